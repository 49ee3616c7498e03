// The operators of fastgl_autograd.cpp in the host module (fastgl_host.cpp).
#pragma once

#include <torch/extension.h>

void bind_recorded_operators(py::module& m);
