// The weight gradient of a layer whose input rows are held in 8 bits (fgl_wgrad8.hip).
#pragma once

#include "fgl_common.hpp"

namespace fgl {

// Steps a column of rows: what a lane loads of them, eight at a time, exists also for the last rows.
inline int64_t w8_step_ld(int64_t n_rows) { return (n_rows + 15) / 16 * 16; }

size_t wgrad8_workspace_bytes(int64_t k, int m, int n, int dtype);
// C[m, n] (row stride ldc) = A[k, m]^T (codes times steps)[k, n], steps w8_step_ld(k) apart; sum_a (may be null) = A's column sums.  Sizes and pointers have been checked.
int launch_wgrad8(const void* a, int64_t lda, const uint8_t* codes, const uint8_t* steps, int64_t k, int m, int n, int dtype, void* c, int64_t ldc, void* sum_a, void* ws,
                  size_t ws_bytes, hipStream_t stream);

}  // namespace fgl
