// Column sums of a matrix's rows, a bias gradient without the weight's (fgl_column_sums.hip).
#pragma once

#include "fgl_common.hpp"

namespace fgl {

// How a weight gradient's kernel splits its k rows, and in which order a lane adds up: every other of a step's eight rows (fp32 instructions) or eight neighbours of sixteen
struct ColumnSplit {
    int splits;
    int64_t k_per_split;
    bool every_other;
};
ColumnSplit wgrad_column_split(int64_t k, int m, int n, int dtype);   // fgl_wgrad.hip (bf16 rows start on words)
ColumnSplit wgrad8_column_split(int64_t k, int m, int n, int dtype);  // fgl_wgrad8.hip (the same)

size_t column_sums_workspace_bytes(const ColumnSplit& split, int m);
// out[m] = sums over k >= 1 rows of A (row stride lda): the bits that the weight gradient's kernel of that split leaves beside the weight's.  Sizes and pointers have been checked.
int launch_column_sums(const void* a, int64_t lda, int64_t k, int m, int dtype, const ColumnSplit& split, void* out, void* ws, size_t ws_bytes, hipStream_t stream);

}  // namespace fgl
