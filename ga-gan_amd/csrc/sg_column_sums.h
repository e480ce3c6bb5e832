// Column sums of a matrix (bias gradients), shared by the fully connected layer and the table lookup.
#pragma once

#include "sg_common.h"

namespace sg {

size_t column_sums_workspace_bytes(int64_t rows, int64_t cols);

// out[c] = scale * sum over r of g[r * ld + c], in g's element type (sums in float32, in an order that depends on the sizes
// alone).  `workspace`: column_sums_workspace_bytes(rows, cols) bytes of 16-byte aligned device memory.
int column_sums(const void* g, int dtype, int64_t rows, int64_t cols, int64_t ld, float scale, void* out, void* workspace, hipStream_t stream);

}  // namespace sg
