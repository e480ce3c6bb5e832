// The last step of column sums (bias gradients), shared by the fully connected layer and the table lookup.
#pragma once

#include "sg_common.h"

namespace sg {

// out[c] = scale * sum over b of partial[b][c] (float32, in an order that depends on their number alone), in element type `dtype`.
int join_column_sums(const float* partial, int blocks, int64_t cols, float scale, int dtype, void* out, hipStream_t stream);

}  // namespace sg
