// The last step of column sums (bias gradients), shared by the fully connected layer and the table lookup: out[c] = scale * sum over b of
// partial[b][c], in an order that depends on the number of partial sums alone.
#pragma once

#include "sg_common.h"

namespace sg {

struct ColumnJoin {
    const float* partial;                // [blocks][cols]
    void* out;                           // [cols]
    int64_t cols;
    int blocks;
    float scale;
};

// 64 columns a workgroup of WAVES waves: sixteen shares of every 16th partial sum, sixteen under way at a time, whichever waves take them.
template <class T, int WAVES> __device__ __forceinline__ void join_columns(const ColumnJoin& p, unsigned block, float* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)block * 64 + lane;
#pragma unroll
    for (int share = wave; share < 16; share += WAVES) {
        float sum = 0.f;
        for (int b = share; b < p.blocks; b += 16 * 16) {
            float v[16];
#pragma unroll
            for (int u = 0; u < 16; u++) v[u] = b + 16 * u < p.blocks && c < p.cols ? p.partial[(int64_t)(b + 16 * u) * p.cols + c] : 0.f;
#pragma unroll
            for (int u = 0; u < 16; u++) sum += v[u];
        }
        part[share * 64 + lane] = sum;
    }
    __syncthreads();
    if (wave == 0 && c < p.cols) {
        float sum = 0.f;
#pragma unroll
        for (int share = 0; share < 16; share++) sum += part[share * 64 + lane];
        ((T*)p.out)[c] = Elem<T>::store(sum * p.scale);
    }
}

}  // namespace sg
