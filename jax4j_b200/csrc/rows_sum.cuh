// rows_sum.cuh -- sums over the rows of an array, in a fixed order.
#pragma once

#include "common.cuh"

namespace j4c {
namespace {

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// out[j] = sum over r of in[r, j], r < rows, for two [rows, cols] arrays back
// to back (blockIdx.y; one array: a grid of one row): 32 columns and 32 lanes
// of rows a CTA; either output may be NULL.
template <typename T>
__global__ void __launch_bounds__(1024) sum_rows_kernel(const T *__restrict__ in, int64_t rows, int64_t cols, T *out0,
                                                        T *out1) {
    __shared__ T part[32][33];
    const int lane = threadIdx.x % 32, rl = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    T *out = blockIdx.y ? out1 : out0;
    if (!out) return;
    in += blockIdx.y * rows * cols;
    T v = T(0);
    if (c < cols) {
        int64_t r = rl;
        for (; r + 96 < rows; r += 128) {
            T w[4];
#pragma unroll
            for (int u = 0; u < 4; u++) w[u] = in[(r + 32 * u) * cols + c];
            v += (w[0] + w[1]) + (w[2] + w[3]);
        }
        for (; r < rows; r += 32) v += in[r * cols + c];
    }
    part[rl][lane] = v;
    __syncthreads();
    // the warp of a column adds the column's 32 lanes
    v = warp_sum(part[lane][rl]);
    const int64_t mine = (int64_t)blockIdx.x * 32 + rl;
    if (lane == 0 && mine < cols) out[mine] = v;
}

}  // namespace
}  // namespace j4c
