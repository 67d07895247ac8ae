// rows_sum.cuh -- sums over the rows of an array, in a fixed order.
#pragma once

#include "common.cuh"

namespace j4c {
namespace {

// Additions in a row that a thread makes at most, where a sum may be long.  Each
// in FP32 loses up to half a step of the running sum, so the error grows with the
// row; cut rows' sums are added after them.
constexpr int64_t kMaxTerms = 1024;

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The sums over the rows r < rows of an array [rows, cols], 32 columns a CTA and
// 32 lanes of rows (1024 threads): lane 0 of warp w gets that of column
// 32 blockIdx.x + w.  Every thread of the CTA comes along.
template <typename T>
__device__ __forceinline__ T column_sum(const T *__restrict__ in, int64_t rows, int64_t cols) {
    __shared__ T part[32][33];
    const int lane = threadIdx.x % 32, rl = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
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
    return warp_sum(part[lane][rl]);
}

// out[j] = sum over r of in[r, j], r < rows, for two [rows, cols] arrays back
// to back (blockIdx.y; one array: a grid of one row); either output may be NULL.
template <typename T>
__global__ void __launch_bounds__(1024) sum_rows_kernel(const T *__restrict__ in, int64_t rows, int64_t cols, T *out0,
                                                        T *out1) {
    T *out = blockIdx.y ? out1 : out0;
    if (!out) return;
    const T v = column_sum(in + blockIdx.y * rows * cols, rows, cols);
    const int64_t mine = (int64_t)blockIdx.x * 32 + threadIdx.x / 32;
    if (threadIdx.x % 32 == 0 && mine < cols) out[mine] = v;
}

}  // namespace
}  // namespace j4c
