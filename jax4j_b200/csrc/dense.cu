// dense.cu -- what a dense layer needs beside the tensor-core product:
// y = act(x . w + bias) + residual for small products, its elementwise part
// for FLOAT64, and the pass over the output gradient.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "rows_sum.cuh"

namespace cg = cooperative_groups;

namespace j4c {

int tc_gemm_act(const float *ah, const float *al, const float *bh, const float *bl, int64_t M, int64_t K, int64_t N,
                const float *bias, int act, const float *residual, float *z, float *y, cudaStream_t s);
bool tc_gemm_supported(int64_t M, int64_t K, int64_t N);

namespace {

// ---- small FLOAT32 products ----------------------------------------------------------
// A product too small for the tensor-core kernel's splits to pay (each operand
// is read and written twice before the first MMA, eight launches in all) runs
// on the CUDA cores in one launch, in FP32 FMAs.  K is cut over a cluster of
// CTAs so that few output tiles still fill the GPU; their partial sums meet
// through distributed shared memory and are added in rank order.
struct Product {
    const float *A, *B, *bias, *residual;
    float *z, *y;  // z may be NULL
    int64_t M, K, N;
    int act;
};

// acc -> y (and z) at row m, column n.
__device__ __forceinline__ void finish(const Product &p, int64_t m, int64_t n, float v) {
    const int64_t at = m * p.N + n;
    if (p.bias) v = __fadd_rn(v, p.bias[n]);
    if (p.z) p.z[at] = v;
    float o[1] = {v};
    act_values(p.act, o);
    p.y[at] = p.residual ? __fadd_rn(o[0], p.residual[at]) : o[0];
}

// Up to 16 rows of x against a weight [K, N], bound by reading the weight: a
// CTA holds 32 V columns, its eight warps take turns along K, a thread V
// columns of MT rows; x comes from shared memory, one value for the warp.
constexpr int kRowsThreads = 256, kRowsK = 256;  // rows of the weight whose x is staged together
template <int MT, int V>
__global__ void __launch_bounds__(kRowsThreads) rows_kernel(const Product p) {
    constexpr int COLS = 32 * V;
    extern __shared__ __align__(16) float smem[];
    float *xs = smem;   // [kRowsK][MT]
    float *sum = smem;  // [8 warps][MT][COLS], then [MT][COLS]: after the last use of xs
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t n0 = (int64_t)(blockIdx.x / ranks) * COLS + lane * V, m0 = (int64_t)blockIdx.y * MT;
    const int64_t k0 = p.K * rank / ranks, k1 = p.K * (rank + 1) / ranks;
    float acc[MT][V];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int v = 0; v < V; v++) acc[m][v] = 0.0f;
    for (int64_t kb = k0; kb < k1; kb += kRowsK) {
        const int len = (int)min((int64_t)kRowsK, k1 - kb);
        __syncthreads();
        for (int e = threadIdx.x; e < MT * len; e += kRowsThreads) {
            const int m = e / len, k = e - m * len;
            xs[k * MT + m] = m0 + m < p.M ? p.A[(m0 + m) * p.K + kb + k] : 0.0f;
        }
        __syncthreads();
        if (n0 < p.N) {  // V divides N
            const float *w = p.B + kb * p.N + n0;
            constexpr int U = 8;  // loads of the weight in flight
            for (int k = warp; k < len; k += 8 * U) {
                float b[U][V];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const float *at = w + (int64_t)(k + 8 * u) * p.N;
                    const bool in = k + 8 * u < len;
                    if constexpr (V == 4) {
                        const float4 t = in ? __ldg(reinterpret_cast<const float4 *>(at)) : float4{0, 0, 0, 0};
                        b[u][0] = t.x, b[u][1] = t.y, b[u][2] = t.z, b[u][3] = t.w;
                    } else if constexpr (V == 2) {
                        const float2 t = in ? __ldg(reinterpret_cast<const float2 *>(at)) : float2{0, 0};
                        b[u][0] = t.x, b[u][1] = t.y;
                    } else {
                        b[u][0] = in ? __ldg(at) : 0.0f;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (k + 8 * u >= len) break;
                    const float *x = xs + (k + 8 * u) * MT;
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int v = 0; v < V; v++) acc[m][v] = fmaf(x[m], b[u][v], acc[m][v]);
                }
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int v = 0; v < V; v++) sum[(warp * MT + m) * COLS + lane * V + v] = acc[m][v];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * COLS; e += kRowsThreads) {
        float v = sum[e];
#pragma unroll
        for (int w = 1; w < 8; w++) v += sum[w * MT * COLS + e];
        sum[e] = v;
    }
    cluster.sync();  // every rank's sums are there
    const int64_t c0 = (int64_t)(blockIdx.x / ranks) * COLS;
    for (int e = rank * kRowsThreads + threadIdx.x; e < MT * COLS; e += ranks * kRowsThreads) {
        const int m = e / COLS, c = e - m * COLS;
        if (m0 + m >= p.M || c0 + c >= p.N) continue;
        float v = 0.0f;
        for (int r = 0; r < ranks; r++) v += *cluster.map_shared_rank(sum + e, r);
        finish(p, m0 + m, c0 + c, v);
    }
    cluster.sync();  // no rank leaves while its sums are read
}

// The general form, op(A) [M, K] . op(B) [K, N] with either operand stored
// transposed: 64 x 64 tiles of 128 threads (8 x 4 results each), K in steps of
// 16 through a ring of three buffers filled by asynchronous copies, two steps
// ahead: a CTA's share of K is a few steps, each bound by the copies' latency.
// Also measured, and no faster at [256,784]x[784,512] (13.4 us) to 1024^3 (81
// us): rings of four and six buffers, 8 x 8 results a thread, and two or four
// shares of K within a CTA.
constexpr int kTM = 64, kTN = 64, kTK = 16, kPitch = 68;  // a row of a buffer: padded, 16-byte multiples
constexpr int kRing = 3, kTileThreads = 128;
struct TileStep {
    float A[kTK][kPitch], B[kTK][kPitch];
};
__device__ __forceinline__ void copy4_async(float *to, const float *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
                 : "memory");
}
template <bool TA, bool TB>
__device__ __forceinline__ void tile_product(const Product &p, int64_t tile_m, int64_t tile_n, TileStep *ring) {
    // the tile's sums take the ring's place once it has been read
    float(*const part)[kTN] = reinterpret_cast<float(*)[kTN]>(ring);
    static_assert(kRing * sizeof(TileStep) >= kTM * kTN * sizeof(float), "the tile's sums take the ring's place");
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int64_t n0 = tile_n * kTN, m0 = tile_m * kTM;
    const int64_t k0 = p.K * rank / ranks, k1 = p.K * (rank + 1) / ranks;
    const int steps = (int)((k1 - k0 + kTK - 1) / kTK);
    // This thread copies eight values of each operand a step: of one stored
    // along K, one K of every eighth row; of one stored across, every second K
    // of a row.  Bit i of the masks: its i-th row (or its row) is in the operand.
    const int am = TA ? tid % kTM : tid / kTK, ak = TA ? tid / kTM : tid % kTK;
    const int bn = TB ? tid / kTK : tid % kTN, bk = TB ? tid % kTK : tid / kTN;
    const float *a = p.A + (TA ? (k0 + ak) * p.M + m0 + am : (m0 + am) * p.K + k0 + ak);
    const float *b = p.B + (TB ? (n0 + bn) * p.K + k0 + bk : (k0 + bk) * p.N + n0 + bn);
    const int64_t a_next = TA ? 2 * p.M : 8 * p.K, b_next = TB ? 8 * p.K : 2 * p.N;  // to the thread's next value
    const int64_t a_step = TA ? kTK * p.M : kTK, b_step = TB ? kTK : kTK * p.N;      // to the next step
    uint32_t a_in = 0, b_in = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        a_in |= (m0 + am + (TA ? 0 : 8 * i) < p.M ? 1u : 0u) << i;
        b_in |= (n0 + bn + (TB ? 8 * i : 0) < p.N ? 1u : 0u) << i;
    }
    auto fetch = [&](int step) {
        if (step < steps) {
            TileStep &to = ring[step % kRing];
            const int left = (int)min((int64_t)kTK, k1 - k0 - (int64_t)step * kTK);  // Ks of this step
            const float *pa = a, *pb = b;
#pragma unroll
            for (int i = 0; i < 8; i++, pa += a_next) {
                const int m = TA ? am : am + 8 * i, k = TA ? ak + 2 * i : ak;
                if ((a_in >> i & 1u) && k < left) copy4_async(&to.A[k][m], pa);
                else to.A[k][m] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++, pb += b_next) {
                const int n = TB ? bn + 8 * i : bn, k = TB ? bk : bk + 2 * i;
                if ((b_in >> i & 1u) && k < left) copy4_async(&to.B[k][n], pb);
                else to.B[k][n] = 0.0f;
            }
            a += a_step, b += b_step;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0.0f;
#pragma unroll
    for (int i = 0; i < kRing - 1; i++) fetch(i);
    for (int step = 0; step < steps; step++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
        __syncthreads();  // this step's copies are everyone's, and the buffer of the step before has been read
        fetch(step + kRing - 1);
        const TileStep &at = ring[step % kRing];
#pragma unroll
        for (int k = 0; k < kTK; k++) {
            const float4 a0 = *reinterpret_cast<const float4 *>(&at.A[k][ty * 8]);
            const float4 a1 = *reinterpret_cast<const float4 *>(&at.A[k][ty * 8 + 4]);
            const float4 b0 = *reinterpret_cast<const float4 *>(&at.B[k][tx * 4]);
            const float av[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w}, bv[4] = {b0.x, b0.y, b0.z, b0.w};
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++)
        *reinterpret_cast<float4 *>(&part[ty * 8 + i][tx * 4]) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    cluster.sync();
    // Rank r finishes rows r, r + ranks, ... of the tile: a thread every second
    // of them in its column, eight at a time so that their residuals are on
    // their way together.  Shares are added in order.
    const int n = tid % kTN, mine = kTM / ranks;
    if (n0 + n < p.N) {
        const float bias = p.bias ? p.bias[n0 + n] : 0.0f;
        for (int i0 = tid / kTN; i0 < mine; i0 += 16) {
            float v[8], res[8];
            int64_t at[8];
            bool in[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int idx = i0 + 2 * i, m = idx * ranks + rank;
                in[i] = idx < mine && m0 + m < p.M;
                at[i] = (m0 + m) * p.N + n0 + n;
                res[i] = p.residual && in[i] ? p.residual[at[i]] : 0.0f;
                v[i] = 0.0f;
                if (in[i])
                    for (int r = 0; r < ranks; r++) v[i] += *cluster.map_shared_rank(&part[m][n], r);
                if (p.bias) v[i] = __fadd_rn(v[i], bias);
            }
            if (p.z) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (in[i]) p.z[at[i]] = v[i];
            }
            act_values(p.act, v);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (in[i]) p.y[at[i]] = p.residual ? __fadd_rn(v[i], res[i]) : v[i];
        }
    }
    cluster.sync();
}

template <bool TA, bool TB>
__global__ void __launch_bounds__(kTileThreads) tile_kernel(const Product p) {
    __shared__ __align__(16) TileStep ring[kRing];
    const int64_t tile = blockIdx.x / cg::this_cluster().num_blocks(), tiles_n = (p.N + kTN - 1) / kTN;
    tile_product<TA, TB>(p, tile / tiles_n, tile % tiles_n, ring);
}

// Two products in one launch, x's gradient dz . w^T and w's x^T . dz: neither
// fills the GPU, and together they cost one launch.
struct TwoProducts {
    Product dx, dw;
    int64_t dx_tiles;
};
__global__ void __launch_bounds__(kTileThreads) two_products_kernel(const TwoProducts p) {
    __shared__ __align__(16) TileStep ring[kRing];
    const int64_t tile = blockIdx.x / cg::this_cluster().num_blocks();
    if (tile < p.dx_tiles) {
        const int64_t tiles_n = (p.dx.N + kTN - 1) / kTN;
        tile_product<false, true>(p.dx, tile / tiles_n, tile % tiles_n, ring);
    } else {
        const int64_t tiles_n = (p.dw.N + kTN - 1) / kTN, t = tile - p.dx_tiles;
        tile_product<true, false>(p.dw, t / tiles_n, t % tiles_n, ring);
    }
}

template <typename Kernel, typename Arg>
int launch_cluster(Kernel kernel, dim3 grid, int threads, size_t smem, int ranks, const Arg &p, cudaStream_t s) {
    if (smem > 48 * 1024)
        J4C_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid.x * ranks, grid.y);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    J4C_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    count_launch();
    return J4C_OK;
}

// CTAs along K: two output tiles' worth of CTAs an SM where K has 64 for each.
int ranks_for(int64_t tiles, int64_t K, int64_t most_k) {
    int ranks = 1;
    while (ranks < 8 && tiles * ranks < 2 * sm_count() && K >= 2 * ranks * most_k) ranks *= 2;
    return ranks;
}

template <int MT, int V>
int launch_rows(const Product &p, cudaStream_t s) {
    constexpr size_t smem = std::max<size_t>(8 * MT * 32 * V, kRowsK * MT) * sizeof(float);
    const dim3 grid((unsigned)ceil_div(p.N, 32 * V), (unsigned)ceil_div(p.M, MT));
    return launch_cluster(rows_kernel<MT, V>, grid, kRowsThreads, smem, ranks_for((int64_t)grid.x * grid.y, p.K, 64), p, s);
}
template <int V>
int launch_rows_m(const Product &p, cudaStream_t s) {
    if (p.M == 1) return launch_rows<1, V>(p, s);
    if (p.M == 2) return launch_rows<2, V>(p, s);
    if (p.M <= 4) return launch_rows<4, V>(p, s);
    if (p.M <= 8) return launch_rows<8, V>(p, s);
    return launch_rows<16, V>(p, s);
}

int64_t tiles_of(const Product &p) { return ceil_div(p.M, kTM) * ceil_div(p.N, kTN); }

// ranks: CTAs along K of the tile form (0: by the product's own size).
int small_product(const Product &p, int ta, int tb, int ranks, cudaStream_t s) {
    if (p.M <= 16 && !ta && !tb) {
        // the widest loads that still give every SM a strip of columns
        auto fits = [&](int v) {
            return p.N % v == 0 && reinterpret_cast<uintptr_t>(p.B) % (4 * v) == 0 && p.N / (32 * v) * 8 >= sm_count();
        };
        return fits(4) ? launch_rows_m<4>(p, s) : fits(2) ? launch_rows_m<2>(p, s) : launch_rows_m<1>(p, s);
    }
    const int64_t tiles = tiles_of(p);
    if (!ranks) ranks = ranks_for(tiles, p.K, 64);
    auto launch = [&](auto kernel) {
        return launch_cluster(kernel, dim3((unsigned)tiles), kTileThreads, 0, ranks, p, s);
    };
    if (ta) return tb ? launch(tile_kernel<true, true>) : launch(tile_kernel<true, false>);
    return tb ? launch(tile_kernel<false, true>) : launch(tile_kernel<false, false>);
}

// ---- the elementwise part alone (FLOAT64, whose product is the DMMA kernel's) ---------
// y = act(z) + residual with z += bias first; z is written back unless y is z.
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(T *z, int64_t M, int64_t N, const T *__restrict__ bias, int act,
                                                     const T *__restrict__ residual, T *y) {
    const int64_t all = M * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        T v = z[i];
        if (bias) {
            v += bias[i % N];
            if (y != z) z[i] = v;
        }
        T o[1] = {v};
        act_values(act, o);
        y[i] = residual ? o[0] + residual[i] : o[0];
    }
}

// ---- the pass over the output gradient ------------------------------------------------
// dz = dy act'(z) from the pre-activation z, or from the output where it tells
// (relu, tanh, sigmoid without a residual: 4 B per value less kept); the column
// sums of dz (the bias's gradient) and dz's line words, which the products'
// splits take instead of a max pass: 12 B per FLOAT32 value, one pass.  A CTA
// holds 256 columns of a group of rows, a warp every eighth row, a lane eight
// columns; a warp adds its rows in order and the warps' and groups' sums are
// added in order, so the bias's gradient repeats bit for bit.
template <typename T>
__device__ __forceinline__ void slopes_of_output(int act, const T (&h)[8], T (&d)[8]) {
    switch (act) {
    case J4C_ACT_RELU:
#pragma unroll
        for (int i = 0; i < 8; i++) d[i] = h[i] > T(0) ? d[i] : T(0);
        break;
    case J4C_ACT_TANH:
#pragma unroll
        for (int i = 0; i < 8; i++) d[i] *= T(1) - h[i] * h[i];
        break;
    case J4C_ACT_SIGMOID:
#pragma unroll
        for (int i = 0; i < 8; i++) d[i] *= h[i] * (T(1) - h[i]);
        break;
    default: break;
    }
}

template <typename T>
struct GradArgs {
    const T *dy, *u;  // u: z, or the output; NULL for no activation
    T *dz, *sums;     // sums [groups][N]; each may be NULL
    uint32_t *lines;  // FLOAT32: rows, columns, flag (zeroed), or NULL
    int64_t M, N, groups;
    int act, from_output;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};

// CLUSTER: the groups of rows of a strip are one cluster, which adds its column
// sums through distributed shared memory: a.sums is the bias's gradient itself.
template <typename T, int V, bool CLUSTER>
__global__ void __launch_bounds__(256) dense_grad_kernel(const GradArgs<T> a) {
    __shared__ T sums[8][256];
    __shared__ uint32_t tops[8][256];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t c0 = (int64_t)blockIdx.x * 256, g = blockIdx.y;
    const int64_t r0 = g * a.M / a.groups, r1 = (g + 1) * a.M / a.groups;
    // column i of this lane: V together, 32 V apart
    auto col = [&](int i) { return (i / V) * (32 * V) + lane * V + i % V; };
    T sum[8];
    uint32_t top[8];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = T(0), top[i] = 0;
    constexpr int U = 2;  // rows in flight
    for (int64_t r = r0 + warp; r < r1; r += 8 * U) {
        T d[U][8], u[U][8];
#pragma unroll
        for (int k = 0; k < U; k++) {
#pragma unroll
            for (int i = 0; i < 8; i += V) {
                Vec<T, V> x{}, z{};
                if (r + 8 * k < r1 && c0 + col(i) < a.N) {  // V divides N
                    const int64_t at = (r + 8 * k) * a.N + c0 + col(i);
                    x = *reinterpret_cast<const Vec<T, V> *>(a.dy + at);
                    if (a.u) z = *reinterpret_cast<const Vec<T, V> *>(a.u + at);
                }
#pragma unroll
                for (int e = 0; e < V; e++) d[k][i + e] = x.e[e], u[k][i + e] = z.e[e];
            }
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            if (r + 8 * k >= r1) break;  // the whole warp
            if (a.from_output) slopes_of_output(a.act, u[k], d[k]);
            else act_slopes(a.act, u[k], d[k]);
            uint32_t rtop = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                sum[i] += d[k][i];
                if constexpr (sizeof(T) == 4) {
                    const uint32_t b = __float_as_uint((float)d[k][i]) & 0x7FFFFFFFu;
                    const bool fin = b < 0x7F800000u;
                    bad |= !fin && c0 + col(i) < a.N;
                    top[i] = max(top[i], fin ? b : 0u);
                    rtop = max(rtop, fin ? b : 0u);
                }
            }
            if (a.dz) {
#pragma unroll
                for (int i = 0; i < 8; i += V)
                    if (c0 + col(i) < a.N) {
                        Vec<T, V> x;
#pragma unroll
                        for (int e = 0; e < V; e++) x.e[e] = d[k][i + e];
                        *reinterpret_cast<Vec<T, V> *>(a.dz + (r + 8 * k) * a.N + c0 + col(i)) = x;
                    }
            }
            if (sizeof(T) == 4 && a.lines) {
                rtop = __reduce_max_sync(0xffffffffu, rtop);
                if (lane == 0 && rtop) atomicMax(a.lines + r + 8 * k, rtop);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        sums[warp][col(i)] = sum[i];
        tops[warp][col(i)] = top[i];
    }
    __syncthreads();
    const int c = threadIdx.x;
    if (c0 + c < a.N) {
        T v = sums[0][c];
        uint32_t m = tops[0][c];
#pragma unroll
        for (int w = 1; w < 8; w++) v += sums[w][c], m = max(m, tops[w][c]);
        if (CLUSTER) sums[0][c] = v;
        else if (a.sums) a.sums[g * a.N + c0 + c] = v;
        if (a.lines && m) atomicMax(a.lines + a.M + c0 + c, m);
    }
    if constexpr (CLUSTER) {
        const cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        // rank r takes columns r, r + ranks, ...
        const int ranks = cluster.num_blocks();
        for (int cc = cluster.block_rank() + threadIdx.x * ranks; cc < 256 && c0 + cc < a.N; cc += 256 * ranks) {
            T v = T(0);
            for (int r = 0; r < ranks; r++) v += *cluster.map_shared_rank(&sums[0][cc], r);
            a.sums[c0 + cc] = v;
        }
        cluster.sync();
    }
    if (a.lines && __any_sync(0xffffffffu, bad) && lane == 0) atomicOr(a.lines + a.M + a.N, 1u);
}

// Groups of rows: four CTAs an SM, at least 32 rows each; where eight are
// enough for that, or for 512 rows, they are a cluster and need no second launch.
int64_t grad_groups(int64_t M, int64_t N) {
    const int64_t groups = std::max<int64_t>(
        1, std::min(ceil_div(M, 32), ceil_div((int64_t)sm_count() * 4, ceil_div(N, 256))));
    return M <= 512 ? std::min<int64_t>(groups, 8) : groups;
}

template <typename T>
int dense_grad(int64_t M, int64_t N, const T *dy, const T *u, int act, int from_output, T *dz, T *dbias, uint32_t *lines,
               void *ws, cudaStream_t s) {
    const int64_t groups = grad_groups(M, N);
    if (lines) J4C_CUDA(cudaMemsetAsync(lines, 0, (size_t)(M + N + 1) * sizeof(uint32_t), s));
    const bool cluster = dbias && groups > 1 && groups <= 8;
    T *sums = !dbias ? nullptr : groups <= 8 ? dbias : static_cast<T *>(ws);
    const GradArgs<T> a{dy, act == J4C_ACT_NONE ? nullptr : u, dz, sums, lines, M, N, groups, act, from_output};
    constexpr int W = 16 / sizeof(T);
    auto fits = [&](int v) {
        auto ok = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (v * sizeof(T)) == 0; };
        return N % v == 0 && ok(dy) && ok(u) && ok(dz);
    };
    auto launch = [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)ceil_div(N, 256), (unsigned)groups);
        cfg.blockDim = dim3(256);
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
        attr[0].val.clusterDim.y = (unsigned)groups;
        cfg.attrs = attr;
        cfg.numAttrs = cluster ? 1 : 0;
        J4C_CUDA(cluster ? cudaLaunchKernelEx(&cfg, dense_grad_kernel<T, V, true>, a)
                         : cudaLaunchKernelEx(&cfg, dense_grad_kernel<T, V, false>, a));
        count_launch();
        return (int)J4C_OK;
    };
    if (int rc = fits(W)   ? launch(std::integral_constant<int, W>{})
                 : fits(2) ? launch(std::integral_constant<int, 2>{})
                           : launch(std::integral_constant<int, 1>{}))
        return rc;
    if (dbias && groups > 8) {
        sum_rows_kernel<T><<<(unsigned)ceil_div(N, 32), 1024, 0, s>>>(sums, groups, N, dbias, nullptr);
        J4C_LAUNCH_CHECK("sum_rows_kernel");
    }
    return J4C_OK;
}

}  // namespace
}  // namespace j4c

using namespace j4c;

// More tiles (eight CTAs each) than a grid takes.
static bool too_many(int64_t M, int64_t N) {
    return M >= (1ll << 40) || N >= (1ll << 33) || ceil_div(M, kTM) * ceil_div(N, 32) >= (1ll << 27);
}

extern "C" {

int j4c_dot_act(const float *a, const float *b, int64_t M, int64_t K, int64_t N, int trans_a, int trans_b,
                const float *bias, int act, const float *residual, float *z, float *y, j4c_stream stream) {
    J4C_REQUIRE(M >= 0 && K >= 0 && N >= 0, "j4c_dot_act: negative dimension");
    J4C_REQUIRE(act_known(act), "j4c_dot_act: unknown activation %d", act);
    if (M == 0 || N == 0) return J4C_OK;
    J4C_REQUIRE(y && (K == 0 || (a && b)), "j4c_dot_act: NULL pointer");
    if (too_many(M, N))
        return set_error(J4C_E_UNSUPPORTED, "j4c_dot_act: %lld x %lld results are too many", (long long)M, (long long)N);
    return small_product(Product{a, b, bias, residual, z, y, M, K, N, act}, trans_a, trans_b, 0, as_stream(stream));
}

int j4c_dot_split_act(const float *a_hi, const float *a_lo, const float *bt_hi, const float *bt_lo, int64_t M, int64_t K,
                      int64_t N, const float *bias, int act, const float *residual, float *z, float *y,
                      j4c_stream stream) {
    J4C_REQUIRE(M >= 0 && K >= 0 && N >= 0, "j4c_dot_split_act: negative dimension");
    J4C_REQUIRE(act_known(act), "j4c_dot_split_act: unknown activation %d", act);
    if (M == 0 || N == 0) return J4C_OK;
    J4C_REQUIRE(y && a_hi && a_lo && bt_hi && bt_lo, "j4c_dot_split_act: NULL pointer");
    J4C_REQUIRE(K > 0, "j4c_dot_split_act: K = 0");
    if (!tc_gemm_supported(M, K, N))
        return set_error(J4C_E_UNSUPPORTED, "j4c_dot_split_act: shape %lld x %lld x %lld is too large", (long long)M,
                         (long long)K, (long long)N);
    return tc_gemm_act(a_hi, a_lo, bt_hi, bt_lo, M, K, N, bias, act, residual, z, y, as_stream(stream));
}

int j4c_dense_finish(int dtype, void *z, int64_t M, int64_t N, const void *bias, int act, const void *residual, void *y,
                     j4c_stream stream) {
    J4C_REQUIRE(dtype == J4C_FLOAT32 || dtype == J4C_FLOAT64, "j4c_dense_finish requires FLOAT32 or FLOAT64 arrays, got %s",
                dtype_name(dtype));
    J4C_REQUIRE(M >= 0 && N >= 0, "j4c_dense_finish: negative dimension");
    J4C_REQUIRE(act_known(act), "j4c_dense_finish: unknown activation %d", act);
    if (M == 0 || N == 0) return J4C_OK;
    J4C_REQUIRE(z && y, "j4c_dense_finish: NULL pointer");
    auto run = [&](auto t) {
        using T = decltype(t);
        finish_kernel<T><<<grid_for(M * N, 256), 256, 0, as_stream(stream)>>>((T *)z, M, N, (const T *)bias, act,
                                                                              (const T *)residual, (T *)y);
        J4C_LAUNCH_CHECK("finish_kernel");
        return (int)J4C_OK;
    };
    return dtype == J4C_FLOAT64 ? run(0.0) : run(0.0f);
}

size_t j4c_dense_grad_workspace(int dtype, int64_t M, int64_t N) {
    if (M <= 0 || N <= 0) return 0;
    const int64_t groups = grad_groups(M, N);
    return groups <= 8 ? 0 : (size_t)(groups * N) * dtype_size(dtype);
}

int j4c_dense_grad(int dtype, int64_t M, int64_t N, const void *dy, const void *u, int act, int from_output, void *dz,
                   void *dbias, uint32_t *lines, void *ws, size_t ws_bytes, j4c_stream stream) {
    J4C_REQUIRE(dtype == J4C_FLOAT32 || dtype == J4C_FLOAT64, "j4c_dense_grad requires FLOAT32 or FLOAT64 arrays, got %s",
                dtype_name(dtype));
    J4C_REQUIRE(M >= 0 && N >= 0, "j4c_dense_grad: negative dimension");
    J4C_REQUIRE(act_known(act), "j4c_dense_grad: unknown activation %d", act);
    J4C_REQUIRE(!from_output || act <= J4C_ACT_SIGMOID, "j4c_dense_grad: the output of silu and gelu does not tell the slope");
    J4C_REQUIRE(!lines || dtype == J4C_FLOAT32, "j4c_dense_grad: line words are for FLOAT32");
    cudaStream_t s = as_stream(stream);
    if (M == 0 || N == 0) {
        if (dbias && N) J4C_CUDA(cudaMemsetAsync(dbias, 0, (size_t)N * dtype_size(dtype), s));
        if (lines) J4C_CUDA(cudaMemsetAsync(lines, 0, (size_t)(M + N + 1) * sizeof(uint32_t), s));
        return J4C_OK;
    }
    J4C_REQUIRE(dy && (u || act == J4C_ACT_NONE) && (dz || act == J4C_ACT_NONE), "j4c_dense_grad: NULL pointer");
    const size_t need = dbias ? j4c_dense_grad_workspace(dtype, M, N) : 0;
    J4C_REQUIRE(need == 0 || (ws && aligned16(ws) && ws_bytes >= need), "j4c_dense_grad: needs %zu bytes of workspace", need);
    if (ceil_div(N, 256) >= (1ll << 31))
        return set_error(J4C_E_UNSUPPORTED, "j4c_dense_grad: %lld columns are too many", (long long)N);
    auto run = [&](auto t) {
        using T = decltype(t);
        return dense_grad<T>(M, N, (const T *)dy, (const T *)u, act, from_output, (T *)dz, (T *)dbias, lines, ws, s);
    };
    return dtype == J4C_FLOAT64 ? run(0.0) : run(0.0f);
}

int j4c_dense_backward(const float *x, const float *w, int64_t M, int64_t K, int64_t N, const float *dy, const float *u,
                       int act, int from_output, float *dz, float *dx, float *dw, float *dbias, void *ws, size_t ws_bytes,
                       j4c_stream stream) {
    J4C_REQUIRE(M >= 0 && K >= 0 && N >= 0, "j4c_dense_backward: negative dimension");
    J4C_REQUIRE(dx || dw || K == 0 || (M == 0 && N == 0),
                "j4c_dense_backward: neither product is wanted (j4c_dense_grad gives dbias alone)");
    const float *d = dy;
    if (dbias || act != J4C_ACT_NONE) {
        if (int rc = j4c_dense_grad(J4C_FLOAT32, M, N, dy, u, act, from_output, dz, dbias, nullptr, ws, ws_bytes, stream))
            return rc;
        if (act != J4C_ACT_NONE) d = dz;
    }
    const bool dx_too = dx && M && K, dw_too = dw && K && N;
    J4C_REQUIRE((!dx_too || N == 0 || (d && w)) && (!dw_too || M == 0 || (d && x)), "j4c_dense_backward: NULL pointer");
    const Product px{d, w, nullptr, nullptr, nullptr, dx, M, N, K, J4C_ACT_NONE};
    const Product pw{x, d, nullptr, nullptr, nullptr, dw, K, M, N, J4C_ACT_NONE};
    if ((dx_too && too_many(M, K)) || (dw_too && too_many(K, N)))
        return set_error(J4C_E_UNSUPPORTED, "j4c_dense_backward: %lld x %lld x %lld is too large", (long long)M,
                         (long long)K, (long long)N);
    cudaStream_t s = as_stream(stream);
    // the same cut of K whether one product is wanted or both: the same bits
    const int64_t tx = tiles_of(px), tw = tiles_of(pw);
    const int ranks = ranks_for(tx + tw, std::max(M, N), 64);
    if (dx_too && dw_too)
        return launch_cluster(two_products_kernel, dim3((unsigned)(tx + tw)), kTileThreads, 0, ranks,
                              TwoProducts{px, pw, tx}, s);
    if (dx_too) return small_product(px, 0, 1, ranks, s);
    return dw_too ? small_product(pw, 1, 0, ranks, s) : (int)J4C_OK;
}

}  // extern "C"
