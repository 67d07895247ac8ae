// dense.cu -- what a dense layer needs beside the tensor-core product:
// y = act(x . w + bias) + residual for small products and for FLOAT64, and the
// pass over the output gradient.
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

// ---- products straight from the arrays --------------------------------------------------------
// A FLOAT32 product too small for the tcgen05 kernel's splits to pay (before the
// first MMA the operands are read, once or twice, and written as halves; four
// launches in all) runs here in one launch of FP32 FMAs, and every FLOAT64 product with the
// FP64 tensor instruction (tcgen05 has no FP64 kind).  K is cut over a cluster
// of CTAs so that few output tiles still fill the GPU; their partial sums meet
// through distributed shared memory and are added in rank order.  A sum too long
// for one cluster is cut into parts first (gridDim.z, parts_for): each part's
// results go to its own [M, N] of y, and join_kernel adds the parts in order and
// applies the rest.
template <typename T>
struct Product {
    const T *A, *B, *bias, *residual;
    T *z, *y;  // z may be NULL
    int64_t M, K, N;
    int act;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};

// acc -> y (and z) at row m, column n.
template <typename T>
__device__ __forceinline__ void finish(const Product<T> &p, T *y, int64_t m, int64_t n, T v) {
    const int64_t at = m * p.N + n;
    if (p.bias) v = r_add(v, p.bias[n]);
    if (p.z) p.z[at] = v;
    T o[1] = {v};
    act_values(p.act, o);
    y[at] = p.residual ? r_add(o[0], p.residual[at]) : o[0];
}

// The sums over K of the calling CTA: [from, to) of its part and its rank in the
// cluster; and its part's results.
template <typename T>
struct Share {
    int64_t from, to;
    T *y;
    __device__ __forceinline__ Share(const Product<T> &p, int rank, int ranks) {
        const int64_t at = (int64_t)blockIdx.z * ranks + rank, all = (int64_t)gridDim.z * ranks;
        from = p.K * at / all;
        to = p.K * (at + 1) / all;
        y = p.y + blockIdx.z * p.M * p.N;
    }
};

template <typename T>
__global__ void __launch_bounds__(1024) join_kernel(const Product<T> p, const T *__restrict__ sums, int64_t parts) {
    const T v = column_sum(sums, parts, p.M * p.N);
    const int64_t e = (int64_t)blockIdx.x * 32 + threadIdx.x / 32;
    if (threadIdx.x % 32 == 0 && e < p.M * p.N) finish(p, p.y, e / p.N, e % p.N, v);
}

// Up to 16 rows of x against a weight [K, N], bound by reading the weight: a
// CTA holds 32 V columns, its eight warps take turns along K, a thread V
// columns of MT rows; x comes from shared memory, one value for the warp.
constexpr int kRowsThreads = 256, kRowsK = 256;  // rows of the weight whose x is staged together
template <typename T, int MT, int V>
__global__ void __launch_bounds__(kRowsThreads) rows_kernel(const Product<T> p) {
    constexpr int COLS = 32 * V;
    extern __shared__ __align__(16) unsigned char smem[];
    T *xs = reinterpret_cast<T *>(smem);   // [kRowsK][MT]
    T *sum = reinterpret_cast<T *>(smem);  // [8 warps][MT][COLS], then [MT][COLS]: after the last use of xs
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t n0 = (int64_t)(blockIdx.x / ranks) * COLS + lane * V, m0 = (int64_t)blockIdx.y * MT;
    const Share<T> share(p, rank, ranks);
    const int64_t k0 = share.from, k1 = share.to;
    T acc[MT][V];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int v = 0; v < V; v++) acc[m][v] = T(0);
    for (int64_t kb = k0; kb < k1; kb += kRowsK) {
        const int len = (int)min((int64_t)kRowsK, k1 - kb);
        __syncthreads();
        for (int e = threadIdx.x; e < MT * len; e += kRowsThreads) {
            const int m = e / len, k = e - m * len;
            xs[k * MT + m] = m0 + m < p.M ? p.A[(m0 + m) * p.K + kb + k] : T(0);
        }
        __syncthreads();
        if (n0 < p.N) {  // V divides N
            const T *w = p.B + kb * p.N + n0;
            constexpr int U = 8;  // loads of the weight in flight
            for (int k = warp; k < len; k += 8 * U) {
                Vec<T, V> b[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const T *at = w + (int64_t)(k + 8 * u) * p.N;
                    if (k + 8 * u < len) b[u] = *reinterpret_cast<const Vec<T, V> *>(at);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (k + 8 * u >= len) break;
                    const T *x = xs + (k + 8 * u) * MT;
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int v = 0; v < V; v++) acc[m][v] = fma(x[m], b[u].e[v], acc[m][v]);
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
        T v = sum[e];
#pragma unroll
        for (int w = 1; w < 8; w++) v += sum[w * MT * COLS + e];
        sum[e] = v;
    }
    cluster.sync();  // every rank's sums are there
    const int64_t c0 = (int64_t)(blockIdx.x / ranks) * COLS;
    for (int e = rank * kRowsThreads + threadIdx.x; e < MT * COLS; e += ranks * kRowsThreads) {
        const int m = e / COLS, c = e - m * COLS;
        if (m0 + m >= p.M || c0 + c >= p.N) continue;
        T v = T(0);
        for (int r = 0; r < ranks; r++) v += *cluster.map_shared_rank(sum + e, r);
        finish(p, share.y, m0 + m, c0 + c, v);
    }
    cluster.sync();  // no rank leaves while its sums are read
}

// The general form, op(A) [M, K] . op(B) [K, N] with either operand stored
// transposed: 64 x 64 tiles of 128 threads, K in steps of 16 (FLOAT64: 8) through
// a ring of three buffers (four) filled by asynchronous copies, two steps (three)
// ahead: a CTA's share of K is a few steps, each bound by the copies' latency.
// FLOAT32: 8 x 4 results a thread.  FLOAT64: a warp has a quarter of the tile as
// 4 x 4 tiles of m8n8k4 (A element: row lane / 4, k lane % 4; B: k lane % 4,
// column lane / 4; results: row lane / 4, columns 2 (lane % 4) and the next).
// FLOAT32 [256,784]x[784,512] takes 18 us, [1024,1024]x[1024,512] 47; FLOAT64 18
// and, at 2048^3, 592 us (29 TFLOP/s).  Also measured, and no faster in FLOAT32:
// rings of four and six buffers, 8 x 8 results a thread, and two or four shares
// of K within a CTA; in FLOAT64 FMAs instead of the tensor instruction: 22 and
// 1021 us.
constexpr int kTM = 64, kTN = 64, kPitch = 68;  // kPitch: a row of a buffer, padded, 16-byte multiples
constexpr int kTileThreads = 128;
template <typename T>
constexpr int kTK = sizeof(T) == 8 ? 8 : 16;
template <typename T>
constexpr int kRing = sizeof(T) == 8 ? 4 : 3;
template <typename T>
struct alignas(16) TileStep {
    T A[kTK<T>][kPitch], B[kTK<T>][kPitch];
};
template <typename T>
__device__ __forceinline__ void copy_async(T *to, const T *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from),
                 "n"(sizeof(T))
                 : "memory");
}
__device__ __forceinline__ void mma_8x8x4(double &d0, double &d1, double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                 : "+d"(d0), "+d"(d1)
                 : "d"(a), "d"(b));
}
template <typename T, bool TA, bool TB>
__device__ __forceinline__ void tile_product(const Product<T> &p, int64_t tile_m, int64_t tile_n, TileStep<T> *ring) {
    constexpr int TK = kTK<T>, RING = kRing<T>;
    constexpr int PER = kTM * TK / kTileThreads, ROWS = kTileThreads / TK;  // values a thread copies of an operand
    // the tile's sums take the ring's place once it has been read
    T(*const part)[kTN] = reinterpret_cast<T(*)[kTN]>(ring);
    static_assert(RING * sizeof(TileStep<T>) >= kTM * kTN * sizeof(T), "the tile's sums take the ring's place");
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int64_t n0 = tile_n * kTN, m0 = tile_m * kTM;
    const Share<T> share(p, rank, ranks);
    const int64_t k0 = share.from, k1 = share.to;
    const int steps = (int)((k1 - k0 + TK - 1) / TK);
    // This thread copies PER values of each operand a step: of one stored along
    // K, one K of every ROWS-th row; of one stored across, every second K of a
    // row.  Bit i of the masks: its i-th row (or its row) is in the operand.
    const int am = TA ? tid % kTM : tid / TK, ak = TA ? tid / kTM : tid % TK;
    const int bn = TB ? tid / TK : tid % kTN, bk = TB ? tid % TK : tid / kTN;
    const T *a = p.A + (TA ? (k0 + ak) * p.M + m0 + am : (m0 + am) * p.K + k0 + ak);
    const T *b = p.B + (TB ? (n0 + bn) * p.K + k0 + bk : (k0 + bk) * p.N + n0 + bn);
    const int64_t a_next = TA ? 2 * p.M : ROWS * p.K, b_next = TB ? ROWS * p.K : 2 * p.N;  // to the thread's next value
    const int64_t a_step = TA ? TK * p.M : TK, b_step = TB ? TK : TK * p.N;                // to the next step
    uint32_t a_in = 0, b_in = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        a_in |= (m0 + am + (TA ? 0 : ROWS * i) < p.M ? 1u : 0u) << i;
        b_in |= (n0 + bn + (TB ? ROWS * i : 0) < p.N ? 1u : 0u) << i;
    }
    auto fetch = [&](int step) {
        if (step < steps) {
            TileStep<T> &to = ring[step % RING];
            const int left = (int)min((int64_t)TK, k1 - k0 - (int64_t)step * TK);  // Ks of this step
            const T *pa = a, *pb = b;
#pragma unroll
            for (int i = 0; i < PER; i++, pa += a_next) {
                const int m = TA ? am : am + ROWS * i, k = TA ? ak + 2 * i : ak;
                if ((a_in >> i & 1u) && k < left) copy_async(&to.A[k][m], pa);
                else to.A[k][m] = T(0);
            }
#pragma unroll
            for (int i = 0; i < PER; i++, pb += b_next) {
                const int n = TB ? bn + ROWS * i : bn, k = TB ? bk : bk + 2 * i;
                if ((b_in >> i & 1u) && k < left) copy_async(&to.B[k][n], pb);
                else to.B[k][n] = T(0);
            }
            a += a_step, b += b_step;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    constexpr bool MMA = sizeof(T) == 8;
    T acc[8][4];  // with MMA: tile (i, j) of 8 x 8 is acc[2 i + j / 2][2 (j % 2) ..]
    const int fr = tid % 32 / 4, fk = tid % 4, wm = tid / 64 * 32, wn = tid / 32 % 2 * 32;
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = T(0);
#pragma unroll
    for (int i = 0; i < RING - 1; i++) fetch(i);
    for (int step = 0; step < steps; step++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
        __syncthreads();  // this step's copies are everyone's, and the buffer of the step before has been read
        fetch(step + RING - 1);
        const TileStep<T> &at = ring[step % RING];
        if constexpr (MMA) {
#pragma unroll
            for (int k = 0; k < TK; k += 4) {
                T av[4], bv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) av[i] = at.A[k + fk][wm + i * 8 + fr], bv[i] = at.B[k + fk][wn + i * 8 + fr];
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        mma_8x8x4(acc[2 * i + j / 2][j % 2 * 2], acc[2 * i + j / 2][j % 2 * 2 + 1], av[i], bv[j]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < TK; k++) {
                Vec<T, 4> av[2];
                av[0] = *reinterpret_cast<const Vec<T, 4> *>(&at.A[k][ty * 8]);
                av[1] = *reinterpret_cast<const Vec<T, 4> *>(&at.A[k][ty * 8 + 4]);
                const Vec<T, 4> bv = *reinterpret_cast<const Vec<T, 4> *>(&at.B[k][tx * 4]);
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][j] = fma(av[i / 4].e[i % 4], bv.e[j], acc[i][j]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (MMA) {
#pragma unroll
            for (int j = 0; j < 4; j += 2)
                *reinterpret_cast<Vec<T, 2> *>(&part[wm + i / 2 * 8 + fr][wn + (i % 2 * 2 + j / 2) * 8 + 2 * fk]) =
                    Vec<T, 2>{acc[i][j], acc[i][j + 1]};
        } else {
            *reinterpret_cast<Vec<T, 4> *>(&part[ty * 8 + i][tx * 4]) = Vec<T, 4>{acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
        }
    }
    cluster.sync();
    // Rank r finishes rows r, r + ranks, ... of the tile: a thread every second
    // of them in its column, eight at a time so that their residuals are on
    // their way together.  Shares are added in order.
    const int n = tid % kTN, mine = kTM / ranks;
    if (n0 + n < p.N) {
        const T bias = p.bias ? p.bias[n0 + n] : T(0);
        for (int i0 = tid / kTN; i0 < mine; i0 += 16) {
            T v[8], res[8];
            int64_t at[8];
            bool in[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int idx = i0 + 2 * i, m = idx * ranks + rank;
                in[i] = idx < mine && m0 + m < p.M;
                at[i] = (m0 + m) * p.N + n0 + n;
                res[i] = p.residual && in[i] ? p.residual[at[i]] : T(0);
                v[i] = T(0);
                if (in[i])
                    for (int r = 0; r < ranks; r++) v[i] += *cluster.map_shared_rank(&part[m][n], r);
                if (p.bias) v[i] = r_add(v[i], bias);
            }
            if (p.z) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (in[i]) p.z[at[i]] = v[i];
            }
            act_values(p.act, v);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (in[i]) share.y[at[i]] = p.residual ? r_add(v[i], res[i]) : v[i];
        }
    }
    cluster.sync();
}

template <typename T, bool TA, bool TB>
__global__ void __launch_bounds__(kTileThreads) tile_kernel(const Product<T> p) {
    __shared__ TileStep<T> ring[kRing<T>];
    const int64_t tile = blockIdx.x / cg::this_cluster().num_blocks(), tiles_n = (p.N + kTN - 1) / kTN;
    tile_product<T, TA, TB>(p, tile / tiles_n, tile % tiles_n, ring);
}

// Two products in one launch, x's gradient dz . w^T and w's x^T . dz: neither
// fills the GPU, and together they cost one launch.
template <typename T>
struct TwoProducts {
    Product<T> dx, dw;
    int64_t dx_tiles;
};
template <typename T>
__global__ void __launch_bounds__(kTileThreads) two_products_kernel(const TwoProducts<T> p) {
    __shared__ TileStep<T> ring[kRing<T>];
    const int64_t tile = blockIdx.x / cg::this_cluster().num_blocks();
    if (tile < p.dx_tiles) {
        const int64_t tiles_n = (p.dx.N + kTN - 1) / kTN;
        tile_product<T, false, true>(p.dx, tile / tiles_n, tile % tiles_n, ring);
    } else {
        const int64_t tiles_n = (p.dw.N + kTN - 1) / kTN, t = tile - p.dx_tiles;
        tile_product<T, true, false>(p.dw, t / tiles_n, t % tiles_n, ring);
    }
}

template <typename Kernel, typename Arg>
int launch_cluster(Kernel kernel, dim3 grid, int threads, size_t smem, int ranks, const Arg &p, cudaStream_t s) {
    if (smem > 48 * 1024)
        J4C_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (ranks > 8) J4C_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid.x * ranks, grid.y, grid.z);
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

// CTAs along K: two output tiles' worth of CTAs an SM where K has 64 (FLOAT64:
// 32) for each; clusters of 16 only where few of them are wanted (64 rows of
// [4096,512] 41 -> 29 us, but [256,784]x[784,512] FLOAT64 15 -> 22 us).
template <typename T>
int ranks_for(int64_t tiles, int64_t K) {
    int ranks = 1;
    while (ranks < 16 && tiles * ranks < (ranks < 8 ? 2 : 1) * sm_count() && K >= 2 * ranks * (256 / (int)sizeof(T))) ranks *= 2;
    return ranks;
}

// Parts of a sum of K terms whose `ctas` CTAs have `adders` threads after one
// another along K: so many that no thread adds more than kMaxTerms of them in a
// row.  The weight's gradient of [4000000,8]x[8,8], values of one sign, came out
// 1.4e-5 off from the 16 CTAs of one cluster (250000 terms a thread) and 8e-8 in
// parts, and forward and gradients take 3.1 ms instead of 13.6.  FLOAT64 has the
// digits to spare; there parts only fill idle SMs.
template <typename T>
int64_t parts_for(int64_t ctas, int64_t adders, int64_t K) {
    int64_t parts = std::min<int64_t>(ceil_div(K, adders * kMaxTerms), 65535);
    if (sizeof(T) == 8) parts = std::min(parts, 2 * sm_count() / std::max<int64_t>(ctas, 1));
    return std::max<int64_t>(parts, 1);
}

template <typename T, typename Kernel>
int launch_parts(Kernel kernel, dim3 grid, int threads, size_t smem, int ranks, int64_t parts, const Product<T> &p,
                 cudaStream_t s) {
    if (parts == 1) return launch_cluster(kernel, grid, threads, smem, ranks, p, s);
    void *sums = nullptr;
    if (int rc = scratch_alloc((size_t)(parts * p.M * p.N) * sizeof(T), &sums, s)) return rc;
    grid.z = (unsigned)parts;
    int rc = launch_cluster(kernel, grid, threads, smem, ranks,
                            Product<T>{p.A, p.B, nullptr, nullptr, nullptr, (T *)sums, p.M, p.K, p.N, J4C_ACT_NONE}, s);
    if (rc == J4C_OK) {
        join_kernel<T><<<(unsigned)ceil_div(p.M * p.N, 32), 1024, 0, s>>>(p, (const T *)sums, parts);
        count_launch();
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) rc = cuda_status(e, "join_kernel");
    }
    const int freed = scratch_free(sums, s);
    return rc ? rc : freed;
}

template <typename T, int MT, int V>
int launch_rows(const Product<T> &p, cudaStream_t s) {
    constexpr size_t smem = std::max<size_t>(8 * MT * 32 * V, kRowsK * MT) * sizeof(T);
    const dim3 grid((unsigned)ceil_div(p.N, 32 * V), (unsigned)ceil_div(p.M, MT));
    const int64_t strips = (int64_t)grid.x * grid.y;
    const int ranks = ranks_for<T>(strips, p.K);
    return launch_parts(rows_kernel<T, MT, V>, grid, kRowsThreads, smem, ranks,
                        parts_for<T>(strips * ranks, ranks * (kRowsThreads / 32), p.K), p, s);
}
template <typename T, int V>
int launch_rows_m(const Product<T> &p, cudaStream_t s) {
    if (p.M == 1) return launch_rows<T, 1, V>(p, s);
    if (p.M == 2) return launch_rows<T, 2, V>(p, s);
    if (p.M <= 4) return launch_rows<T, 4, V>(p, s);
    if (p.M <= 8) return launch_rows<T, 8, V>(p, s);
    return launch_rows<T, 16, V>(p, s);
}

template <typename T>
int64_t tiles_of(const Product<T> &p) {
    return ceil_div(p.M, kTM) * ceil_div(p.N, kTN);
}

// ranks: CTAs along K of the tile form (0: by the product's own size).
template <typename T>
int small_product(const Product<T> &p, int ta, int tb, int ranks, cudaStream_t s) {
    if (p.M <= 16 && !ta && !tb) {
        // the widest loads that still give every SM a strip of columns
        auto fits = [&](int v) {
            return p.N % v == 0 && reinterpret_cast<uintptr_t>(p.B) % (sizeof(T) * v) == 0 &&
                   p.N / (32 * v) * 8 >= sm_count();
        };
        if constexpr (sizeof(T) == 4)
            if (fits(4)) return launch_rows_m<T, 4>(p, s);
        return fits(2) ? launch_rows_m<T, 2>(p, s) : launch_rows_m<T, 1>(p, s);
    }
    const int64_t tiles = tiles_of(p);
    if (!ranks) ranks = ranks_for<T>(tiles, p.K);
    const int64_t parts = parts_for<T>(tiles * ranks, ranks, p.K);
    auto launch = [&](auto kernel) {
        return launch_parts(kernel, dim3((unsigned)tiles), kTileThreads, 0, ranks, parts, p, s);
    };
    if (ta) return tb ? launch(tile_kernel<T, true, true>) : launch(tile_kernel<T, true, false>);
    return tb ? launch(tile_kernel<T, false, true>) : launch(tile_kernel<T, false, false>);
}

// x's and w's gradients, in one launch (a cut of K for both) unless that left
// one of them more than 256 K a CTA that its own cut would not, or one comes in
// parts: the gradients of [1839,2090]x[2090,6], dw with 1839 K, 191 us in one
// launch, 46 in two.  How K is
// cut depends on the layer's sizes alone, not on which of the two are wanted: the
// same bits.
template <typename T>
int gradients(const Product<T> &dx, const Product<T> &dw, bool dx_too, bool dw_too, cudaStream_t s) {
    const int64_t tx = tiles_of(dx), tw = tiles_of(dw);
    const int both = ranks_for<T>(tx + tw, std::max(dx.K, dw.K));
    const int rx = ranks_for<T>(tx, dx.K), rw = ranks_for<T>(tw, dw.K);
    const bool parts = parts_for<T>(tx * both, both, dx.K) > 1 || parts_for<T>(tw * both, both, dw.K) > 1;
    const bool together = !parts && (std::max(dx.K, dw.K) <= both * 256ll || (rx <= both && rw <= both));
    if (together && dx_too && dw_too)
        return launch_cluster(two_products_kernel<T>, dim3((unsigned)(tx + tw)), kTileThreads, 0, both,
                              TwoProducts<T>{dx, dw, tx}, s);
    if (dx_too)
        if (int rc = small_product(dx, 0, 1, together ? both : rx, s)) return rc;
    return dw_too ? small_product(dw, 1, 0, together ? both : rw, s) : (int)J4C_OK;
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

// CLUSTER: the groups of rows of a strip are one cluster, which adds its column
// sums through distributed shared memory: a.sums is the bias's gradient itself.
template <typename T, int V, bool CLUSTER>
__global__ void __launch_bounds__(256, 4) dense_grad_kernel(const GradArgs<T> a) {
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
    for (int64_t r = r0 + warp; r < r1; r += 8) {
        T d[8], u[8];
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            Vec<T, V> x{}, z{};
            if (c0 + col(i) < a.N) {  // V divides N
                const int64_t at = r * a.N + c0 + col(i);
                x = *reinterpret_cast<const Vec<T, V> *>(a.dy + at);
                if (a.u) z = *reinterpret_cast<const Vec<T, V> *>(a.u + at);
            }
#pragma unroll
            for (int e = 0; e < V; e++) d[i + e] = x.e[e], u[i + e] = z.e[e];
        }
        if (a.from_output) slopes_of_output(a.act, u, d);
        else act_slopes(a.act, u, d);
        uint32_t rtop = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            sum[i] += d[i];
            if constexpr (sizeof(T) == 4) {
                const uint32_t b = __float_as_uint((float)d[i]) & 0x7FFFFFFFu;
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
                    for (int e = 0; e < V; e++) x.e[e] = d[i + e];
                    *reinterpret_cast<Vec<T, V> *>(a.dz + r * a.N + c0 + col(i)) = x;
                }
        }
        if (sizeof(T) == 4 && a.lines) {
            rtop = __reduce_max_sync(0xffffffffu, rtop);
            if (lane == 0 && rtop) atomicMax(a.lines + r, rtop);
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

// Groups of rows: four CTAs an SM (64 registers a thread, one row of a warp in
// flight: [8192,4096] gelu 68 us, 5.9 TB/s; two rows in flight and two CTAs an SM
// 75) and no more unless a warp had more than kMaxTerms rows, at least 32 rows
// each; where eight are enough for that, or for 512 rows, they are a cluster and
// need no second launch.
int64_t grad_groups(int64_t M, int64_t N) {
    const int64_t groups = std::max<int64_t>(
        1, std::min(ceil_div(M, 32), (int64_t)sm_count() * 4 / ceil_div(N, 256)));
    if (M <= 512) return std::min<int64_t>(groups, 8);
    return std::max(groups, std::min<int64_t>(ceil_div(M, 8 * kMaxTerms), 65535));
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

// More tiles than a grid takes.
static bool too_many(int64_t M, int64_t N) {
    return M >= (1ll << 40) || N >= (1ll << 33) || ceil_div(M, kTM) * ceil_div(N, 32) >= (1ll << 27);
}

extern "C" {

int j4c_dot_act(int dtype, const void *a, const void *b, int64_t M, int64_t K, int64_t N, int trans_a, int trans_b,
                const void *bias, int act, const void *residual, void *z, void *y, j4c_stream stream) {
    J4C_REQUIRE(dtype == J4C_FLOAT32 || dtype == J4C_FLOAT64, "j4c_dot_act requires FLOAT32 or FLOAT64 arrays, got %s",
                dtype_name(dtype));
    J4C_REQUIRE(M >= 0 && K >= 0 && N >= 0, "j4c_dot_act: negative dimension");
    J4C_REQUIRE(act_known(act), "j4c_dot_act: unknown activation %d", act);
    if (M == 0 || N == 0) return J4C_OK;
    J4C_REQUIRE(y && (K == 0 || (a && b)), "j4c_dot_act: NULL pointer");
    if (too_many(M, N))
        return set_error(J4C_E_UNSUPPORTED, "j4c_dot_act: %lld x %lld results are too many", (long long)M, (long long)N);
    auto run = [&](auto t) {
        using T = decltype(t);
        return small_product(Product<T>{(const T *)a, (const T *)b, (const T *)bias, (const T *)residual, (T *)z, (T *)y, M,
                                        K, N, act},
                             trans_a, trans_b, 0, as_stream(stream));
    };
    return dtype == J4C_FLOAT64 ? run(0.0) : run(0.0f);
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

int j4c_dense_backward(int dtype, const void *x, const void *w, int64_t M, int64_t K, int64_t N, const void *dy,
                       const void *u, int act, int from_output, void *dz, void *dx, void *dw, void *dbias, void *ws,
                       size_t ws_bytes, j4c_stream stream) {
    J4C_REQUIRE(dtype == J4C_FLOAT32 || dtype == J4C_FLOAT64, "j4c_dense_backward requires FLOAT32 or FLOAT64 arrays, got %s",
                dtype_name(dtype));
    J4C_REQUIRE(M >= 0 && K >= 0 && N >= 0, "j4c_dense_backward: negative dimension");
    // (an empty gradient's pointer is NULL too)
    J4C_REQUIRE(dx || dw || M == 0 || K == 0 || N == 0,
                "j4c_dense_backward: neither product is wanted (j4c_dense_grad gives dbias alone)");
    const void *d = dy;
    if (dbias || act != J4C_ACT_NONE) {
        if (int rc = j4c_dense_grad(dtype, M, N, dy, u, act, from_output, dz, dbias, nullptr, ws, ws_bytes, stream)) return rc;
        if (act != J4C_ACT_NONE) d = dz;
    }
    const bool dx_too = dx && M && K, dw_too = dw && K && N;
    J4C_REQUIRE((!dx_too || N == 0 || (d && w)) && (!dw_too || M == 0 || (d && x)), "j4c_dense_backward: NULL pointer");
    if ((dx_too && too_many(M, K)) || (dw_too && too_many(K, N)))
        return set_error(J4C_E_UNSUPPORTED, "j4c_dense_backward: %lld x %lld x %lld is too large", (long long)M,
                         (long long)K, (long long)N);
    auto run = [&](auto t) {
        using T = decltype(t);
        const Product<T> px{(const T *)d, (const T *)w, nullptr, nullptr, nullptr, (T *)dx, M, N, K, J4C_ACT_NONE};
        const Product<T> pw{(const T *)x, (const T *)d, nullptr, nullptr, nullptr, (T *)dw, K, M, N, J4C_ACT_NONE};
        return gradients(px, pw, dx_too, dw_too, as_stream(stream));
    };
    return dtype == J4C_FLOAT64 ? run(0.0) : run(0.0f);
}

}  // extern "C"
