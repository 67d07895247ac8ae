// group_norm.cu -- group norm with an activation over channels-last arrays.
//
// x is [B, S, C]: B samples of S positions with C contiguous channels, in G
// groups of D = C / G neighbouring channels.  Over the n = S * D values of a
// (sample, group):
//   xhat = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   u = gamma[c] xhat + beta[c],  y = act(u)
// and for the gradient, with du = dy act'(u) and h = gamma du:
//   dbeta[c] = sum du,  dgamma[c] = sum du xhat     (over samples and positions)
//   dx = rstd (h - mean(h) - xhat mean(h xhat))     (means over the group)
// Variances are sums of squared differences from the mean, never differences
// of sums, so a mean far from zero costs no digits.  Everything is summed in
// the arrays' type in a fixed order: results repeat bit for bit.
//
// All of it is bound by HBM: x in, y out (8 B per FLOAT32 value) forward; x and
// dy in, dx out backward (12 B).  Two forms:
//  * Groups of at most 8192 values (rows of features are S = 1, G = 1: layer
//    norm) are held in registers, eight values a thread, by 1 to 32 warps:
//    every value is read once.  Backward a warp set keeps its group and walks
//    over samples, so dgamma and dbeta gather in registers too.
//  * Larger groups are cut into tiles of rows.  Forward, one kernel reads a
//    tile into shared memory and leaves its mean and squared differences per
//    group; a second one merges the tiles' (Chan, Golub and LeVeque's pairwise
//    update, in FP64) and applies.  Backward the same with per-channel sums of
//    du and du xhat.  The second read of a tile comes from L2: the batch is
//    walked in parts of at most kL2Part bytes.
#include <algorithm>
#include <type_traits>

#include "act.cuh"
#include "common.cuh"

namespace j4c {
namespace {

constexpr int kHeld = 8;             // values a thread holds
constexpr int64_t kMaxHeld = 32 * 32 * kHeld;
constexpr int kTileThreads = 256;
constexpr int kTileBytes = 48 * 1024;
constexpr int kTileChannels = 2048;  // channels of a tile at most
constexpr int64_t kL2Part = 40ll << 20;

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};

template <typename T>
struct Args {
    int64_t B, S, C, G, D;
    const T *x, *gamma, *beta, *dy;
    T *mean, *rstd;  // [B, G]
    T eps;
    int act;
    T *y;   // y or dx
    T *dpart;  // per-channel sums of du, then of du xhat: see the kernels
};

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float inv_sqrt(float x) { return __frcp_rn(__fsqrt_rn(x)); }
__device__ __forceinline__ double inv_sqrt(double x) { return 1.0 / sqrt(x); }

// ---- groups held in registers ------------------------------------------------------
// WARPS warps hold one (sample, group); a CTA of max(8, WARPS) warps has CTA / WARPS sets.
template <int WARPS>
struct Held {
    static constexpr int CTA = WARPS < 8 ? 8 : WARPS;
    static constexpr int SETS = CTA / WARPS;
    static constexpr int THREADS = 32 * WARPS;  // of a set
};

// The sum over a set.  Consecutive sums alternate between two buffers: a
// barrier of the second is behind every read of the first.
template <typename T, int WARPS>
__device__ __forceinline__ T set_sum(T v, T *buf, int set) {
    v = warp_sum(v);
    if constexpr (WARPS > 1) {
        const int warp = (threadIdx.x / 32) % WARPS;
        if (threadIdx.x % 32 == 0) buf[set * WARPS + warp] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + set), "n"(32 * WARPS) : "memory");
        v = T(0);
#pragma unroll
        for (int w = 0; w < WARPS; w++) v += buf[set * WARPS + w];
    }
    return v;
}

// Where thread t of a set finds its values: value i * V + e of its kHeld is
// channel col[i] + e of the group, off[i] + e elements behind the group's first.
template <int V, int WARPS, int NV>
struct Place {
    int64_t off[NV];
    int col[NV];
    __device__ __forceinline__ Place(int t, int64_t S, int64_t C, int64_t D) {
        const int per_row = (int)(D / V), all = (int)(S * per_row);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int v = t + i * Held<WARPS>::THREADS;
            const int s = v / per_row;
            col[i] = v < all ? (v - s * per_row) * V : -1;
            off[i] = (int64_t)s * C + col[i];
        }
    }
};

template <typename T, int V, int WARPS>
__global__ void __launch_bounds__(32 * Held<WARPS>::CTA) held_forward_kernel(const Args<T> a) {
    using H = Held<WARPS>;
    constexpr int NV = kHeld / V;
    __shared__ T sums[2][H::CTA];
    const int set = threadIdx.x / H::THREADS, t = threadIdx.x % H::THREADS;
    const Place<V, WARPS, NV> at(t, a.S, a.C, a.D);
    const int64_t items = a.B * a.G;
    const T n = (T)(a.S * a.D);
    for (int64_t item = (int64_t)blockIdx.x * H::SETS + set; item < items; item += (int64_t)gridDim.x * H::SETS) {
        const int64_t b = item / a.G, g = item - b * a.G;
        const int64_t base = b * a.S * a.C + g * a.D;
        Vec<T, V> x[NV];
        T sum = T(0);
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) x[i] = *reinterpret_cast<const Vec<T, V> *>(a.x + base + at.off[i]);
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) {
#pragma unroll
                for (int e = 0; e < V; e++) sum += x[i].e[e];
            }
        const T mean = set_sum<T, WARPS>(sum, sums[0], set) / n;
        T sq = T(0);
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    x[i].e[e] -= mean;
                    sq += x[i].e[e] * x[i].e[e];
                }
            }
        const T rstd = inv_sqrt(set_sum<T, WARPS>(sq, sums[1], set) / n + a.eps);
        if (t == 0 && a.mean) {
            a.mean[item] = mean;
            a.rstd[item] = rstd;
        }
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) {
                const int64_t c = g * a.D + at.col[i];
#pragma unroll
                for (int e = 0; e < V; e++) {
                    T u = x[i].e[e] * rstd;
                    if (a.gamma) u *= a.gamma[c + e];
                    if (a.beta) u += a.beta[c + e];
                    x[i].e[e] = act_value(a.act, u);
                }
                *reinterpret_cast<Vec<T, V> *>(a.y + base + at.off[i]) = x[i];
            }
    }
}

// Set k of the grid holds group k % G and walks over samples k / G, k / G + nb, ...
// (nb sets for every group).  a.dpart, unless NULL, gets its sums over samples
// and positions: [nb, C] of du, then [nb, C] of du xhat.
template <typename T, int V, int WARPS>
__global__ void __launch_bounds__(32 * Held<WARPS>::CTA) held_backward_kernel(const Args<T> a, int64_t nb) {
    using H = Held<WARPS>;
    constexpr int NV = kHeld / V;
    __shared__ T sums[2][H::CTA];
    extern __shared__ __align__(16) unsigned char raw[];
    const int set = threadIdx.x / H::THREADS, t = threadIdx.x % H::THREADS;
    const Place<V, WARPS, NV> at(t, a.S, a.C, a.D);
    const int64_t k = (int64_t)blockIdx.x * H::SETS + set;
    if (k >= nb * a.G) return;  // a whole set: barriers are the set's own
    const int64_t g = k % a.G;
    const T n = (T)(a.S * a.D);
    T du_sum[kHeld], dux_sum[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; i++) du_sum[i] = dux_sum[i] = T(0);
    for (int64_t b = k / a.G; b < a.B; b += nb) {
        const int64_t base = b * a.S * a.C + g * a.D;
        Vec<T, V> x[NV], h[NV];
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) {
                x[i] = *reinterpret_cast<const Vec<T, V> *>(a.x + base + at.off[i]);
                h[i] = *reinterpret_cast<const Vec<T, V> *>(a.dy + base + at.off[i]);
            }
        const T mean = a.mean[b * a.G + g], rstd = a.rstd[b * a.G + g];
        T s1 = T(0), s2 = T(0);
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) {
                const int64_t c = g * a.D + at.col[i];
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const T xhat = (x[i].e[e] - mean) * rstd;
                    const T gm = a.gamma ? a.gamma[c + e] : T(1);
                    T u = xhat * gm;
                    if (a.beta) u += a.beta[c + e];
                    const T du = h[i].e[e] * act_slope(a.act, u);
                    du_sum[i * V + e] += du;
                    dux_sum[i * V + e] += du * xhat;
                    x[i].e[e] = xhat;
                    h[i].e[e] = du * gm;
                    s1 += h[i].e[e];
                    s2 += h[i].e[e] * xhat;
                }
            }
        s1 = set_sum<T, WARPS>(s1, sums[0], set) / n;
        s2 = set_sum<T, WARPS>(s2, sums[1], set) / n;
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) {
#pragma unroll
                for (int e = 0; e < V; e++) x[i].e[e] = rstd * (h[i].e[e] - s1 - x[i].e[e] * s2);
                *reinterpret_cast<Vec<T, V> *>(a.y + base + at.off[i]) = x[i];
            }
    }
    if (!a.dpart) return;
    // sums over samples: now over the positions of a channel, through shared memory
    T *buf = reinterpret_cast<T *>(raw) + (size_t)set * a.S * a.D;
    for (int which = 0; which < 2; which++) {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (at.col[i] >= 0) {
                const int64_t s = (at.off[i] - at.col[i]) / a.C;
#pragma unroll
                for (int e = 0; e < V; e++)
                    buf[s * a.D + at.col[i] + e] = which ? dux_sum[i * V + e] : du_sum[i * V + e];
            }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + set), "n"(32 * WARPS) : "memory");
        for (int c = t; c < a.D; c += H::THREADS) {
            T v = T(0);
            for (int s = 0; s < a.S; s++) v += buf[s * a.D + c];
            a.dpart[((int64_t)which * nb + k / a.G) * a.C + g * a.D + c] = v;
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + set), "n"(32 * WARPS) : "memory");
    }
}

// out[j] = sum over r of in[r, j], r < rows, for two [rows, cols] arrays back
// to back: 32 columns and 8 lanes of rows a CTA; either output may be NULL.
template <typename T>
__global__ void __launch_bounds__(256) sum_rows_kernel(const T *__restrict__ in, int64_t rows, int64_t cols, T *out0,
                                                       T *out1) {
    __shared__ T part[8][33];
    const int lane = threadIdx.x % 32, rl = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    T *out = blockIdx.y ? out1 : out0;
    if (!out) return;
    in += blockIdx.y * rows * cols;
    T v = T(0);
    if (c < cols) {
        int64_t r = rl;
        for (; r + 24 < rows; r += 32) {
            T w[4];
#pragma unroll
            for (int u = 0; u < 4; u++) w[u] = in[(r + 8 * u) * cols + c];
            v += (w[0] + w[1]) + (w[2] + w[3]);
        }
        for (; r < rows; r += 8) v += in[r * cols + c];
    }
    part[rl][lane] = v;
    __syncthreads();
    if (rl == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 8; i++) v += part[i][lane];
        out[c] = v;
    }
}

// ---- groups cut into tiles ------------------------------------------------------------
// A tile is `rows` positions of one sample by some channels: whole groups
// (per > 0 of them), or a stretch of one group wider than kTileChannels
// (per = 0, `cuts` stretches a group).
struct Geo {
    int64_t S, C, G, D;
    int rows, row_tiles, width, col_tiles, per, cuts;
    __host__ __device__ int parts() const { return row_tiles * cuts; }  // tiles of a (sample, group)
};

struct Tile {
    int64_t b, c0, g0;
    int r0, rows, width, groups, cut;
    __device__ __forceinline__ Tile(const Geo &q, int64_t block) {
        const int ct = (int)(block % q.col_tiles);
        const int64_t br = block / q.col_tiles;
        const int rt = (int)(br % q.row_tiles);
        b = br / q.row_tiles;
        r0 = rt * q.rows;
        rows = (int)min((int64_t)q.rows, q.S - r0);
        if (q.per) {
            g0 = (int64_t)ct * q.per;
            groups = (int)min((int64_t)q.per, q.G - g0);
            c0 = g0 * q.D;
            width = (int)(groups * q.D);
            cut = 0;
        } else {
            g0 = ct / q.cuts;
            cut = ct % q.cuts;
            groups = 1;
            c0 = g0 * q.D + (int64_t)cut * q.width;
            width = (int)min((int64_t)q.width, q.D - (int64_t)cut * q.width);
        }
    }
};

// The threads of a tile: columns of V channels, and lanes of rows where a row
// has fewer columns than the CTA threads.
struct Lanes {
    int cols, rows, j, r;
    bool on;
    __device__ __forceinline__ Lanes(int width, int V) {
        cols = width / V;
        rows = cols >= kTileThreads ? 1 : kTileThreads / cols;
        j = cols >= kTileThreads ? threadIdx.x : threadIdx.x % cols;
        r = cols >= kTileThreads ? 0 : threadIdx.x / cols;
        on = r < rows;
    }
};

// Sums red[lane of rows][column] over each group's columns; out[group], by one warp a group.
template <typename T, typename Store>
__device__ __forceinline__ void sum_groups(const T *red, const Lanes &l, int groups, Store store) {
    const int per = l.cols / groups, all = per * l.rows;
    for (int g = threadIdx.x / 32; g < groups; g += kTileThreads / 32) {
        T v = T(0);
        for (int k = threadIdx.x % 32; k < all; k += 32) {
            const int r = k / per;
            v += red[r * l.cols + g * per + (k - r * per)];
        }
        v = warp_sum(v);
        if (threadIdx.x % 32 == 0) store(g, v);
    }
}

// stats[(b G + g) parts + part] = (mean, sum of squared differences from it) of a tile's part of a group.
template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads) tile_stats_kernel(const Args<T> a, const Geo q, T *__restrict__ stats) {
    extern __shared__ __align__(16) unsigned char raw[];
    T *tile = reinterpret_cast<T *>(raw);
    T *red = tile + (size_t)q.rows * q.width;
    T *means = red + max(kTileThreads, q.width / V);
    const Tile w(q, blockIdx.x);
    const Lanes l(w.width, V);
    const T *x = a.x + (w.b * q.S + w.r0) * q.C + w.c0;
    if (l.on)
        for (int j = l.j; j < l.cols; j += kTileThreads) {
            T sum = T(0);
#pragma unroll 8
            for (int r = l.r; r < w.rows; r += l.rows) {
                const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(x + r * q.C + j * V);
                *reinterpret_cast<Vec<T, V> *>(tile + (size_t)r * w.width + j * V) = v;
#pragma unroll
                for (int e = 0; e < V; e++) sum += v.e[e];
            }
            red[l.r * l.cols + j] = sum;
        }
    __syncthreads();
    const T n = (T)((int64_t)w.rows * (w.width / w.groups));
    sum_groups(red, l, w.groups, [&](int g, T v) { means[g] = v / n; });
    __syncthreads();
    const int per = l.cols / w.groups;
    if (l.on)
        for (int j = l.j; j < l.cols; j += kTileThreads) {
            const T mean = means[j / per];
            T sum = T(0);
#pragma unroll 4
            for (int r = l.r; r < w.rows; r += l.rows) {
                const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(tile + (size_t)r * w.width + j * V);
#pragma unroll
                for (int e = 0; e < V; e++) sum += (v.e[e] - mean) * (v.e[e] - mean);
            }
            red[l.r * l.cols + j] = sum;
        }
    __syncthreads();
    const int part = (w.r0 / q.rows) * q.cuts + w.cut;
    sum_groups(red, l, w.groups, [&](int g, T v) {
        T *s = stats + 2 * ((w.b * q.G + w.g0 + g) * q.parts() + part);
        s[0] = means[g];
        s[1] = v;
    });
}

template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads) tile_apply_kernel(const Args<T> a, const Geo q,
                                                                  const T *__restrict__ stats) {
    extern __shared__ __align__(16) unsigned char raw[];
    const Tile w(q, blockIdx.x);
    T *means = reinterpret_cast<T *>(raw), *rstds = means + w.groups;
    // merge the group's parts, one warp a group
    const int lane = threadIdx.x % 32;
    for (int g = threadIdx.x / 32; g < w.groups; g += kTileThreads / 32) {
        const T *s = stats + 2 * (w.b * q.G + w.g0 + g) * q.parts();
        const double n = (double)q.S * q.D;
        auto count = [&](int p) {
            const int rows = (int)min((int64_t)q.rows, q.S - (int64_t)(p / q.cuts) * q.rows);
            const int64_t cols = q.per ? q.D : min((int64_t)q.width, q.D - (int64_t)(p % q.cuts) * q.width);
            return (double)(rows * cols);
        };
        double sum = 0.0;
        for (int p = lane; p < q.parts(); p += 32) sum += count(p) * (double)s[2 * p];
        const double mean = warp_sum(sum) / n;
        double m2 = 0.0;
        for (int p = lane; p < q.parts(); p += 32) {
            const double d = (double)s[2 * p] - mean;
            m2 += (double)s[2 * p + 1] + count(p) * d * d;
        }
        m2 = warp_sum(m2);
        if (lane == 0) {
            means[g] = (T)mean;
            rstds[g] = inv_sqrt((T)(m2 / n) + a.eps);
            if (w.r0 == 0 && w.cut == 0 && a.mean) {
                a.mean[w.b * q.G + w.g0 + g] = means[g];
                a.rstd[w.b * q.G + w.g0 + g] = rstds[g];
            }
        }
    }
    __syncthreads();
    const Lanes l(w.width, V);
    const int per = l.cols / w.groups;
    const int64_t base = (w.b * q.S + w.r0) * q.C + w.c0;
    if (!l.on) return;
    for (int j = l.j; j < l.cols; j += kTileThreads) {
        const T mean = means[j / per], rstd = rstds[j / per];
        Vec<T, V> gm, bt;
#pragma unroll
        for (int e = 0; e < V; e++) {
            gm.e[e] = a.gamma ? a.gamma[w.c0 + j * V + e] : T(1);
            bt.e[e] = a.beta ? a.beta[w.c0 + j * V + e] : T(0);
        }
#pragma unroll 4
        for (int r = l.r; r < w.rows; r += l.rows) {
            Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(a.x + base + r * q.C + j * V);
#pragma unroll
            for (int e = 0; e < V; e++) {
                T u = (v.e[e] - mean) * rstd * gm.e[e];
                if (a.beta) u += bt.e[e];
                v.e[e] = act_value(a.act, u);
            }
            *reinterpret_cast<Vec<T, V> *>(a.y + base + r * q.C + j * V) = v;
        }
    }
}

// sums[(b row_tiles + rt) C + c] = sum over the tile's rows of du, and behind
// all of these ([B row_tiles, C]) of du xhat.
template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads) tile_sums_kernel(const Args<T> a, const Geo q, int64_t samples,
                                                                 T *__restrict__ sums) {
    extern __shared__ __align__(16) unsigned char raw[];
    T *red = reinterpret_cast<T *>(raw);  // [2][lanes of rows][width], where there are several lanes of rows
    const Tile w(q, blockIdx.x);
    const Lanes l(w.width, V);
    const int per = l.cols / w.groups;
    const int64_t base = (w.b * q.S + w.r0) * q.C + w.c0;
    T *out0 = sums + (w.b * q.row_tiles + w.r0 / q.rows) * q.C + w.c0, *out1 = out0 + samples * q.row_tiles * q.C;
    if (l.on)
        for (int j = l.j; j < l.cols; j += kTileThreads) {
            const int64_t g = w.g0 + j / per;
            const T mean = a.mean[w.b * q.G + g], rstd = a.rstd[w.b * q.G + g];
            Vec<T, V> gm, bt, s1, s2;
#pragma unroll
            for (int e = 0; e < V; e++) {
                gm.e[e] = a.gamma ? a.gamma[w.c0 + j * V + e] : T(1);
                bt.e[e] = a.beta ? a.beta[w.c0 + j * V + e] : T(0);
                s1.e[e] = s2.e[e] = T(0);
            }
#pragma unroll 4
            for (int r = l.r; r < w.rows; r += l.rows) {
                const Vec<T, V> x = *reinterpret_cast<const Vec<T, V> *>(a.x + base + r * q.C + j * V);
                const Vec<T, V> dy = *reinterpret_cast<const Vec<T, V> *>(a.dy + base + r * q.C + j * V);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const T xhat = (x.e[e] - mean) * rstd;
                    T u = xhat * gm.e[e];
                    if (a.beta) u += bt.e[e];
                    const T du = dy.e[e] * act_slope(a.act, u);
                    s1.e[e] += du;
                    s2.e[e] += du * xhat;
                }
            }
#pragma unroll
            for (int e = 0; e < V; e++) {
                if (l.rows == 1) {
                    out0[j * V + e] = s1.e[e];
                    out1[j * V + e] = s2.e[e];
                } else {
                    red[l.r * w.width + j * V + e] = s1.e[e];
                    red[(l.rows + l.r) * w.width + j * V + e] = s2.e[e];
                }
            }
        }
    if (l.rows == 1) return;
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * w.width; c += kTileThreads) {
        const int which = c >= w.width, cc = c - which * w.width;
        T v = T(0);
        for (int r = 0; r < l.rows; r++) v += red[(which * l.rows + r) * w.width + cc];
        (which ? out1 : out0)[cc] = v;
    }
}

// Per (sample, group), one CTA: the tiles' sums added up per channel (chan[b C + c],
// and chan_half behind it the ones of du xhat) and, weighted with gamma, over the
// group: group[2 (b G + g)] = mean(h), mean(h xhat).
template <typename T>
__global__ void __launch_bounds__(256) merge_sums_kernel(const Args<T> a, const Geo q, int64_t samples,
                                                         const T *__restrict__ sums, T *__restrict__ chan,
                                                         int64_t chan_half, T *__restrict__ group) {
    __shared__ T part[2][8];
    const int64_t b = blockIdx.x / q.G, g = blockIdx.x - b * q.G;
    const int64_t half = samples * q.row_tiles * q.C;
    T s1 = T(0), s2 = T(0);
    for (int64_t d = threadIdx.x; d < q.D; d += 256) {
        const int64_t c = g * q.D + d;
        const T *p = sums + b * q.row_tiles * q.C + c;
        T v1 = T(0), v2 = T(0);
#pragma unroll 4
        for (int r = 0; r < q.row_tiles; r++) {
            v1 += p[r * q.C];
            v2 += p[half + r * q.C];
        }
        chan[b * q.C + c] = v1;
        chan[chan_half + b * q.C + c] = v2;
        const T gm = a.gamma ? a.gamma[c] : T(1);
        s1 += gm * v1;
        s2 += gm * v2;
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (threadIdx.x % 32 == 0) {
        part[0][threadIdx.x / 32] = s1;
        part[1][threadIdx.x / 32] = s2;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        T v = T(0);
        for (int i = 0; i < 8; i++) v += part[threadIdx.x][i];
        group[2 * (b * q.G + g) + threadIdx.x] = v / (T)(q.S * q.D);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads) tile_grad_kernel(const Args<T> a, const Geo q,
                                                                 const T *__restrict__ group) {
    const Tile w(q, blockIdx.x);
    const Lanes l(w.width, V);
    const int per = l.cols / w.groups;
    const int64_t base = (w.b * q.S + w.r0) * q.C + w.c0;
    if (!l.on) return;
    for (int j = l.j; j < l.cols; j += kTileThreads) {
        const int64_t bg = w.b * q.G + w.g0 + j / per;
        const T mean = a.mean[bg], rstd = a.rstd[bg], h1 = group[2 * bg], h2 = group[2 * bg + 1];
        Vec<T, V> gm, bt;
#pragma unroll
        for (int e = 0; e < V; e++) {
            gm.e[e] = a.gamma ? a.gamma[w.c0 + j * V + e] : T(1);
            bt.e[e] = a.beta ? a.beta[w.c0 + j * V + e] : T(0);
        }
#pragma unroll 4
        for (int r = l.r; r < w.rows; r += l.rows) {
            Vec<T, V> x = *reinterpret_cast<const Vec<T, V> *>(a.x + base + r * q.C + j * V);
            const Vec<T, V> dy = *reinterpret_cast<const Vec<T, V> *>(a.dy + base + r * q.C + j * V);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const T xhat = (x.e[e] - mean) * rstd;
                T u = xhat * gm.e[e];
                if (a.beta) u += bt.e[e];
                const T h = dy.e[e] * act_slope(a.act, u) * gm.e[e];
                x.e[e] = rstd * (h - h1 - xhat * h2);
            }
            *reinterpret_cast<Vec<T, V> *>(a.y + base + r * q.C + j * V) = x;
        }
    }
}

// ---- host ----------------------------------------------------------------------------
inline bool held(int64_t S, int64_t D) { return D <= kMaxHeld && S <= kMaxHeld && S * D <= kMaxHeld; }

// Rows of a tile: as many as shared memory takes, fewer when the batch would
// leave SMs without a tile; at most `most` (the backward sums need no shared
// memory, and a tile's sums cost 2 / rows of a pass).
template <typename T>
Geo make_geo(int64_t B, int64_t S, int64_t C, int64_t G, bool backward) {
    Geo q;
    q.S = S, q.C = C, q.G = G, q.D = C / G;
    if (q.D <= kTileChannels) {
        q.per = (int)std::min<int64_t>(G, kTileChannels / q.D);
        q.width = (int)(q.per * q.D);
        q.col_tiles = (int)ceil_div(G, q.per);
        q.cuts = 1;
    } else {
        q.per = 0;
        q.width = kTileChannels;
        q.cuts = (int)ceil_div(q.D, q.width);
        q.col_tiles = (int)(G * q.cuts);
    }
    const int64_t fit = std::max<int64_t>(1, kTileBytes / ((int64_t)q.width * sizeof(T)));
    int64_t rows = fit;
    if (backward) rows = std::max<int64_t>(fit, ceil_div(B * S * q.col_tiles, (int64_t)sm_count() * 16));
    // two tiles for every SM, where there are rows enough
    const int64_t tiles_wanted = ceil_div((int64_t)sm_count() * 2, B * q.col_tiles);
    rows = std::min(rows, std::max<int64_t>(4, ceil_div(S, tiles_wanted)));
    rows = std::min(rows, S);
    q.rows = (int)rows;
    q.row_tiles = (int)ceil_div(S, rows);
    return q;
}

int64_t samples_of_part(int64_t B, int64_t bytes_per_sample) {
    return std::max<int64_t>(1, std::min(B, kL2Part / std::max<int64_t>(1, bytes_per_sample)));
}

// Warps that hold a group of n values, eight values a thread.
inline int held_warps(int64_t n) {
    int warps = 1;
    while (warps * 32 * kHeld < n) warps *= 2;
    return warps;
}

// Backward, the sets that share a group's samples: two CTAs of 512 threads an
// SM (64 registers each) or as many threads in smaller ones, no more than samples.
inline int64_t held_sets(int64_t B, int64_t G, int warps) {
    const int cta = std::max(8, warps);
    return std::min(B, std::max<int64_t>(1, ceil_div((int64_t)sm_count() * (32 / cta) * (cta / warps), G)));
}

template <typename T>
size_t workspace(int64_t B, int64_t S, int64_t C, int64_t G, bool backward) {
    const int64_t es = sizeof(T);
    if (held(S, C / G)) return backward ? (size_t)(2 * es * C * held_sets(B, G, held_warps(S * (C / G)))) : 0;
    const int64_t part = samples_of_part(B, (backward ? 2 : 1) * S * C * es);
    const Geo q = make_geo<T>(part, S, C, G, backward);
    if (!backward) return (size_t)(2 * es * part * G * q.parts());
    return (size_t)(es * (2 * part * q.row_tiles * C + 2 * B * C + 2 * part * G));
}

template <typename T, int V, int WARPS>
int launch_held(const Args<T> &a, bool backward, T *dgamma, T *dbeta, cudaStream_t s) {
    using H = Held<WARPS>;
    const int threads = 32 * H::CTA;
    if (!backward) {
        const int64_t ctas = ceil_div(a.B * a.G, H::SETS);
        const unsigned grid = (unsigned)std::min<int64_t>(ctas, (int64_t)sm_count() * (2048 / threads));
        held_forward_kernel<T, V, WARPS><<<grid, threads, 0, s>>>(a);
        J4C_LAUNCH_CHECK("held_forward_kernel");
        return J4C_OK;
    }
    const int64_t nb = held_sets(a.B, a.G, WARPS);
    if (ceil_div(nb * a.G, H::SETS) >= (1ll << 31)) return set_error(J4C_E_UNSUPPORTED, "j4c_group_norm: too many groups");
    const size_t smem = a.dpart ? (size_t)H::SETS * a.S * a.D * sizeof(T) : 0;
    if (smem > 48 * 1024)
        J4C_CUDA(cudaFuncSetAttribute(held_backward_kernel<T, V, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)smem));
    held_backward_kernel<T, V, WARPS><<<(unsigned)ceil_div(nb * a.G, H::SETS), threads, smem, s>>>(a, nb);
    J4C_LAUNCH_CHECK("held_backward_kernel");
    if (a.dpart) {
        sum_rows_kernel<T><<<dim3((unsigned)ceil_div(a.C, 32), 2), 256, 0, s>>>(a.dpart, nb, a.C, dbeta, dgamma);
        J4C_LAUNCH_CHECK("sum_rows_kernel");
    }
    return J4C_OK;
}

template <typename T, int V>
int run_held(const Args<T> &a, bool backward, T *dgamma, T *dbeta, cudaStream_t s) {
    switch (held_warps(a.S * a.D)) {
    case 1: return launch_held<T, V, 1>(a, backward, dgamma, dbeta, s);
    case 2: return launch_held<T, V, 2>(a, backward, dgamma, dbeta, s);
    case 4: return launch_held<T, V, 4>(a, backward, dgamma, dbeta, s);
    case 8: return launch_held<T, V, 8>(a, backward, dgamma, dbeta, s);
    case 16: return launch_held<T, V, 16>(a, backward, dgamma, dbeta, s);
    default: return launch_held<T, V, 32>(a, backward, dgamma, dbeta, s);
    }
}

template <typename T, int V>
int run_tiles(const Args<T> &whole, bool backward, T *dgamma, T *dbeta, void *ws, cudaStream_t s) {
    const int64_t B = whole.B, S = whole.S, C = whole.C, G = whole.G;
    const int64_t part = samples_of_part(B, (backward ? 2 : 1) * S * C * (int64_t)sizeof(T));
    const Geo q = make_geo<T>(part, S, C, G, backward);
    const int64_t tiles_of_sample = (int64_t)q.row_tiles * q.col_tiles;
    if (part * tiles_of_sample >= (1ll << 31) || part * G >= (1ll << 31))
        return set_error(J4C_E_UNSUPPORTED, "j4c_group_norm: too many tiles");
    T *w = static_cast<T *>(ws);
    for (int64_t b0 = 0; b0 < B; b0 += part) {
        const int64_t nb = std::min(part, B - b0);
        Args<T> a = whole;
        a.B = nb;
        a.x += b0 * S * C, a.y += b0 * S * C;
        if (a.mean) a.mean += b0 * G, a.rstd += b0 * G;
        const unsigned grid = (unsigned)(nb * tiles_of_sample);
        if (!backward) {
            const size_t smem = ((size_t)q.rows * q.width + std::max(kTileThreads, q.width / V) + std::max(q.per, 1)) *
                                sizeof(T);
            if (smem > 48 * 1024)  // the tile and the columns' sums: at most 72 KB
                J4C_CUDA(cudaFuncSetAttribute(tile_stats_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              96 * 1024));
            tile_stats_kernel<T, V><<<grid, kTileThreads, smem, s>>>(a, q, w);
            J4C_LAUNCH_CHECK("tile_stats_kernel");
            tile_apply_kernel<T, V><<<grid, kTileThreads, 2 * std::max(q.per, 1) * sizeof(T), s>>>(a, q, w);
            J4C_LAUNCH_CHECK("tile_apply_kernel");
            continue;
        }
        a.dy += b0 * S * C;
        T *sums = w, *chan = w + 2 * part * q.row_tiles * C, *group = chan + 2 * B * C;
        const size_t smem = 2 * (size_t)std::max(kTileThreads * V, q.width) * sizeof(T);
        tile_sums_kernel<T, V><<<grid, kTileThreads, smem, s>>>(a, q, nb, sums);
        J4C_LAUNCH_CHECK("tile_sums_kernel");
        // chan is [2, B, C] over the whole batch: this part's rows of each half
        merge_sums_kernel<T><<<(unsigned)(nb * G), 256, 0, s>>>(a, q, nb, sums, chan + b0 * C, B * C, group);
        J4C_LAUNCH_CHECK("merge_sums_kernel");
        tile_grad_kernel<T, V><<<grid, kTileThreads, 0, s>>>(a, q, group);
        J4C_LAUNCH_CHECK("tile_grad_kernel");
    }
    if (backward && (dgamma || dbeta)) {
        sum_rows_kernel<T><<<dim3((unsigned)ceil_div(C, 32), 2), 256, 0, s>>>(w + 2 * part * q.row_tiles * C, B, C, dbeta,
                                                                              dgamma);
        J4C_LAUNCH_CHECK("sum_rows_kernel");
    }
    return J4C_OK;
}

template <typename T>
int group_norm(const Args<T> &a, bool backward, T *dgamma, T *dbeta, void *ws, cudaStream_t s) {
    // vectors of neighbouring channels lie within a group
    constexpr int W = 16 / sizeof(T);
    auto fits = [&](int v) {
        auto ok = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (v * sizeof(T)) == 0; };
        return a.D % v == 0 && ok(a.x) && ok(a.y) && ok(a.dy);
    };
    const int v = fits(W) ? W : W > 2 && fits(2) ? 2 : 1;
    const bool small = held(a.S, a.D);
    auto run = [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        return small ? run_held<T, V>(a, backward, dgamma, dbeta, s) : run_tiles<T, V>(a, backward, dgamma, dbeta, ws, s);
    };
    if (v == W) return run(std::integral_constant<int, W>{});
    if (v == 2) return run(std::integral_constant<int, 2>{});
    return run(std::integral_constant<int, 1>{});
}

}  // namespace
}  // namespace j4c

using namespace j4c;

extern "C" {

static int check_shape(const char *name, int dtype, int64_t B, int64_t S, int64_t C, int64_t groups, double eps, int act) {
    J4C_REQUIRE(dtype == J4C_FLOAT32 || dtype == J4C_FLOAT64, "%s requires FLOAT32 or FLOAT64 arrays, got %s", name,
                dtype_name(dtype));
    J4C_REQUIRE(B >= 0 && S >= 0 && C >= 1, "%s: bad extents [%lld, %lld, %lld]", name, (long long)B, (long long)S,
                (long long)C);
    J4C_REQUIRE(groups >= 1 && C % groups == 0, "%s: %lld channels do not divide into %lld groups", name, (long long)C,
                (long long)groups);
    J4C_REQUIRE(eps >= 0.0, "%s: negative eps", name);
    J4C_REQUIRE(act_known(act), "%s: unknown activation %d", name, act);
    J4C_REQUIRE(S < (1ll << 31) && C < (1ll << 31), "%s: extents of 2^31 and more are not supported", name);
    return J4C_OK;
}

size_t j4c_group_norm_workspace(int dtype, int64_t B, int64_t S, int64_t C, int64_t groups, int backward) {
    if (B <= 0 || S <= 0 || C < 1 || groups < 1 || C % groups) return 0;
    return dtype == J4C_FLOAT64 ? workspace<double>(B, S, C, groups, backward != 0)
                                : workspace<float>(B, S, C, groups, backward != 0);
}

int j4c_group_norm(int dtype, int64_t B, int64_t S, int64_t C, int64_t groups, const void *x, const void *gamma,
                   const void *beta, double eps, int act, void *y, void *mean, void *rstd, void *ws, size_t ws_bytes,
                   j4c_stream stream) {
    if (int rc = check_shape("j4c_group_norm", dtype, B, S, C, groups, eps, act)) return rc;
    J4C_REQUIRE(!mean == !rstd, "j4c_group_norm: mean and rstd go together");
    if (B == 0 || S == 0) return J4C_OK;
    J4C_REQUIRE(x && y, "j4c_group_norm: NULL pointer");
    const size_t need = j4c_group_norm_workspace(dtype, B, S, C, groups, 0);
    J4C_REQUIRE(need == 0 || (ws && aligned16(ws) && ws_bytes >= need), "j4c_group_norm: needs %zu bytes of workspace", need);
    auto run = [&](auto t) {
        using T = decltype(t);
        Args<T> a{B, S, C, groups, C / groups, (const T *)x, (const T *)gamma, (const T *)beta, nullptr, (T *)mean,
                  (T *)rstd, (T)eps, act, (T *)y, nullptr};
        return group_norm<T>(a, false, nullptr, nullptr, ws, as_stream(stream));
    };
    return dtype == J4C_FLOAT64 ? run(0.0) : run(0.0f);
}

int j4c_group_norm_grad(int dtype, int64_t B, int64_t S, int64_t C, int64_t groups, const void *x, const void *gamma,
                        const void *beta, int act, const void *mean, const void *rstd, const void *dy, void *dx,
                        void *dgamma, void *dbeta, void *ws, size_t ws_bytes, j4c_stream stream) {
    if (int rc = check_shape("j4c_group_norm_grad", dtype, B, S, C, groups, 0.0, act)) return rc;
    const size_t es = dtype_size(dtype);
    if (B == 0 || S == 0) {
        for (void *p : {dgamma, dbeta})
            if (p) J4C_CUDA(cudaMemsetAsync(p, 0, (size_t)C * es, as_stream(stream)));
        return J4C_OK;
    }
    J4C_REQUIRE(x && mean && rstd && dy && dx, "j4c_group_norm_grad: NULL pointer");
    const size_t need = j4c_group_norm_workspace(dtype, B, S, C, groups, 1);
    J4C_REQUIRE(ws && aligned16(ws) && ws_bytes >= need, "j4c_group_norm_grad: needs %zu bytes of workspace", need);
    auto run = [&](auto t) {
        using T = decltype(t);
        const bool sums = dgamma || dbeta;
        Args<T> a{B, S, C, groups, C / groups, (const T *)x, (const T *)gamma, (const T *)beta, (const T *)dy,
                  (T *)mean, (T *)rstd, T(0), act, (T *)dx, sums ? (T *)ws : nullptr};
        return group_norm<T>(a, true, (T *)dgamma, (T *)dbeta, ws, as_stream(stream));
    };
    return dtype == J4C_FLOAT64 ? run(0.0) : run(0.0f);
}

}  // extern "C"
