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
//    norm) are held in registers by 1 to 32 warps, sixteen values a thread where
//    they come four at a time, else eight: every value is read once, and while a
//    group is worked on the thread's values of the next one are on their way to
//    shared memory (cp.async).  Backward a warp set keeps its group and walks
//    over samples, so dgamma and dbeta gather in registers too.
//  * Larger groups are cut into tiles of rows.  Forward, one kernel leaves every
//    tile's mean and squared differences per group -- of a thread's batch of
//    values from registers, merged by Chan, Golub and LeVeque's pairwise update,
//    so one read is enough; a second one merges the tiles' in FP64 and applies.
//    Backward the same with the tiles' sums of h and h xhat.  The second read
//    of a tile comes from L2: the batch is walked in parts of kL2Part bytes.
#include <algorithm>
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "rows_sum.cuh"

namespace j4c {
namespace {

template <typename T, int V>
constexpr int kHeld = sizeof(T) * V == 16 && V == 4 ? 16 : 8;  // values a thread holds
constexpr int64_t kMaxHeld = 8192;
constexpr int kTileThreads = 512;    // at most: a tile's CTA has whole rows of columns
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

// An asynchronous copy of 4, 8 or 16 bytes to shared memory.
template <typename V>
__device__ __forceinline__ void copy_async(V *to, const V *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from),
                 "n"(sizeof(V))
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last LEFT committed groups have arrived.
template <int LEFT>
__device__ __forceinline__ void copies_done() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
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

// Threads an SM: 64 registers each, and 128 where two arrays and their sums of
// sixteen values are held.
template <typename T, int V, bool BACKWARD>
constexpr int kResident = kHeld<T, V> == 16 && BACKWARD ? 512 : 1024;

// The sum over a set.  Consecutive sums alternate between two buffers: a
// barrier of the second is behind every read of the first.
template <typename T, int WARPS>
__device__ __forceinline__ T set_sum(T v, T *buf, int set) {
    v = warp_sum(v);
    if constexpr (WARPS > 1) {
        const int warp = (threadIdx.x / 32) % WARPS;
        if (threadIdx.x % 32 == 0) buf[set * WARPS + warp] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + set), "n"(32 * WARPS) : "memory");
        v = buf[set * WARPS + threadIdx.x % WARPS];
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// Where thread t of a set finds its values: value i * V + e of those it holds is
// channel col[i] + e of the group, off[i] + e elements behind the group's first.
template <int V, int WARPS, int NV>
struct Place {
    uint32_t off[NV];
    int col[NV];
    __device__ __forceinline__ Place(int t, int64_t S, int64_t C, int64_t D) {
        const int per_row = (int)(D / V), all = (int)(S * per_row);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int v = t + i * Held<WARPS>::THREADS;
            const int s = v / per_row;
            col[i] = v < all ? (v - s * per_row) * V : -1;
            off[i] = (uint32_t)((int64_t)s * C + col[i]);
        }
    }
};

// A thread's slots in shared memory for its values of an item: slot i of
// thread t at i * blockDim + t.  Nobody else touches them.  Two sets of slots
// take turns: the copies of the next item start before the current one is
// read, into the set whose values the item before has used up.  FLOAT64
// backward has room for one set only, and no item ahead.
template <typename T, bool BACKWARD>
constexpr int kAhead = sizeof(T) == 8 && BACKWARD ? 0 : 1;
template <typename T, int V, int WARPS, int NV>
__device__ __forceinline__ void fetch(Vec<T, V> *slots, const T *from, const Place<V, WARPS, NV> &at) {
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (at.col[i] >= 0)
            copy_async(slots + i * blockDim.x + threadIdx.x, reinterpret_cast<const Vec<T, V> *>(from + at.off[i]));
}
template <typename T, int V, int WARPS, int NV>
__device__ __forceinline__ void take(const Vec<T, V> *slots, T (&x)[kHeld<T, V>], const Place<V, WARPS, NV> &at) {
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (at.col[i] >= 0) {
            const Vec<T, V> v = slots[i * blockDim.x + threadIdx.x];
#pragma unroll
            for (int e = 0; e < V; e++) x[i * V + e] = v.e[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[i * V + e] = T(0);
        }
}
template <typename T, int V, int WARPS, int NV>
__device__ __forceinline__ void put(T *to, const T (&x)[kHeld<T, V>], const Place<V, WARPS, NV> &at) {
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (at.col[i] >= 0) {
            Vec<T, V> v;
#pragma unroll
            for (int e = 0; e < V; e++) v.e[e] = x[i * V + e];
            *reinterpret_cast<Vec<T, V> *>(to + at.off[i]) = v;
        }
}
// The group's parameters of the thread's values (from L1 after the first item).
template <typename T, int V, int WARPS, int NV>
__device__ __forceinline__ void params(const T *p, int64_t c0, T (&v)[kHeld<T, V>], const Place<V, WARPS, NV> &at) {
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (at.col[i] >= 0) {
            const Vec<T, V> w = *reinterpret_cast<const Vec<T, V> *>(p + c0 + at.col[i]);
#pragma unroll
            for (int e = 0; e < V; e++) v[i * V + e] = w.e[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) v[i * V + e] = T(0);
        }
}

template <typename T, int V, int WARPS>
__global__ void __launch_bounds__(32 * Held<WARPS>::CTA, kResident<T, V, false> / (32 * Held<WARPS>::CTA))
held_forward_kernel(const Args<T> a) {
    using H = Held<WARPS>;
    constexpr int NV = kHeld<T, V> / V;
    __shared__ T sums[2][H::CTA];
    extern __shared__ __align__(16) unsigned char raw[];
    Vec<T, V> *slots = reinterpret_cast<Vec<T, V> *>(raw);
    const int set = threadIdx.x / H::THREADS, t = threadIdx.x % H::THREADS;
    const Place<V, WARPS, NV> at(t, a.S, a.C, a.D);
    const int64_t items = a.B * a.G, step = (int64_t)gridDim.x * H::SETS;
    const T n = (T)(a.S * a.D);
    const int64_t sample = a.S * a.C, b_step = step / a.G, g_step = step - b_step * a.G;
    const int turn = NV * blockDim.x;
    int64_t item = (int64_t)blockIdx.x * H::SETS + set;
    int64_t b = item / a.G, g = item - b * a.G;
    if (item < items) fetch(slots, a.x + b * sample + g * a.D, at);
    copies_commit();
    for (int now = 0; item < items; item += step, now ^= 1) {
        const int64_t base = b * sample + g * a.D, c0 = g * a.D;
        T x[kHeld<T, V>], p[kHeld<T, V>];
        b += b_step, g += g_step;  // the next item's, without a division
        if (g >= a.G) b++, g -= a.G;
        if (item + step < items) fetch(slots + (now ^ 1) * turn, a.x + b * sample + g * a.D, at);
        copies_commit();
        copies_done<1>();
        take(slots + now * turn, x, at);
        T sum = T(0);
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++) sum += x[i];
        const T mean = set_sum<T, WARPS>(sum, sums[0], set) / n;
        T sq = T(0);
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++)
            if (at.col[i / V] >= 0) {
                x[i] -= mean;
                sq += x[i] * x[i];
            }
        const T rstd = inv_sqrt(set_sum<T, WARPS>(sq, sums[1], set) / n + a.eps);
        if (t == 0 && a.mean) {
            a.mean[item] = mean;
            a.rstd[item] = rstd;
        }
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++) x[i] *= rstd;
        if (a.gamma) {
            params(a.gamma, c0, p, at);
#pragma unroll
            for (int i = 0; i < kHeld<T, V>; i++) x[i] *= p[i];
        }
        if (a.beta) {
            params(a.beta, c0, p, at);
#pragma unroll
            for (int i = 0; i < kHeld<T, V>; i++) x[i] += p[i];
        }
        act_values(a.act, x);
        put(a.y + base, x, at);
    }
}

// Set k of the grid holds group k % G and walks over samples k / G, k / G + nb, ...
// (nb sets for every group).  a.dpart, unless NULL, gets its sums over samples
// and positions: [nb, C] of du, then [nb, C] of du xhat.
template <typename T, int V, int WARPS>
__global__ void __launch_bounds__(32 * Held<WARPS>::CTA, kResident<T, V, true> / (32 * Held<WARPS>::CTA))
held_backward_kernel(const Args<T> a, int64_t nb) {
    using H = Held<WARPS>;
    constexpr int NV = kHeld<T, V> / V;
    __shared__ T sums[2][H::CTA];
    extern __shared__ __align__(16) unsigned char raw[];
    constexpr int AHEAD = kAhead<T, true>;
    const int turn = NV * blockDim.x;
    Vec<T, V> *xs = reinterpret_cast<Vec<T, V> *>(raw), *ds = xs + (1 + AHEAD) * turn;
    const int set = threadIdx.x / H::THREADS, t = threadIdx.x % H::THREADS;
    const Place<V, WARPS, NV> at(t, a.S, a.C, a.D);
    const int64_t k = (int64_t)blockIdx.x * H::SETS + set;
    const bool on = k < nb * a.G;  // a whole set: the barriers in the loop are the set's own
    const int64_t g = k % a.G, sample = a.S * a.C;
    const T n = (T)(a.S * a.D);
    T du_sum[kHeld<T, V>], dux_sum[kHeld<T, V>];
#pragma unroll
    for (int i = 0; i < kHeld<T, V>; i++) du_sum[i] = dux_sum[i] = T(0);
    auto fetch_both = [&](int64_t sb, int to) {
        if (sb < a.B) {
            fetch(xs + to * turn, a.x + sb * sample + g * a.D, at);
            fetch(ds + to * turn, a.dy + sb * sample + g * a.D, at);
        }
        copies_commit();
    };
    int64_t b = on ? k / a.G : a.B;
    if (AHEAD) fetch_both(b, 0);
    for (int now = 0; b < a.B; b += nb, now ^= AHEAD) {
        fetch_both(b + AHEAD * nb, now ^ AHEAD);
        const T mean = a.mean[b * a.G + g], rstd = a.rstd[b * a.G + g];
        T x[kHeld<T, V>], h[kHeld<T, V>], u[kHeld<T, V>], p[kHeld<T, V>];
        copies_done<AHEAD>();
        take(xs + now * turn, x, at);
        take(ds + now * turn, h, at);
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++) x[i] = at.col[i / V] >= 0 ? (x[i] - mean) * rstd : T(0);
        if (a.act != J4C_ACT_NONE) {
#pragma unroll
            for (int i = 0; i < kHeld<T, V>; i++) u[i] = x[i];
            if (a.gamma) {
                params(a.gamma, g * a.D, p, at);
#pragma unroll
                for (int i = 0; i < kHeld<T, V>; i++) u[i] *= p[i];
            }
            if (a.beta) {
                params(a.beta, g * a.D, p, at);
#pragma unroll
                for (int i = 0; i < kHeld<T, V>; i++) u[i] += p[i];
            }
            act_slopes(a.act, u, h);
        }
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++) {
            du_sum[i] += h[i];
            dux_sum[i] += h[i] * x[i];
        }
        if (a.gamma) {
            params(a.gamma, g * a.D, p, at);
#pragma unroll
            for (int i = 0; i < kHeld<T, V>; i++) h[i] *= p[i];
        }
        T s1 = T(0), s2 = T(0);
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++) {
            s1 += h[i];
            s2 += h[i] * x[i];
        }
        s1 = set_sum<T, WARPS>(s1, sums[0], set) / n;
        s2 = set_sum<T, WARPS>(s2, sums[1], set) / n;
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++) x[i] = rstd * (h[i] - s1 - x[i] * s2);
        put(a.y + b * sample + g * a.D, x, at);
    }
    if (!a.dpart) return;
    // sums over samples: now over the positions of a channel, through shared
    // memory (the slots' space: every set's copies have been read)
    copies_done<0>();
    __syncthreads();
    T *buf = reinterpret_cast<T *>(raw) + (size_t)set * H::THREADS * kHeld<T, V>;
    for (int which = 0; which < 2; which++) {
#pragma unroll
        for (int i = 0; i < kHeld<T, V>; i++)
            if (at.col[i / V] >= 0) {
                const int64_t s = (at.off[i / V] - (uint32_t)at.col[i / V]) / (uint32_t)a.C;
                buf[s * a.D + at.col[i / V] + i % V] = which ? dux_sum[i] : du_sum[i];
            }
        __syncthreads();
        if (on)
            for (int c = t; c < a.D; c += H::THREADS) {
                T v = T(0);
                for (int s0 = 0; s0 < a.S; s0 += 64) {  // up to 8192 positions: 64 at a time
                    T w = T(0);
                    for (int s = s0; s < min((int)a.S, s0 + 64); s++) w += buf[s * a.D + c];
                    v += w;
                }
                a.dpart[((int64_t)which * nb + k / a.G) * a.C + g * a.D + c] = v;
            }
        __syncthreads();
    }
}

// ---- groups cut into tiles ------------------------------------------------------------
// A tile is `rows` positions of one sample by some channels: whole groups
// (per > 0 of them), or a stretch of one group wider than kTileChannels
// (per = 0, `cuts` stretches a group).
struct Geo {
    int64_t S, C, G, D;
    int rows, row_tiles, width, col_tiles, per, cuts;
    int dcols;  // columns of V channels of a group (of a tile, where per = 0)
    __host__ __device__ int parts() const { return row_tiles * cuts; }  // tiles of a (sample, group)
};

struct Tile {
    int64_t b, c0, g0;
    int r0, rows, width, groups, cut;
    // grid: row tiles, column tiles, samples
    __device__ __forceinline__ explicit Tile(const Geo &q) {
        const int ct = blockIdx.y;
        b = blockIdx.z;
        r0 = blockIdx.x * q.rows;
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
        rows = cols >= (int)blockDim.x ? 1 : blockDim.x / cols;
        j = cols >= (int)blockDim.x ? threadIdx.x : threadIdx.x % cols;
        r = cols >= (int)blockDim.x ? 0 : threadIdx.x / cols;
        on = r < rows;
    }
};

// Every group of the tile by a power of two of lanes, as many as there are
// threads for (at most a warp): body(group, whether it is one, lane, lanes).
// All threads get there as often.
template <typename Body>
__device__ __forceinline__ void by_group(int groups, Body body) {
    int lanes = 1;
    while (lanes < 32 && 2 * lanes * groups <= (int)blockDim.x) lanes *= 2;
    for (int g0 = 0; g0 < groups; g0 += blockDim.x / lanes) {
        const int g = g0 + threadIdx.x / lanes;
        body(g, g < groups, threadIdx.x % lanes, lanes);
    }
}
template <typename T>
__device__ __forceinline__ T lanes_sum(T v, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A thread's values of a column, in batches of VALUES whose loads are in flight
// together: f(the batch's first row, whether it is whole, its rows) -- whole
// batches, but for the last, without a test for every row.
template <int V, int VALUES>
constexpr int kRows = VALUES / V;
template <int U, typename F>
__device__ __forceinline__ void by_batch(const Lanes &l, int rows, F f) {
    int left = (rows - l.r + l.rows - 1) / l.rows, r = l.r;
    for (; left >= U; left -= U, r += U * l.rows) f(r, std::true_type{}, U);
    if (left > 0) f(r, std::false_type{}, left);
}
template <bool WHOLE, typename T, int V, int N>
__device__ __forceinline__ void load_rows(T (&x)[N], const T *p, int64_t pitch, int rows) {
#pragma unroll
    for (int i = 0; i < N / V; i++, p += pitch) {
        Vec<T, V> v{};
        if (WHOLE || i < rows) v = *reinterpret_cast<const Vec<T, V> *>(p);
#pragma unroll
        for (int e = 0; e < V; e++) x[i * V + e] = v.e[e];
    }
}
template <bool WHOLE, typename T, int V, int N>
__device__ __forceinline__ void store_rows(T *p, const T (&x)[N], int64_t pitch, int rows) {
#pragma unroll
    for (int i = 0; i < N / V; i++, p += pitch) {
        Vec<T, V> v;
#pragma unroll
        for (int e = 0; e < V; e++) v.e[e] = x[i * V + e];
        if (WHOLE || i < rows) *reinterpret_cast<Vec<T, V> *>(p) = v;
    }
}

// (mean, m2) of n values joined by those of n2 more.
template <typename T>
__device__ __forceinline__ void join(T &n, T &mean, T &m2, T n2, T mean2, T m22) {
    const T all = n + n2, d = mean2 - mean, share = n2 / all;
    mean += d * share;
    m2 += m22 + d * d * (n * share);
    n = all;
}

// stats[((b G + g) parts + part) 2] = mean, sum of squared differences from it, of a tile's part of a group.
template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads, 2) tile_stats_kernel(const Args<T> a, const Geo q,
                                                                     T *__restrict__ stats) {
    constexpr int N = 16, U = kRows<V, N>;
    extern __shared__ __align__(16) unsigned char raw[];
    T *red = reinterpret_cast<T *>(raw);  // (mean, m2) of [lanes of rows][columns]
    const Tile w(q);
    const Lanes l(w.width, V);
    const T *x = a.x + (w.b * q.S + w.r0) * q.C + w.c0;
    const int64_t pitch = l.rows * q.C;
    if (l.on)
        for (int j = l.j; j < l.cols; j += blockDim.x) {
            T n = T(0), mean = T(0), m2 = T(0);
            by_batch<U>(l, w.rows, [&](int r, auto whole, int rows) {
                constexpr bool WHOLE = decltype(whole)::value;
                T v[N];
                load_rows<WHOLE, T, V>(v, x + r * q.C + j * V, pitch, rows);
                T sum = T(0), sq = T(0);
#pragma unroll
                for (int i = 0; i < N; i++) sum += v[i];
                const T count = (T)(rows * V), mb = WHOLE ? sum * T(1.0 / N) : sum / count;
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (WHOLE || i / V < rows) sq += (v[i] - mb) * (v[i] - mb);
                if (r == l.r) n = count, mean = mb, m2 = sq;
                else join(n, mean, m2, count, mb, sq);
            });
            red[2 * (l.r * l.cols + j)] = mean;
            red[2 * (l.r * l.cols + j) + 1] = m2;
        }
    __syncthreads();
    // the threads of a group: lane r of a column has rows r, r + l.rows, ...
    by_group(w.groups, [&](int g, bool is, int lane, int lanes) {
        auto each = [&](auto f) {
            if (!is) return;
            for (int r = 0; r < l.rows && r < w.rows; r++) {
                const T n = (T)(V * ((w.rows - r + l.rows - 1) / l.rows));
                const T *p = red + 2 * (r * l.cols + g * q.dcols);
                const int cols = min(q.dcols, l.cols - g * q.dcols);
                for (int k = lane; k < cols; k += lanes) f(n, p + 2 * k);
            }
        };
        T sum = T(0), m2 = T(0);
        each([&](T n, const T *p) { sum += n * p[0]; });
        const T mean = lanes_sum(sum, lanes) / (T)((int64_t)w.rows * (q.per ? (int)q.D : w.width));
        each([&](T n, const T *p) { m2 += p[1] + n * (p[0] - mean) * (p[0] - mean); });
        m2 = lanes_sum(m2, lanes);
        if (is && lane == 0) {
            T *s = stats + 2 * ((w.b * q.G + w.g0 + g) * q.parts() + (int)blockIdx.x * q.cuts + w.cut);
            s[0] = mean;
            s[1] = m2;
        }
    });
}

template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads, 2) tile_apply_kernel(const Args<T> a, const Geo q,
                                                                     const T *__restrict__ stats) {
    constexpr int N = 8, U = kRows<V, N>;
    extern __shared__ __align__(16) unsigned char raw[];
    const Tile w(q);
    T *means = reinterpret_cast<T *>(raw), *rstds = means + w.groups;
    const double n = (double)q.S * q.D;
    by_group(w.groups, [&](int g, bool is, int lane, int lanes) {
        const T *s = stats + 2 * (w.b * q.G + w.g0 + g) * q.parts();
        const int parts = q.parts();
        double sum = 0.0, m2 = 0.0, mean;
        if (q.cuts == 1) {
            // every part but the last has `full` values: weights come in once
            const int64_t cols = q.D, last_rows = q.S - (int64_t)(q.row_tiles - 1) * q.rows;
            const double full = (double)(q.rows * cols), less = full - (double)(last_rows * cols);
            const double tail = is ? (double)s[2 * parts - 2] : 0.0;
            if (is) {
#pragma unroll 4
                for (int p = lane; p < parts; p += lanes) sum += (double)s[2 * p];
            }
            mean = (lanes_sum(sum, lanes) * full - less * tail) / n;
            double sq = 0.0;
            if (is) {
#pragma unroll 4
                for (int p = lane; p < parts; p += lanes) {
                    const double d = (double)s[2 * p] - mean;
                    sq += d * d;
                    m2 += (double)s[2 * p + 1];
                }
            }
            m2 = lanes_sum(m2 + full * sq, lanes) - less * (tail - mean) * (tail - mean);
        } else {
            auto count = [&](int p) {
                const int64_t cols = p % q.cuts == q.cuts - 1 ? q.D - (int64_t)(q.cuts - 1) * q.width : q.width;
                const int64_t rows = p / q.cuts == q.row_tiles - 1 ? q.S - (int64_t)(q.row_tiles - 1) * q.rows : q.rows;
                return (double)(rows * cols);
            };
            if (is)
                for (int p = lane; p < parts; p += lanes) sum += count(p) * (double)s[2 * p];
            mean = lanes_sum(sum, lanes) / n;
            if (is)
                for (int p = lane; p < parts; p += lanes) {
                    const double d = (double)s[2 * p] - mean;
                    m2 += (double)s[2 * p + 1] + count(p) * d * d;
                }
            m2 = lanes_sum(m2, lanes);
        }
        if (is && lane == 0) {
            means[g] = (T)mean;
            rstds[g] = inv_sqrt((T)((m2 < 0.0 ? 0.0 : m2) / n) + a.eps);  // NaN stays
            if (w.r0 == 0 && w.cut == 0 && a.mean) {
                a.mean[w.b * q.G + w.g0 + g] = means[g];
                a.rstd[w.b * q.G + w.g0 + g] = rstds[g];
            }
        }
    });
    __syncthreads();
    const Lanes l(w.width, V);
    const int64_t base = (w.b * q.S + w.r0) * q.C + w.c0, pitch = l.rows * q.C;
    if (!l.on) return;
    for (int j = l.j; j < l.cols; j += blockDim.x) {
        const int g = j / q.dcols;
        const T mean = means[g];
        T scale[V], shift[V];
#pragma unroll
        for (int e = 0; e < V; e++) {
            scale[e] = a.gamma ? rstds[g] * a.gamma[w.c0 + j * V + e] : rstds[g];
            shift[e] = a.beta ? a.beta[w.c0 + j * V + e] : T(0);
        }
        by_batch<U>(l, w.rows, [&](int r, auto whole, int rows) {
            constexpr bool WHOLE = decltype(whole)::value;
            const int64_t at = base + r * q.C + j * V;
            T u[N];
            load_rows<WHOLE, T, V>(u, a.x + at, pitch, rows);
#pragma unroll
            for (int i = 0; i < N; i++) u[i] = (u[i] - mean) * scale[i % V] + shift[i % V];
            act_values(a.act, u);
            store_rows<WHOLE, T, V>(a.y + at, u, pitch, rows);
        });
    }
}

// A column's parameters in the gradient.
template <typename T, int V>
struct Column {
    T mean, rstd, gm[V], bt[V];
    __device__ __forceinline__ void set(const Args<T> &a, int64_t bg, int64_t c) {
        mean = a.mean[bg], rstd = a.rstd[bg];
#pragma unroll
        for (int e = 0; e < V; e++) {
            gm[e] = a.gamma ? a.gamma[c + e] : T(1);
            bt[e] = a.beta ? a.beta[c + e] : T(0);
        }
    }
    // x <- xhat, d <- du, for a batch of x and dy
    __device__ __forceinline__ void du(int act, T (&x)[8], T (&d)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (x[i] - mean) * rstd;
        if (act != J4C_ACT_NONE) {
            T u[8];
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = x[i] * gm[i % V] + bt[i % V];
            act_slopes(act, u, d);
        }
    }
};

// hsums[((b G + g) parts + part) 2] = sum of h, of h xhat, over a tile's part of
// a group; and, unless a.dpart is NULL, its per-channel sums over the tile's
// rows: dpart[(b row_tiles + rt) C + c] of du, `half` behind it of du xhat.
template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads, 2) tile_sums_kernel(const Args<T> a, const Geo q, int64_t half,
                                                                    T *__restrict__ hsums) {
    constexpr int N = 8, U = kRows<V, N>;
    extern __shared__ __align__(16) unsigned char raw[];
    T *red = reinterpret_cast<T *>(raw);  // [2][lanes of rows][width]
    const Tile w(q);
    const Lanes l(w.width, V);
    const int64_t base = (w.b * q.S + w.r0) * q.C + w.c0, pitch = l.rows * q.C;
    if (l.on)
        for (int j = l.j; j < l.cols; j += blockDim.x) {
            Column<T, V> k;
            k.set(a, w.b * q.G + w.g0 + j / q.dcols, w.c0 + j * V);
            T s1[V], s2[V];
#pragma unroll
            for (int e = 0; e < V; e++) s1[e] = s2[e] = T(0);
            by_batch<U>(l, w.rows, [&](int r, auto whole, int rows) {
                constexpr bool WHOLE = decltype(whole)::value;
                const int64_t at = base + r * q.C + j * V;
                T x[N], d[N];
                load_rows<WHOLE, T, V>(x, a.x + at, pitch, rows);
                load_rows<WHOLE, T, V>(d, a.dy + at, pitch, rows);
                k.du(a.act, x, d);
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (WHOLE || i / V < rows) {  // behind the tile x is 0, which may lie at infinity from the mean
                        s1[i % V] += d[i];
                        s2[i % V] += d[i] * x[i];
                    }
            });
#pragma unroll
            for (int e = 0; e < V; e++) {
                red[l.r * w.width + j * V + e] = s1[e];
                red[(l.rows + l.r) * w.width + j * V + e] = s2[e];
            }
        }
    __syncthreads();
    // over the lanes of rows: red[which][0][c] is the channel's sum
    const int64_t row = (w.b * q.row_tiles + (int)blockIdx.x) * q.C + w.c0;
    for (int c = threadIdx.x; c < 2 * w.width; c += blockDim.x) {
        const int which = c >= w.width, cc = c - which * w.width;
        T v = T(0);
        for (int r = 0; r < l.rows; r++) v += red[(which * l.rows + r) * w.width + cc];
        red[which * l.rows * w.width + cc] = v;
        if (a.dpart) a.dpart[which * half + row + cc] = v;
    }
    __syncthreads();
    const int part = (int)blockIdx.x * q.cuts + w.cut, span = q.per ? (int)q.D : w.width;
    by_group(w.groups, [&](int g, bool is, int lane, int lanes) {
        T s1 = T(0), s2 = T(0);
        if (is)
            for (int k = lane; k < span; k += lanes) {
                const int c = g * span + k;
                const T gm = a.gamma ? a.gamma[w.c0 + c] : T(1);
                s1 += gm * red[c];
                s2 += gm * red[l.rows * w.width + c];
            }
        s1 = lanes_sum(s1, lanes);
        s2 = lanes_sum(s2, lanes);
        if (is && lane == 0) {
            T *s = hsums + 2 * ((w.b * q.G + w.g0 + g) * q.parts() + part);
            s[0] = s1;
            s[1] = s2;
        }
    });
}

template <typename T, int V>
__global__ void __launch_bounds__(kTileThreads, 2) tile_grad_kernel(const Args<T> a, const Geo q,
                                                                    const T *__restrict__ hsums) {
    constexpr int N = 8, U = kRows<V, N>;
    extern __shared__ __align__(16) unsigned char raw[];
    const Tile w(q);
    T *mean_h = reinterpret_cast<T *>(raw), *mean_hx = mean_h + w.groups;
    by_group(w.groups, [&](int g, bool is, int lane, int lanes) {
        const T *s = hsums + 2 * (w.b * q.G + w.g0 + g) * q.parts();
        T s1 = T(0), s2 = T(0);
        if (is)
#pragma unroll 4
            for (int p = lane; p < q.parts(); p += lanes) {
                s1 += s[2 * p];
                s2 += s[2 * p + 1];
            }
        s1 = lanes_sum(s1, lanes);
        s2 = lanes_sum(s2, lanes);
        if (is && lane == 0) {
            mean_h[g] = s1 / (T)(q.S * q.D);
            mean_hx[g] = s2 / (T)(q.S * q.D);
        }
    });
    __syncthreads();
    const Lanes l(w.width, V);
    const int64_t base = (w.b * q.S + w.r0) * q.C + w.c0, pitch = l.rows * q.C;
    if (!l.on) return;
    for (int j = l.j; j < l.cols; j += blockDim.x) {
        const int g = j / q.dcols;
        Column<T, V> k;
        k.set(a, w.b * q.G + w.g0 + g, w.c0 + j * V);
        const T h1 = mean_h[g], h2 = mean_hx[g];
        by_batch<U>(l, w.rows, [&](int r, auto whole, int rows) {
            constexpr bool WHOLE = decltype(whole)::value;
            const int64_t at = base + r * q.C + j * V;
            T x[N], d[N];
            load_rows<WHOLE, T, V>(x, a.x + at, pitch, rows);
            load_rows<WHOLE, T, V>(d, a.dy + at, pitch, rows);
            k.du(a.act, x, d);
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = k.rstd * (d[i] * k.gm[i % V] - h1 - x[i] * h2);
            store_rows<WHOLE, T, V>(a.y + at, x, pitch, rows);
        });
    }
}

// ---- host ----------------------------------------------------------------------------
inline bool held(int64_t S, int64_t C, int64_t G) {
    const int64_t D = C / G;
    return D <= kMaxHeld && S <= kMaxHeld && S * D <= kMaxHeld && S * C < (1ll << 32);
}

template <typename T>
Geo make_geo(int64_t B, int64_t S, int64_t C, int64_t G) {
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
    // Tiles of about 192 KB, as many as fill whole waves of two CTAs an SM: a tile
    // costs its threads some 500 instructions beside its values.  At least four rows.
    const int64_t slots = (int64_t)sm_count() * 2;
    const int64_t target = std::max<int64_t>(4, 192 * 1024 / ((int64_t)q.width * sizeof(T)));
    const int64_t waves = std::max<int64_t>(1, (B * S * q.col_tiles + target * slots / 2) / (target * slots));
    const int64_t per_sample = std::max<int64_t>(1, waves * slots / (B * q.col_tiles));  // tiles of rows
    const int64_t rows = std::min(S, std::max<int64_t>(4, ceil_div(S, per_sample)));
    q.rows = (int)rows;
    q.row_tiles = (int)ceil_div(S, rows);
    return q;
}

int64_t samples_of_part(int64_t B, int64_t bytes_per_sample) {
    return std::max<int64_t>(1, std::min(B, kL2Part / std::max<int64_t>(1, bytes_per_sample)));
}

// Warps that hold a group of n values.
template <typename T, int V>
int held_warps(int64_t n) {
    int warps = 1;
    while (warps * 32 * kHeld<T, V> < n) warps *= 2;
    return warps;
}

// Backward, the sets that share a group's samples: as many as are resident, more
// where one would add more than kMaxTerms of them, no more than samples.
template <typename T, int V>
int64_t held_sets(int64_t B, int64_t G, int warps) {
    const int cta = std::max(8, warps);
    const int64_t resident = (int64_t)sm_count() * (kResident<T, V, true> / 32 / cta) * (cta / warps);
    return std::min(B, std::max(ceil_div(resident, G), ceil_div(B, kMaxTerms)));
}

template <typename T>
size_t workspace(int64_t B, int64_t S, int64_t C, int64_t G, bool backward) {
    const int64_t es = sizeof(T);
    if (held(S, C, G)) {
        // with either width of vector
        const int64_t n = S * (C / G);
        const int64_t sets = std::max(held_sets<T, 1>(B, G, held_warps<T, 1>(n)), held_sets<T, 4>(B, G, held_warps<T, 4>(n)));
        return backward ? (size_t)(2 * es * C * sets) : 0;
    }
    const int64_t part = samples_of_part(B, (backward ? 2 : 1) * S * C * es);
    const Geo q = make_geo<T>(part, S, C, G);
    // the parts' statistics, and backward the tiles' sums of every channel
    return (size_t)(2 * es * (part * G * q.parts() + (backward ? B * q.row_tiles * C : 0)));
}

template <typename T, int V, int WARPS>
int launch_held(const Args<T> &a, bool backward, T *dgamma, T *dbeta, cudaStream_t s) {
    using H = Held<WARPS>;
    const int threads = 32 * H::CTA;
    const size_t smem = (size_t)threads * kHeld<T, V> * sizeof(T) *
                        (backward ? 2 * (1 + kAhead<T, true>) : 1 + kAhead<T, false>);
    auto allow = [&](auto kernel) {
        return smem > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)
                                : cudaSuccess;
    };
    if (!backward) {
        const int64_t ctas = ceil_div(a.B * a.G, H::SETS);
        const unsigned grid = (unsigned)std::min<int64_t>(ctas, (int64_t)sm_count() * (kResident<T, V, false> / threads));
        J4C_CUDA(allow(held_forward_kernel<T, V, WARPS>));
        held_forward_kernel<T, V, WARPS><<<grid, threads, smem, s>>>(a);
        J4C_LAUNCH_CHECK("held_forward_kernel");
        return J4C_OK;
    }
    const int64_t nb = held_sets<T, V>(a.B, a.G, WARPS);
    if (ceil_div(nb * a.G, H::SETS) >= (1ll << 31)) return set_error(J4C_E_UNSUPPORTED, "j4c_group_norm: too many groups");
    J4C_CUDA(allow(held_backward_kernel<T, V, WARPS>));
    held_backward_kernel<T, V, WARPS><<<(unsigned)ceil_div(nb * a.G, H::SETS), threads, smem, s>>>(a, nb);
    J4C_LAUNCH_CHECK("held_backward_kernel");
    if (a.dpart) {
        sum_rows_kernel<T><<<dim3((unsigned)ceil_div(a.C, 32), 2), 1024, 0, s>>>(a.dpart, nb, a.C, dbeta, dgamma);
        J4C_LAUNCH_CHECK("sum_rows_kernel");
    }
    return J4C_OK;
}

template <typename T, int V>
int run_held(const Args<T> &a, bool backward, T *dgamma, T *dbeta, cudaStream_t s) {
    switch (held_warps<T, V>(a.S * a.D)) {
    case 1: return launch_held<T, V, 1>(a, backward, dgamma, dbeta, s);
    case 2: return launch_held<T, V, 2>(a, backward, dgamma, dbeta, s);
    case 4: return launch_held<T, V, 4>(a, backward, dgamma, dbeta, s);
    case 8: return launch_held<T, V, 8>(a, backward, dgamma, dbeta, s);
    case 16: return launch_held<T, V, 16>(a, backward, dgamma, dbeta, s);
    default:
        if constexpr (kHeld<T, V> == 8) return launch_held<T, V, 32>(a, backward, dgamma, dbeta, s);
        return set_error(J4C_E_UNSUPPORTED, "j4c_group_norm: a group of %lld values", (long long)(a.S * a.D));  // > kMaxHeld
    }
}

template <typename T, int V>
int run_tiles(const Args<T> &whole, bool backward, T *dgamma, T *dbeta, void *ws, cudaStream_t s) {
    const int64_t B = whole.B, S = whole.S, C = whole.C, G = whole.G;
    const int64_t part = samples_of_part(B, (backward ? 2 : 1) * S * C * (int64_t)sizeof(T));
    Geo q = make_geo<T>(part, S, C, G);
    q.dcols = (q.per ? (int)q.D : q.width) / V;
    if (q.col_tiles > 65535 || part > 65535)
        return set_error(J4C_E_UNSUPPORTED, "j4c_group_norm: %lld channels are too many", (long long)C);
    T *stats = static_cast<T *>(ws), *sums = stats + 2 * part * G * q.parts();
    const int cols = q.width / V;
    const int threads = cols >= kTileThreads ? kTileThreads : (int)ceil_div(kTileThreads / cols * cols, 32) * 32;
    const size_t per_group = 2 * (size_t)std::max(q.per, 1) * sizeof(T);
    const size_t stats_smem = 2 * (size_t)std::max(kTileThreads, cols) * sizeof(T);
    const size_t sums_smem = 2 * (size_t)std::max(kTileThreads * V, q.width) * sizeof(T);
    for (int64_t b0 = 0; b0 < B; b0 += part) {
        const int64_t nb = std::min(part, B - b0);
        Args<T> a = whole;
        a.B = nb;
        a.x += b0 * S * C, a.y += b0 * S * C;
        if (a.mean) a.mean += b0 * G, a.rstd += b0 * G;
        const dim3 grid((unsigned)q.row_tiles, (unsigned)q.col_tiles, (unsigned)nb);
        if (!backward) {
            tile_stats_kernel<T, V><<<grid, threads, stats_smem, s>>>(a, q, stats);
            J4C_LAUNCH_CHECK("tile_stats_kernel");
            tile_apply_kernel<T, V><<<grid, threads, per_group, s>>>(a, q, stats);
            J4C_LAUNCH_CHECK("tile_apply_kernel");
            continue;
        }
        a.dy += b0 * S * C;
        if (a.dpart) a.dpart = sums + b0 * q.row_tiles * C;
        tile_sums_kernel<T, V><<<grid, threads, sums_smem, s>>>(a, q, B * q.row_tiles * C, stats);
        J4C_LAUNCH_CHECK("tile_sums_kernel");
        tile_grad_kernel<T, V><<<grid, threads, per_group, s>>>(a, q, stats);
        J4C_LAUNCH_CHECK("tile_grad_kernel");
    }
    if (backward && whole.dpart) {
        sum_rows_kernel<T><<<dim3((unsigned)ceil_div(C, 32), 2), 1024, 0, s>>>(sums, B * q.row_tiles, C, dbeta, dgamma);
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
        return a.D % v == 0 && ok(a.x) && ok(a.y) && ok(a.dy) && ok(a.gamma) && ok(a.beta);
    };
    const int v = fits(W) ? W : W > 2 && fits(2) ? 2 : 1;
    const bool small = held(a.S, a.C, a.G);
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
    J4C_REQUIRE((double)B * (double)S * (double)C < 1e18, "%s: [%lld, %lld, %lld] is too large", name, (long long)B,
                (long long)S, (long long)C);
    return J4C_OK;
}

size_t j4c_group_norm_workspace(int dtype, int64_t B, int64_t S, int64_t C, int64_t groups, int backward) {
    if (B <= 0 || S <= 0 || C < 1 || groups < 1 || C % groups) return 0;
    if ((double)B * (double)S * (double)C >= 1e18) return 0;  // refused by the calls
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
