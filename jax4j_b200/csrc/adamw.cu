// adamw.cu -- the AdamW step of many tensors in one launch.
//
// For every element, with g' = g * scale and t the step being taken:
//   m' = beta1 m + (1 - beta1) g'          v' = beta2 v + (1 - beta2) g'^2
//   w' = w - lr wd w - lr (m' / (1 - beta1^t)) / (sqrt(v' / (1 - beta2^t)) + eps)
// evaluated as m' * a / (sqrt(v') * b + eps) with a = 1 / (1 - beta1^t) and
// b = 1 / sqrt(1 - beta2^t) computed in FP64 from the running powers of the
// betas that travel with the state (no host knows t, so a recorded graph
// counts on).  Every product and sum is rounded on its own (no FMA), so an
// elementwise evaluation of the same expressions gives the same bits (with
// moments in 8 bits the quotient is within 2 ulp).
//
// Bound by HBM with moments in the tensors' type: 28 B per FLOAT32 element (w,
// g, m, v read; w, m, v written), 41.9 M elements in 209 us = 5.6 TB/s.  With
// moments in 8 bits 16.1 B, and bound by instructions (some 100 an element, a
// third of them the IEEE root and quotient and the root's encoding): 172 us =
// 3.9 TB/s; without the copies a chunk ahead 188 us.  All tensors of a tree share
// one launch: the table of pointers travels in the kernel's parameters (no copy
// to the device, nothing a captured graph would have to keep alive), and a CTA
// takes chunks of consecutive elements, finding a chunk's tensor by bisection.
//
// Moments in 8 bits.  A tensor is cut into blocks of 128 elements, half a
// warp's eight elements per lane, so a block's largest value is one reduction
// of registers.  First moments are e4m3 floats; of the second moment the root is
// held (the update needs the root anyway, and it has half the range), in
// unsigned floats of 4 exponent and 4 fraction bits, whose smallest value a
// non-zero root never falls below -- a zero would divide by eps alone.  Each
// code times the block's FLOAT32 step (largest value / largest code) is the
// value.  The step is not rounded to a power of two: a block whose moments all
// decay by beta must follow, and does, through its step.  Rounding to nearest
// costs at most 2^-4 of a first moment and 2^-5 of a root; only the state is
// rounded, the update uses the moments before rounding.
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"

namespace j4c {
namespace {

constexpr int kThreads = 256;
constexpr int kCtas = 4;                 // per SM: 64 registers a thread
constexpr int kQCtas = 3;                // with 8-bit moments, 80 registers a thread (2: 199 us, 4: as fast, with spills)
constexpr int kQBlock = 128;             // elements that share a step
constexpr float kTopM = 448.0f;          // largest e4m3 value
constexpr float kTopR = 480.0f;          // largest code of a root (0xFE; 0xFF is NaN)
constexpr int kSmallTable = 24, kLargeTable = 380;  // tensors of one launch

struct Tensor {
    const void *w, *g, *m, *v;  // 8-bit moments: m is the packed state, v unused
    void *w_out, *m_out, *v_out;
    int64_t n;
    double wd;
    int first;  // its first chunk
    int vec;    // 16-byte loads and stores
};

template <int N>
struct Table {
    Tensor t[N];
    int count;
    int chunks;       // of all tensors
    int chunk_elems;  // a multiple of kThreads * 4
};
static_assert(sizeof(Table<kLargeTable>) <= 32000, "kernel parameters");

struct Hyper {
    const double *steps;  // steps taken, beta1^steps, beta2^steps
    double *steps_out;    // may be NULL
    const float *lr_dev;  // may be NULL: lr
    double lr, scale, beta1, beta2, eps;
};

template <int N>
__device__ __forceinline__ const Tensor &tensor_of(const Table<N> &tab, int chunk) {
    int lo = 0, hi = tab.count - 1;  // the last tensor whose first chunk is not behind `chunk`
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.t[mid].first <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return tab.t[lo];
}

__device__ __forceinline__ float r_sqrt(float x) { return __fsqrt_rn(x); }
__device__ __forceinline__ double r_sqrt(double x) { return __dsqrt_rn(x); }
// r_div without its shortcut for zero dividends, which are rare here
__device__ __forceinline__ float q_div(float a, float b) { return __fdiv_rn(a, b); }
__device__ __forceinline__ double q_div(double a, double b) { return __ddiv_rn(a, b); }
// Within 2 ulp for divisors of 2^-126 to 2^126, and x / 0 as it should be: the
// divisor is a root, 0 or from 2^-75 to 2^64, times b (1 to 2^27), plus eps, which
// the call checks.  No branch, so eight of them overlap.
__device__ __forceinline__ float fast_div(float a, float b) { return __fdividef(a, b); }

// What a step needs beside the elements, in the elements' type.
template <typename T>
struct Coef {
    T scale, b1, c1, b2, c2, a, b, eps, lr;
    bool scaled;

    __device__ __forceinline__ explicit Coef(const Hyper &h) {
        const double p1 = h.steps[1] * h.beta1, p2 = h.steps[2] * h.beta2;
        if (h.steps_out && blockIdx.x == 0 && threadIdx.x == 0) {
            h.steps_out[0] = h.steps[0] + 1.0;
            h.steps_out[1] = p1;
            h.steps_out[2] = p2;
        }
        scale = (T)h.scale;
        scaled = h.scale != 1.0;
        b1 = (T)h.beta1;
        c1 = (T)(1.0 - h.beta1);
        b2 = (T)h.beta2;
        c2 = (T)(1.0 - h.beta2);
        a = (T)(1.0 / (1.0 - p1));
        b = (T)(1.0 / sqrt(1.0 - p2));
        eps = (T)h.eps;
        lr = h.lr_dev ? (T)*h.lr_dev : (T)h.lr;
    }
    // lr * weight decay, rounded once when lr is the host's
    __device__ __forceinline__ T decay(const Hyper &h, double wd) const {
        return h.lr_dev ? (T)((double)*h.lr_dev * wd) : (T)(h.lr * wd);
    }
};

// m, v in: the old moments; out: the new ones and the root of v.  FAST: the
// update's quotient within 2 ulp.
template <typename T, bool FAST = false>
__device__ __forceinline__ T adamw_element(const Coef<T> &k, T decay, T w, T g, T &m, T &v, T &root) {
    if (k.scaled) g = r_mul(g, k.scale);
    m = r_add(r_mul(m, k.b1), r_mul(g, k.c1));
    v = r_add(r_mul(v, k.b2), r_mul(r_mul(g, g), k.c2));
    root = r_sqrt(v);
    const T up = r_mul(m, k.a), down = r_add(r_mul(root, k.b), k.eps);
    T update;
    if constexpr (FAST) update = fast_div(up, down);
    else update = q_div(up, down);
    return r_sub(r_sub(w, r_mul(w, decay)), r_mul(update, k.lr));
}

template <typename T>
struct alignas(16) Vec {
    T e[16 / sizeof(T)];
};

// Moments in the elements' type.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads, kCtas) adamw_kernel(const __grid_constant__ Table<N> tab,
                                                         const __grid_constant__ Hyper h) {
    constexpr int V = 16 / sizeof(T);
    const Coef<T> k(h);
    for (int chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
        const Tensor &t = tensor_of(tab, chunk);
        const int64_t from = (int64_t)(chunk - t.first) * tab.chunk_elems;
        const int64_t end = min(t.n, from + tab.chunk_elems);
        const T *w = static_cast<const T *>(t.w), *g = static_cast<const T *>(t.g);
        const T *m = static_cast<const T *>(t.m), *v = static_cast<const T *>(t.v);
        T *wo = static_cast<T *>(t.w_out), *mo = static_cast<T *>(t.m_out), *vo = static_cast<T *>(t.v_out);
        const T decay = k.decay(h, t.wd);
        int64_t done = from;
        if (t.vec) {
            const int64_t vend = from + (end - from) / V * V;
            for (int64_t i = from + threadIdx.x * V; i < vend; i += 2 * kThreads * V) {
                // two vectors of every array in flight: the outputs may be the
                // inputs, so no load moves above an earlier vector's stores
                Vec<T> ww[2], gg[2], mm[2], vv[2];
                const int64_t at[2] = {i, i + kThreads * V};
                const bool both = at[1] < vend;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u == 1 && !both) break;
                    ww[u] = *reinterpret_cast<const Vec<T> *>(w + at[u]);
                    gg[u] = *reinterpret_cast<const Vec<T> *>(g + at[u]);
                    mm[u] = *reinterpret_cast<const Vec<T> *>(m + at[u]);
                    vv[u] = *reinterpret_cast<const Vec<T> *>(v + at[u]);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u == 1 && !both) break;
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        T root;
                        ww[u].e[e] = adamw_element(k, decay, ww[u].e[e], gg[u].e[e], mm[u].e[e], vv[u].e[e], root);
                    }
                    *reinterpret_cast<Vec<T> *>(wo + at[u]) = ww[u];
                    *reinterpret_cast<Vec<T> *>(mo + at[u]) = mm[u];
                    *reinterpret_cast<Vec<T> *>(vo + at[u]) = vv[u];
                }
            }
            done = vend;
        }
        for (int64_t i = done + threadIdx.x; i < end; i += kThreads) {
            T mm = m[i], vv = v[i], root;
            wo[i] = adamw_element(k, decay, w[i], g[i], mm, vv, root);
            mo[i] = mm;
            vo[i] = vv;
        }
    }
}

// ---- moments in 8 bits -----------------------------------------------------------
// A packed state of nb blocks: nb * 32 words of first-moment codes, nb * 32 of
// root codes, nb steps of the first moments, nb steps of the roots.
// Four codes of a word each way.
__device__ __forceinline__ void decode_m(uint32_t codes, float step, float *x) {
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * p)), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        x[2 * p] = r_mul(f.x, step);
        x[2 * p + 1] = r_mul(f.y, step);
    }
}
// Bits 7..4 the exponent, 3..0 the fraction: read as an FP32 number's (its
// subnormals included) and scaled by 2^120, exponent 0 is 2^-6 and below it
// the code counts 2^-10s.  0xFF is NaN.
__device__ __forceinline__ void decode_r(uint32_t codes, float step, float *x) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t at = e < 3 ? codes << (19 - 8 * e) : codes >> 5;  // this code's bits at 26..19
        x[e] = r_mul(r_mul(__uint_as_float(at & (0xFFu << 19)), 0x1p120f), step);
    }
    const uint32_t z = ~codes;
    if ((z - 0x01010101u) & codes & 0x80808080u) {  // a byte of z is zero
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (((codes >> (8 * e)) & 0xFFu) == 0xFFu) x[e] = __int_as_float(0x7FC00000);
    }
}
__device__ __forceinline__ uint32_t encode_m(const float *y) {
    uint32_t c = 0;
#pragma unroll
    for (int p = 0; p < 2; p++)
        c |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[2 * p], y[2 * p + 1]), __NV_SATFINITE, __NV_E4M3)
             << (16 * p);
    return c;
}
// y >= 0 and finite.
__device__ __forceinline__ uint32_t encode_r(float y) {
    const uint32_t b = __float_as_uint(y);
    const uint32_t big = min(((b + 0x3FFFFu + ((b >> 19) & 1u)) >> 19) - (120u << 4), 0xFEu);
    // 8192 counts in steps of 2^-10: the sum's low bits are y rounded to them
    uint32_t small = __float_as_uint(__fadd_rn(y, 8192.0f)) & 0x1Fu;
    small = max(small, y > 0.0f ? 1u : 0u);
    return y < 0x1p-6f ? small : big;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
constexpr uint32_t kInfBits = 0x7F800000u;
// The factor that brings a block's largest value to the largest code, and the
// step that brings it back; a block below 2^-100 is held as zeros (its inverse
// would overflow; no root of a FLOAT32 second moment lies there).
__device__ __forceinline__ void block_scale(uint32_t top_bits, float top_code, float &inv, float &step) {
    const float top = __uint_as_float(top_bits);
    const bool held = top >= 0x1p-100f;
    inv = held ? r_mul(__frcp_rn(top), top_code) : 0.0f;
    step = held ? r_mul(top, 1.0f / top_code) : 0.0f;
}

// A warp takes two neighbouring blocks, half a warp each and eight elements a
// lane: what a lane computes for its block (addresses, the step, its inverse)
// is shared by eight.
__device__ __forceinline__ uint32_t half_max(uint32_t v) {
    return __reduce_max_sync(threadIdx.x % 32 < 16 ? 0x0000FFFFu : 0xFFFF0000u, v);
}
struct Packed {  // a packed state's parts
    uint32_t *m, *r;
    float *steps_m, *steps_r;
    __device__ __forceinline__ Packed(const void *q, int64_t nb) {
        m = static_cast<uint32_t *>(const_cast<void *>(q));
        r = m + nb * 32;
        steps_m = reinterpret_cast<float *>(r + nb * 32);
        steps_r = steps_m + nb;
    }
};
// Eight codes of a lane, at word `at`: one load where the state is 8-byte aligned.
__device__ __forceinline__ uint2 load_codes(const uint32_t *p, int64_t at, bool vec) {
    return vec ? *reinterpret_cast<const uint2 *>(p + at) : make_uint2(p[at], p[at + 1]);
}
__device__ __forceinline__ void store_codes(uint32_t *p, int64_t at, bool vec, uint2 c) {
    if (vec) *reinterpret_cast<uint2 *>(p + at) = c;
    else p[at] = c.x, p[at + 1] = c.y;
}
// Eight values at p, those from `left` on behind the tensor.
__device__ __forceinline__ void load8(const float *p, int left, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = e < left ? p[e] : 0.0f;
}
__device__ __forceinline__ void store8(float *p, bool whole, int left, const float (&x)[8]) {
    if (whole) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) p[e] = x[e];
    }
}

// What a half warp does of a chunk: one block (a chunk has at most 16).
struct Share {
    int64_t b, i, at, nb;  // the block, its first element and word of the lane, the tensor's blocks
    int left;              // of the lane's elements, those in the tensor
    bool is, vec, whole;   // is there a block; 16-byte loads; of all eight elements
};
template <int N>
__device__ __forceinline__ Share share_of(const Table<N> &tab, const Tensor &t, int chunk) {
    const int lane = threadIdx.x % 16, half = threadIdx.x / 16, per = tab.chunk_elems / kQBlock;
    Share p;
    p.nb = (t.n + kQBlock - 1) / kQBlock;
    p.b = (int64_t)(chunk - t.first) * per + half;
    p.is = half < per && p.b < p.nb;
    p.i = p.b * kQBlock + lane * 8;
    p.at = p.b * 32 + lane * 2;
    p.left = (int)max((int64_t)0, min((int64_t)8, t.n - p.i));
    p.vec = t.vec;
    p.whole = p.vec && p.left == 8;
    return p;
}
template <int BYTES, typename V>
__device__ __forceinline__ void copy_async(V *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from),
                 "n"(BYTES)
                 : "memory");
}

// While a chunk is worked on the next one's values are on their way, to the
// threads' own slots in shared memory (two sets take turns) and the steps to
// registers.
template <int N>
__global__ void __launch_bounds__(kThreads, kQCtas) adamw_q8_kernel(const __grid_constant__ Table<N> tab,
                                                                   const __grid_constant__ Hyper h) {
    __shared__ __align__(16) float4 slots[2][4][kThreads];  // w, g
    __shared__ __align__(16) uint2 codes[2][2][kThreads];   // of m, of the roots
    const Coef<float> k(h);
    const int tid = threadIdx.x;
    float next_m = 0.0f, next_r = 0.0f;
    auto fetch = [&](int64_t chunk, int to) {
        if (chunk < tab.chunks) {
            const Tensor &t = tensor_of(tab, (int)chunk);
            const Share p = share_of(tab, t, (int)chunk);
            if (p.is) {
                const Packed q(t.m, p.nb);
                next_m = q.steps_m[p.b], next_r = q.steps_r[p.b];
                if (p.vec) {
                    copy_async<8>(&codes[to][0][tid], q.m + p.at);
                    copy_async<8>(&codes[to][1][tid], q.r + p.at);
                }
                if (p.whole) {
                    const float *w = static_cast<const float *>(t.w) + p.i, *g = static_cast<const float *>(t.g) + p.i;
                    copy_async<16>(&slots[to][0][tid], w);
                    copy_async<16>(&slots[to][1][tid], w + 4);
                    copy_async<16>(&slots[to][2][tid], g);
                    copy_async<16>(&slots[to][3][tid], g + 4);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(blockIdx.x, 0);
    int turn = 0;
    for (int chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x, turn ^= 1) {
        const Tensor &t = tensor_of(tab, chunk);
        const Share p = share_of(tab, t, chunk);
        const int64_t b = p.b, i = p.i, at = p.at;
        const int left = p.left;
        const bool vec = p.vec, whole = p.whole;
        const Packed q(t.m, p.nb), qo(t.m_out, p.nb);
        float *wo = static_cast<float *>(t.w_out);
        const float decay = k.decay(h, t.wd);
        const float sm = next_m, sr = next_r;
        fetch(chunk + (int64_t)gridDim.x, turn ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (p.is) {
            float ww[8], gg[8], mm[8], rr[8];
            if (whole) {
                const float4 x[4] = {slots[turn][0][tid], slots[turn][1][tid], slots[turn][2][tid], slots[turn][3][tid]};
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    ww[4 * e] = x[e].x, ww[4 * e + 1] = x[e].y, ww[4 * e + 2] = x[e].z, ww[4 * e + 3] = x[e].w;
                    gg[4 * e] = x[2 + e].x, gg[4 * e + 1] = x[2 + e].y, gg[4 * e + 2] = x[2 + e].z, gg[4 * e + 3] = x[2 + e].w;
                }
            } else {
                load8(static_cast<const float *>(t.w) + i, left, ww);
                load8(static_cast<const float *>(t.g) + i, left, gg);
            }
            const uint2 cm = vec ? codes[turn][0][tid] : load_codes(q.m, at, false);
            const uint2 cr = vec ? codes[turn][1][tid] : load_codes(q.r, at, false);
            decode_m(cm.x, sm, mm);
            decode_m(cm.y, sm, mm + 4);
            decode_r(cr.x, sr, rr);
            decode_r(cr.y, sr, rr + 4);
            uint32_t top_m = 0, top_r = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float v = r_mul(rr[e], rr[e]);
                ww[e] = adamw_element<float, true>(k, decay, ww[e], gg[e], mm[e], v, rr[e]);
            }
            if (left < 8) {  // behind the tensor: zeros
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (e >= left) mm[e] = rr[e] = 0.0f;
            }
            store8(wo + i, whole, left, ww);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                top_m = max(top_m, abs_bits(mm[e]));
                top_r = max(top_r, abs_bits(rr[e]));
            }
            top_m = half_max(top_m);
            top_r = half_max(top_r);
            const bool odd = max(top_m, top_r) >= kInfBits;  // of the whole block: a value is not finite
            if (odd) {
                top_m = top_r = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (abs_bits(mm[e]) < kInfBits) top_m = max(top_m, abs_bits(mm[e]));
                    if (abs_bits(rr[e]) < kInfBits) top_r = max(top_r, abs_bits(rr[e]));
                }
                top_m = half_max(top_m);
                top_r = half_max(top_r);
            }
            float inv_m, inv_r, step_m, step_r;
            block_scale(top_m, kTopM, inv_m, step_m);
            block_scale(top_r, kTopR, inv_r, step_r);
            float ym[8];
            uint32_t om[2], orr[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                ym[e] = r_mul(mm[e], inv_m);
                orr[e / 4] |= encode_r(r_mul(rr[e], inv_r)) << (8 * (e % 4));
            }
            om[0] = encode_m(ym);
            om[1] = encode_m(ym + 4);
            if (odd) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int s = 8 * (e % 4);
                    if (abs_bits(mm[e]) >= kInfBits) om[e / 4] = (om[e / 4] & ~(0xFFu << s)) | 0x7Fu << s;
                    if (abs_bits(rr[e]) >= kInfBits) orr[e / 4] |= 0xFFu << s;
                }
            }
            store_codes(qo.m, at, vec, make_uint2(om[0], om[1]));
            store_codes(qo.r, at, vec, make_uint2(orr[0], orr[1]));
            if (tid % 16 == 0) {
                qo.steps_m[b] = step_m;
                qo.steps_r[b] = step_r;
            }
        }
    }
}

// The values a packed state stands for: m and v = (root)^2 as FLOAT32.  Bound
// by writing 8 B per element.
template <int N>
__global__ void __launch_bounds__(kThreads, kCtas) adamw_moments_kernel(const __grid_constant__ Table<N> tab) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
        const Tensor &t = tensor_of(tab, chunk);
        const int64_t n = t.n, nb = (n + kQBlock - 1) / kQBlock;
        const bool vec = t.vec;
        const int per = tab.chunk_elems / kQBlock;
        const int64_t b0 = (int64_t)(chunk - t.first) * per, b1 = min(nb, b0 + per);
        const Packed q(t.m, nb);
        float *mo = static_cast<float *>(t.m_out), *vo = static_cast<float *>(t.v_out);
        for (int64_t b = b0 + 2 * warp + lane / 16; b < b1; b += 2 * (kThreads / 32)) {
            const int64_t i = b * kQBlock + (lane % 16) * 8, at = b * 32 + (lane % 16) * 2;
            const int left = (int)max((int64_t)0, min((int64_t)8, n - i));
            const bool whole = vec && left == 8;
            const uint2 cm = load_codes(q.m, at, vec), cr = load_codes(q.r, at, vec);
            const float sm = q.steps_m[b], sr = q.steps_r[b];
            float m[8], r[8];
            decode_m(cm.x, sm, m);
            decode_m(cm.y, sm, m + 4);
            decode_r(cr.x, sr, r);
            decode_r(cr.y, sr, r + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) r[e] = r_mul(r[e], r[e]);
            store8(mo + i, whole, left, m);
            store8(vo + i, whole, left, r);
        }
    }
}

bool aligned8(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// Lays the tensors' chunks out and launches; chunks of 2048 elements (two
// vectors of every thread), or of 1024 when that leaves SMs without one.
template <int N, typename Launch>
int launch_table(Table<N> &tab, int count, int ctas, Launch launch) {
    int64_t total = 0;
    for (int i = 0; i < count; i++) total += tab.t[i].n;
    const int64_t slots = (int64_t)sm_count() * ctas;
    tab.count = count;
    tab.chunk_elems = total >= 2048 * slots ? 2048 : 1024;
    int64_t chunks = 0;
    for (int i = 0; i < count; i++) {
        tab.t[i].first = (int)chunks;
        chunks += ceil_div(tab.t[i].n, tab.chunk_elems);
        if (chunks >= (1ll << 31)) return set_error(J4C_E_UNSUPPORTED, "j4c_adamw: too many elements in one call");
    }
    tab.chunks = (int)chunks;
    return launch((unsigned)std::min<int64_t>(chunks, slots));
}

// fill(i, tensor) for every non-empty tensor i; launch(table, grid) per table.
template <typename Fill, typename Launch>
int for_tables(int ntensors, const int64_t *numel, int ctas, Fill fill, Launch launch) {
    int nonempty = 0;
    for (int i = 0; i < ntensors; i++) nonempty += numel[i] > 0;
    auto run = [&](auto &tab, int cap) {
        int i = 0;
        while (true) {
            int count = 0;
            for (; i < ntensors && count < cap; i++) {
                if (numel[i] == 0) continue;
                tab.t[count] = Tensor{};
                tab.t[count].n = numel[i];
                fill(i, tab.t[count]);
                count++;
            }
            if (count == 0) return (int)J4C_OK;
            if (int rc = launch_table(tab, count, ctas, [&](unsigned grid) { return launch(tab, grid); })) return rc;
        }
    };
    if (nonempty <= kSmallTable) {
        Table<kSmallTable> tab;
        return run(tab, kSmallTable);
    }
    Table<kLargeTable> tab;
    return run(tab, kLargeTable);
}

__global__ void advance_kernel(Hyper h) { const Coef<double> k(h); }

}  // namespace
}  // namespace j4c

using namespace j4c;

extern "C" {

int64_t j4c_adamw_q8_words(int64_t n) { return n < 0 ? -1 : ceil_div(n, kQBlock) * (kQBlock / 2 + 2); }

int j4c_adamw_step(int dtype, int state_bits, int ntensors, const int64_t *numel, const void *const *w,
                   const void *const *g, const void *const *state, void *const *w_out, void *const *state_out,
                   const double *weight_decay, const double *steps, double *steps_out, const float *lr_dev, double lr,
                   double scale, double beta1, double beta2, double eps, j4c_stream stream) {
    J4C_REQUIRE(dtype == J4C_FLOAT32 || dtype == J4C_FLOAT64, "j4c_adamw_step: FLOAT32 or FLOAT64 tensors, got %s",
                dtype_name(dtype));
    J4C_REQUIRE(state_bits == 8 || state_bits == 32, "j4c_adamw_step: moments in 8 or 32 bits, got %d", state_bits);
    J4C_REQUIRE(state_bits == 32 || dtype == J4C_FLOAT32, "j4c_adamw_step: 8-bit moments are for FLOAT32 tensors");
    J4C_REQUIRE(ntensors >= 0 && (ntensors == 0 || (numel && w && g && state && w_out && state_out && weight_decay)),
                "j4c_adamw_step: NULL table");
    J4C_REQUIRE(steps && steps != steps_out, "j4c_adamw_step: steps is NULL or steps_out");
    J4C_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "j4c_adamw_step: betas lie in [0, 1)");
    J4C_REQUIRE(eps >= 0.0, "j4c_adamw_step: negative eps");
    J4C_REQUIRE(state_bits == 32 || eps == 0.0 || (eps >= 0x1p-126 && eps <= 0x1p125),
                "j4c_adamw_step: with 8-bit moments eps is 0 or from 2^-126 to 2^125, got %g", eps);
    const int per = state_bits == 8 ? 1 : 2;
    for (int i = 0; i < ntensors; i++) {
        J4C_REQUIRE(numel[i] >= 0, "j4c_adamw_step: tensor %d has a negative size", i);
        if (numel[i] == 0) continue;
        bool there = w[i] && g[i] && w_out[i];
        for (int j = 0; j < per; j++) there = there && state[per * i + j] && state_out[per * i + j];
        J4C_REQUIRE(there, "j4c_adamw_step: tensor %d has a NULL pointer", i);
    }
    cudaStream_t s = as_stream(stream);
    Hyper h{steps, steps_out, lr_dev, lr, scale, beta1, beta2, eps};
    auto fill = [&](int i, Tensor &t) {
        t.w = w[i], t.g = g[i], t.w_out = w_out[i], t.wd = weight_decay[i];
        t.m = state[per * i], t.m_out = state_out[per * i];
        t.vec = aligned16(t.w) && aligned16(t.g) && aligned16(t.w_out);
        if (per == 1) t.vec = t.vec && aligned8(t.m) && aligned8(t.m_out);
        if (per == 2) {
            t.v = state[2 * i + 1], t.v_out = state_out[2 * i + 1];
            t.vec = t.vec && aligned16(t.m) && aligned16(t.v) && aligned16(t.m_out) && aligned16(t.v_out);
        }
    };
    bool any = false;
    auto launch = [&](auto &tab, unsigned grid) {
        constexpr int N = sizeof(tab.t) / sizeof(tab.t[0]);
        if (state_bits == 8) adamw_q8_kernel<N><<<grid, kThreads, 0, s>>>(tab, h);
        else if (dtype == J4C_FLOAT32) adamw_kernel<float, N><<<grid, kThreads, 0, s>>>(tab, h);
        else adamw_kernel<double, N><<<grid, kThreads, 0, s>>>(tab, h);
        J4C_LAUNCH_CHECK("adamw_kernel");
        any = true;
        h.steps_out = nullptr;  // one launch advances the counter
        return (int)J4C_OK;
    };
    if (int rc = for_tables(ntensors, numel, state_bits == 8 ? kQCtas : kCtas, fill, launch)) return rc;
    if (!any && steps_out) {  // nothing but empty tensors: the counter still advances
        advance_kernel<<<1, 1, 0, s>>>(h);
        J4C_LAUNCH_CHECK("advance_kernel");
    }
    return J4C_OK;
}

int j4c_adamw_moments(int ntensors, const int64_t *numel, const void *const *state, float *const *m_out,
                      float *const *v_out, j4c_stream stream) {
    J4C_REQUIRE(ntensors >= 0 && (ntensors == 0 || (numel && state && m_out && v_out)),
                "j4c_adamw_moments: NULL table");
    for (int i = 0; i < ntensors; i++) {
        J4C_REQUIRE(numel[i] >= 0, "j4c_adamw_moments: tensor %d has a negative size", i);
        J4C_REQUIRE(numel[i] == 0 || (state[i] && m_out[i] && v_out[i]), "j4c_adamw_moments: tensor %d has a NULL pointer",
                    i);
    }
    cudaStream_t s = as_stream(stream);
    auto fill = [&](int i, Tensor &t) {
        t.m = state[i], t.m_out = m_out[i], t.v_out = v_out[i];
        t.vec = aligned16(t.m_out) && aligned16(t.v_out) && aligned8(t.m);
    };
    auto launch = [&](auto &tab, unsigned grid) {
        constexpr int N = sizeof(tab.t) / sizeof(tab.t[0]);
        adamw_moments_kernel<N><<<grid, kThreads, 0, s>>>(tab);
        J4C_LAUNCH_CHECK("adamw_moments_kernel");
        return (int)J4C_OK;
    };
    return for_tables(ntensors, numel, kCtas, fill, launch);
}

}  // extern "C"
