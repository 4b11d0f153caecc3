// paged_append.cu - one layer's rows between the QKV projection and the attention: q/k RMSNorm, rotary
// positions, rotated queries out, K and V quantised into the step's 8-bit pages.  And the way back:
// rows of the cache as numbers.
//
// y = x / sqrt(mean(x^2) + eps) * w;  a pair (a, b) at angle t becomes (a cos t - b sin t, a sin t + b cos t).
// Angles: f_i comes as turns per position in two f32 parts (hi + lo = f_i / 2 pi to ~48 bits).  The
// product with the position keeps its rounding error (one fma), whole turns leave exactly, and what is left
// is under one turn, so the angle is good to f32 rounding at any position.
// A page and head has one scale s = max(s_old, amax / 127).  One block owns all of a page's new rows for one
// kv head of K or V, so the maximum, the scale and the rounding of the codes already there need no
// atomics and no second launch.  The block keeps its rows in registers between the maximum and the
// rounding: each row is read once.
//
// A block takes one page's new rows (or one row of a decode step) and some of the heads: first the cosines
// and sines of its tokens, once, into shared memory; then K and V of each kv head; then the query rows.
// Eight consecutive elements of a row per thread (HD/8 threads per row, all in one warp).  Two forms,
// by the most rows that the step can bring to one page:
//   up to 4   a row's threads own a (kv head, K or V) by themselves: the maximum is a few shuffles
//   more      the whole block takes a kv head's K and V rows at once: one barrier per head; queries keep their
//             token's rotation in registers over the heads
// The rotation and the norm weight of an element are one factor: y = n (x (w c) + x' (w' s)), n the row's norm.
// Bound: HBM (f16 projections in, f16 queries and codes out); latency for a few tokens.
#include <cmath>
#include <cstring>
#include <new>

#include "common.cuh"
#include "paged.hpp"

namespace svkv {

namespace {

constexpr int kThreads = 256;       // of the read kernel

struct AppendArgs {
    sv_paged kv;
    const uint8_t *q, *k, *v;
    size_t q_nb, k_nb, v_nb;
    const float *qn, *kn;
    float eps;
    const float4* pairs;      // null: no rotation
    int mode, n_dims;         // n_dims = 0 without rotation
    float mag;
    const int32_t* pos;       // [T], or [4][T] for IMROPE
    int T, NH, G;
    const int4* pages;
    const int* head;
    int kv_per;               // kv heads per block
    void* q_out;
    bool q_out_f32;
};

template <bool F32>
struct Raw8 { uint4 w[F32 ? 2 : 1]; };

template <bool F32>
__device__ __forceinline__ Raw8<F32> fetch8(const uint8_t* row, int e) {
    Raw8<F32> r;
    const uint4* p = reinterpret_cast<const uint4*>(row + (size_t)e * (F32 ? 4 : 2));
    r.w[0] = p[0];
    if constexpr (F32) r.w[1] = p[1];
    return r;
}

template <bool F32>
__device__ __forceinline__ void to_f32(const Raw8<F32>& r, float* x) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

template <bool F32>
__device__ __forceinline__ float load1(const uint8_t* row, int e) {
    if constexpr (F32) return *reinterpret_cast<const float*>(row + (size_t)e * 4);
    else return __half2float(*reinterpret_cast<const __half*>(row + (size_t)e * 2));
}

__device__ __forceinline__ void store8(void* out, size_t at, bool f32, const float* x) {
    if (f32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<__half*>(out) + at) =
            make_uint4(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7]));
    }
}

// (cos, sin) of a pair's angle at a position, times mag.  The angle is brought to one eighth of a turn on
// either side of a quarter; there the Taylor series to x^9 and x^8 are exact to f32 (next terms below 2^-25).
__device__ __forceinline__ float2 turn(const float4 f, int pos, float mag) {
    const float p = (float)pos;
    const float rest = (float)(int)((long long)pos - (long long)p);   // 0 below 2^24
    const float t = p * f.x, e = fmaf(p, f.x, -t);
    float r = t - rintf(t);
    r += fmaf(p, f.y, e) + rest * f.x;
    const float q = rintf(4.0f * r);
    const float a = fmaf(-0.25f, q, r) * 6.28318530717958647693f, a2 = a * a;
    const float sn = mag * a * fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    const float cn = mag * fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, 1.0f / 40320, -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int i = (int)q;
    const float2 z = i & 1 ? make_float2(-sn, cn) : make_float2(cn, sn);
    return i & 2 ? make_float2(-z.x, -z.y) : z;
}

// Factors of a thread's 8 elements [e, e + 8) and of their partners: y_i = x_i c_i + x'_i s_i.
struct Rotation {
    float c[8], s[8];
};

// cs: the token's cosines [n_dims/2], then its sines.  w: norm weights or null.
__device__ __forceinline__ void rotation_of(const AppendArgs& a, const float* cs, int e, const float* w, Rotation* r) {
    const int half = a.n_dims >> 1;
    const bool norm_mode = a.mode == SV_ROPE_NORM;
    if (e >= a.n_dims) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            r->c[i] = w ? __ldg(w + e + i) : 1.0f;
            r->s[i] = 0.0f;
        }
    } else if ((a.n_dims & 15) == 0) {             // whole runs of 8: 16-byte reads
        if (norm_mode) {
            const float4 c = *reinterpret_cast<const float4*>(cs + (e >> 1)), s = *reinterpret_cast<const float4*>(cs + half + (e >> 1));
            const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                r->c[i] = cc[i >> 1];
                r->s[i] = i & 1 ? ss[i >> 1] : -ss[i >> 1];
            }
        } else {
            const float4* c = reinterpret_cast<const float4*>(cs + (e < half ? e : e - half));
            const float4* s = reinterpret_cast<const float4*>(cs + half + (e < half ? e : e - half));
            const float sg = e < half ? -1.0f : 1.0f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float4 x = c[i], y = s[i];
                r->c[4 * i] = x.x; r->c[4 * i + 1] = x.y; r->c[4 * i + 2] = x.z; r->c[4 * i + 3] = x.w;
                r->s[4 * i] = sg * y.x; r->s[4 * i + 1] = sg * y.y; r->s[4 * i + 2] = sg * y.z; r->s[4 * i + 3] = sg * y.w;
            }
        }
        if (w) {
            const int pe = norm_mode ? e : (e < half ? e + half : e - half);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                r->c[i] *= __ldg(w + e + i);
                r->s[i] *= __ldg(w + pe + (norm_mode ? i ^ 1 : i));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = e + i;
            float c = 1.0f, s = 0.0f;
            int pd = d;
            if (d < a.n_dims) {
                const bool second = norm_mode ? (i & 1) : d >= half;
                const int pair = norm_mode ? d >> 1 : (second ? d - half : d);
                pd = norm_mode ? d ^ 1 : (second ? d - half : d + half);
                c = cs[pair];
                s = second ? cs[half + pair] : -cs[half + pair];
            }
            r->c[i] = w ? c * __ldg(w + d) : c;
            r->s[i] = w ? s * __ldg(w + pd) : s;
        }
    }
}

// The partners of a thread's elements, from the row again (L1) where they lie with another thread.
enum : int { PART_NONE = 0, PART_OWN = 1, PART_VEC = 2, PART_ONE = 3 };
__device__ __forceinline__ int partners_by(const AppendArgs& a, int e) {
    if (e >= a.n_dims) return PART_NONE;
    if (a.mode == SV_ROPE_NORM) return PART_OWN;
    return (a.n_dims & 15) == 0 ? PART_VEC : PART_ONE;
}
__device__ __forceinline__ int partner_at(const AppendArgs& a, int e) {
    const int half = a.n_dims >> 1;
    return e < half ? e + half : e - half;
}
template <bool F32>
__device__ __forceinline__ void partners(const AppendArgs& a, int by, const Raw8<F32>& pr, const uint8_t* row, int e, const float* x,
                                         float* y) {
    if (by == PART_VEC) {
        to_f32<F32>(pr, y);
    } else if (by == PART_OWN) {
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = x[i ^ 1];
    } else {
        const int half = a.n_dims >> 1;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = e + i;
            y[i] = by == PART_ONE && d < a.n_dims ? load1<F32>(row, d < half ? d + half : d - half) : 0.0f;
        }
    }
}

// 1 / rms over the row's lanes
template <int HD>
__device__ __forceinline__ float row_norm(const float* x, float eps) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return 1.0f / sqrtf(ss / (float)HD + eps);
}

template <int HD>
__device__ __forceinline__ void apply(const AppendArgs& a, bool normed, const Rotation& r, const float* y, float* x) {
    const float n = normed ? row_norm<HD>(x, a.eps) : 1.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = n * fmaf(x[i], r.c[i], y[i] * r.s[i]);
}

// ---- quantising
// Running maximum of |x|, and NaN in *bad once a value is not finite (0 x is NaN then).
__device__ __forceinline__ void watch(const float* x, float* amax, float* bad) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        *amax = fmaxf(*amax, fabsf(x[i]));
        *bad = fmaf(x[i], 0.0f, *bad);
    }
}
__device__ __forceinline__ float finite_max(const float* x) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (fabsf(x[i]) <= 3.402823466e38f) m = fmaxf(m, fabsf(x[i]));
    return m;
}
__device__ __forceinline__ void page_scale(float amax, float s_old, float* s, float* inv) {
    if (amax < 7.8886090522101181e-31f) amax = 0.0f;   // 2^-100: 1 / s stays finite
    *s = fmaxf(s_old, __fdiv_rn(amax, 127.0f));
    *inv = *s > 0.0f ? __fdiv_rn(1.0f, *s) : 0.0f;
}
// Codes of 8 values, round-half-even of x inv: the sum with 1.5 2^23 leaves the integer in its low byte.
// |x inv| is at most 127 (1 + 2^-23), which rounds to 127.
__device__ __forceinline__ uint2 codes8(const float* x, float inv) {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[4 * j + i], inv), 12582912.0f));
        w[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    return make_uint2(w[0], w[1]);
}
// infinities to +-127, NaN to 0
__device__ __forceinline__ void tame(float* x, float s) {
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (!(fabsf(x[i]) <= 3.402823466e38f)) x[i] = x[i] > 0.0f ? 127.0f * s : (x[i] < 0.0f ? -127.0f * s : 0.0f);
}
// eight codes that the page holds, rounded to its new scale (f = s_old / s)
__device__ __forceinline__ uint2 recode8(uint2 c, float f) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)(int8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    return codes8(x, f);
}
// rows [first, end) of a page, `step` apart, this thread's 8 codes of each
template <int HD>
__device__ __forceinline__ void recode_rows(uint8_t* page, int first, int end, int step, int e, float f) {
    for (int r = first; r < end; r += 4 * step) {
        uint2 c[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (r + i * step < end) c[i] = *reinterpret_cast<const uint2*>(page + (size_t)(r + i * step) * HD + e);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (r + i * step < end) *reinterpret_cast<uint2*>(page + (size_t)(r + i * step) * HD + e) = recode8(c[i], f);
    }
}

// cosines and sines of `rows` tokens from t0: [rows][n_dims/2 cosines, n_dims/2 sines]
__device__ __forceinline__ void fill_turns(const AppendArgs& a, int t0, int rows, float* cs) {
    const int half = a.n_dims >> 1;
    for (int i = threadIdx.x; i < rows * half; i += blockDim.x) {
        const int r = i / half, p = i - r * half;
        const float4 f = __ldg(a.pairs + p);
        const float2 z = turn(f, __ldg(a.pos + (size_t)__float_as_int(f.z) * a.T + t0 + r), a.mag);
        cs[r * a.n_dims + p] = z.x;
        cs[r * a.n_dims + half + p] = z.y;
    }
}

// ---------------- up to NV rows per page
template <int HD, bool F32, int NV>
__global__ void __launch_bounds__(256, NV == 1 ? 3 : 2) paged_append_few(const __grid_constant__ AppendArgs a) {
    constexpr int C = HD / 8, PER = 256 / C;       // threads per row, rows at once
    constexpr int ES = F32 ? 4 : 2;
    extern __shared__ float cs[];
    pdl_wait();
    if (threadIdx.x == 0) pdl_trigger();
    if ((int)blockIdx.x >= a.head[PH_PAGES]) return;
    const int4 it = a.pages[blockIdx.x];           // first row, page, offset in it, rows
    const int n = min(it.w, NV);
    const int e = (threadIdx.x % C) * 8, u = threadIdx.x / C;
    const int kv0 = blockIdx.y * a.kv_per, kvn = min(a.kv_per, a.kv.n_kv_head - kv0);
    if (a.pairs) {
        fill_turns(a, it.x, n, cs);
        __syncthreads();
    }
    const int by = partners_by(a, e);
    // ---- units: kv head 2 i / 2, K or V
    for (int i0 = 0; it.y >= 0 && i0 < 2 * kvn; i0 += PER) {
        const bool live = i0 + u < 2 * kvn;
        const int i = live ? i0 + u : 0;
        const int h = kv0 + (i >> 1);
        const bool is_k = (i & 1) == 0;
        const uint8_t* src = (is_k ? a.k + (size_t)it.x * a.k_nb : a.v + (size_t)it.x * a.v_nb) + (size_t)h * HD * ES;
        const size_t nb = is_k ? a.k_nb : a.v_nb;
        const size_t unit = (size_t)it.y * a.kv.n_kv_head + h;
        float* sp = (is_k ? a.kv.k_scale : a.kv.v_scale) + unit;
        const float s_old = it.z > 0 ? *sp : 0.0f;
        Raw8<F32> raw[NV], praw[NV];
#pragma unroll
        for (int r = 0; r < NV; r++)
            if (r < n) {
                raw[r] = fetch8<F32>(src + r * nb, e);
                if (is_k && by == PART_VEC) praw[r] = fetch8<F32>(src + r * nb, partner_at(a, e));
            }
        float x[NV][8], amax = 0.0f, bad = 0.0f;
#pragma unroll
        for (int r = 0; r < NV; r++) {
            if (r >= n) break;
            to_f32<F32>(raw[r], x[r]);
            // K and V rows share warps: the norm's shuffles run for both
            const float nrm = a.kn ? row_norm<HD>(x[r], a.eps) : 1.0f;
            if (is_k && (a.pairs || a.kn)) {
                float y[8];
                Rotation rot;
                partners<F32>(a, by, praw[r], src + r * nb, e, x[r], y);
                rotation_of(a, cs + r * a.n_dims, e, a.kn, &rot);
#pragma unroll
                for (int j = 0; j < 8; j++) x[r][j] = nrm * fmaf(x[r][j], rot.c[j], y[j] * rot.s[j]);
            }
            watch(x[r], &amax, &bad);
        }
        if (__any_sync(0xffffffffu, bad != 0.0f)) {     // NaN
            amax = 0.0f;
#pragma unroll
            for (int r = 0; r < NV; r++)
                if (r < n) amax = fmaxf(amax, finite_max(x[r]));
        }
#pragma unroll
        for (int o = C / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        float s, inv;
        page_scale(amax, s_old, &s, &inv);
        __syncwarp();                              // the row's threads have read the old scale
        if (live) {
            if (e == 0) *sp = s;
            uint8_t* page = static_cast<uint8_t*>(is_k ? a.kv.k : a.kv.v) + unit * a.kv.page_size * HD;
#pragma unroll
            for (int r = 0; r < NV; r++)
                if (r < n) {
                    if (bad != 0.0f) tame(x[r], s);
                    *reinterpret_cast<uint2*>(page + (size_t)(it.z + r) * HD + e) = codes8(x[r], inv);
                }
            if (s > s_old && it.z > 0) recode_rows<HD>(page, 0, it.z, 1, e, __fmul_rn(s_old, inv));
        }
    }
    // ---- query rows
    const int q0 = kv0 * a.G, qn = kvn * a.G;
    for (int i0 = 0; i0 < n * qn; i0 += PER) {
        const bool live = i0 + u < n * qn;
        const int i = live ? i0 + u : 0, r = i / qn, h = q0 + i - r * qn;
        const uint8_t* row = a.q + (size_t)(it.x + r) * a.q_nb + (size_t)h * HD * ES;
        float x[8];
        const Raw8<F32> raw = fetch8<F32>(row, e);
        Raw8<F32> praw;
        if (by == PART_VEC) praw = fetch8<F32>(row, partner_at(a, e));
        to_f32<F32>(raw, x);
        if (a.pairs || a.qn) {
            float y[8];
            Rotation rot;
            partners<F32>(a, by, praw, row, e, x, y);
            rotation_of(a, cs + r * a.n_dims, e, a.qn, &rot);
            apply<HD>(a, a.qn != nullptr, rot, y, x);
        }
        __syncwarp();                              // q_out may be q: the row's partners have been read
        if (live) store8(a.q_out, ((size_t)(it.x + r) * a.NH + h) * HD + e, a.q_out_f32, x);
    }
}

// ---------------- up to NV x (THREADS / C) rows per page
template <int HD, bool F32, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 1 : NV <= 2 ? 3 : 2) paged_append_many(const __grid_constant__ AppendArgs a) {
    constexpr int C = HD / 8, RP = THREADS / C;    // threads per row, rows per pass
    constexpr int ES = F32 ? 4 : 2, W = THREADS / 32;
    extern __shared__ float cs[];
    __shared__ float s_max[2][2][W];               // [parity of the head][K, V]
    __shared__ int s_bad[2];
    pdl_wait();
    if (threadIdx.x == 0) pdl_trigger();
    if ((int)blockIdx.x >= a.head[PH_PAGES]) return;
    const int4 it = a.pages[blockIdx.x];
    const int n = min(it.w, NV * RP);
    const int e = (threadIdx.x % C) * 8, r0 = threadIdx.x / C;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv0 = blockIdx.y * a.kv_per, kvn = min(a.kv_per, a.kv.n_kv_head - kv0);
    const int by = partners_by(a, e);
    if (threadIdx.x < 2) s_bad[threadIdx.x] = 0;
    if (a.pairs) fill_turns(a, it.x, n, cs);
    __syncthreads();
    for (int hi = 0; it.y >= 0 && hi < kvn; hi++) {
        const int h = kv0 + hi, par = hi & 1;
        const uint8_t* ks = a.k + (size_t)it.x * a.k_nb + (size_t)h * HD * ES;
        const uint8_t* vs = a.v + (size_t)it.x * a.v_nb + (size_t)h * HD * ES;
        const size_t unit = (size_t)it.y * a.kv.n_kv_head + h;
        Raw8<F32> kr[NV], vr[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int r = r0 + i * RP;
            if (r < n) {
                kr[i] = fetch8<F32>(ks + (size_t)r * a.k_nb, e);
                vr[i] = fetch8<F32>(vs + (size_t)r * a.v_nb, e);
            }
        }
        const float k_old = it.z > 0 ? a.kv.k_scale[unit] : 0.0f, v_old = it.z > 0 ? a.kv.v_scale[unit] : 0.0f;
        float x[NV][8], kmax = 0.0f, vmax = 0.0f, bad = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (i * RP >= n) break;
            const int r = r0 + i * RP;
            const bool live = r < n;
            if (live) {
                to_f32<F32>(kr[i], x[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = 0.0f;
            }
            if (a.pairs || a.kn) {                 // whole warps go through (the norm's shuffles)
                const int rr = live ? r : 0;
                const uint8_t* row = ks + (size_t)rr * a.k_nb;
                Raw8<F32> pr;
                if (by == PART_VEC) pr = fetch8<F32>(row, partner_at(a, e));
                float y[8];
                Rotation rot;
                partners<F32>(a, by, pr, row, e, x[i], y);
                rotation_of(a, cs + rr * a.n_dims, e, a.kn, &rot);
                apply<HD>(a, a.kn != nullptr, rot, y, x[i]);
            }
            if (live) {
                watch(x[i], &kmax, &bad);
                float v[8];
                to_f32<F32>(vr[i], v);
                watch(v, &vmax, &bad);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
            vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
        }
        if (lane == 0) {
            s_max[par][0][warp] = kmax;
            s_max[par][1][warp] = vmax;
        }
        if (__any_sync(0xffffffffu, bad != 0.0f) && lane == 0) s_bad[par] = 1;
        __syncthreads();                           // maxima meet; every thread has read the old scales
        if (s_bad[par]) {                          // once more over the finite values
            kmax = vmax = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (r0 + i * RP < n) {
                    float v[8];
                    to_f32<F32>(vr[i], v);
                    kmax = fmaxf(kmax, finite_max(x[i]));
                    vmax = fmaxf(vmax, finite_max(v));
                }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
                vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
            }
            __syncthreads();
            if (lane == 0) {
                s_max[par][0][warp] = kmax;
                s_max[par][1][warp] = vmax;
            }
            __syncthreads();
        }
        const bool any_bad = s_bad[par] != 0;
        kmax = vmax = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            kmax = fmaxf(kmax, s_max[par][0][w]);
            vmax = fmaxf(vmax, s_max[par][1][w]);
        }
        if (threadIdx.x == 0) s_bad[par ^ 1] = 0;  // the next head's; its last reader is a barrier behind
        float sk, ik, sv, iv;
        page_scale(kmax, k_old, &sk, &ik);
        page_scale(vmax, v_old, &sv, &iv);
        if (threadIdx.x == 0) {
            a.kv.k_scale[unit] = sk;
            a.kv.v_scale[unit] = sv;
        }
        uint8_t* kp = static_cast<uint8_t*>(a.kv.k) + unit * a.kv.page_size * HD;
        uint8_t* vp = static_cast<uint8_t*>(a.kv.v) + unit * a.kv.page_size * HD;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int r = r0 + i * RP;
            if (r < n) {
                float v[8];
                to_f32<F32>(vr[i], v);
                if (any_bad) {
                    tame(x[i], sk);
                    tame(v, sv);
                }
                *reinterpret_cast<uint2*>(kp + (size_t)(it.z + r) * HD + e) = codes8(x[i], ik);
                *reinterpret_cast<uint2*>(vp + (size_t)(it.z + r) * HD + e) = codes8(v, iv);
            }
        }
        if (it.z > 0) {
            if (sk > k_old) recode_rows<HD>(kp, r0, it.z, RP, e, __fmul_rn(k_old, ik));
            if (sv > v_old) recode_rows<HD>(vp, r0, it.z, RP, e, __fmul_rn(v_old, iv));
        }
    }
    // ---- query rows: a thread keeps its token and chunk over the heads
    constexpr int U = F32 ? 2 : 4;                 // heads whose loads are in flight
    const int q0 = kv0 * a.G, qe = q0 + kvn * a.G;
    const bool turned = a.pairs || a.qn;
    for (int rb = 0; rb < n; rb += RP) {
        const bool live = rb + r0 < n;
        const int t = it.x + (live ? rb + r0 : 0);
        Rotation rot;
        if (turned) rotation_of(a, cs + (t - it.x) * a.n_dims, e, a.qn, &rot);
        for (int hb = q0; hb < qe; hb += U) {
            Raw8<F32> raw[U], pr[U];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint8_t* row = a.q + (size_t)t * a.q_nb + (size_t)min(hb + j, qe - 1) * HD * ES;
                raw[j] = fetch8<F32>(row, e);
                if (by == PART_VEC) pr[j] = fetch8<F32>(row, partner_at(a, e));
            }
            __syncwarp();                          // q_out may be q: these heads' partners have been read
#pragma unroll
            for (int j = 0; j < U; j++) {
                float x[8];
                to_f32<F32>(raw[j], x);
                if (turned) {
                    float y[8];
                    partners<F32>(a, by, pr[j], a.q + (size_t)t * a.q_nb + (size_t)min(hb + j, qe - 1) * HD * ES, e, x, y);
                    apply<HD>(a, a.qn != nullptr, rot, y, x);
                }
                __syncwarp();                      // as above, for partners that were read one by one
                if (live && hb + j < qe) store8(a.q_out, ((size_t)t * a.NH + hb + j) * HD + e, a.q_out_f32, x);
            }
        }
    }
}

template <bool F32>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const __grid_constant__ sv_paged kv, const int32_t* slots,
                                                              int n, void* k_out, void* v_out) {
    pdl_wait();
    const int C = kv.head_dim / 8, per = kv.n_kv_head * C;
    const long long all = (long long)n * per;
    const int lg = 31 - __clz(kv.page_size);
    for (long long id = (long long)blockIdx.x * kThreads + threadIdx.x; id < all; id += (long long)gridDim.x * kThreads) {
        const long long i = id / per;
        const int at = (int)(id % per), h = at / C, e = (at % C) * 8;
        const int slot = __ldg(slots + i);
        const bool ok = slot >= 0 && (slot >> lg) < kv.n_pages;
        if (!ok && slot != -1 && at == 0 && kv.err) atomicOr(kv.err, ERRBIT_ROW_RANGE);
        float x[2][8] = {};
        if (ok) {
            const size_t unit = (size_t)(slot >> lg) * kv.n_kv_head + h;
            const size_t off = (unit * kv.page_size + (slot & (kv.page_size - 1))) * kv.head_dim + e;
            const uint2 w[2] = {*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(kv.k) + off),
                                *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(kv.v) + off)};
            const float s[2] = {kv.k_scale[unit], kv.v_scale[unit]};
#pragma unroll
            for (int o = 0; o < 2; o++)
#pragma unroll
                for (int b = 0; b < 8; b++)
                    x[o][b] = (float)(int8_t)((b < 4 ? w[o].x : w[o].y) >> (8 * (b & 3))) * s[o];
        }
        store8(k_out, (size_t)id * 8, F32, x[0]);
        store8(v_out, (size_t)id * 8, F32, x[1]);
    }
}

}  // namespace

cudaError_t launch_paged_append(const sv_paged& kv, const sv_paged_step& s, const StepLayout& l,
                                const sv_paged_rows& r, cudaStream_t st) {
    AppendArgs a{};
    const uint8_t* work = static_cast<const uint8_t*>(s.work);
    a.kv = kv;
    a.q = static_cast<const uint8_t*>(r.q);
    a.k = static_cast<const uint8_t*>(r.k);
    a.v = static_cast<const uint8_t*>(r.v);
    a.q_nb = r.q_nb;
    a.k_nb = r.k_nb;
    a.v_nb = r.v_nb;
    a.qn = r.q_norm;
    a.kn = r.k_norm;
    a.eps = r.eps;
    if (r.rope) {
        a.pairs = r.rope->pairs;
        a.mode = r.rope->mode;
        a.n_dims = r.rope->n_dims;
        a.mag = r.rope->mag;
    }
    a.pos = r.pos ? r.pos : s.tok_pos;
    a.T = s.n_tokens;
    a.NH = s.n_head;
    a.G = s.n_head / s.n_kv_head;
    a.pages = reinterpret_cast<const int4*>(work + l.page);
    a.head = reinterpret_cast<const int*>(work + l.head);
    a.q_out = r.q_out;
    a.q_out_f32 = r.q_out_type == SV_TYPE_F32;
    // Heads are split over blocks until there are about four blocks per SM: below that the rows of a page
    // leave SMs idle, above it the tokens' sines are computed more often than needed.
    const int want = ceil_div(4 * device_sm_count(), l.page_cap);
    const int groups = want < 1 ? 1 : want > kv.n_kv_head ? kv.n_kv_head : want;
    a.kv_per = ceil_div(kv.n_kv_head, groups);
    const dim3 grid((unsigned)l.page_cap, (unsigned)ceil_div(kv.n_kv_head, a.kv_per));
    const int rows = kv.page_size < s.max_new ? kv.page_size : s.max_new;    // new rows of one page, at most
    const int smem = rows * a.n_dims * 4;
    const bool f32 = r.type == SV_TYPE_F32;
#define SV_TRY(...)                                                                          \
    {                                                                                        \
        auto* k32 = __VA_ARGS__;                                                             \
        if (smem > 40 * 1024) {                                                              \
            const cudaError_t e = cudaFuncSetAttribute(k32, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024); \
            if (e != cudaSuccess) return e;                                                  \
        }                                                                                    \
        return launch_pdl(k32, grid, dim3(threads), (size_t)smem, st, a);                    \
    }
#define SV_FEW(HD_, NV_)                                                                     \
    if (kv.head_dim == HD_ && rows <= NV_) {                                                 \
        const int threads = 256;                                                             \
        if (f32) SV_TRY(paged_append_few<HD_, true, NV_>) else SV_TRY(paged_append_few<HD_, false, NV_>) \
    }
#define SV_MANY(HD_, TH_, NV_)                                                               \
    if (kv.head_dim == HD_ && rows <= NV_ * TH_ * 8 / HD_) {                                 \
        const int threads = TH_;                                                             \
        if (f32) SV_TRY(paged_append_many<HD_, true, TH_, NV_>) else SV_TRY(paged_append_many<HD_, false, TH_, NV_>) \
    }
    SV_FEW(64, 1) SV_FEW(64, 4) SV_MANY(64, 256, 1) SV_MANY(64, 256, 4)
    SV_FEW(128, 1) SV_FEW(128, 4) SV_MANY(128, 256, 2) SV_MANY(128, 256, 4) SV_MANY(128, 512, 4)
    SV_FEW(256, 1) SV_FEW(256, 4) SV_MANY(256, 256, 2) SV_MANY(256, 256, 4) SV_MANY(256, 512, 8)
#undef SV_FEW
#undef SV_MANY
#undef SV_TRY
    return cudaErrorInvalidValue;
}

cudaError_t launch_paged_read(const sv_paged& kv, const int32_t* slots, int n, void* k_out, void* v_out, int out_type,
                              cudaStream_t st) {
    const int64_t all = (int64_t)n * kv.n_kv_head * (kv.head_dim / 8);
    const int64_t most = (int64_t)device_sm_count() * 8;
    const int64_t blocks = (all + kThreads - 1) / kThreads;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    return out_type == SV_TYPE_F32 ? launch_pdl(paged_read_kernel<true>, grid, dim3(kThreads), 0, st, kv, slots, n, k_out, v_out)
                                   : launch_pdl(paged_read_kernel<false>, grid, dim3(kThreads), 0, st, kv, slots, n, k_out, v_out);
}

}  // namespace svkv

extern "C" {

int sv_rope_table_create(int device, const sv_rope_params* p, sv_rope_table** out) {
    using namespace svkv;
    if (!out) return SV_ERR_INVALID;
    *out = nullptr;
    if (!p || !(p->freq_base > 0.0) || !std::isfinite(p->freq_base) || !(p->freq_scale > 0.0) || !(p->ext_factor >= 0.0) ||
        !std::isfinite(p->attn_factor))
        return SV_ERR_INVALID;
    if (p->mode != SV_ROPE_NORM && p->mode != SV_ROPE_NEOX && p->mode != SV_ROPE_IMROPE) return SV_ERR_UNSUPPORTED;
    if (p->n_dims < 2 || p->n_dims > 256 || (p->n_dims & 1)) return SV_ERR_UNSUPPORTED;
    if (p->ext_factor > 0.0 && (p->n_ctx_orig < 1 || !(p->beta_fast > 0.0) || !(p->beta_slow > 0.0) || p->freq_base <= 1.0))
        return SV_ERR_INVALID;
    int sum = 0;
    for (int i = 0; i < 4; i++) {
        if (p->mode == SV_ROPE_IMROPE && (p->sections[i] < 0 || p->sections[i] > 128)) return SV_ERR_INVALID;
        sum += p->mode == SV_ROPE_IMROPE ? p->sections[i] : 0;
    }
    const int half = p->n_dims / 2;
    const double two_pi = 6.283185307179586476925, base = p->freq_base, scale = p->freq_scale;
    float4 host[128];
    double low = 0.0, high = 0.0;
    if (p->ext_factor > 0.0) {
        // the pair that turns `turns` times in the original context
        auto pair_of = [&](double turns) {
            return p->n_dims * std::log(p->n_ctx_orig / (turns * two_pi)) / (2.0 * std::log(base));
        };
        low = std::fmax(0.0, std::floor(pair_of(p->beta_fast)));
        high = std::fmin(p->n_dims - 1.0, std::ceil(pair_of(p->beta_slow)));
    }
    for (int i = 0; i < half; i++) {
        double f = std::pow(base, -2.0 * i / p->n_dims);
        if (p->freq_factors) {
            if (!(p->freq_factors[i] > 0.0f)) return SV_ERR_INVALID;
            f /= p->freq_factors[i];
        }
        double keep = 0.0;
        if (p->ext_factor > 0.0) {
            const double y = (i - low) / std::fmax(0.001, high - low);
            keep = (1.0 - std::fmin(1.0, std::fmax(0.0, y))) * p->ext_factor;
        }
        f = f * scale * (1.0 - keep) + f * keep;
        const double turns = f / two_pi;
        int axis = 0;
        if (p->mode == SV_ROPE_IMROPE) {
            const int j = sum > 0 ? i % sum : i;
            axis = j % 3 == 1 && j < 3 * p->sections[1] ? 1 : j % 3 == 2 && j < 3 * p->sections[2] ? 2
                   : j % 3 == 0 && j < 3 * p->sections[0] ? 0 : 3;
        }
        host[i].x = (float)turns;
        host[i].y = (float)(turns - (double)host[i].x);
        memcpy(&host[i].z, &axis, 4);
        host[i].w = 0.0f;
    }
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return SV_ERR_CUDA;
    float4* dev = nullptr;
    int rc = SV_OK;
    if (cudaMalloc(&dev, sizeof(float4) * half) != cudaSuccess) rc = SV_ERR_NOMEM;
    else if (cudaMemcpy(dev, host, sizeof(float4) * half, cudaMemcpyHostToDevice) != cudaSuccess) rc = SV_ERR_CUDA;
    sv_rope_table* t = rc == SV_OK ? new (std::nothrow) sv_rope_table() : nullptr;
    if (rc == SV_OK && !t) rc = SV_ERR_NOMEM;
    if (rc != SV_OK) {
        if (dev) cudaFree(dev);
    } else {
        t->device = device;
        t->mode = p->mode;
        t->n_dims = p->n_dims;
        t->mag = (float)(p->attn_factor * (p->ext_factor > 0.0 ? 1.0 + 0.1 * std::log(1.0 / scale) : 1.0));
        t->pairs = dev;
        *out = t;
    }
    cudaSetDevice(prev);
    return rc;
}

int sv_rope_table_destroy(sv_rope_table* t) {
    if (!t) return SV_ERR_INVALID;
    int prev = -1;
    if (cudaGetDevice(&prev) == cudaSuccess) {
        cudaSetDevice(t->device);
        cudaFree(t->pairs);
        cudaSetDevice(prev);
    }
    delete t;
    return SV_OK;
}

}  // extern "C"
