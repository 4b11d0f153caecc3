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
// Each thread holds 8 consecutive elements of a row (HD/8 threads per row, all in one warp).
//   blocks [0, KV)  one (page, kv head, K or V) each
//   the rest        query rows: a thread does its 8 elements of `loop` heads of one token, so the sines
//                   and cosines are computed once for them
// Bound: HBM (f16 projections in, f16 queries and codes out); latency for a few tokens.
#include <cmath>
#include <cstring>
#include <new>

#include "common.cuh"
#include "paged.hpp"

namespace svkv {

namespace {

constexpr int kThreads = 256;

struct AppendArgs {
    sv_paged kv;
    const uint8_t *q, *k, *v;
    size_t q_nb, k_nb, v_nb;
    const float *qn, *kn;
    float eps;
    const float4* pairs;      // null: no rotation
    int mode, n_dims;
    float mag;
    const int32_t* pos;       // [T], or [4][T] for IMROPE
    int T, NH;
    const int4* pages;
    const int* head;
    int n_kv_blocks;          // blocks of the first kind
    int loop, n_groups;       // query heads per thread, groups of heads
    void* q_out;
    bool q_out_f32;
    const int32_t* q_start;   // [n_req + 1]; the last is the step's row count
    int n_req;
    int* err;
};

template <bool F32>
__device__ __forceinline__ void load8(const uint8_t* row, int e, float* x) {
    if constexpr (F32) {
        const float4 a = *reinterpret_cast<const float4*>(row + (size_t)e * 4);
        const float4 b = *reinterpret_cast<const float4*>(row + (size_t)e * 4 + 16);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(row + (size_t)e * 2);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
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

// cos and sin (times mag) of a pair's angle at a position
__device__ __forceinline__ float2 turn(const float4 f, int pos, float mag) {
    const float p = (float)pos;
    const float rest = (float)(int)((long long)pos - (long long)p);   // 0 below 2^24
    const float t = p * f.x, e = fmaf(p, f.x, -t);
    float r = t - rintf(t);
    r += fmaf(p, f.y, e) + rest * f.x;
    float sn, cn;
    sincospif(2.0f * r, &sn, &cn);
    return make_float2(cn * mag, sn * mag);
}

// The rotation of a thread's 8 elements [e, e + 8): y_i = x_i c_i + partner_i s_i, with the pair's sine signed
// by the element's place in it.  Elements past n_dims keep c = 1, s = 0.
struct Rotation {
    float c[8], s[8];
};

__device__ __forceinline__ void rotation_of(const AppendArgs& a, int t, int e, Rotation* r) {
    const int half = a.n_dims >> 1;
    if (a.mode == SV_ROPE_NORM) {
        const int pos = __ldg(a.pos + t);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float2 w = make_float2(1.0f, 0.0f);
            if (e + i < a.n_dims) w = turn(__ldg(a.pairs + ((e + i) >> 1)), pos, a.mag);
            r->c[i] = r->c[i + 1] = w.x;
            r->s[i] = -w.y;
            r->s[i + 1] = w.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float2 w = make_float2(1.0f, 0.0f);
            const int d = e + i;
            if (d < a.n_dims) {
                const float4 f = __ldg(a.pairs + (d < half ? d : d - half));
                w = turn(f, __ldg(a.pos + (size_t)__float_as_int(f.z) * a.T + t), a.mag);
            }
            r->c[i] = w.x;
            r->s[i] = d < half ? -w.y : w.y;
        }
    }
}

// norm and rotation of one row's 8 elements; every thread of the row calls it.  The partner's elements
// are read again from the row (L1), so any n_dims does.
template <int HD, bool F32>
__device__ __forceinline__ void norm_turn(const AppendArgs& a, const uint8_t* row, int e, const float* w,
                                          const Rotation& r, float* x) {
    float scale = 1.0f;
    if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        scale = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = x[i] * scale * __ldg(w + e + i);
    }
    if (a.pairs && e < a.n_dims) {
        float y[8];
        const int half = a.n_dims >> 1;
        if (a.mode == SV_ROPE_NORM) {
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = x[i ^ 1];
        } else if ((half & 7) == 0) {
            const int pe = e < half ? e + half : e - half;
            load8<F32>(row, pe, y);
            if (w) {
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = y[i] * scale * __ldg(w + pe + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = e + i, pd = d < half ? d + half : d - half;
                y[i] = 0.0f;
                if (d < a.n_dims) y[i] = load1<F32>(row, pd) * (w ? scale * __ldg(w + pd) : 1.0f);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = fmaf(x[i], r.c[i], y[i] * r.s[i]);
    }
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// the code of x: round-half-even of x / s, held to +-127; NaN -> 0
__device__ __forceinline__ int code_of(float x, float inv) {
    if (!finite(x)) return x > 0.0f ? 127 : (x < 0.0f ? -127 : 0);
    return (int)fminf(fmaxf(rintf(__fmul_rn(x, inv)), -127.0f), 127.0f);
}

// NV: row passes of a block, page_size * HD / 8 / kThreads at most
template <int HD, bool F32, int NV>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int C = HD / 8;                  // threads per row
    constexpr int RP = kThreads / C;           // rows per pass
    pdl_wait();
    if (threadIdx.x == 0) pdl_trigger();
    const int e = (threadIdx.x % C) * 8;
    if ((int)blockIdx.x < a.n_kv_blocks) {
        // ---------------- one page's new rows of one kv head, K or V
        __shared__ float s_max[kThreads / 32];
        const int NKV = a.kv.n_kv_head;
        const int which = blockIdx.x & 1, h = (blockIdx.x >> 1) % NKV, item = (blockIdx.x >> 1) / NKV;
        if (item >= a.head[PH_PAGES]) return;
        const int4 it = a.pages[item];         // first row, page, offset in it, rows
        if (it.y < 0) return;                  // no page: dropped (the plan raised the error)
        const bool is_k = which == 0;
        const uint8_t* src = is_k ? a.k : a.v;
        const size_t nb = is_k ? a.k_nb : a.v_nb;
        const int r0 = threadIdx.x / C;
        float x[NV][8];
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int r = r0 + i * RP;
            if (r < it.w) load8<F32>(src + (size_t)(it.x + r) * nb + (size_t)h * HD * (F32 ? 4 : 2), e, x[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int r = r0 + i * RP;
            if (i * RP >= it.w) break;
            const bool live = r < it.w;
            if (!live) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = 0.0f;
            }
            if (is_k) {
                // whole warps go through (the norm's shuffles); a dead row takes the page's first
                const int t = it.x + (live ? r : 0);
                Rotation rot;
                if (a.pairs && e < a.n_dims) rotation_of(a, t, e, &rot);
                norm_turn<HD, F32>(a, a.k + (size_t)t * a.k_nb + (size_t)h * HD * (F32 ? 4 : 2), e, a.kn, rot, x[i]);
            }
            if (live) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (finite(x[i][j])) amax = fmaxf(amax, fabsf(x[i][j]));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
        float* sp = (is_k ? a.kv.k_scale : a.kv.v_scale) + (size_t)it.y * NKV + h;
        const float s_old = it.z > 0 ? *sp : 0.0f;
        __syncthreads();                       // the scale is read by all before one writes it
#pragma unroll
        for (int w = 0; w < kThreads / 32; w++) amax = fmaxf(amax, s_max[w]);
        if (amax < 7.8886090522101181e-31f) amax = 0.0f;   // 2^-100: 1 / s stays finite
        const float s = fmaxf(s_old, __fdiv_rn(amax, 127.0f));
        const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
        if (threadIdx.x == 0) *sp = s;
        uint8_t* page = static_cast<uint8_t*>(is_k ? a.kv.k : a.kv.v) + ((size_t)it.y * NKV + h) * a.kv.page_size * HD;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int r = r0 + i * RP;
            if (r < it.w) {
                uint32_t w[2];
#pragma unroll
                for (int j = 0; j < 2; j++)
                    w[j] = (uint32_t)(code_of(x[i][4 * j], inv) & 255) | (uint32_t)(code_of(x[i][4 * j + 1], inv) & 255) << 8 |
                           (uint32_t)(code_of(x[i][4 * j + 2], inv) & 255) << 16 |
                           (uint32_t)(code_of(x[i][4 * j + 3], inv) & 255) << 24;
                *reinterpret_cast<uint2*>(page + (size_t)(it.z + r) * HD + e) = make_uint2(w[0], w[1]);
            }
        }
        if (s > s_old && it.z > 0) {           // the rows that the page holds, rounded to the new scale
            const float f = __fmul_rn(s_old, inv);
            for (int r = r0; r < it.z; r += RP) {
                uint2* p = reinterpret_cast<uint2*>(page + (size_t)r * HD + e);
                uint2 w = *p;
                uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    uint32_t o = 0;
#pragma unroll
                    for (int b = 0; b < 4; b++)
                        o |= (uint32_t)(code_of((float)(int8_t)(ww[j] >> (8 * b)), f) & 255) << (8 * b);
                    ww[j] = o;
                }
                *p = w;
            }
        }
    } else {
        // ---------------- query rows: 8 elements of `loop` heads of one token per thread
        const long long id = (long long)(blockIdx.x - a.n_kv_blocks) * RP + threadIdx.x / C;
        const int g = (int)(id % a.n_groups);
        const long long t64 = id / a.n_groups;
        const int live_rows = __ldg(a.q_start + a.n_req);
        const bool live = t64 < live_rows;
        const int t = live ? (int)t64 : 0;
        if (!__any_sync(0xffffffffu, live)) return;
        Rotation rot;
        if (a.pairs && e < a.n_dims) rotation_of(a, t, e, &rot);
        for (int i = 0; i < a.loop; i++) {         // the same count in every lane: the norm's shuffles
            const int h = min(g * a.loop + i, a.NH - 1);
            const uint8_t* row = a.q + (size_t)t * a.q_nb + (size_t)h * HD * (F32 ? 4 : 2);
            float x[8];
            load8<F32>(row, e, x);
            norm_turn<HD, F32>(a, row, e, a.qn, rot, x);
            __syncwarp();                      // q_out may be q: the row's partners have been read
            if (live && g * a.loop + i < a.NH) store8(a.q_out, ((size_t)t * a.NH + h) * HD + e, a.q_out_f32, x);
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
    a.pages = reinterpret_cast<const int4*>(work + l.page);
    a.head = reinterpret_cast<const int*>(work + l.head);
    a.n_kv_blocks = l.page_cap * kv.n_kv_head * 2;
    a.q_out = r.q_out;
    a.q_out_f32 = r.q_out_type == SV_TYPE_F32;
    a.q_start = s.q_start;
    a.n_req = s.n_req;
    a.err = kv.err;
    // One head per thread while that still fits the GPU at once (latency); eight otherwise, which
    // computes the sines an eighth as often.
    const int C = kv.head_dim / 8;
    a.loop = (int64_t)s.n_tokens * s.n_head * C > (int64_t)device_sm_count() * 1024 ? 8 : 1;
    a.n_groups = ceil_div(s.n_head, a.loop);
    const int64_t q_blocks = ((int64_t)s.n_tokens * a.n_groups + kThreads / C - 1) / (kThreads / C);
    const dim3 grid((unsigned)(a.n_kv_blocks + q_blocks)), block(kThreads);
    const int rows = kv.page_size < s.max_new ? kv.page_size : s.max_new;    // new rows of one page, at most
    const int nv = ceil_div(rows, kThreads / C);
    const bool f32 = r.type == SV_TYPE_F32;
#define SV_APPEND(HD_, NV_)                                                                              \
    if (kv.head_dim == HD_ && nv <= NV_)                                                                 \
        return f32 ? launch_pdl(paged_append_kernel<HD_, true, NV_>, grid, block, 0, st, a)              \
                   : launch_pdl(paged_append_kernel<HD_, false, NV_>, grid, block, 0, st, a);
    SV_APPEND(64, 1) SV_APPEND(64, 4)
    SV_APPEND(128, 1) SV_APPEND(128, 4) SV_APPEND(128, 8)
    SV_APPEND(256, 1) SV_APPEND(256, 4) SV_APPEND(256, 16)
#undef SV_APPEND
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
