// paged_prefill.cu - attention of requests with many rows over the paged 8-bit cache, one warp per query row and head.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = exp2(s_j - m), s_j = scale log2(e) ks[page] (q . c_j), m the running
// maximum.  Lane l holds elements l + 32 i of q and o.
#include "common.cuh"
#include "paged.hpp"

namespace svkv {

namespace {

template <int HD>
__global__ void __launch_bounds__(256) paged_attn_kernel(const __grid_constant__ PagedAttn a) {
    constexpr int N = HD / 32;
    pdl_wait();
    const int4* req = reinterpret_cast<const int4*>(a.work + a.l.req);
    const int lane = threadIdx.x & 31;
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = (int)(id / a.n_head), head = (int)(id % a.n_head), h = head / a.G;
    if (t >= a.n_tokens) return;
    int r = 0;
    for (int lo = 0, hi = a.n_req; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (req[mid].x <= t) lo = mid;
        else hi = mid;
        r = lo;
    }
    const int4 q = req[r];
    if (t >= q.x + q.y || q.y * a.G <= kDecRows) return;
    const int pos = q.z + t - q.x, end = min(pos + 1, q.w), begin = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int ps = a.kv.page_size, NKV = a.kv.n_kv_head;
    float x[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const size_t e = (size_t)head * HD + lane + 32 * i;
        x[i] = a.q_type == SV_TYPE_F32 ? __half2float(__float2half_rn(reinterpret_cast<const float*>(a.q + (size_t)t * a.q_nb)[e]))
                                       : __half2float(reinterpret_cast<const __half*>(a.q + (size_t)t * a.q_nb)[e]);
        o[i] = 0.0f;
    }
    for (int j = begin; j < end; j++) {
        const int page = a.table[(size_t)r * a.max_blocks + j / ps];
        if (page < 0 || page >= a.kv.n_pages) {
            if (a.err) atomicOr(a.err, SV_DEVERR_PAGES);
            continue;
        }
        const size_t unit = (size_t)page * NKV + h, off = (unit * ps + j % ps) * HD;
        const int8_t* k = static_cast<const int8_t*>(a.kv.k) + off;
        const int8_t* v = static_cast<const int8_t*>(a.kv.v) + off;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) s = fmaf(x[i], (float)k[lane + 32 * i], s);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        s *= a.kv.k_scale[unit] * a.scale_log2;
        const float mn = fmaxf(m, s), f = exp2f(m - mn), p = exp2f(s - mn), pv = p * a.kv.v_scale[unit];
        l = l * f + p;
        m = mn;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = fmaf(pv, (float)v[lane + 32 * i], o[i] * f);
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const size_t e = ((size_t)t * a.n_head + head) * HD + lane + 32 * i;
        if (a.out_type == SV_TYPE_F32) static_cast<float*>(a.out)[e] = o[i] * inv;
        else static_cast<__half*>(a.out)[e] = __float2half_rn(o[i] * inv);
    }
}

}  // namespace

cudaError_t launch_paged_prefill(const PagedAttn& a, cudaStream_t st) {
    if (a.l.pre_cap == 0) return cudaSuccess;
    const dim3 grid((unsigned)(((int64_t)a.n_tokens * a.n_head + 7) / 8));
    if (a.kv.head_dim == 64) return launch_pdl(paged_attn_kernel<64>, grid, dim3(256), 0, st, a);
    if (a.kv.head_dim == 128) return launch_pdl(paged_attn_kernel<128>, grid, dim3(256), 0, st, a);
    return launch_pdl(paged_attn_kernel<256>, grid, dim3(256), 0, st, a);
}

}  // namespace svkv
