// paged_attn.hip — attention of new tokens over the pages of their sequences (gfx950): fp16 or
// 4-bit pages (layout: paged.hpp), one token per sequence or many, scores capped, lowered by
// distance, limited to a window and a prefix.
//
// Reference: Kernels::multi_head_attention (kernels/attention_kernels.cpp:26-113) with the cache
// kernels/flash_attention.cpp:165-247 intends; repeat_kv_heads (api/cortex_sdk.cpp:1453-1478).
//
//   s = scale q.k;  s = cap tanh(s / cap);  s -= slope_h |pq - p|
//   seen: p < len and (p < prefix or (p <= pq and pq - p < window));  out = softmax(s) V
#include <hip/hip_runtime.h>

#include <cmath>

#include "paged.hpp"

namespace {

using csdr::PagedView;
using csdr::SeqRows;
using csdr::set_error;

struct AttnArgs {
    PagedView pv;
    const void* q;
    void* out;
    long long q_stride;
    int hq;
    float scale;
    float cap, inv_cap;  // cap 0: none
    int window;          // 0: none
    const float* slopes;
    const int32_t* prefix;
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}

// Positions that a token of sequence b sees, besides those of its own past.
struct Seen {
    int keys, window, prefix;
    __device__ bool at(int pq, int p) const {
        return p < keys && (p < prefix || (p <= pq && pq - p < window));
    }
};

__device__ __forceinline__ Seen seen_of(const AttnArgs& a, int b, const SeqRows& r) {
    Seen s;
    s.keys = min(r.len, a.pv.capacity());
    s.window = a.window > 0 ? a.window : 0x7fffffff;
    s.prefix = a.prefix ? a.prefix[b] : 0;
    return s;
}

__device__ __forceinline__ float shaped(const AttnArgs& a, float s, float slope, int dist) {
    if (a.cap > 0.0f) s = a.cap * tanhf(s * a.inv_cap);
    return s - slope * (float)abs(dist);
}

// One row (token, head) by one wave, position by position: lanes over 64 positions for the scores,
// over the dims for the values. Nothing of an unseen position is used.
template <int HD, bool Q4, typename XT>
__device__ void attend_row(const AttnArgs& a, int b, const SeqRows& r, int t, int h) {
    const PagedView& pv = a.pv;
    const int lane = threadIdx.x & 63;
    const int kvh = h / (a.hq / pv.hkv), ps = pv.page_size();
    const Seen seen = seen_of(a, b, r);
    const int pq = r.p0 + t;
    const long long row = (long long)r.first + t;
    const XT* q = static_cast<const XT*>(a.q) + row * a.q_stride + (long long)h * HD;
    const float slope = a.slopes ? a.slopes[h] : 0.0f;
    float m = -INFINITY, l = 0.0f, o[HD / 64] = {};
    const int end = pq < 0 ? 0 : max(min(pq + 1, seen.keys), min(seen.prefix, seen.keys));
    for (int p0 = 0; p0 < end; p0 += 64) {
        const int p = p0 + lane;
        const int page = seen.at(pq, p) ? csdr::page_of(pv, b, p) : -1;
        const uint64_t live = __ballot(page >= 0);
        if (!live) continue;
        float s = -INFINITY;
        if (page >= 0) {
            const uint8_t* kp = pv.k + csdr::head_offset<Q4>(pv, HD, page, kvh);
            float d = 0.0f;
            for (int i = 0; i < HD; ++i)
                d = fmaf((float)q[i], csdr::cache_value<HD, Q4>(kp, false, ps, p & (ps - 1), i), d);
            s = shaped(a, d * a.scale, slope, pq - p);
        }
        const float mn = fmaxf(m, wave_max(s));
        // NaN is not seen by the maxima: it reaches the sum through its own weight
        if (mn == -INFINITY && !__any(s != s)) continue;
        const float alpha = m == -INFINITY ? 0.0f : expf(m - mn);
        const float w = page >= 0 ? expf(s - mn) : 0.0f;
        l = l * alpha + csdr::wave_sum(w);
        m = mn;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) o[c] *= alpha;
        for (int j = 0; j < 64; ++j) {
            if (!(live >> j & 1)) continue;
            const float wj = __shfl(w, j, 64);
            const int pj = __shfl(page, j, 64), sj = (p0 + j) & (ps - 1);
            const uint8_t* vp = pv.v + csdr::head_offset<Q4>(pv, HD, pj, kvh);
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
                o[c] = fmaf(wj, csdr::cache_value<HD, Q4>(vp, true, ps, sj, lane + 64 * c), o[c]);
        }
    }
    XT* out = static_cast<XT*>(a.out) + (row * a.hq + h) * HD;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) out[lane + 64 * c] = (XT)(l == 0.0f ? 0.0f : o[c] / l);
}

template <int HD, bool Q4, typename XT>
__global__ __launch_bounds__(64) void row_kernel(AttnArgs a) {
    const int b = blockIdx.x / a.pv.max_q, t = blockIdx.x % a.pv.max_q;
    const SeqRows r = csdr::seq_rows(a.pv, b);
    if (t >= r.n) return;
    attend_row<HD, Q4, XT>(a, b, r, t, blockIdx.y);
}

template <int HD, bool Q4>
void launch(const AttnArgs& a, int dtype, hipStream_t st) {
    const dim3 grid((unsigned)((long long)a.pv.n_seqs * a.pv.max_q), a.hq);
    if (dtype == CSDR_F32) row_kernel<HD, Q4, float><<<grid, 64, 0, st>>>(a);
    else row_kernel<HD, Q4, _Float16><<<grid, 64, 0, st>>>(a);
}

}  // namespace

extern "C" {

CSDR_API size_t csdr_paged_attn_workspace_bytes(const csdr_paged_kv* kv, int n_tokens,
                                                const int32_t* q_start, int max_q, int Hq,
                                                int max_len) {
    (void)kv, (void)n_tokens, (void)q_start, (void)max_q, (void)Hq, (void)max_len;
    return 0;
}

CSDR_API int csdr_paged_attn(const csdr_paged_kv* kv, const void* q, int dtype, int n_tokens,
                             const int32_t* q_start, int max_q, int Hq, int64_t q_stride,
                             int max_len, float scale, const csdr_attn_options* options, void* out,
                             void* workspace, size_t workspace_bytes, void* hip_stream) {
    (void)workspace, (void)workspace_bytes;
    AttnArgs a{};
    if (int rc = csdr::paged_check("paged_attn", kv, n_tokens, q_start, max_q, &a.pv)) return rc;
    if (!q || !out) return set_error(CSDR_E_INVALID, "paged_attn: a pointer is NULL");
    if (dtype != CSDR_F32 && dtype != CSDR_F16)
        return set_error(CSDR_E_INVALID, "paged_attn: dtype must be CSDR_F32 or CSDR_F16");
    if (Hq <= 0 || Hq > 65535 || Hq % kv->n_kv_heads)
        return set_error(CSDR_E_INVALID, "paged_attn: bad number of heads");
    if (max_len < 0) return set_error(CSDR_E_INVALID, "paged_attn: max_len is negative");
    const int hd = kv->head_dim;
    a.q_stride = q_stride ? q_stride : (int64_t)Hq * hd;
    if (a.q_stride < (int64_t)Hq * hd)
        return set_error(CSDR_E_INVALID, "paged_attn: the token stride is below a token's values");
    if (!(std::fabs(scale) < INFINITY))
        return set_error(CSDR_E_INVALID, "paged_attn: the scale is not finite");
    a.scale = scale == 0.0f ? 1.0f / std::sqrt((float)hd) : scale;
    if (options) {
        if (!(options->softcap >= 0.0f && options->softcap < INFINITY) || options->window < 0)
            return set_error(CSDR_E_INVALID, "paged_attn: bad options");
        a.cap = options->softcap;
        a.inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
        a.window = options->window;
        a.slopes = options->slopes;
        a.prefix = options->prefix;
    }
    a.q = q;
    a.out = out;
    a.hq = Hq;
    if ((long long)kv->n_seqs * a.pv.max_q > 0x7fffffffLL)
        return set_error(CSDR_E_INVALID, "paged_attn: too many tokens");
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const bool q4 = kv->kv_dtype == CSDR_Q4;
    if (hd == 64) {
        if (q4) launch<64, true>(a, dtype, st);
        else launch<64, false>(a, dtype, st);
    } else {
        if (q4) launch<128, true>(a, dtype, st);
        else launch<128, false>(a, dtype, st);
    }
    CSDR_LAUNCH_CHECK("paged_attn");
    return CSDR_OK;
}

}  // extern "C"
