// paged_cache.hip — appending new tokens to a paged K/V cache, with the position rotation on the
// way, and reading rows back (gfx950). The cache's layout: paged.hpp.
//
// Rotation as apply_rope_inplace (api/cortex_sdk.cpp:1395-1423), adjacent pairs:
//   (x0, x1) -> (x0 c - x1 s, x0 s + x1 c),  c + i s = exp(i pos theta^(-2j / hd)) for pair j.
// The angle is held in turns in fp64 (an fp32 angle is off by 2^-24 of itself: 4e-3 rad at
// position 65536), its whole turns dropped before sincos; the pairs are turned in fp64, which runs
// at the fp32 rate here, and rounded once to fp32, so that a 4-bit row is what the formulas say
// and not a neighbour across a border between codes.
//
// 4 bits, per position and group of 32 dims x: minimum m = fp16(min x), scale s = fp16(max(0,
// (max x - m) / 15)), code = clamp(rint((x - m) / s), 0, 15), ties to even; codes 0 where s = 0. A
// group holding a NaN or an infinity, or whose minimum or scale leaves fp16, gets NaN for both and
// reads as NaN.
//
// One wave takes a head (HD / 2 lanes, a pair of dims each; two heads at HD 64) at 8 consecutive
// positions, aligned to 8: the unit in which V's pages are laid out, so that one thread writes all
// of a word or piece that the block's tokens share, and no two threads of a call write one word.
//
// Bound by memory: 5751 fp32 tokens of 32 + 2 x 8 heads of 128 take 43 us into fp16 pages, 6.0
// TB/s, and 58 into 4-bit ones, 4.2 TB/s (243 MB, and the codes' work beside them); a step's tokens
// are one round trip (64 sequences 5 us, one 3). The read of their rows as fp16 takes 10 and 12 us where 47
// and 31 MB are 9 and 6: a lane stores 4 bytes a row, and on 4-bit pages four lanes share a word.
#include <hip/hip_runtime.h>

#include <cmath>

#include "paged.hpp"

namespace {

using csdr::kGroup;
using csdr::PagedView;
using csdr::SeqRows;
using csdr::set_error;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr long long kMaxBlocks = (1LL << 32) / kThreads - 1;  // fewer than 2^32 threads a launch

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Two values at any alignment of their type.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Pair {
    T a, b;
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(dpp<CTRL>(__float_as_uint(v)));
}
// lane ^ 1, lane ^ 2, mirrored within 8 and within 16 lanes: after the first two every quad holds
// one value, so the mirrors join the quads and the halves of a row of 16 lanes (a group's 32 dims).
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;

__device__ __forceinline__ float row_min(float v) {
    v = fminf(v, dpp<kXor1>(v));
    v = fminf(v, dpp<kXor2>(v));
    v = fminf(v, dpp<kHalfMirror>(v));
    return fminf(v, dpp<kMirror>(v));
}
__device__ __forceinline__ uint32_t quad_or(uint32_t v) {
    v |= dpp<kXor1>(v);
    return v | dpp<kXor2>(v);
}
__device__ __forceinline__ uint32_t row_or(uint32_t v) {
    v = quad_or(v);
    v |= dpp<kHalfMirror>(v);
    return v | dpp<kMirror>(v);
}

struct Quant {
    _Float16 s, m;
};

// Scale and minimum of the group that a row of 16 lanes holds (x0, x1 in each lane).
__device__ __forceinline__ Quant group_range(float x0, float x1) {
    const bool bad = !(fabsf(x0) < INFINITY) || !(fabsf(x1) < INFINITY);
    const float lo = row_min(fminf(x0, x1)), hi = -row_min(-fmaxf(x0, x1));
    Quant q;
    q.m = (_Float16)lo;
    q.s = (_Float16)fmaxf((hi - (float)q.m) / 15.0f, 0.0f);
    if (row_or(bad) || !(fabsf((float)q.m) < INFINITY) || !((float)q.s < INFINITY)) {
        q.m = (_Float16)NAN;
        q.s = (_Float16)NAN;
    }
    return q;
}

// rint((x - m) / s) within [0, 15], in exact arithmetic: the quotient is estimated in fp32 and
// corrected by the fp64 remainder (x - m and code * s are exact in fp64).
__device__ __forceinline__ uint32_t code_of(float x, Quant q) {
    const float s = (float)q.s;
    if (!(s > 0.0f)) return 0u;
    const double d = (double)x - (double)(float)q.m, ds = (double)s;
    float c = fminf(fmaxf(rintf((float)d / s), 0.0f), 15.0f);
    const double r2 = 2.0 * fma(-(double)c, ds, d);
    const bool odd = ((int)c & 1) != 0;
    if (r2 > ds || (r2 == ds && odd)) c += 1.0f;
    else if (r2 < -ds || (r2 == -ds && odd)) c -= 1.0f;
    return (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);
}

struct AppendArgs {
    PagedView pv;
    const void *q, *k, *v;
    void* q_out;
    long long q_stride, k_stride, v_stride;  // elements between tokens
    int hq, nblk;
    bool rotate;
    double log2_theta;
};

// XT: the element type of q, k, v and q_out.
template <int HD, bool Q4, typename XT>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
    constexpr int LANES = HD / 2;       // lanes per head
    constexpr int HPW = 64 / LANES;     // heads per wave
    const PagedView& pv = a.pv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int li = lane % LANES;
    const int unit = (blockIdx.y * kWaves + wave) * HPW + lane / LANES;
    if (unit >= a.hq + 2 * pv.hkv) return;
    const int b = blockIdx.x / a.nblk;
    const SeqRows r = csdr::seq_rows(pv, b);
    const int j0 = max(r.p0, 0) & ~7;  // the block of the first position
    const int base = j0 + 8 * (int)(blockIdx.x % a.nblk);
    // this block's tokens: positions [t0, t1), rows shift + position
    const int t0 = max(base, max(r.p0, 0)), t1 = min(base + 8, r.p0 + r.n);
    if (t0 >= t1) return;
    const long long row0 = (long long)r.first - r.p0;

    const bool is_q = unit < a.hq, is_v = unit >= a.hq + pv.hkv;
    const int head = is_q ? unit : (unit - a.hq) % pv.hkv;
    if (is_q && !a.q) return;
    const XT* src = static_cast<const XT*>(is_q ? a.q : is_v ? a.v : a.k);
    const long long stride = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;

    float x[8][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int p = base + i;
        const bool mine = p >= t0 && p < t1;
        const long long row = row0 + (mine ? p : t0);
        const Pair<XT> w = *reinterpret_cast<const Pair<XT>*>(src + row * stride +
                                                             (long long)head * HD + 2 * li);
        x[i][0] = (float)w.a;
        x[i][1] = (float)w.b;
    }
    if (!is_v && a.rotate) {
        // turns per position, the block's angle, then one position further each time
        const double f = exp2(-(double)(2 * li) / HD * a.log2_theta) * 0.15915494309189533577;
        double c, s, cf = 1.0, sf = 0.0;
        const double turns = (double)t0 * f;
        sincospi(2.0 * (turns - rint(turns)), &s, &c);
        if (t1 - t0 > 1) sincospi(2.0 * (f - rint(f)), &sf, &cf);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = base + i;
            if (p < t0 || p >= t1) continue;
            const double x0 = x[i][0], x1 = x[i][1];
            x[i][0] = (float)fma(x0, c, -(x1 * s));
            x[i][1] = (float)fma(x0, s, x1 * c);
            const double cn = fma(c, cf, -(s * sf));
            s = fma(c, sf, s * cf);
            c = cn;
        }
    }
    if (is_q) {
        XT* dst = static_cast<XT*>(a.q_out) + (long long)head * HD + 2 * li;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = base + i;
            if (p < t0 || p >= t1) continue;
            Pair<XT> w;
            w.a = (XT)x[i][0];
            w.b = (XT)x[i][1];
            *reinterpret_cast<Pair<XT>*>(dst + (row0 + p) * ((long long)a.hq * HD)) = w;
        }
        return;
    }
    const int page = csdr::page_of(pv, b, base);
    if (page < 0) return;
    uint8_t* hp = (is_v ? pv.v : pv.k) + csdr::head_offset<Q4>(pv, HD, page, head);
    const int ps = pv.page_size(), slot0 = base & (ps - 1);
    const bool whole = t1 - t0 == 8;
    if constexpr (!Q4) {
        _Float16* h = reinterpret_cast<_Float16*>(hp);
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int p = base + i;
                if (p < t0 || p >= t1) continue;
                *reinterpret_cast<h2*>(h + (slot0 + i) * HD + 2 * li) =
                    h2{(_Float16)x[i][0], (_Float16)x[i][1]};
            }
        } else {
            _Float16* d = h + ((size_t)(slot0 >> 3) * HD + 2 * li) * 8;
            if (whole) {
                h8 v0, v1;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v0[i] = (_Float16)x[i][0];
                    v1[i] = (_Float16)x[i][1];
                }
                reinterpret_cast<h8*>(d)[0] = v0;
                reinterpret_cast<h8*>(d)[1] = v1;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int p = base + i;
                    if (p < t0 || p >= t1) continue;
                    d[i] = (_Float16)x[i][0];
                    d[8 + i] = (_Float16)x[i][1];
                }
            }
        }
    } else {
        const int g = 2 * li / kGroup;
        uint32_t w0 = 0u, w1 = 0u, mask = 0u;  // V: the words of this lane's two dims
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = base + i;
            if (p < t0 || p >= t1) continue;
            const Quant qn = group_range(x[i][0], x[i][1]);
            const uint32_t c0 = code_of(x[i][0], qn), c1 = code_of(x[i][1], qn);
            if (!is_v) {
                // dims 2 li, 2 li + 1 are codes 2 (li % 4) and the next of their word
                const uint32_t w = quad_or((c0 | c1 << 16) << (4 * (li & 3)));
                if ((li & 3) == 0)
                    reinterpret_cast<uint32_t*>(hp)[csdr::k_word<HD>(slot0 + i, 2 * li)] = w;
            } else {
                const int sh = csdr::code_shift(i);
                w0 |= c0 << sh;
                w1 |= c1 << sh;
                mask |= 15u << sh;
            }
            if ((li & 15) == 0) {
                *reinterpret_cast<_Float16*>(hp + csdr::scale_offset(HD, ps, g, slot0 + i)) = qn.s;
                *reinterpret_cast<_Float16*>(hp + csdr::min_offset(HD, ps, g, slot0 + i)) = qn.m;
            }
        }
        if (is_v) {
            uint32_t* d0 = reinterpret_cast<uint32_t*>(hp) + csdr::v_word<HD>(slot0, 2 * li);
            uint32_t* d1 = reinterpret_cast<uint32_t*>(hp) + csdr::v_word<HD>(slot0, 2 * li + 1);
            if (!whole) {  // the block's other positions keep their codes
                w0 |= *d0 & ~mask;
                w1 |= *d1 & ~mask;
            }
            *d0 = w0;
            *d1 = w1;
        }
    }
}

struct ReadArgs {
    PagedView pv;
    void *k, *v;
    int nblk;
};

// The rows of a call's tokens as the values the cache holds; zeros where it holds none.
template <int HD, bool Q4, typename XT>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
    constexpr int LANES = HD / 2;
    constexpr int HPW = 64 / LANES;
    const PagedView& pv = a.pv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int li = lane % LANES;
    const int unit = (blockIdx.y * kWaves + wave) * HPW + lane / LANES;
    if (unit >= 2 * pv.hkv) return;
    const int b = blockIdx.x / a.nblk;
    const SeqRows r = csdr::seq_rows(pv, b);
    const int base = (r.p0 & ~7) + 8 * (int)(blockIdx.x % a.nblk);  // p0 may be negative
    const int t0 = max(base, r.p0), t1 = min(base + 8, r.p0 + r.n);
    if (t0 >= t1) return;
    const bool is_v = unit >= pv.hkv;
    const int head = unit % pv.hkv;
    const int page = csdr::page_of(pv, b, base);
    const int ps = pv.page_size(), slot0 = base & (ps - 1);
    const uint8_t* hp =
        (is_v ? pv.v : pv.k) + csdr::head_offset<Q4>(pv, HD, max(page, 0), head);
    XT* dst = static_cast<XT*>(is_v ? a.v : a.k) + (long long)head * HD + 2 * li;
    // the block's data first, all of it (page 0 stands in for none)
    float x[8][2];
    if constexpr (!Q4) {
        const _Float16* h = reinterpret_cast<const _Float16*>(hp);
        if (!is_v) {
            h2 w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = *reinterpret_cast<const h2*>(h + (slot0 + i) * HD + 2 * li);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i][0] = (float)w[i][0];
                x[i][1] = (float)w[i][1];
            }
        } else {
            const h8* d = reinterpret_cast<const h8*>(h + ((slot0 >> 3) * HD + 2 * li) * 8);
            const h8 v0 = d[0], v1 = d[1];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i][0] = (float)v0[i];
                x[i][1] = (float)v1[i];
            }
        }
    } else {
        const int g = 2 * li / kGroup;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(hp);
        const h8 sc = *reinterpret_cast<const h8*>(hp + csdr::scale_offset(HD, ps, g, slot0));
        const h8 mn = *reinterpret_cast<const h8*>(hp + csdr::min_offset(HD, ps, g, slot0));
        uint32_t w[8];  // K: the word of each position; V: the words of the lane's two dims
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = words[is_v ? csdr::v_word<HD>(slot0, 2 * li + (i & 1))
                              : csdr::k_word<HD>(slot0 + i, 2 * li)];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t code = is_v ? w[u] >> csdr::code_shift(i)
                                           : w[i] >> (4 * (li & 3) + 16 * u);
                x[i][u] = fmaf((float)sc[i], (float)(code & 15u), (float)mn[i]);
            }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int p = base + i;
        if (p < t0 || p >= t1) continue;
        const long long row = (long long)r.first + (p - r.p0);
        Pair<XT> w{};
        if (page >= 0) {
            w.a = (XT)x[i][0];
            w.b = (XT)x[i][1];
        }
        *reinterpret_cast<Pair<XT>*>(dst + row * ((long long)pv.hkv * HD)) = w;
    }
}

// 8-position blocks that max_q consecutive positions can touch
int blocks_of(int max_q) { return (int)(((long long)max_q + 14) / 8); }

template <int HD, bool Q4>
void launch_append(const AppendArgs& a, int dtype, dim3 grid, hipStream_t st) {
    if (dtype == CSDR_F32) append_kernel<HD, Q4, float><<<grid, kThreads, 0, st>>>(a);
    else append_kernel<HD, Q4, _Float16><<<grid, kThreads, 0, st>>>(a);
}

template <int HD, bool Q4>
void launch_read(const ReadArgs& a, int dtype, dim3 grid, hipStream_t st) {
    if (dtype == CSDR_F32) read_kernel<HD, Q4, float><<<grid, kThreads, 0, st>>>(a);
    else read_kernel<HD, Q4, _Float16><<<grid, kThreads, 0, st>>>(a);
}

}  // namespace

namespace csdr {

int paged_check(const char* what, const csdr_paged_kv* kv, int n_tokens, const int32_t* q_start,
                int max_q, PagedView* out) {
    const std::string w = what;
    if (!kv) return set_error(CSDR_E_INVALID, w + ": no cache");
    if (!kv->k_pages || !kv->v_pages || !kv->page_table || !kv->lens)
        return set_error(CSDR_E_INVALID, w + ": a pointer of the cache is NULL");
    if (kv->kv_dtype != CSDR_F16 && kv->kv_dtype != CSDR_Q4)
        return set_error(CSDR_E_UNSUPPORTED, w + ": kv_dtype must be CSDR_F16 or CSDR_Q4");
    if (kv->head_dim != 64 && kv->head_dim != 128)
        return set_error(CSDR_E_UNSUPPORTED, w + ": head_dim must be 64 or 128");
    int shift = 4;
    while (shift < 12 && (1 << shift) != kv->page_size) ++shift;
    if ((1 << shift) != kv->page_size)
        return set_error(CSDR_E_UNSUPPORTED,
                         w + ": page_size must be a power of two from 16 to 4096");
    if (kv->n_pages <= 0 || kv->n_kv_heads <= 0 || kv->n_kv_heads > 65535 || kv->n_seqs <= 0 ||
        kv->table_stride <= 0)
        return set_error(CSDR_E_INVALID, w + ": bad cache shape");
    if (((long long)kv->table_stride << shift) > kMaxPositions)
        return set_error(CSDR_E_INVALID, w + ": the table holds more than 2^30 positions");
    if ((reinterpret_cast<uintptr_t>(kv->k_pages) | reinterpret_cast<uintptr_t>(kv->v_pages)) % 16)
        return set_error(CSDR_E_INVALID, w + ": pages must be 16-byte aligned");
    if (n_tokens <= 0) return set_error(CSDR_E_INVALID, w + ": no tokens");
    int T = 0;
    if (q_start) {
        if (max_q <= 0) return set_error(CSDR_E_INVALID, w + ": max_q must be positive");
        if (max_q > n_tokens) max_q = n_tokens;
    } else {
        if (n_tokens % kv->n_seqs)
            return set_error(CSDR_E_INVALID,
                             w + ": without q_start every sequence has as many tokens");
        T = max_q = n_tokens / kv->n_seqs;
    }
    *out = PagedView{static_cast<uint8_t*>(kv->k_pages), static_cast<uint8_t*>(kv->v_pages),
                     kv->page_table, kv->lens, q_start, kv->n_pages, shift, kv->n_kv_heads,
                     kv->table_stride, kv->n_seqs, n_tokens, T, max_q};
    return CSDR_OK;
}

}  // namespace csdr

extern "C" {

CSDR_API size_t csdr_paged_page_bytes(int kv_dtype, int page_size, int n_kv_heads, int head_dim) {
    if ((kv_dtype != CSDR_F16 && kv_dtype != CSDR_Q4) || page_size < 16 || page_size > 4096 ||
        (page_size & (page_size - 1)) || n_kv_heads <= 0 || n_kv_heads > 65535 ||
        (head_dim != 64 && head_dim != 128))
        return 0;
    return (size_t)n_kv_heads * csdr::paged_head_bytes(kv_dtype == CSDR_Q4, page_size, head_dim);
}

CSDR_API int csdr_paged_append(const csdr_paged_kv* kv, const void* q, const void* k,
                               const void* v, int dtype, int n_tokens, const int32_t* q_start,
                               int max_q, int Hq, int64_t q_stride, int64_t k_stride,
                               int64_t v_stride, float theta, void* q_out, void* hip_stream) {
    AppendArgs a{};
    if (int rc = csdr::paged_check("paged_append", kv, n_tokens, q_start, max_q, &a.pv)) return rc;
    if (!k || !v || (q != nullptr) != (q_out != nullptr))
        return set_error(CSDR_E_INVALID, "paged_append: a pointer is NULL");
    if (dtype != CSDR_F32 && dtype != CSDR_F16)
        return set_error(CSDR_E_INVALID, "paged_append: dtype must be CSDR_F32 or CSDR_F16");
    if (q && (Hq <= 0 || Hq > 65535 || Hq % kv->n_kv_heads))
        return set_error(CSDR_E_INVALID, "paged_append: bad number of heads");
    if (q && q_out == q && q_stride != 0 && q_stride != (int64_t)Hq * kv->head_dim)
        return set_error(CSDR_E_INVALID, "paged_append: q in place must be packed");
    if (!(theta >= 0.0f) || theta == INFINITY)
        return set_error(CSDR_E_INVALID, "paged_append: theta must be positive, or 0 for none");
    const int hd = kv->head_dim;
    const int64_t kvw = (int64_t)kv->n_kv_heads * hd, qw = (int64_t)Hq * hd;
    a.q_stride = q_stride ? q_stride : qw;
    a.k_stride = k_stride ? k_stride : kvw;
    a.v_stride = v_stride ? v_stride : kvw;
    if (a.k_stride < kvw || a.v_stride < kvw || (q && a.q_stride < qw))
        return set_error(CSDR_E_INVALID, "paged_append: a token stride is below a token's values");
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.hq = q ? Hq : 0;
    a.nblk = blocks_of(a.pv.max_q);
    a.rotate = theta > 0.0f;
    a.log2_theta = a.rotate ? std::log2((double)theta) : 0.0;
    const int upw = kWaves * (128 / hd), units = a.hq + 2 * kv->n_kv_heads;
    const long long gx = (long long)kv->n_seqs * a.nblk;
    if (gx > kMaxBlocks) return set_error(CSDR_E_INVALID, "paged_append: too many tokens");
    const dim3 grid((unsigned)gx, (units + upw - 1) / upw);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const bool q4 = kv->kv_dtype == CSDR_Q4;
    if (hd == 64) {
        if (q4) launch_append<64, true>(a, dtype, grid, st);
        else launch_append<64, false>(a, dtype, grid, st);
    } else {
        if (q4) launch_append<128, true>(a, dtype, grid, st);
        else launch_append<128, false>(a, dtype, grid, st);
    }
    CSDR_LAUNCH_CHECK("paged_append");
    return CSDR_OK;
}

CSDR_API int csdr_paged_read(const csdr_paged_kv* kv, int n_tokens, const int32_t* q_start,
                             int max_q, void* k, void* v, int dtype, void* hip_stream) {
    ReadArgs a{};
    if (int rc = csdr::paged_check("paged_read", kv, n_tokens, q_start, max_q, &a.pv)) return rc;
    if (!k || !v) return set_error(CSDR_E_INVALID, "paged_read: a pointer is NULL");
    if (dtype != CSDR_F32 && dtype != CSDR_F16)
        return set_error(CSDR_E_INVALID, "paged_read: dtype must be CSDR_F32 or CSDR_F16");
    a.k = k;
    a.v = v;
    a.nblk = blocks_of(a.pv.max_q);
    const int hd = kv->head_dim, upw = kWaves * (128 / hd);
    const long long gx = (long long)kv->n_seqs * a.nblk;
    if (gx > kMaxBlocks) return set_error(CSDR_E_INVALID, "paged_read: too many tokens");
    const dim3 grid((unsigned)gx, (2 * kv->n_kv_heads + upw - 1) / upw);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const bool q4 = kv->kv_dtype == CSDR_Q4;
    if (hd == 64) {
        if (q4) launch_read<64, true>(a, dtype, grid, st);
        else launch_read<64, false>(a, dtype, grid, st);
    } else {
        if (q4) launch_read<128, true>(a, dtype, grid, st);
        else launch_read<128, false>(a, dtype, grid, st);
    }
    CSDR_LAUNCH_CHECK("paged_read");
    return CSDR_OK;
}

}  // extern "C"
