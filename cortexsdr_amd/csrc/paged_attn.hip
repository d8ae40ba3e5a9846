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

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

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
        // (no short cuts: they compile to branches)
        return (p < keys) & ((p < prefix) | ((p <= pq) & (pq - p < window)));
    }
};

__device__ __forceinline__ Seen seen_of(const AttnArgs& a, int b, const SeqRows& r) {
    Seen s;
    s.keys = min(r.len, a.pv.capacity());
    s.window = a.window > 0 ? a.window : 0x7fffffff;
    s.prefix = a.prefix ? a.prefix[b] : 0;
    return s;
}

// The tiles of T positions that columns at positions pq0 .. pq1 see: `low` tiles from 0 on
// (prefix), then those from w0 on (window and causal part), n in all.
template <int T>
struct Tiles {
    int low, w0, n;
    __device__ Tiles(const Seen& s, int pq0, int pq1) {
        const int first = max(0, pq0 - min(pq0 + 1, s.window) + 1) / T * T;
        const int end = pq1 < 0 ? 0 : min(s.keys, max(pq1 + 1, s.prefix));
        const int prefix = min(max(s.prefix, 0), s.keys);
        w0 = first;
        low = pq1 < 0 ? 0 : min((prefix + T - 1) / T, first / T);
        n = low + max(0, (end - first + T - 1) / T);
    }
    __device__ int at(int i) const { return i < low ? i * T : w0 + (i - low) * T; }
    // Tiles [lo, hi) of a split: equal shares of what there is, in whole units of tiles.
    __device__ void share(int split, int splits, int unit, int& lo, int& hi) const {
        const int each = ((n + splits - 1) / splits + unit - 1) / unit * unit;
        lo = min(n, split * each);
        hi = min(n, lo + each);
    }
};

__device__ __forceinline__ float shaped(const AttnArgs& a, float s, float slope, int dist) {
    if (a.cap > 0.0f) s = a.cap * tanhf(s * a.inv_cap);
    return s - slope * (float)abs(dist);
}

// One row (token, head) by one wave, position by position: lanes over 64 positions for the scores,
// over the dims for the values. Nothing of an unseen position is used. (The sum is 0 for a row that
// sees nothing, and for one whose scores are all -infinity: zeros and NaN.)
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
    bool sees = false;
    const int end = pq < 0 ? 0 : max(min(pq + 1, seen.keys), min(seen.prefix, seen.keys));
    for (int p0 = 0; p0 < end; p0 += 64) {
        const int p = p0 + lane;
        const int page = seen.at(pq, p) ? csdr::page_of(pv, b, p) : -1;
        const uint64_t live = __ballot(page >= 0);
        if (!live) continue;
        sees = true;
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
    for (int c = 0; c < HD / 64; ++c) out[lane + 64 * c] = (XT)(sees ? o[c] / l : 0.0f);
}

// ---------------------------------------------------------------- few tokens: split positions

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;       // positions per step of a wave
constexpr int kCols = 16;       // (token, query head) pairs per wave
constexpr int kStepWaves = 4;
constexpr float kLog2e = 1.44269504088896341f;
// Weights are 2^(s - m + bias) in the log2 domain, m a maximum that may lag `lag` behind, so that m
// moves, and the sums with it, only now and then: at most 2^15, near the top of fp16. fp32 calls: a
// pair keeps its 22 bits down to 2^(bias - 30) of the largest weight (the step of its low half is
// 2^-24); with a bias of 8, rows with a high maximum were 2e-5 to 1.6e-4 off. fp16 calls: 11 bits
// down to 2^-21 of it do, which leaves more room to lag. One rounding to those 11 bits is a choice
// of speed: outputs are 2.7e-4 to 3.0e-4 off where their own rounding makes 2.05e-4, and pairs, which
// leave just that, cost 161 -> 205 us (prompt of 4096 on fp16 pages), 461 -> 537 (prompts on 4-bit
// pages), 118 -> 135 and 46 -> 52 (single tokens on 4-bit pages). Single tokens on fp16 pages take
// pairs in fp16 calls too: there they cost nothing (78.1 us both, 32 sequences of 4096).
template <typename XT>
constexpr float kLag = sizeof(XT) == 4 ? 2.0f : 8.0f;
template <typename XT>
constexpr float kBias = 15.0f - kLag<XT>;
constexpr float kNoMax = -1e30f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 + code for the eight codes of a word: the codes shifted into an fp16 mantissa. `magic` is
// 16.0 twice, in a vector register: with the mask that makes one and-or a pair.
__device__ __forceinline__ h8 codes16(uint32_t w, uint32_t magic) {
    u4 r;
    r.x = ((w << 6) & 0x03C003C0u) | magic;
    r.y = ((w << 2) & 0x03C003C0u) | magic;
    r.z = ((w >> 2) & 0x03C003C0u) | magic;
    r.w = ((w >> 6) & 0x03C003C0u) | magic;
    return __builtin_bit_cast(h8, r);
}

// code - 8: the codes at the foot of a mantissa of 1024 or, four bits up, of 64, where pairs need
// no shift of their own (`m0`, `m1`: 1024.0 and 64.0 twice, in vector registers).
__device__ __forceinline__ h8 codes8(uint32_t w, uint32_t m0, uint32_t m1) {
    const uint32_t v = w >> 8;
    const h2 a = __builtin_bit_cast(h2, (w & 0x000F000Fu) | m0) - (_Float16)1032.0f;
    const h2 b = __builtin_bit_cast(h2, (w & 0x00F000F0u) | m1) - (_Float16)72.0f;
    const h2 c = __builtin_bit_cast(h2, (v & 0x000F000Fu) | m0) - (_Float16)1032.0f;
    const h2 d = __builtin_bit_cast(h2, (v & 0x00F000F0u) | m1) - (_Float16)72.0f;
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x times y (fp32 values with fp16 factors), rounded to fp16, and what the rounding left: both
// straight from the exact product (v_fma_mix).
template <bool PAIR>
__device__ __forceinline__ void split8(const float* x, h8 y, h8& hi, h8& lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        hi[j] = (_Float16)fmaf(x[j], (float)y[j], 0.0f);
        if constexpr (PAIR) lo[j] = (_Float16)fmaf(x[j], (float)y[j], -(float)hi[j]);
    }
}
template <bool PAIR>
__device__ __forceinline__ void split8(const float* x, h8& hi, h8& lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        hi[j] = (_Float16)x[j];
        if constexpr (PAIR) lo[j] = (_Float16)(x[j] - (float)hi[j]);
    }
}

__device__ __forceinline__ float lanes16_max(float v) {  // over the four lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float lanes16_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// A tile's operands as they come from memory. Lane (c, g) = (lane % 16, lane / 16) holds, for the
// scores, the rows of positions 8 (c / 4) + 4 t + c % 4 of tile t, and for the values positions
// 8 g .. 8 g + 7.
template <int HD, bool Q4>
struct Tile;
template <int HD>
struct Tile<HD, false> {
    h8 k[2][HD / 32];  // dims 32 s + 8 g ..
    h8 v[HD / 16];     // dim 16 d + c
};
template <int HD>
struct Tile<HD, true> {
    uint32_t k[2][HD / 32], v[HD / 16];
    h8 par;  // piece `lane` of the tile's 64 pieces of scales and minima (see TileParams)
};

// A tile's scales and minima, 16-byte pieces of 8 positions: piece 4 r + i holds positions 8 i ..
// of row r: K's scales of the HD / 32 groups, K's minima, then from piece 32 V's likewise. A lane
// loads one piece; the wave shares them through LDS, where four lanes' addresses serve all 64
// (what each lane needs, loaded by itself, takes 14 loads and 56 registers a tile). `k` holds K's
// once more, the rows of each position side by side.
template <int HD>
struct TileParams {
    static constexpr int kMin = HD / 32, kV = 8;  // first rows
    h8 piece[64];
    h8 k[32];
    __device__ h8 at(int row, int i) const { return piece[4 * row + i]; }
};

// Orders a wave's LDS accesses on both sides: lanes read what others have written. (LDS serves a
// wave in order, so this costs no wait.)
__device__ __forceinline__ void lanes_meet() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
}

// Where a tile's data lie: a pointer for positions tb .. tb + 15 of the head and one for the rest
// (the same page unless pages hold 16), and the lane's offsets, which do not change.
struct Pages {
    const uint8_t *a, *b;
};
template <int HD, bool Q4>
struct LaneOffsets {
    int k, v, par;  // bytes
    bool khigh, high, parhigh, parv;
    __device__ LaneOffsets(const PagedView& pv, int lane) {
        const int c = lane & 15, g = lane >> 4, ps = pv.page_size();
        khigh = c >= 8;
        high = g >= 2;
        const int slot = (8 * (c >> 2) + (c & 3)) & (ps - 1), s8 = (8 * g) & (ps - 1);
        parv = lane >= 32;
        parhigh = (lane & 3) >= 2;
        if constexpr (!Q4) {
            k = 2 * (slot * HD + 8 * g);
            v = 2 * (s8 * HD + c * 8);
            par = 0;
        } else {
            k = 4 * (slot * (HD / 8) + g * (HD / 32));
            v = 4 * ((s8 >> 3) * HD + c * (HD / 16));
            // minima follow the scales; HD 64 has four rows, and lanes that load one twice
            const int row = (lane >> 2 & 7) % (2 * HD / 32);
            par = csdr::scale_offset(HD, ps, row, (8 * (lane & 3)) & (ps - 1));
        }
    }
};

template <int HD, bool Q4>
__device__ __forceinline__ Pages pages_of(const uint8_t* pool, const PagedView& pv, int kvh,
                                          int page0, int page1) {
    return Pages{pool + csdr::head_offset<Q4>(pv, HD, max(page0, 0), kvh),
                 pool + csdr::head_offset<Q4>(pv, HD, max(page1, 0), kvh)};
}

template <int HD, bool Q4>
__device__ __forceinline__ void load_k(Tile<HD, Q4>& t, const PagedView& pv, Pages p, int tb,
                                       const LaneOffsets<HD, Q4>& at) {
    const int ps = pv.page_size();
    const int slot = tb & (ps - 1) & ~15;  // uniform; pages of 16: 0
    if constexpr (!Q4) {
        const uint8_t* hp = (at.khigh ? p.b : p.a) + slot * (HD * 2) + at.k;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int s = 0; s < HD / 32; ++s)
                t.k[u][s] = *reinterpret_cast<const h8*>(hp + 2 * (4 * u * HD + 32 * s));
    } else {
        const uint8_t* hp = (at.khigh ? p.b : p.a) + slot * (HD / 2) + at.k;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            __builtin_memcpy(t.k[u], __builtin_assume_aligned(hp + 4 * u * (HD / 2), HD / 8), HD / 8);
    }
}

template <int HD, bool Q4>
__device__ __forceinline__ void load_v(Tile<HD, Q4>& t, const PagedView& pv, Pages p, int tb,
                                       const LaneOffsets<HD, Q4>& at) {
    const int ps = pv.page_size();
    const int slot = tb & (ps - 1) & ~15;
    const uint8_t* hp = at.high ? p.b : p.a;
    if constexpr (!Q4) {
        hp += slot * (HD * 2) + at.v;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) t.v[d] = *reinterpret_cast<const h8*>(hp + 256 * d);
    } else {
        __builtin_memcpy(t.v, __builtin_assume_aligned(hp + slot * (HD / 2) + at.v, 16), HD / 4);
    }
}

template <int HD>
__device__ __forceinline__ void load_par(Tile<HD, true>& t, const PagedView& pv, Pages k, Pages v,
                                         int tb, const LaneOffsets<HD, true>& at) {
    const int slot = tb & (pv.page_size() - 1) & ~15;
    const uint8_t* a = at.parv ? v.a : k.a;
    const uint8_t* b = at.parv ? v.b : k.b;
    t.par = *reinterpret_cast<const h8*>((at.parhigh ? b : a) + 2 * slot + at.par);
}

// The eight halves of `v` whose bit of `live` is set, zero elsewhere.
__device__ __forceinline__ h8 only(h8 v, uint32_t live) {
    u4 w = __builtin_bit_cast(u4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (live >> (2 * i) & 1) ? 0x0000FFFFu : 0u;
        const uint32_t hi = (live >> (2 * i + 1) & 1) ? 0xFFFF0000u : 0u;
        w[i] &= lo | hi;
    }
    return __builtin_bit_cast(h8, w);
}

// Eight scores with the options, in the log2 domain, of positions `back`, back - 1 .. behind the
// token (ahead of it below 0); `x` the products q.k in units of 1 / unit. (One branch for all eight:
// with one at each score, no two are on their way together.)
__device__ __forceinline__ void shape8(const AttnArgs& a, float* x, float unit, float slope,
                                       int back) {
    if (a.cap > 0.0f) {
        const float to = unit * a.inv_cap, cap = a.cap * kLog2e;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = x[j] * to, b = fabsf(t);
            // tanh: 1 - 2 / (e^2b + 1), absolutely exact to 2^-23, and its series for small b
            const float e = exp2_fast(2.0f * kLog2e * b);
            const float y = fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
            const float t2 = t * t;
            const float p = b * fmaf(t2, fmaf(t2, fmaf(t2, -17.0f / 315, 2.0f / 15), -1.0f / 3), 1.0f);
            x[j] = cap * copysignf(b < 0.2f ? p : y, t);
        }
    } else {
        const float to = unit * kLog2e;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= to;
    }
    if (a.slopes) {
        const float s = -slope * kLog2e, d = (float)back;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(s, fabsf(d - (float)j), x[j]);
    }
}

// A column's query as B operand: dims 32 s + 8 g .. for lane group g. fp32: the row scaled by a
// power of two that puts its largest magnitude in [2^TOP, 2^(TOP + 1)), then in pairs of fp16
// (fp16: as it is unless TOP is given). A negative scale turns the query round. Returns the
// (positive) factor from products to scores, in the log2 domain if there are no options.
template <int HD, typename XT, bool OPTS, int TOP = sizeof(XT) == 4 ? 13 : 0>
__device__ __forceinline__ float load_query(const AttnArgs& a, const XT* qp, int g, h8* qh,
                                            h8* ql) {
    constexpr bool PAIR = sizeof(XT) == 4;
    float unit = fabsf(OPTS ? a.scale : a.scale * kLog2e);
    float x[HD / 32][8], big = 0.0f, f = 1.0f;
#pragma unroll
    for (int s = 0; s < HD / 32; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[s][j] = (float)qp[32 * s + 8 * g + j];
            big = fmaxf(big, fabsf(x[s][j]));
        }
    if constexpr (TOP != 0) {
        big = lanes16_max(big);
        const int e = (int)(__float_as_uint(big) >> 23) - 127;
        const int k = big > 0.0f ? min(max(TOP - e, -120), 120) : 0;
        f = __uint_as_float((uint32_t)(127 + k) << 23);
        unit *= __uint_as_float((uint32_t)(127 - k) << 23);
    }
    f = copysignf(f, a.scale);
#pragma unroll
    for (int s = 0; s < HD / 32; ++s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[s][j] *= f;
        split8<PAIR>(x[s], qh[s], ql[PAIR ? s : 0]);
    }
    return unit;
}

struct Splits {
    bool step;     // step_kernel, else prompt_kernel
    int n;         // of the tiles that a workgroup's columns see
    float* stats;  // 2 per (row, head, split): exponent offset and sum
    float* vecs;   // HD per (row, head, split)
};

// Split attention of up to 16 (token, head) columns of one KV head. One wave runs a softmax with
// a running maximum over tiles of 32 positions, all operands straight from memory in the order
// the matrix cores take them:
//   S^T = K Q^T, two 16x16 tiles of rows = positions; lane (c, g) ends with column c's scores at
//     positions 8 g .. 8 g + 7, which is just what it has to give as B operand of
//   O^T += V^T P^T, whose A operand is a 16-byte piece of V's page.
// So nothing crosses lanes but the maximum, and that only when it moves by more than kLag.
// 4 bits: codes enter the products as whole numbers (16 + code for K; code - 8 for V, centred, so
// that sums do not cancel); K's scale is applied to the group's 32-dim partial score, V's to the
// weights, and what the minima (and the 16) add comes from small products of their own. fp32 calls
// carry q and the weights as pairs of fp16 (22 bits), fp16 calls on fp16 pages the weights; those on
// 4-bit pages round weights, and sum what they rounded (so that constant values come back).
// fp16 pages: bound by their stream (32 sequences, fp16 calls: 81 us, 4.7 TB/s). 4 bits: by vector
// instructions, about 450 beside 39 matrix ones a tile (64 sequences of 4096 to 8192, fp32 calls:
// 137 to 143 us, 3.5 TB/s; one of 131071, fp16 calls: 47 us); with fewer than 16 query heads to a KV
// head and a token each, the columns past them repeat the last one, and that work with them.
template <int HD, bool Q4, typename XT, bool OPTS>
__global__ __launch_bounds__(64 * kStepWaves, 3) void step_kernel(AttnArgs a, Splits sp) {
    constexpr bool PAIR = sizeof(XT) == 4, WPAIR = PAIR || !Q4;  // queries, weights
    constexpr int NS = HD / 32, ND = HD / 16;
    const PagedView& pv = a.pv;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.hq / pv.hkv;
    const int b = blockIdx.x / pv.hkv, kvh = blockIdx.x % pv.hkv, split = blockIdx.y;
    const SeqRows r = csdr::seq_rows(pv, b);
    const int col0 = blockIdx.z * kCols, ncol = min(r.n * G - col0, kCols);
    if (ncol <= 0) return;
    const Seen seen = seen_of(a, b, r);
    const int col = col0 + min(c, ncol - 1);
    const int h = kvh * G + col % G, pq = r.p0 + col / G;
    const long long row = (long long)r.first + col / G;
    const int pq0 = r.p0 + col0 / G, pq1 = r.p0 + (col0 + ncol - 1) / G;
    const float slope = OPTS && a.slopes ? a.slopes[h] : 0.0f;

    const Tiles<kTile> tiles(seen, pq0, pq1);
    const int first = max(0, pq0 - min(pq0 + 1, seen.window) + 1);  // below: only the prefix
    int lo, hi;
    tiles.share(split, sp.n, kStepWaves, lo, hi);

    h8 qh[NS], ql[NS];
    const XT* qp = static_cast<const XT*>(a.q) + row * a.q_stride + (long long)h * HD;
    const float unit = load_query<HD, XT, OPTS, Q4 ? 5 : PAIR ? 13 : 0>(a, qp, g, qh, ql);
    // 4 bits: what the groups' minima and the 16 too many in the codes add to a score, the sum over
    // groups of minimum * qsum - scale * 16 qsum, is a product of its own: row 0 .. of a position's
    // parameters against these (in two halves; |q| below 2^6 keeps 16 qsum in fp16)
    h8 sh, sl;
    if constexpr (Q4) {
        float x[8] = {};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            float t = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) t += PAIR ? (float)qh[s][j] + (float)ql[s][j] : (float)qh[s][j];
            t = lanes16_sum(t);
            x[s] = g == 0 ? -16.0f * t : 0.0f;
            x[NS + s] = g == 0 ? t : 0.0f;
        }
        split8<true>(x, sh, sl);
    }
    __shared__ TileParams<HD> params[Q4 ? kStepWaves : 1];
    TileParams<HD>& tp = params[Q4 ? wave : 0];
    if (Q4 && NS < 4) tp.k[lane & 31] = h8{};  // (its unused half meets zeros)

    f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f4{0.f, 0.f, 0.f, 0.f};
    f4 par = {0.f, 0.f, 0.f, 0.f};  // 4 bits: sums of weights times what code 8 stands for
    f4 lw = {0.f, 0.f, 0.f, 0.f};   // sums of weights rounded once, in par's units, in all rows
    const h8 ones = h8{} + (_Float16)1.0f;
    float m = kNoMax, l = 0.0f;       // the (lagging) maximum, log2 domain; this lane's sum
    // exponent above V's largest scale (from fp16's smallest): weights are 2^-ev of the above
    float ev = Q4 ? -24.0f : 0.0f, vtop = 0x1p-24f;
    uint32_t magic = 0x4C004C00u;
    uint32_t m0 = 0x64006400u, m1 = 0x54005400u;
    asm("" : "+v"(magic), "+v"(m0), "+v"(m1));  // (kept in registers)

    const LaneOffsets<HD, Q4> at(pv, lane);
    Tile<HD, Q4> t;
    // One tile at tb (pages pg0, pg1); with MORE, the loads of the next one (nb, ng0, ng1) are
    // issued as soon as its registers are free. (The last tile, which has no next one, is code of
    // its own.)
    auto tile = [&](auto more, int tb, int pg0, int pg1, int nb, int ng0, int ng1) {
        constexpr bool MORE = decltype(more)::value;
        // the lane's positions that its column sees; whole tiles need no mask
        const int p8 = tb + 8 * g;
        const bool whole = pg0 >= 0 && pg1 >= 0 && pq0 >= 0 && tb + kTile <= seen.keys &&
                           (tb + kTile <= seen.prefix || (tb + kTile - 1 <= pq0 && tb >= first &&
                                                          pq1 - tb < seen.window));
        uint32_t live = 0xFFu, mine = 0xFFu;  // seen by some column; by this one
        uint32_t plive = 0u;                  // the same for the positions of the lane's piece
        if (!whole) {
            live = mine = 0u;
            auto some = [&](int p) {
                return (p < seen.keys) & ((p < seen.prefix) | ((p >= first) & (p <= pq1)));
            };
            if (Q4 && (at.parhigh ? pg1 : pg0) >= 0)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    plive |= (uint32_t)some(tb + 8 * (lane & 3) + j) << j;
            if ((g >= 2 ? pg1 : pg0) >= 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int p = p8 + j;
                    mine |= (uint32_t)((pq >= 0) & seen.at(pq, p)) << j;
                    live |= (uint32_t)some(p) << j;
                }
            }
        }

        float vscale = 0.0f;  // the largest of V's scales that this lane loaded
        if constexpr (Q4) {
            if (!whole && at.parv) t.par = only(t.par, plive);
            lanes_meet();  // (the last tile's reads are done)
            if (at.parv && (lane & 31) < 4 * NS)
#pragma unroll
                for (int j = 0; j < 8; ++j) vscale = fmaxf(vscale, (float)t.par[j]);
            tp.piece[lane] = t.par;
            if (lane < 8 * NS)  // K's row lane / 4 of positions 8 (lane % 4) ..
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    reinterpret_cast<_Float16*>(&tp.k[8 * (lane & 3) + j])[lane >> 2] = t.par[j];
            lanes_meet();
        }

        // scores of positions p8 + j
        float s8[8];
        f4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if constexpr (Q4) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const h8 kp = tp.k[8 * (c >> 2) + 4 * u + (c & 3)];
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kp, sh, acc[u], 0, 0, 0);
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kp, sl, acc[u], 0, 0, 0);
            }
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if constexpr (!Q4) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[u][s], qh[s], acc[u], 0, 0, 0);
                    if constexpr (PAIR)
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[u][s], ql[s], acc[u], 0, 0, 0);
                }
            } else {
                const h8 ks = tp.at(s, g);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const h8 kc = codes16(t.k[u][s], magic);
                    f4 part = {0.f, 0.f, 0.f, 0.f};
                    part = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qh[s], part, 0, 0, 0);
                    if constexpr (PAIR)
                        part = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, ql[s], part, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[u][i] = fmaf((float)ks[4 * u + i], part[i], acc[u][i]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s8[j] = OPTS ? acc[j >> 2][j & 3] : acc[j >> 2][j & 3] * unit;
        if constexpr (OPTS) shape8(a, s8, unit, slope, pq - p8);
        if constexpr (MORE) {
            const Pages kp = pages_of<HD, Q4>(pv.k, pv, kvh, ng0, ng1);
            load_k<HD, Q4>(t, pv, kp, nb, at);
            if constexpr (Q4)
                load_par<HD>(t, pv, kp, pages_of<HD, Q4>(pv.v, pv, kvh, ng0, ng1), nb, at);
        }

        float top = kNoMax;
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(mine >> j & 1)) s8[j] = -INFINITY;
            if constexpr (!Q4) {
#pragma unroll
                for (int d = 0; d < ND; ++d) t.v[d] = only(t.v[d], live);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, s8[j]);
        bool move = top > m + kLag<XT>;
        if constexpr (Q4) {
            move = move || vscale > vtop;
        }
        if (__any(move)) {
            const float mn = fmaxf(m, lanes16_max(top));
            float en = ev;
            if constexpr (Q4) {
                const float big = wave_max(vscale);
                if (big > vtop) {
                    en = (float)((int)(__float_as_uint(big) >> 23) - 126);
                    vtop = __uint_as_float((uint32_t)((int)en + 127) << 23);
                }
            }
            const float f = exp2_fast((m + ev) - (mn + en));
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= f;
            if constexpr (Q4) {
                const float fp = exp2_fast(m - mn);
                par *= fp;
                if constexpr (!WPAIR) lw *= fp;
            }
            m = mn;
            ev = en;
        }
        const float off = kBias<XT> - ev - m;
        float w8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w8[j] = exp2_fast(s8[j] + off);
            if constexpr (WPAIR) l += w8[j];
        }
        if constexpr (!Q4) {
            h8 wh, wl;
            split8<WPAIR>(w8, wh, wl);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.v[d], wh, o[d], 0, 0, 0);
                if constexpr (WPAIR)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.v[d], wl, o[d], 0, 0, 0);
            }
        } else {
            // value = scale (code - 8) + (8 scale + minimum): the second, of group c mod NS, as A
            // operand, in two halves as well; its sum over positions is the same for the group's
            // dims. (Scales and minima summed apart cancel: 7e-6 off in place of 7e-7.) Weights
            // without 2^-ev, which would take them past fp16 where scales are small.
            h8 ch, cl, wh, wl;
            const h8 rs = tp.at(TileParams<HD>::kV + c % NS, g);
            const h8 rm = tp.at(TileParams<HD>::kV + TileParams<HD>::kMin + c % NS, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float ctr = fmaf(8.0f, (float)rs[j], (float)rm[j]);
                ch[j] = (_Float16)ctr;
                cl[j] = (_Float16)(ctr - (float)ch[j]);
            }
            split8<WPAIR>(w8, h8{} + (_Float16)vtop, wh, wl);
            par = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, wh, par, 0, 0, 0);
            par = __builtin_amdgcn_mfma_f32_16x16x32_f16(cl, wh, par, 0, 0, 0);
            if constexpr (WPAIR)
                par = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, wl, par, 0, 0, 0);
            else
                lw = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, wh, lw, 0, 0, 0);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                split8<WPAIR>(w8, tp.at(TileParams<HD>::kV + s, g), wh, wl);
#pragma unroll
                for (int d = 2 * s; d < 2 * s + 2; ++d) {
                    const h8 vc = codes8(t.v[d], m0, m1);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, wh, o[d], 0, 0, 0);
                    if constexpr (WPAIR)
                        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, wl, o[d], 0, 0, 0);
                }
            }
        }
        if constexpr (MORE) load_v<HD, Q4>(t, pv, pages_of<HD, Q4>(pv.v, pv, kvh, ng0, ng1), nb, at);
    };
    int i = lo + wave;
    if (i < hi) {
        auto pages_at = [&](int p, int& x, int& y) {
            x = csdr::page_of(pv, b, p);
            y = pv.shift == 4 ? csdr::page_of(pv, b, p + 16) : x;
        };
        int tb = tiles.at(i), nb = tiles.at(i + kStepWaves);
        int pg0, pg1, ng0, ng1;
        pages_at(tb, pg0, pg1);
        const Pages kp = pages_of<HD, Q4>(pv.k, pv, kvh, pg0, pg1);
        const Pages vp = pages_of<HD, Q4>(pv.v, pv, kvh, pg0, pg1);
        load_k<HD, Q4>(t, pv, kp, tb, at);
        if constexpr (Q4) load_par<HD>(t, pv, kp, vp, tb, at);
        load_v<HD, Q4>(t, pv, vp, tb, at);
        pages_at(nb, ng0, ng1);  // (-1 past the table)
        for (i += kStepWaves; i < hi; i += kStepWaves) {
            // the page ids of the tile after the next are on their way during this one
            const int nn = tiles.at(i + kStepWaves);
            int nng0, nng1;
            pages_at(nn, nng0, nng1);
            tile(std::true_type{}, tb, pg0, pg1, nb, ng0, ng1);
            tb = nb;
            pg0 = ng0;
            pg1 = ng1;
            nb = nn;
            ng0 = nng0;
            ng1 = nng1;
        }
        tile(std::false_type{}, tb, pg0, pg1, 0, 0, 0);
    }

    // join the waves: sums in units of 2^(m + ev)
    __shared__ float stat[kStepWaves][2][kCols];
    __shared__ float vec[kStepWaves][kCols][HD + 4];
    if constexpr (WPAIR) l = lanes16_sum(l);
    else l = lw[0] * (1.0f / vtop);
    float corr[Q4 ? NS : 1];
    if constexpr (Q4) {
        // row 4 g + i of the product is group (4 g + i) mod NS
        const float f = 1.0f / vtop;
#pragma unroll
        for (int s = 0; s < NS; ++s) corr[s] = par[s] * f;
    }
    if (g == 0) {
        stat[wave][0][c] = m + ev;
        stat[wave][1][c] = l;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        if constexpr (Q4) o[d] += corr[d / 2];
        *reinterpret_cast<f4*>(&vec[wave][c][16 * d + 4 * g]) = o[d];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ncol * HD; i += 64 * kStepWaves) {
        const int cc = i / HD, d = i % HD;
        float e = stat[0][0][cc];
#pragma unroll
        for (int w = 1; w < kStepWaves; ++w) e = fmaxf(e, stat[w][0][cc]);
        float sum = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < kStepWaves; ++w) {
            const float f = exp2_fast(stat[w][0][cc] - e);
            den = fmaf(f, stat[w][1][cc], den);
            sum = fmaf(f, vec[w][cc][d], sum);
        }
        const int ci = col0 + cc;
        const size_t part =
            (((size_t)r.first + ci / G) * a.hq + kvh * G + ci % G) * sp.n + split;
        sp.vecs[part * HD + d] = sum;
        if (d == 0) {
            sp.stats[2 * part] = e;
            sp.stats[2 * part + 1] = den;
        }
    }
}

// Joins a row's splits, one workgroup of 1 or 4 waves per (token, head). A row whose sum is not
// positive or whose result is not finite is done again position by position (attend_row): rows
// that see nothing, NaN or infinities that a token sees or that lie in a shared tile unseen.
template <int HD, bool Q4, typename XT>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a, Splits sp) {
    constexpr int VPL = HD / 64;
    const int b = blockIdx.x / a.pv.max_q, tq = blockIdx.x % a.pv.max_q, h = blockIdx.y;
    const SeqRows r = csdr::seq_rows(a.pv, b);
    if (tq >= r.n) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const long long row = (long long)r.first + tq;
    const size_t part = ((size_t)row * a.hq + h) * sp.n;
    const float* st = sp.stats + 2 * part;
    const float* vec = sp.vecs + part * HD + VPL * lane;
    float e = kNoMax;
    for (int i = lane; i < sp.n; i += 64) e = fmaxf(e, st[2 * i]);
    e = wave_max(e);
    float den = 0.0f, num[VPL] = {};
    for (int i0 = wave; i0 < sp.n; i0 += 8 * nw) {
        float x[8][VPL], f[8], ls[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = min(i0 + k * nw, sp.n - 1);
            f[k] = st[2 * i];
            ls[k] = st[2 * i + 1];
#pragma unroll
            for (int v = 0; v < VPL; ++v) x[k][v] = vec[(size_t)i * HD + v];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float w = i0 + k * nw < sp.n ? exp2_fast(f[k] - e) : 0.0f;
            den = fmaf(w, ls[k], den);
#pragma unroll
            for (int v = 0; v < VPL; ++v)
                num[v] = i0 + k * nw < sp.n ? fmaf(w, x[k][v], num[v]) : num[v];
        }
    }
    if (nw > 1) {
        __shared__ float red[4][HD + 1];
#pragma unroll
        for (int v = 0; v < VPL; ++v) red[wave][VPL * lane + v] = num[v];
        if (lane == 0) red[wave][HD] = den;
        __syncthreads();
        if (wave > 0) return;
        den = red[0][HD] + red[1][HD] + red[2][HD] + red[3][HD];
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int i = VPL * lane + v;
            num[v] = red[0][i] + red[1][i] + red[2][i] + red[3][i];
        }
    }
    bool fine = den > 0.0f && den < INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) fine = fine && fabsf(num[v]) < INFINITY;
    if (!__all(fine)) {
        attend_row<HD, Q4, XT>(a, b, r, tq, h);
        return;
    }
    XT* out = static_cast<XT*>(a.out) + (row * a.hq + h) * HD + VPL * lane;
#pragma unroll
    for (int v = 0; v < VPL; ++v) out[v] = (XT)(num[v] / den);
}

// ---------------------------------------------------------------- prompts: tiles shared in LDS

typedef const __attribute__((address_space(1))) void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

// Attention of many columns, the (token, query head) pairs of one sequence and KV head: a workgroup
// of NW waves takes 16 NQ NW of them, a wave NQ tiles of 16 (column tiles are dealt to the waves in
// turn, so that under a causal mask all see about as many positions). Tiles of TP positions of K
// and V lie in LDS twice, the next one being brought in while the current one is worked on; a wave
// reads each operand once for its NQ column tiles. The products, the running maximum and what a
// lane holds are step_kernel's, all NQ column tiles beside each other.
//
// fp16 pages go straight to LDS (16 bytes a lane); K's 16-byte chunks of a row are permuted within
// the row on the way (chunk j of row r at j ^ key(r)), so that the 16 rows of an operand read fall
// on distinct banks; V's pieces lie in operand order already. 4-bit pages are turned into fp16
// values by the threads, in two planes: value = hi + lo to 22 bits, and products hi hi, lo hi and
// for fp32 calls hi lo. (One plane, values rounded to 11 bits, would do with half the products for
// fp16 calls, but left them 2.2 times as far off as the rounding of their outputs alone.)
// Bound by matrix and vector instructions in turn: 4096 tokens on fp16 pages, fp16 calls, 159 to
// 168 us from card to card, 820 to 865 TFLOP/s (fp32 calls 269); prompts on 4-bit pages, fp32 calls,
// 598 us, 263 TFLOP/s, three products for each (fp16 calls 461, two).
template <int HD, bool Q4, typename XT, int NQ, int NW>
struct PromptShape {
    static constexpr bool kPair = sizeof(XT) == 4;
    static constexpr int kPlanes = Q4 ? 2 : 1;
    // positions per tile, and waves per SIMD: LDS for two workgroups of four waves or one of eight
    // on a CU; three of four where 168 registers do (4096 tokens of fp16, HD 128: tiles of 64 and
    // two waves 171 us, of 32 and three 164)
    static constexpr bool kLean = !Q4 && !kPair && HD == 128;
    static constexpr int kSimdWaves = kLean ? 3 : 2;
    static constexpr int TP = (kPlanes == 2 && HD == 128 && NW == 4) || kLean ? 32 : 64;
    static constexpr int kPlane = TP * HD;                          // halves
    static constexpr int kLds = 2 * 2 * kPlanes * kPlane * 2;       // bytes
    static constexpr int kColumns = NW * 16 * NQ;
};

// Where the LDS row of position r of a tile keeps chunk j.
template <int HD>
__device__ __forceinline__ int chunk_key(int r) {
    return HD == 128 ? 4 * ((r >> 3) & 3) + (r & 3) : 2 * ((r >> 3) & 3) + ((r >> 1) & 1);
}

template <int HD, bool Q4, typename XT, bool OPTS, int NQ, int NW>
__global__ __launch_bounds__(64 * NW, (PromptShape<HD, Q4, XT, NQ, NW>::kSimdWaves)) void
prompt_kernel(AttnArgs a, Splits sp) {
    using Shape = PromptShape<HD, Q4, XT, NQ, NW>;
    constexpr bool PAIR = Shape::kPair;
    constexpr int NS = HD / 32, ND = HD / 16, TP = Shape::TP, PLANES = Shape::kPlanes;
    constexpr int PLANE = Shape::kPlane, GR = TP / 16;
    extern __shared__ __attribute__((aligned(16))) _Float16 lds[];  // [2][K, V][planes][TP * HD]
    const PagedView& pv = a.pv;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.hq / pv.hkv;
    // (sequence, KV head) fastest: on a chip of 8 dies that take workgroups in turn, the blocks of
    // one KV head meet in one L2 where there are 8 (or a multiple) of them. Latest columns, which
    // see most, first; where a CU takes two workgroups, the second 256 in the opposite order, so
    // that a CU with the longest of the first has the shortest of the second (14 heads of 64, two
    // prompts of 4096 tokens: 111 -> 106 us, one of 8192: 215 -> 203). Where it takes three, that
    // gains nothing (32 heads of 128, 4096 tokens: 167 and 168, 8192: 567 and 572).
    const int pairs = pv.n_seqs * pv.hkv, blocks = gridDim.x / pairs;
    const int bh = blockIdx.x % pairs, around = max(1, 256 / pairs);
    int rank = blockIdx.x / pairs;
    if (NW == 4 && Shape::kSimdWaves == 2 && rank >= around && rank < min(2 * around, blocks))
        rank = around + min(2 * around, blocks) - 1 - rank;
    const int block = blocks - 1 - rank;
    const int b = bh / pv.hkv, kvh = bh % pv.hkv, split = blockIdx.y;
    const SeqRows r = csdr::seq_rows(pv, b);
    const int ncols = r.n * G, col0 = block * Shape::kColumns;
    if (col0 >= ncols) return;
    const Seen seen = seen_of(a, b, r);
    const int ps = pv.page_size();
    auto pos_of = [&](int col) { return r.p0 + col / G; };
    const int last_col = min(ncols, col0 + Shape::kColumns) - 1;
    const int pq0 = pos_of(col0), pq1 = pos_of(last_col);  // of the workgroup

    const Tiles<TP> tiles(seen, pq0, pq1);
    const int first = max(0, pq0 - min(pq0 + 1, seen.window) + 1);  // below: only the prefix
    int lo, hi;
    tiles.share(split, sp.n, 256 / TP, lo, hi);

    // the columns of this lane: tile q holds columns col0 + 16 (NW q + wave) + c
    h8 qh[NQ][NS], ql[PAIR ? NQ : 1][NS];
    float unit[NQ], slope[NQ];
    int pq[NQ];
    int wp0 = 0x7fffffff, wp1 = -0x7fffffff;  // first and last position of the wave's columns
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int t0 = col0 + 16 * (NW * q + wave);
        const int col = min(t0 + c, ncols - 1);
        if (t0 < ncols) {
            wp0 = min(wp0, pos_of(t0));
            wp1 = max(wp1, pos_of(min(t0 + 15, ncols - 1)));
        }
        const int h = kvh * G + col % G;
        pq[q] = pos_of(col);
        slope[q] = OPTS && a.slopes ? a.slopes[h] : 0.0f;
        const XT* qp = static_cast<const XT*>(a.q) + ((long long)r.first + col / G) * a.q_stride +
                       (long long)h * HD;
        unit[q] = load_query<HD, XT, OPTS>(a, qp, g, qh[q], ql[PAIR ? q : 0]);
    }

    f4 o[NQ][ND], l[NQ];  // l: the sum of the weights, in all four rows (a product with ones)
    float m[NQ];
    const h8 ones = h8{} + (_Float16)1.0f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        m[q] = kNoMax;
        l[q] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < ND; ++d) o[q][d] = f4{0.f, 0.f, 0.f, 0.f};
    }

    auto buffer = [&](int buf, int v, int plane) {
        return lds + ((buf * 2 + v) * PLANES + plane) * PLANE;
    };
    // page ids of a tile's granules of 16 positions (uniform; through the scalar cache 164 -> 157
    // us for 4096 tokens on fp16 pages, but 600 -> 644 where 4-bit pages are unpacked between)
    auto pages_at = [&](int tb, int* pg) {
#pragma unroll
        for (int i = 0; i < GR; ++i)
            pg[i] = i > 0 && ps >= TP ? pg[0] : csdr::page_of<!Q4>(pv, b, tb + 16 * i);
    };

    // 4 bits: the words this thread turns into values, and their groups' scales and minima
    constexpr int W = TP * HD / 8 / (64 * NW);  // words per thread: 2 or 4
    struct Codes {
        uint32_t k[W], v[W];
        _Float16 ks[W], km[W];
        h8 vs[W / 2], vm[W / 2];
    };
    Codes cd;

    // brings the tile at tb into buffer `buf` (fp16 pages) or its codes into registers
    auto fetch = [&](int tb, int buf, const int* pg) {
        if constexpr (!Q4) {
            constexpr int N = PLANE * 2 / 1024 / NW;  // 1 KB pieces per wave, for K and for V
            constexpr int R = 512 / HD;               // K: rows a piece
            // the lane's chunk of a piece of K (a key depends on the piece only by R = 4)
            const int in = lane / (HD / 8), ch = lane % (HD / 8);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int piece = NW * i + wave, row = piece * R;
                const int page = max(pg[row / 16], 0);
                const size_t head = csdr::head_offset<Q4>(pv, HD, page, kvh);
                const int slot = (tb + row) & (ps - 1);
                __builtin_amdgcn_global_load_lds(
                    (GlobalPtr)(pv.k + head + slot * (HD * 2) +
                                (in * (HD * 2) + (ch ^ chunk_key<HD>(row + in)) * 16)),
                    (LdsPtr)(buffer(buf, 0, 0) + piece * 512), 16, 0, 0);
                // V: [8 positions][dim][8]: the same piece of memory, R of 8 rows of a block
                __builtin_amdgcn_global_load_lds((GlobalPtr)(pv.v + head + slot * (HD * 2) + lane * 16),
                                                 (LdsPtr)(buffer(buf, 1, 0) + piece * 512), 16, 0, 0);
            }
        } else {
            // K: words [slot][dim % 32 / 8][dim / 32]; V: words [slot / 8][dim % 16][dim / 16]
            const int w0 = tid * W;
            const int kr = w0 / (HD / 8), vr = w0 / HD * 8;
            int kpage = max(pg[0], 0), vpage = kpage;
#pragma unroll
            for (int i = 1; i < GR; ++i) {
                kpage = kr / 16 == i ? max(pg[i], 0) : kpage;
                vpage = vr / 16 == i ? max(pg[i], 0) : vpage;
            }
            const uint8_t* kb = pv.k + csdr::head_offset<Q4>(pv, HD, kpage, kvh);
            const uint8_t* vb = pv.v + csdr::head_offset<Q4>(pv, HD, vpage, kvh);
            const int ks = (tb + kr) & (ps - 1), vs = (tb + vr) & (ps - 1);
            __builtin_memcpy(cd.k, __builtin_assume_aligned(
                                       kb + 4 * (ks * (HD / 8) + w0 % (HD / 8)), 4 * W), 4 * W);
            __builtin_memcpy(cd.v, __builtin_assume_aligned(
                                       vb + 4 * ((vs >> 3) * HD + w0 % HD), 4 * W), 4 * W);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int grp = (w0 + i) % NS;
                cd.ks[i] = *reinterpret_cast<const _Float16*>(kb + csdr::scale_offset(HD, ps, grp, ks));
                cd.km[i] = *reinterpret_cast<const _Float16*>(kb + csdr::min_offset(HD, ps, grp, ks));
            }
#pragma unroll
            for (int i = 0; i < W / 2; ++i) {
                const int grp = (w0 % ND) / 2 + i;
                cd.vs[i] = *reinterpret_cast<const h8*>(vb + csdr::scale_offset(HD, ps, grp, vs));
                cd.vm[i] = *reinterpret_cast<const h8*>(vb + csdr::min_offset(HD, ps, grp, vs));
            }
        }
    };
    // 4 bits: this thread's words as values into buffer `buf`
    uint32_t magic = 0x4C004C00u;
    asm("" : "+v"(magic));
    auto put = [&](_Float16* at, uint32_t w, auto scale, auto low) {
        const h8 code = codes16(w, magic) - (_Float16)16.0f;
        h8 hi8, lo8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = fmaf((float)scale(e), (float)code[e], (float)low(e));
            hi8[e] = (_Float16)x;
            if constexpr (PLANES == 2) lo8[e] = (_Float16)(x - (float)hi8[e]);
        }
        *reinterpret_cast<h8*>(at) = hi8;
        if constexpr (PLANES == 2) *reinterpret_cast<h8*>(at + PLANE) = lo8;
    };
    auto unpack = [&](int buf) {
        const int w0 = tid * W, kr = w0 / (HD / 8);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int kw = w0 % (HD / 8) + i, ch = kw % NS * 4 + kw / NS;  // dims 8 ch ..
            put(buffer(buf, 0, 0) + kr * HD + (ch ^ chunk_key<HD>(kr)) * 8, cd.k[i],
                [&](int) { return cd.ks[i]; }, [&](int) { return cd.km[i]; });
            const int vw = w0 % HD + i, d = vw % ND * 16 + vw / ND;
            put(buffer(buf, 1, 0) + (w0 / HD * HD + d) * 8, cd.v[i],
                [&](int e) { return cd.vs[i / 2][e]; }, [&](int e) { return cd.vm[i / 2][e]; });
        }
    };
    // zeros for V at positions of the tile that hold nothing (their weights are zero)
    auto clear = [&](int tb, int buf, const int* pg) {
        for (int i = tid; i < TP * HD; i += 64 * NW) {
            const int pos = i / (8 * HD) * 8 + i % 8;
            int page = pg[0];
#pragma unroll
            for (int k = 1; k < GR; ++k) page = pos / 16 == k ? pg[k] : page;
            if (page >= 0 && tb + pos < seen.keys) continue;
#pragma unroll
            for (int k = 0; k < PLANES; ++k) buffer(buf, 1, k)[i] = (_Float16)0.0f;
        }
    };

    int buf = 0;
    int pg[GR] = {};
    if (lo < hi) {
        pages_at(tiles.at(lo), pg);
        fetch(tiles.at(lo), 0, pg);
        if constexpr (Q4) unpack(0);
    }
    for (int i = lo; i < hi; ++i) {
        const int tb = tiles.at(i);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (this wave's pieces are in LDS)
        __syncthreads();  // the tile is whole, and everyone is done with the other buffer
        bool held = tb + TP <= seen.keys;
        uint32_t have = 0u;  // granules with a page
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            held = held && pg[i] >= 0;
            have |= (uint32_t)(pg[i] >= 0) << i;
        }
        if (!held) {
            clear(tb, buf, pg);
            __syncthreads();
        }
        if (Q4 || i + 1 < hi) {  // (4 bits: the last tile again, which nobody reads)
            const int nb = tiles.at(min(i + 1, hi - 1));
            pages_at(nb, pg);
            fetch(nb, buf ^ 1, pg);
        }
        const bool any = wp0 <= wp1 && ((tb <= wp1 && tb + TP > first) || tb < seen.prefix);
        const bool whole = held && wp0 >= 0 &&
                           (tb + TP <= seen.prefix ||
                            (tb + TP - 1 <= wp0 && tb >= 0 && wp1 - tb < seen.window));
        if (any) {
#pragma unroll
            for (int hb = 0; hb < TP / 32; ++hb) {
                const _Float16* kt = buffer(buf, 0, 0) + (32 * hb + 8 * (c >> 2) + (c & 3)) * HD;
                const _Float16* vt = buffer(buf, 1, 0) + (4 * hb + g) * (8 * HD) + c * 8;
                const int key = chunk_key<HD>(8 * (c >> 2) + (c & 3));
                f4 acc[NQ][2];
#pragma unroll
                for (int q = 0; q < NQ; ++q) acc[q][0] = acc[q][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const _Float16* kp = kt + 4 * u * HD + ((4 * s + g) ^ key) * 8;
                        const h8 k0 = *reinterpret_cast<const h8*>(kp);
#pragma unroll
                        for (int q = 0; q < NQ; ++q) {
                            acc[q][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[q][s],
                                                                               acc[q][u], 0, 0, 0);
                            if constexpr (PAIR)
                                acc[q][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    k0, ql[q][s], acc[q][u], 0, 0, 0);
                        }
                        if constexpr (PLANES == 2) {
                            const h8 k1 = *reinterpret_cast<const h8*>(kp + PLANE);
#pragma unroll
                            for (int q = 0; q < NQ; ++q)
                                acc[q][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    k1, qh[q][s], acc[q][u], 0, 0, 0);
                        }
                    }
                const int p8 = tb + 32 * hb + 8 * g;
                h8 wh[NQ], wl[PAIR ? NQ : 1];
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    // scores, without options still in the products' units
                    float x[8], top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = acc[q][j >> 2][j & 3];
                    if constexpr (OPTS) shape8(a, x, unit[q], slope[q], pq[q] - p8);
                    if (!whole) {
                        const bool row = (have >> ((32 * hb + 8 * g) / 16) & 1) & (pq[q] >= 0);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (!(row & seen.at(pq[q], p8 + j))) x[j] = -INFINITY;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
                    if constexpr (!OPTS) top *= unit[q];
                    if (__any(top > m[q] + kLag<XT>)) {
                        const float mn = fmaxf(m[q], lanes16_max(top));
                        const float f = exp2_fast(m[q] - mn);
                        l[q] *= f;
#pragma unroll
                        for (int d = 0; d < ND; ++d) o[q][d] *= f;
                        m[q] = mn;
                    }
                    const float off = kBias<XT> - m[q];
                    float w8[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w8[j] = exp2_fast(OPTS ? x[j] + off : fmaf(x[j], unit[q], off));
                    split8<PAIR>(w8, wh[q], wl[PAIR ? q : 0]);
                    l[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, wh[q], l[q], 0, 0, 0);
                    if constexpr (PAIR)
                        l[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, wl[q], l[q], 0, 0, 0);
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const h8 v0 = *reinterpret_cast<const h8*>(vt + d * 128);
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        o[q][d] =
                            __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, wh[q], o[q][d], 0, 0, 0);
                        if constexpr (PAIR)
                            o[q][d] =
                                __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, wl[q], o[q][d], 0, 0, 0);
                    }
                    if constexpr (PLANES == 2) {
                        const h8 v1 = *reinterpret_cast<const h8*>(vt + d * 128 + PLANE);
#pragma unroll
                        for (int q = 0; q < NQ; ++q)
                            o[q][d] =
                                __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, wh[q], o[q][d], 0, 0, 0);
                    }
                }
            }
        }
        if constexpr (Q4) unpack(buf ^ 1);
        buf ^= 1;
    }

#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int t0 = col0 + 16 * (NW * q + wave), col = t0 + c;
        const float sum = l[q][0];
        const long long row = (long long)r.first + col / G;
        const int h = kvh * G + col % G;
        if (sp.n > 1) {
            if (col < ncols) {
                const size_t part = ((size_t)row * a.hq + h) * sp.n + split;
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    *reinterpret_cast<f4*>(sp.vecs + part * HD + 16 * d + 4 * g) = o[q][d];
                if (g == 0) {
                    sp.stats[2 * part] = m[q];
                    sp.stats[2 * part + 1] = sum;
                }
            }
            continue;
        }
        bool fine = sum > 0.0f && sum < INFINITY;
        const float inv = 1.0f / sum;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            o[q][d] *= inv;
#pragma unroll
            for (int i = 0; i < 4; ++i) fine = fine && fabsf(o[q][d][i]) < INFINITY;
        }
        XT* out = static_cast<XT*>(a.out) + (row * a.hq + h) * HD + 4 * g;
        if (col < ncols)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) out[16 * d + i] = (XT)o[q][d][i];
        // rows that see nothing, or something that is not finite (perhaps unseen): once more
        uint64_t redo = __ballot(!fine && col < ncols);
        redo |= redo >> 32;
        redo = (redo | redo >> 16) & 0xFFFFu;
        while (redo) {
            const int k = __builtin_ctzll(redo);
            redo &= redo - 1;
            const int col1 = t0 + k;
            attend_row<HD, Q4, XT>(a, b, r, col1 / G, kvh * G + col1 % G);
        }
    }
}

// Whether step_kernel takes the columns of a KV head, 16 at a time, or prompt_kernel all. A second
// block of 16 reads the pages once more, which on fp16 pages pays while that is little: up to 128 MB
// in all (17 to 64 columns, step and prompt: 20 MB 13.6 and 12.9 us, 39 MB 15.3 and 19.9, 14.9 and
// 18.5, 79 MB 20.4 and 21.6, 118 MB 21.6 both, 17.6 and 21.1, 157 MB 27.3 and 24.3, 21.5 and 23.1,
// 1.26 GB 279 and 104). On 4-bit pages, which prompt_kernel unpacks for 128 columns at once or
// more, it pays up to 64 columns (32: 18.5 and 39.3, 57 and 100; 64: 24 and 39, 92.6 and 108; but
// short sequences that are many, 16 of 300 positions: 49 and 29), and from 1024 positions on up to
// 128 (80: 25.8 and 41.0, 86 and 182; 128: 31 and 41, 144 and 183, 170 and 155; 300 positions 13 and
// 25, or 85 and 54).
bool takes_step(const PagedView& pv, bool q4, int hd, long long cols, long long len) {
    if (cols <= kCols) return true;
    if (q4)  // (the last: more would be too many for its join)
        return cols <= 64 ||
               (cols <= 128 && len > 1024 && (long long)pv.n_seqs * pv.max_q < 1LL << 24);
    const double blocks = (double)pv.n_seqs * pv.hkv * (double)((cols + kCols - 1) / kCols);
    return cols <= 64 && blocks * (double)len * (4 * hd) <= 128e6;
}

constexpr long long kPromptBlocks = 512;  // two workgroups to a CU
constexpr int kSmallColumns = 64;         // of the smallest workgroup of prompt_kernel

// Splits of the positions: for step_kernel 768 workgroups in all (the three that a CU holds at
// once), or 1536, which even out sequences of different lengths, where there is work enough for
// their joins: 2^21 positions of a head and 16 columns on 4-bit pages, 2^20 on fp16 ones (heads of
// 128, 768 and 1536 workgroups: 4-bit pages, 2^20 positions 26.9 and 30.4, 38.1 and 39.6 us, 2^21
// 66.5 and 61.5, 71.1 and 64.3, 64.9 and 62.8; fp16 pages, 2^18 positions 23.8 and 24.1, 15.4 and
// 16.6, 2^20 79.6 and 78.5, 87.9 and 90.2, 2^21 154.8 and 156.5, 155.7 and 154.2),
// 128 positions (a tile per wave) each at least; for prompt_kernel one if there are 512 workgroups,
// else enough for that, 512 positions at least. A sequence's positions are shared out equally, so a
// call with sequences of different lengths, or of lengths far below the bound, stays balanced. A
// window, or a smaller bound, only ever makes fewer splits; beside a prefix, whose length is device memory, no fewer than 4096
// positions have (one sequence, a window of 256 and a prefix of 32000: 80 -> 26 us, 128 tokens of
// one: 259 -> 122; a window of 1024 and a prefix of 4: 14 us either way, but for all of the length's
// splits 0 to 2 us more).
constexpr long long kPrefixSeen = 4096;

Splits splits_of(const PagedView& pv, bool q4, int hq, bool step, long long len, int window,
                 bool prefix) {
    const int G = hq / pv.hkv;
    const long long cols = (long long)pv.max_q * G;
    const long long per = step ? kCols : kSmallColumns, unit = step ? kTile * kStepWaves : 512;
    const long long wgs = (long long)pv.n_seqs * pv.hkv * ((cols + per - 1) / per);
    const long long target =
        !step ? kPromptBlocks : (double)wgs * (double)len < (q4 ? 0x1p21 : 0x1p20) ? 768 : 1536;
    // (a block's columns see a window each, and two tiles more where these do not fall on tiles)
    long long seen = window > 0 ? std::min(len, window + std::min(cols, per) / G + 2 * 64) : len;
    if (prefix) seen = std::max(seen, std::min(len, kPrefixSeen));
    Splits s{};
    s.step = step;
    s.n = (int)std::max(1LL, std::min((seen + unit - 1) / unit,
                                      step ? (target + wgs - 1) / wgs : target / wgs));
    return s;
}

long long bound_of(const PagedView& pv, int max_len) {
    return std::max(1, max_len > 0 ? std::min(max_len, pv.capacity()) : pv.capacity());
}

// A call of prompt_kernel without splits needs none.
bool one_launch(const Splits& s) { return !s.step && s.n == 1; }

size_t workspace_of(const PagedView& pv, int hq, int hd, const Splits& s) {
    if (one_launch(s)) return 0;
    const size_t parts = (size_t)pv.n_tokens * hq * s.n;
    return csdr::align_up(parts * 8, 16) + parts * hd * 4;
}

// Column tiles per wave of prompt_kernel: as many as 256 registers hold (sums, queries, weights),
// or one where that would leave the chip without two workgroups a CU (SMALL). Waves per workgroup:
// eight where 4-bit rows of 128 are unpacked, which then serves twice the columns.
template <int HD, bool Q4, typename XT, bool SMALL>
struct PromptConfig {
    static constexpr int NQ =
        SMALL ? 1 : HD == 128 ? 2 : sizeof(XT) == 4 || Q4 ? 3 : 4;
    static constexpr int NW = !SMALL && Q4 && HD == 128 ? 8 : 4;
    using Shape = PromptShape<HD, Q4, XT, NQ, NW>;
};

template <int HD, bool Q4, typename XT, bool OPTS, bool SMALL>
void launch_prompt(const AttnArgs& a, const Splits& s, hipStream_t st) {
    using Config = PromptConfig<HD, Q4, XT, SMALL>;
    using Shape = typename Config::Shape;
    constexpr auto kernel = &prompt_kernel<HD, Q4, XT, OPTS, Config::NQ, Config::NW>;
    if constexpr (Shape::kLds > 65536) {  // beyond the default: allowed once per device
        static std::atomic<uint64_t> allowed{0};
        int dev = 0;
        (void)hipGetDevice(&dev);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (!(allowed.load(std::memory_order_relaxed) & bit)) {
            (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, Shape::kLds);
            allowed.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const int cols = a.pv.max_q * (a.hq / a.pv.hkv);
    const int blocks = (cols + Shape::kColumns - 1) / Shape::kColumns;
    const dim3 grid((unsigned)(a.pv.n_seqs * a.pv.hkv * blocks), s.n);
    kernel<<<grid, 64 * Config::NW, Shape::kLds, st>>>(a, s);
}

template <int HD, bool Q4, typename XT, bool OPTS>
void launch_kernel(const AttnArgs& a, const Splits& s, hipStream_t st) {
    const int cols = a.pv.max_q * (a.hq / a.pv.hkv);
    if (!s.step) {
        const long long columns = PromptConfig<HD, Q4, XT, false>::Shape::kColumns;
        if ((long long)a.pv.n_seqs * a.pv.hkv * cols < kPromptBlocks * columns)
            launch_prompt<HD, Q4, XT, OPTS, true>(a, s, st);
        else
            launch_prompt<HD, Q4, XT, OPTS, false>(a, s, st);
        if (s.n == 1) return;
    } else {
        const dim3 grid(a.pv.n_seqs * a.pv.hkv, s.n, (cols + kCols - 1) / kCols);
        step_kernel<HD, Q4, XT, OPTS><<<grid, 64 * kStepWaves, 0, st>>>(a, s);
    }
    join_kernel<HD, Q4, XT>
        <<<dim3(a.pv.n_seqs * a.pv.max_q, a.hq), s.n > 8 ? 256 : 64, 0, st>>>(a, s);
}

template <int HD, bool Q4, typename XT>
void launch_step(const AttnArgs& a, const Splits& s, hipStream_t st) {
    if (a.cap > 0.0f || a.slopes) launch_kernel<HD, Q4, XT, true>(a, s, st);
    else launch_kernel<HD, Q4, XT, false>(a, s, st);
}

template <int HD, bool Q4>
void launch(const AttnArgs& a, int dtype, const Splits& s, hipStream_t st) {
    if (dtype == CSDR_F32) launch_step<HD, Q4, float>(a, s, st);
    else launch_step<HD, Q4, _Float16>(a, s, st);
}

}  // namespace

extern "C" {

CSDR_API size_t csdr_paged_attn_workspace_bytes(const csdr_paged_kv* kv, int n_tokens,
                                                const int32_t* q_start, int max_q, int Hq,
                                                int max_len) {
    PagedView pv;
    if (csdr::paged_check("paged_attn", kv, n_tokens, q_start, max_q, &pv) != CSDR_OK || Hq <= 0 ||
        Hq > 65535 || Hq % kv->n_kv_heads || max_len < 0)
        return 0;
    // (a smaller bound, which may choose the other kernel, needs no more)
    const bool q4 = kv->kv_dtype == CSDR_Q4;
    const long long cols = (long long)pv.max_q * (Hq / kv->n_kv_heads), len = bound_of(pv, max_len);
    size_t need = 0;
    if (takes_step(pv, q4, kv->head_dim, cols, 1) || takes_step(pv, q4, kv->head_dim, cols, len))
        need = workspace_of(pv, Hq, kv->head_dim, splits_of(pv, q4, Hq, true, len, 0, false));
    if (!takes_step(pv, q4, kv->head_dim, cols, 1) || !takes_step(pv, q4, kv->head_dim, cols, len))
        need = std::max(need, workspace_of(pv, Hq, kv->head_dim,
                                           splits_of(pv, q4, Hq, false, len, 0, false)));
    return need;
}

CSDR_API int csdr_paged_attn(const csdr_paged_kv* kv, const void* q, int dtype, int n_tokens,
                             const int32_t* q_start, int max_q, int Hq, int64_t q_stride,
                             int max_len, float scale, const csdr_attn_options* options, void* out,
                             void* workspace, size_t workspace_bytes, void* hip_stream) {
    AttnArgs a{};
    if (int rc = csdr::paged_check("paged_attn", kv, n_tokens, q_start, max_q, &a.pv)) return rc;
    if (!q || !out) return set_error(CSDR_E_INVALID, "paged_attn: a pointer is NULL");
    if (q == out)  // (rows with values that are not finite are read again)
        return set_error(CSDR_E_INVALID, "paged_attn: out must not be q");
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
        // (a denormal cap has no finite reciprocal)
        if (!(options->softcap == 0.0f ||
              (options->softcap >= FLT_MIN && options->softcap < INFINITY)) ||
            options->window < 0)
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
    const bool q4 = kv->kv_dtype == CSDR_Q4;
    const long long len = bound_of(a.pv, max_len);
    const long long cols = (long long)a.pv.max_q * (Hq / kv->n_kv_heads);
    Splits s = splits_of(a.pv, q4, Hq, takes_step(a.pv, q4, hd, cols, len), len, a.window,
                         a.prefix != nullptr);
    // fewer than 2^32 threads a launch: workgroups of at most 256 (prompt_kernel: two threads a
    // column, except where it has few), join_kernel's where there may be one
    if ((long long)kv->n_seqs * kv->n_kv_heads * ((cols + 127) / 128) >= 1LL << 24 ||
        ((!one_launch(s) || cols <= 64) && (long long)kv->n_seqs * a.pv.max_q >= 1LL << 24))
        return set_error(CSDR_E_INVALID, "paged_attn: too many tokens");
    const size_t need = workspace_of(a.pv, Hq, hd, s);
    if (need && (!workspace || workspace_bytes < need ||
                 reinterpret_cast<uintptr_t>(workspace) % 16))
        return set_error(CSDR_E_WORKSPACE, "paged_attn: workspace missing, too small or unaligned");
    s.stats = static_cast<float*>(workspace);
    s.vecs = s.stats + csdr::align_up((size_t)n_tokens * Hq * s.n * 2, 4);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (hd == 64) {
        if (q4) launch<64, true>(a, dtype, s, st);
        else launch<64, false>(a, dtype, s, st);
    } else {
        if (q4) launch<128, true>(a, dtype, s, st);
        else launch<128, false>(a, dtype, s, st);
    }
    CSDR_LAUNCH_CHECK("paged_attn");
    return CSDR_OK;
}

}  // extern "C"
