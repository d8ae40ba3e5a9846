// rotary.hip — rotary positions for the forms that the cache's own rotation (csdr_paged_append,
// csdr_rope_kv_rows) has not: halves as well as adjacent pairs, the first dims of a head, any frequencies and a
// magnitude (gfx950).
//   (u, v) -> magnitude (u c - v s, u s + v c),  c + i s = exp(i position frequency_j) for pair j
//
// The angle is held in turns in fp64 (an fp32 angle is off by 4e-3 rad at position 65536), its whole turns
// dropped before the fp32 sine and cosine of what is left, at most half a turn. They are computed once per
// token and pair and shared by the heads of a workgroup through LDS. A thread takes 8 pairs, 32 or 64 bytes in
// and out. Bound by memory: 8192 tokens of 32 + 32 heads of 128 in fp16 take 45 us, 5.9 TB/s; a step's tokens
// one round trip (64 of 32 + 8 heads 3.3 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "common.hpp"

namespace {

using csdr::set_error;

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;
constexpr int kUnit = 8;  // pairs of a thread where rows of 8 values are whole

template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[N];
};

struct Side {
    const void* in;
    void* out;
    long long in_stride, out_stride;  // elements between tokens
    int heads;
};

struct Args {
    Side q, k;
    const int32_t* positions;
    const double* turns;  // frequencies / 2 pi, of pair j
    int n_tokens, hd, dims, groups, tokens;  // workgroups of a token, or tokens of a workgroup
    float magnitude;
};

// A workgroup per token and group of heads, or several tokens of few heads. WIDE: 8 pairs a thread; else one. A
// thread's first items are on their way while the sines and cosines are formed (8192 tokens of 64 heads 57 -> 45 us).
template <typename T, bool HALVES, bool WIDE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Args a) {
    __shared__ float2 cs[kMaxDim / 2];
    const int first = (int)(blockIdx.x / a.groups) * a.tokens, group = blockIdx.x % a.groups;
    const int half = a.dims / 2, tokens = min(a.tokens, a.n_tokens - first);
    // items of a head: its pairs, then its other dims (the last one alone where they are odd)
    constexpr int P = WIDE ? kUnit : 1, O = 2 * P, AHEAD = 2;
    const int turned = half / P, items = turned + (a.hd - a.dims) / O + (WIDE ? 0 : (a.hd - a.dims) % O);
    const int each = (a.q.heads + a.k.heads) * items, all = tokens * each, step = a.groups * kThreads;

    // what item i is: where its two pieces lie, and which sines are its pairs' (-1: none, as they are)
    struct Item {
        const T* in;
        T* out;
        int second, pair;
        bool one, none;
    };
    auto item_of = [&](int i) {
        const int local = tokens > 1 ? i / each : 0, head = (i - local * each) / items, item = i % items;
        const int token = first + local;
        const bool is_k = head >= a.q.heads;
        const Side& s = is_k ? a.k : a.q;
        const long long h = (long long)(is_k ? head - a.q.heads : head) * a.hd;
        const bool pairs = item < turned;
        const int at = pairs ? (HALVES ? item * P : item * O) : a.dims + (item - turned) * O;
        Item t;
        t.in = static_cast<const T*>(s.in) + token * s.in_stride + h + at;
        t.out = static_cast<T*>(s.out) + token * s.out_stride + h + at;
        t.second = HALVES && pairs ? half : P;
        t.pair = pairs ? local * half + item * P : -1;
        t.none = a.positions[token] < 0;  // no token
        t.one = !WIDE && at + 1 == a.hd;
        return t;
    };
    using V = Vec<T, P>;
    auto load = [&](const Item& t, V& u, V& v) {
        u = *reinterpret_cast<const V*>(t.in);
        v = *reinterpret_cast<const V*>(t.in + (t.one ? 0 : t.second));
    };
    auto put = [&](const Item& t, const V& u, const V& v) {
        if (t.none) return;
        V p = u, w = v;
        if (t.pair >= 0) {
            float x[O];  // (u, v) of the pairs, one after the other
#pragma unroll
            for (int e = 0; e < P; ++e) {
                x[HALVES ? 2 * e : e] = csdr::to_f32(u.v[e]);
                x[HALVES ? 2 * e + 1 : P + e] = csdr::to_f32(v.v[e]);
            }
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float2 c = cs[t.pair + e];
                const float y = x[2 * e] * c.x - x[2 * e + 1] * c.y;
                x[2 * e + 1] = x[2 * e] * c.y + x[2 * e + 1] * c.x;
                x[2 * e] = y;
            }
#pragma unroll
            for (int e = 0; e < P; ++e) {
                p.v[e] = (T)x[HALVES ? 2 * e : e];
                w.v[e] = (T)x[HALVES ? 2 * e + 1 : P + e];
            }
        }
        *reinterpret_cast<V*>(t.out) = p;
        if (!t.one) *reinterpret_cast<V*>(t.out + t.second) = w;
    };

    const int mine = group * kThreads + threadIdx.x;
    Item t[AHEAD];
    V u[AHEAD], v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (i * step < all) {
            t[i] = item_of(min(mine + i * step, all - 1));
            load(t[i], u[i], v[i]);
        }
    for (int j = threadIdx.x; j < tokens * half; j += kThreads) {
        const int local = tokens > 1 ? j / half : 0;
        const double r = (double)a.positions[first + local] * a.turns[j - local * half];
        const float f = (float)(r - rint(r));
        float s, c;
        sincospif(2.0f * f, &s, &c);
        cs[j] = make_float2(c * a.magnitude, s * a.magnitude);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (mine + i * step < all) put(t[i], u[i], v[i]);
    for (int i = mine + AHEAD * step; i < all; i += step) {
        t[0] = item_of(i);
        load(t[0], u[0], v[0]);
        put(t[0], u[0], v[0]);
    }
}

template <typename T>
void launch(const Args& a, bool halves, bool wide, hipStream_t st) {
    const unsigned grid = (unsigned)((a.n_tokens + a.tokens - 1) / a.tokens) * (unsigned)a.groups;
    if (halves) {
        if (wide) rotary_kernel<T, true, true><<<grid, kThreads, 0, st>>>(a);
        else rotary_kernel<T, true, false><<<grid, kThreads, 0, st>>>(a);
    } else {
        if (wide) rotary_kernel<T, false, true><<<grid, kThreads, 0, st>>>(a);
        else rotary_kernel<T, false, false><<<grid, kThreads, 0, st>>>(a);
    }
}

}  // namespace

extern "C" {

CSDR_API int csdr_rotary(const void* q, void* q_out, int Hq, int64_t q_stride, int64_t q_out_stride,
                         const void* k, void* k_out, int Hk, int64_t k_stride, int64_t k_out_stride,
                         int dtype, int n_tokens, int head_dim, int dims, int layout,
                         const int32_t* positions, const double* turns, float magnitude,
                         void* hip_stream) {
    if (!q || !q_out || !positions || !turns || (k != nullptr) != (k_out != nullptr))
        return set_error(CSDR_E_INVALID, "rotary: a pointer is NULL");
    if (dtype != CSDR_F32 && dtype != CSDR_F16)
        return set_error(CSDR_E_INVALID, "rotary: dtype must be CSDR_F32 or CSDR_F16");
    if (layout != CSDR_ROTARY_ADJACENT && layout != CSDR_ROTARY_HALVES)
        return set_error(CSDR_E_INVALID, "rotary: layout must be CSDR_ROTARY_ADJACENT or _HALVES");
    if (n_tokens <= 0 || Hq <= 0 || (k && Hk <= 0) || Hq > 65535 || Hk > 65535)
        return set_error(CSDR_E_INVALID, "rotary: bad sizes");
    if (head_dim <= 0 || head_dim > kMaxDim || dims <= 0 || dims > head_dim || dims % 2)
        return set_error(CSDR_E_UNSUPPORTED,
                         "rotary: dims must be even and up to head_dim, head_dim up to 1024");
    if (!(fabsf(magnitude) < INFINITY))
        return set_error(CSDR_E_INVALID, "rotary: the magnitude is not finite");
    Args a{};
    const int64_t nq = (int64_t)Hq * head_dim, nk = k ? (int64_t)Hk * head_dim : 0;
    a.q = {q, q_out, q_stride ? q_stride : nq, q_out_stride ? q_out_stride : nq, Hq};
    a.k = {k, k_out, k_stride ? k_stride : nk, k_out_stride ? k_out_stride : nk, k ? Hk : 0};
    if (a.q.in_stride < nq || a.q.out_stride < nq || a.k.in_stride < nk || a.k.out_stride < nk)
        return set_error(CSDR_E_INVALID, "rotary: a token stride is below its heads");
    if (n_tokens > 1 && ((q == q_out && a.q.in_stride != a.q.out_stride) ||
                         (k && k == k_out && a.k.in_stride != a.k.out_stride)))
        return set_error(CSDR_E_INVALID, "rotary: in place both strides must be the same");
    if (k && (q_out == k || k_out == q || q_out == k_out))
        return set_error(CSDR_E_INVALID, "rotary: an output is the other's input or output");
    a.positions = positions;
    a.turns = turns;
    a.n_tokens = n_tokens;
    a.hd = head_dim;
    a.dims = dims;
    a.magnitude = magnitude;
    const bool wide = dims % (2 * kUnit) == 0 && head_dim % (2 * kUnit) == 0;
    // few tokens: their heads over more workgroups; many of few heads: several to a workgroup
    const long long items = (nq + nk) / (wide ? 2 * kUnit : 2);
    a.groups = (int)std::min<long long>((items + kThreads - 1) / kThreads, std::max(1, 1024 / n_tokens));
    a.tokens = 1;
    if (a.groups == 1 && n_tokens > 1024)
        a.tokens = (int)std::max<long long>(1, std::min<long long>(kThreads / items, kMaxDim / dims));
    if ((long long)n_tokens * a.groups >= (1LL << 24))
        return set_error(CSDR_E_INVALID, "rotary: more than 2^24 - 1 tokens");
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (dtype == CSDR_F32) launch<float>(a, layout == CSDR_ROTARY_HALVES, wide, st);
    else launch<_Float16>(a, layout == CSDR_ROTARY_HALVES, wide, st);
    CSDR_LAUNCH_CHECK("rotary");
    return CSDR_OK;
}

}  // extern "C"
