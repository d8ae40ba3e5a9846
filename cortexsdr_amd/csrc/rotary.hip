// rotary.hip — rotary positions for the forms that the cache's own rotation (csdr_paged_append,
// csdr_rope_kv_rows) has not: halves as well as adjacent pairs, the first dims of a head, any frequencies and a
// magnitude (gfx950).
//   (u, v) -> magnitude (u c - v s, u s + v c),  c + i s = exp(i position frequency_j) for pair j
//
// The angle is held in turns in fp64 (an fp32 angle is off by 4e-3 rad at position 65536), its whole turns
// dropped before the fp32 sine and cosine of what is left, at most half a turn. They are computed once per
// token and pair and shared by the heads of a workgroup through LDS. A thread takes 8 pairs, 32 or 64 bytes in
// and out. Bound by memory: 8192 tokens of 32 + 32 heads of 128 in fp16 take 56 us, 4.8 TB/s; a step's tokens
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
    int n_tokens, hd, dims, groups;
    float magnitude;
};

// A workgroup per token and group of heads. WIDE: 8 pairs a thread; else one.
template <typename T, bool HALVES, bool WIDE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Args a) {
    __shared__ float2 cs[kMaxDim / 2];
    const int token = blockIdx.x / a.groups, group = blockIdx.x % a.groups;
    const int pos = a.positions[token];
    if (pos < 0) return;  // no token
    const int half = a.dims / 2;
    for (int j = threadIdx.x; j < half; j += kThreads) {
        const double u = (double)pos * a.turns[j];
        const float f = (float)(u - rint(u));
        float s, c;
        sincospif(2.0f * f, &s, &c);
        cs[j] = make_float2(c * a.magnitude, s * a.magnitude);
    }
    __syncthreads();
    // items of a head: its pairs, then its other dims
    constexpr int P = WIDE ? kUnit : 1, O = 2 * P;
    const int turned = half / P, items = turned + (a.hd - a.dims) / O + (WIDE ? 0 : (a.hd - a.dims) % O);
    const int heads = a.q.heads + a.k.heads;
    for (int i = group * kThreads + threadIdx.x; i < heads * items; i += a.groups * kThreads) {
        const int head = i / items, item = i % items;
        const bool is_k = head >= a.q.heads;
        const Side& s = is_k ? a.k : a.q;
        const int h = is_k ? head - a.q.heads : head;
        const T* in = static_cast<const T*>(s.in) + token * s.in_stride + (long long)h * a.hd;
        T* out = static_cast<T*>(s.out) + token * s.out_stride + (long long)h * a.hd;
        if (item >= turned) {  // as they are
            const int at = a.dims + (item - turned) * O;
            if (in != out) {
                if (at + O <= a.hd)
                    *reinterpret_cast<Vec<T, O>*>(out + at) = *reinterpret_cast<const Vec<T, O>*>(in + at);
                else
                    out[at] = in[at];
            }
            continue;
        }
        const int j = item * P;
        float u[P], v[P];
        if (HALVES) {
            const Vec<T, P> x0 = *reinterpret_cast<const Vec<T, P>*>(in + j);
            const Vec<T, P> x1 = *reinterpret_cast<const Vec<T, P>*>(in + half + j);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                u[e] = csdr::to_f32(x0.v[e]);
                v[e] = csdr::to_f32(x1.v[e]);
            }
        } else {
            const Vec<T, O> x = *reinterpret_cast<const Vec<T, O>*>(in + 2 * j);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                u[e] = csdr::to_f32(x.v[2 * e]);
                v[e] = csdr::to_f32(x.v[2 * e + 1]);
            }
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const float2 t = cs[j + e];
            const float p = u[e] * t.x - v[e] * t.y;
            v[e] = u[e] * t.y + v[e] * t.x;
            u[e] = p;
        }
        if (HALVES) {
            Vec<T, P> y0, y1;
#pragma unroll
            for (int e = 0; e < P; ++e) {
                y0.v[e] = (T)u[e];
                y1.v[e] = (T)v[e];
            }
            *reinterpret_cast<Vec<T, P>*>(out + j) = y0;
            *reinterpret_cast<Vec<T, P>*>(out + half + j) = y1;
        } else {
            Vec<T, O> y;
#pragma unroll
            for (int e = 0; e < P; ++e) {
                y.v[2 * e] = (T)u[e];
                y.v[2 * e + 1] = (T)v[e];
            }
            *reinterpret_cast<Vec<T, O>*>(out + 2 * j) = y;
        }
    }
}

template <typename T>
void launch(const Args& a, bool halves, bool wide, hipStream_t st) {
    const unsigned grid = (unsigned)a.n_tokens * (unsigned)a.groups;
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
    a.positions = positions;
    a.turns = turns;
    a.n_tokens = n_tokens;
    a.hd = head_dim;
    a.dims = dims;
    a.magnitude = magnitude;
    const bool wide = dims % (2 * kUnit) == 0 && head_dim % (2 * kUnit) == 0;
    // few tokens: their heads over more workgroups
    const long long items = (nq + nk) / (wide ? 2 * kUnit : 2);
    a.groups = (int)std::min<long long>((items + kThreads - 1) / kThreads,
                                        std::max(1, 1024 / n_tokens));
    if ((long long)n_tokens * a.groups >= (1LL << 24))
        return set_error(CSDR_E_INVALID, "rotary: more than 2^24 - 1 tokens");
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (dtype == CSDR_F32) launch<float>(a, layout == CSDR_ROTARY_HALVES, wide, st);
    else launch<_Float16>(a, layout == CSDR_ROTARY_HALVES, wide, st);
    CSDR_LAUNCH_CHECK("rotary");
    return CSDR_OK;
}

}  // extern "C"
