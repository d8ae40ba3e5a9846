// q8_rows.hip — rows of values as 8-bit codes with a scale each, from a root-mean-square norm with the
// residual's addition, from values as they are, or from silu(gate) * x; and back to values (gfx950).
//
// A row v: top = max |v|, code = rint(127 v / top) (ties to even), scale = top / 127 in fp32. The codes are
// those of exact arithmetic (of a gated value as fp64 forms it, but within 2^-42 of a border), so that a code does
// not depend on the order of a sum or on which kernel made it.
// The norm's 1 / rms is in every value of a row and cancels in its codes: they come from t = h w alone, a
// product of two fp32 numbers that fp64 holds exactly, and one pass over the row gives both the sum of squares
// (fp64) and top. Values, their largest and their codes are formed in fp32, and in fp64 only where that may not
// be enough: the values that may be the row's largest, the codes next to a border between two (one of several
// thousand), rows so small that fp32 holds their values with few bits or so large that it does not hold them.
//
// A workgroup takes a row, and its values stay in registers between the pass that finds their largest and the
// one that writes codes. Bound by memory: the norm of 4096 rows of 4096 in fp16 with its residual takes 22 us,
// 5.3 TB/s; the gated rows of 4096 x 11008 in fp16 49 us, 4.6 TB/s (an exponential and a reciprocal a value, 30
// instructions in all, beside the loads); 22016 x 4096 fp32 weights 75 us, 6.0 TB/s; the way back to fp16 of
// 4096 x 11008 22 us. Few rows are one round trip and two barriers (one row 3 us).
//
// A row that holds a value which is not finite (or whose scale passes fp32) has the scale NaN and codes 0, so
// it reads as NaN; a row of zeros has the scale 0 (a norm's without eps is NaN).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "q8.hpp"

namespace {

using csdr::kMaxWidth;
using csdr::q8_pitch;
using csdr::set_error;

constexpr int kChunk = 8;  // consecutive values of a thread: one 8-byte store of codes
constexpr int kMaxThreads = 1024;
constexpr int kCUs = 256;
constexpr int kMaxRows = (1 << 22) - 1;  // fewer than 2^32 threads a launch

typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// Consecutive values at any alignment of their type.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[kChunk];
};

// The chunk at `at` of a row of n values as it lies there, without a branch (another chunk of the row where it
// is not whole), so that a thread's loads are on their way together; then its values, zeros behind the last.
template <typename T>
__device__ __forceinline__ Vec<T> raw_of(const T* row, int at, int n) {
    return *reinterpret_cast<const Vec<T>*>(row + (at + kChunk <= n ? at : 0));
}
template <typename T>
__device__ __forceinline__ void values_of(const Vec<T>& raw, const T* row, int at, int n, float* f) {
    if (at + kChunk <= n) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) f[i] = csdr::to_f32(raw.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) f[i] = at + i < n ? csdr::to_f32(row[at + i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void load(const T* p, int left, float* f) {
    if (left >= kChunk) {
        const Vec<T> a = *reinterpret_cast<const Vec<T>*>(p);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) f[i] = csdr::to_f32(a.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) f[i] = i < left ? csdr::to_f32(p[i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store(T* p, int left, const float* f) {
    if (left >= kChunk) {
        Vec<T> a;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) a.v[i] = (T)f[i];
        *reinterpret_cast<Vec<T>*>(p) = a;
    } else {
        for (int i = 0; i < left; ++i) p[i] = (T)f[i];
    }
}

__device__ __forceinline__ uint64_t bits_of(double v) { return __builtin_bit_cast(uint64_t, v); }
__device__ __forceinline__ double of_bits(uint64_t v) { return __builtin_bit_cast(double, v); }

// How far a value formed in fp32 is off at most, of itself: 8 roundings for a gated value (the exponential and
// the reciprocal are off by a step), one for a norm's; and then its code, of 127 at most: with a quarter to
// spare.
constexpr float kValueOff = 1.2e-6f, kCodeOff = 1e-4f;
// Rows whose largest value is below kTiny are formed in fp64 throughout.
constexpr float kTiny = 1e-25f;
// Rows with a gate below it too: the sigmoid leaves the normal numbers of fp32.
constexpr float kLow = -87.0f;

// What a row's threads have to agree on, and what they pass it through.
struct Joined {
    double sum;
    uint32_t most;  // bits of the largest magnitude in fp32; a NaN's are larger than any number's
    bool low;
};
struct Shared {
    double sum[kMaxThreads / 64];
    uint32_t most[kMaxThreads / 64];
    unsigned long long top;
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const u2 b = __builtin_bit_cast(u2, v);
    return __builtin_bit_cast(double, u2{dpp<CTRL>(b[0]), dpp<CTRL>(b[1])});
}
// lane ^ 1, lane ^ 2, mirrored within 8 and within 16 lanes, which then hold one value
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;

template <bool SUM>
__device__ __forceinline__ Joined join(Joined r, Shared& lds) {
    r.most = max(r.most, dpp<kXor1>(r.most));
    r.most = max(r.most, dpp<kXor2>(r.most));
    r.most = max(r.most, dpp<kHalfMirror>(r.most));
    r.most = max(r.most, dpp<kMirror>(r.most));
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, (uint32_t)__builtin_amdgcn_readlane((int)r.most, 16 * i));
    if (SUM) {
        r.sum += dpp<kXor1>(r.sum);
        r.sum += dpp<kXor2>(r.sum);
        r.sum += dpp<kHalfMirror>(r.sum);
        r.sum += dpp<kMirror>(r.sum);
        r.sum += __shfl_xor(r.sum, 16, 64);
        r.sum += __shfl_xor(r.sum, 32, 64);
    }
    r.low = __any(r.low);
    if (threadIdx.x == 0) lds.top = 0;
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        if (SUM) lds.sum[threadIdx.x >> 6] = r.sum;
        lds.most[threadIdx.x >> 6] = most << 1 | (r.low ? 1u : 0u);  // (the sign's bit is free)
    }
    __syncthreads();
    r.sum = 0.0;
    uint32_t both = 0, low = 0;
    for (int i = 0; i < waves; ++i) {
        if (SUM) r.sum += lds.sum[i];
        both = max(both, lds.most[i]);
        low |= lds.most[i] & 1u;
    }
    r.most = both >> 1;
    r.low = low != 0;
    return r;
}

// 1 / v and 1 / sqrt(v) to about 2^-50, for v normal, by Newton's steps from the instruction's estimate: every
// thread of a row forms them (norm of 4096 x 4096 in fp16 24.0 us with the full division and root, 22.3 so).
__device__ __forceinline__ double reciprocal(double v) {
    double r = __builtin_amdgcn_rcp(v);
    r = fma(fma(-v, r, 1.0), r, r);
    return fma(fma(-v, r, 1.0), r, r);
}
__device__ __forceinline__ double inverse_root(double v) {
    if (v == INFINITY) return 0.0;
    double r = __builtin_amdgcn_rsq(v);
    r = fma(fma(-v * r, r, 1.0), 0.5 * r, r);
    return fma(fma(-v * r, r, 1.0), 0.5 * r, r);
}

struct Scale {
    double inv, top;  // 127 / top (0 for rows without codes)
    float inv32, value;
    bool wide;        // codes in fp64 throughout
};

__device__ __forceinline__ Scale scale_of(double top, double factor, bool wide) {
    Scale s;
    s.top = top;
    s.value = (float)(top * factor * (1.0 / 127.0));
    const bool fine = s.value < INFINITY;  // (not for a NaN)
    if (!fine) s.value = NAN;
    s.inv = fine && top > 0.0 ? 127.0 * reciprocal(top) : 0.0;
    s.inv32 = (float)s.inv;
    s.wide = wide;
    return s;
}

// The nearest code of t, in exact arithmetic but for 1e-13 of the product with the reciprocal. Next to a border (k + 1/2
// of a code) of |t|, EXACT (for t and top of 48 bits, products of two fp32 numbers): 254 |t| against (2 k + 1) top, the
// second as a product and what it is rounded by, and their difference, a multiple of top's last place, too small to be
// rounded; ties to even. Otherwise the quotient as fp64 rounds it: a gated value has fp64's roundings in itself, and
// values of one gate that tie in the formula are to tie here.
template <bool EXACT>
__device__ __forceinline__ int code_of(double t, const Scale& s) {
    const double q = t * s.inv;
    double r = rint(q);
    if (__builtin_expect(fabs(fabs(q - r) - 0.5) < 1e-9, 0)) {
        if (EXACT) {
            const double k = floor(fabs(q)), odd = 2.0 * k + 1.0, border = odd * s.top;
            const double over = fma(254.0, fabs(t), -border), rounded = fma(odd, s.top, -border);
            const bool up = over > rounded || (over == rounded && ((int)k & 1));
            r = copysign(up ? k + 1.0 : k, t);
        } else {
            r = rint(127.0 * t / s.top);
        }
    }
    return (int)r;
}

// The codes of a chunk's values t, exact(i) being value i in fp64. 3 2^22 + q holds rint(q) in its low bits.
template <bool EXACT, typename Exact>
__device__ __forceinline__ void put_codes(int8_t* p, const float* t, const Scale& s, Exact exact) {
    u2 v = {0, 0};
    if (s.inv > 0.0) {
        constexpr float kMagic = 12582912.0f;
        uint32_t c[kChunk];
        float d[kChunk], most = 0.0f;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            const float u = fmaf(t[i], s.inv32, kMagic);
            d[i] = fabsf(fmaf(t[i], s.inv32, -(u - kMagic)));
            c[i] = __float_as_uint(u);
            most = fmaxf(most, d[i]);
        }
        if (__builtin_expect(most > 0.5f - kCodeOff || s.wide, 0)) {
#pragma unroll
            for (int i = 0; i < kChunk; ++i)
                if (d[i] > 0.5f - kCodeOff || s.wide) c[i] = (uint32_t)code_of<EXACT>(exact(i), s);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            v[i] = __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0c0c0400u) |
                   __builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x04000c0cu);
    }
    *reinterpret_cast<u2*>(p) = v;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// ------------------------------------------------------------------ norm

struct NormArgs {
    const void *x, *residual;
    void *residual_out, *y;
    const float* w;
    int8_t* codes;
    float* scales;
    long long x_stride, residual_stride;
    int n, pitch;
    float eps;
    double inv_n;
};

// h = x + residual as the stream holds it.
template <typename TX, typename TR, bool RES>
__device__ __forceinline__ void load_h(const NormArgs& a, long long row, int at, float* h) {
    load(static_cast<const TX*>(a.x) + row * a.x_stride + at, a.n - at, h);
    if (RES) {
        float r[kChunk];
        load(static_cast<const TR*>(a.residual) + row * a.residual_stride + at, a.n - at, r);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) h[i] = (float)(TR)(h[i] + r[i]);
    }
}

// A row per workgroup. NV > 0: its values stay in registers, NV chunks a thread; 0: rows of any width,
// formed again for each step. What fp64 needs comes from memory again.
template <typename TX, typename TR, bool RES, int NV>
__global__ __launch_bounds__(kMaxThreads) void norm_kernel(NormArgs a) {
    __shared__ Shared lds;
    const long long row = blockIdx.x;
    const int step = blockDim.x * kChunk, first = threadIdx.x * kChunk;
    constexpr int N = NV > 0 ? NV : 1;
    float t[N][kChunk] = {};  // h w
    Joined r = {0.0, 0, false};
    TR* out = RES ? static_cast<TR*>(a.residual_out) + row * a.n : nullptr;

    auto each = [&](int end, auto f) {
        if (NV > 0) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (first + j * step < end) f(j, first + j * step);
        } else {
            for (int at = first; at < end; at += step) f(0, at);
        }
    };
    // h as the stream holds it (where that is updated in place its old values are gone)
    auto load_again = [&](int at, float* h, float* w) {
        load(a.w + at, a.n - at, w);
        if (RES) load(out + at, a.n - at, h);
        else load_h<TX, TR, RES>(a, row, at, h);
    };
    auto again = [&](int at) {
        if (NV > 0) return;
        float h[kChunk], w[kChunk];
        load_again(at, h, w);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) t[0][i] = h[i] * w[i];
    };
    auto exact = [&](int at) {  // (at < n)
        const float h = RES ? csdr::to_f32(out[at])
                            : csdr::to_f32(static_cast<const TX*>(a.x)[row * a.x_stride + at]);
        return (double)h * (double)a.w[at];
    };
    const TX* px = static_cast<const TX*>(a.x) + row * a.x_stride;
    const TR* pr = static_cast<const TR*>(a.residual) + row * a.residual_stride;
    auto take = [&](int j, int at, const Vec<TX>& x, const Vec<TR>& res, const Vec<float>& wv) {
        float h[kChunk], w[kChunk], u[kChunk];
        values_of(wv, a.w, at, a.n, w);
        values_of(x, px, at, a.n, h);
        if (RES) {
            values_of(res, pr, at, a.n, u);
#pragma unroll
            for (int i = 0; i < kChunk; ++i) h[i] = (float)(TR)(h[i] + u[i]);
            store(out + at, a.n - at, h);
        }
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            t[j][i] = h[i] * w[i];
            r.sum = fma((double)h[i], (double)h[i], r.sum);
            r.most = max(r.most, magnitude(t[j][i]));
        }
    };
    Vec<TX> x[N];
    Vec<TR> res[N];
    Vec<float> wv[N];
    auto fetch = [&](int j, int at) {
        x[j] = raw_of(px, at, a.n);
        if (RES) res[j] = raw_of(pr, at, a.n);
        wv[j] = raw_of(a.w, at, a.n);
    };
    if (NV > 0 && a.n >= kChunk) {
#pragma unroll
        for (int j = 0; j < N; ++j) fetch(j, first + j * step);
    }
    each(a.n, [&](int j, int at) {
        if (NV == 0) fetch(0, at);
        take(j, at, x[j], res[j], wv[j]);
    });
    const uint32_t mine = r.most;
    r = join<true>(r, lds);
    const float top32 = __uint_as_float(r.most);
    const bool wide = !(top32 >= kTiny) || top32 == INFINITY;
    if (wide || __uint_as_float(mine) >= top32 * (1.0f - kValueOff)) {
        each(a.n, [&](int j, int at) {
            again(at);
#pragma unroll
            for (int i = 0; i < kChunk; ++i)
                if ((wide || fabsf(t[j][i]) >= top32 * (1.0f - kValueOff)) && at + i < a.n)
                    atomicMax(&lds.top, (unsigned long long)bits_of(fabs(exact(at + i))));
        });
    }
    __syncthreads();
    const double rms = inverse_root(r.sum * a.inv_n + (double)a.eps);
    // (a finite top beside a sum that is not: a weight of 0 under a value that is not finite)
    const Scale s = scale_of(r.sum < INFINITY && top32 == top32 ? of_bits(lds.top) : (double)NAN, rms, wide);
    if (threadIdx.x == 0 && a.scales) a.scales[row] = s.value;

    if (a.codes)
        each(a.pitch, [&](int j, int at) {
            again(at);
            put_codes<true>(a.codes + row * a.pitch + at, t[j], s,
                            [&](int i) { return at + i < a.n ? exact(at + i) : 0.0; });
        });
    if (a.y)
        each(a.n, [&](int, int at) {
            float h[kChunk], w[kChunk];
            load_again(at, h, w);
#pragma unroll
            for (int i = 0; i < kChunk; ++i) h[i] = (float)((double)h[i] * rms * (double)w[i]);
            store(static_cast<TX*>(a.y) + row * a.n + at, a.n - at, h);
        });
}

// ------------------------------------------------------------------ rows as they are, or gated

struct RowsArgs {
    const void *x, *gate;
    int8_t* codes;
    float* scales;
    long long x_stride, gate_stride;
    int n, pitch;
};

// silu(g) x. exp(-g) = 2^p (1 + rest ln 2), p and the rest of its rounding from two parts of 1 / ln 2, so that
// a large gate costs no bits; beyond kLow the gate is held where the sigmoid is a normal number, and above 150 the
// exponential is nothing beside 1. The sigmoid comes last: a subnormal gate has all its bits in g x (gate times sigmoid
// would round to a few), where g x is itself subnormal the value is far below kTiny / 127, and where g x passes fp32 the
// value is infinite here, so that its row is formed in fp64.
__device__ __forceinline__ float gated(float g, float x) {
    constexpr float kHi = 1.44269502162933349609375f, kLo = 1.92596299e-8f, kLn2 = 0.69314718f;
    const float v = __builtin_amdgcn_fmed3f(-g, -150.0f, -kLow), p = v * kHi;
    const float rest = fmaf(v, kLo, fmaf(v, kHi, -p));
    const float e2 = __builtin_amdgcn_exp2f(p), e = fmaf(e2, rest * kLn2, e2);
    return g * x * __builtin_amdgcn_rcpf(1.0f + e);
}
__device__ __forceinline__ double gated(double g, double x) { return g / (1.0 + exp(-g)) * x; }

template <typename T, bool GATE, int NV>
__global__ __launch_bounds__(kMaxThreads) void rows_kernel(RowsArgs a) {
    __shared__ Shared lds;
    const long long row = blockIdx.x;
    const int step = blockDim.x * kChunk, first = threadIdx.x * kChunk;
    constexpr int N = NV > 0 ? NV : 1;
    float t[N][kChunk] = {};
    Joined r = {0.0, 0, false};
    const T* px = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* pg = static_cast<const T*>(a.gate) + row * a.gate_stride;

    auto each = [&](int end, auto f) {
        if (NV > 0) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (first + j * step < end) f(j, first + j * step);
        } else {
            for (int at = first; at < end; at += step) f(0, at);
        }
    };
    Vec<T> x[N], gate[N];
    auto fetch = [&](int j, int at) {
        x[j] = raw_of(px, at, a.n);
        if (GATE) gate[j] = raw_of(pg, at, a.n);
    };
    auto take = [&](int j, int at, bool look) {
        float g[kChunk];
        if (NV == 0) fetch(0, at);
        values_of(x[j], px, at, a.n, t[j]);
        if (GATE) {
            values_of(gate[j], pg, at, a.n, g);
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
                // (in fp16 what the exponential loses is below kTiny / 127 of any row formed in fp32)
                if (sizeof(T) == 4 && look) r.low |= g[i] < kLow;
                t[j][i] = gated(g[i], t[j][i]);
            }
        }
    };
    if (NV > 0 && a.n >= kChunk) {
#pragma unroll
        for (int j = 0; j < N; ++j) fetch(j, first + j * step);
    }
    auto again = [&](int at) {
        if (NV == 0) take(0, at, false);
    };
    auto exact = [&](int at) {  // (at < n)
        const double x = (double)csdr::to_f32(px[at]);
        return GATE ? gated((double)csdr::to_f32(pg[at]), x) : x;
    };
    each(a.n, [&](int j, int at) {
        take(j, at, true);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) r.most = max(r.most, magnitude(t[j][i]));
    });
    const uint32_t mine = r.most;
    r = join<false>(r, lds);
    const float top32 = __uint_as_float(r.most);
    double top = (double)top32;
    bool wide = !(top32 >= kTiny);
    if (GATE) {
        wide = wide || r.low || top32 == INFINITY;
        if (wide || __uint_as_float(mine) >= top32 * (1.0f - kValueOff)) {
            each(a.n, [&](int j, int at) {
                again(at);
#pragma unroll
                for (int i = 0; i < kChunk; ++i)
                    if ((wide || fabsf(t[j][i]) >= top32 * (1.0f - kValueOff)) && at + i < a.n)
                        atomicMax(&lds.top, (unsigned long long)bits_of(fabs(exact(at + i))));
            });
        }
        __syncthreads();
        if (top32 == top32) top = of_bits(lds.top);
    }
    const Scale s = scale_of(top, 1.0, wide);
    if (threadIdx.x == 0) a.scales[row] = s.value;
    each(a.pitch, [&](int j, int at) {
        again(at);
        put_codes<!GATE>(a.codes + row * a.pitch + at, t[j], s,
                         [&](int i) { return at + i < a.n ? exact(at + i) : 0.0; });
    });
}

// ------------------------------------------------------------------ back to values

// 16 codes a thread.
template <typename T>
__global__ __launch_bounds__(256) void values_kernel(const int8_t* codes, const float* scales, int n,
                                                     int pitch, int per_row, T* out) {
    const long long row = blockIdx.x / per_row;
    const int at = ((int)(blockIdx.x % per_row) * 256 + (int)threadIdx.x) * 16;
    if (at >= n) return;
    const float s = scales[row];
    const uint4 c = *reinterpret_cast<const uint4*>(codes + row * pitch + at);
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
    T* o = out + row * n + at;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float f[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
            f[i] = s * (float)(int8_t)(words[2 * k + i / 4] >> (8 * (i % 4)));
        if (at + 8 * k < n) store(o + 8 * k, n - at - 8 * k, f);
    }
}

// Threads of a row and chunks a thread (0: more than the registers hold). Many rows take up to 512 threads, so that more
// of them are on a CU, one's loads beside another's codes (gated fp16 rows of 11008, 4096 of them: 47 to 50 us with
// three chunks a thread, 54 to 57 with two; of 14336, 3000: 53 with four, 59 with two); few take as many as there may
// be (64 gated rows of 14336: 6.8 us with two chunks, 7.8 with four).
struct Shape {
    int threads, nv;
};
Shape shape_of(int width, int rows) {
    const int chunks = (width + kChunk - 1) / kChunk, want = rows < 2 * kCUs ? kMaxThreads : 512;
    if (chunks > 4 * kMaxThreads) return {kMaxThreads, 0};
    const int nv = std::min((chunks + want - 1) / want, 4);
    return {((chunks + nv - 1) / nv + 63) / 64 * 64, nv};
}

template <typename TX, typename TR, bool RES>
void launch_norm(const NormArgs& a, int rows, hipStream_t st) {
    const Shape s = shape_of(a.codes ? a.pitch : a.n, rows);
    if (s.nv == 1) norm_kernel<TX, TR, RES, 1><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 2) norm_kernel<TX, TR, RES, 2><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 3) norm_kernel<TX, TR, RES, 3><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 4) norm_kernel<TX, TR, RES, 4><<<rows, s.threads, 0, st>>>(a);
    else norm_kernel<TX, TR, RES, 0><<<rows, s.threads, 0, st>>>(a);
}

template <typename T, bool GATE>
void launch_rows(const RowsArgs& a, int rows, hipStream_t st) {
    const Shape s = shape_of(a.pitch, rows);
    if (s.nv == 1) rows_kernel<T, GATE, 1><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 2) rows_kernel<T, GATE, 2><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 3) rows_kernel<T, GATE, 3><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 4) rows_kernel<T, GATE, 4><<<rows, s.threads, 0, st>>>(a);
    else rows_kernel<T, GATE, 0><<<rows, s.threads, 0, st>>>(a);
}

bool type_ok(int dtype) { return dtype == CSDR_F32 || dtype == CSDR_F16; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int check_rows(const char* what, int rows, int n) {
    if (rows <= 0 || n <= 0) return set_error(CSDR_E_INVALID, std::string(what) + ": bad sizes");
    if (rows > kMaxRows)
        return set_error(CSDR_E_INVALID, std::string(what) + ": more than 2^22 - 1 rows");
    if (n > kMaxWidth)
        return set_error(CSDR_E_UNSUPPORTED, std::string(what) + ": more than 131071 columns");
    return CSDR_OK;
}

}  // namespace

extern "C" {

CSDR_API size_t csdr_q8_pitch(int n) { return n <= 0 || n > kMaxWidth ? 0 : q8_pitch(n); }

CSDR_API int csdr_q8_quantize(const void* x, const void* gate, int dtype, int rows, int n,
                              int64_t x_stride, int64_t gate_stride, int8_t* codes, float* scales,
                              void* hip_stream) {
    if (!x || !codes || !scales) return set_error(CSDR_E_INVALID, "q8_quantize: a pointer is NULL");
    if (!type_ok(dtype))
        return set_error(CSDR_E_INVALID, "q8_quantize: dtype must be CSDR_F32 or CSDR_F16");
    if (int rc = check_rows("q8_quantize", rows, n)) return rc;
    if ((x_stride != 0 && x_stride < n) || (gate && gate_stride != 0 && gate_stride < n))
        return set_error(CSDR_E_INVALID, "q8_quantize: a row stride is below n");
    if (!aligned(codes, 16))
        return set_error(CSDR_E_INVALID, "q8_quantize: codes must be 16-byte aligned");
    if (codes == x || codes == gate) return set_error(CSDR_E_INVALID, "q8_quantize: codes are an input");
    RowsArgs a{x, gate, codes, scales, x_stride ? x_stride : n, gate_stride ? gate_stride : n, n,
               (int)q8_pitch(n)};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (dtype == CSDR_F32) {
        if (gate) launch_rows<float, true>(a, rows, st);
        else launch_rows<float, false>(a, rows, st);
    } else {
        if (gate) launch_rows<_Float16, true>(a, rows, st);
        else launch_rows<_Float16, false>(a, rows, st);
    }
    CSDR_LAUNCH_CHECK("q8_quantize");
    return CSDR_OK;
}

CSDR_API int csdr_q8_dequantize(const int8_t* codes, const float* scales, int rows, int n, void* out,
                                int dtype, void* hip_stream) {
    if (!codes || !scales || !out)
        return set_error(CSDR_E_INVALID, "q8_dequantize: a pointer is NULL");
    if (!type_ok(dtype))
        return set_error(CSDR_E_INVALID, "q8_dequantize: dtype must be CSDR_F32 or CSDR_F16");
    if (int rc = check_rows("q8_dequantize", rows, n)) return rc;
    if (!aligned(codes, 16))
        return set_error(CSDR_E_INVALID, "q8_dequantize: codes must be 16-byte aligned");
    if (out == codes) return set_error(CSDR_E_INVALID, "q8_dequantize: out is codes");
    const int per_row = (n + 16 * 256 - 1) / (16 * 256);
    const long long blocks = (long long)rows * per_row;
    if (blocks >= (1LL << 24))
        return set_error(CSDR_E_INVALID, "q8_dequantize: more workgroups than a launch may have");
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int pitch = (int)q8_pitch(n);
    if (dtype == CSDR_F32)
        values_kernel<<<(unsigned)blocks, 256, 0, st>>>(codes, scales, n, pitch, per_row,
                                                        static_cast<float*>(out));
    else
        values_kernel<<<(unsigned)blocks, 256, 0, st>>>(codes, scales, n, pitch, per_row,
                                                        static_cast<_Float16*>(out));
    CSDR_LAUNCH_CHECK("q8_dequantize");
    return CSDR_OK;
}

CSDR_API int csdr_add_rms_norm(const void* x, int dtype, int64_t x_stride, const void* residual,
                               int residual_dtype, int64_t residual_stride, void* residual_out,
                               const float* w, float eps, int rows, int n, void* y, int8_t* codes,
                               float* scales, void* hip_stream) {
    if (!x || !w || (!y && !codes) || (codes != nullptr) != (scales != nullptr) ||
        (residual != nullptr) != (residual_out != nullptr))
        return set_error(CSDR_E_INVALID, "add_rms_norm: a pointer is NULL");
    if (!type_ok(dtype) || (residual && !type_ok(residual_dtype)))
        return set_error(CSDR_E_INVALID, "add_rms_norm: types must be CSDR_F32 or CSDR_F16");
    if (int rc = check_rows("add_rms_norm", rows, n)) return rc;
    if (!(eps >= 0.0f && eps < INFINITY))
        return set_error(CSDR_E_INVALID, "add_rms_norm: eps must be finite and not negative");
    if ((x_stride != 0 && x_stride < n) || (residual && residual_stride != 0 && residual_stride < n))
        return set_error(CSDR_E_INVALID, "add_rms_norm: a row stride is below n");
    if (codes && !aligned(codes, 16))
        return set_error(CSDR_E_INVALID, "add_rms_norm: codes must be 16-byte aligned");
    if (residual && residual_out == residual && rows > 1 && residual_stride != 0 &&
        residual_stride != n)
        return set_error(CSDR_E_INVALID, "add_rms_norm: a stream updated in place must be packed");
    if ((residual && residual_out == x) || (y && (y == x || y == residual || y == residual_out)) ||
        (codes && (codes == x || codes == residual || codes == residual_out || codes == y)))
        return set_error(CSDR_E_INVALID, "add_rms_norm: an output is an input or another output");
    NormArgs a{};
    a.x = x;
    a.residual = residual;
    a.residual_out = residual_out;
    a.y = y;
    a.w = w;
    a.codes = codes;
    a.scales = scales;
    a.x_stride = x_stride ? x_stride : n;
    a.residual_stride = residual_stride ? residual_stride : n;
    a.n = n;
    a.pitch = (int)q8_pitch(n);
    a.eps = eps;
    a.inv_n = 1.0 / n;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const bool xh = dtype == CSDR_F16, rh = residual_dtype == CSDR_F16;
    if (!residual) {
        if (xh) launch_norm<_Float16, _Float16, false>(a, rows, st);
        else launch_norm<float, float, false>(a, rows, st);
    } else if (xh) {
        if (rh) launch_norm<_Float16, _Float16, true>(a, rows, st);
        else launch_norm<_Float16, float, true>(a, rows, st);
    } else {
        if (rh) launch_norm<float, _Float16, true>(a, rows, st);
        else launch_norm<float, float, true>(a, rows, st);
    }
    CSDR_LAUNCH_CHECK("add_rms_norm");
    return CSDR_OK;
}

}  // extern "C"
