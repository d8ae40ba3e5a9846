// q8_rows.hip — rows of values as 8-bit codes with a scale each, from a root-mean-square norm with the
// residual's addition, from values as they are, or from silu(gate) * x; and back to values (gfx950).
//
// A row v: top = max |v|, code = rint(127 v / top) (ties to even), scale = top / 127 in fp32. The codes
// are those of exact arithmetic, so that a code does not depend on the order of a sum or on which kernel
// made it. The norm's 1 / rms is in every value of a row and cancels in its codes: they come from
// t = h w alone, a product of two fp32 numbers that fp64 holds exactly, and one pass over the row gives
// both the sum of squares and top. fp64 runs at the fp32 rate here. 127 t / top is taken as a product
// with the reciprocal (off by 1e-13), and divided only where that lies next to a border. A gated value
// costs an exponential: those are computed in fp32 (off by less than 4e-7 of themselves), and in fp64
// where the code lies next to a border or the value may be the row's largest.
//
// A row that holds a value which is not finite (or whose largest value passes fp32) has the scale NaN
// and codes 0, so it reads as NaN; a row of zeros has the scale 0.
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
constexpr int kMaxRows = (1 << 22) - 1;  // fewer than 2^32 threads a launch

typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// Consecutive values at any alignment of their type.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[kChunk];
};

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

// What a row's threads have to agree on.
struct Row {
    double sum, top;
};

__device__ __forceinline__ uint64_t bits_of(double v) { return __builtin_bit_cast(uint64_t, v); }
__device__ __forceinline__ double of_bits(uint64_t v) { return __builtin_bit_cast(double, v); }
// The larger magnitude; a NaN is larger than any number.
__device__ __forceinline__ double larger(double a, double b) {
    return of_bits(max(bits_of(a), bits_of(b)));
}

// Over the workgroup; `lds` has a Row per wave.
__device__ __forceinline__ Row join(Row r, Row* lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        r.sum += __shfl_xor(r.sum, off, 64);
        r.top = larger(r.top, __shfl_xor(r.top, off, 64));
    }
    const int waves = blockDim.x >> 6;
    if (waves == 1) return r;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = r;
    __syncthreads();
    r = lds[0];
    for (int i = 1; i < waves; ++i) {
        r.sum += lds[i].sum;
        r.top = larger(r.top, lds[i].top);
    }
    return r;
}

// Next to a border between two codes, as a distance of q from a half.
__device__ __forceinline__ bool at_border(double q, double r) { return fabs(fabs(q - r) - 0.5) < 1e-9; }

struct Scale {
    double inv, top;  // 127 / top (0 for rows without codes)
    float value;
};

__device__ __forceinline__ Scale scale_of(double top, double factor) {
    Scale s;
    s.top = top;
    s.value = (float)(top * factor / 127.0);
    const bool fine = s.value < INFINITY;  // (not for a NaN)
    if (!fine) s.value = NAN;
    s.inv = fine && top > 0.0 ? 127.0 / top : 0.0;
    return s;
}

__device__ __forceinline__ int code_of(double t, const Scale& s) {
    const double q = t * s.inv;
    double r = rint(q);
    if (__builtin_expect(at_border(q, r), 0)) r = rint(127.0 * t / s.top);
    return (int)r;
}

__device__ __forceinline__ void store_codes(int8_t* p, const int* c) {
    u2 v = {0, 0};
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i / 4] |= (uint32_t)(c[i] & 255) << (8 * (i % 4));
    *reinterpret_cast<u2*>(p) = v;
}

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
// read twice.
template <typename TX, typename TR, bool RES, int NV>
__global__ __launch_bounds__(kMaxThreads) void norm_kernel(NormArgs a) {
    __shared__ Row lds[kMaxThreads / 64];
    const long long row = blockIdx.x;
    const int step = blockDim.x * kChunk, first = threadIdx.x * kChunk;
    constexpr int N = NV > 0 ? NV : 1;
    float h[N][kChunk];
    double sum = 0.0, top = 0.0;
    TR* out = RES ? static_cast<TR*>(a.residual_out) + row * a.n : nullptr;

    auto take = [&](float* v, int at) {
        float w[kChunk];
        load(a.w + at, a.n - at, w);
        load_h<TX, TR, RES>(a, row, at, v);
        if (RES) store(out + at, a.n - at, v);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            sum = fma((double)v[i], (double)v[i], sum);
            top = larger(top, fabs((double)v[i] * (double)w[i]));
        }
    };
    if (NV > 0) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (first + j * step < a.n) take(h[j], first + j * step);
    } else {
        for (int at = first; at < a.n; at += step) take(h[0], at);
    }
    const Row r = join({sum, top}, lds);
    const double rms = 1.0 / sqrt(r.sum / a.n + (double)a.eps);
    // (a finite top beside a sum that is not: a weight of 0 under a value that is not finite)
    const Scale s = scale_of(r.sum < INFINITY ? r.top : (double)NAN, rms);
    if (threadIdx.x == 0 && a.scales) a.scales[row] = s.value;

    auto put = [&](const float* v, int at) {
        float w[kChunk];
        load(a.w + at, a.n - at, w);
        if (a.codes) {
            int c[kChunk];
#pragma unroll
            for (int i = 0; i < kChunk; ++i) c[i] = code_of((double)v[i] * (double)w[i], s);
            store_codes(a.codes + row * a.pitch + at, c);
        }
        if (a.y && at < a.n) {
            float y[kChunk];
#pragma unroll
            for (int i = 0; i < kChunk; ++i) y[i] = (float)((double)v[i] * rms * (double)w[i]);
            store(static_cast<TX*>(a.y) + row * a.n + at, a.n - at, y);
        }
    };
    const int end = a.codes ? a.pitch : a.n;
    if (NV > 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = first + j * step;
            if (at >= a.n) {
#pragma unroll
                for (int i = 0; i < kChunk; ++i) h[j][i] = 0.0f;
            }
            if (at < end) put(h[j], at);
        }
    } else {
        for (int at = first; at < end; at += step) {
            // (where the stream is updated in place its old values are gone: the sums are read back)
            if (RES) load(out + at, a.n - at, h[0]);
            else load_h<TX, TR, RES>(a, row, at, h[0]);
            put(h[0], at);
        }
    }
}

// ------------------------------------------------------------------ rows as they are, or gated

struct RowsArgs {
    const void *x, *gate;
    int8_t* codes;
    float* scales;
    long long x_stride, gate_stride;
    int n, pitch;
};

// How far a gated value computed in fp32 may be off, of itself, and its code, with both to spare.
constexpr float kGatedOff = 2e-6f, kCodeOff = 2e-4f;
// In fp64 throughout: rows whose largest value is below kTiny, whose smaller ones fp32 holds with few
// bits or none; values whose gate is below kLow, where the exponential passes fp32.
constexpr float kTiny = 1e-30f, kLow = -88.0f;

__device__ __forceinline__ float gated(float g, float x) { return g / (1.0f + expf(-g)) * x; }
__device__ __forceinline__ double gated(double g, double x) { return g / (1.0 + exp(-g)) * x; }

template <typename T, bool GATE, int NV>
__global__ __launch_bounds__(kMaxThreads) void rows_kernel(RowsArgs a) {
    __shared__ Row lds[kMaxThreads / 64];
    __shared__ unsigned long long exact_top;
    const long long row = blockIdx.x;
    const int step = blockDim.x * kChunk, first = threadIdx.x * kChunk;
    constexpr int N = NV > 0 ? NV : 1;
    float x[N][kChunk], g[N][GATE ? kChunk : 1];
    const T* px = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* pg = static_cast<const T*>(a.gate) + row * a.gate_stride;
    uint32_t most = 0;  // bits of the largest magnitude; a NaN's are larger than any number's

    auto take = [&](float* v, float* u, int at) {
        load(px + at, a.n - at, v);
        if (GATE) load(pg + at, a.n - at, u);
    };
    auto value = [&](const float* v, const float* u, int i) { return GATE ? gated(u[i], v[i]) : v[i]; };
    auto look = [&](const float* v, const float* u) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
            most = max(most, __float_as_uint(value(v, u, i)) & 0x7FFFFFFFu);
    };
    if (NV > 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = first + j * step;
            if (at < a.n) {
                take(x[j], g[j], at);
                look(x[j], g[j]);
            }
        }
    } else {
        for (int at = first; at < a.n; at += step) {
            take(x[0], g[0], at);
            look(x[0], g[0]);
        }
    }
    if (GATE && threadIdx.x == 0) exact_top = 0;
    const Row r = join({0.0, (double)__uint_as_float(most)}, lds);
    const float top32 = (float)r.top;
    double top = r.top;
    const bool tiny = GATE && top32 < kTiny;
    if (GATE) {
        if (blockDim.x <= 64) __syncthreads();  // (else join has had one)
        auto check = [&](const float* v, const float* u) {
#pragma unroll
            for (int i = 0; i < kChunk; ++i)
                if (fabsf(value(v, u, i)) >= top32 * (1.0f - kGatedOff) || u[i] < kLow || tiny)
                    atomicMax(&exact_top, (unsigned long long)bits_of(fabs(
                                              gated((double)u[i], (double)v[i]))));
        };
        if (NV > 0) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (first + j * step < a.n) check(x[j], g[j]);
        } else {
            for (int at = first; at < a.n; at += step) {
                take(x[0], g[0], at);
                check(x[0], g[0]);
            }
        }
        __syncthreads();
        if (r.top < INFINITY) top = of_bits(exact_top);
    }
    const Scale s = scale_of(top, 1.0);
    if (threadIdx.x == 0) a.scales[row] = s.value;
    const float inv32 = (float)s.inv;

    auto put = [&](const float* v, const float* u, int at) {
        int c[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            if (GATE) {
                const float q = value(v, u, i) * inv32, f = rintf(q);
                c[i] = (int)f;
                if (__builtin_expect(fabsf(fabsf(q - f) - 0.5f) < kCodeOff || u[i] < kLow || tiny, 0))
                    c[i] = s.inv > 0.0 ? code_of(gated((double)u[i], (double)v[i]), s) : 0;
            } else {
                c[i] = code_of((double)v[i], s);
            }
            if (!(s.inv > 0.0)) c[i] = 0;
        }
        store_codes(a.codes + row * a.pitch + at, c);
    };
    if (NV > 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = first + j * step;
            if (at >= a.n) {
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    x[j][i] = 0.0f;
                    if (GATE) g[j][i] = 0.0f;
                }
            }
            if (at < a.pitch) put(x[j], g[j], at);
        }
    } else {
        for (int at = first; at < a.pitch; at += step) {
            take(x[0], g[0], at);
            put(x[0], g[0], at);
        }
    }
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

// Threads of a row and chunks a thread (0: more than four, which the registers do not hold).
struct Shape {
    int threads, nv;
};
Shape shape_of(int width) {
    const int chunks = (width + kChunk - 1) / kChunk;
    Shape s;
    s.threads = std::min(256, (chunks + 63) / 64 * 64);
    if (chunks > 4 * 256) s.threads = std::min(kMaxThreads, (chunks / 4 + 63) / 64 * 64);
    const int nv = (chunks + s.threads - 1) / s.threads;
    s.nv = nv <= 1 ? 1 : nv == 2 ? 2 : nv <= 4 ? 4 : 0;
    return s;
}

template <typename TX, typename TR, bool RES>
void launch_norm(const NormArgs& a, int rows, hipStream_t st) {
    const Shape s = shape_of(a.codes ? a.pitch : a.n);
    if (s.nv == 1) norm_kernel<TX, TR, RES, 1><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 2) norm_kernel<TX, TR, RES, 2><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 4) norm_kernel<TX, TR, RES, 4><<<rows, s.threads, 0, st>>>(a);
    else norm_kernel<TX, TR, RES, 0><<<rows, s.threads, 0, st>>>(a);
}

template <typename T, bool GATE>
void launch_rows(const RowsArgs& a, int rows, hipStream_t st) {
    const Shape s = shape_of(a.pitch);
    if (s.nv == 1) rows_kernel<T, GATE, 1><<<rows, s.threads, 0, st>>>(a);
    else if (s.nv == 2) rows_kernel<T, GATE, 2><<<rows, s.threads, 0, st>>>(a);
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
