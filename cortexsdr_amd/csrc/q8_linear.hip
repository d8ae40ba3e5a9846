// q8_linear.hip — products of 8-bit rows on the integer matrix cores (gfx950):
//   y[m][r] = x_scales[m] * w_scales[r] * sum_c x[m][c] w[r][c] (+ bias[r]) (+ add[m][r])
// The sums are exact (32-bit integers), so no order of summation shows in the result: it is rounded as
// a sum is converted to fp32, by two products and the additions in fp32, and once to y's type.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "q8.hpp"

namespace {

using csdr::kMaxWidth;
using csdr::q8_pitch;
using csdr::set_error;

typedef int i4 __attribute__((ext_vector_type(4)));

struct Args {
    const int8_t *w, *x;
    const float *w_scales, *x_scales, *bias;
    const void* add;
    void* y;
    long long y_stride, add_stride;
    int R, M, pitch;
};

// Four neighbouring outputs of a token, as many of them as there are.
template <typename T>
__device__ __forceinline__ void finish(const Args& a, int m, int r, const i4& sum) {
    if (m >= a.M || r >= a.R) return;
    const float xs = a.x_scales[m];
    const int n = min(4, a.R - r);
    T* y = static_cast<T*>(a.y) + m * a.y_stride + r;
    const T* add = static_cast<const T*>(a.add) + m * a.add_stride + r;
    for (int i = 0; i < n; ++i) {
        float v = (float)sum[i] * xs * a.w_scales[r + i];
        if (a.bias) v += a.bias[r + i];
        if (a.add) v += csdr::to_f32(add[i]);
        y[i] = (T)v;
    }
}

// 16 rows of w times 16 MT tokens; the waves take steps of 64 columns in turn and add up through LDS.
// w and x come from memory straight into the operands: lane l holds row l % 16, columns 16 (l / 16) and
// on of a step (both operands alike, so their order within a step does not matter).
template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void rows16_kernel(Args a) {
    __shared__ i4 part[WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
    const long long at = 16 * (lane >> 4);
    const int8_t* w = a.w + (long long)min(r0 + (lane & 15), a.R - 1) * a.pitch + at;
    const int8_t* x[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j)
        x[j] = a.x + (long long)min(m0 + 16 * j + (lane & 15), a.M - 1) * a.pitch + at;
    i4 acc[MT] = {};
    const int steps = a.pitch / 64;
#pragma unroll 4
    for (int s = wave; s < steps; s += WAVES) {
        const i4 wv = *reinterpret_cast<const i4*>(w + 64 * s);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const i4 xv = *reinterpret_cast<const i4*>(x[j] + 64 * s);
            acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xv, acc[j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    // D: lane l holds rows 4 (l / 16) and on, column l % 16
    for (int i = threadIdx.x; i < MT * 64; i += WAVES * 64) {
        const int j = i >> 6, l = i & 63;
        i4 sum = part[0][j][l];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) sum += part[k][j][l];
        finish<T>(a, m0 + 16 * j + (l & 15), r0 + 4 * (l >> 4), sum);
    }
}

template <typename T>
void launch(const Args& a, hipStream_t st) {
    const unsigned rows = (unsigned)((a.R + 15) / 16);
    if (a.M <= 16) rows16_kernel<T, 1, 8><<<dim3(rows, 1), 512, 0, st>>>(a);
    else rows16_kernel<T, 4, 8><<<dim3(rows, (a.M + 63) / 64), 512, 0, st>>>(a);
}

}  // namespace

extern "C" {

CSDR_API int csdr_q8_linear(const int8_t* w, const float* w_scales, int R, const int8_t* x,
                            const float* x_scales, int M, int C, const float* bias, const void* add,
                            int64_t add_stride, void* y, int y_dtype, int64_t y_stride,
                            void* hip_stream) {
    if (!w || !w_scales || !x || !x_scales || !y)
        return set_error(CSDR_E_INVALID, "q8_linear: a pointer is NULL");
    if (R <= 0 || M <= 0 || C <= 0) return set_error(CSDR_E_INVALID, "q8_linear: bad sizes");
    if (C > kMaxWidth)
        return set_error(CSDR_E_UNSUPPORTED, "q8_linear: more than 131071 columns");
    if (y_dtype != CSDR_F32 && y_dtype != CSDR_F16)
        return set_error(CSDR_E_INVALID, "q8_linear: y_dtype must be CSDR_F32 or CSDR_F16");
    if (M > (1 << 22) - 1 || R > INT_MAX - 256)
        return set_error(CSDR_E_INVALID, "q8_linear: more than 2^22 - 1 tokens or 2^31 - 257 rows");
    if ((y_stride != 0 && y_stride < R) || (add && add_stride != 0 && add_stride < R))
        return set_error(CSDR_E_INVALID, "q8_linear: a row stride is below R");
    if (add == y && M > 1 && (add_stride ? add_stride : R) != (y_stride ? y_stride : R))
        return set_error(CSDR_E_INVALID, "q8_linear: in place add and y must have the same stride");
    if (reinterpret_cast<uintptr_t>(w) % 16 || reinterpret_cast<uintptr_t>(x) % 16)
        return set_error(CSDR_E_INVALID, "q8_linear: codes must be 16-byte aligned");
    Args a{};
    a.w = w;
    a.x = x;
    a.w_scales = w_scales;
    a.x_scales = x_scales;
    a.bias = bias;
    a.add = add;
    a.y = y;
    a.y_stride = y_stride ? y_stride : R;
    a.add_stride = add_stride ? add_stride : R;
    a.R = R;
    a.M = M;
    a.pitch = (int)q8_pitch(C);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (y_dtype == CSDR_F32) launch<float>(a, st);
    else launch<_Float16>(a, st);
    CSDR_LAUNCH_CHECK("q8_linear");
    return CSDR_OK;
}

}  // extern "C"
