// logprobs.hip — log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits (gfx950).
//
//   y = x / temperature; Z = sum exp(y - m); logprob_t = y_t - m - log Z
//   entropy = log Z - sum exp(y - m) (y - m) / Z
// The order of the top: larger y first, among equals the lower id.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"

namespace {

using csdr::set_error;

constexpr int kThreads = 256;
constexpr int kMaxTop = 64;

struct Args {
    const void* x;
    int n;
    long long stride;
    float inv_t;
    const int32_t* tokens;
    float *logprobs, *entropy, *top_logprobs;
    int32_t* top_ids;
    int top_n;
};

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = csdr::wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < kThreads / 64; ++i) s += red[i];
    return s;
}

// The better of two (value, id) by the top's order.
__device__ __forceinline__ void better(float& v, int& i, float v2, int i2) {
    if (i2 >= 0 && (i < 0 || v2 > v || (v2 == v && i2 < i))) {
        v = v2;
        i = i2;
    }
}

__device__ __forceinline__ void block_best(float& v, int& i, float* rv, int* ri) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float v2 = __shfl_xor(v, off, 64);
        const int i2 = __shfl_xor(i, off, 64);
        better(v, i, v2, i2);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        rv[threadIdx.x >> 6] = v;
        ri[threadIdx.x >> 6] = i;
    }
    __syncthreads();
    v = rv[0];
    i = ri[0];
    for (int w = 1; w < kThreads / 64; ++w) better(v, i, rv[w], ri[w]);
}

template <typename XT>
__global__ __launch_bounds__(kThreads) void row_kernel(Args a) {
    __shared__ float rv[kThreads / 64];
    __shared__ int ri[kThreads / 64];
    const int row = blockIdx.x;
    const XT* x = static_cast<const XT*>(a.x) + (long long)row * a.stride;
    float m = -INFINITY;
    int mi = -1;
    bool bad = false;
    for (int i = threadIdx.x; i < a.n; i += kThreads) {
        const float y = (float)x[i] * a.inv_t;
        if (!(y < INFINITY)) bad = true;
        else if (y > -INFINITY) better(m, mi, y, i);
    }
    block_best(m, mi, rv, ri);
    bad = __syncthreads_or(bad);
    float z = 0.0f, w = 0.0f;
    for (int i = threadIdx.x; i < a.n; i += kThreads) {
        const float y = (float)x[i] * a.inv_t;
        if (!(y > -INFINITY && y < INFINITY)) continue;
        const float d = y - m, e = expf(d);
        z += e;
        w = fmaf(e, d, w);
    }
    z = block_sum(z, rv);
    w = block_sum(w, rv);
    const float lz = bad ? NAN : mi < 0 ? 0.0f : logf(z);
    if (threadIdx.x == 0) {
        if (a.entropy) a.entropy[row] = mi < 0 ? lz : lz - w / z;
        if (a.tokens) {
            const int t = a.tokens[row];
            float lp = t < 0 ? 0.0f : NAN;
            if (t >= 0 && t < a.n) {
                const float y = (float)x[t] * a.inv_t;
                lp = bad ? NAN : y == -INFINITY ? y : y - m - lz;
            }
            a.logprobs[row] = lp;
        }
    }
    float lv = m;
    int li = mi;
    for (int k = 0; k < a.top_n; ++k) {
        if (threadIdx.x == 0) {
            a.top_ids[(long long)row * a.top_n + k] = li;
            a.top_logprobs[(long long)row * a.top_n + k] = li < 0 ? -INFINITY : lv - m - lz;
        }
        if (li < 0) continue;
        float v = -INFINITY;
        int vi = -1;
        for (int i = threadIdx.x; i < a.n; i += kThreads) {
            const float y = (float)x[i] * a.inv_t;
            if (!(y > -INFINITY && y < INFINITY)) continue;
            if (y < lv || (y == lv && i > li)) better(v, vi, y, i);
        }
        block_best(v, vi, rv, ri);
        lv = v;
        li = vi;
    }
}

}  // namespace

extern "C" {

CSDR_API size_t csdr_token_logprobs_workspace_bytes(int rows, int n, int top_n) {
    (void)rows, (void)n, (void)top_n;
    return 0;
}

CSDR_API int csdr_token_logprobs(const void* logits, int dtype, int rows, int n,
                                 int64_t row_stride, float temperature, const int32_t* tokens,
                                 float* logprobs, float* entropy, int top_n, int32_t* top_ids,
                                 float* top_logprobs, void* workspace, size_t workspace_bytes,
                                 void* hip_stream) {
    (void)workspace, (void)workspace_bytes;
    if (!logits || rows <= 0 || n <= 0)
        return set_error(CSDR_E_INVALID, "token_logprobs: bad argument");
    if (dtype != CSDR_F32 && dtype != CSDR_F16)
        return set_error(CSDR_E_INVALID, "token_logprobs: dtype must be CSDR_F32 or CSDR_F16");
    if (top_n < 0 || top_n > kMaxTop)
        return set_error(CSDR_E_UNSUPPORTED, "token_logprobs: top_n must be 0 to 64");
    if ((tokens != nullptr) != (logprobs != nullptr) ||
        (top_n > 0 && (!top_ids || !top_logprobs)))
        return set_error(CSDR_E_INVALID, "token_logprobs: a pointer is NULL");
    if (row_stride != 0 && row_stride < n)
        return set_error(CSDR_E_INVALID, "token_logprobs: the row stride is below n");
    if (!(temperature < INFINITY) || temperature == -INFINITY)
        return set_error(CSDR_E_INVALID, "token_logprobs: the temperature is not finite");
    Args a{logits, n, row_stride ? row_stride : n, temperature > 0.0f ? 1.0f / temperature : 1.0f,
           tokens, logprobs, entropy, top_logprobs, top_ids, top_n};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (dtype == CSDR_F32) row_kernel<float><<<rows, kThreads, 0, st>>>(a);
    else row_kernel<_Float16><<<rows, kThreads, 0, st>>>(a);
    CSDR_LAUNCH_CHECK("token_logprobs");
    return CSDR_OK;
}

}  // extern "C"
