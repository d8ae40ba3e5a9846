// q8_linear.hip — products of 8-bit rows on the integer matrix cores (gfx950):
//   y[m][r] = x_scales[m] * w_scales[r] * sum_c x[m][c] w[r][c] (+ bias[r]) (+ add[m][r])
// The sums are exact (32-bit integers), so no order of summation shows in the result: it is rounded as
// a sum is converted to fp32, by two products and the additions in fp32, and once to y's type.
#include <hip/hip_runtime.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

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
    bool wide;  // four outputs at a multiple of four may be moved at once
};

template <typename T>
struct Four;
template <>
struct Four<float> {
    typedef float type __attribute__((ext_vector_type(4)));
};
template <>
struct Four<_Float16> {
    typedef _Float16 type __attribute__((ext_vector_type(4)));
};
typedef float f4 __attribute__((ext_vector_type(4)));

// The scales and biases of four neighbouring rows of w (the last one's again where there are fewer).
__device__ __forceinline__ f4 four_of(const float* p, int r, int R) {
    f4 v;
    if (r + 3 < R) __builtin_memcpy(&v, p + r, 16);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[min(r + i, R - 1)];
    return v;
}

__device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) {
    return (float)sum * xs * ws + bias;
}

// Four neighbouring outputs of a token at once (a.wide, r + 3 < R, m < M).
template <typename T>
__device__ __forceinline__ void finish_wide(const Args& a, int m, int r, const i4& sum, float xs, const f4& ws,
                                            const f4& bias, const typename Four<T>::type& add) {
    typename Four<T>::type o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (T)(scaled(sum[i], xs, ws[i], bias[i]) + (float)add[i]);
    *reinterpret_cast<typename Four<T>::type*>(static_cast<T*>(a.y) + m * a.y_stride + r) = o;
}
template <typename T>
__device__ __forceinline__ typename Four<T>::type wide_added(const Args& a, int m, int r) {
    using V = typename Four<T>::type;
    return *reinterpret_cast<const V*>(static_cast<const T*>(a.add) + m * a.add_stride + r);
}

// One by one, as many of them as there are.
template <typename T>
__device__ __forceinline__ void finish(const Args& a, int m, int r, const i4& sum, float xs, const f4& ws,
                                       const f4& bias) {
    if (m >= a.M) return;
    T* y = static_cast<T*>(a.y) + m * a.y_stride + r;
    const T* add = static_cast<const T*>(a.add) + m * a.add_stride + r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r + i < a.R)
            y[i] = (T)(scaled(sum[i], xs, ws[i], bias[i]) + (a.add ? (float)add[i] : 0.0f));
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
        const int m = m0 + 16 * j + (l & 15), r = r0 + 4 * (l >> 4);
        const int rc = min(r, a.R - 1), mc = min(m, a.M - 1);
        const float xs = a.x_scales[mc];
        const f4 ws = four_of(a.w_scales, rc, a.R), bias = a.bias ? four_of(a.bias, rc, a.R) : f4{};
        if (!a.wide || r + 3 >= a.R) finish<T>(a, m, r, sum, xs, ws, bias);
        else if (m < a.M)
            finish_wide<T>(a, m, r, sum, xs, ws, bias,
                           a.add ? wide_added<T>(a, m, r) : typename Four<T>::type{});
    }
}

// ------------------------------------------------------------------ tiles through LDS

typedef __attribute__((address_space(3))) void* LdsPtr;

// TR rows of w times TM tokens a workgroup, in WR x WM waves. A step is 128 columns; its rows lie in LDS 128
// bytes apart, 16-byte chunk c of row i at c ^ (i % 8), so that the 16 rows of an operand's chunk fall on
// different banks.
template <int TR, int TM, int WR, int WM>
struct Tile {
    static constexpr int kWaves = WR * WM, kThreads = 64 * kWaves;
    static constexpr int FR = TR / WR / 16, FM = TM / WM / 16;  // operands of a wave
    static constexpr int kBytes = (TR + TM) * 128;              // a step's
    static constexpr int kPieces = kBytes / 1024 / kWaves;      // 1 KB loads a wave
    static constexpr int kLds = 2 * kBytes;
    // through how many parts of the LDS a wave's sums go
    static constexpr int kPasses = TR * TM * 4 > kLds ? 2 : 1;
    static_assert(TR * TM * 4 <= kLds * kPasses, "sums of a pass");
};

constexpr int kRsrc = 0x00027000;  // a raw buffer

// This wave's loads into LDS have arrived and its reads are done; then every wave's.
__device__ __forceinline__ void arrived() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// sum += w . x. Written out so that the sums stay where they are: from the builtin the compiler gives results
// other registers than their operands, and with all 256 accumulator registers in use copies them about in every
// step. The next product of the same sum is (FR FM - 1) products away; the last ones are builtins, so that the
// compiler knows what to wait for before it reads a sum.
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass knows no such registers)
__device__ __forceinline__ void product(i4& sum, const i4& w, const i4& x) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(sum) : "v"(w), "v"(x));
}
#endif

template <typename T, int TR, int TM, int WR, int WM>
__global__ __launch_bounds__(64 * WR * WM) void tile_kernel(Args a, int tiles_r, int tiles_m) {
#ifdef __HIP_DEVICE_COMPILE__
    using S = Tile<TR, TM, WR, WM>;
    constexpr int FR = S::FR, FM = S::FM, NP = S::kPieces, NW = TR / (8 * S::kWaves);
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroups go to the eight XCDs in turn: each XCD takes a run of tiles, eight columns of tokens by
    // as many rows as it has, so that its L2 serves what they share.
    int tr, tm;
    {
        const int n = tiles_r * tiles_m, b = blockIdx.x, per = n / 8, rest = n % 8;
        const int xcd = b % 8;
        const int t = xcd * per + min(xcd, rest) + b / 8;
        const int group = t / (8 * tiles_r), width = min(8, tiles_m - 8 * group);
        const int in = t - group * 8 * tiles_r;
        tr = in / width;
        tm = 8 * group + in % width;
    }
    const int r0 = tr * TR, m0 = tm * TM;

    // the lane's part of the wave's loads: 8 rows of a piece (the last row again where there are fewer), its
    // chunk as the row's key says
    static_assert(TR % (8 * S::kWaves) == 0, "a piece is of one operand");
    const auto wb = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (long long)r0 * a.pitch), 0, -1, kRsrc);
    const auto xb = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + (long long)m0 * a.pitch), 0, -1, kRsrc);
    int off[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int row = (i * S::kWaves + wave) * 8 + (lane >> 3);
        const int in = i < NW ? min(row, a.R - 1 - r0) : min(row - TR, a.M - 1 - m0);
        off[i] = in * a.pitch + 16 * ((lane & 7) ^ (lane >> 3));
    }
    // piece i of a step, into buffer `buf`
    auto fetch = [&](int i, int buf, int step) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            i < NW ? wb : xb, (LdsPtr)(lds + buf * S::kBytes + (i * S::kWaves + wave) * 1024), 16, off[i],
            step * 128, 0, 0);
    };
    const int steps = a.pitch / 128;
#pragma unroll
    for (int i = 0; i < NP; ++i) fetch(i, 0, 0);
    if (steps > 1) {
#pragma unroll
        for (int i = 0; i < NP; ++i) fetch(i, 1, 1);
    }
    const int wr = wave / WM, wm = wave % WM;
    const int at = (lane & 15) * 128 + 16 * ((lane >> 4) ^ (lane & 7));
    const int at_w = wr * FR * 2048 + at, at_x = TR * 128 + wm * FM * 2048 + at;
    i4 wf[2][FR], xf[2][FM];
    // operand f of half a step
    auto read = [&](int f, int half, int buf) {
        const int8_t* base = lds + buf * S::kBytes;
        if (f < FM) xf[half][f] = *reinterpret_cast<const i4*>(base + (at_x ^ (64 * half)) + f * 2048);
        else wf[half][f - FM] = *reinterpret_cast<const i4*>(base + (at_w ^ (64 * half)) + (f - FM) * 2048);
    };
    i4 acc[FR][FM] = {};
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) asm volatile("" : "+a"(acc[i][j]));  // (zero while the first loads run)
    constexpr int NF = FR + FM, N = FR * FM;
    // The products of half a step, with the reads of the next half's operands (NR of them) and loads (NL) spread
    // over the first three quarters of them.
    auto multiply = [&](int half, auto nr, int read_buf, auto nl, int load_buf, int load_step) {
        constexpr int NR = decltype(nr)::value, NL = decltype(nl)::value, MOST = NR > NL ? NR : NL;
        constexpr int EACH = MOST == 0 ? N : N * 3 / 4 / MOST > 0 ? N * 3 / 4 / MOST : 1;
        static_assert(MOST <= N, "more reads than products");
        asm volatile("s_nop 1");  // (registers written just before a product written out need two states)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            // (behind a product: the first one's wait for its operands is not one for these reads)
            product(acc[k / FM][k % FM], wf[half][k / FM], xf[half][k % FM]);
            if (k % EACH == 0) {
                if (k / EACH < NL) fetch(k / EACH, load_buf, load_step);
                if (k / EACH < NR) read(k / EACH, half ^ 1, read_buf);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // A step: the products of its first half while the second half's operands are read; then every wave is
    // done with the step's buffer and the next step has arrived in the other one: the products of the second
    // half while the step after next is fetched into the buffer and the next one's first operands are read.
    using Reads = std::integral_constant<int, NF>;
    using Loads = std::integral_constant<int, NP>;
    using None = std::integral_constant<int, 0>;
    auto step = [&](int s, auto loads) {
        const int cur = s & 1;
        multiply(0, Reads(), cur, None(), 0, 0);
        arrived();
        multiply(1, Reads(), cur ^ 1, loads, cur, s + 2);
    };
    arrived();
#pragma unroll
    for (int f = 0; f < NF; ++f) read(f, 0, 0);
    for (int s = 0; s < steps - 2; ++s) step(s, Loads());
    if (steps > 1) step(steps - 2, None());
    multiply(0, Reads(), (steps - 1) & 1, None(), 0, 0);
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[1][i], xf[1][j], acc[i][j], 0, 0, 0);
    // Each wave turns its sums through its part of the LDS, `TOKENS` tokens at a time (token-major, 16-byte chunk c
    // of token m at c ^ (m % 8)): a lane then has neighbouring rows for whole lines of y, and a short loop writes
    // them, where straight code over the registers was 40 KB of instructions that came from memory at each launch
    // (14 us of a launch, 3 with the loop).
    constexpr int CHUNKS = TR / WR / 4, PASSES = S::kPasses, TOKENS = TM / WM / PASSES;
    constexpr int PER = 64 / CHUNKS;  // tokens at once
    constexpr int BATCH = TOKENS / PER < 16 ? TOKENS / PER : 16;
    using V = typename Four<T>::type;
    i4* part = reinterpret_cast<i4*>(lds) + wave * (TOKENS * CHUNKS);
    const int c = lane % CHUNKS, mine = lane / CHUNKS;
    const int r = r0 + wr * (TR / WR) + 4 * c;
    const f4 ws = four_of(a.w_scales, min(r, a.R - 1), a.R);
    const f4 bias = a.bias ? four_of(a.bias, min(r, a.R - 1), a.R) : f4{};
    const bool whole = a.wide && r + 3 < a.R;
    arrived();  // every wave is done with the tiles
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
#pragma unroll
        for (int j = 0; j < TOKENS / 16; ++j)
#pragma unroll
            for (int i = 0; i < FR; ++i) {
                const int m = 16 * j + (lane & 15);
                part[m * CHUNKS + ((4 * i + (lane >> 4)) ^ (m & 7))] = acc[i][p * (TOKENS / 16) + j];
            }
        const int first = m0 + wm * (TM / WM) + p * TOKENS + mine;
        auto sum_of = [&](int k) { return part[(k + mine) * CHUNKS + (c ^ ((k + mine) & 7))]; };
        if (whole) {
#pragma unroll 1
            for (int k = 0; k < TOKENS; k += BATCH * PER) {
                float xs[BATCH];
                V add[BATCH] = {};
#pragma unroll
                for (int q = 0; q < BATCH; ++q) {
                    const int m = min(first + k + q * PER, a.M - 1);
                    xs[q] = a.x_scales[m];
                    if (a.add) add[q] = wide_added<T>(a, m, r);
                }
#pragma unroll
                for (int q = 0; q < BATCH; ++q)
                    if (first + k + q * PER < a.M)
                        finish_wide<T>(a, first + k + q * PER, r, sum_of(k + q * PER), xs[q], ws, bias, add[q]);
            }
        } else if (r < a.R) {
#pragma unroll 1
            for (int k = 0; k < TOKENS; k += PER)
                finish<T>(a, first + k, r, sum_of(k), a.x_scales[min(first + k, a.M - 1)], ws, bias);
        }
    }
#endif
}

template <typename T, int TR, int TM, int WR, int WM>
void launch_tiles(const Args& a, hipStream_t st) {
    using S = Tile<TR, TM, WR, WM>;
    auto kernel = tile_kernel<T, TR, TM, WR, WM>;
    if constexpr (S::kLds > 65536) {  // beyond the default: allowed once per device
        static std::atomic<uint64_t> allowed{0};
        int dev = 0;
        (void)hipGetDevice(&dev);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (!(allowed.load(std::memory_order_relaxed) & bit)) {
            (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds);
            allowed.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const int tiles_r = (a.R + TR - 1) / TR, tiles_m = (a.M + TM - 1) / TM;
    kernel<<<(unsigned)(tiles_r * tiles_m), S::kThreads, S::kLds, st>>>(a, tiles_r, tiles_m);
}

template <typename T>
void launch(const Args& a, hipStream_t st) {
    const unsigned rows = (unsigned)((a.R + 15) / 16);
    if (a.M <= 16) rows16_kernel<T, 1, 8><<<dim3(rows, 1), 512, 0, st>>>(a);
    else if (a.M > 64) {
        const char* e = getenv("TILE");
        const int t = e ? atoi(e) : 0;
        if (t == 0) launch_tiles<T, 256, 256, 2, 2>(a, st);
        else if (t == 1) launch_tiles<T, 256, 128, 2, 2>(a, st);
        else if (t == 2) launch_tiles<T, 128, 128, 2, 2>(a, st);
        else if (t == 3) launch_tiles<T, 64, 64, 2, 2>(a, st);
        else if (t == 4) launch_tiles<T, 128, 64, 2, 2>(a, st);
        else if (t == 5) launch_tiles<T, 64, 128, 2, 2>(a, st);
        else if (t == 6) launch_tiles<T, 128, 256, 2, 2>(a, st);
        else if (t == 7) rows16_kernel<T, 4, 8><<<dim3(rows, (a.M + 63) / 64), 512, 0, st>>>(a);
    }
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
    const size_t four = y_dtype == CSDR_F32 ? 16 : 8;
    a.wide = a.y_stride % 4 == 0 && reinterpret_cast<uintptr_t>(y) % four == 0 &&
             (!add || (a.add_stride % 4 == 0 && reinterpret_cast<uintptr_t>(add) % four == 0));
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (y_dtype == CSDR_F32) launch<float>(a, st);
    else launch<_Float16>(a, st);
    CSDR_LAUNCH_CHECK("q8_linear");
    return CSDR_OK;
}

}  // extern "C"
