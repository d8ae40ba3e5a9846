// q8_linear.hip — products of 8-bit rows on the integer matrix cores (gfx950):
//   y[m][r] = x_scales[m] * w_scales[r] * sum_c x[m][c] w[r][c] (+ bias[r]) (+ add[m][r])
// The sums are exact (32-bit integers), so no order of summation shows in the result: it is rounded as a sum is
// converted to fp32, by two products and the additions in fp32, and once to y's type.
//
// One kernel, seven tiles. Rows of codes come from memory straight into LDS (no register, no instruction of the
// waves between), several stages ahead; a wave reads its operands for the next half step while the matrix cores
// work on this one, with one barrier a stage. What bounds it, by the number of tokens (times of launches in a
// graph):
//   one to 16    the stream of the weights: 22016 x 4096 for one token 18 us with them in the Infinity Cache, 23 us (3.9
//                TB/s) where 720 MB of them are read in turn; small ones the chain of a launch, first loads,
//                barrier, sums (1152 x 896 2.9 us)
//   up to some   reads of L2: 12 to 14 TB/s over a launch with its start and end, seven tenths of them hits or more,
//   hundreds     the matrix cores busy in a tenth to a quarter of the time: 64 tokens, 4096 x 11008, 13 us (18 with
//                540 MB of weights in turn); there large tiles take fewer bytes and leave CUs without work, so tiles
//                are chosen by what they cost (kCosts)
//   thousands    the matrix cores at the clock that they can be fed at: 4096 tokens, 4096 x 11008, 135 us, 2.74
//                POPS, busy in 68% of the cycles counted around a launch (nothing but the products runs at 1.9
//                GHz, 3.9 POPS; taking the same rows for every tile, so that all loads hit L2, changes nothing, nor
//                does the order of loads, reads and products, nor the waves' priority); 12 us of it start and end,
//                67 MB of y and `add`
#include <hip/hip_runtime.h>

#include <algorithm>
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
};

// Four neighbouring values at any alignment of their type.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T v[4];
};
typedef float f4 __attribute__((ext_vector_type(4)));

// The scales and biases of four neighbouring rows of w (the last one's again where there are fewer).
[[maybe_unused]] __device__ __forceinline__ f4 four_of(const float* p, int r, int R) {
    f4 v;
    if (r + 3 < R) __builtin_memcpy(&v, p + r, 16);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[min(r + i, R - 1)];
    return v;
}

// A sum times both scales. With a channel's scale below kLarge first the product passes fp32 in no sum (at most 2^31)
// and, as a whole number of the scale's last place, loses nothing below the normal numbers; from there on the token's
// scale goes first, and where that product passes fp32 the result does.
constexpr float kLarge = 0x1p96f;
[[maybe_unused]] __device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) {
    return (float)sum * ws * xs + bias;
}

// Four neighbouring outputs of a token at once (r + 3 < R, m < M, no large scale among theirs).
template <typename T>
__device__ __forceinline__ void finish_four(const Args& a, int m, int r, const i4& sum, float xs, const f4& ws,
                                            const f4& bias, const Four<T>& add) {
    Four<T> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = (T)(scaled(sum[i], xs, ws[i], bias[i]) + (float)add.v[i]);
    *reinterpret_cast<Four<T>*>(static_cast<T*>(a.y) + m * a.y_stride + r) = o;
}

// One by one, as many of them as there are, with any scales.
template <typename T>
__device__ __forceinline__ void finish(const Args& a, int m, int r, const i4& sum, float xs, const f4& ws,
                                       const f4& bias) {
    if (m >= a.M) return;
    T* y = static_cast<T*>(a.y) + m * a.y_stride + r;
    const T* add = static_cast<const T*>(a.add) + m * a.add_stride + r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r + i < a.R) {
            const bool large = fabsf(ws[i]) >= kLarge;
            y[i] = (T)(scaled(sum[i], large ? ws[i] : xs, large ? xs : ws[i], bias[i]) + (a.add ? (float)add[i] : 0.0f));
        }
}

typedef __attribute__((address_space(3))) void* LdsPtr;

// TR rows of w times TM tokens a workgroup, in WR x WM waves. A step is 128 columns; its rows lie in LDS 128
// bytes apart, 16-byte chunk c of row i at c ^ (i % 8), so that the 16 rows of an operand's chunk fall on
// different banks. KG groups of waves take a step each of a stage's KG and add up at the end; NBUF stages are
// in LDS or on their way.
template <int TR, int TM, int KG, int WR, int WM, int NBUF>
struct Tile {
    static constexpr int kWaves = KG * WR * WM, kThreads = 64 * kWaves;
    static constexpr int FR = TR / WR / 16, FM = TM / WM / 16;  // operands of a wave
    static constexpr int kGroup = (TR + TM) * 128;              // a step's bytes
    static constexpr int kBytes = KG * kGroup;                  // a stage's
    static constexpr int kPieces = kBytes / 1024 / kWaves;      // 1 KB loads a wave
    static_assert(kPieces * 1024 * kWaves == kBytes, "whole pieces");
    static constexpr int kLds = NBUF * kBytes;
    // through how many parts the sums go to the other threads
    static constexpr int kPasses = KG * TR * TM * 4 > kLds ? 2 : 1;
    static_assert(KG * TR * TM * 4 <= kLds * kPasses && kLds <= 160 * 1024, "LDS");
};

[[maybe_unused]] constexpr int kRsrc = 0x00027000;  // a raw buffer

// This wave's loads into LDS have arrived and its reads are done; then every wave's.
// (LATER: loads of steps that need not have.)
template <int LATER>
__device__ __forceinline__ void arrived() {
    static_assert(LATER < 64, "the counter's width");
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// sum += w . x. Written out so that the sums stay where they are: from the builtin the compiler gives results
// other registers than their operands, and copies them about in every step of the larger tiles. The next
// product of the same sum is three others away at least, longer than one takes; the last ones are builtins, so
// that the compiler knows what to wait for before it reads a sum.
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass knows no such registers)
__device__ __forceinline__ void product(i4& sum, const i4& w, const i4& x) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(sum) : "v"(w), "v"(x));
}
#endif

template <typename T, int TR, int TM, int KG, int WR, int WM, int NBUF>
__global__ __launch_bounds__(64 * KG * WR * WM) void tile_kernel(Args a, int tiles_r, int tiles_m) {
#ifdef __HIP_DEVICE_COMPILE__
    using S = Tile<TR, TM, KG, WR, WM, NBUF>;
    constexpr int FR = S::FR, FM = S::FM, NP = S::kPieces;
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroups go to the eight XCDs in turn: each XCD takes a run of tiles, eight tiles of tokens by
    // as many of rows as it has, so that its L2 serves what they share.
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
    const int steps = a.pitch / 128, stages = (steps + KG - 1) / KG;
    constexpr int PW = TR / 8, PG = (TR + TM) / 8;  // pieces of w, and of a step
    int off[NP];
    auto of_w = [&](int i) {  // which operand piece i is of: known when compiled where TR is whole pieces of all
        if constexpr (KG == 1 && PW % S::kWaves == 0) return i < PW / S::kWaves;
        else return (i * S::kWaves + wave) % PG < PW;
    };
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int row = (i * S::kWaves + wave) % PG * 8 + (lane >> 3);
        const int in = of_w(i) ? min(row, a.R - 1 - r0) : min(row - TR, a.M - 1 - m0);
        off[i] = in * a.pitch + 16 * ((lane & 7) ^ (lane >> 3));
    }
    // piece i of a stage, into buffer `buf` (the last step again behind the end)
    auto fetch = [&](int i, int buf, int stage) {
        const int8_t* base = of_w(i) ? a.w + (long long)r0 * a.pitch : a.x + (long long)m0 * a.pitch;
        const int p = i * S::kWaves + wave, step = KG == 1 ? stage : min(stage * KG + p / PG, steps - 1);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, -1, kRsrc), (LdsPtr)(lds + buf * S::kBytes + p * 1024),
            16, off[i], step * 128, 0, 0);
    };
#pragma unroll
    for (int b = 0; b < NBUF; ++b)
        if (b < stages) {
#pragma unroll
            for (int i = 0; i < NP; ++i) fetch(i, b, b);
        }
    const int group = wave / (WR * WM), wr = wave / WM % WR, wm = wave % WM;
    const int at = group * S::kGroup + (lane & 15) * 128 + 16 * ((lane >> 4) ^ (lane & 7));
    const int at_w = wr * FR * 2048 + at, at_x = TR * 128 + wm * FM * 2048 + at;
    i4 wf[2][FR], xf[2][FM];
    // operand f of half a step
    auto read = [&](int f, int half, int buf) {
        const int8_t* base = lds + buf * S::kBytes;
        if (f < FM) xf[half][f] = *reinterpret_cast<const i4*>(base + (at_x ^ (64 * half)) + f * 2048);
        else wf[half][f - FM] = *reinterpret_cast<const i4*>(base + (at_w ^ (64 * half)) + (f - FM) * 2048);
    };
    constexpr int NF = FR + FM, N = FR * FM;
    constexpr bool OUT = N >= 4;  // products written out: three others at least between two of a sum
    // (a group without a last step would end on products written out, with nothing to wait for their sums)
    static_assert(KG == 1 || !OUT, "waves that share the columns end on builtin products");
    i4 acc[FR][FM] = {};
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
            if constexpr (OUT) asm volatile("" : "+a"(acc[i][j]));  // (zero while the first loads run)

    // The products of half a step, with the reads of the next half's operands (NR of them) and loads (NL)
    // spread over the first three quarters of them.
    auto multiply = [&](int half, auto nr, int read_buf, auto nl, int load_buf, int load_step) {
        constexpr int NR = decltype(nr)::value, NL = decltype(nl)::value, MOST = NR > NL ? NR : NL;
        constexpr int EACH = MOST == 0 ? N : N * 3 / 4 / MOST > 0 ? N * 3 / 4 / MOST : 1;
        constexpr int GROUP = (MOST + N - 1) / N;  // of them behind a product
        if constexpr (OUT) asm volatile("s_nop 1");  // (registers written just before need two states)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            // (behind a product: the first one's wait for its operands is not one for these reads)
            i4& sum = acc[k / FM][k % FM];
            if constexpr (OUT) product(sum, wf[half][k / FM], xf[half][k % FM]);
            else sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[half][k / FM], xf[half][k % FM], sum, 0, 0, 0);
            if (k % EACH == 0) {
#pragma unroll
                for (int i = k / EACH * GROUP; i < (k / EACH + 1) * GROUP; ++i) {
                    if (i < NL) fetch(i, load_buf, load_step);
                    if (i < NR) read(i, half ^ 1, read_buf);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // A step: the products of its first half while the second half's operands are read; then every wave is
    // done with the step's buffer and the next step has arrived in its own: the products of the second half
    // while a later step is fetched into the buffer and the next one's first operands are read.
    using Reads = std::integral_constant<int, NF>;
    using Loads = std::integral_constant<int, NP>;
    using None = std::integral_constant<int, 0>;
    int buf = 0;
    auto step = [&](int s, auto loads) {
        const int next = buf + 1 < NBUF ? buf + 1 : 0;
        multiply(0, Reads(), buf, None(), 0, 0);
        if constexpr (decltype(loads)::value > 0) arrived<(NBUF - 2) * NP>();
        else arrived<0>();
        multiply(1, Reads(), next, loads, buf, s + NBUF);
        buf = next;
    };
    if (stages >= NBUF) arrived<(NBUF - 1) * NP>();
    else arrived<0>();
#pragma unroll
    for (int f = 0; f < NF; ++f) read(f, 0, 0);
    int s = 0;
    for (; s < stages - NBUF; ++s) step(s, Loads());
#pragma unroll 1
    for (; s < stages - 1; ++s) step(s, None());
    if (KG == 1 || s * KG + group < steps) {
        multiply(0, Reads(), buf, None(), 0, 0);
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[1][i], xf[1][j], acc[i][j], 0, 0, 0);
    }
    // The sums go through LDS (token-major, 16-byte chunk c of token m at c ^ (m % 8)): a thread then has
    // neighbouring rows for whole lines of y, and a short loop writes them, eight tokens' reads of `add`
    // together. (Straight code over the registers was 30 KB of instructions, read for every tile, with one read
    // of `add` after another: 163 us where this takes 137, for 4096 tokens onto a residual.)
    constexpr int CHUNKS = TR / 4, KEYS = CHUNKS < 8 ? CHUNKS : 8, PASSES = S::kPasses;
    constexpr int TOKENS = TM / PASSES, MINE = TOKENS / WM;      // of a pass, and of those a wave's
    constexpr int PER = S::kThreads / CHUNKS;                    // tokens at once
    constexpr int ROUNDS = TOKENS > PER ? TOKENS / PER : 1, BATCH = ROUNDS < 8 ? ROUNDS : 8;
    i4* part = reinterpret_cast<i4*>(lds);
    const int c = threadIdx.x % CHUNKS, mine = threadIdx.x / CHUNKS;
    const int r = r0 + 4 * c;
    const f4 ws = four_of(a.w_scales, min(r, a.R - 1), a.R);
    const f4 bias = a.bias ? four_of(a.bias, min(r, a.R - 1), a.R) : f4{};
    const float most = fmaxf(fmaxf(fabsf(ws[0]), fabsf(ws[1])), fmaxf(fabsf(ws[2]), fabsf(ws[3])));
    const bool whole = r + 3 < a.R && !(most >= kLarge);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        arrived<0>();  // every wave is done with what lay there
#pragma unroll
        for (int j = 0; j < MINE / 16; ++j)
#pragma unroll
            for (int i = 0; i < FR; ++i) {
                const int m = wm * MINE + 16 * j + (lane & 15), k = (wr * FR + i) * 4 + (lane >> 4);
                part[(group * TOKENS + m) * CHUNKS + (k ^ (m & (KEYS - 1)))] = acc[i][p * (MINE / 16) + j];
            }
        arrived<0>();
        // token m of a pass: the wave of its columns has it there
        auto token = [&](int m) { return m0 + m / MINE * (TM / WM) + p * MINE + m % MINE; };
        auto sum_of = [&](int m) {
            i4 sum = part[m * CHUNKS + (c ^ (m & (KEYS - 1)))];
#pragma unroll
            for (int g = 1; g < KG; ++g) sum += part[(g * TOKENS + m) * CHUNKS + (c ^ (m & (KEYS - 1)))];
            return sum;
        };
        if (whole) {
#pragma unroll 1
            for (int k = mine; k < TOKENS; k += BATCH * PER) {
                float xs[BATCH];
                Four<T> add[BATCH] = {};
                int m[BATCH];
#pragma unroll
                for (int q = 0; q < BATCH; ++q) {
                    m[q] = token(k + q * PER);
                    xs[q] = a.x_scales[min(m[q], a.M - 1)];
                }
                if (a.add) {
#pragma unroll
                    for (int q = 0; q < BATCH; ++q)
                        add[q] = *reinterpret_cast<const Four<T>*>(
                            static_cast<const T*>(a.add) + min(m[q], a.M - 1) * a.add_stride + r);
                }
#pragma unroll
                for (int q = 0; q < BATCH; ++q)
                    if (m[q] < a.M)
                        finish_four<T>(a, m[q], r, sum_of(k + q * PER), xs[q], ws, bias, add[q]);
            }
        } else if (r < a.R) {
#pragma unroll 1
            for (int k = mine; k < TOKENS; k += PER) {
                const int m = token(k);
                finish<T>(a, m, r, sum_of(k), a.x_scales[min(m, a.M - 1)], ws, bias);
            }
        }
    }
#endif
}

template <typename T, int TR, int TM, int KG, int WR, int WM, int NBUF>
int launch_tiles(const Args& a, hipStream_t st) {
    using S = Tile<TR, TM, KG, WR, WM, NBUF>;
    auto kernel = tile_kernel<T, TR, TM, KG, WR, WM, NBUF>;
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
    if ((long long)tiles_r * tiles_m >= (1LL << 32) / S::kThreads)
        return set_error(CSDR_E_INVALID, "q8_linear: more workgroups than a launch may have");
    kernel<<<(unsigned)(tiles_r * tiles_m), S::kThreads, S::kLds, st>>>(a, tiles_r, tiles_m);
    return CSDR_OK;
}

// What a tile costs, in us: `fixed` for a workgroup's start and end, a step of 128 columns `alone` for one
// workgroup on a CU and `each` for every one of `held` (as many as a CU's LDS holds). Fitted to products of 1
// to 4096 tokens with 1152 to 11008 rows and 896 to 11008 columns whose codes lie in the Infinity Cache, which they
// give within a tenth to a fifth; the rule has only to tell tiles apart. Codes from memory have no term in it (one
// token, 22016 x 4096: 13.6 us here, 18 to 23 measured). Both sides of its borders, measured for 4096 x 4096: 64 tokens
// 6.3 us in tiles of 32 x 32, 8.1 of 32 x 64; 128 tokens 8.1 of 32 x 32, 8.2 of 32 x 64, 10.6 of 64 x 64; 512 tokens
// 13.8 of 128 x 64, 15 of 64 x 64, 22.7 of 128 x 128; 2048 tokens 34 of 128 x 128, 42 of 128 x 64, 46 of 256 x
// 256; 4096 tokens 58 of 256 x 256, 66 of 128 x 128.
struct Cost {
    int tr, tm, held;
    float fixed, alone, each;
};
constexpr Cost kCosts[] = {
    {256, 256, 1, 11.0f, 1.35f, 1.35f}, {128, 128, 2, 5.0f, 0.53f, 0.445f}, {128, 64, 2, 3.0f, 0.33f, 0.30f},
    {64, 64, 3, 3.0f, 0.235f, 0.197f},  {32, 64, 3, 3.0f, 0.165f, 0.122f},  {32, 32, 2, 2.4f, 0.122f, 0.10f},
    {16, 16, 3, 2.3f, 0.088f, 0.073f},
};
constexpr int kCUs = 256;

float cost_of(const Cost& c, const Args& a) {
    const long long tiles = (long long)((a.R + c.tr - 1) / c.tr) * ((a.M + c.tm - 1) / c.tm);
    const long long most = (tiles + kCUs - 1) / kCUs;  // of a CU
    const int steps = a.pitch / 128, rest = (int)(most % c.held);
    float us = (float)(most / c.held) * (c.fixed + steps * c.held * c.each);
    if (rest) us += c.fixed + steps * std::max(c.alone, rest * c.each);
    return us;
}

template <typename T>
int launch(const Args& a, hipStream_t st) {
    int best = 0;
    float least = INFINITY;
    for (int i = 0; i < (int)(sizeof kCosts / sizeof *kCosts); ++i) {
        const float us = cost_of(kCosts[i], a);
        if (us < least) {
            least = us;
            best = i;
        }
    }
    switch (best) {
        case 0: return launch_tiles<T, 256, 256, 1, 4, 2, 2>(a, st);
        case 1: return launch_tiles<T, 128, 128, 1, 4, 2, 2>(a, st);
        case 2: return launch_tiles<T, 128, 64, 1, 2, 2, 3>(a, st);
        case 3: return launch_tiles<T, 64, 64, 1, 2, 2, 3>(a, st);
        case 4: return launch_tiles<T, 32, 64, 1, 1, 4, 4>(a, st);
        case 5: return launch_tiles<T, 32, 32, 2, 1, 2, 4>(a, st);
        default: return launch_tiles<T, 16, 16, 4, 1, 1, 3>(a, st);
    }
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
    if (y == w || y == x) return set_error(CSDR_E_INVALID, "q8_linear: y is an input");
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
    const int rc = y_dtype == CSDR_F32 ? launch<float>(a, st) : launch<_Float16>(a, st);
    if (rc != CSDR_OK) return rc;
    CSDR_LAUNCH_CHECK("q8_linear");
    return CSDR_OK;
}

}  // extern "C"
