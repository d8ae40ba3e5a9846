// logprobs.hip — log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits (gfx950).
//
//   m = max x; d = (x - m) / temperature; Z = sum exp d; logprob_t = d_t - log Z
//   entropy = log Z - sum exp(d) d / Z
// (Differences first: x / temperature alone may be past fp32 where d is not.)
// The order of the top: larger x first, among equals the lower id.
//
// Bound by the read of the logits: 2048 rows of 151936 fp32 with the top 5 take 233 us, 5.3 TB/s
// (of fp16 196 us, 3.2 TB/s, since a value's vector work stays).
// segment_kernel reads them once: a wave takes a segment of a row in rounds of 2048 values that
// stay in registers, the next round's loads issued before the current one is worked on. Per round:
// the maximum, then the two sums about the running maximum; for the top, values that beat the
// wave's n-th best so far go to a list in LDS, which is cut to the best n when it fills. The first
// round's bound is the n-th largest of 128 group maxima (there are n values no smaller), found bit
// by bit with ballots, so that about n values pass it and not all. join_kernel joins a row's
// segments: sums rescaled to one maximum; of the segments' lists the entries no smaller than the
// n-th largest of their heads, which are few, are ranked. Where they are many (equals; fewer
// segments than places), the n-th best is found bit by bit over all entries first, then, if there
// are more equals of it than places, the last id among them (8 rows of 151936, top 20: always bit
// by bit 13.2 us, heads first 9.4).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "common.hpp"

namespace {

using csdr::set_error;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kMaxTop = 64;
constexpr int kPer = 32;               // values per lane and round
constexpr int kRound = 64 * kPer;
constexpr int kList = 192;             // entries of a wave's list: room for 64 more at 128
constexpr int kMaxSegments = 128;
constexpr int kListEntries = 7168;     // of a row's segments' lists in all: 56 KB
constexpr float kLog2e = 1.44269504088896341f;

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct Args {
    const void* x;
    int rows, n;
    long long stride;
    float inv_t;
    const int32_t* tokens;
    float *logprobs, *entropy, *top_logprobs;
    int32_t* top_ids;
    int top_n, segments, rounds;  // segments per row, rounds per segment
    float4* sums;                 // per (row, segment): maximum, Z, weighted sum, 1 if not finite
    float* top_v;                 // per (row, segment): top_n values and ids, best first
    int32_t* top_i;
};

struct Entry {
    float v;
    int i;
};
__device__ __forceinline__ bool beats(Entry a, Entry b) {
    return a.v > b.v || (a.v == b.v && a.i < b.i);
}

// 16 bytes at any alignment of the element
template <typename XT>
struct __attribute__((packed, aligned(sizeof(XT)))) Piece {
    u4 v;
};

template <typename XT>
__device__ __forceinline__ float element(const u4& p, int e) {
    if constexpr (sizeof(XT) == 4) return __uint_as_float(p[e]);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(p[e >> 1] >> (16 * (e & 1))));
}

// fp32 values as whole numbers of the same order (both zeros as one).
__device__ __forceinline__ uint32_t key_of(float v) {
    const int b = __float_as_int(v + 0.0f);
    return (uint32_t)(b ^ ((b >> 31) & 0x7FFFFFFF)) ^ 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    const int b = (int)(k ^ 0x80000000u);
    return __int_as_float(b ^ ((b >> 31) & 0x7FFFFFFF));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The list's best n, in order, by one wave: each lane ranks up to three entries against all.
// Returns how many are left.
__device__ int cut_list(Entry* list, int count, int n) {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    Entry mine[kList / 64];
    int rank[kList / 64];
#pragma unroll
    for (int k = 0; k < kList / 64; ++k) {
        mine[k] = list[min(lane + 64 * k, count - 1)];
        rank[k] = 0;
    }
    for (int j = 0; j < count; j += 4) {  // (four reads in flight; entries past the end repeat)
        Entry e[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) e[u] = list[min(j + u, count - 1)];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int k = 0; k < kList / 64; ++k) rank[k] += j + u < count && beats(e[u], mine[k]);
    }
#pragma unroll
    for (int k = 0; k < kList / 64; ++k)
        if (lane + 64 * k < count && rank[k] < n) list[rank[k]] = mine[k];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return min(count, n);
}

template <typename XT, bool TOP>
__global__ __launch_bounds__(kThreads) void segment_kernel(Args a) {
    constexpr int VEC = 16 / sizeof(XT), NP = kPer / VEC;
    __shared__ Entry lists[TOP ? kWaves : 1][TOP ? kList : 1];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long unit = (long long)blockIdx.x * kWaves + wave;
    const int row = (int)(unit / a.segments), seg = (int)(unit % a.segments);
    if (row >= a.rows) return;
    const XT* x = static_cast<const XT*>(a.x) + (long long)row * a.stride;
    const long long from = (long long)seg * a.rounds * kRound;
    const int rounds =
        (int)max(0LL, min((long long)a.rounds, (a.n - from + kRound - 1) / kRound));
    Entry* list = lists[TOP ? wave : 0];
    int count = 0;
    float bar = -INFINITY;  // a value below is not among the segment's best
    float m = -INFINITY, z = 0.0f, w = 0.0f;
    bool bad = false;

    // round r's values of this lane: element e of piece p is id
    // from + r kRound + (64 p + lane) VEC + e
    u4 next[NP];
    auto load = [&](int r) {
        const long long base = from + (long long)r * kRound;
        if (base + kRound <= a.n) {
#pragma unroll
            for (int p = 0; p < NP; ++p)
                next[p] =
                    reinterpret_cast<const Piece<XT>*>(x + base + (64 * p + lane) * VEC)->v;
        } else {
            constexpr uint32_t low = sizeof(XT) == 4 ? 0xFF800000u : 0xFC00FC00u;  // -infinity
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const long long i = base + (64 * p + lane) * VEC;
                next[p] = u4{low, low, low, low};
                if (i + VEC <= a.n) {
                    next[p] = reinterpret_cast<const Piece<XT>*>(x + i)->v;
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (i + e < a.n) {
                            if constexpr (sizeof(XT) == 4) {
                                next[p][e] = __float_as_uint((float)x[i + e]);
                            } else {
                                const uint32_t h = __builtin_bit_cast(uint16_t, x[i + e]);
                                const int sh = 16 * (e & 1);
                                next[p][e >> 1] = (next[p][e >> 1] & ~(0xFFFFu << sh)) | h << sh;
                            }
                        }
                }
            }
        }
    };
    if (rounds > 0) load(0);
    for (int r = 0; r < rounds; ++r) {
        float y[kPer];                          // the round's logits
        float big[2] = {-INFINITY, -INFINITY};  // maxima of the lane's two groups of 16
        int hi = 0x80000000;                    // NaN and +infinity, by their bits
        uint32_t lo = 0u;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            y[k] = element<XT>(next[k / VEC], k % VEC);
            hi = max(hi, __float_as_int(y[k]));
            lo = max(lo, __float_as_uint(y[k]));
        }
        if (r + 1 < rounds) load(r + 1);
        if (__any(hi >= 0x7F800000 || lo > 0xFF800000u)) {
            bad = true;
#pragma unroll
            for (int k = 0; k < kPer; ++k)
                if (!(y[k] < INFINITY)) y[k] = -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) big[k / 16] = fmaxf(big[k / 16], y[k]);
        const float top = wave_max(fmaxf(big[0], big[1]));
        if (top == -INFINITY) continue;
        if (top > m) {
            // (f = 0: what came before is nothing beside this round, and its z d may be past
            // fp32, as after rounds of the type's lowest value)
            const float d = (m - top) * a.inv_t, f = exp2f(d * kLog2e);
            w = f > 0.0f ? f * fmaf(z, d, w) : 0.0f;
            z *= f;
            m = top;
        }
        float zr = 0.0f, wr = 0.0f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            // exp(-200) is 0 here, 0 * -200 too
            const float d = fmaxf((y[k] - m) * a.inv_t, -200.0f);
            const float e = __builtin_amdgcn_exp2f(d * kLog2e);
            zr += e;
            wr = fmaf(e, d, wr);
        }
        z += zr;
        w += wr;
        if constexpr (TOP) {
            if (!(top >= bar)) continue;
            const int n = a.top_n;
            if (count < n) {
                // about the n-th largest group maximum, its key from the highest bit down: n values
                // of this round, and not many more, are no smaller
                const uint32_t k0 = key_of(big[0]), k1 = key_of(big[1]);
                uint32_t t = 0u;
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t c = t | 1u << bit;
                    const int above = __popcll(__ballot(k0 >= c)) + __popcll(__ballot(k1 >= c));
                    if (above >= n) t = c;
                    if (above >= n && above <= n + 4) break;
                }
                bar = value_of(max(t, key_of(-INFINITY)));
            }
            const int id0 = (int)(from + (long long)r * kRound) + lane * VEC;
            const int before = count;
            bool cut = false;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const bool in = y[k] >= bar && y[k] > -INFINITY;
                const uint64_t mask = __ballot(in);
                if (mask) {
                    if (in)
                        list[count + lanes_below(mask)] =
                            Entry{y[k], id0 + (k / VEC) * 64 * VEC + k % VEC};
                    count += __popcll(mask);
                    if (count > kList - 64) {
                        count = cut_list(list, count, n);
                        cut = true;
                        bar = list[n - 1].v;  // (equals still pass: their ids may be lower)
                    }
                }
            }
            if (r + 1 < rounds && count >= n && (cut || count > before)) {
                // the ids of later rounds are higher: an equal of the n-th best loses
                count = cut_list(list, count, n);
                bar = value_of(key_of(list[n - 1].v) + 1u);
            }
        }
    }
    z = csdr::wave_sum(z);
    w = csdr::wave_sum(w);
    const long long at = (long long)row * a.segments + seg;
    if (lane == 0) a.sums[at] = float4{m, z, w, bad ? 1.0f : 0.0f};
    if constexpr (TOP) {
        if (count > 0) count = cut_list(list, count, a.top_n);
        for (int i = lane; i < a.top_n; i += 64) {
            a.top_v[at * a.top_n + i] = i < count ? list[i].v : -INFINITY;
            a.top_i[at * a.top_n + i] = i < count ? list[i].i : -1;
        }
    }
}

// A row's segments joined, one workgroup per row.
template <typename XT, bool TOP>
__global__ __launch_bounds__(kThreads) void join_kernel(Args a) {
    extern __shared__ uint32_t shared[];  // segments x top_n keys, then ids
    const int row = blockIdx.x, lane = threadIdx.x & 63, S = a.segments;
    const float4* s = a.sums + (long long)row * S;
    // every load that waits for nothing first; each wave joins the sums for itself (at most two
    // segments a lane)
    const int token = a.tokens ? a.tokens[row] : -1;
    float4 p[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
        p[k] = lane + 64 * k < S ? s[lane + 64 * k] : float4{-INFINITY, 0.0f, 0.0f, 0.0f};
    const int n = a.top_n, all = S * n;
    const long long at = (long long)row * all;
    uint32_t* key = shared;
    uint32_t* id = shared + all;
    if constexpr (TOP)
        for (int i0 = threadIdx.x; i0 < all; i0 += 8 * kThreads) {
            int32_t e[8];  // (eight loads in flight: one at a time took 6 of 9 us)
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = min(i0 + k * kThreads, all - 1);
                e[k] = a.top_i[at + i];
                v[k] = a.top_v[at + i];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = i0 + k * kThreads;
                if (i >= all) break;
                key[i] = e[k] < 0 ? 0u : key_of(v[k]);  // (no finite value has key 0)
                id[i] = (uint32_t)e[k];
            }
        }
    float xt = 0.0f;
    if (token >= 0 && token < a.n)
        xt = (float)static_cast<const XT*>(a.x)[(long long)row * a.stride + token];
    const float m = wave_max(fmaxf(p[0].x, p[1].x));
    float z = 0.0f, w = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (p[k].x == -INFINITY) continue;
        const float d = (p[k].x - m) * a.inv_t, f = expf(d);
        z = fmaf(f, p[k].y, z);
        w += f * (p[k].z + (f > 0.0f ? p[k].y * d : 0.0f));
    }
    z = csdr::wave_sum(z);
    w = csdr::wave_sum(w);
    const bool bad = __any(p[0].w + p[1].w > 0.0f), none = m == -INFINITY;
    const float lz = bad ? NAN : none ? 0.0f : logf(z);
    if (threadIdx.x == 0) {
        if (a.entropy) a.entropy[row] = none ? lz : lz - w / z;
        if (a.tokens) {
            float lp = token < 0 ? 0.0f : NAN;
            if (token >= 0 && token < a.n && !bad)
                lp = xt == -INFINITY ? xt : (xt - m) * a.inv_t - lz;
            a.logprobs[row] = lp;
        }
    }
    if constexpr (TOP) {
        __shared__ int part[2][kWaves];
        __shared__ Entry best[kThreads];
        __shared__ int nbest;
        if (threadIdx.x == 0) nbest = 0;
        __syncthreads();
        // entries with keys no smaller than t, of the equals those with ids up to `last`
        auto gather = [&](uint32_t t, uint32_t last) {
            for (int i = threadIdx.x; i < all; i += kThreads) {
                if (key[i] == 0u || key[i] < t || (key[i] == t && id[i] > last)) continue;
                const int k = atomicAdd(&nbest, 1);
                if (k < kThreads) best[k] = Entry{value_of(key[i]), (int)id[i]};
            }
            __syncthreads();
        };
        uint32_t heads = 0u;
        if (S >= n) {  // (every wave for itself: at most two heads a lane)
            const uint32_t k0 = lane < S ? key[lane * n] : 0u;
            const uint32_t k1 = lane + 64 < S ? key[(lane + 64) * n] : 0u;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t c = heads | 1u << bit;
                const int above = __popcll(__ballot(k0 >= c)) + __popcll(__ballot(k1 >= c));
                if (above >= n) heads = c;
                if (above >= n && above <= 2 * n) break;
            }
        }
        gather(heads, 0x7FFFFFFFu);
        if (nbest > kThreads) {
            int turn = 0;
            // the first eight entries of each thread stay in registers
            constexpr int kKept = 8;
            uint32_t kk[kKept], ki[kKept];
#pragma unroll
            for (int k = 0; k < kKept; ++k) {
                const int i = threadIdx.x + k * kThreads;
                kk[k] = i < all ? key[i] : 0u;
                ki[k] = i < all ? id[i] : 0xFFFFFFFFu;
            }
            auto count = [&](auto pred) {  // over all entries; the same in every thread
                int c = 0;
#pragma unroll
                for (int k = 0; k < kKept; ++k)
                    if (k * kThreads < all) c += __popcll(__ballot(pred(kk[k], ki[k])));
                for (int i = threadIdx.x + kKept * kThreads; i - (int)threadIdx.x < all; i += kThreads)
                    c += __popcll(__ballot(i < all && pred(key[min(i, all - 1)], id[min(i, all - 1)])));
                if (lane == 0) part[turn][threadIdx.x >> 6] = c;
                __syncthreads();
                c = 0;
#pragma unroll
                for (int k = 0; k < kWaves; ++k) c += part[turn][k];
                turn ^= 1;
                return c;
            };
            // the n-th best key t (0: fewer than n entries) and how many are no smaller
            uint32_t t = 0u;
            int above = all;
            for (int bit = 31; bit >= 0 && above != n; --bit) {
                const uint32_t c = t | 1u << bit;
                const int k = count([&](uint32_t x, uint32_t) { return x >= c; });
                if (k >= n) {
                    t = c;
                    above = k;
                }
            }
            uint32_t last = 0x7FFFFFFFu;  // of the equals of t, ids up to this one
            if (above > n && t > 0u) {
                const int more = count([&](uint32_t x, uint32_t) { return x > t; });
                uint32_t below = 0u;  // ids < below: fewer than the places left
                for (int bit = 30; bit >= 0; --bit) {
                    const uint32_t c = below | 1u << bit;
                    if (count([&](uint32_t x, uint32_t y) { return x == t && y < c; }) < n - more)
                        below = c;
                }
                last = below;
            }
            __syncthreads();  // (everyone has read nbest)
            if (threadIdx.x == 0) nbest = 0;
            __syncthreads();
            gather(t, last);
        }
        if ((int)threadIdx.x < nbest) {
            const Entry e = best[threadIdx.x];
            int rank = 0;
            for (int j = 0; j < nbest; j += 4) {
                Entry o[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) o[u] = best[min(j + u, nbest - 1)];
#pragma unroll
                for (int u = 0; u < 4; ++u) rank += j + u < nbest && beats(o[u], e);
            }
            if (rank < n) {
                a.top_ids[(long long)row * n + rank] = e.i;
                a.top_logprobs[(long long)row * n + rank] = (e.v - m) * a.inv_t - lz;
            }
        }
        for (int i = nbest + threadIdx.x; i < n; i += kThreads) {
            a.top_ids[(long long)row * n + i] = -1;
            a.top_logprobs[(long long)row * n + i] = -INFINITY;
        }
    }
}

// Segments of a row: whole rounds, about 8192 waves in all, as many as leave join_kernel's lists
// and its few KB beside them in the 64 KB of LDS that every launch may have.
void set_segments(Args& a) {
    const int all = (int)(((long long)a.n + kRound - 1) / kRound);
    const int most = std::min(kMaxSegments, kListEntries / std::max(a.top_n, 1));
    const int want = std::min(std::max(8192 / a.rows, 1), most);
    a.rounds = (all + want - 1) / want;
    a.segments = (all + a.rounds - 1) / a.rounds;
}

size_t workspace_of(const Args& a) {
    const size_t parts = (size_t)a.rows * a.segments;
    return parts * sizeof(float4) + parts * a.top_n * 8;
}

template <typename XT, bool TOP>
void launch(const Args& a, hipStream_t st) {
    const long long units = (long long)a.rows * a.segments;
    segment_kernel<XT, TOP><<<(unsigned)((units + kWaves - 1) / kWaves), kThreads, 0, st>>>(a);
    join_kernel<XT, TOP><<<a.rows, kThreads, (size_t)a.segments * a.top_n * sizeof(Entry), st>>>(a);
}

}  // namespace

extern "C" {

CSDR_API size_t csdr_token_logprobs_workspace_bytes(int rows, int n, int top_n) {
    if (rows <= 0 || n <= 0 || top_n < 0 || top_n > kMaxTop) return 0;
    Args a{};
    a.rows = rows;
    a.n = n;
    a.top_n = top_n;
    set_segments(a);
    return workspace_of(a);
}

CSDR_API int csdr_token_logprobs(const void* logits, int dtype, int rows, int n,
                                 int64_t row_stride, float temperature, const int32_t* tokens,
                                 float* logprobs, float* entropy, int top_n, int32_t* top_ids,
                                 float* top_logprobs, void* workspace, size_t workspace_bytes,
                                 void* hip_stream) {
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
    if (temperature > 0.0f && temperature < FLT_MIN)  // (its reciprocal may be infinite)
        return set_error(CSDR_E_INVALID, "token_logprobs: the temperature is a denormal number");
    if (rows > (1 << 24) - 1)  // (workgroups of a launch: 2^32 threads)
        return set_error(CSDR_E_INVALID, "token_logprobs: more than 2^24 - 1 rows");
    Args a{};
    a.x = logits;
    a.rows = rows;
    a.n = n;
    a.stride = row_stride ? row_stride : n;
    a.inv_t = temperature > 0.0f ? 1.0f / temperature : 1.0f;
    a.tokens = tokens;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.top_n = top_n;
    set_segments(a);
    if (!workspace || workspace_bytes < workspace_of(a) ||
        reinterpret_cast<uintptr_t>(workspace) % 16)
        return set_error(CSDR_E_WORKSPACE,
                         "token_logprobs: workspace missing, too small or unaligned");
    const size_t parts = (size_t)rows * a.segments;
    a.sums = static_cast<float4*>(workspace);
    a.top_v = reinterpret_cast<float*>(a.sums + parts);
    a.top_i = reinterpret_cast<int32_t*>(a.top_v + parts * top_n);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (dtype == CSDR_F32) {
        if (top_n) launch<float, true>(a, st);
        else launch<float, false>(a, st);
    } else {
        if (top_n) launch<_Float16, true>(a, st);
        else launch<_Float16, false>(a, st);
    }
    CSDR_LAUNCH_CHECK("token_logprobs");
    return CSDR_OK;
}

}  // extern "C"
