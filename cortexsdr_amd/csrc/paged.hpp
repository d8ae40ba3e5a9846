// paged.hpp — layout of the paged K/V cache (csdr_paged_kv) and the lookups its kernels share.
//
// A page holds page_size positions (a power of two, 16 or more) of every KV head; K and V have
// pages of their own. Per KV head, hd dims, page_size ps:
//   CSDR_F16  K [position][dim]: a row is the A operand of a score tile as it lies. V [position /
//             8][dim][position % 8]: 16 bytes are 8 positions of one dim, the A operand of
//             O^T = V^T P^T, so neither is transposed on the way to the matrix cores.
//   CSDR_Q4   codes, then per group of 32 dims and position a scale, then a minimum (fp16,
//             [group][position] each); value = minimum + scale * code. Eight codes share a 32-bit
//             word, code e in bits 4 (e / 2) + 16 (e % 2): one shift and one mask bring the pair
//             (2j, 2j + 1) into the two halves of a register. K: per position, words [dim % 32 /
//             8][dim / 32] of 8 dims: lane group g of a score tile loads its words of all groups
//             of dims at once. V: per 8 positions, words [dim % 16][dim / 16] of those positions:
//             a lane loads its dim's words of all output tiles at once.
#pragma once

#include "common.hpp"

namespace csdr {

constexpr int kGroup = 32;  // dims that share a 4-bit scale and minimum
constexpr int kMaxPositions = 1 << 30;

// Bytes of one KV head in a page.
__host__ __device__ constexpr int paged_head_bytes(bool q4, int ps, int hd) {
    return q4 ? ps * (hd / 2 + hd / kGroup * 4) : ps * hd * 2;
}

struct PagedView {
    uint8_t* k;
    uint8_t* v;
    const int32_t* table;    // n_seqs x stride page ids
    const int32_t* lens;     // positions of each sequence, the call's tokens included
    const int32_t* q_start;  // n_seqs + 1 first rows, or NULL: T rows each
    int n_pages, shift, hkv, stride, n_seqs;
    int n_tokens, T, max_q;

    __host__ __device__ int capacity() const { return stride << shift; }
    __host__ __device__ int page_size() const { return 1 << shift; }
};

// The rows of a call that belong to one sequence: rows first .. first + n - 1 at positions p0 ..;
// the sequence holds len positions in all.
struct SeqRows {
    int first, n, p0, len;
};

__host__ __device__ __forceinline__ SeqRows seq_rows(const PagedView& pv, int b) {
    SeqRows r;
    int n;
    if (pv.q_start) {
        r.first = min(max(pv.q_start[b], 0), pv.n_tokens);
        n = min(max(pv.q_start[b + 1], r.first), pv.n_tokens) - r.first;
    } else {
        r.first = b * pv.T;
        n = pv.T;
    }
    r.len = min(max(pv.lens[b], 0), kMaxPositions + (kMaxPositions >> 1));  // no sum overflows
    r.p0 = r.len - n;
    r.n = min(n, pv.max_q);
    return r;
}

// The page of position p of sequence b (SCALAR: the same in the whole wave, looked up through the
// scalar cache also behind barriers, which a constant table allows), or -1 where the table has none
// (positions past its end, ids outside [0, n_pages)).
template <bool SCALAR = false>
__host__ __device__ __forceinline__ int page_of(const PagedView& pv, int b, int p) {
    const int i = p >> pv.shift;
    if (p < 0 || i >= pv.stride) return -1;
    const size_t at = (size_t)b * pv.stride + i;
#if defined(__HIP_DEVICE_COMPILE__)
    const int pg = SCALAR ? ((const __attribute__((address_space(4))) int32_t*)pv.table)[at]
                          : pv.table[at];
#else
    const int pg = pv.table[at];
#endif
    return (unsigned)pg < (unsigned)pv.n_pages ? pg : -1;
}

template <bool Q4>
__device__ __forceinline__ size_t head_offset(const PagedView& pv, int hd, int page, int head) {
    return ((size_t)page * pv.hkv + head) * (size_t)paged_head_bytes(Q4, pv.page_size(), hd);
}

// Byte offsets of a group's scale and minimum of one position inside a head (4 bits).
__host__ __device__ __forceinline__ int scale_offset(int hd, int ps, int group, int slot) {
    return ps * (hd / 2) + 2 * (group * ps + slot);
}
__host__ __device__ __forceinline__ int min_offset(int hd, int ps, int group, int slot) {
    return scale_offset(hd, ps, group, slot) + 2 * ps * (hd / kGroup);
}

__host__ __device__ __forceinline__ int code_shift(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

// Word index of K's 8 dims d .. d + 7 (d % 8 == 0) of a position, and of V's dim d of 8 positions.
template <int HD>
__host__ __device__ __forceinline__ int k_word(int slot, int d) {
    return slot * (HD / 8) + ((d & 31) >> 3) * (HD / kGroup) + (d >> 5);
}
template <int HD>
__host__ __device__ __forceinline__ int v_word(int slot, int d) {
    return (slot >> 3) * HD + (d & 15) * (HD / 16) + (d >> 4);
}

// One value of the cache, for the kernels that read few of them. `p` is the head's base.
template <int HD, bool Q4>
__device__ __forceinline__ float cache_value(const uint8_t* p, bool is_v, int ps, int slot, int d) {
    if (!Q4) {
        const int i = is_v ? ((slot >> 3) * HD + d) * 8 + (slot & 7) : slot * HD + d;
        return (float)reinterpret_cast<const _Float16*>(p)[i];
    }
    const uint32_t w =
        reinterpret_cast<const uint32_t*>(p)[is_v ? v_word<HD>(slot, d) : k_word<HD>(slot, d)];
    const float c = (float)((w >> code_shift(is_v ? slot & 7 : d & 7)) & 15u);
    const int g = d / kGroup;
    const float s = (float)*reinterpret_cast<const _Float16*>(p + scale_offset(HD, ps, g, slot));
    const float m = (float)*reinterpret_cast<const _Float16*>(p + min_offset(HD, ps, g, slot));
    return fmaf(s, c, m);
}

// Host: the descriptor's checks, shared by the entry points (paged_cache.hip).
int paged_check(const char* what, const csdr_paged_kv* kv, int n_tokens, const int32_t* q_start,
                int max_q, PagedView* out);

}  // namespace csdr
