// q8.hpp — the layout of 8-bit rows that q8_rows.hip writes and q8_linear.hip multiplies.
#pragma once

#include "common.hpp"

namespace csdr {

// Codes of a row lie side by side, zeros behind the last up to a whole number of 128 bytes (two
// matrix-core steps over the columns, 16-byte loads at every row): no product has a rest of columns.
constexpr int kRowBytes = 128;
// Widest row: a sum of products of two codes (at most 2^14 each) stays within 32 bits.
constexpr int kMaxWidth = (1 << 17) - 1;

inline size_t q8_pitch(int n) { return align_up((size_t)n, kRowBytes); }

}  // namespace csdr
