// Eights of a row of C values: the whole ones, and the last, of C % 8, value by value.
// Rows may start at any element.
#pragma once

#include "logits_rows.h"

namespace rwkv7 {

// How many of the b-th eight's values the row has.
RWKV7_DEV int part_len(int64_t b, int C) {
  const int64_t n = C - 8 * b;
  return n < 0 ? 0 : n > 8 ? 8 : (int)n;
}

// The b-th eight of a row, zeros where it has none; `n` = part_len(b, C).
// EIGHTS: n is 0 or 8.
template <int FMT, bool EIGHTS = false>
RWKV7_DEV void load_part(Chunk<FMT> &x, const void *row, uint32_t b, int n) {
  if (n == 8) {
    x.load_whole(row, b);
    return;
  }
#pragma unroll
  for (int i = 0; i < Chunk<FMT>::kWords; ++i) x.w[i] = 0u;
  if (EIGHTS || n == 0) return;
  if constexpr (FMT == 1) {
    const uint32_t *p = static_cast<const uint32_t *>(row) + 8 * b;
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) x.w[e] = p[e];
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(row) + 8 * b;
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) x.w[e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
  }
}

// Eight values as the b-th eight of a row, as far as it has them.
template <int FMT, bool EIGHTS = false>
RWKV7_DEV void store_part(void *row, uint32_t b, int n, const float (&f)[8]) {
  if (n == 8) {
    store_chunk<FMT>(row, b, f);
    return;
  }
  if (EIGHTS) return;
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < n) store_logit<FMT>(row, 8 * (int64_t)b + e, f[e]);
}

// Eight values of a vector of either type, as f32.
template <int FMT, bool EIGHTS = false>
RWKV7_DEV void load_part_f(float (&f)[8], const void *row, uint32_t b, int n) {
  Chunk<FMT> x;
  load_part<FMT, EIGHTS>(x, row, b, n);
  x.get(f);
}

}  // namespace rwkv7
