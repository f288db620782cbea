// Packed batches: sequences of different lengths one behind the other, cu[b] the first row
// of sequence b.
#pragma once

#include "ia_common.hpp"

namespace ia {

// A tile of up to `size` rows of one sequence.  Sequence b's tiles are numbered from
// cu[b] / size + b: floor sums leave every sequence room for its own and at least one
// number (an empty sequence has a tile of no rows), so a workgroup finds its sequence from
// cu alone, 64 candidates at a time, with no scan over the batch.  n_rows / size + n_seq
// numbers cover every batch of n_rows rows.  With `spare` 2 a sequence has room for one tile
// more: tiles that begin at multiples of `size` of another count than its own rows.
struct PackedTile {
  int b, tok0, n_tok;  // sequence, first row, rows; n_tok 0: no rows
  int first, count;    // the sequence's first row and row count
  int local;           // the tile's number in its sequence (negative: none)
};

__device__ __forceinline__ PackedTile packed_tile(const int32_t* cus, int n_seq, int n_rows, int size, int tile,
                                                  int lane, int spare = 1) {
  PackedTile r{};
  int lo = 0, len = n_seq;
  auto cu = [&](int i) {
    const int x = cus[i];
    return x < 0 ? 0 : x > n_rows ? n_rows : x;
  };
  while (len > 1) {
    const int step = (len + 63) / 64, i = lo + lane * step;
    const bool in = lane * step < len;
    const unsigned long long at = __ballot(in && cu(i) / size + spare * i <= tile);
    const int n = at ? 64 - __builtin_clzll(at) : 1;  // the last candidate that starts at or before the tile
    len = len - (n - 1) * step < step ? len - (n - 1) * step : step;
    lo += (n - 1) * step;
  }
  const int c0 = cu(lo), c1 = cu(lo + 1);
  r.b = lo;
  r.first = c0;
  r.count = c1 > c0 ? c1 - c0 : 0;
  r.local = tile - (c0 / size + spare * lo);
  const int64_t t0 = (int64_t)r.local * size;
  if (r.local < 0 || t0 >= r.count) return r;
  r.tok0 = c0 + (int)t0;
  r.n_tok = r.count - (int)t0 < size ? r.count - (int)t0 : size;
  return r;
}

}  // namespace ia
