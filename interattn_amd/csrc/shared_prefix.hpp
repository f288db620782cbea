// Decode attention of a batch whose sequences share long prefixes: parameters shared by the
// host side and the per-type kernel instances.
//
// A group's members attend the same first tokens.  Their query rows are put together, so
// the prefix's K/V is read once per (group, kv head) instead of once per sequence; each
// sequence's own tokens are a second, small range.  Both kinds of range are cut into items
// of about the same number of key tiles, one workgroup each, and a row's partials (its
// prefix's items, then its own) are merged in that order: sums do not depend on timing.
#pragma once

#include "attend_rows.hpp"

namespace ia {

// one item: rows of the sequences [tok0, tok0 + n_tok), keys [k_lo, k_hi) of sequence table_seq
struct PrefixItem {
  int32_t tok0, n_tok, k_lo, k_hi, table_seq, slot, pad0, pad1;
};
// the partials of one range: n items of rows rows each, from row slot on
struct PrefixEntry {
  int32_t slot, n, rows, pad;
};

struct PrefixParams {
  ArParams ar;
  const int32_t* seq_lens;
  const int32_t* group_starts;  // [n_groups + 1]
  const int32_t* shared_lens;   // [n_groups]
  int32_t batch, n_groups;
  int32_t tile_seqs;            // sequences of a row tile (128 / group)
  int32_t n_tiles;              // bound of the prefixes' row tiles
  int32_t max_items;            // per kv head
  int32_t target;               // items per kv head the device runs at once
  int64_t kv_cap;
  int64_t rows;                 // partial rows per kv head
  int32_t* n_items;
  PrefixItem* items;
  PrefixEntry* entries;         // [n_tiles + batch]: the row tiles, then the sequences
  int32_t* tile_of;             // [batch] a sequence's row tile, -1: none
  float* part_ml;               // [n_kv_heads, rows, 2]
  float* part_acc;              // [n_kv_heads, rows, D]
};

constexpr int kPrefixMinTiles = 2;  // fewest key tiles an item is cut to

int launch_prefix_bf16(const PrefixParams& p, int d, hipStream_t st);
int launch_prefix_f32(const PrefixParams& p, int d, hipStream_t st);
int launch_prefix_fp8(const PrefixParams& p, int d, hipStream_t st);

template <int KV, int D>
__global__ __launch_bounds__(kArThreads, KV == kArF32 ? 1 : 2) void ia_shared_prefix_attend(PrefixParams p) {
  __shared__ __align__(1024) char smem[ArShape<KV, D>::kSmem];
  const int head = blockIdx.x % p.ar.n_kv_heads, i = blockIdx.x / p.ar.n_kv_heads;
  if (i >= *p.n_items) return;
  const PrefixItem x = p.items[i];
  ArItem it{};
  it.table = p.ar.kv.table ? p.ar.kv.table + (int64_t)x.table_seq * p.ar.kv.bt_stride : nullptr;
  it.head = head;
  it.tok0 = x.tok0;
  it.n_rows = x.n_tok * p.ar.group;
  it.k_lo = x.k_lo;
  it.k_hi = x.k_hi;
  it.lens = p.seq_lens;
  const int64_t row = (int64_t)head * p.rows + x.slot;
  it.part_ml = p.part_ml + 2 * row;
  it.part_acc = p.part_acc + row * D;
  ar_attend<KV, D>(p.ar, it, smem);
}

template <int KV, int D>
int launch_prefix(const PrefixParams& p, hipStream_t st) {
  hipLaunchKernelGGL((ia_shared_prefix_attend<KV, D>), dim3((unsigned)p.max_items * p.ar.n_kv_heads), dim3(kArThreads),
                     0, st, p);
  return check_launch("shared-prefix decode");
}

}  // namespace ia
