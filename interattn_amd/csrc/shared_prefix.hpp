// Decode attention of a batch whose sequences share long prefixes: parameters shared by the
// host side and the per-type kernel instances.
//
// A group's members attend the same first tokens.  Their query rows are put together, so
// the prefix's K/V is read once per (group, kv head) instead of once per sequence; each
// sequence's own tokens are a second, small range.  Both kinds of range are cut into items
// of at most a cut of key tiles, one workgroup each, and a row's partials (its
// prefix's items, then its own) are merged in that order: sums do not depend on timing.
//
// Bound by the K/V stream where prefixes are long: 32 sequences behind 32,768 shared tokens (8
// kv heads of 128, groups of 4, bf16; 212 MB of K/V) take 50.4 us, 4.2 TB/s, while 17 MB of
// partials are written, and 8.2 us to merge them; 70 us with inputs that no cache holds.  Items
// on two workgroups per CU: with one of eight waves and a deeper ring the same took 87-91 us,
// since its waves load, multiply and exponentiate in step.  fp8 (5, 1, 9 and 4 members on
// 1,000-8,200 tokens): 34.9 us and 6.5 us of merge, a tile's latency with half the bytes in flight.
#pragma once

#include "attend_rows.hpp"

namespace ia {

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
  int32_t tile_seqs;            // sequences of a row tile (128 / group; float32 32 / group)
  int32_t n_tiles;              // bound of the prefixes' row tiles
  int32_t max_items;            // per kv head: workgroups launched
  int32_t target;               // items per kv head the device runs at once
  int64_t kv_cap;
  int64_t rows;                 // partial rows per kv head
  PrefixEntry* entries;         // [n_tiles + batch]: the row tiles, then the sequences
  float* part_ml;               // [n_kv_heads, rows, 2]
  float* part_acc;              // [n_kv_heads, rows, D]
};

constexpr int kPrefixMinTiles = 2;  // fewest key tiles an item is cut to

int launch_prefix_bf16(const PrefixParams& p, int d, hipStream_t st);
int launch_prefix_f32(const PrefixParams& p, int d, hipStream_t st);
int launch_prefix_fp8(const PrefixParams& p, int d, hipStream_t st);

__device__ __forceinline__ int prefix_start(const PrefixParams& p, int g) {
  const int s = p.group_starts[g];
  return s < 0 ? 0 : s > p.batch ? p.batch : s;
}

__device__ __forceinline__ int prefix_len(const PrefixParams& p, int b) {
  const int n = p.seq_lens[b];
  return n < 0 ? 0 : n > p.kv_cap ? (int)p.kv_cap : n;
}

// The plan's view of the groups: their starts and shared lengths, held in LDS where they
// fit (every entry looks its group up).
struct PrefixGroups {
  const PrefixParams& p;
  const int* starts;  // null: global memory
  const int* shared;

  __device__ __forceinline__ int start(int g) const { return starts ? starts[g] : prefix_start(p, g); }

  // tokens the prefix pass of group g covers: as many as its first sequence, whose pages it
  // reads, has.  A group of one shares with nobody: its tokens are its own range.
  __device__ __forceinline__ int covers(int g) const {
    if (shared) return shared[g];
    const int s0 = start(g), s1 = start(g + 1);
    if (s1 - s0 < 2) return 0;
    const int n = p.shared_lens[g], have = prefix_len(p, s0);
    return n < 0 ? 0 : n < have ? n : have;
  }

  // the last g with start(g) / div + g * mul <= x, or -1
  __device__ __forceinline__ int last(int x, int div, int mul) const {
    int lo = 0, hi = p.n_groups;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) / div + mid * mul <= x) lo = mid + 1; else hi = mid;
    }
    return lo - 1;
  }
  __device__ __forceinline__ int of(int b) const {
    const int g = last(b, 1, 0);
    return g >= 0 && b < start(g + 1) ? g : -1;
  }
};

struct PrefixRange {
  int tok0, n_tok, k_lo, k_hi, table_seq;
};

// entry e: a row tile of a group's prefix (e < n_tiles) or a sequence's own tokens.  Row
// tiles are numbered as in PackedTile.
__device__ __forceinline__ PrefixRange prefix_range(const PrefixParams& p, const PrefixGroups& gr, int e) {
  PrefixRange r{};
  if (e >= p.n_tiles) {
    const int b = e - p.n_tiles, g = gr.of(b);
    r.tok0 = r.table_seq = b;
    r.n_tok = 1;
    r.k_lo = g < 0 ? 0 : gr.covers(g);
    r.k_hi = prefix_len(p, b);
    return r;
  }
  const int g = gr.last(e, p.tile_seqs, 1);
  if (g < 0) return r;
  const int s0 = gr.start(g), s1 = gr.start(g + 1);
  const int64_t at = s0 + (int64_t)(e - (s0 / p.tile_seqs + g)) * p.tile_seqs;
  if (at >= s1) return r;
  r.tok0 = (int)at;
  r.n_tok = s1 - (int)at < p.tile_seqs ? s1 - (int)at : p.tile_seqs;
  r.k_hi = gr.covers(g);
  r.table_seq = s0;
  return r;
}

__device__ __forceinline__ int prefix_tiles(const PrefixRange& r) {
  return r.n_tok == 0 || r.k_hi <= r.k_lo ? 0 : (r.k_hi - (r.k_lo & ~15) + kArTile - 1) / kArTile;
}

constexpr int kPrefixHeld = 4096;  // most entries and groups whose plan data fits LDS (32 KB)
constexpr int kPrefixCuts = 16;    // cuts tried: 1, 17/16, ... of an even share

// Item `want`: every workgroup makes the plan for itself from the device's lengths, which
// costs less than a launch of its own.  The cut is the smallest of 16 tried (an even share
// of all tiles, up to twice that) at which the items, rounded up range by range, still run
// at once; workgroup 0 also records where each range's partials are, for the merge.
// Returns false past the last item.
__device__ __forceinline__ bool prefix_plan(const PrefixParams& p, int want, char* smem, PrefixRange* out, int* slot) {
  __shared__ long long sums[kPrefixCuts + 1];
  __shared__ int wave_n[kArThreads / 64], wave_rows[kArThreads / 64], found[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = p.n_tiles + p.batch;
  const bool held = n + 2 * (int64_t)p.n_groups + 1 <= 2 * kPrefixHeld;
  int* tiles = reinterpret_cast<int*>(smem);
  int* starts = tiles + n;
  int* shared = starts + p.n_groups + 1;
  if (tid <= kPrefixCuts) sums[tid] = 0;
  if (held)
    for (int g = tid; g <= p.n_groups && p.n_groups; g += kArThreads) starts[g] = prefix_start(p, g);
  __syncthreads();
  PrefixGroups gr{p, held ? starts : nullptr, nullptr};
  if (held) {
    for (int g = tid; g < p.n_groups; g += kArThreads) shared[g] = gr.covers(g);
    __syncthreads();
    gr.shared = shared;
  }
  long long mine = 0;
  for (int e = tid; e < n; e += kArThreads) {
    const int t = prefix_tiles(prefix_range(p, gr, e));
    if (held) tiles[e] = t;
    mine += t;
  }
  for (int s = 32; s > 0; s >>= 1) mine += __shfl_xor(mine, s, 64);
  if (lane == 0 && mine) atomicAdd(reinterpret_cast<unsigned long long*>(&sums[kPrefixCuts]), (unsigned long long)mine);
  __syncthreads();
  const long long even = (sums[kPrefixCuts] + p.target - 1) / p.target;
  auto cut_at = [&](int j) {
    const long long c = (even * (16 + j) + 15) / 16;
    return (int)(c < kPrefixMinTiles ? kPrefixMinTiles : c);
  };
  // wave w tries cuts w, w + 4, ... (batches too wide for LDS take the last: a trial is a
  // pass over them)
  for (int j = wave; j < kPrefixCuts && held; j += kArThreads / 64) {
    const u32 cut = cut_at(j);
    long long items = 0;
    for (int e = lane; e < n; e += 64) {
      const u32 t = tiles[e];
      items += (t + cut - 1) / cut;
    }
    for (int s = 32; s > 0; s >>= 1) items += __shfl_xor(items, s, 64);
    if (lane == 0) sums[j] = items;
  }
  if (tid < 8) found[tid] = -1;
  __syncthreads();
  int j = 0;
  while (j < kPrefixCuts - 1 && (!held || sums[j] > p.target)) ++j;
  const u32 cut = cut_at(j);
  int base = 0, rows0 = 0;
  for (int e0 = 0; e0 < n; e0 += kArThreads) {
    const int e = e0 + tid;
    PrefixRange r{};
    int items = 0, rows = 0, t = 0;
    if (e < n) {
      r = prefix_range(p, gr, e);
      t = prefix_tiles(r);
      items = (t + cut - 1) / cut;
      rows = r.n_tok * p.ar.group;
    }
    const int upto = wave_inclusive_scan(items), rows_upto = wave_inclusive_scan(items * rows);
    if (lane == 63) {
      wave_n[wave] = upto;
      wave_rows[wave] = rows_upto;
    }
    __syncthreads();
    int at = base + upto - items, row = rows0 + rows_upto - items * rows;
#pragma unroll
    for (int w = 0; w < kArThreads / 64; ++w) {
      if (w < wave) {
        at += wave_n[w];
        row += wave_rows[w];
      }
      base += wave_n[w];
      rows0 += wave_rows[w];
    }
    // (starts that decrease put a sequence in several tiles: past the partials' room, none)
    const bool room = row + items * rows <= p.rows;
    if (blockIdx.x == 0 && e < n) p.entries[e] = PrefixEntry{row, room ? items : 0, rows, 0};
    if (want >= at && want < at + items && room) {
      const int i = want - at, per = (t + items - 1) / items, tb = r.k_lo & ~15;
      const int lo = tb + i * per * kArTile, hi = lo + per * kArTile;
      found[0] = r.tok0;
      found[1] = r.n_tok;
      found[2] = lo < r.k_lo ? r.k_lo : lo;
      found[3] = hi < r.k_hi ? hi : r.k_hi;
      found[4] = r.table_seq;
      found[5] = row + i * rows;
    }
    __syncthreads();
    if (want < base && blockIdx.x != 0) break;
  }
  if (found[1] <= 0) return false;
  *out = PrefixRange{found[0], found[1], found[2], found[3], found[4]};
  *slot = found[5];
  return true;
}

template <int KV, int D>
__global__ __launch_bounds__(kArThreads, KV == kArF32 ? 1 : 2) void ia_shared_prefix_attend(PrefixParams p) {
  __shared__ __align__(1024) char smem[ArShape<KV, D>::kSmem];
  static_assert(ArShape<KV, D>::kSmem >= 2 * kPrefixHeld * 4, "the plan's data in the tiles' LDS");
  const int head = blockIdx.x % p.ar.n_kv_heads;
  PrefixRange x;
  int slot;
  if (!prefix_plan(p, blockIdx.x / p.ar.n_kv_heads, smem, &x, &slot)) return;
  ArItem it{};
  it.table = p.ar.kv.table ? p.ar.kv.table + (int64_t)x.table_seq * p.ar.kv.bt_stride : nullptr;
  it.head = head;
  it.tok0 = x.tok0;
  it.n_rows = x.n_tok * p.ar.group;
  it.k_lo = x.k_lo;
  it.k_hi = x.k_hi;
  it.lens = p.seq_lens;
  const int64_t row = (int64_t)head * p.rows + slot;
  it.part_ml = p.part_ml + 2 * row;
  it.part_acc = p.part_acc + row * D;
  __syncthreads();  // (the plan's data is no longer read)
  ar_attend<KV, D>(p.ar, it, smem);
}

template <int KV, int D>
int launch_prefix(const PrefixParams& p, hipStream_t st) {
  hipLaunchKernelGGL((ia_shared_prefix_attend<KV, D>), dim3((unsigned)p.max_items * p.ar.n_kv_heads), dim3(kArThreads),
                     0, st, p);
  return check_launch("shared-prefix decode");
}

}  // namespace ia
