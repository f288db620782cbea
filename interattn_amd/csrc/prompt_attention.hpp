// Causal attention of packed prompts: parameters shared by the host side and the per-type
// kernel instances.
//
// 4 D flops per visible (row, key) pair, on the matrix cores.  Two prompts of 8,192 tokens (8
// kv heads of 128, groups of 4, bf16) take 1,192 us, 920 TFLOP/s: of the cycles that a SIMD
// has work, the matrix unit is busy 44% and a vector instruction issues in 54%, so the
// products and the softmax take turns.  At D = 64 (24 prompts of 1-2,000 tokens, groups of 8:
// 218 us, 570 TFLOP/s) the vector side is 72% and the matrix side 29%.
#pragma once

#include "attend_rows.hpp"
#include "packed_rows.hpp"

namespace ia {

struct PromptParams {
  ArParams ar;
  const int32_t* cu;        // [n_seq + 1] first token of each sequence in q
  const int32_t* seq_lens;  // paged: [n_seq] keys of each sequence; null: its own tokens
  int64_t kv_cap;           // paged: keys a block-table row can hold
  int32_t n_seq, n_tokens;
  int32_t tile_rows;        // rows of a row tile: 128 or 32
  int32_t tile_tokens;      // its tokens, tile_rows / group
  int32_t n_tiles;          // bound over all sequences
  int32_t slices;           // most key slices of a row tile
  int32_t slice_tiles;      // fewest key tiles a slice is worth
  float* part_ml;
  float* part_acc;
};

// slices the keys of a row tile are cut into
__host__ __device__ inline int prompt_slices(const PromptParams& p, int key_tiles) {
  int n = (key_tiles + p.slice_tiles - 1) / p.slice_tiles;
  return n < 1 ? 1 : n > p.slices ? p.slices : n;
}

int launch_prompt_bf16(const PromptParams& p, int d, hipStream_t st);
int launch_prompt_f32(const PromptParams& p, int d, hipStream_t st);
int launch_prompt_fp8(const PromptParams& p, int d, hipStream_t st);

__device__ __forceinline__ PackedTile prompt_tile(const PromptParams& p, int tile, int lane) {
  return packed_tile(p.cu, p.n_seq, p.n_tokens, p.tile_tokens, tile, lane);
}

// keys the tile's last row sees, and the first row's limit
__device__ __forceinline__ void prompt_keys(const PromptParams& p, const PackedTile& t, int* limit0, int* k_hi) {
  int64_t total = t.count;
  if (p.seq_lens) total = p.seq_lens[t.b];
  const int64_t first = total - t.count + (t.tok0 - t.first) + 1;  // keys the tile's first token sees
  *limit0 = (int)first;
  int64_t hi = first + t.n_tok - 1;
  if (p.seq_lens && hi > p.kv_cap) hi = p.kv_cap;
  *k_hi = hi < 0 ? 0 : (int)hi;
}

template <int KV, int D>
__global__ __launch_bounds__(kArThreads, KV == kArF32 ? 1 : 2) void ia_prompt_attention(PromptParams p) {
  __shared__ __align__(1024) char smem[ArShape<KV, D>::kSmem];
  // heads fastest, so that with 2^n heads a head's tiles share XCDs (their L2 holds its
  // K/V); later tiles of the batch, which see more keys, first
  int id = blockIdx.x;
  const int head = id % p.ar.n_kv_heads;
  id /= p.ar.n_kv_heads;
  const int slice = id % p.slices, tile = p.n_tiles - 1 - id / p.slices;
  const PackedTile t = prompt_tile(p, tile, threadIdx.x & 63);
  if (t.n_tok == 0) return;
  ArItem it{};
  int k_end = 0;
  prompt_keys(p, t, &it.limit0, &k_end);
  const int key_tiles = (k_end + kArTile - 1) / kArTile;
  const int n = prompt_slices(p, key_tiles);
  if (slice >= n) return;
  const int per = (key_tiles + n - 1) / n;
  it.k_lo = slice * per * kArTile;
  it.k_hi = (slice + 1) * per * kArTile < k_end ? (slice + 1) * per * kArTile : k_end;
  it.table = p.ar.kv.table ? p.ar.kv.table + (int64_t)t.b * p.ar.kv.bt_stride : nullptr;
  it.row0 = p.seq_lens ? 0 : t.first;
  it.head = head;
  it.tok0 = t.tok0;
  it.n_rows = t.n_tok * p.ar.group;
  if (n > 1) {
    const int64_t slot = ((int64_t)tile * p.ar.n_kv_heads + head) * p.slices + slice;
    it.part_ml = p.part_ml + slot * p.tile_rows * 2;
    it.part_acc = p.part_acc + slot * p.tile_rows * D;
  }
  ar_attend<KV, D>(p.ar, it, smem);
}

template <int KV, int D>
int launch_prompt(const PromptParams& p, hipStream_t st) {
  const unsigned tiles = (unsigned)p.n_tiles * p.ar.n_kv_heads;
  hipLaunchKernelGGL((ia_prompt_attention<KV, D>), dim3(tiles * p.slices), dim3(kArThreads), 0, st, p);
  return check_launch("prompt attention");
}

}  // namespace ia
