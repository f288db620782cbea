// The K/V rows of packed prompts into the paged pool for gfx950.
//
//   ia_append_prompt_rows: a workgroup per tile of one sequence's new tokens (256 threads
//   cover the 16-byte chunks of a head's row for 8, 16 or 32 tokens), looping over its
//   heads with every K and V load of a pass in flight.  A thread's token and page are
//   fixed, so the block table is read once per thread.  Bound by HBM: each row is read and
//   written once (16 prompts of 500-4,000 tokens, 8 heads of 128 bf16: 322 MB in 53.0 us,
//   6.1 TB/s); 37 tokens take 3.3 us, a workgroup per head and 16 of them.
#include <algorithm>

#include "packed_rows.hpp"
#include "row_spans.hpp"

namespace ia {

int check_kv(const ia_paged_kv* kv, int d);

namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendHeads = 4;  // heads whose loads are in flight together

struct PromptAppendParams {
  char* k;
  char* v;
  int64_t k_page, k_head, k_tok, v_page, v_head, v_tok;  // bytes
  const char* k_new;
  const char* v_new;
  int64_t kn_tok, kn_head, vn_tok, vn_head;              // bytes
  const int32_t* table;
  int64_t bt_stride, bt_cols, n_pages;
  int32_t page_rows;
  const int32_t* cu;
  const int32_t* seq_lens;
  int32_t* new_lens;
  int32_t n_seq, n_tokens, n_kv_heads, heads_per_wg;
  int32_t chunks;      // 16-byte chunks of a head's row
  int32_t tile;        // tokens of a tile
};

__device__ __forceinline__ int64_t page_at(const PromptAppendParams& p, int b, int64_t lp) {
  int64_t pg = lp;
  if (p.table) pg = lp < p.bt_cols ? p.table[(int64_t)b * p.bt_stride + lp] : -1;
  return pg < 0 || pg >= p.n_pages ? -1 : pg;
}

__global__ __launch_bounds__(kAppendThreads) void ia_append_prompt_rows(PromptAppendParams p) {
  __shared__ int first_gap;
  const int tid = threadIdx.x;
  const PackedTile t = packed_tile(p.cu, p.n_seq, p.n_tokens, p.tile, blockIdx.x, tid & 63);
  if (t.local < 0) return;
  const int64_t past = p.seq_lens[t.b];
  if (t.local == 0 && blockIdx.y == 0) {
    // the length: up to the first position without a page
    if (tid == 0) first_gap = INT32_MAX;
    __syncthreads();
    const int64_t end = past + t.count;
    if (past >= 0 && t.count > 0)
      for (int64_t lp = past / p.page_rows + tid; lp * p.page_rows < end; lp += kAppendThreads)
        if (page_at(p, t.b, lp) < 0) {
          atomicMin(&first_gap, (int)lp);
          break;
        }
    __syncthreads();
    if (tid == 0) {
      int64_t len = past;
      if (past >= 0) {
        const int64_t gap = (int64_t)first_gap * p.page_rows;
        len = end < gap ? end : past > gap ? past : gap;
      }
      p.new_lens[t.b] = (int)len;
    }
  }
  const int tok = tid / p.chunks, off = (tid % p.chunks) * 16;
  if (tok >= t.n_tok || past < 0) return;
  const int64_t pos = past + t.local * (int64_t)p.tile + tok;
  const int64_t lp = pos / p.page_rows, pg = page_at(p, t.b, lp);
  if (pg < 0) return;
  const int64_t in = pos - lp * p.page_rows;
  const int h0 = blockIdx.y * p.heads_per_wg, h1 = min(h0 + p.heads_per_wg, p.n_kv_heads);
  const char* ks = p.k_new + (t.tok0 + tok) * p.kn_tok + off;
  const char* vs = p.v_new + (t.tok0 + tok) * p.vn_tok + off;
  char* kd = p.k + pg * p.k_page + in * p.k_tok + off;
  char* vd = p.v + pg * p.v_page + in * p.v_tok + off;
  for (int h = h0; h < h1; h += kAppendHeads) {
    u32x4_t a[kAppendHeads], b[kAppendHeads];
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i)
      if (h + i < h1) {
        a[i] = ld_stream16(ks + (h + i) * p.kn_head);
        b[i] = ld_stream16(vs + (h + i) * p.vn_head);
      }
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i)
      if (h + i < h1) {
        *reinterpret_cast<u32x4_t*>(kd + (h + i) * p.k_head) = a[i];
        *reinterpret_cast<u32x4_t*>(vd + (h + i) * p.v_head) = b[i];
      }
  }
}

}  // namespace
}  // namespace ia

extern "C" int ia_append_prompt_kv(const ia_paged_kv* kv, const ia_packed_kv* rows, const int32_t* cu_seqlens,
                                   const int32_t* seq_lens, int32_t* new_seq_lens, int32_t n_seq, int32_t n_tokens,
                                   int32_t n_kv_heads, int32_t head_dim, void* stream) {
  using namespace ia;
  // (arrays without entries have no address)
  if (!rows || (n_seq > 0 && (!cu_seqlens || !seq_lens || !new_seq_lens)))
    return fail(IA_ERR_INVALID, "null pointer argument");
  if (head_dim != 64 && head_dim != 128) return fail(IA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (kv && kv->dtype != IA_F32 && kv->dtype != IA_BF16)
    return fail(IA_ERR_UNSUPPORTED, "append takes bf16 or f32 pools");
  int rc = check_kv(kv, head_dim);
  if (rc) return rc;
  if (rows->dtype != kv->dtype) return fail(IA_ERR_INVALID, "the new rows must have the pool's dtype");
  if (n_seq < 0 || n_tokens < 0 || n_kv_heads <= 0) return fail(IA_ERR_INVALID, "sequence, token or head counts");
  if (n_tokens > 0 && (!rows->k || !rows->v)) return fail(IA_ERR_INVALID, "null pointer argument");
  if (n_seq > 0 && new_seq_lens == seq_lens) return fail(IA_ERR_INVALID, "new_seq_lens must not be seq_lens");
  const int eb = kv->dtype == IA_F32 ? 4 : 2;
  const int64_t strides[4] = {rows->k_token_stride, rows->k_head_stride, rows->v_token_stride, rows->v_head_stride};
  for (int64_t s : strides)
    if (s < 0 || (s * eb) % 16) return fail(IA_ERR_INVALID, "row strides must be non-negative 16-byte multiples");
  if ((reinterpret_cast<uintptr_t>(rows->k) | reinterpret_cast<uintptr_t>(rows->v)) % 16)
    return fail(IA_ERR_INVALID, "rows must be 16-byte aligned");
  if (n_seq == 0) return IA_OK;
  PromptAppendParams p{};
  p.k = static_cast<char*>(const_cast<void*>(kv->k));
  p.v = static_cast<char*>(const_cast<void*>(kv->v));
  p.k_page = kv->k_page_stride * eb;
  p.k_head = kv->k_head_stride * eb;
  p.k_tok = kv->k_token_stride * eb;
  p.v_page = kv->v_page_stride * eb;
  p.v_head = kv->v_head_stride * eb;
  p.v_tok = kv->v_token_stride * eb;
  p.k_new = static_cast<const char*>(rows->k);
  p.v_new = static_cast<const char*>(rows->v);
  p.kn_tok = rows->k_token_stride * eb;
  p.kn_head = rows->k_head_stride * eb;
  p.vn_tok = rows->v_token_stride * eb;
  p.vn_head = rows->v_head_stride * eb;
  p.table = kv->block_table;
  p.bt_stride = kv->bt_stride;
  p.bt_cols = kv->bt_cols;
  p.n_pages = kv->n_pages;
  p.page_rows = kv->page_size;
  p.cu = cu_seqlens;
  p.seq_lens = seq_lens;
  p.new_lens = new_seq_lens;
  p.n_seq = n_seq;
  p.n_tokens = n_tokens;
  p.n_kv_heads = n_kv_heads;
  p.chunks = head_dim * eb / 16;
  p.tile = kAppendThreads / p.chunks;
  const int64_t tiles = (int64_t)n_tokens / p.tile + n_seq;
  if (tiles >= (int64_t)1 << 23) return fail(IA_ERR_UNSUPPORTED, "too many tokens for one launch");
  // few tiles: a workgroup per head, so that a short prompt is one round trip
  p.heads_per_wg = tiles >= 2 * device_cus() ? n_kv_heads : 1;
  const dim3 grid((unsigned)tiles, (unsigned)((n_kv_heads + p.heads_per_wg - 1) / p.heads_per_wg));
  // (a sequence's length is written while other workgroups still read theirs, and where they begin)
  if (ints_meet(new_seq_lens, n_seq, seq_lens, n_seq))
    return fail(IA_ERR_INVALID, "new_seq_lens must not overlap seq_lens");
  if (ints_meet(new_seq_lens, n_seq, cu_seqlens, (int64_t)n_seq + 1))
    return fail(IA_ERR_INVALID, "new_seq_lens must not overlap cu_seqlens");
  hipLaunchKernelGGL(ia_append_prompt_rows, grid, dim3(kAppendThreads), 0, static_cast<hipStream_t>(stream), p);
  return check_launch("append prompt kv");
}
