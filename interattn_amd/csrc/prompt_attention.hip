// Prompt attention, host side: argument checks, how far the keys are cut, dispatch to the
// per-type instances (prompt_attention_{bf16,f32,fp8}.hip), and the merge of cut rows.
#include <algorithm>
#include <cstdlib>

#include "prompt_attention.hpp"

namespace ia {

// Rows of tiles whose keys were cut: their slices' partials, in slice order.
template <int D>
__global__ __launch_bounds__(kArThreads) void ia_prompt_merge(PromptParams p) {
  const int head = blockIdx.x % p.ar.n_kv_heads, tile = blockIdx.x / p.ar.n_kv_heads;
  const PackedTile t = prompt_tile(p, tile, threadIdx.x & 63);
  if (t.n_tok == 0) return;
  int limit0, k_end;
  prompt_keys(p, t, &limit0, &k_end);
  const int n = prompt_slices(p, (k_end + kArTile - 1) / kArTile);
  if (n <= 1) return;
  const int64_t slot = ((int64_t)tile * p.ar.n_kv_heads + head) * p.slices;
  ArItem it{};
  it.head = head;
  it.tok0 = t.tok0;
  const int rows = t.n_tok * p.ar.group;
  for (int i = threadIdx.x; i < rows * (D / 4); i += kArThreads) {
    const int r = i / (D / 4), e = (i % (D / 4)) * 4;
    float m = kNegInf;
    for (int s = 0; s < n; ++s) m = fmaxf(m, p.part_ml[((slot + s) * p.tile_rows + r) * 2]);
    const float mu = m == kNegInf ? 0.f : m;
    float l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < n; ++s) {
      const f32x2_t ml = *reinterpret_cast<const f32x2_t*>(p.part_ml + ((slot + s) * p.tile_rows + r) * 2);
      const float a = __builtin_amdgcn_exp2f(ml[0] - mu);
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(p.part_acc + ((slot + s) * p.tile_rows + r) * D + e);
      l += a * ml[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += a * y[j];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= inv;
    ar_store4(p.ar, ar_out_row(p.ar, it, r, D) + e, x);
  }
}

namespace {

constexpr int kPromptMaxSlices = 64;

// Fewest key tiles a slice is worth.  Merging 128 rows takes as long as ten key tiles of
// bf16 or fp8 products (1,000 tokens in halves of 8 tiles 50 us, uncut 33), but as two of
// float32's (eight of 1-500 tokens at 0-1,500 keys: 8 tiles 79, 16 tiles 104); with tiles of
// 32 rows, 16 instead of 8 took 33 us for 27 (16 tokens at 4,000 keys).
int least_key_tiles(int kv_dtype, int rows) { return rows == kArNarrow || kv_dtype == IA_F32 ? 8 : 16; }

int check_prompt_shape(const ia_prompt_shape* s) {
  if (!s) return fail(IA_ERR_INVALID, "shape is null");
  if (s->n_seq < 0 || s->n_tokens < 0 || s->n_q_heads <= 0 || s->n_kv_heads <= 0)
    return fail(IA_ERR_INVALID, "sequence and token counts must be >= 0 and head counts positive");
  if (s->n_q_heads % s->n_kv_heads != 0)
    return fail(IA_ERR_INVALID, "n_q_heads must be a multiple of n_kv_heads (grouped query attention)");
  if (s->n_q_heads / s->n_kv_heads > kArMaxGroup)
    return fail(IA_ERR_UNSUPPORTED, "GQA group size must not exceed " + std::to_string(kArMaxGroup));
  if (s->head_dim != 64 && s->head_dim != 128) return fail(IA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  return check_ar_q(s->q_dtype, s->q_token_stride, s->q_head_stride);
}

int64_t resident_wgs(int kv_dtype) { return (int64_t)device_cus() * (kv_dtype == IA_F32 ? 1 : 2); }

// Row tiles (a bound from the token and sequence counts alone), and the slices their keys
// may be cut into.  Times are of the launches alone, in us, groups of 4, D = 128 unless said.
//
// Tiles of 128 rows read K/V least often and keep the matrix cores busiest; tiles of 32
// rows spread a key tile over four waves, a quarter of the time for each.  They pay where
// all of them run at once and, over bf16 and fp8 caches, the keys are long enough to be cut
// but 128-row tiles, cut or not, leave a quarter of the device idle.  bf16, 8 kv heads, 32
// rows / 128: 16 tokens at 4,000 keys 28 / 35, 64 at 8,000 55 / 95, four of 32 at 2,000
// 38 / 58; but prompts of 333 tokens 19 / 17, of 1,000 49 / 33, and four of 64 tokens at
// 8,000 keys 113 / 112.  float32, whose products are as dense in both (4 kv heads of 64):
// one prompt of 500 25 / 47, four of 500 (1,016 tiles of 32 for 256 places) 66 / 50.
//
// Keys are cut into as many slices as all run at once.  One more round of workgroups undoes
// the gain (five of 320 tokens at 8,000 keys, 400 tiles: uncut 277, halves 308).  In
// place: 256 tokens at 32,000 keys, 64 tiles, 8 slices 216 against 841; four of 256 at
// 20,000, 256 tiles in halves 423 against 634; eight single tokens at 8,000 keys 55 against
// 153.
void prompt_grid(const ia_prompt_shape* s, int kv_dtype, int64_t most_keys, PromptParams* p) {
  const int group = s->n_q_heads / s->n_kv_heads;
  const int64_t resident = resident_wgs(kv_dtype);
  const int64_t key_tiles = (most_keys + kArTile - 1) / kArTile;
  auto slices = [&](int rows) {
    const int least = least_key_tiles(kv_dtype, rows);
    return (key_tiles + least - 1) / least;
  };
  // tiles of `rows` rows, at least: one for each sequence, as many as whole ones hold
  auto tiles_of = [&](int rows) {
    return std::max<int64_t>(s->n_tokens / (rows / group), std::min(s->n_seq, s->n_tokens)) * s->n_kv_heads;
  };
  const bool small =
      group <= kArNarrow && tiles_of(kArNarrow) <= resident &&
      (kv_dtype == IA_F32 || (key_tiles > least_key_tiles(kv_dtype, kArNarrow) &&
                              4 * tiles_of(kArRows) * std::min(slices(kArRows), resident) <= 3 * resident));
  p->tile_rows = small ? kArNarrow : kArRows;
  p->tile_tokens = p->tile_rows / group;
  p->n_tiles = (int)std::min<int64_t>((int64_t)s->n_tokens / p->tile_tokens + s->n_seq, INT32_MAX);
  p->slice_tiles = least_key_tiles(kv_dtype, p->tile_rows);
  const int64_t bound = std::max<int64_t>(1, (int64_t)p->n_tiles * s->n_kv_heads);
  int64_t n = resident / std::max<int64_t>(1, tiles_of(p->tile_rows));
  n = std::min<int64_t>(n, kPromptMaxSlices);
  n = std::min<int64_t>(n, 2 * resident / bound);
  n = std::min(n, slices(p->tile_rows));
  p->slices = (int)std::max<int64_t>(1, n);
}

// One size for every call that cuts (a cut call has at most two slices per resident
// workgroup), so a buffer kept from call to call never has to be replaced by a larger one
// while a captured graph still uses it.
size_t prompt_ws_size(const ia_prompt_shape* s, int kv_dtype, const PromptParams& p) {
  return p.slices <= 1 ? 0 : (size_t)(2 * resident_wgs(kv_dtype)) * kArRows * (s->head_dim + 2) * 4;
}

int run_prompt(const ia_prompt_shape* s, const void* q, int kv_dtype, PromptParams& p, const int32_t* cu, float scale,
               void* out, int32_t out_dtype, void* workspace, size_t workspace_bytes, int64_t most_keys,
               hipStream_t st) {
  int rc = set_ar_params(&p.ar, q, s->q_dtype, s->q_token_stride, s->q_head_stride, s->n_q_heads / s->n_kv_heads,
                         s->n_kv_heads, kv_dtype, scale, out, out_dtype);
  if (rc) return rc;
  if (!cu) return fail(IA_ERR_INVALID, "null pointer argument");
  if (s->n_seq == 0 || s->n_tokens == 0) return IA_OK;
  p.cu = cu;
  p.n_seq = s->n_seq;
  p.n_tokens = s->n_tokens;
  prompt_grid(s, kv_dtype, most_keys, &p);
  if ((int64_t)p.n_tiles * s->n_kv_heads * p.slices >= kArMaxGrid)
    return fail(IA_ERR_UNSUPPORTED, "too many row tiles for one launch");
  const size_t need = prompt_ws_size(s, kv_dtype, p);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(IA_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned: " + std::to_string(need) +
                                      " bytes needed");
  p.part_acc = reinterpret_cast<float*>(workspace);
  if (need) p.part_ml = p.part_acc + (size_t)p.n_tiles * s->n_kv_heads * p.slices * p.tile_rows * s->head_dim;
  const int d = s->head_dim;
  rc = kv_dtype == IA_BF16 ? launch_prompt_bf16(p, d, st)
                           : kv_dtype == IA_F32 ? launch_prompt_f32(p, d, st) : launch_prompt_fp8(p, d, st);
  if (rc || p.slices <= 1) return rc;
  const dim3 grid((unsigned)p.n_tiles * s->n_kv_heads);
  if (d == 128)
    hipLaunchKernelGGL((ia_prompt_merge<128>), grid, dim3(kArThreads), 0, st, p);
  else
    hipLaunchKernelGGL((ia_prompt_merge<64>), grid, dim3(kArThreads), 0, st, p);
  return check_launch("prompt merge");
}

}  // namespace

int check_ar_q(int q_dtype, int64_t q_tok, int64_t q_head) {
  if (q_dtype != IA_F32 && q_dtype != IA_BF16) return fail(IA_ERR_INVALID, "q dtype must be IA_F32 or IA_BF16");
  const int eb = q_dtype == IA_F32 ? 4 : 2;
  if (q_tok < 0 || q_head < 0 || (q_tok * eb) % 16 || (q_head * eb) % 16)
    return fail(IA_ERR_INVALID, "q strides must be non-negative 16-byte multiples");
  return IA_OK;
}

int set_ar_params(ArParams* p, const void* q, int q_dtype, int64_t q_tok, int64_t q_head, int group, int n_kv_heads,
                  int kv_dtype, float scale, void* out, int out_dtype) {
  if (!q || !out) return fail(IA_ERR_INVALID, "null pointer argument");
  if (out_dtype != IA_F32 && out_dtype != IA_BF16) return fail(IA_ERR_INVALID, "out dtype must be IA_F32 or IA_BF16");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16)
    return fail(IA_ERR_INVALID, "q and out must be 16-byte aligned");
  if (kv_dtype == IA_F32 && q_dtype != IA_F32) return fail(IA_ERR_UNSUPPORTED, "fp32 kv needs fp32 q");
  if (kv_dtype != IA_F32 && q_dtype == IA_F32 && kv_dtype == IA_FP8_E4M3)
    return fail(IA_ERR_UNSUPPORTED, "fp8 kv needs bf16 q");
  if (!(std::fabs(scale) < __builtin_huge_valf())) return fail(IA_ERR_INVALID, "scale must be finite");
  p->q = q;
  p->q_tok = q_tok;
  p->q_head = q_head;
  p->out = out;
  p->out_f32 = out_dtype == IA_F32;
  p->q_f32 = q_dtype == IA_F32;
  p->group = group;
  p->n_kv_heads = n_kv_heads;
  p->scale_log2 = std::fabs(scale) * kLog2e;
  p->q_flip = scale < 0 ? 0x8000u : 0u;
  return IA_OK;
}

void set_ar_pages(ArSource* s, const ia_paged_kv* kv) {
  const int eb = kv->dtype == IA_F32 ? 4 : (kv->dtype == IA_BF16 ? 2 : 1);
  s->k = static_cast<const char*>(kv->k);
  s->v = static_cast<const char*>(kv->v);
  s->k_page = kv->k_page_stride * eb;
  s->k_head = kv->k_head_stride * eb;
  s->k_tok = kv->k_token_stride * eb;
  s->v_page = kv->v_page_stride * eb;
  s->v_head = kv->v_head_stride * eb;
  s->v_tok = kv->v_token_stride * eb;
  s->table = kv->block_table;
  s->bt_stride = kv->bt_stride;
  s->bt_cols = kv->bt_cols;
  s->n_pages = kv->n_pages;
  s->page_rows = kv->page_size;
  s->k_scale = kv->k_scale;
  s->v_scale = kv->v_scale;
  s->scale_page = kv->scale_page_stride;
}

int64_t ar_key_cap(const ia_paged_kv* kv) {
  const int64_t keys = (kv->block_table ? kv->bt_cols : kv->n_pages) * (int64_t)kv->page_size;
  return std::min<int64_t>(keys, INT32_MAX - 1024);
}

}  // namespace ia

extern "C" {

size_t ia_prompt_attention_workspace_size(const ia_prompt_shape* shape, int32_t kv_dtype, int64_t max_keys) {
  if (ia::check_prompt_shape(shape)) return 0;
  ia::PromptParams p{};
  ia::prompt_grid(shape, kv_dtype, max_keys, &p);
  return ia::prompt_ws_size(shape, kv_dtype, p);
}

int ia_prompt_attention(const ia_prompt_shape* shape, const void* q, const ia_packed_kv* kv, const int32_t* cu_seqlens,
                        float scale, void* out, int32_t out_dtype, void* workspace, size_t workspace_bytes,
                        void* stream) {
  using namespace ia;
  int rc = check_prompt_shape(shape);
  if (rc) return rc;
  if (!kv || !kv->k || !kv->v) return fail(IA_ERR_INVALID, "k and v must be non-null");
  if (kv->dtype != IA_F32 && kv->dtype != IA_BF16) return fail(IA_ERR_UNSUPPORTED, "packed k and v are bf16 or f32");
  const int eb = kv->dtype == IA_F32 ? 4 : 2;
  const int64_t strides[4] = {kv->k_token_stride, kv->k_head_stride, kv->v_token_stride, kv->v_head_stride};
  for (int64_t s : strides)
    if (s < 0 || (s * eb) % 16) return fail(IA_ERR_INVALID, "k and v strides must be non-negative 16-byte multiples");
  if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) % 16)
    return fail(IA_ERR_INVALID, "k and v must be 16-byte aligned");
  PromptParams p{};
  ArSource& s = p.ar.kv;
  s.k = static_cast<const char*>(kv->k);
  s.v = static_cast<const char*>(kv->v);
  s.k_tok = kv->k_token_stride * eb;
  s.k_head = kv->k_head_stride * eb;
  s.v_tok = kv->v_token_stride * eb;
  s.v_head = kv->v_head_stride * eb;
  s.k_page = 16 * s.k_tok;
  s.v_page = 16 * s.v_tok;
  s.n_pages = INT64_MAX;
  s.page_rows = 16;
  // (what is cut for: a sequence of the mean length)
  const int64_t keys = shape->n_seq ? ((int64_t)shape->n_tokens + shape->n_seq - 1) / shape->n_seq : 0;
  return run_prompt(shape, q, kv->dtype, p, cu_seqlens, scale, out, out_dtype, workspace, workspace_bytes, keys,
                    static_cast<hipStream_t>(stream));
}

int ia_paged_prompt_attention(const ia_prompt_shape* shape, const void* q, const ia_paged_kv* kv,
                              const int32_t* seq_lens, const int32_t* cu_seqlens, float scale, void* out,
                              int32_t out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ia;
  int rc = check_prompt_shape(shape);
  if (rc) return rc;
  rc = check_kv(kv, shape->head_dim);
  if (rc) return rc;
  if (!seq_lens) return fail(IA_ERR_INVALID, "null pointer argument");
  PromptParams p{};
  set_ar_pages(&p.ar.kv, kv);
  p.seq_lens = seq_lens;
  p.kv_cap = ar_key_cap(kv);
  return run_prompt(shape, q, kv->dtype, p, cu_seqlens, scale, out, out_dtype, workspace, workspace_bytes, p.kv_cap,
                    static_cast<hipStream_t>(stream));
}

}  // extern "C"
