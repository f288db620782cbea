// Shared-prefix decode, host side: argument checks, dispatch to the per-type instances
// (shared_prefix_{bf16,f32,fp8}.hip), and the merge.
#include <algorithm>

#include "shared_prefix.hpp"

namespace ia {
namespace {

constexpr int kMergeThreads = 512;
// Every workgroup plans over all sequences and groups, and there is a workgroup for each: the
// call grows with the square of the batch.  Pairs of sequences of 17-31 tokens, 8 kv heads of
// 64: 1.9 ms at 2,048 sequences, 27 ms at 8,192, 110 ms at 16,384; half a second here, minutes
// at a million.
constexpr int kPrefixMaxBatch = 1 << 15;

// One workgroup per (sequence, kv head): its rows' partials, prefix first.  A row's partials
// are dealt to the thread groups of D / 4 that share it, so a sequence of few heads still
// has every partial's load in flight at once; the groups' sums meet in LDS in order.
template <int D>
__global__ __launch_bounds__(kMergeThreads) void ia_shared_prefix_merge(PrefixParams p) {
  constexpr int kCols = D / 4, kGroups = kMergeThreads / kCols;
  __shared__ f32x4_t acc[kGroups][kCols];
  __shared__ float sum_l[kGroups];
  const int b = blockIdx.x / p.ar.n_kv_heads, head = blockIdx.x % p.ar.n_kv_heads;
  const PrefixGroups gr{p, nullptr, nullptr};
  const PrefixEntry own = p.entries[p.n_tiles + b];
  PrefixEntry pre{};
  int in_tile = 0;  // the sequence's first row in its tile's partials
  const int g = p.n_groups ? gr.of(b) : -1;
  if (g >= 0) {
    const int s0 = gr.start(g), tile = s0 / p.tile_seqs + g + (b - s0) / p.tile_seqs;
    if (tile < p.n_tiles) pre = p.entries[tile];
    in_tile = (b - s0) % p.tile_seqs * p.ar.group;
    if (in_tile + p.ar.group > pre.rows) pre.n = 0;  // (starts that decrease)
  }
  const int64_t base = (int64_t)head * p.rows;
  ArItem it{};
  it.head = head;
  it.tok0 = b;
  const int n = pre.n + own.n, per_row = kGroups / p.ar.group > 0 ? kGroups / p.ar.group : 1;
  const int grp = threadIdx.x / kCols, col = threadIdx.x % kCols, part = grp % per_row;
  const int at_once = kGroups / per_row;
  for (int r0 = 0; r0 < p.ar.group; r0 += at_once) {
    const int r = r0 + grp / per_row;
    const bool live = r < p.ar.group && grp < at_once * per_row;
    auto at = [&](int s) {
      return base + (s < pre.n ? pre.slot + s * pre.rows + in_tile + r : own.slot + (s - pre.n) * own.rows + r);
    };
    float m = kNegInf, l = 0.f;
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
    if (live) {
#pragma unroll 8
      for (int s = 0; s < n; ++s) m = fmaxf(m, p.part_ml[2 * at(s)]);
      const float mu = m == kNegInf ? 0.f : m;
#pragma unroll 4
      for (int s = part; s < n; s += per_row) {
        const int64_t row = at(s);
        const f32x2_t ml = *reinterpret_cast<const f32x2_t*>(p.part_ml + 2 * row);
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(p.part_acc + row * D + 4 * col);
        const float a = __builtin_amdgcn_exp2f(ml[0] - mu);
        l += a * ml[1];
        x += a * y;
      }
    }
    __syncthreads();  // (the last round's sums have been read)
    acc[grp][col] = x;
    if (col == 0) sum_l[grp] = l;
    __syncthreads();
    if (live && part == 0) {
      for (int s = 1; s < per_row; ++s) {
        x += acc[grp + s][col];
        l += sum_l[grp + s];
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
      ar_store4(p.ar, ar_out_row(p.ar, it, r, D) + 4 * col, y);
    }
  }
}

int check_prefix_shape(const ia_decode_shape* s, int n_groups) {
  if (!s) return fail(IA_ERR_INVALID, "shape is null");
  if (s->batch < 0 || s->n_kv_heads <= 0 || s->n_q_heads <= 0 || n_groups < 0)
    return fail(IA_ERR_INVALID, "batch and groups must be >= 0 and head counts positive");
  if (s->n_q_heads % s->n_kv_heads != 0)
    return fail(IA_ERR_INVALID, "n_q_heads must be a multiple of n_kv_heads (grouped query attention)");
  if (s->n_q_heads / s->n_kv_heads > kArMaxGroup)
    return fail(IA_ERR_UNSUPPORTED, "GQA group size must not exceed " + std::to_string(kArMaxGroup));
  if (s->head_dim != 64 && s->head_dim != 128) return fail(IA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (s->batch > kPrefixMaxBatch || n_groups > kPrefixMaxBatch)
    return fail(IA_ERR_UNSUPPORTED, "batch too large: at most " + std::to_string(kPrefixMaxBatch) + " sequences or groups");
  return check_ar_q(s->q_dtype, s->q_batch_stride, s->q_row_stride);
}

// sizes of the plan and its partials; `ws` null: the bytes alone
size_t prefix_layout(const ia_decode_shape* s, int kv_dtype, int n_groups, PrefixParams* p, char* ws) {
  const int group = s->n_q_heads / s->n_kv_heads;
  p->batch = s->batch;
  p->n_groups = n_groups;
  // Tiles of 128 rows read a prefix least often.  float32 products are as dense in tiles of
  // 32 rows, which leave no wave idle where a group does not fill 128: 16 members of 4 query
  // heads on 16,000 keys (8 kv heads of 128) 136 us against 180; 32 members, which do, 135
  // against 122 on 8,000 keys.
  p->tile_seqs = (kv_dtype == IA_F32 && group <= kArNarrow ? kArNarrow : kArRows) / group;
  p->n_tiles = n_groups ? s->batch / p->tile_seqs + n_groups : 0;
  const int resident = device_cus() * (kv_dtype == IA_F32 ? 1 : 2);
  p->target = std::max(1, resident / s->n_kv_heads);
  p->max_items = p->target + p->n_tiles + s->batch;
  // Every range has an item (a sequence is in one row tile and has its own tokens), and cuts
  // add at most target more, of a whole tile's rows where there are tiles.
  const int64_t most = n_groups ? std::min(p->tile_seqs, s->batch) : 1;
  p->rows = ((n_groups ? 2 : 1) * (int64_t)s->batch + p->target * most) * group;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* x = ws ? ws + at : nullptr;
    at += align_up(bytes, 256);
    return x;
  };
  p->entries = reinterpret_cast<PrefixEntry*>(take(sizeof(PrefixEntry) * (p->n_tiles + (size_t)s->batch)));
  p->part_ml = reinterpret_cast<float*>(take(8 * (size_t)p->rows * s->n_kv_heads));
  p->part_acc = reinterpret_cast<float*>(take(4 * (size_t)p->rows * s->n_kv_heads * s->head_dim));
  return at;
}

}  // namespace
}  // namespace ia

extern "C" {

size_t ia_shared_prefix_workspace_size(const ia_decode_shape* shape, int32_t kv_dtype, int32_t n_groups) {
  if (ia::check_prefix_shape(shape, n_groups)) return 0;
  ia::PrefixParams p{};
  return ia::prefix_layout(shape, kv_dtype, n_groups, &p, nullptr);
}

int ia_shared_prefix_decode(const ia_decode_shape* shape, const void* q, const ia_paged_kv* kv, const int32_t* seq_lens,
                            const int32_t* group_starts, const int32_t* shared_lens, int32_t n_groups, float scale,
                            void* out, int32_t out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ia;
  int rc = check_prefix_shape(shape, n_groups);
  if (rc) return rc;
  rc = check_kv(kv, shape->head_dim);
  if (rc) return rc;
  if (shape->batch == 0) return IA_OK;  // (arrays without entries have no address)
  if (!seq_lens || (n_groups && (!group_starts || !shared_lens))) return fail(IA_ERR_INVALID, "null pointer argument");
  PrefixParams p{};
  rc = set_ar_params(&p.ar, q, shape->q_dtype, shape->q_batch_stride, shape->q_row_stride,
                     shape->n_q_heads / shape->n_kv_heads, shape->n_kv_heads, kv->dtype, scale, out, out_dtype);
  if (rc) return rc;
  const size_t need = prefix_layout(shape, kv->dtype, n_groups, &p, nullptr);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(IA_ERR_WORKSPACE, "workspace missing, too small or not 256-byte aligned: " + std::to_string(need) +
                                      " bytes needed");
  prefix_layout(shape, kv->dtype, n_groups, &p, static_cast<char*>(workspace));
  set_ar_pages(&p.ar.kv, kv);
  p.kv_cap = ar_key_cap(kv);
  p.seq_lens = seq_lens;
  p.group_starts = group_starts;
  p.shared_lens = shared_lens;
  if ((int64_t)p.max_items * shape->n_kv_heads >= kArMaxGrid || p.rows >= (int64_t)1 << 31)
    return fail(IA_ERR_UNSUPPORTED, "batch too large for one launch");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int d = shape->head_dim;
  rc = kv->dtype == IA_BF16 ? launch_prefix_bf16(p, d, st)
                            : kv->dtype == IA_F32 ? launch_prefix_f32(p, d, st) : launch_prefix_fp8(p, d, st);
  if (rc) return rc;
  const dim3 grid((unsigned)shape->batch * shape->n_kv_heads);
  if (d == 128)
    hipLaunchKernelGGL((ia_shared_prefix_merge<128>), grid, dim3(kMergeThreads), 0, st, p);
  else
    hipLaunchKernelGGL((ia_shared_prefix_merge<64>), grid, dim3(kMergeThreads), 0, st, p);
  return check_launch("shared-prefix merge");
}

}  // extern "C"
