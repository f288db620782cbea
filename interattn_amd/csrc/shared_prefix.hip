// Shared-prefix decode, host side: argument checks, the plan that cuts the ranges into
// items, dispatch to the per-type instances (shared_prefix_{bf16,f32,fp8}.hip), the merge.
#include <algorithm>

#include "shared_prefix.hpp"

namespace ia {
namespace {

constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int group_start(const PrefixParams& p, int g) {
  const int s = p.group_starts[g];
  return s < 0 ? 0 : s > p.batch ? p.batch : s;
}

__device__ __forceinline__ int seq_len(const PrefixParams& p, int b) {
  const int n = p.seq_lens[b];
  return n < 0 ? 0 : n > p.kv_cap ? (int)p.kv_cap : n;
}

// tokens group g's prefix pass covers: as many as its first sequence, whose pages it reads,
// has.  A group of one shares with nobody: its tokens are all its own range.
__device__ __forceinline__ int group_shared(const PrefixParams& p, int g) {
  const int s0 = group_start(p, g), s1 = group_start(p, g + 1);
  if (s1 - s0 < 2) return 0;
  const int n = p.shared_lens[g], have = seq_len(p, s0);
  return n < 0 ? 0 : n < have ? n : have;
}

// the last group that starts at or before sequence b, where b lies in it; else -1
__device__ __forceinline__ int group_of(const PrefixParams& p, int b) {
  int lo = 0, hi = p.n_groups;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (group_start(p, mid) <= b) lo = mid + 1; else hi = mid;
  }
  const int g = lo - 1;
  return g >= 0 && b < group_start(p, g + 1) ? g : -1;
}

struct Range {
  int tok0, n_tok, k_lo, k_hi, table_seq;
};

// entry e: a row tile of a group's prefix (e < n_tiles) or a sequence's own tokens
__device__ __forceinline__ Range plan_range(const PrefixParams& p, int e) {
  Range r{};
  if (e >= p.n_tiles) {
    const int b = e - p.n_tiles, g = group_of(p, b);
    r.tok0 = r.table_seq = b;
    r.n_tok = 1;
    r.k_lo = g < 0 ? 0 : group_shared(p, g);
    r.k_hi = seq_len(p, b);
    return r;
  }
  int lo = 0, hi = p.n_groups;  // the last group whose tiles start at or before e
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (group_start(p, mid) / p.tile_seqs + mid <= e) lo = mid + 1; else hi = mid;
  }
  const int g = lo - 1;
  if (g < 0) return r;
  const int s0 = group_start(p, g), s1 = group_start(p, g + 1);
  const int64_t at = s0 + (int64_t)(e - (s0 / p.tile_seqs + g)) * p.tile_seqs;
  if (at >= s1) return r;
  r.tok0 = (int)at;
  r.n_tok = s1 - (int)at < p.tile_seqs ? s1 - (int)at : p.tile_seqs;
  r.k_hi = group_shared(p, g);
  r.table_seq = s0;
  return r;
}

__device__ __forceinline__ int range_tiles(const Range& r) {
  return r.n_tok == 0 || r.k_hi <= r.k_lo ? 0 : (r.k_hi - (r.k_lo & ~15) + kArTile - 1) / kArTile;
}

// Cuts the ranges into items of at most `cut` key tiles, cut = all tiles over the items the
// device runs at once.  One workgroup: a batch has few ranges.
__global__ __launch_bounds__(kPlanThreads) void ia_shared_prefix_plan(PrefixParams p) {
  __shared__ int wave_a[kPlanThreads / 64], wave_b[kPlanThreads / 64];
  __shared__ long long total;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = p.n_tiles + p.batch;
  if (tid == 0) total = 0;
  __syncthreads();
  long long mine = 0;
  for (int e = tid; e < n; e += kPlanThreads) mine += range_tiles(plan_range(p, e));
  for (int s = 32; s > 0; s >>= 1) mine += __shfl_xor(mine, s, 64);
  if (lane == 0 && mine) atomicAdd(reinterpret_cast<unsigned long long*>(&total), (unsigned long long)mine);
  __syncthreads();
  long long cut = (total + p.target - 1) / p.target;
  if (cut < kPrefixMinTiles) cut = kPrefixMinTiles;
  int base = 0, slot = 0;
  for (int e0 = 0; e0 < n; e0 += kPlanThreads) {
    const int e = e0 + tid;
    Range r{};
    int tiles = 0;
    if (e < n) {
      r = plan_range(p, e);
      tiles = range_tiles(r);
    }
    const int items = (int)((tiles + cut - 1) / cut), rows = r.n_tok * p.ar.group;
    const int ia = wave_inclusive_scan(items), ib = wave_inclusive_scan(items * rows);
    if (lane == 63) {
      wave_a[wave] = ia;
      wave_b[wave] = ib;
    }
    __syncthreads();
    int at = base + ia - items, row = slot + ib - items * rows;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) {
        at += wave_a[w];
        row += wave_b[w];
      }
      base += wave_a[w];
      slot += wave_b[w];
    }
    if (e < n) {
      p.entries[e] = PrefixEntry{row, items, rows, 0};
      if (e >= p.n_tiles) {
        const int b = e - p.n_tiles, g = group_of(p, b);
        int t = -1;
        if (g >= 0) {
          const int s0 = group_start(p, g);
          t = s0 / p.tile_seqs + g + (b - s0) / p.tile_seqs;
        }
        p.tile_of[b] = t < p.n_tiles ? t : -1;
      }
      const int per = items ? (tiles + items - 1) / items : 0, tb = r.k_lo & ~15;
      for (int i = 0; i < items; ++i) {
        const int lo = tb + i * per * kArTile, hi = lo + per * kArTile;
        if (at + i < p.max_items)
          p.items[at + i] = PrefixItem{r.tok0, r.n_tok, lo < r.k_lo ? r.k_lo : lo, hi < r.k_hi ? hi : r.k_hi,
                                       r.table_seq, row + i * rows, 0, 0};
      }
    }
    __syncthreads();
  }
  if (tid == 0) *p.n_items = base < p.max_items ? base : p.max_items;
}

// One workgroup per (sequence, kv head): its rows' partials, prefix first.
template <int D>
__global__ __launch_bounds__(kArThreads) void ia_shared_prefix_merge(PrefixParams p) {
  const int b = blockIdx.x / p.ar.n_kv_heads, head = blockIdx.x % p.ar.n_kv_heads;
  const int tile = p.tile_of[b];
  PrefixEntry pre{}, own = p.entries[p.n_tiles + b];
  int in_tile = 0;  // the sequence's first row in its tile's partials
  if (tile >= 0) {
    pre = p.entries[tile];
    in_tile = (b - group_start(p, group_of(p, b))) % p.tile_seqs * p.ar.group;
    if (in_tile + p.ar.group > pre.rows) pre.n = 0;  // (starts that decrease)
  }
  const int64_t base = (int64_t)head * p.rows;
  ArItem it{};
  it.head = head;
  it.tok0 = b;
  const int n = pre.n + own.n;
  for (int i = threadIdx.x; i < p.ar.group * (D / 4); i += kArThreads) {
    const int r = i / (D / 4), e = (i % (D / 4)) * 4;
    auto at = [&](int s) {
      return base + (s < pre.n ? pre.slot + s * pre.rows + in_tile + r : own.slot + (s - pre.n) * own.rows + r);
    };
    float m = kNegInf;
    for (int s = 0; s < n; ++s) m = fmaxf(m, p.part_ml[2 * at(s)]);
    const float mu = m == kNegInf ? 0.f : m;
    float l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < n; ++s) {
      const int64_t row = at(s);
      const float a = __builtin_amdgcn_exp2f(p.part_ml[2 * row] - mu);
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(p.part_acc + row * D + e);
      l += a * p.part_ml[2 * row + 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += a * y[j];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= inv;
    ar_store4(p.ar, ar_out_row(p.ar, it, r, D) + e, x);
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
  if ((int64_t)s->batch + n_groups > 1 << 20) return fail(IA_ERR_UNSUPPORTED, "batch too large for one plan");
  return check_ar_q(s->q_dtype, s->q_batch_stride, s->q_row_stride);
}

// sizes of the plan and its partials; `ws` null: the bytes alone
size_t prefix_layout(const ia_decode_shape* s, int kv_dtype, int n_groups, PrefixParams* p, char* ws) {
  const int group = s->n_q_heads / s->n_kv_heads;
  p->batch = s->batch;
  p->n_groups = n_groups;
  p->tile_seqs = kArRows / group;
  p->n_tiles = n_groups ? s->batch / p->tile_seqs + n_groups : 0;
  const int resident = device_cus() * (kv_dtype == IA_F32 ? 1 : 2);
  p->target = std::max(1, resident / s->n_kv_heads);
  p->max_items = p->target + p->n_tiles + s->batch;
  // a range is cut into at most its share of target, and one more
  p->rows = (int64_t)(p->n_tiles ? p->target + p->n_tiles : 0) * kArRows + (int64_t)(p->target + s->batch) * group;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* x = ws ? ws + at : nullptr;
    at += align_up(bytes, 256);
    return x;
  };
  p->n_items = reinterpret_cast<int32_t*>(take(4));
  p->items = reinterpret_cast<PrefixItem*>(take(sizeof(PrefixItem) * p->max_items));
  p->entries = reinterpret_cast<PrefixEntry*>(take(sizeof(PrefixEntry) * (p->n_tiles + (size_t)s->batch)));
  p->tile_of = reinterpret_cast<int32_t*>(take(4 * (size_t)s->batch));
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
  if (!seq_lens || (n_groups && (!group_starts || !shared_lens))) return fail(IA_ERR_INVALID, "null pointer argument");
  PrefixParams p{};
  rc = set_ar_params(&p.ar, q, shape->q_dtype, shape->q_batch_stride, shape->q_row_stride,
                     shape->n_q_heads / shape->n_kv_heads, shape->n_kv_heads, kv->dtype, scale, out, out_dtype);
  if (rc) return rc;
  if (shape->batch == 0) return IA_OK;
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
  if ((int64_t)p.max_items * shape->n_kv_heads >= (int64_t)1 << 31 || p.rows >= (int64_t)1 << 31)
    return fail(IA_ERR_UNSUPPORTED, "batch too large for one launch");
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(ia_shared_prefix_plan, dim3(1), dim3(kPlanThreads), 0, st, p);
  rc = check_launch("shared-prefix plan");
  if (rc) return rc;
  const int d = shape->head_dim;
  rc = kv->dtype == IA_BF16 ? launch_prefix_bf16(p, d, st)
                            : kv->dtype == IA_F32 ? launch_prefix_f32(p, d, st) : launch_prefix_fp8(p, d, st);
  if (rc) return rc;
  const dim3 grid((unsigned)shape->batch * shape->n_kv_heads);
  if (d == 128)
    hipLaunchKernelGGL((ia_shared_prefix_merge<128>), grid, dim3(kArThreads), 0, st, p);
  else
    hipLaunchKernelGGL((ia_shared_prefix_merge<64>), grid, dim3(kArThreads), 0, st, p);
  return check_launch("shared-prefix merge");
}

}  // extern "C"
