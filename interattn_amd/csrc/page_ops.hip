// Pages of a cache: copying, forking, reserving, freeing and compacting, for gfx950.
//
// State on the device: block_table [rows, cols] (-1: no page), seq_lens [rows] and
// refs [n_pages], the number of table entries that hold a page; a page is free where
// refs is 0, and allocation takes the lowest free page.  So the state after a call is a
// function of the state before it (no free list whose order depends on timing), and a
// captured serving step can replay every call.
//
// A call is one launch that decides (one workgroup: a few thousand entries and one pass
// over refs, 4 bytes a page; bound by its round trips: 10.4 us for 16 forks among 1,100
// pages, 6.7 us for a reservation, 12.9 us for the plan of 16,384 pages' compaction) and,
// where pages move, one that copies.  Copying is bound by HBM: a workgroup per (page,
// tensor), 16 bytes a lane and eight of them in flight: 700 pages of 8 fp8 pools and their
// scales, 184 MB read and written, in 35.0 us (5.3 TB/s); 4,096 pages of 4 bf16 pools moved
// by a compaction, 1.07 GB, in 255 us (4.2 TB/s).
#include <algorithm>

#include "ia_common.hpp"

namespace ia {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kListMax = 1 << 23;  // entries of a list that has a workgroup for each
constexpr int kForkMax = 8192;   // forks of one call (the plan compares them pairwise)
constexpr int kMaxTensors = 48;  // of one launch (kernel arguments)

struct Tensors {
  ia_page_tensor t[kMaxTensors];
  int32_t n;
};

template <typename W>
__device__ __forceinline__ void copy_words(const ia_page_tensor& t, const char* src, char* dst, int tid) {
  const int per = t.run_bytes / (int)sizeof(W), total = t.n_outer * t.n_inner * per;
  constexpr int kFly = 8;
  for (int i0 = 0; i0 < total; i0 += kFly * kCopyThreads) {
    W w[kFly];
    int64_t off[kFly];
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      const int i = i0 + j * kCopyThreads + tid;
      if (i < total) {
        const int run = i / per;
        off[j] = (run / t.n_inner) * t.outer_stride + (run % t.n_inner) * t.inner_stride + (int64_t)(i - run * per) * (int)sizeof(W);
        w[j] = __builtin_nontemporal_load(reinterpret_cast<const W*>(src + off[j]));
      }
    }
#pragma unroll
    for (int j = 0; j < kFly; ++j)
      if (i0 + j * kCopyThreads + tid < total) *reinterpret_cast<W*>(dst + off[j]) = w[j];
  }
}

__device__ __forceinline__ void copy_page(const ia_page_tensor& t, int64_t src, int64_t dst, int tid) {
  char* base = static_cast<char*>(t.data);
  if (t.word_bytes == 16)
    copy_words<u32x4_t>(t, base + src * t.page_stride, base + dst * t.page_stride, tid);
  else
    copy_words<u32>(t, base + src * t.page_stride, base + dst * t.page_stride, tid);
}

__global__ __launch_bounds__(kCopyThreads) void ia_copy_page_list(Tensors ts, const int32_t* src, const int32_t* dst,
                                                              int n_pages) {
  const int s = src[blockIdx.x], d = dst[blockIdx.x];
  if (s < 0 || d < 0 || s >= n_pages || d >= n_pages || s == d) return;
  copy_page(ts.t[blockIdx.y], s, d, threadIdx.x);
}

// ------------------------------------------------------------------ free pages

// Sum over the workgroup of one value per wave, and the waves' exclusive prefix.
__device__ __forceinline__ void wave_prefix(int mine, int* scratch, int* before, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) scratch[wave] = mine;
  __syncthreads();
  int b = 0, t = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) b += scratch[w];
    t += scratch[w];
  }
  *before = b;
  *total = t;
}

__device__ __forceinline__ int wave_total(int v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s, 64);
  return v;
}

// Wave w's stretch of refs, in words of four pages.
__device__ __forceinline__ void stretch(int n_pages, int* lo, int* hi) {
  const int words = (n_pages + 3) / 4, per = ((words + kPlanWaves - 1) / kPlanWaves + 63) / 64 * 64;
  *lo = min((int)(threadIdx.x >> 6) * per, words);
  *hi = min(*lo + per, words);
}

// refs of the four pages from 4 * i on (1 past the last page: not free)
__device__ __forceinline__ int4 refs4(const int32_t* refs, int n_pages, int i) {
  if (4 * i + 3 < n_pages) return *reinterpret_cast<const int4*>(refs + 4 * i);
  int4 r = {1, 1, 1, 1};
  if (4 * i < n_pages) r.x = refs[4 * i];
  if (4 * i + 1 < n_pages) r.y = refs[4 * i + 1];
  if (4 * i + 2 < n_pages) r.z = refs[4 * i + 2];
  return r;
}

// The free pages in ascending order, the first `want` of them into list; returns how many
// there are, want at most.  All threads of the workgroup.
__device__ int lowest_free(const int32_t* refs, int n_pages, int want, int32_t* list, int* scratch) {
  const int lane = threadIdx.x & 63;
  int lo, hi, mine = 0;
  stretch(n_pages, &lo, &hi);
#pragma unroll 8
  for (int i = lo + lane; i < hi; i += 64) {
    const int4 r = refs4(refs, n_pages, i);
    mine += (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
  }
  int before, total;
  wave_prefix(wave_total(mine), scratch, &before, &total);
  for (int i0 = lo; i0 < hi && before < want; i0 += 64) {
    const int i = i0 + lane;
    const int4 r = i < hi ? refs4(refs, n_pages, i) : int4{1, 1, 1, 1};
    const int z[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
    const int n = z[0] + z[1] + z[2] + z[3], upto = wave_inclusive_scan(n);
    int at = before + upto - n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (z[j]) {
        if (at < want) list[at] = 4 * i + j;
        ++at;
      }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  __syncthreads();
  return total < want ? total : want;
}

// ------------------------------------------------------------------ fork

struct Table {
  int32_t* table;
  int64_t stride;
  int32_t rows, cols;
  int32_t* seq_lens;
  int32_t* refs;
  int32_t n_pages, page_rows;
};

// Per fork: ok, and the page its prompt's last, partial page is copied from and to.
struct ForkPlan {
  int32_t* ok;    // caller's
  int32_t* from;  // workspace [n]
  int32_t* to;    // workspace [n]
  int32_t* list;  // workspace [n]
};

__global__ __launch_bounds__(kPlanThreads) void ia_fork_plan(Table t, const int32_t* src, const int32_t* dst, int n,
                                                             ForkPlan f) {
  __shared__ int scratch[kPlanWaves];
  const int tid = threadIdx.x;
  // a fork fails whose rows do not exist, whose source is longer than a row or is itself
  // written by this call, or whose destination is listed before or holds anything
  for (int i = tid; i < n; i += kPlanThreads) {
    const int s = src[i], d = dst[i];
    int ok = s >= 0 && s < t.rows && d >= 0 && d < t.rows, from = -1;
    if (ok) {
      const int len = t.seq_lens[s];
      ok = len >= 0 && len <= (int64_t)t.cols * t.page_rows && t.seq_lens[d] == 0;
      if (ok && len % t.page_rows) {
        from = t.table[s * t.stride + len / t.page_rows];
        ok = from >= 0 && from < t.n_pages;
      }
    }
    for (int j = 0; j < n && ok; ++j) ok = dst[j] != s && (j >= i || dst[j] != d);
    f.ok[i] = ok;
    f.from[i] = ok ? from : -1;
    f.to[i] = -1;
  }
  __syncthreads();
  for (int64_t k = tid; k < (int64_t)n * t.cols; k += kPlanThreads) {
    const int i = (int)(k / t.cols), d = dst[i];
    if (d >= 0 && d < t.rows && t.table[d * t.stride + (k - (int64_t)i * t.cols)] >= 0) f.ok[i] = 0;
  }
  __syncthreads();
  // pages for the partial ones, in the forks' order
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const int need = i < n && f.ok[i] && f.from[i] >= 0;
    const int upto = wave_inclusive_scan(need);
    int before, total;
    wave_prefix(__builtin_amdgcn_readlane(upto, 63), scratch, &before, &total);
    if (i < n) f.to[i] = need ? base + before + upto - 1 : -1;  // (its rank, for now)
    base += total;
  }
  const int have = lowest_free(t.refs, t.n_pages, base, f.list, scratch);
  for (int i = tid; i < n; i += kPlanThreads) {
    const int rank = f.to[i];
    if (rank < 0) continue;
    if (rank >= have) {
      f.ok[i] = 0;
      f.to[i] = -1;
      continue;
    }
    f.to[i] = f.list[rank];
    t.refs[f.list[rank]] = 1;
  }
}

// y = 0: the table rows and counts; y > 0: tensor y - 1's partial page
__global__ __launch_bounds__(kCopyThreads) void ia_fork_apply(Table t, Tensors ts, const int32_t* src,
                                                              const int32_t* dst, ForkPlan f, int with_table) {
  const int i = blockIdx.x, tid = threadIdx.x;
  if (!f.ok[i]) return;
  const int y = (int)blockIdx.y - with_table;
  if (y >= 0) {
    if (f.to[i] >= 0) copy_page(ts.t[y], f.from[i], f.to[i], tid);
    return;
  }
  const int s = src[i], d = dst[i], len = t.seq_lens[s], whole = len / t.page_rows;
  for (int c = tid; c < whole; c += kCopyThreads) {
    const int pg = t.table[s * t.stride + c];
    t.table[d * t.stride + c] = pg;
    if (pg >= 0 && pg < t.n_pages) atomicAdd(&t.refs[pg], 1);
  }
  if (tid == 0) {
    if (f.to[i] >= 0) t.table[d * t.stride + whole] = f.to[i];
    t.seq_lens[d] = len;
  }
}

// ------------------------------------------------------------------ free, reserve

__global__ __launch_bounds__(kCopyThreads) void ia_free_rows(Table t, const int32_t* rows, int n) {
  const int i = blockIdx.x, tid = threadIdx.x, row = rows[i];
  if (row < 0 || row >= t.rows) return;
  int again = 0;  // a row listed twice is freed once
  for (int j = tid; j < i; j += kCopyThreads) again |= rows[j] == row;
  if (__syncthreads_or(again)) return;
  for (int c = tid; c < t.cols; c += kCopyThreads) {
    int32_t* e = t.table + row * t.stride + c;
    const int pg = *e;
    if (pg >= 0 && pg < t.n_pages) atomicSub(&t.refs[pg], 1);
    *e = -1;
  }
  if (tid == 0) t.seq_lens[row] = 0;
}

// A wave per row counts the entries without a page in the pages its next tokens reach;
// rows are served in order, each whole or not at all; then a wave per row fills them.
__global__ __launch_bounds__(kPlanThreads) void ia_reserve_rows(Table t, const int32_t* grow, int32_t* ok, int32_t* at,
                                                                int32_t* list) {
  __shared__ int scratch[kPlanWaves];
  __shared__ unsigned long long sum;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto span = [&](int row, int* lo, int* hi) {
    const int64_t len = t.seq_lens[row], g = grow[row];
    *lo = 0;
    *hi = 0;
    if (g <= 0) return true;
    if (len < 0 || len + g > (int64_t)t.cols * t.page_rows) return false;
    *lo = (int)(len / t.page_rows);
    *hi = (int)((len + g + t.page_rows - 1) / t.page_rows);
    return true;
  };
  for (int row = wave; row < t.rows; row += kPlanWaves) {
    int lo, hi, need = 0;
    const bool fits = span(row, &lo, &hi);
    for (int c = lo + lane; c < hi; c += 64) need += t.table[row * t.stride + c] < 0;
    need = wave_total(need);
    if (lane == 0) {
      ok[row] = fits;
      at[row] = fits ? need : 0;
    }
  }
  // how many pages there are, then how far they reach
  if (tid == 0) sum = 0;
  __syncthreads();
  long long all = 0;
  for (int row = tid; row < t.rows; row += kPlanThreads) all += at[row];
  for (int s = 32; s > 0; s >>= 1) all += __shfl_xor(all, s, 64);
  if (lane == 0) atomicAdd(&sum, (unsigned long long)all);
  __syncthreads();
  const int want = (int)min(sum, (unsigned long long)t.n_pages);
  const int have = lowest_free(t.refs, t.n_pages, want, list, scratch);
  if (sum <= (unsigned long long)have) {
    int base = 0;
    for (int r0 = 0; r0 < t.rows; r0 += kPlanThreads) {
      const int row = r0 + tid, need = row < t.rows ? at[row] : 0;
      const int upto = wave_inclusive_scan(need);
      int before, total;
      wave_prefix(__builtin_amdgcn_readlane(upto, 63), scratch, &before, &total);
      if (row < t.rows) at[row] = base + before + upto - need;
      base += total;
    }
  } else if (tid == 0) {  // short of pages: in order, rows that the rest still covers
    int base = 0;
    for (int row = 0; row < t.rows; ++row) {
      const int need = at[row];
      if (need > have - base) {
        ok[row] = 0;
        at[row] = have;
      } else {
        at[row] = base;
        base += need;
      }
    }
  }
  __syncthreads();
  for (int row = wave; row < t.rows; row += kPlanWaves) {
    int lo, hi, base = at[row];
    if (!ok[row] || !span(row, &lo, &hi)) continue;
    for (int c0 = lo; c0 < hi; c0 += 64) {
      const int c = c0 + lane;
      const int need = c < hi && t.table[row * t.stride + c] < 0;
      const int upto = wave_inclusive_scan(need);
      if (need) {
        const int pg = list[base + upto - 1];
        t.table[row * t.stride + c] = pg;
        t.refs[pg] = 1;
      }
      base += __builtin_amdgcn_readlane(upto, 63);
    }
  }
}

// ------------------------------------------------------------------ reorder

// Row i becomes what row parents[i] was.  One row takes over what its parent held (the
// parent itself, else the lowest of them); the others share the whole pages and get a copy
// of the partly filled one.  Two launches, each a chain of round trips: 4 rows of 48 bf16
// tensors take 8 + 8 us, 128 rows of 2,000 to 9,000 tokens in 16 fp8 pools and their scales
// 11 + 14 us, of which the copies' bytes are 5.
struct ReorderPlan {
  const int32_t* parents;
  int32_t* ok;     // caller's
  int32_t* kind;   // workspace [rows]: what becomes of the row
  int32_t* len;    // [rows] its length
  int32_t* from;   // [rows] the page it needs a copy of, -1: none
  int32_t* to;     // [rows]
  int32_t* list;   // [rows]
  int32_t* table;  // [rows, cols] its pages
  u32* ended;      // workgroups of ia_reorder_take that have ended (0 between calls)
};
enum { kRowStays = 0, kRowChanges = 1, kRowEmpty = 2 };

// The row's new pages and their counts, by one workgroup a stretch of columns.  The table itself
// is read only; the counts change by sums, whose order does not matter.
__device__ void reorder_row(const Table& t, const ReorderPlan& r, int i, int c0, int c1, bool first) {
  const int tid = threadIdx.x, src = r.parents[i];
  const bool exists = src >= 0 && src < t.rows;
  bool heir = src == i;
  if (exists && !heir) {
    int before = r.parents[src] == src;
    for (int j = tid; j < i && !before; j += kPlanThreads) before = r.parents[j] == src;
    heir = !__syncthreads_or(before);
  }
  int kind = src == i ? kRowStays : exists ? kRowChanges : kRowEmpty, ok = 1, len = 0, whole = 0, from = -1;
  if (exists) {
    len = t.seq_lens[src];
    if (!heir) {
      ok = len >= 0 && len <= (int64_t)t.cols * t.page_rows;
      if (ok) whole = len / t.page_rows;
      if (ok && len % t.page_rows) {
        from = t.table[src * t.stride + whole];
        ok = from >= 0 && from < t.n_pages;
      }
      if (!ok) {
        kind = kRowEmpty;
        len = 0;
        from = -1;
      }
    }
  }
  if (first && tid == 0) {
    r.kind[i] = kind;
    r.len[i] = len;
    // (read by the workgroup that plans)
    st_agent_u32(reinterpret_cast<u32*>(r.ok + i), (u32)ok);
    st_agent_u32(reinterpret_cast<u32*>(r.from + i), (u32)from);
  }
  if (kind == kRowStays) return;
  for (int c = c0 + tid; c < c1; c += kPlanThreads) {
    const int old = t.table[i * t.stride + c];
    int pg = -1;
    if (kind == kRowChanges && (heir || c < whole)) pg = t.table[src * t.stride + c];
    r.table[(int64_t)i * t.cols + c] = pg;
    if (pg == old) continue;
    if (old >= 0 && old < t.n_pages) atomicSub(&t.refs[old], 1);
    if (pg >= 0 && pg < t.n_pages) atomicAdd(&t.refs[pg], 1);
  }
}

// Pages for the copies, in the rows' order.
__device__ void reorder_pages(const Table& t, const ReorderPlan& r, int* scratch) {
  const int tid = threadIdx.x;
  int base = 0;
  for (int i0 = 0; i0 < t.rows; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const int need = i < t.rows && (int)ld_agent_u32(reinterpret_cast<const u32*>(r.from + i)) >= 0;
    const int upto = wave_inclusive_scan(need);
    int before, total;
    wave_prefix(__builtin_amdgcn_readlane(upto, 63), scratch, &before, &total);
    if (i < t.rows) r.to[i] = need ? base + before + upto - 1 : -1;  // (its rank, for now)
    base += total;
  }
  const int have = lowest_free(t.refs, t.n_pages, base, r.list, scratch);
  for (int i = tid; i < t.rows; i += kPlanThreads) {
    const int rank = r.to[i];
    if (rank < 0) continue;
    if (rank >= have) {
      r.ok[i] = 0;
      r.to[i] = -1;
      continue;
    }
    r.to[i] = r.list[rank];
    t.refs[r.list[rank]] = 1;
  }
}

// A workgroup per row and stretch of columns; the one that ends last plans the copies (a launch
// of its own for that costs 3 us more).  What it reads of the others' work is stored at the
// device's coherence point, and the counts are agent-scope atomics: no fence over a whole L2 (one
// in every workgroup took 38 us).
__global__ __launch_bounds__(kPlanThreads) void ia_reorder_take(Table t, ReorderPlan r, int span) {
  __shared__ int scratch[kPlanWaves];
  __shared__ u32 before;
  const int c0 = blockIdx.y * span;
  reorder_row(t, r, blockIdx.x, c0, min(c0 + span, t.cols), blockIdx.y == 0);
  wait_memory();
  __syncthreads();
  if (threadIdx.x == 0) before = fetch_add_agent_u32(r.ended, 1);
  __syncthreads();
  if (before != gridDim.x * gridDim.y - 1) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  if (threadIdx.x == 0) st_agent_u32(r.ended, 0);
  reorder_pages(t, r, scratch);
}

// y = 0: the table rows and lengths; y > 0: tensor y - 1's partly filled page
__global__ __launch_bounds__(kCopyThreads) void ia_reorder_apply(Table t, Tensors ts, ReorderPlan r, int with_table) {
  const int i = blockIdx.x, tid = threadIdx.x, kind = r.kind[i];
  if (kind == kRowStays) return;
  const int y = (int)blockIdx.y - with_table;
  if (y >= 0) {
    if (r.to[i] >= 0) copy_page(ts.t[y], r.from[i], r.to[i], tid);
    return;
  }
  const int len = r.len[i], whole = r.to[i] >= 0 ? len / t.page_rows : -1;
  const bool given_up = kind == kRowChanges && !r.ok[i];  // no page was left: what it shares goes back
  for (int c = tid; c < t.cols; c += kCopyThreads) {
    int pg = r.table[(int64_t)i * t.cols + c];
    if (given_up) {
      if (pg >= 0 && pg < t.n_pages) atomicSub(&t.refs[pg], 1);
      pg = -1;
    }
    t.table[i * t.stride + c] = c == whole ? r.to[i] : pg;
  }
  if (tid == 0) t.seq_lens[i] = given_up ? 0 : len;
}

// ------------------------------------------------------------------ compact

// Live pages at or past the number of live pages move, in ascending order, into the free
// pages before it.  movers / holes [n_pages / 2 + 1]; map [n_pages] where a page at or past
// the count now is; count[0] live pages, count[1] moves.
__global__ __launch_bounds__(kPlanThreads) void ia_compact_plan(int32_t* refs, int n_pages, int32_t* movers,
                                                                int32_t* holes, int32_t* map, int32_t* live_out,
                                                                int32_t* moves_out) {
  __shared__ int scratch[kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  int lo, hi, mine = 0;
  stretch(n_pages, &lo, &hi);
  auto live4 = [&](int i, int* v) {
    const int4 r = i < hi ? refs4(refs, n_pages, i) : int4{0, 0, 0, 0};
    v[0] = r.x > 0 && 4 * i < n_pages;
    v[1] = r.y > 0 && 4 * i + 1 < n_pages;
    v[2] = r.z > 0 && 4 * i + 2 < n_pages;
    v[3] = r.w > 0 && 4 * i + 3 < n_pages;
  };
#pragma unroll 8
  for (int i = lo + lane; i < hi; i += 64) {
    int v[4];
    live4(i, v);
    mine += v[0] + v[1] + v[2] + v[3];
  }
  int before, count, front = 0, unused, low;
  wave_prefix(wave_total(mine), scratch, &before, &count);
  for (int i = lo + lane; i < hi && 4 * i < count; i += 64) {  // live pages that stay
    int v[4];
    live4(i, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) front += v[j] && 4 * i + j < count;
  }
  wave_prefix(wave_total(front), scratch, &unused, &low);
  const int moves = count - low;
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const int i = i0 + lane;
    int v[4];
    live4(i, v);
    const int n = v[0] + v[1] + v[2] + v[3], upto = wave_inclusive_scan(n);
    int at = before + upto - n;  // live pages before this one
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pg = 4 * i + j;
      if (i < hi && pg < n_pages) {
        if (pg >= count) {
          if (v[j]) movers[at - low] = pg; else map[pg] = pg;
        } else if (!v[j]) {
          holes[pg - at] = pg;
        }
      }
      at += v[j];
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  __syncthreads();
  for (int k = tid; k < moves; k += kPlanThreads) {
    const int from = movers[k], to = holes[k];
    map[from] = to;
    refs[to] = refs[from];
    refs[from] = 0;
  }
  if (tid == 0) {
    *live_out = count;
    *moves_out = moves;
  }
}

// The first copy_wgs workgroups move pages, the rest rewrite the table.
__global__ __launch_bounds__(kCopyThreads) void ia_compact_apply(Tensors ts, int copy_wgs, const int32_t* movers,
                                                                 const int32_t* holes, const int32_t* map,
                                                                 const int32_t* live, const int32_t* moves,
                                                                 int32_t* table, int64_t stride, int rows, int cols,
                                                                 int n_pages) {
  if ((int)blockIdx.x < copy_wgs) {
    const int64_t n = (int64_t)*moves * ts.n;
    for (int64_t k = blockIdx.x; k < n; k += copy_wgs)
      copy_page(ts.t[k % ts.n], movers[k / ts.n], holes[k / ts.n], threadIdx.x);
    return;
  }
  const int count = *live;
  const int64_t n = (int64_t)rows * cols, step = (int64_t)(gridDim.x - copy_wgs) * kCopyThreads;
  for (int64_t k = (int64_t)(blockIdx.x - copy_wgs) * kCopyThreads + threadIdx.x; k < n; k += step) {
    int32_t* e = table + (k / cols) * stride + k % cols;
    const int pg = *e;
    if (pg >= count && pg < n_pages) *e = map[pg];
  }
}

// ------------------------------------------------------------------ host

int check_tensors(const ia_page_tensor* t, int n) {
  if (n < 0 || (n && !t)) return fail(IA_ERR_INVALID, "page tensors");
  for (int i = 0; i < n; ++i) {
    const ia_page_tensor& x = t[i];
    if (!x.data || x.n_outer < 1 || x.n_inner < 1 || x.run_bytes < 1 || x.page_stride < 0 || x.outer_stride < 0 ||
        x.inner_stride < 0)
      return fail(IA_ERR_INVALID, "page tensors need non-null data and positive extents");
    if (x.word_bytes != 16 && x.word_bytes != 4) return fail(IA_ERR_INVALID, "page tensor words are 4 or 16 bytes");
    if ((int64_t)x.n_outer * x.n_inner * x.run_bytes >= (int64_t)1 << 31)
      return fail(IA_ERR_UNSUPPORTED, "a page must be smaller than 2 GiB");
    if (reinterpret_cast<uintptr_t>(x.data) % x.word_bytes || x.page_stride % x.word_bytes ||
        x.outer_stride % x.word_bytes || x.inner_stride % x.word_bytes || x.run_bytes % x.word_bytes)
      return fail(IA_ERR_INVALID, "page tensor not aligned to its words");
  }
  return IA_OK;
}

int check_state(const ia_page_state* s, Table* t, bool lens = true) {
  // (arrays without entries have no address)
  if (!s || (!s->block_table && s->rows > 0 && s->cols > 0) || (lens && !s->seq_lens && s->rows > 0) ||
      (!s->refs && s->n_pages > 0))
    return fail(IA_ERR_INVALID, "null pointer argument");
  if (s->rows < 0 || s->cols < 0 || s->bt_stride < s->cols || s->n_pages < 0 || s->page_size <= 0)
    return fail(IA_ERR_INVALID, "page state: rows, cols, n_pages >= 0, bt_stride >= cols, page_size > 0");
  if (s->n_pages > INT32_MAX - 4) return fail(IA_ERR_UNSUPPORTED, "too many pages");
  if (reinterpret_cast<uintptr_t>(s->refs) % 16) return fail(IA_ERR_INVALID, "refs must be 16-byte aligned");
  *t = Table{s->block_table, s->bt_stride, s->rows, s->cols, s->seq_lens, s->refs, (int32_t)s->n_pages, s->page_size};
  return IA_OK;
}

// tensors [at, at + kMaxTensors) of a list
Tensors some_tensors(const ia_page_tensor* t, int n, int at) {
  Tensors ts{};
  ts.n = std::min(n - at, kMaxTensors);
  for (int i = 0; i < ts.n; ++i) ts.t[i] = t[at + i];
  return ts;
}

}  // namespace
}  // namespace ia

extern "C" {

int ia_copy_pages(const ia_page_tensor* tensors, int32_t n_tensors, const int32_t* src, const int32_t* dst, int32_t n,
                  int64_t n_pages, void* stream) {
  using namespace ia;
  int rc = check_tensors(tensors, n_tensors);
  if (rc) return rc;
  if (n < 0 || n >= kListMax || n_pages < 0 || n_pages > INT32_MAX || (n && (!src || !dst)))
    return fail(IA_ERR_INVALID, "page lists");
  if (n == 0) return IA_OK;
  for (int at = 0; at < n_tensors; at += kMaxTensors) {
    const Tensors ts = some_tensors(tensors, n_tensors, at);
    hipLaunchKernelGGL(ia_copy_page_list, dim3(n, ts.n), dim3(kCopyThreads), 0, static_cast<hipStream_t>(stream), ts, src,
                       dst, (int)n_pages);
    rc = check_launch("copy pages");
    if (rc) return rc;
  }
  return IA_OK;
}

size_t ia_fork_workspace_size(int32_t n) { return n > 0 ? 12 * (size_t)n : 0; }

int ia_fork_sequences(const ia_page_state* state, const ia_page_tensor* tensors, int32_t n_tensors, const int32_t* src,
                      const int32_t* dst, int32_t n, int32_t* ok, void* workspace, size_t workspace_bytes,
                      void* stream) {
  using namespace ia;
  Table t;
  int rc = check_state(state, &t);
  if (rc) return rc;
  rc = check_tensors(tensors, n_tensors);
  if (rc) return rc;
  if (n < 0 || n > kForkMax || (n && (!src || !dst || !ok)))
    return fail(IA_ERR_INVALID, "fork lists of up to " + std::to_string(kForkMax) + " rows");
  if (n == 0) return IA_OK;
  if (!workspace || workspace_bytes < ia_fork_workspace_size(n) || reinterpret_cast<uintptr_t>(workspace) % 4)
    return fail(IA_ERR_WORKSPACE, "workspace missing or too small");
  int32_t* w = static_cast<int32_t*>(workspace);
  const ForkPlan f{ok, w, w + n, w + 2 * (size_t)n};
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(ia_fork_plan, dim3(1), dim3(kPlanThreads), 0, st, t, src, dst, n, f);
  rc = check_launch("fork plan");
  for (int at = 0; !rc && (at == 0 || at < n_tensors); at += kMaxTensors) {
    const Tensors ts = some_tensors(tensors, n_tensors, at);
    const int with_table = at == 0;
    hipLaunchKernelGGL(ia_fork_apply, dim3(n, ts.n + with_table), dim3(kCopyThreads), 0, st, t, ts, src, dst, f,
                       with_table);
    rc = check_launch("fork");
  }
  return rc;
}

int ia_free_sequences(const ia_page_state* state, const int32_t* rows, int32_t n, void* stream) {
  using namespace ia;
  Table t;
  int rc = check_state(state, &t);
  if (rc) return rc;
  if (n < 0 || n >= kListMax || (n && !rows)) return fail(IA_ERR_INVALID, "row list");
  if (n == 0) return IA_OK;
  hipLaunchKernelGGL(ia_free_rows, dim3(n), dim3(kCopyThreads), 0, static_cast<hipStream_t>(stream), t, rows, n);
  return check_launch("free sequences");
}

size_t ia_reserve_workspace_size(int32_t rows, int64_t n_pages) {
  return rows > 0 && n_pages >= 0 ? 4 * ((size_t)rows + (size_t)n_pages) : 0;
}

int ia_reserve_pages(const ia_page_state* state, const int32_t* new_tokens, int32_t* ok, void* workspace,
                     size_t workspace_bytes, void* stream) {
  using namespace ia;
  Table t;
  int rc = check_state(state, &t);
  if (rc) return rc;
  if (t.rows == 0) return IA_OK;
  if (!new_tokens || !ok) return fail(IA_ERR_INVALID, "null pointer argument");
  if (!workspace || workspace_bytes < ia_reserve_workspace_size(t.rows, t.n_pages) ||
      reinterpret_cast<uintptr_t>(workspace) % 4)
    return fail(IA_ERR_WORKSPACE, "workspace missing or too small");
  int32_t* w = static_cast<int32_t*>(workspace);
  hipLaunchKernelGGL(ia_reserve_rows, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), t, new_tokens,
                     ok, w, w + t.rows);
  return check_launch("reserve pages");
}

size_t ia_reorder_workspace_size(int32_t rows, int32_t cols) {
  return rows > 0 && cols >= 0 ? 4 * (1 + (size_t)rows * (5 + (size_t)cols)) : 0;
}

int ia_reorder_sequences(const ia_page_state* state, const ia_page_tensor* tensors, int32_t n_tensors,
                         const int32_t* parents, int32_t* ok, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ia;
  Table t;
  int rc = check_state(state, &t);
  if (rc) return rc;
  rc = check_tensors(tensors, n_tensors);
  if (rc) return rc;
  if (t.rows == 0) return IA_OK;
  if (t.rows > kForkMax) return fail(IA_ERR_UNSUPPORTED, "at most " + std::to_string(kForkMax) + " rows are reordered");
  if (!parents || !ok) return fail(IA_ERR_INVALID, "null pointer argument");
  if (!workspace || workspace_bytes < ia_reorder_workspace_size(t.rows, t.cols) ||
      reinterpret_cast<uintptr_t>(workspace) % 4)
    return fail(IA_ERR_WORKSPACE, "workspace missing or too small");
  int32_t* w = static_cast<int32_t*>(workspace) + 1;
  const size_t n = t.rows;
  const ReorderPlan r{parents,   ok,        w,         w + n, w + 2 * n, w + 3 * n, w + 4 * n, w + 5 * n,
                      static_cast<u32*>(workspace)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  // (a row's length and counts are written even where the table has no column)
  const int span = 4 * kPlanThreads, spans = std::max(1, (t.cols + span - 1) / span);
  if (spans > 65535 || (int64_t)t.rows * spans >= 1 << 22) return fail(IA_ERR_UNSUPPORTED, "the table has too many columns");
  hipLaunchKernelGGL(ia_reorder_take, dim3(t.rows, spans), dim3(kPlanThreads), 0, st, t, r, span);
  rc = check_launch("reorder");
  for (int at = 0; !rc && (at == 0 || at < n_tensors); at += kMaxTensors) {
    const Tensors ts = some_tensors(tensors, n_tensors, at);
    const int with_table = at == 0;
    hipLaunchKernelGGL(ia_reorder_apply, dim3(t.rows, ts.n + with_table), dim3(kCopyThreads), 0, st, t, ts, r,
                       with_table);
    rc = check_launch("reorder apply");
  }
  return rc;
}

size_t ia_compact_workspace_size(int64_t n_pages) { return n_pages >= 0 ? 4 * (2 * (size_t)n_pages + 16) : 0; }

int ia_compact_pages(const ia_page_state* state, const ia_page_tensor* tensors, int32_t n_tensors, int32_t* n_live,
                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ia;
  Table t;
  int rc = check_state(state, &t, false);
  if (rc) return rc;
  rc = check_tensors(tensors, n_tensors);
  if (rc) return rc;
  if (!n_live) return fail(IA_ERR_INVALID, "null pointer argument");
  if (!workspace || workspace_bytes < ia_compact_workspace_size(t.n_pages) || reinterpret_cast<uintptr_t>(workspace) % 4)
    return fail(IA_ERR_WORKSPACE, "workspace missing or too small");
  const int half = t.n_pages / 2 + 1;
  int32_t* moves = static_cast<int32_t*>(workspace);
  int32_t *movers = moves + 4, *holes = movers + half, *map = holes + half;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(ia_compact_plan, dim3(1), dim3(kPlanThreads), 0, st, t.refs, t.n_pages, movers, holes, map, n_live,
                     moves);
  rc = check_launch("compact plan");
  const int64_t entries = (int64_t)t.rows * t.cols;
  for (int at = 0; !rc && (at == 0 || at < n_tensors); at += kMaxTensors) {
    const Tensors ts = some_tensors(tensors, n_tensors, at);
    const int copy_wgs = ts.n ? device_cus() * 8 : 0;
    const int table_wgs =
        at == 0 ? (int)std::min<int64_t>((entries + kCopyThreads * 4 - 1) / (kCopyThreads * 4), device_cus()) : 0;
    if (copy_wgs + table_wgs == 0) break;
    hipLaunchKernelGGL(ia_compact_apply, dim3(copy_wgs + table_wgs), dim3(kCopyThreads), 0, st, ts, copy_wgs, movers,
                       holes, map, n_live, moves, t.table, t.stride, t.rows, t.cols, t.n_pages);
    rc = check_launch("compact");
  }
  return rc;
}

}  // extern "C"
