// Attention of a set of query rows over one key range, by one workgroup: the core of the
// prompt and shared-prefix kernels.
//
// A workgroup takes up to 128 rows of one kv head (tokens x the group's query heads, so a
// K/V tile is read once for the whole group) and streams the range in tiles of 64 keys
// through LDS, the next one on its way while one is used.  Row r's softmax runs online in
// base 2 with its scale folded in: s' = q.k * scale * log2(e); (m, l, acc) are float32, the
// products bf16 in, float32 out (float32 caches: float32 products).  P is rounded to bf16
// for the second product, as the cache's values are; l sums the unrounded P.
//
// Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane holds
// scores of ONE row: the row's maximum and sum cost one exchange between half-waves, and
// the P a lane computed is the operand the second product wants from it (contraction order
// is free as long as V^T is read in the same order, which the transposing LDS read does).
//
// Two shapes:
//   wide   (33..128 rows): 32x32 matrix tiles, a wave per 32 rows, all keys of the tile
//   narrow (1..32 rows):   16x16 matrix tiles, a wave per 16 keys, all rows; the four
//                          waves' (m, l, acc) meet in LDS at the end.  Its EXACT form also
//                          does items over, 32 rows at a time
//
// LDS rows are whole cache rows in 16-byte chunks, chunk c of row r at c ^ f(r): f is
// linear over the bits of r and chosen so that neither the row-per-lane key reads nor the
// four-rows-by-sixteen transposing reads put two lanes of one pass on a bank.
#pragma once

#include "ia_common.hpp"

namespace ia {

constexpr int kArTile = 64;       // keys per tile
constexpr int kArThreads = 256;   // four waves
constexpr int kArRows = 128;      // rows of a wide workgroup
constexpr int kArNarrow = 32;     // most rows of a narrow one
constexpr int kArMaxGroup = 64;   // query heads per kv head: a row tile holds at least two tokens
constexpr int64_t kArMaxGrid = 1 << 23;  // workgroups of a launch (work items are 32 bits)
constexpr float kArSlack = 8.f;   // log2 units a row's maximum may rise before it is rescaled
constexpr float kArFar = 65536.f; // log2 units at which a rounded maximum is off by up to 2^-8

typedef __attribute__((ext_vector_type(16))) float f32x16_t;
#define IA_LDS __attribute__((address_space(3)))

// K/V of a call: pages of page_rows tokens (a multiple of 16).  Packed rows are pages of
// 16 rows that follow each other (no table).  Strides in bytes.
struct ArSource {
  const char* k;
  const char* v;
  int64_t k_page, k_head, k_tok, v_page, v_head, v_tok;
  const int32_t* table;
  int64_t bt_stride, bt_cols, n_pages;
  int32_t page_rows;
  const float* k_scale;  // fp8: per (page, kv head)
  const float* v_scale;
  int64_t scale_page;
};

// One workgroup's work: rows r = 0..n_rows-1 are (token tok0 + r / group, query head
// head * group + r % group); row r sees the keys [k_lo, min(k_hi, limit(r))).
struct ArItem {
  const int32_t* table;  // this sequence's row of the block table
  int64_t row0;          // packed: the sequence's first K/V row
  int32_t head;          // kv head
  int32_t tok0, n_rows;
  int32_t k_lo, k_hi;
  const int32_t* lens;   // limit of token t: lens[t] (one per sequence), or
  int32_t limit0;        //   limit0 + (t - tok0) where lens is null
  float* part_ml;        // (m, l) pairs [n_rows]; null: final rows go to out
  float* part_acc;       // [n_rows, D]
};

struct ArParams {
  ArSource kv;
  const void* q;
  int64_t q_tok, q_head;  // elements
  void* out;              // [tokens, n_q_heads, D]
  int32_t out_f32, q_f32;
  int32_t group, n_kv_heads;
  float scale_log2;       // |scale| * log2(e)
  u32 q_flip;             // sign bit mask applied to q (scale < 0), one element
};

// host side (prompt_attention.hip)
int check_kv(const ia_paged_kv* kv, int d);
int check_ar_q(int q_dtype, int64_t q_tok, int64_t q_head);
int set_ar_params(ArParams* p, const void* q, int q_dtype, int64_t q_tok, int64_t q_head, int group, int n_kv_heads,
                  int kv_dtype, float scale, void* out, int out_dtype);
void set_ar_pages(ArSource* s, const ia_paged_kv* kv);
int64_t ar_key_cap(const ia_paged_kv* kv);  // keys a sequence can have in the pool

enum { kArBf16 = 0, kArF32 = 1, kArFp8 = 2 };

template <int KV, int D>
struct ArShape {
  static constexpr int kRowBytes = D * (KV == kArF32 ? 4 : 2);         // a row in LDS
  static constexpr int kSrcRow = D * (KV == kArF32 ? 4 : KV == kArBf16 ? 2 : 1);
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = kArTile * kRowBytes;
  static constexpr int kStage = 2 * kTileBytes;                        // K tile, V tile
  static constexpr int kSmem = 2 * kStage;
  static constexpr int kSrcChunks = kSrcRow / 16;
  static constexpr int kLoads = kArTile * kSrcChunks / kArThreads;     // 16-byte loads per thread and tile
  static constexpr int kLoadRows = kArThreads / kSrcChunks;            // rows one round of loads covers
};

template <int KV, int D>
__device__ __forceinline__ int ar_swizzle(int r) {
  if constexpr (ArShape<KV, D>::kChunks >= 16)
    return ((r & 1) << 2) ^ ((r & 2) ? 10 : 0) ^ ((r >> 2) & 1) ^ ((r & 8) >> 2);
  else
    return ((r & 1) << 1) ^ ((r & 2) << 1) ^ ((r >> 2) & 1) ^ ((r & 8) >> 2);
}

// 16 bytes per lane from global memory to LDS (lane l's at lds + 16 l) past the registers;
// lds is wave-uniform.  Counted by vmcnt, which ar_arrived() waits on.
__device__ __forceinline__ void ar_dma16(const char* src, u32 lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
// x, but nothing computed from it before is kept in registers (for the second pass, for the
// last stores)
__device__ __forceinline__ int ar_anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ void ar_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ u32 lds_addr(const void* p) {
  return (u32)(uintptr_t)(const IA_LDS char*)p;
}

// ------------------------------------------------------------------ tiles

// Loads tiles of one item.  A tile starts at a multiple of 16 keys, so each of its four
// groups of 16 keys lies in one page.  Lane l keeps where group l & 3 lies, fetched one tile
// ahead of the K/V loads that need it: a load's address is two lane reads and one addition.
template <int KV, int D>
struct ArLoader {
  using S = ArShape<KV, D>;
  const ArSource& kv;
  const ArItem& it;
  int lane, wave, tid;
  int page;                // group lane & 3 of the tile to be loaded next: its page, and
  int64_t k_grp, v_grp;    // where its first rows are
  // a lane's row and chunk within the 16 rows of a group (two forms where a round of loads
  // covers half a group): the rest of an address is the same in every lane
  static constexpr int kForms = S::kLoadRows < 16 ? 2 : 1;
  int64_t k_lane[kForms], v_lane[kForms];
  float ks, vs;            // fp8: its scales, of the tile last issued
  u32x4_t kr[KV == kArFp8 ? S::kLoads : 1], vr[KV == kArFp8 ? S::kLoads : 1];

  __device__ __forceinline__ ArLoader(const ArSource& kv_, const ArItem& it_, bool anew) : kv(kv_), it(it_) {
    tid = anew ? ar_anew(threadIdx.x) : threadIdx.x;
    lane = tid & 63;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    ks = vs = 0.f;
#pragma unroll
    for (int f = 0; f < kForms; ++f) {
      const int row = (tid / S::kSrcChunks + f * S::kLoadRows) & 15, slot = tid % S::kSrcChunks;
      const int chunk = KV == kArFp8 ? slot : slot ^ ar_swizzle<KV, D>(row);
      k_lane[f] = row * kv.k_tok + chunk * 16;
      v_lane[f] = row * kv.v_tok + chunk * 16;
    }
  }

  __device__ __forceinline__ void fetch_pages(int tb) {
    const int key = tb + 16 * (lane & 3);
    int pg = -1, in = 0;
    if (key < it.k_hi) {
      const int lp = kv.page_rows == 16 ? key >> 4 : (int)((u32)key / (u32)kv.page_rows);
      in = key - lp * kv.page_rows;
      pg = lp;
      if (kv.table) pg = lp < kv.bt_cols ? it.table[lp] : -1;
      if (pg >= kv.n_pages) pg = -1;
    }
    page = pg;
    k_grp = reinterpret_cast<int64_t>(kv.k) + it.head * kv.k_head + (it.row0 + in) * kv.k_tok + pg * kv.k_page;
    v_grp = reinterpret_cast<int64_t>(kv.v) + it.head * kv.v_head + (it.row0 + in) * kv.v_tok + pg * kv.v_page;
  }
  static __device__ __forceinline__ int64_t lane_i64(int64_t x, int l) {
    const u32 lo = __builtin_amdgcn_readlane((u32)x, l), hi = __builtin_amdgcn_readlane((u32)((unsigned long long)x >> 32), l);
    return (int64_t)(((unsigned long long)hi << 32) | lo);
  }

  // keys of the tile at tb that exist: in range, on a valid page
  __device__ __forceinline__ bool whole(int tb) const {
    return tb >= it.k_lo && tb + kArTile <= it.k_hi && __ballot(page < 0) == 0;
  }

  template <bool WHOLE>
  __device__ __forceinline__ void issue_rows(int tb, char* smem) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int row = i * S::kLoadRows + tid / S::kSrcChunks;
      const int grp = __builtin_amdgcn_readfirstlane(row >> 4);
      // (lane reads before the lanes part ways)
      const int pg = __builtin_amdgcn_readlane(page, grp);
      const char* k_row = reinterpret_cast<const char*>(lane_i64(k_grp, grp) + k_lane[i % kForms]);
      const char* v_row = reinterpret_cast<const char*>(lane_i64(v_grp, grp) + v_lane[i % kForms]);
      const bool live = WHOLE || (pg >= 0 && tb + row >= it.k_lo && tb + row < it.k_hi);
      if constexpr (KV == kArFp8) {
        kr[i] = vr[i] = u32x4_t{0, 0, 0, 0};
        if (live) {
          kr[i] = *reinterpret_cast<const u32x4_t*>(k_row);
          vr[i] = *reinterpret_cast<const u32x4_t*>(v_row);
        }
      } else {
        const u32 dst = lds_addr(smem) + (i * 4 + wave) * 1024;
        if (live) {
          ar_dma16(k_row, dst);
          ar_dma16(v_row, dst + S::kTileBytes);
        } else {
          *reinterpret_cast<u32x4_t*>(smem + S::kTileBytes + (i * kArThreads + tid) * 16) = u32x4_t{0, 0, 0, 0};
        }
      }
    }
  }

  // Start the loads of the tile at tb (its pages fetched) into stage `smem`.  Keys that do
  // not exist get V rows of zeros: their P is 0, and 0 * garbage must not become NaN.
  __device__ __forceinline__ void issue(int tb, char* smem) {
    if (whole(tb))
      issue_rows<true>(tb, smem);
    else
      issue_rows<false>(tb, smem);
    if constexpr (KV == kArFp8) {
      ks = vs = 0.f;
      if (page >= 0) {
        ks = kv.k_scale[(int64_t)page * kv.scale_page + it.head];
        vs = kv.v_scale[(int64_t)page * kv.scale_page + it.head];
      }
    }
  }

  // fp8: the loaded codes, widened (exactly) to bf16, into stage `smem`
  __device__ __forceinline__ void commit(char* smem) {
    if constexpr (KV == kArFp8) {
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int row = i * S::kLoadRows + tid / S::kSrcChunks;
        const int f = ar_swizzle<KV, D>(row), c = 2 * (tid % S::kSrcChunks);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int off = row * S::kRowBytes + ((c + half) ^ f) * 16;
          u32x4_t a, b;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            a[2 * w] = fp8x2_to_bf16x2<false>(kr[i][2 * half + w]);
            a[2 * w + 1] = fp8x2_to_bf16x2<true>(kr[i][2 * half + w]);
            b[2 * w] = fp8x2_to_bf16x2<false>(vr[i][2 * half + w]);
            b[2 * w + 1] = fp8x2_to_bf16x2<true>(vr[i][2 * half + w]);
          }
          *reinterpret_cast<u32x4_t*>(smem + off) = a;
          *reinterpret_cast<u32x4_t*>(smem + S::kTileBytes + off) = b;
        }
      }
    }
  }
};

// four consecutive keys of 16 columns per 16-lane group, transposed: lane i of the group
// gets column i of the four rows whose 8-byte pieces lanes 4j..4j+3 point at
__device__ __forceinline__ u32x2_t ar_read_tr(const char* p) {
  typedef __attribute__((ext_vector_type(4))) short s4;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((IA_LDS s4*)(const IA_LDS char*)p));
}

__device__ __forceinline__ float half_max(float v) {
  auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// over the 64 lanes, in integers (lengths pass 2^24)
__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    const int o = __shfl_xor(v, s, 64);
    v = o < v ? o : v;
  }
  return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ int ar_limit(const ArItem& it, int tok) {
  const int lim = it.lens ? it.lens[tok] : it.limit0 + (tok - it.tok0);
  return lim < 0 ? 0 : lim < it.k_hi ? lim : it.k_hi;  // (0: its negative exists, unlike INT32_MIN's)
}

__device__ __forceinline__ const char* ar_q_row(const ArParams& p, const ArItem& it, int r) {
  const int tok = it.tok0 + r / p.group, g = r % p.group;
  return reinterpret_cast<const char*>(p.q) +
         ((int64_t)tok * p.q_tok + (int64_t)(it.head * p.group + g) * p.q_head) * (p.q_f32 ? 4 : 2);
}

// eight q elements at element e of a row as a bf16 operand (zero rows past the last); a
// float32 q is rounded to bf16, the products' type over these caches, as in the decode calls
__device__ __forceinline__ bf16x8_t ar_q8(const ArParams& p, const char* row, int e, bool live) {
  u32 w[4] = {0, 0, 0, 0};
  if (live) {
    if (p.q_f32) {
      const float* f = reinterpret_cast<const float*>(row) + e;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
    } else {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(row + 2 * e);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = x[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] ^= p.q_flip * 0x10001u;
  }
  return as_bf16x8(w);
}

// four q elements at element e of a float32 row
__device__ __forceinline__ f32x4_t ar_q4(const ArParams& p, const char* row, int e, bool live) {
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    x = *reinterpret_cast<const f32x4_t*>(row + 4 * e);
    if (p.q_flip)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = -x[j];
  }
  return x;
}

// four consecutive output elements of a row, final or partial
__device__ __forceinline__ void ar_store4(const ArParams& p, int64_t e, const float* x) {
  if (p.out_f32) {
    *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(p.out) + e) = f32x4_t{x[0], x[1], x[2], x[3]};
  } else {
    *reinterpret_cast<u32x2_t*>(reinterpret_cast<unsigned short*>(p.out) + e) =
        u32x2_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  }
}

__device__ __forceinline__ int64_t ar_out_row(const ArParams& p, const ArItem& it, int r, int d) {
  const int tok = it.tok0 + r / p.group, g = r % p.group;
  return ((int64_t)tok * p.n_kv_heads * p.group + it.head * p.group + g) * d;
}

// The second pass.  A key hidden from a row meets it with P = 0, and 0 * V is NaN where V is
// not finite.  The shapes do not look: an item whose rows come out not finite while keys are
// hidden from some of them is done over in the narrow shape with EXACT true; so is one of
// the wide shape whose sum l is not finite, where a scale of 0 met a hidden score (-inf,
// which the narrow shape puts in after the scale), or whose maximum lies so far out that its
// own rounding matters (the narrow shape rounds every scaled score alike).  There V
// enters the product with zeros in place of what is not finite, and a second product of
// marks with the rows' visibility (1 or 0) counts what each row sees: +inf is 1, -inf is 128,
// NaN both; sums over a tile's 64 keys stay exact in float32, and 128 keys of one kind would
// be needed for a carry.  A weight too small for float32 counts as positive.
constexpr u32 kMarkUp = 1, kMarkDown = 128;

__device__ __forceinline__ void ar_marks_bf16(u32 w, u32* fin, u32* mark) {
  *fin = *mark = 0;
#pragma unroll
  for (int s = 0; s < 32; s += 16) {
    const u32 x = (w >> s) & 0xffffu;
    const bool bad = (x & 0x7f80u) == 0x7f80u;
    // 1.0, 128.0 and 129.0 as bf16
    const u32 m = x == 0x7f80u ? 0x3f80u : x == 0xff80u ? 0x4300u : 0x4301u;
    *fin |= (bad ? 0u : x) << s;
    *mark |= (bad ? m : 0u) << s;
  }
}
__device__ __forceinline__ void ar_marks_f32(float x, float* fin, float* mark) {
  const bool bad = !(__builtin_fabsf(x) < __builtin_huge_valf());
  const float m = x == __builtin_huge_valf() ? kMarkUp : x == kNegInf ? kMarkDown : kMarkUp + kMarkDown;
  *fin = bad ? 0.f : x;
  *mark = bad ? m : 0.f;
}
// an accumulator and the marks its row saw
__device__ __forceinline__ float ar_marked(float o, float marks) {
  const u32 n = (u32)marks;
  if (n % kMarkDown) o += __builtin_huge_valf();
  if (n / kMarkDown) o += kNegInf;
  return o;
}

// ------------------------------------------------------------------ wide

// returns whether the item has to be done over (the same in every thread)
template <int KV, int D>
__device__ __forceinline__ bool ar_wide(const ArParams& p, const ArItem& it, char* smem) {
  using S = ArShape<KV, D>;
  constexpr int kDb = D / 32;                                // 32-dim blocks of O^T
  constexpr int kQ = KV == kArF32 ? D / 8 : D / 16;          // q operands per lane
  ArLoader<KV, D> ld(p.kv, it, false);
  const int lane = ld.lane, wave = ld.wave, h = lane >> 5, c = lane & 31;
  const int r = wave * 32 + c;
  const bool row_live = r < it.n_rows, wave_live = wave * 32 < it.n_rows;
  const int limit = row_live ? ar_limit(it, it.tok0 + r / p.group) : it.k_hi;
  // the wave's own bounds (rows of a wave are ordered, but lens need not be)
  const int lim_min = wave_min_i32(limit), lim_max = -wave_min_i32(row_live ? -limit : 1);
  bf16x8_t qb[KV == kArF32 ? 1 : kQ];
  f32x4_t qf[KV == kArF32 ? kQ : 1];
  {
    const char* qr = row_live ? ar_q_row(p, it, r) : nullptr;
#pragma unroll
    for (int s = 0; s < kQ; ++s) {
      if constexpr (KV == kArF32)
        qf[s] = ar_q4(p, qr, 8 * s + 4 * h, row_live);
      else
        qb[s] = ar_q8(p, qr, 16 * s + 8 * h, row_live);
    }
  }
  f32x16_t o[kDb];
#pragma unroll
  for (int d = 0; d < kDb; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = kNegInf, l = 0.f;

  // LDS offsets: key row c of a 32-key block; V rows and columns of the transposing read
  const int fk = ar_swizzle<KV, D>(c) ^ h;
  const int k_off = c * S::kRowBytes;
  const int vr0 = 4 * h + ((lane >> 2) & 3);
  const int vc0 = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ ar_swizzle<KV, D>(vr0);
  const int v_off = vr0 * S::kRowBytes + 8 * (lane & 1);

  const int tb0 = it.k_lo & ~15;
  const int n_tiles = (it.k_hi - tb0 + kArTile - 1) / kArTile;
  ld.fetch_pages(tb0);
  ld.issue(tb0, smem);
  int pages_now = ld.page;
  float ks_now = ld.ks, vs_now = ld.vs;
  ld.commit(smem);
  if (n_tiles > 1) ld.fetch_pages(tb0 + kArTile);
  for (int t = 0; t < n_tiles; ++t) {
    const int tb = tb0 + t * kArTile;
    char* cur = smem + (t & 1) * S::kStage;
    char* nxt = smem + ((t + 1) & 1) * S::kStage;
    ar_arrived();
    __syncthreads();  // (the other stage is no longer read, this one has landed)
    const int pg = pages_now;
    const float ks = ks_now, vs = vs_now;
    if (t + 1 < n_tiles) {
      ld.issue(tb + kArTile, nxt);
      pages_now = ld.page;
      ks_now = ld.ks;
      vs_now = ld.vs;
      if (t + 2 < n_tiles) ld.fetch_pages(tb + 2 * kArTile);
    }
    if (wave_live && tb < lim_max) {
      const char* kt = cur;
      const char* vt = cur + S::kTileBytes;
      f32x16_t s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
      if constexpr (KV == kArF32) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int q = 0; q < kQ; ++q) {
            const f32x4_t x = *reinterpret_cast<const f32x4_t*>(kt + kb * 32 * S::kRowBytes + k_off + (((2 * q) ^ fk) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], qf[q][e], s[kb], 0, 0, 0);
          }
      } else {
        // The key operands of 32 keys are read before their products, the next 32 keys'
        // behind them: left to itself the compiler reads, waits and multiplies one by one.
        bf16x8_t ka[kQ], kc[kQ];
        const char* a = kt + k_off;
#pragma unroll
        for (int q = 0; q < kQ; ++q) ka[q] = *reinterpret_cast<const bf16x8_t*>(a + (((2 * q) ^ fk) << 4));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < kQ; ++q)
          kc[q] = *reinterpret_cast<const bf16x8_t*>(a + 32 * S::kRowBytes + (((2 * q) ^ fk) << 4));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < kQ; ++q) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[q], qb[q], s[0], 0, 0, 0);
#pragma unroll
        for (int q = 0; q < kQ; ++q) s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kc[q], qb[q], s[1], 0, 0, 0);
      }
      // V operands, 16 keys at a time: the first are on their way during the softmax, the
      // next during the products of the ones before
      u32x2_t v[2][kDb][2];
      auto read_v = [&](int g) {
        const char* a = vt + v_off + 16 * g * S::kRowBytes;
#pragma unroll
        for (int d = 0; d < kDb; ++d) {
          v[g & 1][d][0] = ar_read_tr(a + (((4 * d) ^ vc0) << 4));
          v[g & 1][d][1] = ar_read_tr(a + 8 * S::kRowBytes + (((4 * d) ^ 2 ^ vc0) << 4));
        }
      };
      if constexpr (KV != kArF32) {
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (KV == kArFp8) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float sc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), g));
#pragma unroll
          for (int i = 0; i < 8; ++i) s[g >> 1][8 * (g & 1) + i] *= sc;
        }
      }
      const bool holes = tb < it.k_lo || tb + kArTile > it.k_hi || __ballot(pg < 0) != 0;
      if (holes || tb + kArTile > lim_min) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const bool gone = __builtin_amdgcn_readlane(pg, g) < 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = tb + 16 * g + 8 * (i >> 2) + 4 * h + (i & 3);
            if (gone || key < it.k_lo || key >= limit) s[g >> 1][8 * (g & 1) + i] = kNegInf;
          }
        }
      }
      float mx = s[0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
      mx = half_max(mx) * p.scale_log2;
      // Rescale only where some row's maximum rose by more than 2^8: until then P stays
      // below 2^8 (the same relative rounding), and the rescale costs as much as the exps.
      if (__ballot(mx > m + kArSlack) != 0) {
        const float mn = fmaxf(m, mx);
        const float a = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= a;
#pragma unroll
        for (int d = 0; d < kDb; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= a;
        m = mn;
      }
      const float mu = m == kNegInf ? 0.f : m;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], p.scale_log2, -mu));
          l += s[kb][i];
        }
      if constexpr (KV == kArFp8) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float sc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), g));
#pragma unroll
          for (int i = 0; i < 8; ++i) s[g >> 1][8 * (g & 1) + i] *= sc;
        }
      }
      if constexpr (KV == kArF32) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int row = kb * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
            const int f = ar_swizzle<KV, D>(row);
#pragma unroll
            for (int d = 0; d < kDb; ++d) {
              const int ch = (8 * d + (c >> 2)) ^ f;
              const float x = *reinterpret_cast<const float*>(vt + row * S::kRowBytes + ch * 16 + 4 * (c & 3));
              o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[kb][i], o[d], 0, 0, 0);
            }
          }
      } else {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (g < 3) read_v(g + 1);
          u32 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(s[g >> 1][8 * (g & 1) + 2 * j], s[g >> 1][8 * (g & 1) + 2 * j + 1]);
          const bf16x8_t pb = as_bf16x8(w);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int d = 0; d < kDb; ++d) {
            const u32 va[4] = {v[g & 1][d][0][0], v[g & 1][d][0][1], v[g & 1][d][1][0], v[g & 1][d][1][1]};
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(va), pb, o[d], 0, 0, 0);
          }
        }
      }
    }
    if (t + 1 < n_tiles) ld.commit(nxt);
  }
  // 0, or NaN: a sum or a value of the row is not finite, or its scores are too far out for
  // the products above, which subtract the rounded maximum from the unrounded score
  float x = m > kArFar || (m < -kArFar && m != kNegInf) ? __builtin_nanf("") : 0.f * l;
  if (it.k_hi > lim_min) {
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) x += 0.f * o[d][i];
  }
  if (__syncthreads_or(row_live && !(x == 0.f))) return true;
  if (!wave_live) return false;
  l = half_sum(l);
  if (!row_live) return false;
  const int lane_out = ar_anew(lane), h_out = lane_out >> 5, r_out = wave * 32 + (lane_out & 31);
  if (it.part_ml) {
    if (h_out == 0) *reinterpret_cast<f32x2_t*>(it.part_ml + 2 * r_out) = f32x2_t{m, l};
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<f32x4_t*>(it.part_acc + (int64_t)r_out * D + 32 * d + 8 * a + 4 * h_out) =
            f32x4_t{o[d][4 * a], o[d][4 * a + 1], o[d][4 * a + 2], o[d][4 * a + 3]};
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = ar_out_row(p, it, r_out, D);
#pragma unroll
    for (int d = 0; d < kDb; ++d)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        float x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = o[d][4 * a + b] * inv;
        ar_store4(p, at + 32 * d + 8 * a + 4 * h_out, x);
      }
  }
  return false;
}

// ------------------------------------------------------------------ narrow

// the rows row0 .. row0 + 16 NRB - 1 of the item; returns whether they have to be done over
// (EXACT false; the same in every thread)
template <int KV, int D, int NRB, bool EXACT>
__device__ __forceinline__ bool ar_narrow(const ArParams& p, const ArItem& it, char* smem, float (*ml)[kArNarrow][2],
                                          int row0) {
  using S = ArShape<KV, D>;
  constexpr int kDb = D / 16;
  constexpr int kQ = KV == kArF32 ? D / 16 : D / 32;
  static_assert(S::kSmem >= 4 * NRB * 16 * D * 4, "the waves' accumulators meet in the tiles' LDS");
  ArLoader<KV, D> ld(p.kv, it, EXACT);
  const int lane = ld.lane, wave = ld.wave, g4 = lane >> 4, c = lane & 15;
  bf16x8_t qb[NRB][KV == kArF32 ? 1 : kQ];
  f32x4_t qf[NRB][KV == kArF32 ? kQ : 1];
  int limit[NRB];
  int lo_lim = it.k_hi;
#pragma unroll
  for (int b = 0; b < NRB; ++b) {
    const int r = row0 + b * 16 + c;
    const bool live = r < it.n_rows;
    limit[b] = live ? ar_limit(it, it.tok0 + r / p.group) : it.k_hi;
    lo_lim = limit[b] < lo_lim ? limit[b] : lo_lim;
    const char* qr = live ? ar_q_row(p, it, r) : nullptr;
#pragma unroll
    for (int s = 0; s < kQ; ++s) {
      if constexpr (KV == kArF32)
        qf[b][s] = ar_q4(p, qr, 16 * s + 4 * g4, live);
      else
        qb[b][s] = ar_q8(p, qr, 32 * s + 8 * g4, live);
    }
  }
  const int lim_min = wave_min_i32(lo_lim);
  f32x4_t o[NRB][kDb];
  float m[NRB], l[NRB];
#pragma unroll
  for (int b = 0; b < NRB; ++b) {
    m[b] = kNegInf;
    l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < kDb; ++d) o[b][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // this wave's 16 keys of a tile: rows wave * 16 + ...
  const int krow = wave * 16 + c;
  const int fk = ar_swizzle<KV, D>(krow) ^ g4;
  const int k_off = krow * S::kRowBytes;
  const int vr0 = wave * 16 + 4 * g4 + (c >> 2);
  const int vc0 = ((c & 3) >> 1) ^ ar_swizzle<KV, D>(vr0);
  const int v_off = vr0 * S::kRowBytes + 8 * (c & 1);

  const int tb0 = it.k_lo & ~15;
  const int n_tiles = (it.k_hi - tb0 + kArTile - 1) / kArTile;
  ld.fetch_pages(tb0);
  ld.issue(tb0, smem);
  int pages_now = ld.page;
  float ks_now = ld.ks, vs_now = ld.vs;
  ld.commit(smem);
  if (n_tiles > 1) ld.fetch_pages(tb0 + kArTile);
  for (int t = 0; t < n_tiles; ++t) {
    const int tb = tb0 + t * kArTile;
    char* cur = smem + (t & 1) * S::kStage;
    char* nxt = smem + ((t + 1) & 1) * S::kStage;
    ar_arrived();
    __syncthreads();
    const int pg = __builtin_amdgcn_readlane(pages_now, wave);
    const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_now), wave));
    const float vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_now), wave));
    if (t + 1 < n_tiles) {
      ld.issue(tb + kArTile, nxt);
      pages_now = ld.page;
      ks_now = ld.ks;
      vs_now = ld.vs;
      if (t + 2 < n_tiles) ld.fetch_pages(tb + 2 * kArTile);
    }
    const int kw = tb + wave * 16;
    if (pg >= 0 && kw < it.k_hi && kw + 16 > it.k_lo) {
      const char* vt = cur + S::kTileBytes;
      f32x4_t s[NRB];
#pragma unroll
      for (int b = 0; b < NRB; ++b) s[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < kQ; ++q) {
        const char* a = cur + k_off + (((4 * q) ^ fk) << 4);
        if constexpr (KV == kArF32) {
          const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a);
#pragma unroll
          for (int b = 0; b < NRB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], qf[b][q][e], s[b], 0, 0, 0);
        } else {
          const bf16x8_t x = *reinterpret_cast<const bf16x8_t*>(a);
#pragma unroll
          for (int b = 0; b < NRB; ++b) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, qb[b][q], s[b], 0, 0, 0);
        }
      }
      u32 w[NRB][2];
#pragma unroll
      for (int b = 0; b < NRB; ++b) {
        float mx = kNegInf;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[b][i] * p.scale_log2;
          if constexpr (KV == kArFp8) x *= ks;
          const int key = kw + 4 * g4 + i;
          x = key < it.k_lo || key >= limit[b] ? kNegInf : x;
          s[b][i] = x;
          mx = fmaxf(mx, x);
        }
        mx = rows_max(mx);
        if (__ballot(mx > m[b] + kArSlack) != 0) {
          const float mn = fmaxf(m[b], mx);
          const float a = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m[b] - mn);
          l[b] *= a;
#pragma unroll
          for (int d = 0; d < kDb; ++d) o[b][d] *= a;
          m[b] = mn;
        }
        const float mu = m[b] == kNegInf ? 0.f : m[b];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[b][i] = __builtin_amdgcn_exp2f(s[b][i] - mu);
          l[b] += s[b][i];
          if constexpr (KV == kArFp8) s[b][i] *= vs;
          if constexpr (EXACT) s[b][i] = kw + 4 * g4 + i < limit[b] ? s[b][i] : 0.f;
        }
        if constexpr (KV != kArF32) {
          w[b][0] = pack_bf16x2(s[b][0], s[b][1]);
          w[b][1] = pack_bf16x2(s[b][2], s[b][3]);
        }
      }
#pragma unroll
      for (int d = 0; d < kDb; ++d) {
        if constexpr (EXACT) {
          auto sees = [&](int b, int i) { return kw + 4 * g4 + i < limit[b]; };
          f32x4_t marks[NRB];
#pragma unroll
          for (int b = 0; b < NRB; ++b) marks[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          if constexpr (KV == kArF32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = wave * 16 + 4 * g4 + i;
              const int ch = (4 * d + (c >> 2)) ^ ar_swizzle<KV, D>(row);
              float x = *reinterpret_cast<const float*>(vt + row * S::kRowBytes + ch * 16 + 4 * (c & 3)), mark;
              ar_marks_f32(x, &x, &mark);
#pragma unroll
              for (int b = 0; b < NRB; ++b) {
                o[b][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[b][i], o[b][d], 0, 0, 0);
                marks[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(mark, sees(b, i) ? 1.f : 0.f, marks[b], 0, 0, 0);
              }
            }
          } else {
            const u32x2_t x = ar_read_tr(vt + v_off + (((2 * d) ^ vc0) << 4));
            u32 fin[2], mark[2];
            ar_marks_bf16(x[0], &fin[0], &mark[0]);
            ar_marks_bf16(x[1], &fin[1], &mark[1]);
#pragma unroll
            for (int b = 0; b < NRB; ++b) {
              const u32 s0 = (sees(b, 0) ? 0x3f80u : 0u) | (sees(b, 1) ? 0x3f800000u : 0u);
              const u32 s1 = (sees(b, 2) ? 0x3f80u : 0u) | (sees(b, 3) ? 0x3f800000u : 0u);
              o[b][d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(as_i16x4(fin[0], fin[1]), as_i16x4(w[b][0], w[b][1]),
                                                                  o[b][d], 0, 0, 0);
              marks[b] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(as_i16x4(mark[0], mark[1]), as_i16x4(s0, s1),
                                                                   marks[b], 0, 0, 0);
            }
          }
#pragma unroll
          for (int b = 0; b < NRB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[b][d][i] = ar_marked(o[b][d][i], marks[b][i]);
        } else if constexpr (KV == kArF32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = wave * 16 + 4 * g4 + i;
            const int ch = (4 * d + (c >> 2)) ^ ar_swizzle<KV, D>(row);
            const float x = *reinterpret_cast<const float*>(vt + row * S::kRowBytes + ch * 16 + 4 * (c & 3));
#pragma unroll
            for (int b = 0; b < NRB; ++b) o[b][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[b][i], o[b][d], 0, 0, 0);
          }
        } else {
          const u32x2_t x = ar_read_tr(vt + v_off + (((2 * d) ^ vc0) << 4));
#pragma unroll
          for (int b = 0; b < NRB; ++b)
            o[b][d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(as_i16x4(x[0], x[1]), as_i16x4(w[b][0], w[b][1]),
                                                                o[b][d], 0, 0, 0);
        }
      }
    }
    if (t + 1 < n_tiles) ld.commit(nxt);
  }
  // the four waves' partials meet in LDS: acc [4][16 NRB][D], then every thread sums its
  // elements in wave order
  bool again = false;
  if (!EXACT && it.k_hi > lim_min) {
#pragma unroll
    for (int b = 0; b < NRB; ++b) {
      float x = 0.f;  // (0, or NaN: a value of the row is not finite)
#pragma unroll
      for (int d = 0; d < kDb; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) x += 0.f * o[b][d][i];
      again |= row0 + b * 16 + c < it.n_rows && !(x == 0.f);
    }
  }
  if (__syncthreads_or(again)) return true;
  float* acc = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int b = 0; b < NRB; ++b) {
    const int r = b * 16 + c;
    const float lt = rows_sum(l[b]);
    if (g4 == 0) {
      ml[wave][r][0] = m[b];
      ml[wave][r][1] = lt;
    }
#pragma unroll
    for (int d = 0; d < kDb; ++d)
      *reinterpret_cast<f32x4_t*>(acc + ((wave * NRB * 16 + r) * D + 16 * d + 4 * g4)) = o[b][d];
  }
  __syncthreads();
  for (int i = wave; i < NRB * 16 && row0 + i < it.n_rows; i += 4) {
    const int r = row0 + i;
    float mt = kNegInf;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, ml[w][i][0]);
    const float mu = mt == kNegInf ? 0.f : mt;
    float a[4], lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      a[w] = __builtin_amdgcn_exp2f(ml[w][i][0] - mu);
      lt += a[w] * ml[w][i][1];
    }
    constexpr int kE = D / 64;
    float x[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      x[e] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) x[e] += a[w] * acc[(w * NRB * 16 + i) * D + lane * kE + e];
    }
    if (it.part_ml) {
      if (lane == 0) *reinterpret_cast<f32x2_t*>(it.part_ml + 2 * r) = f32x2_t{mt, lt};
#pragma unroll
      for (int e = 0; e < kE; ++e) it.part_acc[(int64_t)r * D + lane * kE + e] = x[e];
    } else {
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      const int64_t at = ar_out_row(p, it, r, D) + lane * kE;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        if (p.out_f32)
          reinterpret_cast<float*>(p.out)[at + e] = x[e] * inv;
        else
          reinterpret_cast<unsigned short*>(p.out)[at + e] = f32_to_bf16_bits(x[e] * inv);
      }
    }
  }
  return false;
}

template <int KV, int D>
__device__ __forceinline__ void ar_attend(const ArParams& p, const ArItem& it, char* smem) {
  __shared__ float ml[4][kArNarrow][2];
  bool again;
  if (it.n_rows > kArNarrow)
    again = ar_wide<KV, D>(p, it, smem);
  else if (it.n_rows > 16)
    again = ar_narrow<KV, D, 2, false>(p, it, smem, ml, 0);
  else
    again = ar_narrow<KV, D, 1, false>(p, it, smem, ml, 0);
  if (again)
    for (int r = 0; r < it.n_rows; r += kArNarrow) {
      ar_narrow<KV, D, 2, true>(p, it, smem, ml, r);
      __syncthreads();  // (the rows' sums have been read)
    }
}

}  // namespace ia
