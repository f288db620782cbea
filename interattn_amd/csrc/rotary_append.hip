// Keys rotated into the paged pool, values into the pool, queries rotated out, for gfx950:
// the write side of a serving step, into bf16, f32 and fp8 pages.
//
// Packed rows: a workgroup per (sequence, page its new tokens touch, slice of heads).  A wave takes one
// head's rows of the page, 16 at a time (a part), as units of VEC pairs: lane = (row, unit), so
// that the angles of its rows are computed once and serve every head, and a pair turns inside a
// lane.  Pages of up to four parts give each part a wave of its own.  Single tokens: a workgroup
// per sequence, several rows a wave.
//
// fp8 pages have one float32 scale per (page, kv head).  The waves that hold the page's new
// rows take the largest magnitude a of its finite values (a reduction inside a wave, and over
// its parts through LDS) and
//   s = 2^ceil(log2(a / 448)), at least 2^-126;
// a page that holds earlier tokens keeps its scale s0 where a <= 448 s0, else its earlier codes
// c become e4m3(c * s0 / s).  A power of two costs e4m3 no relative precision (only up to one
// binade of range at the small end) and makes both the division and the re-encoding exact, but
// for values that turn subnormal: a cache written token by token holds what one written at once
// does.  Codes are rounded from float32, without a rounding to bf16 between.
//
// Bound by HBM for prompts: 38k tokens of 8 kv heads of 128 and groups of 4, bf16 rows, are read
// and written in 162 us into fp8 pages (856 MB, 5.3 TB/s) and 164 us into bf16 ones (5.7 TB/s);
// 3.5k tokens of 4 heads of 64 in 11.5 us.  Single tokens, up to what the device holds at once, are
// bound by their round trips (length, page, rows, scale): 1 to 256 sequences of 48 heads into fp8
// pages in 4.4 to 5.1 us.  More are bound by how many run together: the fp8 kernel holds 102
// registers, a CU two of its workgroups of 6 waves, the device 512, so that 2,048 sequences are
// four rounds, 23 us, where their bytes would take 9.  (Through the packed rows' kernel 8.2 to 25
// and 71.)
#include <algorithm>

#include "packed_rows.hpp"
#include "rotary.hpp"
#include "row_spans.hpp"

namespace ia {

int check_kv(const ia_paged_kv* kv, int d);

namespace {

constexpr int kWriteThreads = 256, kWaves = kWriteThreads / 64;
constexpr int kTokenThreads = 1024;  // at most, of a workgroup for one token
constexpr int kWriteBytes = 48 << 10, kWriteBytesFp8 = 96 << 10;
constexpr int kSub = 16;  // rows of a page taken at a time
constexpr float kLargestCode = 448.f;
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126

struct WriteParams {
  // new rows and rotated queries (strides in bytes)
  const char* q;
  char* q_out;
  const char* k_new;
  const char* v_new;
  int64_t q_tok, q_head, qo_tok, qo_head, kn_tok, kn_head, vn_tok, vn_head;
  // pool (strides in bytes)
  char* k;
  char* v;
  int64_t k_page, k_head, k_tok, v_page, v_head, v_tok;
  float* k_scale;
  float* v_scale;
  int64_t scale_page;
  const int32_t* table;
  int64_t bt_stride, bt_cols, n_pages;
  int32_t page_rows;
  // batch
  const int32_t* cu;
  const int32_t* seq_lens;
  int32_t* new_lens;
  const int32_t* positions;  // null: the place in the sequence
  int32_t n_seq, n_tokens, n_kv_heads, group, kv_heads_per_wg, slices;
  RotaryArgs rot;
  bool stream;  // the queries' rows are written past the caches
};

__device__ __forceinline__ int64_t write_page(const WriteParams& p, int b, int64_t lp) {
  int64_t pg = lp;
  if (p.table) pg = lp < p.bt_cols ? p.table[(int64_t)b * p.bt_stride + lp] : -1;
  return pg < 0 || pg >= p.n_pages ? -1 : pg;
}

// The least power of two, 2^-126 at least, that brings a down to 448 or less: with
// a = m 2^e, m in [1, 2), 448 = 1.75 2^8 asks for 2^(e - 8), or twice that for m > 1.75.
__device__ __forceinline__ float page_scale(float a) {
  const u32 bits = __float_as_uint(a);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return __uint_as_float((u32)(max(e, -126) + 127) << 23);
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Four floats, already divided by their scale, as e4m3 codes.
__device__ __forceinline__ u32 fp8_codes(const float* x) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  return (u32)w;
}

// Not finite: NaN, which has a code (infinity has none).
__device__ __forceinline__ float or_nan(float x) { return finite(x) ? x : __uint_as_float(0x7fc00000u); }

// The earlier rows [0, n) of one head's page from scale s0 to s, by LANES lanes.
template <int D, int LANES>
__device__ void recode(char* rows, int64_t tok_stride, int n, float s0, float s, int lane) {
  const float ratio = s0 / s;
  constexpr int kChunks = D / 16;
  for (int i = lane; i < n * kChunks; i += LANES) {
    u32x4_t* at = reinterpret_cast<u32x4_t*>(rows + i / kChunks * tok_stride + i % kChunks * 16);
    u32x4_t w = *at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
      fp8x4_to_f32(w[i], x);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = or_nan(x[j] * ratio);
      w[i] = fp8_codes(x);
    }
    *at = w;
  }
}

// A unit's elements y as codes over the scale s, inv its reciprocal where that is exact (0 where
// not).
template <int LAYOUT, int VEC>
__device__ __forceinline__ void put_unit_codes(char* to, int u, int rot, int d, const float* y, float s, float inv) {
  int a, b;
  unit_chunks<LAYOUT, VEC>(u, rot, d, &a, &b);
  float z[2 * VEC < 4 ? 4 : 2 * VEC] = {};
  if (inv != 0.f) {
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) z[j] = y[j] * inv;
  } else {
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) z[j] = y[j] / s;
  }
  if constexpr (VEC == 8) {
    *reinterpret_cast<u32x2_t*>(to + a) = u32x2_t{fp8_codes(z), fp8_codes(z + 4)};
    *reinterpret_cast<u32x2_t*>(to + b) = u32x2_t{fp8_codes(z + 8), fp8_codes(z + 12)};
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<u32*>(to + a) = fp8_codes(z);
    *reinterpret_cast<u32*>(to + b) = fp8_codes(z + 4);
  } else {
    const u32 c = fp8_codes(z);
    to[a] = (char)(c & 0xff);
    to[b] = (char)(c >> 8 & 0xff);
  }
}

// (a power of two is divided by exactly through its reciprocal)
__device__ __forceinline__ float exact_inverse(float s) { return (__float_as_uint(s) & 0x7fffffu) == 0 ? 1.f / s : 0.f; }

// The scale for new values of magnitude a of a page whose scale was s0; keeps: the earlier
// codes stay as they are.
__device__ __forceinline__ float settle(float a, bool begun, float s0, bool* keeps) {
  *keeps = begun && finite(s0) && s0 >= kLeastScale && a <= kLargestCode * s0;
  return *keeps ? s0 : page_scale(a);
}

// One page of one sequence, as all of its tasks see it.
struct WritePage {
  int64_t page;  // -1: none
  int64_t tok;   // packed row of page row 0 (may lie before the first row)
  int lo, hi;    // the new rows' places in the page
};

// 16 rows of a page by one wave.  Lanes without a new row hold the nearest one: loads need no
// condition (a branch around one would make every load wait for all before it), a maximum is
// the same, and only stores ask.
template <typename T, int D, int LAYOUT>
struct PageRows {
  using Unit = RowUnit<T, LAYOUT>;
  using Turns = typename Unit::Turns;
  static constexpr int kVec = Unit::kVec;
  static constexpr int kUnits = D / (2 * kVec);  // of a row
  static constexpr int kRows = 64 / kUnits;      // a wave's rows at once
  static constexpr int kGroups = kSub / kRows;   // of 16 rows
  static constexpr int kFly = kGroups >= 4 ? 1 : 4 / kGroups;  // heads whose loads are in flight together
  static_assert(kRows >= 1 && kRows <= kSub, "a wave holds 1 to 16 rows, a unit a lane");

  const WriteParams& p;
  const WritePage& w;
  int unit, row;
  Turns turns;  // of q and k
  Turns none;   // of v
  float cs[kGroups][kVec], sn[kGroups][kVec];

  __device__ __forceinline__ PageRows(const WriteParams& p_, const WritePage& w_, int lane)
      : p(p_), w(w_), unit(lane % kUnits), row(lane / kUnits), turns(lane % kUnits, p_.rot.rot, D), none(lane % kUnits, 0, D) {}

  __device__ __forceinline__ int place(int sub, int g) const { return sub * kSub + g * kRows + row; }
  __device__ __forceinline__ bool mine(int at) const { return at >= w.lo && at < w.hi; }
  __device__ __forceinline__ int64_t token(int at) const { return w.tok + min(max(at, w.lo), w.hi - 1); }

  __device__ __forceinline__ void angles(int sub, int64_t shift) {
    if (p.rot.rot == 0) return;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int64_t tok = token(place(sub, g));
      unit_angles<LAYOUT, kVec>(p.rot, p.positions ? p.positions[tok] : (int)(tok + shift), turns, cs[g], sn[g]);
    }
  }

  __device__ __forceinline__ void load(Unit* x, const char* rows, int64_t tok_stride, int sub) const {
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      x[g].template load<false>(reinterpret_cast<const T*>(rows + token(place(sub, g)) * tok_stride), unit, p.rot.rot, D);
  }

  // as rows of T, row0 the row of the page's first place
  __device__ __forceinline__ void put(const Unit* x, const Turns& t, char* rows, int64_t tok_stride, int64_t row0, int sub,
                                      bool stream) const {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int at = place(sub, g);
      float y[2 * kVec];
      x[g].turned(cs[g], sn[g], t, y);
      if (!mine(at)) continue;
      T* to = reinterpret_cast<T*>(rows + (row0 + at) * tok_stride);
      if (stream) {
        // (the asm keeps the two branches' stores from being made one, without the hint)
        asm volatile("");
        store_unit<T, LAYOUT, true>(to, unit, p.rot.rot, D, y);
        asm volatile("");
      } else {
        store_unit<T, LAYOUT, false>(to, unit, p.rot.rot, D, y);
      }
    }
  }

  using Values = float[kGroups][2 * kVec];

  __device__ __forceinline__ void turn(const Unit* x, const Turns& t, Values& y) const {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) x[g].turned(cs[g], sn[g], t, y[g]);
  }

  // Largest finite magnitude of the rows, in every lane; what is not finite becomes NaN.  As
  // integers, floats of either sign rise with their magnitude, and what is not finite is above
  // all others: one maximum of each sign finds both.
  __device__ __forceinline__ float largest(Values& y) const {
    int plus = 0;
    u32 minus = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int j = 0; j < 2 * kVec; ++j) {
        plus = max(plus, __float_as_int(y[g][j]));
        minus = max(minus, __float_as_uint(y[g][j]));
      }
    float a = __uint_as_float(max((u32)plus, minus & 0x7fffffffu));
    if (!finite(a)) {
      a = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int j = 0; j < 2 * kVec; ++j) {
          y[g][j] = or_nan(y[g][j]);
          a = fmaxf(a, fabsf(y[g][j]));  // (a maximum passes over NaN)
        }
    }
    return wave_max(a);
  }

  // as e4m3 codes over the scale s
  __device__ __forceinline__ void put_codes(const Values& y, char* rows, int64_t tok_stride, int sub, float s) const {
    const float inv = exact_inverse(s);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int at = place(sub, g);
      if (mine(at)) put_unit_codes<LAYOUT, kVec>(rows + at * tok_stride, unit, p.rot.rot, D, y[g], s, inv);
    }
  }
};

// A head's tensor of the page's tasks: queries first, then keys, then values.
struct WriteTask {
  const char* from;
  int64_t from_tok;
  char* rows;  // page row 0
  int64_t tok;
  float* scale;
  bool value;
};

__device__ __forceinline__ WriteTask kv_task(const WriteParams& p, int64_t page, int kv0, int n_kv, int i) {
  const bool value = i >= n_kv;
  const int64_t h = kv0 + (value ? i - n_kv : i);
  WriteTask t;
  t.value = value;
  t.from = value ? p.v_new + h * p.vn_head : p.k_new + h * p.kn_head;
  t.from_tok = value ? p.vn_tok : p.kn_tok;
  t.rows = value ? p.v + page * p.v_page + h * p.v_head : p.k + page * p.k_page + h * p.k_head;
  t.tok = value ? p.v_tok : p.k_tok;
  t.scale = value ? p.v_scale + page * p.scale_page + h : p.k_scale + page * p.scale_page + h;
  return t;
}

template <typename T, bool FP8, int D, int LAYOUT>
__global__ __launch_bounds__(kWriteThreads) void ia_write_pages(WriteParams p) {
  using Rows = PageRows<T, D, LAYOUT>;
  using Unit = typename Rows::Unit;
  constexpr int kFly = Rows::kFly, kGroups = Rows::kGroups;
  __shared__ int first_gap;
  __shared__ float parts[2][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // slices of a tile are neighbours, as their rows are in memory (with one slice of every tile
  // behind another, pages of 64 took 207 us instead of 164, pages of 16 165 instead of 162)
  const int tile = blockIdx.x / p.slices, slice = blockIdx.x - tile * p.slices;
  const PackedTile own = packed_tile(p.cu, p.n_seq, p.n_tokens, p.page_rows, tile, lane, 2);
  const int b = own.b, first = own.first, count = own.count;
  const int64_t local = own.local;
  if (local < 0) return;
  const int64_t past = p.seq_lens[b];
  if (local == 0 && slice == 0) {
    // the length: up to the first position without a page
    if (tid == 0) first_gap = INT32_MAX;
    __syncthreads();
    const int64_t end = past + count;
    if (past >= 0 && count > 0)
      for (int64_t lp = past / p.page_rows + tid; lp * p.page_rows < end; lp += blockDim.x)
        if (write_page(p, b, lp) < 0) {
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
      p.new_lens[b] = (int)len;
    }
  }
  const int64_t start = past < 0 ? 0 : past;  // (a negative length: the queries only)
  const int64_t lp = start / p.page_rows + local, base = lp * p.page_rows;
  if (count == 0 || base >= start + count) return;  // (no rows: none to hold in their place either)
  WritePage w;
  w.page = past < 0 ? -1 : write_page(p, b, lp);
  w.tok = first + (base - start);
  w.lo = (int)(start > base ? start - base : 0);
  w.hi = (int)(start + count - base < p.page_rows ? start + count - base : p.page_rows);
  const int64_t shift = past - first;  // a token's position less its packed row
  const int kv0 = slice * p.kv_heads_per_wg, n_kv = min(kv0 + p.kv_heads_per_wg, p.n_kv_heads) - kv0;
  const int n_q = p.q ? n_kv * p.group : 0;

  // parts with new rows: 1, 2 or up to 4 waves share a head's page, each with a part of its own;
  // with more parts each wave goes through several
  const int sub0 = w.lo / kSub, subs = (w.hi + kSub - 1) / kSub - sub0;
  const int share = subs == 1 ? 1 : subs == 2 ? 2 : 4;
  const int step = kWaves / share, slot = wave / share, part = wave % share;
  const int turns_each = (subs + share - 1) / share;
  Rows rows(p, w, lane);
  for (int k = 0; k < turns_each; ++k) {
    const int sub = sub0 + part + k * share;
    rows.angles(sub, shift);
    for (int i = slot; i < n_q; i += kFly * step) {
      Unit x[kFly][kGroups];
#pragma unroll
      for (int f = 0; f < kFly; ++f)
        rows.load(x[f], p.q + ((int64_t)kv0 * p.group + min(i + f * step, n_q - 1)) * p.q_head, p.q_tok, sub);
#pragma unroll
      for (int f = 0; f < kFly; ++f)
        if (i + f * step < n_q)
          rows.put(x[f], rows.turns, p.q_out + ((int64_t)kv0 * p.group + i + f * step) * p.qo_head, p.qo_tok, w.tok, sub,
                   p.stream);
    }
    if (FP8 || w.page < 0) continue;
    for (int i = slot; i < 2 * n_kv; i += kFly * step) {
      Unit x[kFly][kGroups];
#pragma unroll
      for (int f = 0; f < kFly; ++f) {
        const WriteTask t = kv_task(p, w.page, kv0, n_kv, min(i + f * step, 2 * n_kv - 1));
        rows.load(x[f], t.from, t.from_tok, sub);
      }
#pragma unroll
      for (int f = 0; f < kFly; ++f) {
        if (i + f * step >= 2 * n_kv) break;
        const WriteTask t = kv_task(p, w.page, kv0, n_kv, i + f * step);
        rows.put(x[f], t.value ? rows.none : rows.turns, t.rows, t.tok, 0, sub, p.stream);
      }
    }
  }
  if constexpr (FP8) {
    if (w.page < 0) return;
    // (every wave runs every round: the barriers are the workgroup's)
    int exchange = 0;
    for (int i0 = slot; i0 - slot < 2 * n_kv; i0 += kFly * step) {
      Unit x[kFly][kGroups];
      float s0[kFly];
#pragma unroll
      for (int f = 0; f < kFly; ++f) {
        const WriteTask t = kv_task(p, w.page, kv0, n_kv, min(i0 + f * step, 2 * n_kv - 1));
        s0[f] = w.lo > 0 ? *t.scale : 0.f;
        rows.load(x[f], t.from, t.from_tok, sub0 + part);
      }
#pragma unroll
      for (int f = 0; f < kFly; ++f) {
        const int i = i0 + f * step;
        const WriteTask t = kv_task(p, w.page, kv0, n_kv, min(i, 2 * n_kv - 1));
        const typename Rows::Turns& turns = t.value ? rows.none : rows.turns;
        typename Rows::Values y;
        float a = 0.f;
        for (int k = 0; k < turns_each && i < 2 * n_kv; ++k) {
          if (turns_each > 1) {
            rows.load(x[f], t.from, t.from_tok, sub0 + part + k * share);
            if (!t.value) rows.angles(sub0 + part + k * share, shift);
          }
          rows.turn(x[f], turns, y);
          a = fmaxf(a, rows.largest(y));
        }
        if (share > 1) {
          float* mine = parts[exchange++ & 1];
          if (lane == 0) mine[wave] = a;
          __syncthreads();  // (and the earlier scale has been read by every wave)
          for (int o = 0; o < share; ++o) a = fmaxf(a, mine[slot * share + o]);
        }
        if (i >= 2 * n_kv) continue;
        bool keeps;
        const float s = settle(a, w.lo > 0, s0[f], &keeps);
        if (part == 0) {
          if (w.lo > 0 && !keeps) recode<D, 64>(t.rows, t.tok, w.lo, s0[f], s, lane);
          if (lane == 0) *t.scale = s;
        }
        for (int k = 0; k < turns_each; ++k) {
          const int sub = sub0 + part + k * share;
          if (turns_each > 1) {
            rows.load(x[f], t.from, t.from_tok, sub);
            if (!t.value) rows.angles(sub, shift);
            rows.turn(x[f], turns, y);
            rows.largest(y);  // (what is not finite)
          }
          rows.put_codes(y, t.rows, t.tok, sub, s);
        }
      }
    }
  }
}

// One token of one sequence by a workgroup: a unit of a row (a query, key or value head) a lane,
// several rows a wave, so that the call is the chain length -> page -> scale and everything else
// (rows, frequencies) is loaded beside it.
template <typename T, bool FP8, int D, int LAYOUT>
__global__ __launch_bounds__(kTokenThreads) void ia_write_tokens(WriteParams p) {
  using Unit = RowUnit<T, LAYOUT>;
  constexpr int kVec = Unit::kVec, kUnits = D / (2 * kVec);
  const int b = blockIdx.x, tid = threadIdx.x, unit = tid % kUnits;
  const int64_t past = p.seq_lens[b];
  const int n_q = p.q ? p.group * p.n_kv_heads : 0, n_rows = n_q + 2 * p.n_kv_heads, step = blockDim.x / kUnits;
  int64_t page = -1, lp = 0;
  float cs[kVec], sn[kVec];
  for (int r = tid / kUnits; r < n_rows; r += step) {
    const bool query = r < n_q, value = r >= n_q + p.n_kv_heads;
    const int64_t h = query ? r : value ? r - n_q - p.n_kv_heads : r - n_q;
    const char* from = query ? p.q + b * p.q_tok + h * p.q_head
                             : value ? p.v_new + b * p.vn_tok + h * p.vn_head : p.k_new + b * p.kn_tok + h * p.kn_head;
    Unit x;
    x.template load<false>(reinterpret_cast<const T*>(from), unit, p.rot.rot, D);
    if (r < step) {  // (the first of the lane's rows: behind its load)
      if (past >= 0) {
        lp = past / p.page_rows;
        page = write_page(p, b, lp);
      }
      unit_angles<LAYOUT, kVec>(p.rot, p.positions ? p.positions[b] : (int)past,
                                typename Unit::Turns(unit, p.rot.rot, D), cs, sn);
    }
    const int lo = (int)(past - lp * p.page_rows);
    char* rows = value ? p.v + page * p.v_page + h * p.v_head : p.k + page * p.k_page + h * p.k_head;
    const int64_t tok = value ? p.v_tok : p.k_tok;
    float* scale = (value ? p.v_scale : p.k_scale) + page * p.scale_page + h;
    const bool writes = !query && page >= 0;
    float s0 = 0.f;
    if (FP8 && writes && lo > 0) s0 = *scale;
    float y[2 * kVec];
    x.turned(cs, sn, typename Unit::Turns(unit, value ? 0 : p.rot.rot, D), y);
    if (query || (!FP8 && writes)) {
      char* to = query ? p.q_out + b * p.qo_tok + h * p.qo_head : rows + lo * tok;
      store_unit<T, LAYOUT, false>(reinterpret_cast<T*>(to), unit, p.rot.rot, D, y);
    }
    if constexpr (FP8) {
      float a = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * kVec; ++j) {
        y[j] = or_nan(y[j]);
        a = fmaxf(a, fabsf(y[j]));  // (a maximum passes over NaN)
      }
#pragma unroll
      for (int m = 1; m < kUnits; m <<= 1) a = fmaxf(a, __shfl_xor(a, m, 64));
      if (!writes) continue;
      bool keeps;
      const float s = settle(a, lo > 0, s0, &keeps);
      if (lo > 0 && !keeps) recode<D, kUnits>(rows, tok, lo, s0, s, unit);
      put_unit_codes<LAYOUT, kVec>(rows + lo * tok, unit, p.rot.rot, D, y, s, exact_inverse(s));
      if (unit == 0) *scale = s;
    }
  }
  __syncthreads();  // (every thread has read the length, which may be written in place)
  if (tid == 0) p.new_lens[b] = (int)(page >= 0 ? past + 1 : past);
}

template <typename T, bool FP8, int D, int LAYOUT>
void launch_layout(dim3 grid, hipStream_t st, const WriteParams& p) {
  if (p.cu) {
    hipLaunchKernelGGL((ia_write_pages<T, FP8, D, LAYOUT>), grid, dim3(kWriteThreads), 0, st, p);
    return;
  }
  const int64_t lanes = (int64_t)p.n_kv_heads * (2 + (p.q ? p.group : 0)) * (D / (2 * RowVec<T, LAYOUT>::kVec));
  const unsigned threads = (unsigned)std::min<int64_t>((lanes + 63) / 64 * 64, kTokenThreads);
  hipLaunchKernelGGL((ia_write_tokens<T, FP8, D, LAYOUT>), grid, dim3(threads), 0, st, p);
}

template <typename T, bool FP8, int D>
void launch_write(int layout, dim3 grid, hipStream_t st, const WriteParams& p) {
  if (layout == kRowsHalf)
    launch_layout<T, FP8, D, kRowsHalf>(grid, st, p);
  else if (layout == kRowsInterleaved)
    launch_layout<T, FP8, D, kRowsInterleaved>(grid, st, p);
  else
    launch_layout<T, FP8, D, kRowsHalfOdd>(grid, st, p);
}

template <typename T, bool FP8>
void launch_write_d(int d, int layout, dim3 grid, hipStream_t st, const WriteParams& p) {
  if (d == 64)
    launch_write<T, FP8, 64>(layout, grid, st, p);
  else
    launch_write<T, FP8, 128>(layout, grid, st, p);
}

}  // namespace
}  // namespace ia

extern "C" int ia_rotary_append_kv(const ia_rotary* rotary, const ia_rotary_rows* q, const ia_packed_kv* rows,
                                   const ia_paged_kv* kv, const int32_t* cu_seqlens, const int32_t* seq_lens,
                                   int32_t* new_seq_lens, const int32_t* positions, int32_t n_seq, int32_t n_tokens,
                                   int32_t n_kv_heads, int32_t head_dim, void* stream) {
  using namespace ia;
  if (!rows || (n_seq > 0 && (!seq_lens || !new_seq_lens))) return fail(IA_ERR_INVALID, "null pointer argument");
  if (head_dim != 64 && head_dim != 128) return fail(IA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  int rc = check_kv(kv, head_dim);
  if (rc) return rc;
  if (rotary && (rc = check_rotary(rotary, head_dim))) return rc;
  const bool fp8 = kv->dtype == IA_FP8_E4M3;
  if (rows->dtype != IA_F32 && rows->dtype != IA_BF16) return fail(IA_ERR_INVALID, "the new rows must be f32 or bf16");
  if (!fp8 && rows->dtype != kv->dtype) return fail(IA_ERR_INVALID, "the new rows must have the pool's dtype");
  if (fp8 && kv->n_pages > 1 && kv->scale_page_stride < n_kv_heads)
    return fail(IA_ERR_INVALID, "every page needs scales of its own");
  if (kv->seq_scale) return fail(IA_ERR_INVALID, "scales gathered per sequence are not written: pass none");
  if (n_seq < 0 || n_tokens < 0 || n_kv_heads <= 0) return fail(IA_ERR_INVALID, "sequence, token or head counts");
  if (n_tokens > 0 && (!rows->k || !rows->v)) return fail(IA_ERR_INVALID, "null pointer argument");
  if (!cu_seqlens && n_tokens != n_seq)
    return fail(IA_ERR_INVALID, "without cu_seqlens every sequence has one token");
  const int eb = rows->dtype == IA_F32 ? 4 : 2, pb = fp8 ? 1 : eb;
  const int64_t strides[4] = {rows->k_token_stride, rows->k_head_stride, rows->v_token_stride, rows->v_head_stride};
  for (int64_t s : strides)
    if (s < 0 || (s * eb) % 16) return fail(IA_ERR_INVALID, "row strides must be non-negative 16-byte multiples");
  if ((reinterpret_cast<uintptr_t>(rows->k) | reinterpret_cast<uintptr_t>(rows->v)) % 16)
    return fail(IA_ERR_INVALID, "rows must be 16-byte aligned");
  const bool in_place = n_seq > 0 && new_seq_lens == seq_lens;
  if (in_place && cu_seqlens)
    return fail(IA_ERR_INVALID, "lengths advance in place for single tokens only (cu_seqlens null)");
  // (lengths are written while other waves still look for their positions)
  if (positions && ints_meet(positions, n_tokens, new_seq_lens, n_seq))
    return fail(IA_ERR_INVALID, "positions must not overlap new_seq_lens");
  WriteParams p{};
  p.group = 1;
  if (q) {
    if (q->n_heads <= 0 || q->n_heads % n_kv_heads)
      return fail(IA_ERR_INVALID, "n_q_heads must be a positive multiple of n_kv_heads");
    if (n_tokens > 0 && (!q->in || !q->out)) return fail(IA_ERR_INVALID, "null pointer argument");
    const int64_t qs[4] = {q->in_token_stride, q->in_head_stride, q->out_token_stride, q->out_head_stride};
    for (int64_t s : qs)
      if (s < 0 || (s * eb) % 16) return fail(IA_ERR_INVALID, "row strides must be non-negative 16-byte multiples");
    const RowSpan out(q->out, n_tokens, q->n_heads, q->out_token_stride * eb, q->out_head_stride * eb, head_dim * eb);
    if (!out.rows_apart()) return fail(IA_ERR_INVALID, "output rows must not overlap");
    if ((reinterpret_cast<uintptr_t>(q->in) | reinterpret_cast<uintptr_t>(q->out)) % 16)
      return fail(IA_ERR_INVALID, "rows must be 16-byte aligned");
    p.q = static_cast<const char*>(q->in);
    p.q_out = static_cast<char*>(q->out);
    p.q_tok = q->in_token_stride * eb;
    p.q_head = q->in_head_stride * eb;
    p.qo_tok = q->out_token_stride * eb;
    p.qo_head = q->out_head_stride * eb;
    p.group = q->n_heads / n_kv_heads;
  }
  if (n_seq == 0) return IA_OK;
  p.k_new = static_cast<const char*>(rows->k);
  p.v_new = static_cast<const char*>(rows->v);
  p.kn_tok = rows->k_token_stride * eb;
  p.kn_head = rows->k_head_stride * eb;
  p.vn_tok = rows->v_token_stride * eb;
  p.vn_head = rows->v_head_stride * eb;
  p.k = static_cast<char*>(const_cast<void*>(kv->k));
  p.v = static_cast<char*>(const_cast<void*>(kv->v));
  p.k_page = kv->k_page_stride * pb;
  p.k_head = kv->k_head_stride * pb;
  p.k_tok = kv->k_token_stride * pb;
  p.v_page = kv->v_page_stride * pb;
  p.v_head = kv->v_head_stride * pb;
  p.v_tok = kv->v_token_stride * pb;
  p.k_scale = const_cast<float*>(kv->k_scale);
  p.v_scale = const_cast<float*>(kv->v_scale);
  p.scale_page = kv->scale_page_stride;
  p.table = kv->block_table;
  p.bt_stride = kv->bt_stride;
  p.bt_cols = kv->bt_cols;
  p.n_pages = kv->n_pages;
  p.page_rows = kv->page_size;
  p.cu = cu_seqlens;
  p.seq_lens = seq_lens;
  p.new_lens = new_seq_lens;
  p.positions = positions;
  p.n_seq = n_seq;
  p.n_tokens = n_tokens;
  p.n_kv_heads = n_kv_heads;
  p.rot = RotaryArgs{rotary ? reinterpret_cast<const unsigned long long*>(rotary->turns) : nullptr,
                     rotary ? rotary->dim : 0, rotary ? rotary->factor : 1.f, 1.f};
  const int64_t tiles = cu_seqlens ? (int64_t)n_tokens / p.page_rows + 2 * (int64_t)n_seq : n_seq;
  if (tiles >= (int64_t)1 << 23) return fail(IA_ERR_UNSUPPORTED, "too many tokens for one launch");
  // A workgroup takes about kWriteBytes of rows, into 8 bits about as many K and V rows as its
  // waves have in flight: 38k tokens of 8 kv heads of 128 bf16 and groups of 4 into pages of 16
  // took 162 us with half of the heads to a workgroup, 177 with all and 177 with a quarter; into
  // bf16 pages 176 with half, 190 with all, 164 with a quarter and 212 with one.
  // Few tiles: a workgroup for each kv head.
  const int64_t head_rows = (int64_t)p.page_rows * (2 + (q ? p.group : 0)) * head_dim * eb;
  int64_t slices = n_kv_heads;
  if (tiles >= 2 * device_cus())
    slices = std::clamp<int64_t>(n_kv_heads * head_rows / (fp8 ? kWriteBytesFp8 : kWriteBytes), 1, n_kv_heads);
  p.kv_heads_per_wg = (int)((n_kv_heads + slices - 1) / slices);
  p.slices = cu_seqlens ? (n_kv_heads + p.kv_heads_per_wg - 1) / p.kv_heads_per_wg : 1;
  if (tiles * p.slices >= (int64_t)1 << (cu_seqlens ? 23 : 22))
    return fail(IA_ERR_UNSUPPORTED, "too many tokens for one launch");
  // (a sequence's length is written while other workgroups still read theirs, and where they begin)
  if (!in_place && ints_meet(new_seq_lens, n_seq, seq_lens, n_seq))
    return fail(IA_ERR_INVALID, "new_seq_lens must not overlap seq_lens");
  if (cu_seqlens && ints_meet(new_seq_lens, n_seq, cu_seqlens, (int64_t)n_seq + 1))
    return fail(IA_ERR_INVALID, "new_seq_lens must not overlap cu_seqlens");
  // (keys and values are written by different waves)
  if (kv->k == kv->v) return fail(IA_ERR_INVALID, "the K and V pools must not be one");
  if (fp8 && may_meet(RowSpan(kv->k_scale, kv->n_pages, 1, kv->scale_page_stride * 4, 0, (int64_t)n_kv_heads * 4),
                      RowSpan(kv->v_scale, kv->n_pages, 1, kv->scale_page_stride * 4, 0, (int64_t)n_kv_heads * 4)))
    return fail(IA_ERR_INVALID, "k_scale and v_scale must not share memory: the call sets both");
  if (q) {
    // (a lane reads the queries that it writes itself, and nothing else of the output)
    const RowSpan out(p.q_out, n_tokens, q->n_heads, p.qo_tok, p.qo_head, head_dim * eb),
        in(p.q, n_tokens, q->n_heads, p.q_tok, p.q_head, head_dim * eb),
        k(p.k_new, n_tokens, n_kv_heads, p.kn_tok, p.kn_head, head_dim * eb),
        v(p.v_new, n_tokens, n_kv_heads, p.vn_tok, p.vn_head, head_dim * eb);
    if ((may_meet(out, in) && !out.same(in)) || may_meet(out, k) || may_meet(out, v))
      return fail(IA_ERR_INVALID, "the turned queries must be the queries themselves, or overlap no input");
  }
  const dim3 grid((unsigned)(tiles * p.slices));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int layout = rotary_layout(rotary, eb);
  p.stream = stream_rows(rotary, layout, (int64_t)n_tokens * p.group * n_kv_heads * head_dim * eb, eb);
  if (rows->dtype == IA_BF16)
    fp8 ? launch_write_d<bf16_t, true>(head_dim, layout, grid, st, p)
        : launch_write_d<bf16_t, false>(head_dim, layout, grid, st, p);
  else
    fp8 ? launch_write_d<float, true>(head_dim, layout, grid, st, p)
        : launch_write_d<float, false>(head_dim, layout, grid, st, p);
  return check_launch("rotary append kv");
}
