// Rotary positions: angles from whole positions, and rows of a head as pairs.
//
// Pair p of a head at position t turns by t * w[p].  w is held as turns of a circle in 64-bit
// fixed point, rounded once from the model's float64 frequencies, so that t * w modulo one turn
// is an integer product that drops what overflows: every position of 31 bits and sign has its
// frequency's angle to 1.25 * 2^-32 turns (1.8e-9 radians: 2^-32 cut off and 2^31 roundings of
// 2^-65), with no table and no range reduction in floating point (in float32, t * w at t = 10^6
// is off by 0.03).
#pragma once

#include "ia_common.hpp"

namespace ia {

// The angle's turn in 2^-32, of position t and frequency w (2^-64 turns a position): the
// upper half of the low 64 bits of t * w.
__device__ __forceinline__ u32 rotary_turn(int t, unsigned long long w) {
  const u32 lo = (u32)w, hi = (u32)(w >> 32);
  return __umulhi((u32)t, lo) + (u32)t * hi - (t < 0 ? lo : 0u);
}

// Sine and cosine of a turn: the nearest quarter is taken off, and what is left, x in
// [-pi/4, pi/4], goes through the Taylor sums to x^9 and x^8 (remainders 2e-9 and 2.5e-8).
__device__ __forceinline__ void rotary_sincos(u32 turn, float* sn, float* cs) {
  const u32 near = turn + 0x20000000u, quarter = near >> 30;
  const float x = (float)(int)(turn - (near & 0xc0000000u)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float s = fmaf(z, 2.7557319223985891e-6f, -1.9841269841269841e-4f);
  s = fmaf(z, s, 8.3333333333333333e-3f);
  s = fmaf(z, s, -1.6666666666666667e-1f);
  s = fmaf(x * z, s, x);
  float c = fmaf(z, 2.4801587301587302e-5f, -1.3888888888888889e-3f);
  c = fmaf(z, c, 4.1666666666666667e-2f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.f);
  const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
  *sn = quarter & 2 ? -a : a;
  *cs = (quarter + 1) & 2 ? -b : b;
}

// How a head's D elements are taken as D / 2 pairs.  A lane holds a unit of VEC pairs: two
// chunks of VEC elements, so that neighbouring lanes read neighbouring chunks.  VEC fills 16
// bytes but in the last layout.
//   kRowsHalf         pair (i, i + rot / 2): a chunk of each half; rot a multiple of 2 * VEC
//   kRowsInterleaved  pair (2 i, 2 i + 1): chunks u and u + D / (2 VEC), VEC / 2 pairs in each
//   kRowsHalfOdd      as kRowsHalf for any even rot: one pair a lane, so that a wave's accesses
//                     are neighbours though the halves begin anywhere
// Channels past rot are not turned; rot 0 (values) is a row of plain chunks in any layout.
enum RowLayout { kRowsHalf = 0, kRowsInterleaved = 1, kRowsHalfOdd = 2 };

template <typename T, int LAYOUT = kRowsHalf>
struct RowVec {
  static constexpr int kVec = LAYOUT == kRowsHalfOdd ? 1 : 16 / (int)sizeof(T);
};

struct bf16_t {
  unsigned short bits;
};

__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((u32)v.bits << 16); }
__device__ __forceinline__ float to_f32(float v) { return v; }

// 16 bytes of T as floats and back
__device__ __forceinline__ void widen(const u32x4_t& w, float* x, bf16_t) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = bf16_lo(w[j]);
    x[2 * j + 1] = bf16_hi(w[j]);
  }
}
__device__ __forceinline__ void widen(const u32x4_t& w, float* x, float) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]);
}
__device__ __forceinline__ u32x4_t narrow(const float* x, bf16_t) {
  return u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}
__device__ __forceinline__ u32x4_t narrow(const float* x, float) {
  return u32x4_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
}

// Elements at which a unit's two chunks begin.
template <int LAYOUT, int VEC>
__device__ __forceinline__ void unit_chunks(int u, int rot, int d, int* a, int* b) {
  if constexpr (LAYOUT == kRowsInterleaved) rot = 0;  // (its chunks lie as those of a plain row)
  const int turned = rot / (2 * VEC);
  *a = u < turned ? u * VEC : rot + (u - turned) * VEC;
  *b = *a + (u < turned ? rot : d - rot) / 2;
}

// Pair j of unit u; pairs from rot / 2 on are not turned.
template <int LAYOUT, int VEC>
__device__ __forceinline__ int unit_pair(int u, int j, int d) {
  if constexpr (LAYOUT == kRowsInterleaved) return (u * VEC + (j < VEC / 2 ? 0 : d / 2 - VEC)) / 2 + j;
  return u * VEC + j;
}

// Which pairs of a unit turn: those below `end`; in half layouts all or none.
template <int LAYOUT, int VEC>
struct UnitTurns {
  int unit, d, end;
  bool all;
  __device__ __forceinline__ UnitTurns(int u, int rot, int d_) : unit(u), d(d_), end(rot / 2) {
    all = unit_pair<LAYOUT, VEC>(u, VEC - 1, d) < end;  // (the last pair is the unit's highest)
  }
  __device__ __forceinline__ bool turns(int j) const {
    if constexpr (LAYOUT == kRowsInterleaved) return unit_pair<LAYOUT, VEC>(unit, j, d) < end;
    return all;
  }
};

// One unit of a row as it lies in memory.
template <typename T, int LAYOUT>
struct RowUnit {
  static constexpr int kVec = RowVec<T, LAYOUT>::kVec;
  static constexpr int kA = LAYOUT == kRowsInterleaved ? 2 : 1;      // pair j is x[kA j]
  static constexpr int kB = LAYOUT == kRowsInterleaved ? 1 : kVec;  // and x[kA j + kB]
  using Turns = UnitTurns<LAYOUT, kVec>;
  u32x4_t w0, w1;

  // STREAM: past the caches (rows larger than they hold)
  template <bool STREAM>
  __device__ __forceinline__ void load(const T* row, int u, int rot, int d) {
    int a, b;
    unit_chunks<LAYOUT, kVec>(u, rot, d, &a, &b);
    w0 = STREAM ? ld_stream16(row + a) : *reinterpret_cast<const u32x4_t*>(row + a);
    w1 = STREAM ? ld_stream16(row + b) : *reinterpret_cast<const u32x4_t*>(row + b);
  }

  // x[0 .. VEC) and x[VEC .. 2 VEC): the elements of the two chunks, turned where `t` says so
  // (the others as they are, whatever their neighbour holds)
  __device__ __forceinline__ void turned(const float* cs, const float* sn, const Turns& t, float* x) const {
    widen(w0, x, T{});
    widen(w1, x + kVec, T{});
    if constexpr (LAYOUT == kRowsInterleaved) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        float a = x[kA * j], b = x[kA * j + kB];
        turn(a, b, cs[j], sn[j]);
        if (t.turns(j)) {
          x[kA * j] = a;
          x[kA * j + kB] = b;
        }
      }
    } else if (t.all) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) turn(x[kA * j], x[kA * j + kB], cs[j], sn[j]);
    }
  }

  static __device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = a;
    a = fmaf(x, c, -b * s);
    b = fmaf(b, c, x * s);
  }
};

template <typename T>
struct RowUnit<T, kRowsHalfOdd> {
  static constexpr int kVec = 1;
  using Turns = UnitTurns<kRowsHalfOdd, 1>;
  T e0, e1;

  template <bool STREAM>
  __device__ __forceinline__ void load(const T* row, int u, int rot, int d) {
    int a, b;
    unit_chunks<kRowsHalfOdd, 1>(u, rot, d, &a, &b);
    e0 = row[a];
    e1 = row[b];
  }
  __device__ __forceinline__ void turned(const float* cs, const float* sn, const Turns& t, float* x) const {
    x[0] = to_f32(e0);
    x[1] = to_f32(e1);
    if (t.all) RowUnit<T, kRowsHalf>::turn(x[0], x[1], cs[0], sn[0]);
  }
};

__device__ __forceinline__ void put_one(bf16_t* to, float x) { to->bits = f32_to_bf16_bits(x); }
__device__ __forceinline__ void put_one(float* to, float x) { *to = x; }

// The unit's elements to a row of T.  STREAM: past the caches.
template <typename T, int LAYOUT, bool STREAM>
__device__ __forceinline__ void store_unit(T* row, int u, int rot, int d, const float* x) {
  constexpr int kVec = RowVec<T, LAYOUT>::kVec;
  int a, b;
  unit_chunks<LAYOUT, kVec>(u, rot, d, &a, &b);
  if constexpr (LAYOUT == kRowsHalfOdd) {
    put_one(row + a, x[0]);
    put_one(row + b, x[1]);
  } else {
    const u32x4_t w0 = narrow(x, T{}), w1 = narrow(x + kVec, T{});
    if constexpr (STREAM) {
      __builtin_nontemporal_store(w0, reinterpret_cast<u32x4_t*>(row + a));
      __builtin_nontemporal_store(w1, reinterpret_cast<u32x4_t*>(row + b));
    } else {
      *reinterpret_cast<u32x4_t*>(row + a) = w0;
      *reinterpret_cast<u32x4_t*>(row + b) = w1;
    }
  }
}

// The rotation as the kernels take it.
struct RotaryArgs {
  const unsigned long long* w;  // [rot / 2]
  int rot;
  float factor;
  float sign;  // -1: the transposed rotation
};

// Cosines and sines, times the factor, of unit u's pairs at position t.
template <int LAYOUT, int VEC>
__device__ __forceinline__ void unit_angles(const RotaryArgs& r, int t, const UnitTurns<LAYOUT, VEC>& turns, float* cs,
                                            float* sn) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    float s = 0.f, c = 1.f;
    if (turns.turns(j)) rotary_sincos(rotary_turn(t, r.w[unit_pair<LAYOUT, VEC>(turns.unit, j, turns.d)]), &s, &c);
    cs[j] = c * r.factor;
    sn[j] = s * (r.factor * r.sign);
  }
}

int check_rotary(const ia_rotary* r, int head_dim);  // rotary.hip

// The layout whose loads fit: kRowsHalfOdd where the halves are no whole chunks.
inline int rotary_layout(const ia_rotary* r, int elem_bytes) {
  if (!r || r->dim == 0) return kRowsHalf;
  if (r->interleaved) return kRowsInterleaved;
  return r->dim % (2 * (16 / elem_bytes)) ? kRowsHalfOdd : kRowsHalf;
}

// Whether rows of this size are better written past the caches: more than the L2s hold (dirty
// lines are written back when the kernel ends: 24,001 tokens of 36 heads 93 us, past them 86),
// and no chunk that ends inside a 64-byte sector (halves of 96 bytes: 103 us, past them 143).
inline bool stream_rows(const ia_rotary* r, int layout, int64_t bytes, int elem_bytes) {
  return bytes > (32 << 20) && !(layout != kRowsInterleaved && r && r->dim / 2 * elem_bytes % 64);
}

}  // namespace ia
