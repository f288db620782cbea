// Beam search's selection for gfx950: the n best of beams x vocabulary of every batch entry.
//
//   key(j, v) = scores[j] + logits[j, v] - logsumexp(logits[j])
//
// ia_beam_scan, one launch, one pass over the logits.  A wave takes a slice of a row, groups of
// four 16-byte loads a lane, and keeps sum exp(x - M) against a reference M within 1 of its running
// maximum, and the slice's n best logits (the order inside a row is that of the keys).  What is
// below the n-th largest of the lanes' running maxima (found bit by bit with ballots, and over
// the slices of a row that a workgroup holds) cannot be among them, so a group is one comparison
// unless it holds something better; candidates wait in LDS and are cut to the n best when they
// fill up.  The workgroup that ends last of a batch entry joins the slices' sums, forms the
// candidates' keys in 64 bits (float32 keys of magnitude 10 would order equal what differs by
// 10^-6) and ranks those above a threshold, after cutting them to the n best where they are more
// than 128.  Slices are handed over through memory at the device's coherence point (ia_common.hpp).
//
// Equal keys go to the lower beam * vocabulary + token.
//
// 512 rows of 128,000 bf16 logits take 39 us (131 MB; 26 us at the rate of a copy): the vector
// units are busy for half of the time (an exp takes as long as four other instructions, as much as
// all else of an element), with two waves a SIMD to cover the branches of the candidates, and the
// merge behind the last row is 7 us of waiting.  Short calls are a chain of round trips: the scan
// 7 us (its first loads 3, the cut of the candidates 4), handing over 2.5, the merge 6: 80 rows
// of 50,021 take 15 us, 4 of 32,000 10.
#include <algorithm>

#include "rotary.hpp"

namespace ia {
namespace {

constexpr int kScanThreads = 256;
constexpr int kScanWaves = kScanThreads / 64;
constexpr int kFly = 4;              // chunks of a group, and in flight (group_sum joins four)
constexpr int kHeld = 640;           // candidates a wave holds: a chunk's 512 and some
constexpr int kTrim = 128;           // candidates at which they are cut to the n best
constexpr int kWorthFloor = 2;       // lanes with something better for which the floor is raised
constexpr int kMaxSlices = 64;       // of a row: a lane each in the merge
constexpr int kMaxBeams = 64, kMaxBest = 64;
constexpr int kOwn = 8;              // candidates a merging thread keeps in registers
constexpr int kMaxCandidates = kOwn * kScanThreads;  // of a batch entry, where a slice a row is fewer
constexpr int kNear = 1024;          // of those above the threshold, in LDS; more go through memory
constexpr int kRanked = 128;         // of those, as many as are ranked at once; more are cut first
constexpr u32 kLowest = 0x00800000u; // the key of the lowest finite float
constexpr int kWaves = 2048;         // of a call, where slices are long

// Floats as integers of the same order (-0 before +0).
__device__ __forceinline__ u32 order_key(float x) {
  const u32 b = __float_as_uint(x);
  return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(u32 k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ unsigned long long order_key64(double x) {
  const long long b = __double_as_longlong(x);
  return (unsigned long long)b ^ ((unsigned long long)(b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double order_value64(unsigned long long k) {
  return __longlong_as_double((long long)(k >> 63 ? k ^ 0x8000000000000000ull : ~k));
}

// The n-th largest of the lanes' keys (n <= 64), its lower bits cut off: the largest K of BITS
// leading bits that n keys reach.
template <int BITS>
__device__ __forceinline__ u32 nth_of_lanes(u32 key, int n) {
  u32 k = 0;
#pragma unroll
  for (int bit = 31; bit > 31 - BITS; --bit) {
    const u32 t = k | 1u << bit;
    if (__popcll(__ballot(key >= t)) >= n) k = t;
  }
  return k;
}

// The least float above the one of key k.
__device__ __forceinline__ float above(u32 k) { return order_value(k + 1); }

// A candidate: order_key of the logit (-0 as +0) above the token's complement, so that the
// better of two is the larger number.  0: none.
typedef unsigned long long Candidate;
__device__ __forceinline__ u32 key_of(Candidate c) { return (u32)(c >> 32); }
__device__ __forceinline__ u32 token_of(Candidate c) { return ~(u32)c; }
__device__ __forceinline__ Candidate candidate(float x, u32 token) { return (Candidate)order_key(x + 0.f) << 32 | ~token; }

// c of another lane (the same for all)
__device__ __forceinline__ Candidate of_lane(Candidate c, int lane) {
  return (Candidate)(u32)__builtin_amdgcn_readlane((int)(c >> 32), lane) << 32 |
         (u32)__builtin_amdgcn_readlane((int)(u32)c, lane);
}

// The n best of cnt candidates to the front of `held`; returns the least key that stays.
// n < cnt <= kHeld, one wave.
__device__ u32 trim(Candidate* held, int cnt, int n, int lane) {
  wave_lds_sync();
  Candidate edge;  // the least that stays
  Candidate a = lane < cnt ? held[lane] : 0ull, b = 64 + lane < cnt ? held[64 + lane] : 0ull;
  if (cnt <= 128) {  // ranks, by counting what is better (bit by bit as below: 4 us, 32 dependent steps)
    int ra = 0, rb = 0;
    if (cnt <= 64) {
#pragma unroll 4
      for (int o = 0; o < cnt; ++o) ra += of_lane(a, o) > a;
    } else {
#pragma unroll 4
      for (int o = 0; o < 64; ++o) {
        const Candidate x = of_lane(a, o);
        ra += x > a;
        rb += x > b;
      }
#pragma unroll 4
      for (int o = 0; o < cnt - 64; ++o) {
        const Candidate x = of_lane(b, o);
        ra += x > a;
        rb += x > b;
      }
    }
    wave_lds_sync();
    if (lane < cnt && ra < n) held[ra] = a;
    if (64 + lane < cnt && rb < n) held[rb] = b;
    wave_lds_sync();
    edge = held[n - 1];
  } else {  // (many equal ones) the n-th largest number bit by bit: key, then token
    edge = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const Candidate t = edge | 1ull << bit;
      int c = 0;
      for (int i = 0; i < cnt; i += 64) c += __popcll(__ballot(i + lane < cnt && held[min(i + lane, cnt - 1)] >= t));
      if (c >= n) edge = t;
    }
    int kept = 0;
    for (int i = 0; i < cnt; i += 64) {
      const Candidate c = held[min(i + lane, cnt - 1)];
      const bool keep = i + lane < cnt && c >= edge;
      const unsigned long long m = __ballot(keep);
      wave_lds_sync();  // (read before it is written: entries move towards the front)
      if (keep) held[kept + __popcll(m & ((1ull << lane) - 1))] = c;
      kept += __popcll(m);
      wave_lds_sync();
    }
  }
  return key_of(edge);
}

struct BeamParams {
  const char* logits;
  int64_t row_stride;  // bytes
  const float* scores;  // [batch, beams]
  const uint8_t* done;  // null: none
  int32_t beams, vocab, n, slices, slice_chunks, pad_token;
  int32_t groups;  // workgroups of a batch entry
  unsigned long long per_beam_inverse;  // of slices * n, 2^32 times, rounded up
  // per slice of a row: n candidates, the reference and the sum; per entry: workgroups that have
  // ended (0 between calls), candidates' keys and places where kNear is too few
  Candidate* best;
  unsigned long long* sum;  // (a double's bits)
  float* ref;
  u32* ended;
  unsigned long long* far;
  float* out_scores;  // [batch, n]
  int32_t* out_tokens;
  int32_t* out_rows;
};

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {  // 16 bytes at any element
  u32x4_t w;
};

// The sum of `term` over a lane's elements of a group, joined in pairs.
template <typename T, typename F>
__device__ __forceinline__ float group_sum(const u32x4_t* w, F term) {
  constexpr int kVec = RowVec<T>::kVec;
  float part[kFly];
#pragma unroll
  for (int i = 0; i < kFly; ++i) {
    float x[kVec];
    widen(w[i], x, T{});
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = term(x[j]);
#pragma unroll
    for (int m = kVec / 2; m > 0; m /= 2)
#pragma unroll
      for (int j = 0; j < m; ++j) x[j] += x[j + m];
    part[i] = x[0];
  }
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// One slice of one row: its candidates and sum, handed over.  shares[w0 .. w1): the workgroup's
// slices of the row, each with the order_key that its part of n values reach (`wave` this one).
template <typename T>
__device__ __forceinline__ void scan_slice(const BeamParams& p, Candidate* held, u32* shares, int w0, int w1, int wave,
                                           int64_t row, int slice, int64_t id, int lane) {
  constexpr int kVec = RowVec<T>::kVec, kChunk = 64 * kVec;
  const T* x0 = reinterpret_cast<const T*>(p.logits + row * p.row_stride);
  const int chunks = (p.vocab + kChunk - 1) / kChunk;
  const int c0 = slice * p.slice_chunks, c1 = min(c0 + p.slice_chunks, chunks);
  const int n = p.n;

  float ref = kNegInf;
  float lo = -3.402823466e38f;  // what is below cannot be among the n best
  float seen = kNegInf;         // the lane's maximum so far
  double sum = 0.;
  int cnt = 0;

  // a chunk past the slice or the row's end: what is there, -infinity for the rest
  auto load_some = [&](int c) {
    const int at = c * kChunk + lane * kVec;
    float y[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const float x = to_f32(x0[min(at + j, p.vocab - 1)]);  // (loaded by every lane: no branch a value)
      y[j] = c < c1 && at + j < p.vocab ? x : kNegInf;
    }
    return narrow(y, T{});
  };
  auto load = [&](int c) {
    return __builtin_nontemporal_load(&reinterpret_cast<const Loose<T>*>(x0 + (c * kChunk + lane * kVec))->w);
  };
  const int part_of_n = (n + w1 - w0 - 1) / (w1 - w0);
  // n of the row's values reach the least of the shares
  auto joint = [&]() {
    u32 k = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) {
      const u32 x = __hip_atomic_load(shares + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      if (w >= w0 && w < w1) k = min(k, x);
    }
    return k;
  };
  auto take = [&](const u32x4_t* w, int c) {
    const u32 reached = joint();
    float most[kFly], all = kNegInf;
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      float x[kVec];
      widen(w[i], x, T{});
      most[i] = kNegInf;  // (a maximum passes over NaN)
#pragma unroll
      for (int j = 0; j < kVec; ++j) most[i] = fmaxf(most[i], x[j]);
      all = fmaxf(all, most[i]);
    }
    // The reference follows the maximum to within 1: a term's argument, whose roundings are a part
    // of its size, is then no larger than the term lies under the maximum, or 1 (a reference that
    // lagged by 8 put the log of a sum off by 2^-20.5 where one token is most of it).  Most groups
    // raise nothing.  (As a difference, which a constant added to the row does not change.)
    if (__ballot(all - ref > 1.f)) {
      const float to = wave_max(all);
      if (ref != kNegInf) sum *= (double)__builtin_amdgcn_exp2f((ref - to) * kLog2e);
      ref = to;
    }
    const float base = ref == kNegInf ? 0.f : ref;
    // (a tree of additions: 32 equal small terms in a row behind a large one were off by 2^-19.4)
    float part = group_sum<T>(w, [&](float x) { return __builtin_amdgcn_exp2f((x - base) * kLog2e); });
    if (part != part)  // NaN adds nothing; +infinity leaves the sum NaN: the row offers nothing
      part = group_sum<T>(w, [&](float x) { return x == x ? __builtin_amdgcn_exp2f((x - base) * kLog2e) : 0.f; });
    sum += (double)part;
    // (equal ones stay: theirs may be the lower place)
    lo = fmaxf(lo, order_value(reached));
    const unsigned long long hits = __ballot(all >= lo);
    if (!hits) return;
    seen = fmaxf(seen, all);
    // n values of n lanes reach the floor; a single better value is not worth a new one.  The
    // row's n values are sought over all of its slices here: four waves that share them meet a
    // third of the candidates (512 rows of 128,000, n of 16: 39 us, each for itself 44; 64 x 8 of
    // 16,384: 17 and 20; slices of two groups with n of 5 lose half a microsecond)
    u32 floor_ = 0;
    if (__popcll(hits) >= kWorthFloor) {
      const u32 mine = order_key(seen + 0.f);
      if (w1 - w0 > 1) {
        const u32 share = nth_of_lanes<16>(mine, part_of_n);
        if (lane == 0) __hip_atomic_store(shares + wave, share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      if (reached == kLowest) floor_ = nth_of_lanes<16>(mine, n);  // (not every slice has a share yet)
      lo = fmaxf(lo, order_value(max(floor_, joint())));
    }
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      if (!__ballot(most[i] >= lo)) continue;
      float x[kVec];
      widen(w[i], x, T{});
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const bool in = x[j] >= lo;
        const unsigned long long m = __ballot(in);
        if (m) {
          if (in)
            held[cnt + __popcll(m & ((1ull << lane) - 1))] =
                candidate(x[j], (u32)((c + i) * kChunk + lane * kVec + j));
          cnt += __popcll(m);
        }
      }
      if (cnt >= kTrim) {
        lo = fmaxf(lo, above(trim(held, cnt, n, lane)));
        cnt = n;
      }
    }
    // n values at lower places reach the floor: from here on only what is above it counts
    if (floor_ > kLowest) lo = fmaxf(lo, above(floor_));
  };

  // whole groups, one ahead (the last is loaded twice: a load under a condition would make every
  // group wait for the one behind it), then what is left
  const int whole = max(min(c1, p.vocab / kChunk) - c0, 0) / kFly;
  u32x4_t cur[kFly], nxt[kFly];
  if (whole > 0) {
#pragma unroll
    for (int i = 0; i < kFly; ++i) cur[i] = load(c0 + i);
    for (int g = 0; g < whole; ++g) {
      const int next = c0 + min(g + 1, whole - 1) * kFly;
#pragma unroll
      for (int i = 0; i < kFly; ++i) nxt[i] = load(next + i);
      take(cur, c0 + g * kFly);
#pragma unroll
      for (int i = 0; i < kFly; ++i) cur[i] = nxt[i];
    }
  }
  if (c0 + whole * kFly < c1) {
#pragma unroll
    for (int i = 0; i < kFly; ++i) cur[i] = load_some(c0 + whole * kFly + i);
    take(cur, c0 + whole * kFly);
  }
  wave_lds_sync();
  if (cnt > n) {
    trim(held, cnt, n, lane);
    cnt = n;
  }
  if (lane < n) st_agent_u64(p.best + id * n + lane, lane < cnt ? held[lane] : 0ull);
  for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
  if (lane == 0) {
    st_agent_u64(p.sum + id, (unsigned long long)__double_as_longlong(sum));
    st_agent(p.ref + id, ref);
  }
}

struct MergeLds {
  unsigned long long keys[kNear], places[kNear];  // of those that stay
  double log_sum[kMaxBeams];
  float top[kMaxBeams], score[kMaxBeams];
  int ended[kMaxBeams];
  u32 least[2][kScanWaves];
  int stay;
  unsigned long long cut_keys[kMaxBest], cut_places[kMaxBest];  // of more than kRanked, the n best
  int digits[256];                                              // how many have each value
  int cut;
};

// The *want-th largest of the workgroup's values below 2^BITS, eight bits at a time: how many of
// those that agree so far have each next digit.  value(o, &v): whether o counts, and its value.
// *want becomes the number of those equal to the result that belong to the largest *want.
template <int BITS, typename F>
__device__ unsigned long long nth_largest(int count, int* want, int* digits, F value) {
  const int tid = threadIdx.x, lane = tid & 63;
  unsigned long long edge = 0;
  for (int shift = BITS - 8; shift >= 0; shift -= 8) {
    digits[tid] = 0;
    __syncthreads();
    for (int o = tid; o < count; o += kScanThreads) {
      unsigned long long v;
      if (value(o, &v) && ((v ^ edge) >> shift) < 256) atomicAdd(&digits[v >> shift & 255], 1);
    }
    __syncthreads();
    int n[4], mine = 0;  // a lane's four digits, the largest first
#pragma unroll
    for (int j = 0; j < 4; ++j) mine += n[j] = digits[255 - 4 * lane - j];
    const int upto = wave_inclusive_scan(mine);
    const int first = __builtin_ctzll(__ballot(upto >= *want));
    int before = __builtin_amdgcn_readlane(upto - mine, first), digit = 4 * first;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int c = __builtin_amdgcn_readlane(n[j], first);
      if (digit == 4 * first + j && before + c < *want) {
        before += c;
        ++digit;
      }
    }
    *want -= before;
    edge |= (unsigned long long)(255 - digit) << shift;
    __syncthreads();  // (every wave has read the digits)
  }
  return edge;
}

// The n best of `count` candidates (more than n, in LDS and behind kNear in memory) to cut_keys and
// cut_places, in any order.  Candidates are many where keys are equal: beams that hold the same, rows
// that a mask leaves at the type's lowest value.  Ranked each against all, 64 equal beams (n of 64, 4,096
// candidates) took 895 us a call, 12,000 where all keys were equal, and 8 flat rows of 32,000 (n of
// 16) 2,700; cut first 163, 163 and 95.
__device__ void cut_to_best(MergeLds& l, const unsigned long long* far_keys, const unsigned long long* far_places,
                            int count, int n) {
  auto key_at = [&](int o) { return o < kNear ? l.keys[o] : far_keys[o]; };
  // (a beam below 64 and a token below 2^30: 40 bits; lower places are better)
  auto lowness_at = [&](int o) { return ~(o < kNear ? l.places[o] : far_places[o]) & 0xffffffffffull; };
  int want = n;
  const unsigned long long key = nth_largest<64>(count, &want, l.digits, [&](int o, unsigned long long* v) {
    *v = key_at(o);
    return true;
  });
  const unsigned long long low = nth_largest<40>(count, &want, l.digits, [&](int o, unsigned long long* v) {
    if (key_at(o) != key) return false;
    *v = lowness_at(o);
    return true;
  });
  if (threadIdx.x == 0) l.cut = 0;
  __syncthreads();
  for (int o = threadIdx.x; o < count; o += kScanThreads) {
    const unsigned long long k = key_at(o);
    if (k > key || (k == key && lowness_at(o) >= low)) {
      const int to = atomicAdd(&l.cut, 1);
      l.cut_keys[to] = k;
      l.cut_places[to] = o < kNear ? l.places[o] : far_places[o];
    }
  }
  __syncthreads();
}

// The n best of a batch entry's candidates, by the whole workgroup.
__device__ void merge_entry(const BeamParams& p, MergeLds& l, int b) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per_beam = p.slices * p.n, total = p.beams * per_beam;
  const int64_t row0 = (int64_t)b * p.beams;
  unsigned long long* far_keys = p.far + 2 * (size_t)b * total;
  unsigned long long* far_places = far_keys + total;
  Candidate own[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i)
    own[i] = i * kScanThreads + tid < total ? ld_agent_u64(p.best + row0 * per_beam + i * kScanThreads + tid) : 0ull;
  // each beam's reference and log of its sum; +infinity where the beam has nothing to offer.
  // The slices of four beams are in flight together.
  for (int j0 = wave; j0 < p.beams; j0 += 4 * kScanWaves) {
    float r[4];
    double t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * kScanWaves;
      const int64_t at = (row0 + j) * p.slices + lane;
      const bool ended = j < p.beams && p.done && p.done[row0 + j];
      const bool there = j < p.beams && lane < p.slices && !ended;
      if (j < p.beams && lane == 0) {
        l.score[j] = p.scores[row0 + j];
        l.ended[j] = ended;
      }
      r[i] = there ? ld_agent(p.ref + at) : kNegInf;
      t[i] = there ? __longlong_as_double((long long)ld_agent_u64(p.sum + at)) : 0.;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * kScanWaves;
      if (j >= p.beams) break;
      const float m = wave_max(r[i]);
      // (a reference of -infinity: nothing was added)
      double x = r[i] == kNegInf ? 0. : t[i] * exp((double)r[i] - (double)m);
      for (int s = 32; s > 0; s >>= 1) x += __shfl_xor(x, s, 64);
      if (lane == 0) {
        l.top[j] = m;
        l.log_sum[j] = x > 0. ? log(x) : (double)__builtin_huge_valf();
      }
    }
  }
  if (tid == 0) l.stay = 0;
  __syncthreads();
  const unsigned long long none = order_key64((double)kNegInf);
  // key of candidate i (0: cannot be chosen) and its place
  auto key_place = [&](int i, Candidate c, unsigned long long* place) {
    const int j = (int)((u32)i * p.per_beam_inverse >> 32);
    double key = (double)kNegInf;
    u32 at = token_of(c);
    if (l.ended[j]) {
      at = (u32)p.pad_token;
      if (i == j * per_beam) key = (double)l.score[j];
    } else if (c != 0) {
      // (x - top is exact: rows that differ by a constant have the same keys)
      key = (double)l.score[j] + (((double)order_value(key_of(c)) - (double)l.top[j]) - l.log_sum[j]);
    }
    *place = (unsigned long long)j << 32 | at;
    const unsigned long long k = key == key ? order_key64(key + 0.) : none;
    return k <= none ? 0ull : k;
  };
  // a threshold on the keys' upper halves that n candidates reach: n of some wave, or each wave's
  // share of n
  unsigned long long own_key[kOwn], own_place[kOwn];
  u32 mine = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    own_key[i] = 0;
    if (i * kScanThreads + tid < total) own_key[i] = key_place(i * kScanThreads + tid, own[i], &own_place[i]);
    mine = max(mine, (u32)(own_key[i] >> 32));
  }
  for (int i = kMaxCandidates + tid; i < total; i += kScanThreads) {
    unsigned long long place;
    mine = max(mine, (u32)(key_place(i, ld_agent_u64(p.best + row0 * per_beam + i), &place) >> 32));
  }
  const u32 least = nth_of_lanes<24>(mine, p.n), share = nth_of_lanes<24>(mine, (p.n + kScanWaves - 1) / kScanWaves);
  if (lane == 0) {
    l.least[0][wave] = least;
    l.least[1][wave] = share;
  }
  __syncthreads();
  u32 limit = 0, shares = 0xffffffffu;
#pragma unroll
  for (int w = 0; w < kScanWaves; ++w) {
    limit = max(limit, l.least[0][w]);
    shares = min(shares, l.least[1][w]);
  }
  limit = max(limit, shares);
  auto keep = [&](unsigned long long k, unsigned long long place) {
    if (k == 0 || (u32)(k >> 32) < limit) return;
    const int at = atomicAdd(&l.stay, 1);
    if (at < kNear) {
      l.keys[at] = k;
      l.places[at] = place;
    } else {
      far_keys[at] = k;
      far_places[at] = place;
    }
  };
#pragma unroll
  for (int i = 0; i < kOwn; ++i) keep(own_key[i], own_place[i]);
  for (int i = kMaxCandidates + tid; i < total; i += kScanThreads) {
    unsigned long long place;
    const unsigned long long k = key_place(i, ld_agent_u64(p.best + row0 * per_beam + i), &place);
    keep(k, place);
  }
  __threadfence_block();
  __syncthreads();
  // ranks: better keys, and equal ones at lower places
  int count = l.stay;
  const unsigned long long *keys = l.keys, *places = l.places;
  if (count > kRanked) {
    cut_to_best(l, far_keys, far_places, count, p.n);
    keys = l.cut_keys;
    places = l.cut_places;
    count = p.n;
  }
  // a candidate a lane, the others read across the wave
  const unsigned long long k = tid < count ? keys[tid] : 0ull, at = tid < count ? places[tid] : 0ull;
  int rank = 0;
  for (int o0 = 0; o0 < count && wave * 64 < count; o0 += 64) {
    const unsigned long long ok = o0 + lane < count ? keys[o0 + lane] : 0ull;
    const unsigned long long oa = o0 + lane < count ? places[o0 + lane] : 0ull;
    const int many = min(count - o0, 64);
#pragma unroll 8
    for (int o = 0; o < many; ++o) {
      const unsigned long long x = of_lane(ok, o), y = of_lane(oa, o);
      rank += x > k || (x == k && y < at);
    }
  }
  auto put = [&](int to, double score, unsigned long long place) {
    const int64_t i = (int64_t)b * p.n + to;
    p.out_scores[i] = (float)score;
    p.out_tokens[i] = (int32_t)(u32)place;
    p.out_rows[i] = (int)(row0 + (int64_t)(place >> 32));
  };
  if (tid < count && rank < p.n) put(rank, order_value64(k), at);
  // fewer candidates than places: -infinity, the lowest ones that are none
  if (count < p.n && tid == 0) {
    int j = 0, v = 0;
    for (int r = count; r < p.n;) {
      const unsigned long long place = (unsigned long long)j << 32 | (u32)v;
      bool is = false;
      for (int o = 0; o < count; ++o) is |= places[o] == place;
      if (!is) put(r++, (double)kNegInf, place);
      if (++v == p.vocab) {
        v = 0;
        ++j;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kScanThreads) void ia_beam_scan(BeamParams p) {
  __shared__ union {
    Candidate held[kScanWaves][kHeld];
    MergeLds merge;
  } lds;
  __shared__ u32 before, shares[kScanWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x / p.groups, local = (blockIdx.x - b * p.groups) * kScanWaves + wave;
  if (threadIdx.x < kScanWaves) shares[threadIdx.x] = kLowest;
  __syncthreads();
  if (local < p.beams * p.slices) {
    const int j = local / p.slices, slice = local - j * p.slices;
    const int64_t row = (int64_t)b * p.beams + j;
    if (!p.done || !p.done[row]) {
      const int w0 = max(wave - slice, 0), w1 = min(wave - slice + p.slices, kScanWaves);
      scan_slice<T>(p, lds.held[wave], shares, w0, w1, wave, row, slice, row * p.slices + slice, lane);
    }
  }
  // the workgroup that ends last merges
  wait_memory();
  __syncthreads();
  if (threadIdx.x == 0) before = fetch_add_agent_u32(p.ended + b, 1);
  __syncthreads();
  if (before != (u32)p.groups - 1) return;
  if (threadIdx.x == 0) st_agent_u32(p.ended + b, 0);
  merge_entry(p, lds.merge, b);
}

struct BeamPlan {
  int64_t waves;
  int slices, slice_chunks, groups;
  size_t ended, best, sum, ref, far, total;  // offsets in the workspace
};

// Slices of a row: up to kWaves waves in all with two groups a slice, up to half as many with
// one, as many as fill a batch entry's workgroup, and no more candidates for a batch entry than a
// merging workgroup holds in registers.  A wave's first group and its last cut of the candidates
// cost about 4 us, so that more waves are not faster: 512 rows of 128,000 take 39 us in 2,048
// waves, 41 in 4,096, 51 in 8,192 and 50 in 1,024, where too few loads are in flight; 512 of
// 16,384 17.5 in 2,048 and 4,096, 20.7 in 8,192; 80 of 50,021 15.4 with two groups a slice and
// 16.7 with one.  4,096 entries of one beam of 32,000 take 84 us with a workgroup's four waves on
// the row, 149 with one of them.
BeamPlan beam_plan(int64_t batch, int beams, int vocab, int n, int elem_bytes) {
  BeamPlan r{};
  const int64_t rows = batch * beams;
  const int64_t chunk = 64 * (16 / elem_bytes), chunks = (vocab + chunk - 1) / chunk;
  const int64_t per_row = kWaves / std::max<int64_t>(rows, 1);
  int64_t s = std::max(std::min(per_row, chunks / (2 * kFly)), std::min(per_row / 2, (chunks + kFly - 1) / kFly));
  s = std::max({s, std::min<int64_t>((kScanWaves + beams - 1) / beams, chunks / kFly), (int64_t)1});
  s = std::min<int64_t>(s, std::max(1, std::min(kMaxSlices, kMaxCandidates / (beams * n))));
  r.slice_chunks = (int)align_up((chunks + s - 1) / s, kFly);
  r.slices = (int)((chunks + r.slice_chunks - 1) / r.slice_chunks);
  r.groups = (beams * r.slices + kScanWaves - 1) / kScanWaves;
  r.waves = rows * r.slices;
  r.ended = 0;
  r.best = align_up(r.ended + 4 * (size_t)batch, 256);
  r.sum = align_up(r.best + sizeof(Candidate) * (size_t)r.waves * n, 256);
  r.ref = align_up(r.sum + sizeof(double) * (size_t)r.waves, 256);
  r.far = align_up(r.ref + sizeof(float) * (size_t)r.waves, 256);
  r.total = align_up(r.far + 16 * (size_t)r.waves * n, 256);
  return r;
}

bool beam_sizes(int64_t batch, int beams, int vocab, int n, int dtype) {
  return batch >= 0 && batch <= (1 << 20) && batch * beams <= 1 << 24 && beams >= 1 && beams <= kMaxBeams && n >= 1 && n <= kMaxBest && vocab >= 1 &&
         vocab <= 1 << 30 && n <= (int64_t)beams * vocab && (dtype == IA_F32 || dtype == IA_BF16);
}

}  // namespace
}  // namespace ia

extern "C" {

size_t ia_beam_select_workspace_size(int32_t batch, int32_t beams, int32_t vocab, int32_t n, int32_t logits_dtype) {
  using namespace ia;
  if (!beam_sizes(batch, beams, vocab, n, logits_dtype)) return 0;
  return beam_plan(batch, beams, vocab, n, logits_dtype == IA_F32 ? 4 : 2).total;
}

int ia_beam_select(const void* logits, int32_t logits_dtype, int64_t row_stride, const float* scores,
                   const uint8_t* done, int32_t pad_token, int32_t batch, int32_t beams, int32_t vocab, int32_t n,
                   float* out_scores, int32_t* out_tokens, int32_t* out_rows, void* workspace, size_t workspace_bytes,
                   void* stream) {
  using namespace ia;
  if (logits_dtype != IA_F32 && logits_dtype != IA_BF16) return fail(IA_ERR_UNSUPPORTED, "logits must be bf16 or f32");
  if (!beam_sizes(batch, beams, vocab, n, logits_dtype))
    return fail(IA_ERR_INVALID, "beam selection takes 1 to " + std::to_string(kMaxBeams) + " beams and the best 1 to " +
                                    std::to_string(kMaxBest) + " of beams * vocab candidates");
  if (batch == 0) return IA_OK;
  if (!logits || !scores || !out_scores || !out_tokens || !out_rows) return fail(IA_ERR_INVALID, "null pointer argument");
  if (row_stride < 0) return fail(IA_ERR_INVALID, "row stride must be non-negative");
  if (pad_token < 0 || pad_token >= vocab) return fail(IA_ERR_INVALID, "pad_token must be in the vocabulary");
  const int eb = logits_dtype == IA_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % eb) return fail(IA_ERR_INVALID, "logits must be aligned to their elements");
  const BeamPlan plan = beam_plan(batch, beams, vocab, n, eb);
  if (!workspace || workspace_bytes < plan.total || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(IA_ERR_WORKSPACE, "workspace missing, too small or not 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  BeamParams p{};
  p.logits = static_cast<const char*>(logits);
  p.row_stride = row_stride * eb;
  p.scores = scores;
  p.done = done;
  p.beams = beams;
  p.vocab = vocab;
  p.n = n;
  p.slices = plan.slices;
  p.slice_chunks = plan.slice_chunks;
  p.pad_token = pad_token;
  p.groups = plan.groups;
  p.per_beam_inverse = ((1ull << 32) + plan.slices * n - 1) / (plan.slices * n);
  p.best = reinterpret_cast<Candidate*>(ws + plan.best);
  p.sum = reinterpret_cast<unsigned long long*>(ws + plan.sum);
  p.ref = reinterpret_cast<float*>(ws + plan.ref);
  p.ended = reinterpret_cast<u32*>(ws + plan.ended);
  p.far = reinterpret_cast<unsigned long long*>(ws + plan.far);
  p.out_scores = out_scores;
  p.out_tokens = out_tokens;
  p.out_rows = out_rows;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(batch * plan.groups));
  if (logits_dtype == IA_F32)
    hipLaunchKernelGGL(ia_beam_scan<float>, grid, dim3(kScanThreads), 0, st, p);
  else
    hipLaunchKernelGGL(ia_beam_scan<bf16_t>, grid, dim3(kScanThreads), 0, st, p);
  return check_launch("beam select");
}

}  // extern "C"
