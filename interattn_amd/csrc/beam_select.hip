// Beam search's selection for gfx950: the n best of beams x vocabulary of every batch entry.
//
//   key(j, v) = scores[j] + logits[j, v] - logsumexp(logits[j])
//
//   ia_beam_scan: one pass over the logits.  A wave takes a slice of a row, 16 bytes a lane,
//     and keeps sum exp(x - M) against a reference M near its running maximum, and the slice's
//     n best logits (the order inside a row is that of the keys).  A threshold T, below which
//     nothing can be among them any more, makes the common chunk one comparison: the first
//     chunk's T is the n-th largest of its lanes' maxima (found bit by bit with ballots), later
//     ones follow the candidates held.  Candidates wait in LDS and are cut to the n best when
//     they fill up.
//   ia_beam_merge: a workgroup per batch entry joins the slices' sums, forms the candidates'
//     keys in 64 bits (float32 keys of magnitude 10 would order equal what differs by 10^-6)
//     and ranks those above a threshold.
//
// Equal keys go to the lower beam * vocabulary + token.  Bound by reading the logits once.
#include <algorithm>

#include "rotary.hpp"

namespace ia {
namespace {

constexpr int kScanThreads = 256;
constexpr int kScanWaves = kScanThreads / 64;
constexpr int kFly = 4;              // chunks in flight
constexpr int kHeld = 640;           // candidates a wave holds: a chunk's 512 and some
constexpr int kTrim = 128;           // candidates at which they are cut to the n best
constexpr int kMaxBeams = 64, kMaxBest = 64;
constexpr int kMergeThreads = 256;
constexpr int kMaxCandidates = 8192;  // of a batch entry
constexpr int kNear = 1024;           // of those above the threshold, in LDS; more go through memory
constexpr int kTargetWaves = 4096;

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

// The n-th largest of the lanes' keys (n <= 64): the largest K that n keys reach.
__device__ __forceinline__ u32 nth_of_lanes(u32 key, int n) {
  u32 k = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const u32 t = k | 1u << bit;
    if (__popcll(__ballot(key >= t)) >= n) k = t;
  }
  return k;
}

struct Candidate {
  u32 key;  // order_key of the logit, -0 as +0
  u32 at;   // token
};

// The n best of cnt candidates (key descending, token ascending) to the front of `held`, in
// any order; returns their least key.  cnt > n, one wave.
__device__ u32 trim(Candidate* held, int cnt, int n, int lane) {
  auto reach = [&](auto&& test) {
    int c = 0;
    for (int i = 0; i < cnt; i += 64) c += __popcll(__ballot(i + lane < cnt && test(held[min(i + lane, cnt - 1)])));
    return c;
  };
  u32 least = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const u32 t = least | 1u << bit;
    if (reach([&](const Candidate& c) { return c.key >= t; }) >= n) least = t;
  }
  u32 last = 0xffffffffu;  // of those that have the least key, tokens up to `last` stay
  const int above = reach([&](const Candidate& c) { return c.key > least; });
  if (reach([&](const Candidate& c) { return c.key == least; }) > n - above) {
    u32 below = 0;  // the largest bound below which fewer than n - above tokens lie
    for (int bit = 31; bit >= 0; --bit) {
      const u32 t = below | 1u << bit;
      if (reach([&](const Candidate& c) { return c.key == least && c.at < t; }) < n - above) below = t;
    }
    last = below;
  }
  int kept = 0;
  for (int i = 0; i < cnt; i += 64) {
    const Candidate c = held[min(i + lane, cnt - 1)];
    const bool keep = i + lane < cnt && (c.key > least || (c.key == least && c.at <= last));
    const unsigned long long m = __ballot(keep);
    wave_lds_sync();  // (read before it is written: entries move towards the front)
    if (keep) held[kept + __popcll(m & ((1ull << lane) - 1))] = c;
    kept += __popcll(m);
    wave_lds_sync();
  }
  return least;
}

struct ScanParams {
  const char* logits;
  int64_t row_stride;  // bytes
  const uint8_t* done;  // null: none
  int32_t vocab, n, slices, slice_chunks;
  int64_t waves;  // rows * slices
  // per slice: n candidates, the reference and the sum
  Candidate* best;
  double* sum;
  float* ref;
};

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {  // 16 bytes at any element
  u32x4_t w;
};

template <typename T>
__global__ __launch_bounds__(kScanThreads) void ia_beam_scan(ScanParams p) {
  constexpr int kVec = RowVec<T, kRowsPlain>::kVec, kChunk = 64 * kVec;
  __shared__ Candidate all[kScanWaves][kHeld];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * kScanWaves + wave;
  if (id >= p.waves) return;
  const int64_t row = id / p.slices;
  const int slice = (int)(id - row * p.slices);
  if (p.done && p.done[row]) return;
  Candidate* held = all[wave];
  const T* x0 = reinterpret_cast<const T*>(p.logits + row * p.row_stride);
  const int chunks = (p.vocab + kChunk - 1) / kChunk;
  const int c0 = slice * p.slice_chunks, c1 = min(c0 + p.slice_chunks, chunks);
  const int n = p.n;

  float ref = kNegInf, limit = kNegInf;  // candidates are above `limit` (or any finite, to begin with)
  double sum = 0.;
  int cnt = 0;

  auto load = [&](int c) {
    const int at = c * kChunk + lane * kVec;
    u32x4_t w;
    if (c < c1 && at + kVec <= p.vocab) {
      w = __builtin_nontemporal_load(&reinterpret_cast<const Loose<T>*>(x0 + at)->w);
    } else {
      float y[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[j] = c < c1 && at + j < p.vocab ? to_f32(x0[at + j]) : kNegInf;
      w = narrow(y, T{});
    }
    return w;
  };
  auto take = [&](const u32x4_t& w, int c) {
    float x[kVec];
    widen(w, x, T{});
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = fmaxf(x[j], kNegInf);  // NaN: never chosen, adds nothing
    float most = x[0];
#pragma unroll
    for (int j = 1; j < kVec; ++j) most = fmaxf(most, x[j]);
    // (the reference is the maximum of a chunk that is well above the one before: exp stays
    // below e^8 and few chunks pay for a new one)
    if (__ballot(most > ref + 8.f)) {
      const float to = wave_max(most);
      if (ref != kNegInf) sum *= (double)__builtin_amdgcn_exp2f((ref - to) * kLog2e);
      ref = to;
    }
    const float base = ref == kNegInf ? 0.f : ref;
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < kVec; ++j) part += __builtin_amdgcn_exp2f((x[j] - base) * kLog2e);
    sum += (double)part;
    const unsigned long long hits = __ballot(most > limit);
    if (!hits) return;
    float floor_ = kNegInf;  // what the chunk itself rules out
    if (__popcll(hits) >= n) floor_ = order_value(nth_of_lanes(order_key(most + 0.f), n));
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const bool in = x[j] > limit && x[j] >= floor_;
      const unsigned long long m = __ballot(in);
      if (m) {
        if (in)
          held[cnt + __popcll(m & ((1ull << lane) - 1))] =
              Candidate{order_key(x[j] + 0.f), (u32)(c * kChunk + lane * kVec + j)};
        cnt += __popcll(m);
      }
    }
    limit = fmaxf(limit, floor_);
    wave_lds_sync();
    if (cnt >= kTrim) {
      limit = fmaxf(limit, order_value(trim(held, cnt, n, lane)));
      cnt = n;
    }
  };

  u32x4_t cur[kFly], nxt[kFly];
#pragma unroll
  for (int i = 0; i < kFly; ++i) cur[i] = load(c0 + i);
  for (int c = c0; c < c1; c += kFly) {
#pragma unroll
    for (int i = 0; i < kFly; ++i) nxt[i] = load(c + kFly + i);
#pragma unroll
    for (int i = 0; i < kFly; ++i)
      if (c + i < c1) take(cur[i], c + i);
#pragma unroll
    for (int i = 0; i < kFly; ++i) cur[i] = nxt[i];
  }
  if (cnt > n) {
    trim(held, cnt, n, lane);
    cnt = n;
  }
  wave_lds_sync();
  for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
  if (lane < n) p.best[id * n + lane] = lane < cnt ? held[lane] : Candidate{0u, 0xffffffffu};
  if (lane == 0) {
    p.sum[id] = sum;
    p.ref[id] = ref;
  }
}

struct MergeParams {
  const float* scores;  // [batch, beams]
  const uint8_t* done;
  const Candidate* best;
  const double* sum;
  const float* ref;
  unsigned long long* far;  // per batch entry: candidates' keys, then places, where kNear is too few
  int32_t beams, vocab, n, slices, pad_token;
  float* out_scores;  // [batch, n]
  int32_t* out_tokens;
  int32_t* out_rows;
};

__global__ __launch_bounds__(kMergeThreads) void ia_beam_merge(MergeParams p) {
  __shared__ unsigned long long near_keys[kNear], near_places[kNear];  // of those that stay
  __shared__ double log_sum[kMaxBeams];
  __shared__ float top[kMaxBeams];
  __shared__ u32 wave_least[kMergeThreads / 64];
  __shared__ int stay;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int total = p.beams * p.slices * p.n;
  unsigned long long* far_keys = p.far + 2 * (size_t)b * total;
  unsigned long long* far_places = far_keys + total;
  // each beam's reference and log of its sum; +infinity where the beam has nothing to offer
  for (int j = wave; j < p.beams; j += kMergeThreads / 64) {
    const int64_t row = (int64_t)b * p.beams + j;
    float m = kNegInf;
    const bool ended = p.done && p.done[row];
    if (!ended)
      for (int s = lane; s < p.slices; s += 64) m = fmaxf(m, p.ref[row * p.slices + s]);
    m = wave_max(m);
    double l = 0.;
    if (!ended && m != kNegInf)
      for (int s = lane; s < p.slices; s += 64) {
        const float r = p.ref[row * p.slices + s];
        if (r != kNegInf) l += p.sum[row * p.slices + s] * exp((double)r - (double)m);
      }
    for (int s = 32; s > 0; s >>= 1) l += __shfl_xor(l, s, 64);
    if (lane == 0) {
      top[j] = m;
      log_sum[j] = l > 0. ? log(l) : (double)__builtin_huge_valf();
    }
  }
  if (tid == 0) stay = 0;
  __syncthreads();
  const unsigned long long none = order_key64((double)kNegInf);
  auto candidate = [&](int i, unsigned long long* place) {
    const int j = i / (p.slices * p.n);
    const int64_t row = (int64_t)b * p.beams + j;
    double key = (double)kNegInf;
    u32 at = 0;
    if (p.done && p.done[row]) {
      if (i == j * p.slices * p.n) {
        key = (double)p.scores[row];
        at = (u32)p.pad_token;
      }
    } else {
      const Candidate c = p.best[row * p.slices * p.n + (i - j * p.slices * p.n)];
      // (x - top is exact: rows that differ by a constant have the same keys)
      if (c.at != 0xffffffffu)
        key = (double)p.scores[row] + (((double)order_value(c.key) - (double)top[j]) - log_sum[j]);
      at = c.at;
    }
    *place = (unsigned long long)j * (u32)p.vocab + at;
    const unsigned long long k = key == key ? order_key64(key + 0.) : none;
    return k <= none ? 0ull : k;  // (nothing is below -infinity: 0 marks what cannot be chosen)
  };
  // a threshold on the keys' upper halves that n candidates of some wave reach
  u32 mine = 0;
  for (int i = tid; i < total; i += kMergeThreads) {
    unsigned long long place;
    mine = max(mine, (u32)(candidate(i, &place) >> 32));
  }
  const u32 least = nth_of_lanes(mine, p.n);
  if (lane == 0) wave_least[wave] = least;
  __syncthreads();
  u32 limit = 0;
#pragma unroll
  for (int w = 0; w < kMergeThreads / 64; ++w) limit = max(limit, wave_least[w]);
  for (int i = tid; i < total; i += kMergeThreads) {
    unsigned long long place;
    const unsigned long long k = candidate(i, &place);
    if (k == 0 || (u32)(k >> 32) < limit) continue;
    const int at = atomicAdd(&stay, 1);
    if (at < kNear) {
      near_keys[at] = k;
      near_places[at] = place;
    }
    far_keys[at] = k;
    far_places[at] = place;
  }
  __threadfence();
  __syncthreads();
  // ranks: better keys, and equal ones at lower places
  const int count = stay;
  auto rank_all = [&](const unsigned long long* keys, const unsigned long long* places) {
    for (int i = tid; i < count; i += kMergeThreads) {
      const unsigned long long k = keys[i], at = places[i];
      int rank = 0;
      for (int o = 0; o < count; ++o) rank += keys[o] > k || (keys[o] == k && places[o] < at);
      if (rank >= p.n) continue;
      const int64_t to = (int64_t)b * p.n + rank;
      const int j = (int)(at / (u32)p.vocab);
      p.out_scores[to] = (float)order_value64(k);
      p.out_tokens[to] = (int32_t)(at - (unsigned long long)j * (u32)p.vocab);
      p.out_rows[to] = b * p.beams + j;
    }
  };
  if (count <= kNear)
    rank_all(near_keys, near_places);
  else
    rank_all(far_keys, far_places);
  // fewer candidates than places: -infinity, the lowest ones that are none
  if (count < p.n && tid == 0) {
    unsigned long long at = 0;
    for (int r = count; r < p.n; ++at) {
      bool is = false;
      for (int o = 0; o < count; ++o) is |= near_places[o] == at;
      if (is) continue;
      const int64_t to = (int64_t)b * p.n + r++;
      const int j = (int)(at / (u32)p.vocab);
      p.out_scores[to] = kNegInf;
      p.out_tokens[to] = (int32_t)(at - (unsigned long long)j * (u32)p.vocab);
      p.out_rows[to] = b * p.beams + j;
    }
  }
}

struct BeamPlan {
  int64_t rows, waves;
  int slices, slice_chunks;
  size_t best, sum, ref, far, total;  // offsets in the workspace
};

// Slices of a row: about kTargetWaves waves in all, two chunks each at least, and no more
// candidates for a batch entry than the merge holds.
BeamPlan beam_plan(int64_t batch, int beams, int vocab, int n, int elem_bytes) {
  BeamPlan r{};
  r.rows = batch * beams;
  const int64_t chunk = 64 * (16 / elem_bytes), chunks = (vocab + chunk - 1) / chunk;
  int64_t s = std::max<int64_t>(1, kTargetWaves / std::max<int64_t>(r.rows, 1));
  s = std::min<int64_t>(s, std::max<int64_t>(1, chunks / 2));
  s = std::min<int64_t>(s, std::max(1, kMaxCandidates / (beams * n)));
  r.slice_chunks = (int)((chunks + s - 1) / s);
  r.slices = (int)((chunks + r.slice_chunks - 1) / r.slice_chunks);
  r.waves = r.rows * r.slices;
  r.best = 0;
  r.sum = align_up(r.best + sizeof(Candidate) * (size_t)r.waves * n, 256);
  r.ref = align_up(r.sum + sizeof(double) * (size_t)r.waves, 256);
  r.far = align_up(r.ref + sizeof(float) * (size_t)r.waves, 256);
  r.total = align_up(r.far + 16 * (size_t)r.waves * n, 256);
  return r;
}

bool beam_sizes(int64_t batch, int beams, int vocab, int n, int dtype) {
  return batch >= 0 && batch <= (1 << 22) && beams >= 1 && beams <= kMaxBeams && n >= 1 && n <= kMaxBest && vocab >= 1 &&
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
  ScanParams s{};
  s.logits = static_cast<const char*>(logits);
  s.row_stride = row_stride * eb;
  s.done = done;
  s.vocab = vocab;
  s.n = n;
  s.slices = plan.slices;
  s.slice_chunks = plan.slice_chunks;
  s.waves = plan.waves;
  s.best = reinterpret_cast<Candidate*>(ws + plan.best);
  s.sum = reinterpret_cast<double*>(ws + plan.sum);
  s.ref = reinterpret_cast<float*>(ws + plan.ref);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((plan.waves + kScanWaves - 1) / kScanWaves));
  if (logits_dtype == IA_F32)
    hipLaunchKernelGGL(ia_beam_scan<float>, grid, dim3(kScanThreads), 0, st, s);
  else
    hipLaunchKernelGGL(ia_beam_scan<bf16_t>, grid, dim3(kScanThreads), 0, st, s);
  const int rc = check_launch("beam scan");
  if (rc) return rc;
  const MergeParams m{scores, done,        s.best,    s.sum,      s.ref,      reinterpret_cast<unsigned long long*>(ws + plan.far),
                      beams,  vocab,       n,         plan.slices, pad_token, out_scores,
                      out_tokens, out_rows};
  hipLaunchKernelGGL(ia_beam_merge, dim3(batch), dim3(kMergeThreads), 0, st, m);
  return check_launch("beam merge");
}

}  // extern "C"
