// Rotary positions of packed query and key rows for gfx950.
//
//   ia_rotary_turn: a thread holds one unit (VEC pairs) of one token, its cosines and sines
//   computed once, and goes through the heads of its slice with several rows in flight.
//   Bound by HBM (every row read and written once): 24,001 tokens of 36 heads of 128 bf16 in
//   86 us (442 MB, 5.2 TB/s), halves that are no whole 64 bytes in 103 us, halves of no whole
//   chunk (a pair a lane) in 93 us.  Few tokens are cut into one slice of heads per workgroup,
//   so that a decode step is one round trip: 32 tokens of 40 heads in 4.6 us.
#include <algorithm>

#include "rotary.hpp"
#include "row_spans.hpp"

namespace ia {

int check_rotary(const ia_rotary* r, int head_dim) {
  if (!r) return fail(IA_ERR_INVALID, "rotary is null");
  if (r->dim < 0 || r->dim % 2 || r->dim > head_dim)
    return fail(IA_ERR_INVALID, "rotary dim must be even and at most head_dim");
  if (r->dim > 0 && (!r->turns || reinterpret_cast<uintptr_t>(r->turns) % 8))
    return fail(IA_ERR_INVALID, "rotary turns must be 8-byte aligned");
  if (!std::isfinite(r->factor)) return fail(IA_ERR_INVALID, "rotary factor must be finite");
  return IA_OK;
}

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotFly = 4;  // heads in flight

struct RotTensor {
  const char* in;
  char* out;
  int64_t in_tok, in_head, out_tok, out_head;  // bytes
};

struct RotParams {
  RotTensor t[2];
  int heads[2];
  const int32_t* pos;
  RotaryArgs rot;
  int n_tokens, head_dim, units, tile, heads_per_wg;
};

template <typename T, int LAYOUT, bool STREAM>
__global__ __launch_bounds__(kRotThreads) void ia_rotary_turn(RotParams p) {
  constexpr int kVec = RowVec<T, LAYOUT>::kVec;
  const int u = threadIdx.x % p.units, local = threadIdx.x / p.units;
  const int64_t tok = (int64_t)blockIdx.x * p.tile + local;
  if (local >= p.tile || tok >= p.n_tokens) return;
  float cs[kVec], sn[kVec];
  const typename RowUnit<T, LAYOUT>::Turns turns(u, p.rot.rot, p.head_dim);
  unit_angles<LAYOUT, kVec>(p.rot, p.pos[tok], turns, cs, sn);
  const int all = p.heads[0] + p.heads[1];
  const int h0 = blockIdx.y * p.heads_per_wg, h1 = min(h0 + p.heads_per_wg, all);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const RotTensor& t = p.t[which];
    const int off = which ? p.heads[0] : 0;
    const int a = max(h0 - off, 0), b = min(h1 - off, p.heads[which]);
    const char* in = t.in + tok * t.in_tok;
    char* out = t.out + tok * t.out_tok;
    for (int h = a; h < b; h += kRotFly) {
      RowUnit<T, LAYOUT> x[kRotFly];
#pragma unroll
      for (int i = 0; i < kRotFly; ++i)
        if (h + i < b) x[i].template load<STREAM>(reinterpret_cast<const T*>(in + (h + i) * t.in_head), u, p.rot.rot, p.head_dim);
#pragma unroll
      for (int i = 0; i < kRotFly; ++i)
        if (h + i < b) {
          float y[2 * kVec];
          x[i].turned(cs, sn, turns, y);
          store_unit<T, LAYOUT, STREAM>(reinterpret_cast<T*>(out + (h + i) * t.out_head), u, p.rot.rot, p.head_dim, y);
        }
    }
  }
}

template <typename T, int LAYOUT>
void launch_layout(bool stream, dim3 grid, hipStream_t st, const RotParams& p) {
  if (stream)
    hipLaunchKernelGGL((ia_rotary_turn<T, LAYOUT, true>), grid, dim3(kRotThreads), 0, st, p);
  else
    hipLaunchKernelGGL((ia_rotary_turn<T, LAYOUT, false>), grid, dim3(kRotThreads), 0, st, p);
}

template <typename T>
void launch_rotary(int layout, bool stream, dim3 grid, hipStream_t st, const RotParams& p) {
  if (layout == kRowsHalf)
    launch_layout<T, kRowsHalf>(stream, grid, st, p);
  else if (layout == kRowsInterleaved)
    launch_layout<T, kRowsInterleaved>(stream, grid, st, p);
  else
    hipLaunchKernelGGL((ia_rotary_turn<T, kRowsHalfOdd, false>), grid, dim3(kRotThreads), 0, st, p);
}

}  // namespace
}  // namespace ia

extern "C" int ia_apply_rotary(const ia_rotary* rotary, const ia_rotary_rows* rows, int32_t n_tensors, int32_t dtype,
                               int32_t head_dim, const int32_t* positions, int32_t n_tokens, int32_t inverse,
                               void* stream) {
  using namespace ia;
  if (dtype != IA_F32 && dtype != IA_BF16) return fail(IA_ERR_UNSUPPORTED, "rotary takes bf16 or f32 rows");
  if (head_dim <= 0 || head_dim % 16 || head_dim > 256)
    return fail(IA_ERR_UNSUPPORTED, "head_dim must be a multiple of 16, 256 at most");
  int rc = check_rotary(rotary, head_dim);
  if (rc) return rc;
  if (!rows || n_tensors < 1 || n_tensors > 2 || n_tokens < 0) return fail(IA_ERR_INVALID, "row tensors or tokens");
  if (n_tokens == 0) return IA_OK;
  if (!positions) return fail(IA_ERR_INVALID, "null pointer argument");
  const int eb = dtype == IA_F32 ? 4 : 2;
  RotParams p{};
  RowSpan in[2] = {{nullptr, 0, 0, 0, 0, 0}, {nullptr, 0, 0, 0, 0, 0}}, out[2] = {in[0], in[0]};
  for (int i = 0; i < n_tensors; ++i) {
    const ia_rotary_rows& x = rows[i];
    if (x.n_heads < 0) return fail(IA_ERR_INVALID, "head counts");
    if (x.n_heads == 0) continue;
    if (!x.in || !x.out) return fail(IA_ERR_INVALID, "null pointer argument");
    const int64_t strides[4] = {x.in_token_stride, x.in_head_stride, x.out_token_stride, x.out_head_stride};
    for (int64_t s : strides)
      if (s < 0 || (s * eb) % 16) return fail(IA_ERR_INVALID, "row strides must be non-negative 16-byte multiples");
    in[i] = RowSpan(x.in, n_tokens, x.n_heads, x.in_token_stride * eb, x.in_head_stride * eb, head_dim * eb);
    out[i] = RowSpan(x.out, n_tokens, x.n_heads, x.out_token_stride * eb, x.out_head_stride * eb, head_dim * eb);
    if (!out[i].rows_apart()) return fail(IA_ERR_INVALID, "output rows must not overlap");
    if ((reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out)) % 16)
      return fail(IA_ERR_INVALID, "rows must be 16-byte aligned");
    p.t[i] = RotTensor{static_cast<const char*>(x.in), static_cast<char*>(x.out), x.in_token_stride * eb,
                       x.in_head_stride * eb, x.out_token_stride * eb, x.out_head_stride * eb};
    p.heads[i] = x.n_heads;
  }
  const int64_t all = (int64_t)p.heads[0] + p.heads[1];
  if (all == 0) return IA_OK;
  if (all > INT32_MAX / 2) return fail(IA_ERR_UNSUPPORTED, "too many heads");
  p.pos = positions;
  p.rot = RotaryArgs{reinterpret_cast<const unsigned long long*>(rotary->turns), rotary->dim, rotary->factor,
                     inverse ? -1.f : 1.f};
  p.n_tokens = n_tokens;
  p.head_dim = head_dim;
  const int layout = rotary_layout(rotary, eb);
  p.units = layout == kRowsHalfOdd ? head_dim / 2 : head_dim * eb / 32;
  p.tile = kRotThreads / p.units;
  const int64_t tiles = ((int64_t)n_tokens + p.tile - 1) / p.tile;
  if (tiles >= (int64_t)1 << 23) return fail(IA_ERR_UNSUPPORTED, "too many tokens for one launch");
  // few tokens: the heads over as many workgroups as the device runs at once
  const int64_t slices = std::min<int64_t>((all + kRotFly - 1) / kRotFly,
                                           std::max<int64_t>(1, 4 * (int64_t)device_cus() / tiles));
  p.heads_per_wg = (int)((all + slices - 1) / slices);
  const int64_t ny = (all + p.heads_per_wg - 1) / p.heads_per_wg;
  if (ny > 65535) return fail(IA_ERR_UNSUPPORTED, "too many heads");
  // (a thread reads what it writes itself, and nothing else of an output)
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if ((may_meet(out[i], in[j]) && !(i == j && out[i].same(in[j]))) || (i < j && may_meet(out[i], out[j])))
        return fail(IA_ERR_INVALID, "an output must be its input itself, or overlap no input and no other output");
  const dim3 grid((unsigned)tiles, (unsigned)ny);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool stream_them = stream_rows(rotary, layout, n_tokens * all * head_dim * eb, eb);
  if (dtype == IA_F32)
    launch_rotary<float>(layout, stream_them, grid, st, p);
  else
    launch_rotary<bf16_t>(layout, stream_them, grid, st, p);
  return check_launch("rotary");
}
