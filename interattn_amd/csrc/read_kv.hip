// Cached rows as packed tensors for gfx950: the way back from the paged pool.
//
//   ia_read_kv_rows: a workgroup per tile of one sequence's tokens; a thread's token, page and
//   16-byte chunk are fixed, and it goes through the heads of its slice with the K and V loads
//   of a pass in flight.  fp8 codes are widened exactly, times their page's scale, rounded
//   once.  Bound by HBM.
#include <algorithm>

#include "packed_rows.hpp"
#include "rotary.hpp"

namespace ia {

int check_kv(const ia_paged_kv* kv, int d);

namespace {

constexpr int kReadThreads = 256;
constexpr int kReadHeads = 4;  // heads whose loads are in flight together

struct ReadParams {
  const char* k;
  const char* v;
  int64_t k_page, k_head, k_tok, v_page, v_head, v_tok;  // bytes
  const float* k_scale;
  const float* v_scale;
  int64_t scale_page;
  const int32_t* table;
  int64_t bt_stride, bt_cols, n_pages;
  int32_t page_rows;
  char* k_out;  // [n_tokens, n_kv_heads, D], contiguous
  char* v_out;
  const int32_t* starts;
  const int32_t* cu;
  int32_t n_seq, n_tokens, n_kv_heads, heads_per_wg;
  int32_t chunks;  // 16-byte chunks of a pool row
  int32_t tile;    // tokens of a tile
};

// One chunk of a pool row as OutT's elements.
template <typename PoolT, typename OutT>
struct ReadChunk;

template <typename T>
struct ReadChunk<T, T> {
  static constexpr int kElems = RowVec<T>::kVec;
  static __device__ __forceinline__ void put(T* to, const u32x4_t& w, float) { *reinterpret_cast<u32x4_t*>(to) = w; }
};
template <>
struct ReadChunk<bf16_t, float> {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ void put(float* to, const u32x4_t& w, float) {
    float x[8];
    widen(w, x, bf16_t{});
    reinterpret_cast<u32x4_t*>(to)[0] = narrow(x, float{});
    reinterpret_cast<u32x4_t*>(to)[1] = narrow(x + 4, float{});
  }
};
template <>
struct ReadChunk<float, bf16_t> {
  static constexpr int kElems = 4;
  static __device__ __forceinline__ void put(bf16_t* to, const u32x4_t& w, float) {
    float x[4];
    widen(w, x, float{});
    *reinterpret_cast<u32x2_t*>(to) = u32x2_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  }
};
struct fp8_t {
  unsigned char bits;
};
template <typename OutT>
struct ReadChunk<fp8_t, OutT> {
  static constexpr int kElems = 16;
  static __device__ __forceinline__ void put(OutT* to, const u32x4_t& w, float s) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) fp8x4_to_f32(w[i], x + 4 * i);
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] *= s;
    constexpr int kVec = RowVec<OutT>::kVec;
#pragma unroll
    for (int j = 0; j < 16; j += kVec) *reinterpret_cast<u32x4_t*>(to + j) = narrow(x + j, OutT{});
  }
};

template <typename PoolT, typename OutT>
__global__ __launch_bounds__(kReadThreads) void ia_read_kv_rows(ReadParams p) {
  using C = ReadChunk<PoolT, OutT>;
  constexpr bool kScaled = sizeof(PoolT) == 1;
  const int tid = threadIdx.x;
  const PackedTile t = packed_tile(p.cu, p.n_seq, p.n_tokens, p.tile, blockIdx.x, tid & 63);
  const int tok = tid / p.chunks, chunk = tid % p.chunks;
  if (t.local < 0 || tok >= t.n_tok) return;
  const int64_t pos = (int64_t)p.starts[t.b] + t.local * (int64_t)p.tile + tok;
  int64_t pg = -1, in = 0;
  if (pos >= 0) {
    const int64_t lp = pos / p.page_rows;
    in = pos - lp * p.page_rows;
    pg = lp;
    if (p.table) pg = lp < p.bt_cols ? p.table[(int64_t)t.b * p.bt_stride + lp] : -1;
    if (pg >= p.n_pages) pg = -1;
  }
  const bool held = pg >= 0;
  if (!held) pg = 0;
  const int h0 = blockIdx.y * p.heads_per_wg, h1 = min(h0 + p.heads_per_wg, p.n_kv_heads);
  const char* ks = p.k + pg * p.k_page + in * p.k_tok + chunk * 16;
  const char* vs = p.v + pg * p.v_page + in * p.v_tok + chunk * 16;
  const int64_t row = (int64_t)p.chunks * C::kElems;
  const int64_t out = ((int64_t)(t.tok0 + tok) * p.n_kv_heads) * row + chunk * C::kElems;
  OutT* kd = reinterpret_cast<OutT*>(p.k_out) + out;
  OutT* vd = reinterpret_cast<OutT*>(p.v_out) + out;
  for (int h = h0; h < h1; h += kReadHeads) {
    u32x4_t a[kReadHeads], b[kReadHeads];
    float sa[kReadHeads], sb[kReadHeads];
#pragma unroll
    for (int i = 0; i < kReadHeads; ++i) {
      a[i] = b[i] = u32x4_t{0u, 0u, 0u, 0u};
      sa[i] = sb[i] = 1.f;
      if (held && h + i < h1) {
        a[i] = ld_stream16(ks + (h + i) * p.k_head);
        b[i] = ld_stream16(vs + (h + i) * p.v_head);
        if constexpr (kScaled) {
          sa[i] = p.k_scale[pg * p.scale_page + h + i];
          sb[i] = p.v_scale[pg * p.scale_page + h + i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kReadHeads; ++i)
      if (h + i < h1) {
        C::put(kd + (h + i) * row, a[i], sa[i]);
        C::put(vd + (h + i) * row, b[i], sb[i]);
      }
  }
}

template <typename PoolT>
void launch_read(int out_dtype, dim3 grid, hipStream_t st, const ReadParams& p) {
  if (out_dtype == IA_F32)
    hipLaunchKernelGGL((ia_read_kv_rows<PoolT, float>), grid, dim3(kReadThreads), 0, st, p);
  else
    hipLaunchKernelGGL((ia_read_kv_rows<PoolT, bf16_t>), grid, dim3(kReadThreads), 0, st, p);
}

}  // namespace
}  // namespace ia

extern "C" int ia_read_kv(const ia_paged_kv* kv, void* k_out, void* v_out, int32_t out_dtype, const int32_t* starts,
                          const int32_t* cu_seqlens, int32_t n_seq, int32_t n_tokens, int32_t n_kv_heads,
                          int32_t head_dim, void* stream) {
  using namespace ia;
  if (head_dim != 64 && head_dim != 128) return fail(IA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  int rc = check_kv(kv, head_dim);
  if (rc) return rc;
  if (out_dtype != IA_F32 && out_dtype != IA_BF16) return fail(IA_ERR_INVALID, "out dtype must be IA_F32 or IA_BF16");
  if (n_seq < 0 || n_tokens < 0 || n_kv_heads <= 0) return fail(IA_ERR_INVALID, "sequence, token or head counts");
  if (n_seq == 0 || n_tokens == 0) return IA_OK;
  if (!k_out || !v_out || !starts || !cu_seqlens) return fail(IA_ERR_INVALID, "null pointer argument");
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16)
    return fail(IA_ERR_INVALID, "outputs must be 16-byte aligned");
  const int eb = kv->dtype == IA_F32 ? 4 : kv->dtype == IA_BF16 ? 2 : 1;
  ReadParams p{};
  p.k = static_cast<const char*>(kv->k);
  p.v = static_cast<const char*>(kv->v);
  p.k_page = kv->k_page_stride * eb;
  p.k_head = kv->k_head_stride * eb;
  p.k_tok = kv->k_token_stride * eb;
  p.v_page = kv->v_page_stride * eb;
  p.v_head = kv->v_head_stride * eb;
  p.v_tok = kv->v_token_stride * eb;
  p.k_scale = kv->k_scale;
  p.v_scale = kv->v_scale;
  p.scale_page = kv->scale_page_stride;
  p.table = kv->block_table;
  p.bt_stride = kv->bt_stride;
  p.bt_cols = kv->bt_cols;
  p.n_pages = kv->n_pages;
  p.page_rows = kv->page_size;
  p.k_out = static_cast<char*>(k_out);
  p.v_out = static_cast<char*>(v_out);
  p.starts = starts;
  p.cu = cu_seqlens;
  p.n_seq = n_seq;
  p.n_tokens = n_tokens;
  p.n_kv_heads = n_kv_heads;
  p.chunks = head_dim * eb / 16;
  p.tile = kReadThreads / p.chunks;
  const int64_t tiles = (int64_t)n_tokens / p.tile + n_seq;
  if (tiles >= (int64_t)1 << 23) return fail(IA_ERR_UNSUPPORTED, "too many tokens for one launch");
  p.heads_per_wg = tiles >= 2 * device_cus() ? n_kv_heads : 1;
  const int64_t ny = (n_kv_heads + p.heads_per_wg - 1) / p.heads_per_wg;
  if (ny > 65535) return fail(IA_ERR_UNSUPPORTED, "too many heads");
  const dim3 grid((unsigned)tiles, (unsigned)ny);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (kv->dtype == IA_F32)
    launch_read<float>(out_dtype, grid, st, p);
  else if (kv->dtype == IA_BF16)
    launch_read<bf16_t>(out_dtype, grid, st, p);
  else
    launch_read<fp8_t>(out_dtype, grid, st, p);
  return check_launch("read kv");
}
