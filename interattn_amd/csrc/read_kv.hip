// Cached rows as packed tensors for gfx950: the way back from the paged pool.
//
//   ia_read_kv_rows: a workgroup per tile of one sequence's tokens; a thread's token, page and
//   16-byte chunk of the output row are fixed (so that a wave's stores are whole lines), and it
//   goes through the heads of its slice with the K and V loads of a pass in flight.  fp8 codes
//   are widened exactly, times their page's scale, rounded once.  Bound by HBM: 91k bf16 tokens
//   of 8 heads of 128 (746 MB read and written) in 129 us, 5.8 TB/s; 38k fp8 tokens (233 MB) in
//   44 us, 5.3 TB/s.  Few tokens: a head per workgroup, 5.4 us for 4 sequences of 1 to 600.
#include <algorithm>

#include "packed_rows.hpp"
#include "rotary.hpp"
#include "row_spans.hpp"

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
  int32_t chunks;  // 16-byte chunks of an output row
  int32_t tile;    // tokens of a tile
};

struct fp8_t {
  unsigned char bits;
};

// What of a pool row becomes 16 bytes of OutT.
template <typename PoolT, typename OutT>
struct ReadChunk {
  static constexpr int kElems = 16 / (int)sizeof(OutT), kBytes = kElems * (int)sizeof(PoolT), kWords = kBytes / 4;
  u32 w[kWords];

  __device__ __forceinline__ void load(const char* at) {
    if constexpr (kWords == 1) {
      w[0] = ld_stream4(at);
    } else if constexpr (kWords == 2) {
      const u32x2_t x = ld_stream8(at);
      w[0] = x[0];
      w[1] = x[1];
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const u32x4_t x = ld_stream16(at + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = x[j];
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ u32x4_t out(float s) const {
    if constexpr (sizeof(PoolT) == sizeof(OutT)) {
      return u32x4_t{w[0], w[1], w[2], w[3]};
    } else {
      float x[kElems];
      if constexpr (sizeof(PoolT) == 1) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) fp8x4_to_f32(w[i], x + 4 * i);
#pragma unroll
        for (int j = 0; j < kElems; ++j) x[j] *= s;
      } else if constexpr (sizeof(PoolT) == 2) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          x[2 * i] = bf16_lo(w[i]);
          x[2 * i + 1] = bf16_hi(w[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[i] = __uint_as_float(w[i]);
      }
      return narrow(x, OutT{});
    }
  }
};

template <bool STREAM>
__device__ __forceinline__ void put16(char* to, const u32x4_t& w) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4_t*>(to));
  else
    *reinterpret_cast<u32x4_t*>(to) = w;
}

template <typename PoolT, typename OutT, bool STREAM>
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
  const char* ks = p.k + pg * p.k_page + in * p.k_tok + chunk * C::kBytes;
  const char* vs = p.v + pg * p.v_page + in * p.v_tok + chunk * C::kBytes;
  const int64_t row = (int64_t)p.chunks * 16;
  const int64_t out = (int64_t)(t.tok0 + tok) * p.n_kv_heads * row + chunk * 16;
  for (int h = h0; h < h1; h += kReadHeads) {
    C a[kReadHeads], b[kReadHeads];
    float sa[kReadHeads], sb[kReadHeads];
#pragma unroll
    for (int i = 0; i < kReadHeads; ++i) {
      a[i].zero();
      b[i].zero();
      sa[i] = sb[i] = 1.f;
      if (held && h + i < h1) {
        a[i].load(ks + (h + i) * p.k_head);
        b[i].load(vs + (h + i) * p.v_head);
        if constexpr (kScaled) {
          sa[i] = p.k_scale[pg * p.scale_page + h + i];
          sb[i] = p.v_scale[pg * p.scale_page + h + i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kReadHeads; ++i)
      if (h + i < h1) {
        put16<STREAM>(p.k_out + out + (h + i) * row, a[i].out(sa[i]));
        put16<STREAM>(p.v_out + out + (h + i) * row, b[i].out(sb[i]));
      }
  }
}

template <typename PoolT, typename OutT>
void launch_read(bool past_caches, dim3 grid, hipStream_t st, const ReadParams& p) {
  if (past_caches)
    hipLaunchKernelGGL((ia_read_kv_rows<PoolT, OutT, true>), grid, dim3(kReadThreads), 0, st, p);
  else
    hipLaunchKernelGGL((ia_read_kv_rows<PoolT, OutT, false>), grid, dim3(kReadThreads), 0, st, p);
}

template <typename PoolT>
void launch_read_as(int out_dtype, bool past_caches, dim3 grid, hipStream_t st, const ReadParams& p) {
  if (out_dtype == IA_F32)
    launch_read<PoolT, float>(past_caches, grid, st, p);
  else
    launch_read<PoolT, bf16_t>(past_caches, grid, st, p);
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
  const int ob = out_dtype == IA_F32 ? 4 : 2;
  p.chunks = head_dim * ob / 16;
  p.tile = kReadThreads / p.chunks;
  const int64_t tiles = (int64_t)n_tokens / p.tile + n_seq;
  if (tiles >= (int64_t)1 << 23) return fail(IA_ERR_UNSUPPORTED, "too many tokens for one launch");
  p.heads_per_wg = tiles >= 2 * device_cus() ? n_kv_heads : 1;
  const int64_t ny = (n_kv_heads + p.heads_per_wg - 1) / p.heads_per_wg;
  if (ny > 65535) return fail(IA_ERR_UNSUPPORTED, "too many heads");
  const int64_t row_bytes = (int64_t)n_kv_heads * head_dim * ob;
  if (may_meet(RowSpan(k_out, n_tokens, 1, row_bytes, 0, row_bytes), RowSpan(v_out, n_tokens, 1, row_bytes, 0, row_bytes)))
    return fail(IA_ERR_INVALID, "k_out and v_out must not overlap");
  const dim3 grid((unsigned)tiles, (unsigned)ny);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // outputs larger than the L2s are written past them, as stream_rows says
  const bool past = stream_rows(nullptr, kRowsHalf, (int64_t)n_tokens * n_kv_heads * head_dim * ob, ob);
  if (kv->dtype == IA_F32)
    launch_read_as<float>(out_dtype, past, grid, st, p);
  else if (kv->dtype == IA_BF16)
    launch_read_as<bf16_t>(out_dtype, past, grid, st, p);
  else
    launch_read_as<fp8_t>(out_dtype, past, grid, st, p);
  return check_launch("read kv");
}
