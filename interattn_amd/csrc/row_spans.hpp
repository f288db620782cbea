// Rows [tokens, heads, len] in memory, on the host: whether two sets share a byte, so that a
// call whose workgroups write one while others read or write the other can be refused.
#pragma once

#include <stdint.h>

#include <numeric>
#include <utility>

namespace ia {

struct RowSpan {
  uintptr_t base;
  int64_t tokens, heads;             // 0 of either: no row
  int64_t tok_stride, head_stride;  // bytes, not negative
  int64_t len;                       // bytes of a row

  RowSpan(const void* at, int64_t n_tokens, int64_t n_heads, int64_t tok, int64_t head, int64_t bytes)
      : base(reinterpret_cast<uintptr_t>(at)),
        tokens(n_tokens),
        heads(n_heads),
        tok_stride(n_tokens > 1 ? tok : 0),  // (of one token or head a stride means nothing)
        head_stride(n_heads > 1 ? head : 0),
        len(bytes) {}

  bool empty() const { return tokens == 0 || heads == 0; }
  int64_t token_bytes() const { return (heads - 1) * head_stride + len; }  // from a token's first byte to its last
  int64_t head_bytes() const { return (tokens - 1) * tok_stride + len; }
  int64_t bytes() const { return (tokens - 1) * tok_stride + token_bytes(); }

  // no row shares a byte with another: the wider stride steps over all of the narrower one's rows
  bool rows_apart() const {
    if (empty()) return true;
    if (tok_stride >= head_stride)
      return (heads == 1 || head_stride >= len) && (tokens == 1 || tok_stride >= token_bytes());
    return (tokens == 1 || tok_stride >= len) && (heads == 1 || head_stride >= head_bytes());
  }

  bool same(const RowSpan& o) const {
    return base == o.base && tokens == o.tokens && heads == o.heads && tok_stride == o.tok_stride &&
           head_stride == o.head_stride && len == o.len;
  }
};

// Whether every piece of `ea` bytes at a multiple of `period` from a's base is apart from every
// piece of `eb` bytes at one from b's.
inline bool apart_modulo(const RowSpan& a, const RowSpan& b, int64_t period, int64_t ea, int64_t eb) {
  if (period <= 0) return false;
  const int64_t d = (int64_t)(b.base - a.base) % period, off = d < 0 ? d + period : d;
  return off >= ea && off + eb <= period;
}

// Whether a and b may share a byte.  They do not where one ends before the other begins, or
// where their strides have a common period inside which the rows (or all of a token's, or all of
// a head's) are apart: views of one buffer, however it is laid out.  What no such view is may
// be said to meet though it does not.
inline bool may_meet(const RowSpan& a, const RowSpan& b) {
  if (a.empty() || b.empty()) return false;
  if (a.base + a.bytes() <= b.base || b.base + b.bytes() <= a.base) return false;
  const int64_t tok = std::gcd(a.tok_stride, b.tok_stride), head = std::gcd(a.head_stride, b.head_stride);
  return !(apart_modulo(a, b, std::gcd(tok, head), a.len, b.len) ||
           apart_modulo(a, b, tok, a.token_bytes(), b.token_bytes()) ||
           apart_modulo(a, b, head, a.head_bytes(), b.head_bytes()));
}

// The same of two vectors of int32.
inline bool ints_meet(const int32_t* a, int64_t n, const int32_t* b, int64_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return n > 0 && m > 0 && x < y + 4 * (uintptr_t)m && y < x + 4 * (uintptr_t)n;
}

}  // namespace ia
