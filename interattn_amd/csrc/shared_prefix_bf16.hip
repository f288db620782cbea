// Shared-prefix decode over bf16 K/V (compiled apart so that the instances build in parallel).
#include "shared_prefix.hpp"

namespace ia {

int launch_prefix_bf16(const PrefixParams& p, int d, hipStream_t st) {
  return d == 128 ? launch_prefix<kArBf16, 128>(p, st) : launch_prefix<kArBf16, 64>(p, st);
}

}  // namespace ia
