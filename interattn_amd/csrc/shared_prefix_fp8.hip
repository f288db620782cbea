// Shared-prefix decode over fp8 K/V (compiled apart so that the instances build in parallel).
#include "shared_prefix.hpp"

namespace ia {

int launch_prefix_fp8(const PrefixParams& p, int d, hipStream_t st) {
  return d == 128 ? launch_prefix<kArFp8, 128>(p, st) : launch_prefix<kArFp8, 64>(p, st);
}

}  // namespace ia
