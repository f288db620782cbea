// Shared-prefix decode over f32 K/V (compiled apart so that the instances build in parallel).
#include "shared_prefix.hpp"

namespace ia {

int launch_prefix_f32(const PrefixParams& p, int d, hipStream_t st) {
  return d == 128 ? launch_prefix<kArF32, 128>(p, st) : launch_prefix<kArF32, 64>(p, st);
}

}  // namespace ia
