// Prompt attention over f32 K/V (compiled apart so that the instances build in parallel).
#include "prompt_attention.hpp"

namespace ia {

int launch_prompt_f32(const PromptParams& p, int d, hipStream_t st) {
  return d == 128 ? launch_prompt<kArF32, 128>(p, st) : launch_prompt<kArF32, 64>(p, st);
}

}  // namespace ia
