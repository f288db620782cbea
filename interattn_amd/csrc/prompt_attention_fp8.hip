// Prompt attention over fp8 K/V (compiled apart so that the instances build in parallel).
#include "prompt_attention.hpp"

namespace ia {

int launch_prompt_fp8(const PromptParams& p, int d, hipStream_t st) {
  return d == 128 ? launch_prompt<kArFp8, 128>(p, st) : launch_prompt<kArFp8, 64>(p, st);
}

}  // namespace ia
