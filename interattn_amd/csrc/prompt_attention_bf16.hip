// Prompt attention over bf16 K/V (compiled apart so that the instances build in parallel).
#include "prompt_attention.hpp"

namespace ia {

int launch_prompt_bf16(const PromptParams& p, int d, hipStream_t st) {
  return d == 128 ? launch_prompt<kArBf16, 128>(p, st) : launch_prompt<kArBf16, 64>(p, st);
}

}  // namespace ia
