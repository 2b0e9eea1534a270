// Prompt attention, fp16 queries.
#include "attn_prompt_kernel.h"

namespace qlin {

hipError_t launch_prompt_f16(const PromptArgs& a, int hd, hipStream_t st) {
  return prompt_dispatch<F16>(a, hd, st);
}

}  // namespace qlin
