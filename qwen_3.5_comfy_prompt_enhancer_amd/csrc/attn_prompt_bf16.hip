// Prompt attention, bf16 queries, and the choice of type.
#include "attn_prompt_kernel.h"

namespace qlin {

hipError_t launch_prompt_bf16(const PromptArgs& a, int hd, hipStream_t st) {
  return prompt_dispatch<Bf16>(a, hd, st);
}

hipError_t launch_prompt(const PromptArgs& a, int dt, int hd, hipStream_t st) {
  return dt == DT_BF16 ? launch_prompt_bf16(a, hd, st) : launch_prompt_f16(a, hd, st);
}

}  // namespace qlin
