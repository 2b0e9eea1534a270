// Shared-prefix attention of bf16 queries (attn_shared_kernel.h).
#include "attn_shared_kernel.h"

namespace qlin {

hipError_t launch_shared_bf16(const SharedArgs& a, int hd, hipStream_t st) {
  return a.tiles == 8 ? launch_shared_wide_bf16(a, hd, st) : launch_shared_t<Bf16, false>(a, hd, st);
}

}  // namespace qlin
