// Shared-prefix attention of bf16 queries, groups of many rows (attn_shared_kernel.h).
#include "attn_shared_kernel.h"

namespace qlin {

hipError_t launch_shared_wide_bf16(const SharedArgs& a, int hd, hipStream_t st) { return launch_shared_t<Bf16, true>(a, hd, st); }

}  // namespace qlin
