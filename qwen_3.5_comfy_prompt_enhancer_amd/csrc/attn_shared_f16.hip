// Shared-prefix attention of fp16 queries (attn_shared_kernel.h).
#include "attn_shared_kernel.h"

namespace qlin {

hipError_t launch_shared_f16(const SharedArgs& a, int hd, hipStream_t st) { return launch_shared_t<F16>(a, hd, st); }

}  // namespace qlin
