// attn_bf16.hip — the attention kernels of caches in bf16.
#include "attn.h"

namespace smoe {
hipError_t launch_attn_bf16(const AttnArgs& a, bool q_bf16, hipStream_t st) { return launch_attn<false>(a, q_bf16, st); }
}  // namespace smoe
