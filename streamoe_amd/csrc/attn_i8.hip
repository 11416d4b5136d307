// attn_i8.hip — the attention kernels of caches in 8 bits.
#include "attn.h"

namespace smoe {
hipError_t launch_attn_i8(const AttnArgs& a, bool q_bf16, hipStream_t st) { return launch_attn<true>(a, q_bf16, st); }
}  // namespace smoe
