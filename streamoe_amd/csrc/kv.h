// kv.h — where a position of a sequence lies in a paged cache.
#pragma once

#include "common.h"
#include "kernels.h"

namespace smoe {

// Page of the table that holds sixteen n of a sequence's positions.
__device__ __forceinline__ uint32_t kv_page_of(const KvView& c, uint32_t sixteen) {
  return (uint32_t)(((uint64_t)sixteen * c.div_mul) >> c.div_shift);
}

// Whether token t is a position of a sequence; padding is none, and no error.
__device__ __forceinline__ bool kv_token(const KvTokens& k, int32_t seq, int32_t pos, bool* wrong) {
  const bool in = (uint32_t)seq < k.n_seqs && (uint32_t)pos < k.positions;
  *wrong = !in && seq != -1;
  return in;
}

}  // namespace smoe
