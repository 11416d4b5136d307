// rows8_q4.hip — products of 8-bit rows with 4-bit weights (rows8.h).
#include "rows8.h"

namespace smoe {

hipError_t launch_qmm_i8_q4(const Q8Args& a, uint32_t group, bool x_grouped, hipStream_t st) {
  return q8_launch<4>(a, group, x_grouped, st);
}

}  // namespace smoe
