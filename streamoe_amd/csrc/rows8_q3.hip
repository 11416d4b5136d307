// rows8_q3.hip — products of 8-bit rows with 3-bit weights (rows8.h).
#include "rows8.h"

namespace smoe {

hipError_t launch_qmm_i8_q3(const Q8Args& a, uint32_t group, bool x_grouped, hipStream_t st) {
  return q8_launch<3>(a, group, x_grouped, st);
}

}  // namespace smoe
