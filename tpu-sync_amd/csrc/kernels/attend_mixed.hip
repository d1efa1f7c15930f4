// Launch of attend_mixed: pools of the tensors' type, and the choice of the others,
// which are compiled by themselves.
#include "attend_mixed.h"

namespace kvx {

hipError_t LaunchAttendMixed(const AttendLaunch& l, hipStream_t stream) {
  switch (l.pool) {
    case kPoolE4m3:
      return LaunchAttendMixedE4m3(l, stream);
    case kPoolFp4:
      return LaunchAttendMixedFp4(l, stream);
    default:
      return LaunchAttendMixedOf<kPoolSame>(l, stream);
  }
}

}  // namespace kvx
