// Launch of attend_mixed: 4-bit pools.
#include "attend_mixed.h"

namespace kvx {

hipError_t LaunchAttendMixedFp4(const AttendLaunch& l, hipStream_t stream) {
  return LaunchAttendMixedOf<kPoolFp4>(l, stream);
}

}  // namespace kvx
