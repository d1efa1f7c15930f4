// Launch of attend_mixed: e4m3 pools.
#include "attend_mixed.h"

namespace kvx {

hipError_t LaunchAttendMixedE4m3(const AttendLaunch& l, hipStream_t stream) {
  return LaunchAttendMixedOf<kPoolE4m3>(l, stream);
}

}  // namespace kvx
