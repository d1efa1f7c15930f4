// Launch of attend_few: calls whose sequences all have few rows and no group.
#include <algorithm>

#include "attend_few.h"

namespace kvx {
namespace {

template <class E, int POOL, int DP, int RT, bool FULL>
__global__ __launch_bounds__(kAttendThreads, DP <= 128 ? 2 : 1) void attend_few_kernel(
    const AttendLaunch a) {
  extern __shared__ __align__(16) char lds[];
  // With a join to come, the first workgroup leaves the plan for it.
  const int plans = a.join_grid > 0 ? 1 : 0;
  if (plans && blockIdx.x == 0) {
    WritePlan(a, reinterpret_cast<int*>(lds));
  } else {
    AttendFew<E, POOL, DP, RT, FULL>(a, lds, static_cast<int>(blockIdx.x) - plans);
  }
}

template <class E, int POOL, int DP, int RT, bool FULL>
hipError_t Launch(const AttendLaunch& l, hipStream_t stream) {
  const size_t lds = std::max(FewLds(l, DP), PlanSumWords(l) * sizeof(int));
  constexpr auto kernel = attend_few_kernel<E, POOL, DP, RT, FULL>;
  const hipError_t e = AllowDynamicLds<kernel>(lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3(l.few_grid + (l.join_grid > 0 ? 1 : 0)), dim3(kAttendThreads), lds,
                     stream, l);
  return hipGetLastError();
}

template <class E, int POOL, int DP>
hipError_t PickRows(const AttendLaunch& l, hipStream_t stream) {
  if (l.head_dim != DP) return Launch<E, POOL, DP, 2, false>(l, stream);
  return l.few_rows <= 16 ? Launch<E, POOL, DP, 1, true>(l, stream)
                          : Launch<E, POOL, DP, 2, true>(l, stream);
}

template <class E, int POOL>
hipError_t Pick(const AttendLaunch& l, hipStream_t stream) {
  switch (l.padded_dim) {
    case 64:
      return PickRows<E, POOL, 64>(l, stream);
    case 96:
      return PickRows<E, POOL, 96>(l, stream);
    case 128:
      return PickRows<E, POOL, 128>(l, stream);
    default:
      return PickRows<E, POOL, 256>(l, stream);
  }
}

template <class E>
hipError_t PickPool(const AttendLaunch& l, hipStream_t stream) {
  switch (l.pool) {
    case kPoolE4m3:
      return Pick<E, kPoolE4m3>(l, stream);
    case kPoolFp4:
      return Pick<E, kPoolFp4>(l, stream);
    default:
      return Pick<E, kPoolSame>(l, stream);
  }
}

}  // namespace

hipError_t LaunchAttendFew(const AttendLaunch& l, hipStream_t stream) {
  return l.type == kBf16 ? PickPool<Bf16>(l, stream) : PickPool<F16>(l, stream);
}

}  // namespace kvx
