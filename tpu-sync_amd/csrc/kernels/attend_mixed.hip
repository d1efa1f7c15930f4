// Launch of attend_mixed: calls with chunks of queries or with groups. Its
// workgroups take the parts of many rows and those of few in turn, a round of
// every CU at a time, so that the matrix products of the ones and the reading of
// the others share the CUs.
#include <algorithm>

#include "attend_few.h"
#include "attend_many.h"

namespace kvx {
namespace {

constexpr int kRound = 256;  // CUs

// A kind's workgroups, in whole rounds.
__host__ __device__ inline int Rounded(int grid) { return (grid + kRound - 1) / kRound * kRound; }

template <class E, bool E4, int DP, int RT, bool FULL>
__global__ __launch_bounds__(kAttendThreads, DP <= 128 ? 2 : 1) void attend_mixed_kernel(
    const AttendLaunch a) {
  extern __shared__ __align__(16) char lds[];
  const int plans = a.join_grid > 0 ? 1 : 0;
  if (plans && blockIdx.x == 0) {
    WritePlan(a, reinterpret_cast<int*>(lds));
    return;
  }
  // Workgroups go to XCDs in turn, and on an XCD to its CUs in turn: a round of
  // kRound of one kind puts one on every CU.
  const int block = static_cast<int>(blockIdx.x) - plans;
  const int few = Rounded(a.few_grid), many = Rounded(a.many_grid);
  const int round = block / kRound, both = min(few, many) / kRound;
  const bool is_many = round < 2 * both ? round % 2 == 0 : many > few;
  const int mine = (round < 2 * both ? round / 2 : round - both) * kRound + block % kRound;
  if (is_many) {
    AttendMany<E, E4, DP>(a, lds, mine);
  } else {
    if (mine < a.few_grid) AttendFew<E, E4, DP, RT, FULL>(a, lds, mine);
  }
}

template <class E, bool E4, int DP, int RT, bool FULL>
hipError_t Launch(const AttendLaunch& l, hipStream_t stream) {
  const size_t lds =
      std::max({FewLds(l, DP), ManyLds(l, DP), PlanSumWords(l) * sizeof(int)});
  constexpr auto kernel = attend_mixed_kernel<E, E4, DP, RT, FULL>;
  const hipError_t e = AllowDynamicLds<kernel>(lds);
  if (e != hipSuccess) return e;
  const int grid = Rounded(l.few_grid) + Rounded(l.many_grid);
  hipLaunchKernelGGL(kernel, dim3(grid + (l.join_grid > 0 ? 1 : 0)), dim3(kAttendThreads), lds,
                     stream, l);
  return hipGetLastError();
}

template <class E, bool E4, int DP>
hipError_t PickRows(const AttendLaunch& l, hipStream_t stream) {
  if (l.head_dim != DP) return Launch<E, E4, DP, 2, false>(l, stream);
  return l.few_rows <= 16 ? Launch<E, E4, DP, 1, true>(l, stream)
                          : Launch<E, E4, DP, 2, true>(l, stream);
}

template <class E, bool E4>
hipError_t Pick(const AttendLaunch& l, hipStream_t stream) {
  switch (l.padded_dim) {
    case 64:
      return PickRows<E, E4, 64>(l, stream);
    case 96:
      return PickRows<E, E4, 96>(l, stream);
    case 128:
      return PickRows<E, E4, 128>(l, stream);
    default:
      return PickRows<E, E4, 256>(l, stream);
  }
}

}  // namespace

hipError_t LaunchAttendMixed(const AttendLaunch& l, hipStream_t stream) {
  if (l.type == kBf16) return l.e4m3 ? Pick<Bf16, true>(l, stream) : Pick<Bf16, false>(l, stream);
  return l.e4m3 ? Pick<F16, true>(l, stream) : Pick<F16, false>(l, stream);
}

}  // namespace kvx
