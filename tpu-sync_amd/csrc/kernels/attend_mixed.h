// attend_mixed: calls with chunks of queries or with groups. Its
// workgroups take the parts of many rows and those of few in turn, a round of
// every CU at a time, so that the matrix products of the ones and the reading of
// the others share the CUs.
#ifndef KVX_KERNELS_ATTEND_MIXED_H_
#define KVX_KERNELS_ATTEND_MIXED_H_

#include <algorithm>

#include "attend_few.h"
#include "attend_many.h"

namespace kvx {
namespace {

constexpr int kRound = 256;  // CUs

// A kind's workgroups, in whole rounds.
__host__ __device__ inline int Rounded(int grid) { return (grid + kRound - 1) / kRound * kRound; }

template <class E, int POOL, int DP, int RT, bool FULL>
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
    AttendMany<E, POOL, DP>(a, lds, mine);
  } else {
    if (mine < a.few_grid) AttendFew<E, POOL, DP, RT, FULL>(a, lds, mine);
  }
}

template <class E, int POOL, int DP, int RT, bool FULL>
hipError_t Launch(const AttendLaunch& l, hipStream_t stream) {
  const size_t lds =
      std::max({FewLds(l, DP), ManyLds(l, DP), PlanSumWords(l) * sizeof(int)});
  constexpr auto kernel = attend_mixed_kernel<E, POOL, DP, RT, FULL>;
  const hipError_t e = AllowDynamicLds<kernel>(lds);
  if (e != hipSuccess) return e;
  const int grid = Rounded(l.few_grid) + Rounded(l.many_grid);
  hipLaunchKernelGGL(kernel, dim3(grid + (l.join_grid > 0 ? 1 : 0)), dim3(kAttendThreads), lds,
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

}  // namespace

template <int POOL>
hipError_t LaunchAttendMixedOf(const AttendLaunch& l, hipStream_t stream) {
  return l.type == kBf16 ? Pick<Bf16, POOL>(l, stream) : Pick<F16, POOL>(l, stream);
}

}  // namespace kvx

#endif  // KVX_KERNELS_ATTEND_MIXED_H_
