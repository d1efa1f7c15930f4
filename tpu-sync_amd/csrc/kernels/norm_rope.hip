// RMS norm and position rotation of query and key heads in one pass.
//
// Each head row x of a token at position p becomes
//   y = x * w / sqrt(mean(x^2) + eps)            (y = x without a weight)
//   (u, v) -> (u cos a - v sin a, v cos a + u sin a),  a_i = p * inv_freq[i]
// over the pairs (y_i, y_{i + R/2}) or (y_{2i}, y_{2i+1}) of its first R
// dimensions; the rest keep y. Everything between the load and the store is
// fp32 (the angle is reduced in 64 bits), so a value is rounded once.
//
// A workgroup takes a few tokens: it puts their R/2 (cos, sin) into LDS once
// for all heads (one sincos a token and pair instead of one a head), then its
// waves walk the tokens' rows, 16-byte chunks across the lanes.
#include <hip/hip_runtime.h>

#include "head_row.h"
#include "norm_rope.h"

namespace kvx {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;  // of one workgroup

__device__ __forceinline__ int64_t Position(const NormRopeLaunch& a, int64_t t) {
  return a.positions_64 ? static_cast<const int64_t*>(a.positions)[t]
                        : static_cast<const int32_t*>(a.positions)[t];
}

template <class E, int VEC, int LPR>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const NormRopeLaunch a,
                                                             const int tokens_each) {
  extern __shared__ f32x2 cs[];  // [tokens_each][rotary_dim / 2]
  using Scalar = typename E::Scalar;
  constexpr int kRows = kThreads / LPR;
  const int pairs = a.rotary_dim / 2;
  const int t0 = blockIdx.x * tokens_each;
  const int nt = min(tokens_each, a.tokens - t0);
  const int heads = a.q.heads + a.k.heads;
  // The heads of a token are shared out over gridDim.y workgroups.
  const int step = kRows * gridDim.y;
  int h = blockIdx.y * kRows + threadIdx.x / LPR, t = 0;
  while (h >= heads) {
    h -= heads;
    ++t;
  }
  const RowLane<E, VEC, LPR> lane(a.head_dim, a.rotary_dim, a.interleaved);
  Row<E, VEC, LPR> row;
  const auto load = [&]() {
    const bool is_q = h < a.q.heads;
    const int64_t token = t0 + t;
    const int64_t at = is_q ? token * a.q.in_token + h * a.q.in_head
                            : token * a.k.in_token + (h - a.q.heads) * a.k.in_head;
    row.Load(lane, static_cast<const Scalar*>(is_q ? a.q.in : a.k.in) + at);
  };
  if (t < nt) load();  // in flight while the angles are computed
  float wq[lane.kChunks][VEC], wqo[lane.kChunks][VEC], wk[lane.kChunks][VEC],
      wko[lane.kChunks][VEC];
  LoadWeights(lane, a.q.weight, a.weight_f32, wq, wqo);
  LoadWeights(lane, a.k.weight, a.weight_f32, wk, wko);
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int ti = i / pairs;
    cs[i] = Turn(Position(a, t0 + ti), a.inv_freq[i - ti * pairs]);
  }
  __syncthreads();
  while (t < nt) {
    const bool is_q = h < a.q.heads;
    if ((is_q ? a.q.weight : a.k.weight) != nullptr) {
      if (is_q) {
        row.Norm(lane, wq, wqo, a.eps);
      } else {
        row.Norm(lane, wk, wko, a.eps);
      }
    }
    row.Rotate(lane, cs + t * pairs);
    const int64_t token = t0 + t;
    if (is_q) {
      row.Store(lane, static_cast<Scalar*>(a.q.out) + token * a.q.out_token + h * a.q.out_head);
    } else {
      row.Store(lane, static_cast<Scalar*>(a.k.out) + token * a.k.out_token +
                          (h - a.q.heads) * a.k.out_head);
    }
    h += step;
    while (h >= heads) {
      h -= heads;
      ++t;
    }
    if (t < nt) load();
  }
}

template <class E, int VEC, int LPR>
hipError_t Launch(const NormRopeLaunch& l, hipStream_t stream) {
  constexpr int kRows = kThreads / LPR;
  const int heads = l.q.heads + l.k.heads;
  // About 64 rows a workgroup, so the angles are shared out over many; with
  // few tokens one each, and their heads spread over workgroups too.
  int each = 1, split = 1;
  if (l.tokens > 1024) {
    while (each < kMaxTokens && each * heads < 64) each *= 2;
  } else {
    const int groups = (heads + kRows - 1) / kRows;
    while (split < groups && l.tokens * split < 512) ++split;
  }
  const dim3 grid((l.tokens + each - 1) / each, split);
  const size_t lds = static_cast<size_t>(each) * (l.rotary_dim / 2) * sizeof(f32x2);
  hipLaunchKernelGGL((norm_rope_kernel<E, VEC, LPR>), grid, dim3(kThreads), lds, stream, l, each);
  return hipGetLastError();
}

bool Aligned(const HeadRows& r, int vec) {
  if (r.heads == 0) return true;
  const uint64_t at = reinterpret_cast<uint64_t>(r.in) | reinterpret_cast<uint64_t>(r.out);
  return at % 16 == 0 &&
         (r.in_token | r.in_head | r.out_token | r.out_head) % vec == 0;
}

template <class E, int VEC>
hipError_t Pick(const NormRopeLaunch& l, hipStream_t stream) {
  if (Aligned(l.q, VEC) && Aligned(l.k, VEC) &&
      ChunksFit(VEC, l.head_dim, l.rotary_dim, l.interleaved)) {
    const int chunks = l.head_dim / VEC;
    if (chunks <= 8) return Launch<E, VEC, 8>(l, stream);
    if (chunks <= 16) return Launch<E, VEC, 16>(l, stream);
    if (VEC == 8 || chunks <= 32) return Launch<E, VEC, 32>(l, stream);
    return Launch<E, VEC, VEC == 8 ? 32 : 64>(l, stream);
  }
  return Launch<E, 1, 64>(l, stream);
}

}  // namespace

hipError_t LaunchNormRope(const NormRopeLaunch& l, hipStream_t stream) {
  switch (l.type) {
    case kBf16:
      return Pick<Bf16, 8>(l, stream);
    case kF16:
      return Pick<F16, 8>(l, stream);
    default:
      return Pick<F32, 4>(l, stream);
  }
}

}  // namespace kvx
