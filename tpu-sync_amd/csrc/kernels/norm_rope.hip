// RMS norm and position rotation of query and key heads in one pass.
//
// Each head row x of a token at position p becomes
//   y = x * w / sqrt(mean(x^2) + eps)            (y = x without a weight)
//   (u, v) -> (u cos a - v sin a, v cos a + u sin a),  a_i = p * inv_freq[i]
// over the pairs (y_i, y_{i + R/2}) or (y_{2i}, y_{2i+1}) of its first R
// dimensions; the rest keep y. Everything between the load and the store is
// fp32 (the angle is reduced in 64 bits), so a value is rounded once.
//
// A workgroup takes a few tokens and puts their R/2 (cos, sin) into LDS, one
// sincos a token and pair for all heads. Then teams of lanes (head_row.h) take a
// token's heads in turn. Reading and writing the rows bounds it: 8192 tokens x 40
// heads x 128 in bf16, 39.3 us from cold caches (4.3 TB/s both ways), 31.1 us again
// and again on rows that the last-level cache holds in part; 64 tokens 4.9 us, the
// launch and a chain of dependent loads.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "head_row.h"
#include "norm_rope.h"

namespace kvx {
namespace {

constexpr int kThreads = kRowThreads;
// A workgroup takes one token until there are kEnough workgroups, then more, up
// to kMaxTokens. 2048 and 8192 tokens x 40 heads x 128: 12.6 and 31.1 us; with
// 256 as enough 17.8 and 58.9 us, with 4096 the same as here.
constexpr int kMaxTokens = kMostRowTokens;
constexpr int kEnough = 1024;

__device__ __forceinline__ int64_t Position(const NormRopeLaunch& a, int64_t t) {
  return a.positions_64 ? static_cast<const int64_t*>(a.positions)[t]
                        : static_cast<const int32_t*>(a.positions)[t];
}

template <class E, int VEC, int LPR>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const NormRopeLaunch a,
                                                             const int tokens_each,
                                                             const int teams_of_token) {
  extern __shared__ f32x2 cs[];  // [tokens_each][rotary_dim / 2]
  using Scalar = typename E::Scalar;
  const int pairs = a.rotary_dim / 2;
  const int t0 = blockIdx.x * tokens_each;
  const int nt = min(tokens_each, a.tokens - t0);
  const RowLane<E, VEC, LPR> lane(a.head_dim, a.rotary_dim, a.interleaved);
  // The team's first token and head; heads are shared out over the token's
  // teams of gridDim.y workgroups.
  const int team = threadIdx.x / LPR;
  const int first = blockIdx.y * teams_of_token + team % teams_of_token;
  const int step = teams_of_token * gridDim.y;
  const int token_step = kThreads / LPR / teams_of_token;
  RawRow<E, VEC, LPR> raw;
  const auto load = [&](const HeadRows& rows, int t, int h) {
    if (h >= rows.heads) return;
    raw.Load(lane, static_cast<const Scalar*>(rows.in) + (t0 + t) * rows.in_token + h * rows.in_head,
             true);
  };
  int t = team / teams_of_token;
  if (t < nt) load(a.q, t, first);  // in flight while the angles are computed
  Weights<E, VEC, LPR> q_weights, k_weights;
  q_weights.Load(lane, a.q.weight, a.weight_f32);
  k_weights.Load(lane, a.k.weight, a.weight_f32);
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int ti = i / pairs;
    cs[i] = Turn(Position(a, t0 + ti), a.inv_freq[i - ti * pairs]);
  }
  __syncthreads();
  const auto heads_of = [&](const HeadRows& rows, const Weights<E, VEC, LPR>& weights) {
    const Factors<E, VEC, LPR> f(lane, cs + t * pairs, weights);
    Scalar* out = static_cast<Scalar*>(rows.out) + (t0 + t) * rows.out_token;
    for (int h = first; h < rows.heads;) {
      const Row<E, VEC, LPR> row(lane, raw, f, rows.weight != nullptr, a.eps);
      row.Store(lane, out + h * rows.out_head);
      h += step;
      load(rows, t, h);
    }
  };
  for (; t < nt; t += token_step) {
    heads_of(a.q, q_weights);
    load(a.k, t, first);
    heads_of(a.k, k_weights);
    if (t + token_step < nt) load(a.q, t + token_step, first);
  }
}

template <class E, int VEC, int LPR>
hipError_t Launch(const NormRopeLaunch& l, hipStream_t stream) {
  const int heads = std::max(l.q.heads, l.k.heads);
  const int of_token = TeamsOfToken(heads, LPR);
  // Some tokens for every team or teams of one, so the angles' latency is paid
  // once; with few tokens one, and their heads spread over workgroups too.
  int each = kThreads / LPR / of_token, split = 1;
  while (each < kMaxTokens && l.tokens / each >= 2 * kEnough) each *= 2;
  while (split * of_token < heads && static_cast<int64_t>(l.tokens) * split < 2048) ++split;
  const dim3 grid((l.tokens + each - 1) / each, split);
  const size_t lds = static_cast<size_t>(each) * (l.rotary_dim / 2) * sizeof(f32x2);
  hipLaunchKernelGGL((norm_rope_kernel<E, VEC, LPR>), grid, dim3(kThreads), lds, stream, l, each,
                     of_token);
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
