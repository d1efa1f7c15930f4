// Which tokens of each sequence and key head stay within a budget.
//
// With L tokens held, L > budget: the first F = min(begin, budget) stay, the last R =
// min(recent, budget - F) stay, and of those between, the N = budget - F - R with the
// largest weights, the earlier one first where weights are equal. Positions come out
// in ascending order.
//
// A workgroup takes one sequence and key head. Weights become unsigned numbers in the
// same order (NaN, and tokens without a place, below all). The N-th largest is found by
// its digits from the top, 11, 11 and 10 bits: a histogram in LDS of the digit among
// those that agree in the digits before, then the digit in which the count from above
// reaches N. With the N-th largest T known, threads count what is above and what equals
// it in their ranges of positions, and write the positions that stay in a second pass, so
// nothing depends on the order of atomic additions. Numbers are kept in LDS between
// passes where they fit.
//
// LDS is taken for as many numbers as the tables have places, so above some 18000 of them
// a CU holds one workgroup, however short the sequences are.
//
// 64 sequences of 1000 to 16384 tokens, 8 heads, cut to 2048: 23.5 us (21 MB): the passes
// of each of the 512 workgroups, two a CU, with barriers between them (one a CU, which is
// what tables of 131072 tokens or scalar registers without a limit allow: 30 us); a cut of
// one sequence of 5000 to 1024 takes 9 us, one of 100000 tokens, whose numbers LDS does not
// hold, 166 us. Four weights a load instead of one: 41 to 39 us; ranges of
// positions for threads instead of ballots over 64 at a time: 39 to 36 us; what stays
// kept as bits of a word between counting and writing: 25.5 to 23.5 us. Equal weights
// make additions to one bin take turns: 88 us where all are equal. (Lanes that first
// agree on a bin halve that, and take a tenth longer for others.)
#include "evict.h"

#include <algorithm>

#include "attend_plan.h"

namespace kvx {
namespace {

constexpr int kWavesHere = kChooseThreads / 64;
constexpr int kBins = 2048;
constexpr int kAtOnce = 4;  // loads that a thread has on the way
// Numbers held in LDS: what its 160 KiB leave beside the histogram.
constexpr int kHeldMost = 36864;

__device__ __forceinline__ uint32_t Ordered(float x) {
  if (x != x) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 is 0
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

template <int VEC>
__global__ __launch_bounds__(kChooseThreads, 8) void choose_kept_kernel(const ChooseLaunch a,
                                                                     const int held_most) {
  extern __shared__ uint32_t held[];  // [held_most]
  __shared__ int bins[kBins];
  __shared__ int wave_sums[kWavesHere], wave_more[kWavesHere];
  __shared__ int found_bin, found_above, found_count;
  const BatchView& b = a.batch;
  const int s = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int length = min(max(b.lengths[s], 0), b.capacity);
  int* kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  if (h == 0 && threadIdx.x == 0 && a.new_lengths != nullptr) {
    a.new_lengths[s] = min(length, a.budget);
  }
  if (length <= a.budget) {
    for (int i = threadIdx.x; i < a.budget; i += kChooseThreads) kept[i] = i < length ? i : -1;
    return;
  }
  const int begin = a.begins != nullptr ? max(a.begins[s], 0) : 0;
  const int first = min(begin, a.budget), recent = min(a.recent, a.budget - first);
  const int wanted = a.budget - first - recent;
  for (int i = threadIdx.x; i < first; i += kChooseThreads) kept[i] = i;
  for (int i = threadIdx.x; i < recent; i += kChooseThreads) {
    kept[a.budget - recent + i] = length - recent + i;
  }
  if (wanted == 0) return;
  const int count = length - recent - first;  // above `wanted`
  const int32_t* table = b.tables + s * b.table_stride;
  // The range in whole groups of VEC tokens, which a block holds.
  const int base = first / VEC * VEC;
  const int span = (first + count - base + VEC - 1) / VEC * VEC;
  const bool holds = span <= held_most;
  // Numbers of neighbouring tokens, VEC from place i0 of the range on and again every VEC
  // kChooseThreads (0 behind the last): all of their blocks, then all of their weights on
  // the way at once.
  const auto load = [&](int i0, uint32_t (&u)[kAtOnce][VEC]) {
    int id[kAtOnce], slot[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const int p = base + min(i0 + n * (VEC * kChooseThreads), span - VEC);
      const int at = FastDivI(a.block_div, p);
      id[n] = table[at];
      slot[n] = p - at * b.block_tokens;
    }
    using Weights = __attribute__((ext_vector_type(VEC))) float;
    Weights w[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const bool has = id[n] >= 0 && id[n] < b.num_blocks;
      w[n] = *reinterpret_cast<const Weights*>(
          a.weights + (static_cast<int64_t>(has ? id[n] : 0) * a.heads + h) * b.block_tokens +
          slot[n]);
      if (!has) id[n] = -1;
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) u[n][j] = id[n] >= 0 ? Ordered(w[n][j]) : 0u;
    }
  };
  const auto number = [&](int i) {
    if (holds) return held[first - base + i];
    const int p = first + i, at = FastDivI(a.block_div, p), id = table[at];
    if (id < 0 || id >= b.num_blocks) return 0u;
    return Ordered(a.weights[(static_cast<int64_t>(id) * a.heads + h) * b.block_tokens +
                             (p - at * b.block_tokens)]);
  };

  // Digits of the number that is the wanted-th largest.
  uint32_t digits = 0;
  int above = 0;  // numbers that are larger in the digits so far
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    for (int i = threadIdx.x; i < kBins; i += kChooseThreads) bins[i] = 0;
    __syncthreads();
    const auto note = [&](uint32_t u) {
      if (pass > 0 && ((u ^ digits) >> (pass == 1 ? 21 : 10)) != 0) return;
      atomicAdd(&bins[u >> shift & mask], 1);
    };
    if (pass > 0 && holds) {
      for (int i = threadIdx.x; i < count; i += kChooseThreads) note(held[first - base + i]);
    } else {
      for (int i0 = threadIdx.x * VEC; i0 < span; i0 += kAtOnce * VEC * kChooseThreads) {
        uint32_t u[kAtOnce][VEC];
        load(i0, u);
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          const int i = i0 + n * (VEC * kChooseThreads);
          if (i >= span) break;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (holds) held[i + j] = u[n][j];
            if (VEC == 1 || (i + j >= first - base && i + j < first - base + count)) note(u[n][j]);
          }
        }
      }
    }
    __syncthreads();
    // Counts from the top: thread t has bins from the top 2t and 2t + 1.
    const int top = kBins - 1 - 2 * static_cast<int>(threadIdx.x);
    const int n0 = bins[top], n1 = bins[top - 1];
    int sum = n0 + n1;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const int o = __shfl_up(sum, m);
      if (lane >= m) sum += o;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int before = above + sum - n0 - n1;
#pragma unroll
    for (int w = 0; w < kWavesHere; ++w) before += w < wave ? wave_sums[w] : 0;
    if (before < wanted && before + n0 >= wanted) {
      found_bin = top;
      found_above = before;
      found_count = n0;
    } else if (before + n0 < wanted && before + n0 + n1 >= wanted) {
      found_bin = top - 1;
      found_above = before + n0;
      found_count = n1;
    }
    __syncthreads();
    digits |= static_cast<uint32_t>(found_bin) << shift;
    above = found_above;
    // All with these digits stay (mostly one, after 22 bits): what is above the number
    // before the least of them does.
    if (above + found_count == wanted && digits != 0) {
      --digits;
      above = wanted;
      break;
    }
  }

  // A thread's range of positions (of an odd length, so that a wave reads LDS on all
  // banks): what is above and what equals the number.
  const int each = (count + kChooseThreads - 1) / kChooseThreads | 1;
  const int i0 = min(static_cast<int>(threadIdx.x) * each, count), i1 = min(i0 + each, count);
  int more = 0, equal = 0;
  // Bit i: place i0 + i, of ranges that have no more than 32.
  const bool masks = holds && each <= 32;
  uint32_t at_least = 0, same = 0;
  if (masks) {
    for (int i = i0; i < i1; ++i) {
      const uint32_t u = held[first - base + i], bit = 1u << (i - i0);
      at_least |= u >= digits ? bit : 0u;
      same |= u == digits ? bit : 0u;
    }
    equal = __popc(same);
    more = __popc(at_least) - equal;
  } else {
    for (int i = i0; i < i1; ++i) {
      const uint32_t u = number(i);
      more += u > digits ? 1 : 0;
      equal += u == digits ? 1 : 0;
    }
  }
  int more_to = more, equal_to = equal;  // with the lanes before
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const int x = __shfl_up(more_to, m), y = __shfl_up(equal_to, m);
    if (lane >= m) {
      more_to += x;
      equal_to += y;
    }
  }
  if (lane == 63) {
    wave_more[wave] = more_to;
    wave_sums[wave] = equal_to;
  }
  __syncthreads();
  more = more_to - more;
  equal = equal_to - equal;
#pragma unroll
  for (int w = 0; w < kWavesHere; ++w) {
    more += w < wave ? wave_more[w] : 0;
    equal += w < wave ? wave_sums[w] : 0;
  }
  const int of_equal = wanted - above;  // so many of those that equal it stay
  if (masks) {
    for (; at_least != 0; at_least &= at_least - 1) {
      const int i = __builtin_ctz(at_least);
      const bool is_equal = (same >> i & 1) != 0;
      if (!is_equal || equal < of_equal) {
        kept[first + more + min(equal, of_equal)] = first + i0 + i;
      }
      equal += is_equal ? 1 : 0;
      more += is_equal ? 0 : 1;
    }
    return;
  }
  for (int i = i0; i < i1; ++i) {
    const uint32_t u = number(i);
    if (u > digits) {
      kept[first + more + min(equal, of_equal)] = first + i;
      ++more;
    } else if (u == digits) {
      if (equal < of_equal) kept[first + more + equal] = first + i;
      ++equal;
    }
  }
}

}  // namespace

hipError_t LaunchChooseKept(const ChooseLaunch& l, hipStream_t stream) {
  // Four weights at a time where blocks hold whole fours.
  const bool fours = l.batch.block_tokens % 4 == 0 && reinterpret_cast<uintptr_t>(l.weights) % 16 == 0;
  const int held = std::min((l.batch.capacity + 3) / 4 * 4, kHeldMost);
  const size_t lds = static_cast<size_t>(held) * sizeof(uint32_t);
  constexpr auto by_four = choose_kept_kernel<4>, by_one = choose_kept_kernel<1>;
  // (The limit counts the kernel's own arrays too.)
  const size_t all = lds + kBins * sizeof(int) + 1024;
  const hipError_t e = fours ? AllowDynamicLds<by_four>(all) : AllowDynamicLds<by_one>(all);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fours ? by_four : by_one, dim3(l.batch.sequences * l.heads),
                     dim3(kChooseThreads), lds, stream, l, held);
  return hipGetLastError();
}

}  // namespace kvx
