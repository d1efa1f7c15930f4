// How attention's work is cut up: device arithmetic that every attention
// kernel repeats over the call's lengths.
#ifndef KVX_KERNELS_ATTEND_PLAN_H_
#define KVX_KERNELS_ATTEND_PLAN_H_

#include <hip/hip_runtime.h>

#include "attend.h"

namespace kvx {

constexpr int kAttendThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int FastDivI(const FastDivU32& f, int n) {
  const uint32_t u = static_cast<uint32_t>(n);
  return static_cast<int>((__umulhi(u, f.m) + u) >> f.s);
}

// In-place inclusive sums of c[0..n) over the workgroup (n <= kMaxSequences *
// 2); c[i] must have been written by any thread before, and is visible to all
// after.
__device__ __forceinline__ void BlockSums(int* c, int n) {
  __shared__ int waves[kAttendThreads / 64];
  const int each = (n + kAttendThreads - 1) / kAttendThreads;
  const int i0 = threadIdx.x * each, i1 = min(i0 + each, n);
  __syncthreads();
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine += c[i];
  int sum = mine;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const int o = __shfl_up(sum, m);
    if (lane >= m) sum += o;
  }
  if (lane == 63) waves[wave] = sum;
  __syncthreads();
  int at = sum - mine;
  for (int w = 0; w < wave; ++w) at += waves[w];
  for (int i = i0; i < i1; ++i) {
    at += c[i];
    c[i] = at;
  }
  __syncthreads();
}

// First i of [0, n) with c[i] > x (c: inclusive sums).
__device__ __forceinline__ int FirstAbove(const int* c, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (c[mid] > x) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

// The group that sequence s belongs to, or -1.
__device__ __forceinline__ int GroupOf(const AttendLaunch& a, int s) {
  int lo = 0, hi = a.groups;  // first g with group_starts[g + 1] > s
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.group_starts[mid + 1] > s) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo < a.groups && a.group_starts[lo] <= s ? lo : -1;
}

__device__ __forceinline__ int PrefixLength(const AttendLaunch& a, int g) {
  return min(max(a.prefix_lengths[g], 0), a.batch.capacity);
}

// A sequence's rows and the keys that it reads by itself: [begin, end).
struct OwnKeys {
  SequenceSpan q;
  int rows;   // a key head
  int begin;  // the tokens before are read with its group's
  int end;
  bool grouped;
};

__device__ __forceinline__ OwnKeys LoadOwnKeys(const AttendLaunch& a, int s) {
  OwnKeys k;
  k.q = LoadSequence(a.batch, s);
  k.rows = k.q.count * (a.q_heads / a.k_heads);
  k.end = min(k.q.length, a.batch.capacity);
  const int g = a.groups > 0 ? GroupOf(a, s) : -1;
  k.grouped = g >= 0;
  k.begin = g >= 0 ? min(PrefixLength(a, g), k.end) : 0;
  return k;
}

// Keys that row r of a sequence sees.
__device__ __forceinline__ int Visible(const AttendLaunch& a, const SequenceSpan& q, int token) {
  const int all = min(q.length, a.batch.capacity);
  return a.causal ? min(max(q.length - q.count + (token - q.first) + 1, 0), all) : all;
}

// -- attend_few: every sequence's steps for each key head in turn make one
// axis, which is cut into equal parts, one a workgroup.

__device__ __forceinline__ int FewSteps(const OwnKeys& k) {
  if (k.rows == 0 || k.rows > kFewRows) return 0;
  return max(1, (k.end - k.begin + kFewStep - 1) / kFewStep);
}

struct FewAxis {
  int total;    // steps of all sequences and key heads
  int workers;  // workgroups that get a part

  __device__ FewAxis(const AttendLaunch& a, int steps)
      : total(steps * a.k_heads), workers(min(a.few_grid, steps * a.k_heads)) {}
  __device__ int Start(int w) const {
    return static_cast<int>(static_cast<int64_t>(w) * total / workers);
  }
  // The workgroup whose part holds step x: the largest w with Start(w) <= x.
  __device__ int Owner(int x) const {
    return static_cast<int>(((static_cast<int64_t>(x) + 1) * workers - 1) / total);
  }
};

// -- attend_many: items (row tile, part of the keys, key head) of groups and
// of sequences with many rows.

struct ManyUnit {
  int first, rows;  // first token, and rows a key head
  int begin, end;   // keys
  int length;       // 0: a group
};

__device__ __forceinline__ ManyUnit LoadGroup(const AttendLaunch& a, int g) {
  ManyUnit u = {0, 0, 0, 0, 0};
  const int s0 = min(max(a.group_starts[g], 0), a.batch.sequences);
  const int s1 = min(max(a.group_starts[g + 1], s0), a.batch.sequences);
  if (s0 == s1) return u;
  const SequenceSpan f = LoadSequence(a.batch, s0), l = LoadSequence(a.batch, s1 - 1);
  u.first = f.first;
  u.rows = max(l.first + l.count - f.first, 0) * (a.q_heads / a.k_heads);
  u.end = PrefixLength(a, g);
  if (u.end == 0) u.rows = 0;
  return u;
}

__device__ __forceinline__ int ManyTiles(const ManyUnit& u) {
  return (u.rows + kManyRows - 1) / kManyRows;
}
__device__ __forceinline__ int ManySteps(const ManyUnit& u) {
  return max(1, (u.end - u.begin + kManyStep - 1) / kManyStep);
}

__device__ __forceinline__ ManyUnit LoadManySequence(const OwnKeys& k) {
  ManyUnit u = {k.q.first, k.rows > kFewRows ? k.rows : 0, k.begin, k.end, k.q.length};
  return u;
}

// Parts that a unit's keys are split into: `each` steps a part where there are
// too few tiles to fill the GPU (each > 0).
__device__ __forceinline__ int ManyParts(int steps, int each) {
  return each > 0 ? (steps + each - 1) / each : 1;
}

// Steps a part (0: no split) for `tiles` tiles with `steps` steps in all.
__device__ __forceinline__ int ManyEach(const AttendLaunch& a, int tiles, int64_t steps) {
  constexpr int kLeast = 8;
  if (tiles >= a.many_target) return 0;
  return max(kLeast, static_cast<int>((steps + a.many_target - 1) / a.many_target));
}

// Slots of parts.
__device__ __forceinline__ int64_t FewSlotRow(const AttendLaunch& a, int slot) {
  return static_cast<int64_t>(slot) * a.few_rows;
}
__device__ __forceinline__ int64_t ManySlotRow(const AttendLaunch& a, int slot) {
  return static_cast<int64_t>(2 * a.few_grid) * a.few_rows +
         static_cast<int64_t>(slot) * kManyRows;
}
// The row of a (token, head) that attend_few did not cut, of a grouped sequence.
__device__ __forceinline__ int64_t WholeRow(const AttendLaunch& a, int64_t token, int head) {
  return ManySlotRow(a, a.many_parts) + token * a.q_heads + head;
}
__device__ __forceinline__ f32x2* PartStats(const AttendLaunch& a) {
  return reinterpret_cast<f32x2*>(a.parts + a.part_rows * a.padded_dim);
}

// Maximum over the four 16-lane rows of a wave, lane by lane.
__device__ __forceinline__ float Across32(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
               __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float Across16(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
               __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}

// 16 x 16 x 32 and 32 x 32 x 16 products.
template <class E>
__device__ __forceinline__ f32x4 Mma16(u32x4 x, u32x4 y, f32x4 c);
template <>
__device__ __forceinline__ f32x4 Mma16<Bf16>(u32x4 x, u32x4 y, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x),
                                                 __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 Mma16<F16>(u32x4 x, u32x4 y, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x),
                                                __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}
template <class E>
__device__ __forceinline__ f32x16 Mma32(u32x4 x, u32x4 y, f32x16 c);
template <>
__device__ __forceinline__ f32x16 Mma32<Bf16>(u32x4 x, u32x4 y, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                 __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 Mma32<F16>(u32x4 x, u32x4 y, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x),
                                                __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// Reads 4 rows x 16 columns of 16-bit elements in LDS, transposed: lane i of a
// 16-lane group names 8 bytes (row i / 4, columns 4 (i % 4)..) and gets column
// i of the four rows.
__device__ __forceinline__ u32x2 ReadTransposed(const void* p) {
  using Lds = __attribute__((address_space(3))) s16x4;
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p)));
}

// Eight e4m3 values as an operand.
template <class E>
__device__ __forceinline__ u32x4 Widen(u32x2 w) {
  return u32x4{FromE4m3<E>(w[0], false), FromE4m3<E>(w[0], true), FromE4m3<E>(w[1], false),
               FromE4m3<E>(w[1], true)};
}

}  // namespace kvx

#endif  // KVX_KERNELS_ATTEND_PLAN_H_
