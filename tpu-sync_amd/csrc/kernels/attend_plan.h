// How attention's work is cut up: device arithmetic that every attention
// kernel repeats over the call's lengths.
#ifndef KVX_KERNELS_ATTEND_PLAN_H_
#define KVX_KERNELS_ATTEND_PLAN_H_

#include <hip/hip_runtime.h>

#include <atomic>
#include <type_traits>

#include "attend.h"

namespace kvx {

constexpr int kAttendThreads = 256;
constexpr int kWaves = kAttendThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;

// Rows may start at any element.
using Bytes16 = u32x4 __attribute__((aligned(2)));
using Bytes8 = u32x2 __attribute__((aligned(1)));

// Raises a kernel's limit of dynamic LDS to the CU's 160 KiB, once a device.
template <auto kernel>
hipError_t AllowDynamicLds(size_t bytes) {
  static std::atomic<uint64_t> allowed{0};
  if (bytes <= 65536) return hipSuccess;
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  const uint64_t bit = uint64_t{1} << (device & 63);
  if (e != hipSuccess || (allowed.load() & bit) != 0) return e;
  // What the kernel's own arrays leave of a CU's.
  hipFuncAttributes own;
  e = hipFuncGetAttributes(&own, reinterpret_cast<const void*>(kernel));
  if (e != hipSuccess) return e;
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize,
                          160 * 1024 - static_cast<int>(own.sharedSizeBytes));
  if (e == hipSuccess) allowed.fetch_or(bit);
  return e;
}

__device__ __forceinline__ int FastDivI(const FastDivU32& f, int n) {
  const uint32_t u = static_cast<uint32_t>(n);
  return static_cast<int>((__umulhi(u, f.m) + u) >> f.s);
}

// In-place inclusive sums of c[0..n) over the workgroup (n <= kMaxSequences *
// 2), none above `most` (AddUpTo). c[i] must have been written by any thread
// before, and is visible to all after.
__device__ __forceinline__ void BlockSums(int* c, int n, int most) {
  __shared__ int waves[kWaves];
  const auto add = [&](int x, int y) { return AddUpTo(x, y, most); };
  const int each = (n + kAttendThreads - 1) / kAttendThreads;
  const int i0 = threadIdx.x * each, i1 = min(i0 + each, n);
  __syncthreads();
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine = add(mine, c[i]);
  int sum = mine;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const int o = __shfl_up(sum, m);
    if (lane >= m) sum = add(sum, o);
  }
  if (lane == 63) waves[wave] = sum;
  // What the lanes before this one have.
  int at = __shfl_up(sum, 1);
  if (lane == 0) at = 0;
  __syncthreads();
  for (int w = 0; w < wave; ++w) at = add(at, waves[w]);
  for (int i = i0; i < i1; ++i) {
    at = add(at, c[i]);
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

// Work of all sequences and key heads laid end to end and cut into parts of
// `each`, one a worker.
struct Axis {
  int total, each, workers;
  float inverse;  // 1 / each

  __device__ Axis(int work, int most) : total(work) {
    each = most > 0 ? max((work + most - 1) / most, 1) : 1;
    workers = most > 0 ? (work + each - 1) / each : 0;
    inverse = 1.0f / static_cast<float>(each);
  }
  __device__ __forceinline__ int Start(int w) const { return min(w * each, total); }
  // The worker whose part holds x. The product is off by under one (x / each is
  // below 2^12, its relative error below 2^-21).
  __device__ __forceinline__ int Owner(int x) const {
    const int w = static_cast<int>(static_cast<float>(x) * inverse);
    const int rest = x - w * each;
    return w + (rest >= each ? 1 : 0) - (rest < 0 ? 1 : 0);
  }
  // Worker w's slot for the piece that starts at x in its part: a part cuts at
  // most the first and the last of its pieces.
  __device__ __forceinline__ int Slot(int w, int x) const {
    return x == w * each ? 2 * w : 2 * w + 1;
  }
};

// -- Few rows: steps of kFewStep tokens; a worker is a wave.

__device__ __forceinline__ int FewSteps(const OwnKeys& k) {
  if (k.rows == 0 || k.rows > kFewRows) return 0;
  return max(1, (k.end - k.begin + kFewStep - 1) / kFewStep);
}

__device__ __forceinline__ Axis FewAxis(const AttendLaunch& a, int steps) {
  return Axis(steps * a.k_heads, a.few_grid * kWaves);
}

// -- Many rows: tiles of kManyRows rows of the groups, then of the sequences
// with more than kFewRows rows; a worker is a workgroup. Under a causal mask
// tile r sees 128 r / G keys more than the first, so the axis gives it
// `base` + 2 r / G steps of 64: C(r) = r base + r (r - 1) / G is where it starts.

struct ManyUnit {
  int first, rows;  // first token, and rows a key head
  int begin, end;   // keys
  int base;         // steps of the first tile
};

__device__ __forceinline__ int ManyTiles(const ManyUnit& u) {
  return (u.rows + kManyRows - 1) / kManyRows;
}

__device__ __forceinline__ int ManyCost(const AttendLaunch& a, bool group, int base, int tile) {
  const int more = group || !a.causal ? 0 : FastDivI(a.group_div, tile * (tile - 1));
  return tile * base + more;
}

// The last of `tiles` tiles that starts at or before `at` of its unit's axis.
__device__ __forceinline__ int TileAt(const AttendLaunch& a, bool group, int base, int tiles,
                                      int at) {
  int tile = 0;
  while (tiles - tile > 1) {
    const int mid = (tile + tiles) / 2;
    if (ManyCost(a, group, base, mid) <= at) {
      tile = mid;
    } else {
      tiles = mid;
    }
  }
  return tile;
}

__device__ __forceinline__ ManyUnit LoadGroup(const AttendLaunch& a, int g) {
  ManyUnit u = {0, 0, 0, 0, 0};
  const int s0 = min(max(a.group_starts[g], 0), a.batch.sequences);
  const int s1 = min(max(a.group_starts[g + 1], s0), a.batch.sequences);
  if (s0 == s1) return u;
  const SequenceSpan f = LoadSequence(a.batch, s0), l = LoadSequence(a.batch, s1 - 1);
  u.first = f.first;
  u.end = PrefixLength(a, g);
  if (u.end > 0) u.rows = max(l.first + l.count - f.first, 0) * (a.q_heads / a.k_heads);
  u.base = (u.end + kManyStep - 1) / kManyStep + 1;
  return u;
}

__device__ __forceinline__ ManyUnit LoadManySequence(const AttendLaunch& a, const OwnKeys& k) {
  ManyUnit u = {k.q.first, k.rows > kFewRows ? k.rows : 0, k.begin, k.end, 0};
  const int ahead = a.causal ? min(k.q.length - k.q.count, k.end) : k.end;
  u.base = max(ahead - k.begin, 0) / kManyStep + 2;
  return u;
}

__device__ __forceinline__ ManyUnit LoadManyUnit(const AttendLaunch& a, int i) {
  return i < a.groups ? LoadGroup(a, i) : LoadManySequence(a, LoadOwnKeys(a, i - a.groups));
}

__device__ __forceinline__ int ManyWork(const AttendLaunch& a, int i, const ManyUnit& u) {
  return ManyCost(a, i < a.groups, u.base, ManyTiles(u));
}

// A worker's least part, in steps of 64 tokens: small calls spread over more
// workgroups, though more of their tiles are cut and joined. 3141 shared tokens of
// one sequence's 32 heads on 8, D = 64: 24.5 us with parts of 8 steps, 17.1 us of
// 2, 17.2 us of 1; 3 chunks of 16 tokens over 4000 keys: 25.3, 21.9 and 27.0 us.
// Large calls have larger parts anyway.
constexpr int kLeastPart = 2;
__device__ __forceinline__ Axis ManyAxis(const AttendLaunch& a, int work) {
  const int total = work * a.k_heads;
  return Axis(total, min(a.many_grid, max(total / kLeastPart, 1)));
}

// Rows of `parts`: two slots a wave of few_rows rows, two slots a workgroup of
// kManyRows rows; with groups a row for every (token, head) that was not cut,
// of its own keys and of its group's.
__device__ __forceinline__ int64_t FewSlotRow(const AttendLaunch& a, int slot) {
  return static_cast<int64_t>(slot) * a.few_rows;
}
__device__ __forceinline__ int64_t ManySlotRow(const AttendLaunch& a, int slot) {
  return 2ll * kWaves * a.few_grid * a.few_rows + static_cast<int64_t>(slot) * kManyRows;
}
__device__ __forceinline__ int64_t WholeRow(const AttendLaunch& a, bool group, int64_t token,
                                            int head) {
  return ManySlotRow(a, 2 * a.many_grid) + (group ? 1ll : 0ll) * a.batch.tokens * a.q_heads +
         token * a.q_heads + head;
}
__device__ __forceinline__ f32x2* PartStats(const AttendLaunch& a) {
  return reinterpret_cast<f32x2*>(a.parts + a.part_rows * a.padded_dim);
}

// The plan that attend_join reads, in words.
struct PlanView {
  int* few;     // [sequences] inclusive sums of FewSteps
  int* many;    // [groups + sequences] inclusive sums of ManyWork
  int* todo;    // [sequences] inclusive sums of grouped sequences' row groups
  int* first;   // [sequences] first token
  int* rows;    // [sequences] rows a key head
  int* group;   // [sequences] group or -1
  int* base;    // [groups + sequences] ManyUnit::base
  int* gfirst;  // [groups] first token

  __device__ PlanView(const AttendLaunch& a, int* at) {
    const int S = a.batch.sequences, units = S + a.groups;
    few = at;
    many = few + S;
    todo = many + units;
    first = todo + S;
    rows = first + S;
    group = rows + S;
    base = group + S;
    gfirst = base + units;
  }
};
__host__ __device__ inline int PlanWords(const AttendLaunch& a) {
  return 7 * a.batch.sequences + 3 * a.groups;
}
// Of those, the ones that are summed up in LDS.
__host__ __device__ inline int PlanSumWords(const AttendLaunch& a) {
  return 3 * a.batch.sequences + a.groups;
}
__device__ __forceinline__ int* Plan(const AttendLaunch& a) {
  return reinterpret_cast<int*>(PartStats(a) + a.part_rows);
}

// Written by one workgroup of the kernel before attend_join. lds: PlanSumWords.
__device__ __forceinline__ void WritePlan(const AttendLaunch& a, int* lds) {
  const int S = a.batch.sequences, units = a.groups + S;
  const PlanView here(a, lds), to(a, Plan(a));
  for (int s = threadIdx.x; s < S; s += kAttendThreads) {
    const OwnKeys k = LoadOwnKeys(a, s);
    here.few[s] = FewSteps(k);
    here.todo[s] = k.grouped ? (k.rows + a.join_rows - 1) / a.join_rows : 0;
    to.first[s] = k.q.first;
    to.rows[s] = k.rows;
    to.group[s] = k.grouped ? GroupOf(a, s) : -1;
  }
  for (int i = threadIdx.x; i < units; i += kAttendThreads) {
    const ManyUnit u = LoadManyUnit(a, i);
    here.many[i] = ManyWork(a, i, u);
    to.base[i] = u.base;
    if (i < a.groups) to.gfirst[i] = u.first;
  }
  BlockSums(here.few, S, a.most_few);
  BlockSums(here.many, units, a.most_many);
  BlockSums(here.todo, S, a.batch.tokens * (a.q_heads / a.k_heads) / a.join_rows + S);
  int* out = Plan(a);
  for (int i = threadIdx.x; i < PlanSumWords(a); i += kAttendThreads) out[i] = lds[i];
}

// o, or zeros where a row or its part sees nothing (l = 0): values that it does
// not see have met exponentials of 0, which leaves NaN of those that are not finite.
__device__ __forceinline__ f32x4 Seen(f32x4 o, float l) {
  return l == 0.0f ? f32x4{0, 0, 0, 0} : o;
}
// 1 / l, and 0 of 0.
__device__ __forceinline__ float InverseSum(float l) {
  return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
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

// Eight e4m3 values times a power of two as an operand.
template <class E>
__device__ __forceinline__ u32x4 Widen(u32x2 w, float power = 1.0f) {
  return u32x4{FromE4m3<E>(w[0], false, power), FromE4m3<E>(w[0], true, power),
               FromE4m3<E>(w[1], false, power), FromE4m3<E>(w[1], true, power)};
}

// The scale of e4m3 values goes to the exponentials, so that the values stay
// exact and a product is rounded once. In bf16 all of it does; an exponential,
// up to 2^8, that takes it could leave fp16's range, so there the values take its
// power of two, as far as they stay exact, and the exponentials the rest.
template <class E>
__device__ __forceinline__ float ValuePower(float scale) {
  if constexpr (!std::is_same_v<E, F16>) return 1.0f;
  const float power = __builtin_bit_cast(
      float, __builtin_bit_cast(uint32_t, scale) & 0x7f800000u);
  return fminf(fmaxf(power, 1.0f / 32768), 128.0f);
}
template <class E>
__device__ __forceinline__ float ValueRest(float scale) {
  if constexpr (!std::is_same_v<E, F16>) return scale;
  return scale * __builtin_bit_cast(
      float, 0x7f000000u - __builtin_bit_cast(uint32_t, ValuePower<E>(scale)));
}

}  // namespace kvx

#endif  // KVX_KERNELS_ATTEND_PLAN_H_
