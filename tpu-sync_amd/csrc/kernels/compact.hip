// The kept tokens of each sequence and key head to the front of the sequence, in place:
// place i gets the key, the value (their scales) and the weight of token kept[i], kept
// ascending, so kept[i] >= i.
//
// In place without a copy: a workgroup goes through the places of one sequence and key
// head, K or V, in ascending rounds. A round reads all of its rows into registers,
// waits for every wave, and writes them; what it writes is below every row that a later
// round reads. Rows of the next round are on their way while this one's are written.
// Where there are few sequences and heads, several workgroups take a part of every
// row's bytes each. Rows that stay at their place are neither read nor written.
//
// e4m3 (compact_e4m3_kernel): rows that meet in a block come from blocks with scales of
// their own, so the block gets the largest of them, and codes are stored again as
// e4m3(code * old / new), which rounds those of smaller scales once. A block's scale is
// replaced when all of its rows are there; later rounds read later blocks.
#include "evict.h"

#include <algorithm>

#include "attend_plan.h"

namespace kvx {
namespace {

constexpr int kThreads = kCompactThreads;
constexpr int kHeldPieces = 8;  // 16-byte pieces of rows that a thread holds

// Row of position p of a sequence: -1 without a place. In a head-major pool rows are
// [block][head][slot], else [block][slot][head].
template <bool HEAD_MAJOR>
__device__ __forceinline__ int64_t RowAt(const CompactLaunch& a, const int32_t* table, int h, int p) {
  if (p < 0 || p >= a.batch.capacity) return -1;
  const int at = FastDivI(a.block_div, p), slot = p - at * a.batch.block_tokens;
  const int64_t id = table[at];
  if (id < 0 || id >= a.batch.num_blocks) return -1;
  return HEAD_MAJOR ? (id * a.heads + h) * a.batch.block_tokens + slot
                    : (id * a.batch.block_tokens + slot) * a.heads + h;
}
// Its place in a table [block][head][slot].
template <bool HEAD_MAJOR>
__device__ __forceinline__ int64_t WeightAt(const CompactLaunch& a, int h, int64_t row, int p) {
  if constexpr (HEAD_MAJOR) return row;
  const int slot = p - FastDivI(a.block_div, p) * a.batch.block_tokens;
  // row = (id B + slot) H + h
  return row - slot * static_cast<int64_t>(a.heads) - h +
         static_cast<int64_t>(h) * a.batch.block_tokens + slot;
}

template <bool FP4>
__global__ __launch_bounds__(kThreads, 2) void compact_kernel(const CompactLaunch a,
                                                              const int places,
                                                              const int slice_bytes) {
  __shared__ int64_t from[3][kThreads], to[3][kThreads];
  const int s = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const bool key = blockIdx.y == 0;
  const int row_bytes = FP4 ? a.head_dim / 2 : a.head_dim * 2;
  char* pool = static_cast<char*>(key ? a.k_pool : a.v_pool) + blockIdx.z * slice_bytes;
  uint8_t* scales = static_cast<uint8_t*>(key ? a.k_scales : a.v_scales);
  const int32_t* table = a.batch.tables + s * a.batch.table_stride;
  const int32_t* kept = a.kept + s * a.kept_sequence + h * a.kept_head;
  const int pieces = slice_bytes / 16, items = places * pieces;
  const int rounds = (a.budget + places - 1) / places;
  // One workgroup of each row takes what lies beside it.
  const bool takes_weight = a.weights != nullptr && key && blockIdx.z == 0;
  const bool takes_scales = FP4 && blockIdx.z == 0;
  const int groups = a.head_dim / kFp4Group;
  int64_t weight_from = -1, weight_to = -1, next_from = -1, next_to = -1;

  // Rows of round r: thread t looks up place t.
  const auto look = [&](int r) {
    int64_t x = -1, y = -1;
    next_from = next_to = -1;
    const int i = r * places + static_cast<int>(threadIdx.x);
    if (static_cast<int>(threadIdx.x) < places && r < rounds && i < a.budget) {
      const int p = kept[i * a.kept_place];
      if (p >= 0 && p != i) {
        x = RowAt<FP4>(a, table, h, p);
        y = RowAt<FP4>(a, table, h, i);
        if (x < 0 || y < 0) x = y = -1;
        if (x >= 0 && takes_weight) {
          next_from = WeightAt<FP4>(a, h, x, p);
          next_to = WeightAt<FP4>(a, h, y, i);
        }
      }
    }
    from[r % 3][threadIdx.x] = x;
    to[r % 3][threadIdx.x] = y;
  };
  u32x4 rows[kHeldPieces];
  float weight = 0.0f;
  uint8_t codes[8] = {};
  const auto load = [&](int r) {
    const int64_t* at = from[r % 3];
#pragma unroll
    for (int n = 0; n < kHeldPieces; ++n) {
      const int item = static_cast<int>(threadIdx.x) + n * kThreads;
      rows[n] = u32x4{0, 0, 0, 0};
      if (item < items) {
        const int64_t x = at[item / pieces];
        if (x >= 0) {
          rows[n] = *reinterpret_cast<const u32x4*>(pool + x * row_bytes + item % pieces * 16);
        }
      }
    }
    weight_from = next_from;
    weight_to = next_to;
    if (weight_from >= 0) weight = a.weights[weight_from];
    if constexpr (FP4) {
      const int64_t x = at[threadIdx.x];
      if (takes_scales && x >= 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < groups) codes[i] = scales[x * groups + i];
        }
      }
    }
  };
  look(0);
  __syncthreads();
  load(0);
  look(1);
  for (int r = 0; r < rounds; ++r) {
    // Every wave has this round's rows before one of them is written over.
#pragma unroll
    for (int n = 0; n < kHeldPieces; ++n) asm volatile("" : : "v"(rows[n]));
    asm volatile("" : : "v"(weight));
    if constexpr (FP4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) asm volatile("" : : "v"(static_cast<uint32_t>(codes[i])));
    }
    __syncthreads();
    u32x4 now[kHeldPieces];
#pragma unroll
    for (int n = 0; n < kHeldPieces; ++n) now[n] = rows[n];
    const float now_weight = weight;
    const int64_t now_to = weight_to;
    uint8_t now_codes[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) now_codes[i] = codes[i];
    load(r + 1);
    const int64_t* at = to[r % 3];
#pragma unroll
    for (int n = 0; n < kHeldPieces; ++n) {
      const int item = static_cast<int>(threadIdx.x) + n * kThreads;
      if (item < items) {
        const int64_t y = at[item / pieces];
        if (y >= 0) {
          *reinterpret_cast<u32x4*>(pool + y * row_bytes + item % pieces * 16) = now[n];
        }
      }
    }
    if (now_to >= 0) a.weights[now_to] = now_weight;
    if constexpr (FP4) {
      const int64_t y = at[threadIdx.x];
      if (takes_scales && y >= 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < groups) scales[y * groups + i] = now_codes[i];
        }
      }
    }
    look(r + 2);
  }
}

// -- e4m3

constexpr int kScaledRows = 128;  // of a round

__device__ __forceinline__ uint32_t Rescaled(uint32_t w, float ratio) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  int q = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * ratio, lo[1] * ratio, 0, false);
  q = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * ratio, hi[1] * ratio, q, true);
  return static_cast<uint32_t>(q);
}

__global__ __launch_bounds__(kThreads, 2) void compact_e4m3_kernel(const CompactLaunch a) {
  // Per block of a group: the new scale's bits, and whether a row moves.
  __shared__ uint32_t largest[kScaledRows];
  __shared__ int moves[kScaledRows];
  __shared__ int64_t from[kScaledRows], to[kScaledRows];
  __shared__ float ratios[kScaledRows];
  constexpr int kPieces = kScaledRows * (kMaxHeadDim / 8) / kThreads;  // of a thread
  const int s = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const bool key = blockIdx.y == 0;
  uint8_t* pool = static_cast<uint8_t*>(key ? a.k_pool : a.v_pool);
  float* scales = static_cast<float*>(key ? a.k_scales : a.v_scales);
  const int32_t* table = a.batch.tables + s * a.batch.table_stride;
  const int32_t* kept = a.kept + s * a.kept_sequence + h * a.kept_head;
  const int B = a.batch.block_tokens, pieces = a.head_dim / 8;
  const bool takes_weight = a.weights != nullptr && key;
  // A group: the blocks that a round holds, or one that takes several rounds.
  const int of_group = B <= kScaledRows ? kScaledRows / B : 1;
  const auto block_of = [&](int p) {  // block id, or -1
    if (p < 0 || p >= a.batch.capacity) return -1;
    const int id = table[FastDivI(a.block_div, p)];
    return id >= 0 && id < a.batch.num_blocks ? id : -1;
  };
  const auto scale_of = [&](int id) {
    const float f = scales[static_cast<int64_t>(id) * a.heads + h];
    return f > 0.0f ? f : 0.0f;
  };
  const int64_t last = min(a.budget, a.batch.capacity);
  for (int64_t first = 0; first < last; first += static_cast<int64_t>(of_group) * B) {
    const int end = static_cast<int>(min(first + static_cast<int64_t>(of_group) * B, last));
    const int begin = static_cast<int>(first);
    for (int i = threadIdx.x; i < of_group; i += kThreads) {
      largest[i] = 0;
      moves[i] = 0;
    }
    __syncthreads();
    for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += kThreads) {
      const int p = kept[i * a.kept_place];
      const int id = block_of(p);
      if (id >= 0) {
        const int g = FastDivI(a.block_div, i - begin);
        atomicMax(&largest[g], __builtin_bit_cast(uint32_t, scale_of(id)));
        if (p != i) atomicOr(&moves[g], 1);
      }
    }
    __syncthreads();
    for (int r0 = begin; r0 < end; r0 += kScaledRows) {
      const int i = r0 + static_cast<int>(threadIdx.x);
      if (threadIdx.x < kScaledRows) {
        int64_t x = -1, y = -1;
        float ratio = 1.0f;
        if (i < end) {
          const int p = kept[i * a.kept_place], id = block_of(p), into = block_of(i);
          const int g = FastDivI(a.block_div, i - begin);
          if (id >= 0 && into >= 0 && moves[g] != 0) {
            const auto row = [&](int of, int at) {
              const int slot = at - FastDivI(a.block_div, at) * B;
              return (static_cast<int64_t>(of) * B + slot) * a.heads + h;
            };
            const float old = scale_of(id), now = __builtin_bit_cast(float, largest[g]);
            if (old != now) ratio = old / now;
            if (p != i || old != now) {
              x = row(id, p);
              y = row(into, i);
            }
          }
        }
        from[threadIdx.x] = x;
        to[threadIdx.x] = y;
        ratios[threadIdx.x] = ratio;
      }
      __syncthreads();
      u32x2 held[kPieces];
      float weight = 0.0f;
      const int items = kScaledRows * pieces;
      int64_t weight_to = -1;
#pragma unroll
      for (int n = 0; n < kPieces; ++n) {
        const int item = static_cast<int>(threadIdx.x) + n * kThreads;
        held[n] = u32x2{0, 0};
        if (item < items && from[item / pieces] >= 0) {
          held[n] = *reinterpret_cast<const Bytes8*>(pool + from[item / pieces] * a.head_dim +
                                                     item % pieces * 8);
        }
      }
      if (takes_weight && threadIdx.x < kScaledRows && from[threadIdx.x] >= 0) {
        weight = a.weights[WeightAt<false>(a, h, from[threadIdx.x], kept[i * a.kept_place])];
        weight_to = WeightAt<false>(a, h, to[threadIdx.x], i);
      }
      // Every wave has this round's rows before one of them is written over.
#pragma unroll
      for (int n = 0; n < kPieces; ++n) asm volatile("" : : "v"(held[n]));
      asm volatile("" : : "v"(weight));
      __syncthreads();
#pragma unroll
      for (int n = 0; n < kPieces; ++n) {
        const int item = static_cast<int>(threadIdx.x) + n * kThreads;
        if (item < items && to[item / pieces] >= 0) {
          const float ratio = ratios[item / pieces];
          if (ratio != 1.0f) held[n] = u32x2{Rescaled(held[n][0], ratio), Rescaled(held[n][1], ratio)};
          *reinterpret_cast<Bytes8*>(pool + to[item / pieces] * a.head_dim + item % pieces * 8) =
              held[n];
        }
      }
      if (weight_to >= 0) a.weights[weight_to] = weight;
      __syncthreads();
    }
    for (int g = threadIdx.x; g < of_group; g += kThreads) {
      const int into = begin + g * static_cast<int64_t>(B) < end ? block_of(begin + g * B) : -1;
      if (into >= 0 && moves[g] != 0) {
        scales[static_cast<int64_t>(into) * a.heads + h] =
            __builtin_bit_cast(float, largest[g]);
      }
    }
    __syncthreads();
  }
}

}  // namespace

hipError_t LaunchCompact(const CompactLaunch& l, hipStream_t stream) {
  const unsigned rows = static_cast<unsigned>(l.batch.sequences) * l.heads;
  if (l.pool == kPoolE4m3) {
    hipLaunchKernelGGL(compact_e4m3_kernel, dim3(rows, 2), dim3(kThreads), 0, stream, l);
    return hipGetLastError();
  }
  const bool fp4 = l.pool == kPoolFp4;
  // Parts of a row: two workgroups a CU, but no less than 64 bytes each.
  int slice = fp4 ? l.head_dim / 2 : l.head_dim * 2, slices = 1;
  while (rows * 2ull * slices < 512 && slice % 32 == 0 && slice >= 128) {
    slice /= 2;
    slices *= 2;
  }
  const int places = std::min(kThreads, kThreads * kHeldPieces / (slice / 16));
  hipLaunchKernelGGL(fp4 ? compact_kernel<true> : compact_kernel<false>, dim3(rows, 2, slices),
                     dim3(kThreads), 0, stream, l, places, slice);
  return hipGetLastError();
}

}  // namespace kvx
