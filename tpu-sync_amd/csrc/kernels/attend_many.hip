// Paged attention of many rows a key head: chunks of new tokens, and all rows
// of sequences that share a prefix against that prefix.
//
// A workgroup takes a tile of 128 rows, 32 a wave, and steps through its keys
// 64 at a time: the tile of K and V lies in LDS for all four waves, the next
// one is on its way from memory in registers. Matrix instructions bound it,
// so the layout keeps everything between the two products in place: S^T = K Q^T
// in 32 x 32 x 16 products leaves lane l with the scores of row l % 32, so a
// row's maximum takes one swap between the wave's halves, and the packed
// exponentials are the operand of O^T = V^T P^T as they stand (the contraction
// runs over tokens in the order that the scores lie in). V is transposed by
// the LDS reads.
//
// Work. Items are (row tile, part of the keys, key head) of the groups first,
// then of the sequences with more than kFewRows rows. Where the row tiles
// alone would not fill the GPU, keys are split into parts of equal steps; parts,
// and all that has to do with a group, go to slots of `parts`, which attend_join
// merges.
#include "attend_plan.h"

namespace kvx {
namespace {

using Bytes16 = u32x4 __attribute__((aligned(2)));
using Bytes8 = u32x2 __attribute__((aligned(1)));

// Bytes of a token in LDS. Keys: an odd multiple of 16, so that the 16-byte
// reads of neighbouring rows fall on different banks; values: 64 beyond a
// multiple of 128, so that the 32-byte reads of four rows do.
constexpr int KeyStride(int dp) { return dp * 2 + 16; }
constexpr int ValueStride(int dp) { return (dp * 2) % 128 == 64 ? dp * 2 : dp * 2 + 64; }

// Places of a step's tokens, looked up two steps ahead.
struct Places {
  int64_t at[kManyStep];  // element offset of the token's row, or -1
  float k_scale[kManyStep], v_scale[kManyStep];
  uint64_t present;  // one bit a token
};

template <class E, bool E4, int DP>
__global__ __launch_bounds__(kAttendThreads, DP <= 128 ? 2 : 1) void
attend_many_kernel(const AttendLaunch a) {
  using P = std::conditional_t<E4, Bf16, E>;
  using Scalar = typename E::Scalar;
  constexpr int KS = DP / 16, DT = DP / 32, KST = KeyStride(DP), VST = ValueStride(DP);
  constexpr int kChunks = kManyStep * (DP / 8) / kAttendThreads;  // of a thread
  constexpr int kTile = kManyStep * (KST + VST);
  extern __shared__ __align__(16) char lds[];
  Places* places = reinterpret_cast<Places*>(lds + 2 * kTile);
  int* sums = reinterpret_cast<int*>(places + 4);  // [groups + sequences]
  const BatchView& b = a.batch;
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };

  // The item.
  const int units = a.groups + b.sequences;
  const auto unit_of = [&](int i) {
    return i < a.groups ? LoadGroup(a, i) : LoadManySequence(LoadOwnKeys(a, i - a.groups));
  };
  for (int i = threadIdx.x; i < units; i += kAttendThreads) sums[i] = ManyTiles(unit_of(i));
  BlockSums(sums, units);
  const int tiles = one(sums[units - 1]) * a.k_heads;
  if (tiles == 0) return;
  int each = 0;
  if (tiles < a.many_target) {
    __syncthreads();
    for (int i = threadIdx.x; i < units; i += kAttendThreads) {
      const ManyUnit u = unit_of(i);
      sums[i] = ManyTiles(u) * ManySteps(u);
    }
    BlockSums(sums, units);
    each = ManyEach(a, tiles, static_cast<int64_t>(one(sums[units - 1])) * a.k_heads);
    __syncthreads();
    for (int i = threadIdx.x; i < units; i += kAttendThreads) {
      const ManyUnit u = unit_of(i);
      sums[i] = ManyTiles(u) * ManyParts(ManySteps(u), each);
    }
    BlockSums(sums, units);
  }
  const int item = blockIdx.x;
  if (item >= one(sums[units - 1]) * a.k_heads) return;
  const int i = one(FirstAbove(sums, units, item / a.k_heads));
  const ManyUnit u = unit_of(i);
  const int rows = one(u.rows), begin = one(u.begin), end = one(u.end), first = one(u.first);
  const int steps = one(ManySteps(u)), parts = one(ManyParts(steps, each));
  int rest = item - (i > 0 ? one(sums[i - 1]) : 0) * a.k_heads;
  // Row tiles from the last: under a causal mask they see most. Neighbouring
  // items share keys: tile by tile within a part of a key head.
  const int unit_tiles = one(ManyTiles(u));
  const int tile = unit_tiles - 1 - rest % unit_tiles;
  rest /= unit_tiles;
  const int part = rest % parts, h = rest / parts;
  const bool grouped = i < a.groups;
  const bool split = parts > 1 || grouped || LoadOwnKeys(a, i - a.groups).grouped;
  const int sequence = grouped ? min(max(one(a.group_starts[i]), 0), b.sequences - 1)
                               : i - a.groups;
  const SequenceSpan span = LoadSequence(b, sequence);
  const int part_steps = (steps + parts - 1) / parts;
  const int step0 = part * part_steps;
  int step1 = min(steps, step0 + part_steps);
  const int G = a.q_heads / a.k_heads;

  // Queries: row l % 32 of the wave's 32, as an operand.
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int in32 = lane % 32, half = lane / 32;
  const int row = tile * kManyRows + wave * 32 + in32;
  const int t = FastDivI(a.group_div, row);
  const int64_t token = first + t;
  const int head = h * G + (row - t * G);
  int seen = INT_MAX;
  if (row < rows) {
    if (!grouped) {
      seen = Visible(a, span, first + t);
    } else {
      int s = static_cast<int>(token);
      if (b.starts != nullptr) {
        int lo = 0, hi = b.sequences;  // first s with starts[s + 1] > token
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (b.starts[mid + 1] > token) {
            hi = mid;
          } else {
            lo = mid + 1;
          }
        }
        s = min(lo, b.sequences - 1);
      }
      seen = min(Visible(a, LoadSequence(b, s), static_cast<int>(token)), end);
    }
  }
  int least = seen, most_seen = row < rows ? seen : 0;
#pragma unroll
  for (int m = 32; m > 0; m /= 2) {
    least = min(least, __shfl_xor(least, m));
    most_seen = max(most_seen, __shfl_xor(most_seen, m));
  }
  least = one(least);
  most_seen = one(most_seen);
  if (!grouped && a.causal) {
    // Keys behind the tile's last row are seen by none of its rows.
    const int last = min(rows, (tile + 1) * kManyRows) - 1;
    const int all = Visible(a, span, first + FastDivI(a.group_div, last));
    step1 = min(step1, (max(all - begin, 0) + kManyStep - 1) / kManyStep);
  }
  u32x4 q[KS];
  {
    const Scalar* p = static_cast<const Scalar*>(a.q) + token * a.q_token + head * a.q_head +
                      half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[ks] = u32x4{0, 0, 0, 0};
      if (row < rows && ks * 16 + half * 8 < a.head_dim) {
        q[ks] = *reinterpret_cast<const Bytes16*>(p + ks * 16);
      }
    }
  }

  const int32_t* table = b.tables + sequence * b.table_stride;
  const int64_t row_stride = static_cast<int64_t>(a.k_heads) * a.head_dim;
  // One wave looks up a step's 64 tokens.
  const auto find = [&](int step) {
    Places& to = places[step & 3];
    const int p = begin + step * kManyStep + lane;
    int64_t at = -1;
    if (step < step1 && p < end) {
      const int n = FastDivI(a.block_div, p), id = table[n];
      if (id >= 0 && id < b.num_blocks) {
        at = (static_cast<int64_t>(id) * b.block_tokens + (p - n * b.block_tokens)) * row_stride +
             h * a.head_dim;
        if constexpr (E4) {
          to.k_scale[lane] = a.k_scales[static_cast<int64_t>(id) * a.k_heads + h];
          to.v_scale[lane] = a.v_scales[static_cast<int64_t>(id) * a.k_heads + h];
        }
      }
    }
    to.at[lane] = at;
    const uint64_t present = __ballot(at >= 0);
    if (lane == 0) to.present = present;
  };
  constexpr int W = E4 ? 2 : 4;
  using Words = __attribute__((ext_vector_type(W))) uint32_t;
  Words kw[kChunks], vw[kChunks];
  const auto load = [&](int step) {
    const Places& from = places[step & 3];
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      const int chunk = threadIdx.x + n * kAttendThreads;
      const int tok = chunk / (DP / 8), d = chunk % (DP / 8) * 8;
      const int64_t at = from.at[tok];
      kw[n] = vw[n] = Words(0);
      if (at >= 0 && d < a.head_dim) {
        if constexpr (E4) {
          kw[n] = *reinterpret_cast<const Bytes8*>(static_cast<const uint8_t*>(a.k_pool) + at + d);
          vw[n] = *reinterpret_cast<const Bytes8*>(static_cast<const uint8_t*>(a.v_pool) + at + d);
        } else {
          kw[n] = *reinterpret_cast<const Bytes16*>(static_cast<const Scalar*>(a.k_pool) + at + d);
          vw[n] = *reinterpret_cast<const Bytes16*>(static_cast<const Scalar*>(a.v_pool) + at + d);
        }
      }
    }
  };
  const auto store = [&](int step) {
    char* to = lds + (step & 1) * kTile;
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      const int chunk = threadIdx.x + n * kAttendThreads;
      const int tok = chunk / (DP / 8), d = chunk % (DP / 8) * 8;
      u32x4 k, v;
      if constexpr (E4) {
        k = Widen<E>(kw[n]);
        v = Widen<P>(vw[n]);
      } else {
        k = kw[n];
        v = vw[n];
      }
      *reinterpret_cast<u32x4*>(to + tok * KST + d * 2) = k;
      *reinterpret_cast<u32x4*>(to + kManyStep * KST + tok * VST + d * 2) = v;
    }
  };

  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16(0.0f);
  float top = -__builtin_inff(), sum = 0.0f;
  const float c = a.scale * kLog2e;
  if (step0 < step1) {
    if (wave < 2) find(step0 + wave);
    __syncthreads();
    load(step0);
    store(step0);
  }
  for (int step = step0; step < step1; ++step) {
    __syncthreads();
    if (step + 1 < step1) load(step + 1);
    if (wave == (step & 3)) find(step + 2);
    const Places& here = places[step & 3];
    const int p0 = begin + step * kManyStep;
    if (p0 < most_seen) {
      const char* keys = lds + (step & 1) * kTile;
      const char* values = keys + kManyStep * KST;
      f32x16 sc[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sc[u] = f32x16(0.0f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 key = *reinterpret_cast<const u32x4*>(keys + (u * 32 + in32) * KST +
                                                            ks * 32 + half * 16);
          sc[u] = Mma32<E>(key, q[ks], sc[u]);
        }
      }
      // Lane: row l % 32, tokens 32 u + 8 (i / 4) + 4 (l / 32) + i % 4.
      if constexpr (E4) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4 f =
                *reinterpret_cast<const f32x4*>(&here.k_scale[u * 32 + i * 2 + half * 4]);
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[u][i + j] *= f[j];
          }
        }
      }
      const uint64_t present = here.present;
      if (p0 + kManyStep > least || present != ~uint64_t{0}) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int j = u * 32 + (i / 4) * 8 + half * 4 + i % 4;
            if (p0 + j >= seen || (present >> j & 1) == 0) sc[u][i] = -__builtin_inff();
          }
        }
      }
      float most = sc[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) most = fmaxf(most, sc[i / 16][i % 16]);
      most = Across32(most) * c;
      // The maximum is only moved when it falls behind by 2^8.
      if (__any(most > top + 8.0f)) {
        const float now = fmaxf(top, most);
        const float back = now == -__builtin_inff() ? 0.0f : now;
        const float shrink = __builtin_amdgcn_exp2f(top - back);
        top = now;
        sum *= shrink;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] *= shrink;
      }
      const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sc[u][i] = __builtin_amdgcn_exp2f(fmaf(sc[u][i], c, -base));
          sum += sc[u][i];
        }
      }
      if constexpr (E4) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4 f =
                *reinterpret_cast<const f32x4*>(&here.v_scale[u * 32 + i * 2 + half * 4]);
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[u][i + j] *= f[j];
          }
        }
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int u = kk / 2, i = kk % 2 * 8;
        const u32x4 p = {Pack2<P>(sc[u][i], sc[u][i + 1]), Pack2<P>(sc[u][i + 2], sc[u][i + 3]),
                         Pack2<P>(sc[u][i + 4], sc[u][i + 5]),
                         Pack2<P>(sc[u][i + 6], sc[u][i + 7])};
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const char* from = values + (kk * 16 + half * 4 + lane % 16 / 4) * VST + dt * 64 +
                             lane / 16 % 2 * 32 + lane % 4 * 8;
          const u32x2 lo = ReadTransposed(from), hi = ReadTransposed(from + 8 * VST);
          o[dt] = Mma32<P>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p, o[dt]);
        }
      }
    }
    if (step + 1 < step1) store(step + 1);
  }

  // Lane: row l % 32, dimensions 32 dt + 8 (i / 4) + 4 (l / 32) + i % 4.
  sum += __shfl_xor(sum, 32);
  if (row >= rows) return;
  if (split) {
    const int64_t to = ManySlotRow(a, item) + wave * 32 + in32;
    if (half == 0) PartStats(a)[to] = f32x2{top, sum};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        *reinterpret_cast<f32x4*>(a.parts + to * DP + dt * 32 + i * 2 + half * 4) =
            f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
      }
    }
    return;
  }
  const float inverse = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  Scalar* out = static_cast<Scalar*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = dt * 32 + i * 2 + half * 4;
      using Pair = u32x2 __attribute__((aligned(2)));
      if (d < a.head_dim) {
        *reinterpret_cast<Pair*>(out + d) =
            u32x2{Pack2<E>(o[dt][i] * inverse, o[dt][i + 1] * inverse),
                  Pack2<E>(o[dt][i + 2] * inverse, o[dt][i + 3] * inverse)};
      }
    }
  }
  if (a.lse != nullptr && half == 0) {
    a.lse[token * a.q_heads + head] = (top + log2f(sum)) / kLog2e;
  }
}

template <class E, bool E4, int DP>
hipError_t Launch(const AttendLaunch& l, hipStream_t stream) {
  const size_t lds = 2 * kManyStep * (KeyStride(DP) + ValueStride(DP)) + 4 * sizeof(Places) +
                     static_cast<size_t>(l.groups + l.batch.sequences) * sizeof(int);
  const auto kernel = attend_many_kernel<E, E4, DP>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(lds));
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, dim3(l.many_grid), dim3(kAttendThreads), lds, stream, l);
  return hipGetLastError();
}

template <class E, bool E4>
hipError_t Pick(const AttendLaunch& l, hipStream_t stream) {
  switch (l.padded_dim) {
    case 64:
      return Launch<E, E4, 64>(l, stream);
    case 96:
      return Launch<E, E4, 96>(l, stream);
    case 128:
      return Launch<E, E4, 128>(l, stream);
    default:
      return Launch<E, E4, 256>(l, stream);
  }
}

}  // namespace

hipError_t LaunchAttendMany(const AttendLaunch& l, hipStream_t stream) {
  if (l.type == kBf16) return l.e4m3 ? Pick<Bf16, true>(l, stream) : Pick<Bf16, false>(l, stream);
  return l.e4m3 ? Pick<F16, true>(l, stream) : Pick<F16, false>(l, stream);
}

}  // namespace kvx
