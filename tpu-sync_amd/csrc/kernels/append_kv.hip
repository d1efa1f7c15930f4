// New keys and values into the paged pool.
//
// Token i of sequence s sits at position p = lengths[s] - count[s] + i, slot
// p % B of block tables[s][p / B]. A key is normed and rotated on the way
// (head_row.h); a value is copied. A token whose position or block id has no
// place is dropped.
//
// Pool of the inputs' type (append_kv_kernel): a workgroup takes a few tokens,
// finds their sequences (all lengths at once, one a lane), puts places and
// (cos, sin) into LDS; teams of lanes (head_row.h) take a token's key heads and
// value heads in turn. Reading and writing the rows bounds it: 16384 tokens x 8
// heads x 128, normed, 34.5 us from cold caches (3.9 TB/s both ways), 26.3 us
// again and again on rows that the last-level cache holds; one token of each of
// 64 sequences 4.1 us, which is the launch and its dependent loads.
//
// 4-bit pool: the same kernel with another way to store a row (Fp4Row). Every 32
// dimensions of a token's head have a power-of-two scale of their own, so a row is
// stored by itself, whatever the block holds: four lanes find the largest of the 32
// values as the bits of integers, the scale is integer arithmetic on its exponent, and
// the conversion divides by it exactly and rounds once. 16384 tokens x 8 heads x 128,
// normed, 26.0 us (67 MB read, 18 written; 134 MB in 16 bits 26.1). Without the norm 24.2,
// without the rotation too 21.2: most of it is reading and packing. Vector instructions
// take 55 % of the SIMDs' cycles, 45 % without norm and rotation, and waves wait half of
// theirs. One token of each of 64 sequences: 4.3 us.
//
// e4m3 pool (append_e4m3_kernel): one fp32 scale per (block, head), so all
// rows of a block and head have to be seen before the first is written. A
// workgroup takes the new rows of one block, K or V, a wave the heads in turn:
//   amax = max |x| over the finite new values
//   new  = max(old, amax / 448),  old = 0 where no earlier token is in the block
//   q    = e4m3(clamp(x / new, -448, 448)).
// A wave holds up to kHeld rows a lane of one head in registers, all loaded
// before the first is worked on (one, where there is one new token), so that the
// rows are read once; a block with more new rows is read once for amax and again
// (from the cache) to be stored. Registers decide: 8201 tokens x 8 heads x 128
// took 23 us with 8 rows held by 2 waves a SIMD (256 registers), 32 us with 4 by
// 3, 61 us with 4 by 4 (spilled); 25.4 us since codes are exact quotients.
// Workgroups have as many waves as heads, up to four: 85624 tokens of one head,
// normed, 41 us; with three waves idle 76 us.
// Earlier tokens of the block are stored again at old / new where new is
// larger, so they keep their values within e4m3's rounding. Nothing is
// accumulated over blocks or waves: the same call gives the same bytes.
#include <hip/hip_runtime.h>

#include "append_kv.h"
#include "head_row.h"

namespace kvx {
namespace {

constexpr int kThreads = kRowThreads;
constexpr int kWaves = kThreads / 64;
// append_kv_kernel: a workgroup takes one token until there are kEnough
// workgroups, then more, up to kMaxTokens. 2048 and 8192 tokens x 8 heads x 128:
// 6.5 and 15.0 us; with 256 as enough 8.0 and 23.0 us, with 4096 6.5 and 16.2 us.
constexpr int kMaxTokens = kMostRowTokens;
constexpr int kEnough = 1024;

__device__ __forceinline__ int FastDiv(const FastDivU32& f, int n) {
  const uint32_t u = static_cast<uint32_t>(n);
  return static_cast<int>((__umulhi(u, f.m) + u) >> f.s);
}

__device__ __forceinline__ int64_t RotationPosition(const AppendLaunch& a, int64_t token,
                                                    int place) {
  if (a.positions == nullptr) return place;
  return a.positions_64 ? static_cast<const int64_t*>(a.positions)[token]
                        : static_cast<const int32_t*>(a.positions)[token];
}

// A row's codes and scales in a 4-bit pool. A lane holds 8 neighbouring values
// and four lanes a group (VEC 8), or a lane one value and half a wave a group.
template <class E, int VEC, int LPR>
struct Fp4Row {
  using Lane = RowLane<E, VEC, LPR>;
  static __device__ __forceinline__ uint32_t GroupMost(uint32_t m) {
    if constexpr (VEC == 8) {
      const auto most = [&m](auto control) {
        m = max(m, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
                       0, static_cast<int>(m), decltype(control)::value, 0xf, 0xf, true)));
      };
      most(std::integral_constant<int, 0xb1>{});  // lanes 1 0 3 2
      most(std::integral_constant<int, 0x4e>{});  // lanes 2 3 0 1
    } else {
#pragma unroll
      for (int i = 1; i < 32; i *= 2) {
        m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), i)));
      }
    }
    return m;
  }
  // Every lane of a wave takes part.
  static __device__ __forceinline__ void Store(const Lane& l, const float (*x)[VEC], bool stores,
                                               uint8_t* codes, uint8_t* scales) {
    constexpr uint32_t kEndless = 0x7f800000u;
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        m = max(m, __builtin_bit_cast(uint32_t, x[n][j]) & 0x7fffffffu);
      }
      m = GroupMost(m);
      // Infinities are no part of the largest value, and are clamped.
      if (__any(m == kEndless)) {
        uint32_t finite = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint32_t u = __builtin_bit_cast(uint32_t, x[n][j]) & 0x7fffffffu;
          finite = max(finite, u < kEndless ? u : 0u);
        }
        finite = GroupMost(finite);
        if (m == kEndless) m = finite;
      }
      // The smallest power of two s with m <= 7 s: 6 is the largest code, and up to 7
      // it is the nearest one. Bounded, so that 6 s is finite and the smallest code
      // no subnormal number. A NaN makes NaN of its group.
      constexpr uint32_t top = std::is_same_v<E, F16> ? kFp4MostF16 : kFp4Most;
      const uint32_t code = m > kEndless
                                ? 255u
                                : min(max((m + 0x1fffffu) >> 23, kFp4Least + 2) - 2, top);
      const float scale = __builtin_bit_cast(float, code << 23);
      const bool writes = stores && l.Has(n);
      // The quotient by a power of two is exact, and the instruction rounds to the
      // nearest code, to the even one in the middle, and to 6 above it.
      if constexpr (VEC == 8) {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[n][0], x[n][1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[n][2], x[n][3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[n][4], x[n][5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[n][6], x[n][7], scale, 3);
        if (writes) *reinterpret_cast<uint32_t*>(codes + l.Dim(n) / 2) = w;
      } else {
        const float other = __shfl_xor(x[n][0], 1);
        const uint32_t w =
            __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[n][0], other, scale, 0);
        if (writes && l.Dim(n) % 2 == 0) codes[l.Dim(n) / 2] = static_cast<uint8_t>(w);
      }
      if (writes && l.Dim(n) % kFp4Group == 0) {
        scales[l.Dim(n) / kFp4Group] = static_cast<uint8_t>(code);
      }
    }
  }
};

template <class E, int VEC, int LPR, bool FP4>
__global__ __launch_bounds__(kThreads) void append_kv_kernel(const AppendLaunch a,
                                                             const int tokens_each,
                                                             const int teams_of_token) {
  extern __shared__ f32x2 cs[];  // [tokens_each][rotary_dim / 2]
  __shared__ int sequence[kMaxTokens], place[kMaxTokens];
  // First element of the token's rows (in 4 bits its first head's row), or -1.
  __shared__ int64_t row_at[kMaxTokens];
  using Scalar = typename E::Scalar;
  const int pairs = a.rotary_dim / 2;
  const int t0 = blockIdx.x * tokens_each;
  const int nt = min(tokens_each, a.batch.tokens - t0);
  const RowLane<E, VEC, LPR> lane(a.head_dim, a.rotary_dim, a.interleaved);
  // The team's first token and head; heads are shared out over the token's
  // teams of gridDim.y workgroups.
  const int team = threadIdx.x / LPR;
  const int first = blockIdx.y * teams_of_token + team % teams_of_token;
  const int step = teams_of_token * gridDim.y;
  const int token_step = kThreads / LPR / teams_of_token;
  RawRow<E, VEC, LPR> keys, values;
  const auto load = [&](int t, int h) {
    if (h >= a.heads) return;
    keys.Load(lane, static_cast<const Scalar*>(a.k) + (t0 + t) * a.k_token + h * a.k_head, true);
    values.Load(lane, static_cast<const Scalar*>(a.v) + (t0 + t) * a.v_token + h * a.v_head, false);
  };
  int t = team / teams_of_token;
  if (t < nt) load(t, first);  // in flight while the places are found
  Weights<E, VEC, LPR> weights;
  weights.Load(lane, a.k_weight, a.weight_f32);

  if (threadIdx.x < kMaxTokens) sequence[threadIdx.x] = -1;
  __syncthreads();
  if (a.batch.starts == nullptr) {
    if (threadIdx.x < nt) {
      const int s = t0 + threadIdx.x;
      const SequenceSpan q = LoadSequence(a.batch, s);
      sequence[threadIdx.x] = s;
      place[threadIdx.x] = q.length - 1;
    }
  } else {
    for (int s = threadIdx.x; s < a.batch.sequences; s += kThreads) {
      const SequenceSpan q = LoadSequence(a.batch, s);
      const int end = min(q.first + q.count, t0 + nt);
      for (int i = max(q.first, t0); i < end; ++i) {
        sequence[i - t0] = s;
        place[i - t0] = q.length - q.count + (i - q.first);
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < nt) {
    const int s = sequence[threadIdx.x], p = place[threadIdx.x];
    int64_t at = -1;
    if (s >= 0 && p >= 0 && p < a.batch.capacity) {
      const int b = FastDiv(a.block_div, p);
      const int id = a.batch.tables[s * a.batch.table_stride + b];
      if (id >= 0 && id < a.batch.num_blocks) {
        const int slot = p - b * a.batch.block_tokens;
        if constexpr (FP4) {
          at = static_cast<int64_t>(id) * a.heads * a.batch.block_tokens + slot;
        } else {
          at = (static_cast<int64_t>(id) * a.batch.block_tokens + slot) * a.heads * a.head_dim;
        }
      }
    }
    row_at[threadIdx.x] = at;
  }
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int ti = i / pairs;
    if (sequence[ti] >= 0) {
      cs[i] = Turn(RotationPosition(a, t0 + ti, place[ti]), a.inv_freq[i - ti * pairs]);
    }
  }
  __syncthreads();
  for (; t < nt; t += token_step) {
    const Factors<E, VEC, LPR> f(lane, cs + t * pairs, weights);
    const int64_t at = row_at[t];
    for (int h = first; h < a.heads;) {
      const int64_t to = at + h * (FP4 ? a.batch.block_tokens : a.head_dim);
      const Row<E, VEC, LPR> row(lane, keys, f, a.k_weight != nullptr, a.eps);
      if constexpr (FP4) {
        const int64_t codes = to * (a.head_dim / 2), scales = to * (a.head_dim / kFp4Group);
        using Q = Fp4Row<E, VEC, LPR>;
        Q::Store(lane, row.x, at >= 0, static_cast<uint8_t*>(a.k_pool) + codes,
                 static_cast<uint8_t*>(a.k_scales) + scales);
        Q::Store(lane, Row<E, VEC, LPR>(values).x, at >= 0,
                 static_cast<uint8_t*>(a.v_pool) + codes,
                 static_cast<uint8_t*>(a.v_scales) + scales);
      } else if (at >= 0) {
        row.Store(lane, static_cast<Scalar*>(a.k_pool) + to);
        values.Store(lane, static_cast<Scalar*>(a.v_pool) + to);
      }
      h += step;
      load(t, h);
    }
    if (t + token_step < nt) load(t + token_step, first);
  }
}

// The new rows of one block.
struct BlockRows {
  int id;      // the block
  int token;   // first new token in it
  int count;   // new tokens in it
  int place;   // position of the first
  int slot;    // its slot: the block holds as many earlier tokens
};

template <class E, int VEC, int LPR>
struct E4m3Row {
  using Lane = RowLane<E, VEC, LPR>;
  static __device__ __forceinline__ void Clamp(float* y) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      y[j] = y[j] > kE4m3Max ? kE4m3Max : y[j] < -kE4m3Max ? -kE4m3Max : y[j];  // NaN stays
    }
  }
  static __device__ __forceinline__ void Store(uint8_t* p, const float* y) {
    if constexpr (VEC == 8) {
      u32x2 w = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        int q = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j], y[4 * j + 1], 0, false);
        q = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2], y[4 * j + 3], q, true);
        w[j] = static_cast<uint32_t>(q);
      }
      *reinterpret_cast<u32x2*>(p) = w;
    } else {
      *p = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[0], 0, false));
    }
  }
  static __device__ __forceinline__ void Load(const uint8_t* p, float* y) {
    if constexpr (VEC == 8) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[j]), false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[j]), true);
        y[4 * j] = lo[0];
        y[4 * j + 1] = lo[1];
        y[4 * j + 2] = hi[0];
        y[4 * j + 3] = hi[1];
      }
    } else {
      y[0] = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(*p), false)[0];
    }
  }
};

constexpr int kHeld = 8;  // rows of one head that a lane holds

template <class E, int VEC, int LPR>
__global__ __launch_bounds__(kThreads, 2) void append_e4m3_kernel(const AppendLaunch a) {
  extern __shared__ f32x2 cs[];  // [kRows][rotary_dim / 2], then amax [heads]
  __shared__ int counted[kWaves];
  __shared__ BlockRows found;
  using Scalar = typename E::Scalar;
  using Q = E4m3Row<E, VEC, LPR>;
  constexpr int kWaveRows = 64 / LPR, kRows = kHeld * kWaveRows;
  const int pairs = a.rotary_dim / 2;
  float* amax = reinterpret_cast<float*>(cs + kRows * pairs);
  const BatchView& b = a.batch;
  const int threads = blockDim.x;  // a wave a head, up to kWaves
  const int wave = threadIdx.x / 64, in_wave = threadIdx.x % 64;

  // The block: the blockIdx.x-th of those that the sequences touch, in order.
  // Sums stop at the grid's size, so that one sequence at most has it.
  if (threadIdx.x == 0) found.id = -1;
  const auto add = [](int x, int y) { return AddUpTo(x, y, static_cast<int>(gridDim.x)); };
  const auto touched = [&](const SequenceSpan& q, int& lo, int& hi) {
    lo = max(q.length - q.count, 0);
    hi = min(q.length, b.capacity);
    if (q.count == 0 || hi <= lo) return 0;
    return FastDiv(a.block_div, hi - 1) - FastDiv(a.block_div, lo) + 1;
  };
  int before = 0;  // blocks of the sequences before this thread's
  const int each = (b.sequences + threads - 1) / threads;
  const int s0 = threadIdx.x * each, s1 = min(s0 + each, b.sequences);
  if (b.starts != nullptr) {
    int mine = 0, lo, hi;
    for (int s = s0; s < s1; ++s) mine = add(mine, touched(LoadSequence(b, s), lo, hi));
    int sum = mine;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const int o = __shfl_up(sum, m);
      if (in_wave >= m) sum = add(sum, o);
    }
    if (in_wave == 63) counted[wave] = sum;
    // What the lanes before this one have.
    before = __shfl_up(sum, 1);
    if (in_wave == 0) before = 0;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before = add(before, counted[w]);
  } else {
    before = s0;  // one token, so one block, a sequence
    __syncthreads();
  }
  for (int s = s0; s < s1; ++s) {
    if (b.starts == nullptr && s != static_cast<int>(blockIdx.x)) continue;
    int lo, hi;
    const SequenceSpan q = LoadSequence(b, s);
    const int n = touched(q, lo, hi), j = static_cast<int>(blockIdx.x) - (b.starts ? before : s);
    if (j >= 0 && j < n) {
      const int at = FastDiv(a.block_div, lo) + j, from = at * b.block_tokens;
      found.place = max(lo, from);
      found.slot = found.place - from;
      found.count = min(hi, from + b.block_tokens) - found.place;
      found.token = q.first + found.place - (q.length - q.count);
      const int id = b.tables[s * b.table_stride + at];
      found.id = id < b.num_blocks ? id : -1;
    }
    before = add(before, n);
  }
  for (int h = threadIdx.x; h < a.heads; h += threads) amax[h] = 0.0f;
  __syncthreads();
  const BlockRows rows = found;
  if (rows.id < 0) return;

  const bool key = blockIdx.y == 0;
  const Scalar* in = static_cast<const Scalar*>(key ? a.k : a.v);
  const int64_t token_stride = key ? a.k_token : a.v_token;
  const int64_t head_stride = key ? a.k_head : a.v_head;
  const int64_t slot_bytes = static_cast<int64_t>(a.heads) * a.head_dim;
  uint8_t* block = static_cast<uint8_t*>(key ? a.k_pool : a.v_pool) +
                   rows.id * (slot_bytes * b.block_tokens);
  float* scales = static_cast<float*>(key ? a.k_scales : a.v_scales) +
                  static_cast<int64_t>(rows.id) * a.heads;
  const RowLane<E, VEC, LPR> lane(a.head_dim, a.rotary_dim, a.interleaved);
  Weights<E, VEC, LPR> weights;
  weights.Load(lane, key ? a.k_weight : nullptr, a.weight_f32);
  const int heads_step = threads / 64 * gridDim.z;

  // One head of a chunk of rows, held.
  const auto one_head = [&](auto held_rows, int pass, bool at_once, int c0, int nc, int h) {
    constexpr int held = decltype(held_rows)::value;
    // Row i of the chunk: lane group i % kWaveRows, register i / kWaveRows.
    // Every lane takes part in the rows' sums; those behind the last row
    // repeat it.
    RawRow<E, VEC, LPR> raw[held];
#pragma unroll
    for (int n = 0; n < held; ++n) {
      const int i = min(n * kWaveRows + in_wave / LPR, nc - 1);
      raw[n].Load(lane, in + (rows.token + c0 + i) * token_stride + h * head_stride, key);
    }
    float x[held][lane.kChunks][VEC];
    float largest = 0.0f;
#pragma unroll
    for (int n = 0; n < held; ++n) {
      const auto keep = [&](const Row<E, VEC, LPR>& row) {
#pragma unroll
        for (int m = 0; m < lane.kChunks; ++m) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            x[n][m][j] = row.x[m][j];
            largest = fmaxf(largest, fabsf(row.x[m][j]));
          }
        }
      };
      if (key) {
        const int i = min(n * kWaveRows + in_wave / LPR, nc - 1);
        const Factors<E, VEC, LPR> f(lane, cs + i * pairs, weights);
        keep(Row<E, VEC, LPR>(lane, raw[n], f, a.k_weight != nullptr, a.eps));
      } else {
        keep(Row<E, VEC, LPR>(raw[n]));
      }
    }
    // Infinities are no part of the largest value, and are clamped.
    const bool endless = __any(largest == __builtin_inff());
    if (endless) {
      largest = 0.0f;
#pragma unroll
      for (int n = 0; n < held; ++n) {
#pragma unroll
        for (int m = 0; m < lane.kChunks; ++m) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float size = fabsf(x[n][m][j]);
            largest = fmaxf(largest, size < __builtin_inff() ? size : 0.0f);
          }
        }
      }
    }
    if (pass == 0 || at_once) {
#pragma unroll
      for (int m = 32; m > 0; m /= 2) largest = fmaxf(largest, __shfl_xor(largest, m));
    }
    if (pass == 0) {
      if (in_wave == 0) amax[h] = fmaxf(amax[h], largest);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      return;
    }
    // The scale: found with the first rows, and kept in LDS for later ones as
    // the largest value that it comes from, or as minus the scale that stays.
    float from;
    if (c0 == 0) {
      float old = rows.slot > 0 ? scales[h] : 0.0f;
      old = old > 0.0f ? old : 0.0f;
      if (!at_once) largest = amax[h];
      const float wanted = largest / kE4m3Max;
      const float scale = fmaxf(old, wanted);
      const bool grown = scale > old;
      if (grown && rows.slot > 0) {
        const float ratio = old / scale;
        for (int i = in_wave / LPR; i < rows.slot; i += kWaveRows) {
          uint8_t* p = block + i * slot_bytes + h * a.head_dim;
#pragma unroll
          for (int n = 0; n < lane.kChunks; ++n) {
            if (!lane.Has(n)) continue;
            float y[VEC];
            Q::Load(p + lane.Dim(n), y);
#pragma unroll
            for (int j = 0; j < VEC; ++j) y[j] *= ratio;
            Q::Store(p + lane.Dim(n), y);
          }
        }
      }
      // (Also where the scale already is what these rows want: the same call
      // on its own result stores the same codes.)
      from = wanted >= old ? largest : -old;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (in_wave == 0) {
        scales[h] = scale;
        amax[h] = from;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else {
      from = amax[h];
    }
    // q = x / scale. A scale that comes from a largest value has been rounded,
    // and rows of few bits often meet the middle between two codes, where that
    // rounding would decide: their quotient is 0.875 x / (largest / 512), both
    // exact, by its remainder.
    const float part = from > 0.0f ? 0.875f : 1.0f;
    const float whole = from > 0.0f ? from * (1.0f / 512) : -from;
    const float inverse = whole > 0.0f ? fminf(1.0f / whole, 3.0e38f) : 0.0f;
    // Infinities, and quotients that are not normal numbers throughout.
    const bool clamp = endless || whole < 1.0e-30f;
#pragma unroll
    for (int n = 0; n < held; ++n) {
      const int i = n * kWaveRows + in_wave / LPR;
      if (i >= nc) continue;
      uint8_t* p = block + (rows.slot + c0 + i) * slot_bytes + h * a.head_dim;
#pragma unroll
      for (int m = 0; m < lane.kChunks; ++m) {
        if (!lane.Has(m)) continue;
        float y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = part * x[n][m][j] * inverse;
        if (clamp) {
          // A scale of 0 belongs to zeros, infinities and NaN, which stay.
          if (whole <= 0.0f) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) y[j] = x[n][m][j];
          }
          Q::Clamp(y);
        } else {
          // The quotient itself, by its remainder: bf16 rows often meet the
          // middle between two codes, where the product's error decides.
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            y[j] = __builtin_fmaf(__builtin_fmaf(-y[j], whole, part * x[n][m][j]), inverse, y[j]);
          }
        }
        Q::Store(p + lane.Dim(m), y);
      }
    }
  };

  // Passes: one that finds the largest values, one that stores; in one go where
  // the new rows fit a wave's registers.
  const bool at_once = rows.count <= kRows;
  for (int pass = at_once ? 1 : 0; pass < 2; ++pass) {
    for (int c0 = 0; c0 < rows.count; c0 += kRows) {
      const int nc = min(kRows, rows.count - c0);
      if (key && pairs > 0) {
        __syncthreads();
        for (int i = threadIdx.x; i < nc * pairs; i += threads) {
          const int ti = i / pairs;
          cs[i] = Turn(RotationPosition(a, rows.token + c0 + ti, rows.place + c0 + ti),
                       a.inv_freq[i - ti * pairs]);
        }
        __syncthreads();
      }
      for (int h = blockIdx.z * (threads / 64) + wave; h < a.heads; h += heads_step) {
        if (nc <= kWaveRows) {
          one_head(std::integral_constant<int, 1>{}, pass, at_once, c0, nc, h);
        } else {
          one_head(std::integral_constant<int, kHeld>{}, pass, at_once, c0, nc, h);
        }
      }
    }
  }
}

template <class E, int VEC, int LPR>
hipError_t Launch(const AppendLaunch& l, hipStream_t stream) {
  const size_t pairs = static_cast<size_t>(l.rotary_dim / 2) * sizeof(f32x2);
  const int tokens = l.batch.tokens;
  if (l.pool == kPoolE4m3) {
    const int64_t blocks = MostBlocks(l);
    // Few blocks: their heads spread over workgroups.
    int split = 1;
    const int waves = BlockThreads(l) / 64;
    while (split * waves < l.heads && blocks * 2 * split < 1024) ++split;
    const dim3 grid(static_cast<unsigned>(blocks), 2, split);
    const size_t lds = kHeld * (64 / LPR) * pairs +
                       static_cast<size_t>(l.heads) * sizeof(float);
    hipLaunchKernelGGL((append_e4m3_kernel<E, VEC, LPR>), grid, dim3(waves * 64), lds, stream, l);
    return hipGetLastError();
  }
  const int of_token = TeamsOfToken(l.heads, LPR);
  int each = kThreads / LPR / of_token, split = 1;
  while (each < kMaxTokens && tokens / each >= 2 * kEnough) each *= 2;
  while (split * of_token < l.heads && static_cast<int64_t>(tokens) * split < 2048) ++split;
  const dim3 grid((tokens + each - 1) / each, split);
  constexpr auto same = append_kv_kernel<E, VEC, LPR, false>, fp4 = append_kv_kernel<E, VEC, LPR, true>;
  hipLaunchKernelGGL(l.pool == kPoolFp4 ? fp4 : same, grid, dim3(kThreads), each * pairs, stream, l,
                     each, of_token);
  return hipGetLastError();
}

template <class E>
hipError_t Pick(const AppendLaunch& l, hipStream_t stream) {
  const auto at = [](const void* p) { return reinterpret_cast<uint64_t>(p); };
  if ((at(l.k) | at(l.v)) % 16 == 0 && (at(l.k_pool) | at(l.v_pool)) % 16 == 0 &&
      (l.k_token | l.k_head | l.v_token | l.v_head) % 8 == 0 &&
      ChunksFit(8, l.head_dim, l.rotary_dim, l.interleaved)) {
    const int chunks = l.head_dim / 8;
    if (chunks <= 8) return Launch<E, 8, 8>(l, stream);
    if (chunks <= 16) return Launch<E, 8, 16>(l, stream);
    return Launch<E, 8, 32>(l, stream);
  }
  return Launch<E, 1, 64>(l, stream);
}

}  // namespace

hipError_t LaunchAppendKv(const AppendLaunch& l, hipStream_t stream) {
  return l.type == kBf16 ? Pick<Bf16>(l, stream) : Pick<F16>(l, stream);
}

}  // namespace kvx
