// The attention that each cached token got, added to a table of what it got before:
//   w_j = decay w_j + sum over the rows of its key head that see it of
//         e^{scale q.k_j - lse},
// w_j = 0 before where the token is one of the call's own or has not been weighed yet.
// lse is what attention returns for the row, so that the exponentials of a row add up to
// 1. Everything after the product is fp32.
//
// Tokens take the place of the output's columns, S = Q K^T, so a lane holds one
// token's scores against several rows: the sum over rows stays in the lane but for
// swaps at the end, and every token is added up by one wave in a fixed order, or from
// such parts in order.
//
// weigh_few (up to kFewRows rows a key head): as attend_few a wave takes an equal part
// of the axis of all sequences' steps of 32 tokens; keys go from memory straight into
// operands. Reading them bounds it: 64 sequences of 65 to 8192 tokens, 32 heads on 8, D =
// 128, bf16: 126 us for 565 MB (4.5 TB/s; 121 us without the table's scattered writes; a
// kernel that only reads such rows 95 us). 8 heads on one of a 4-bit pool, 128
// sequences of 300 to 16384: 21.5 us for 79 MB, of which 20 are left when all tokens come
// from the L2: the start of a wave and its 8 steps. Two steps of keys on their way instead
// of one: 124 and 21.9 us, and short sequences slower. The first of these batches over an
// e4m3 pool 74 us for 291 MB, over a 4-bit one 46 us for 163.
//
// weigh_many (chunks): a workgroup takes WeighTile tokens of one sequence and key
// head, keeps their keys in registers and goes through the rows that see them, 64 at a
// time in LDS. The products and the exponentials (16 a lane for 8 products at D = 128)
// bound it. Tiles' stages of 64 rows make one axis that is cut into equal parts, one a
// workgroup; sums of tiles that a cut goes through are joined in order. 2051 new tokens
// of 3 sequences of 2500 to 7700, 32 heads on 8, D = 128: 101 us with the join (6 us),
// 600 TFLOP/s; whole tiles of 128 tokens handed out in turn 158 us, cut into parts 117
// us, 64 tokens a wave instead of 32 (half of the LDS reads) 109 us with a launch of its
// own for few rows. Over an e4m3 or a 4-bit pool 103 and 104 us. Over 36000 tokens 808
// TFLOP/s. One workgroup more a CU with 32 tokens a wave: 712; a wave's products beside the
// exponentials of its last 32 rows, 253 registers: 765.
#include "weigh.h"

#include <algorithm>

#include "attend_many.h"
#include "pool_lane.h"

namespace kvx {
namespace {

// Workgroups of a CU with few rows.
constexpr int WeighFewGroups(int padded_dim, int row_tiles, bool full) {
  return padded_dim > 128 ? 1 : row_tiles == 1 && full ? 4 : 2;
}

struct WeighKeys {
  SequenceSpan q;
  int rows, begin, end;
  int held;  // tokens that hold a weight
};

__device__ __forceinline__ WeighKeys LoadWeighKeys(const WeighLaunch& w, int s) {
  WeighKeys k;
  k.q = LoadSequence(w.attend.batch, s);
  k.rows = k.q.count * (w.attend.q_heads / w.attend.k_heads);
  k.end = min(k.q.length, w.attend.batch.capacity);
  k.begin = w.begins != nullptr ? min(max(w.begins[s], 0), k.end) : 0;
  k.held = k.q.length - k.q.count;
  if (w.weighed != nullptr) k.held = min(k.held, w.weighed[s]);
  return k;
}

__device__ __forceinline__ float Plus16(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) +
         __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}
__device__ __forceinline__ float Plus32(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) +
         __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}

// -- Few rows.

__device__ __forceinline__ int WeighSteps(const WeighKeys& k) {
  if (k.rows == 0 || k.rows > kFewRows) return 0;
  return (k.end - k.begin + kFewStep - 1) / kFewStep;
}

// `group`: number of the workgroup; sums: [sequences] in LDS.
template <class E, int POOL, int DP, int RT, bool FULL>
__device__ __forceinline__ void WeighFew(const WeighLaunch& w, int* sums, int group) {
  using Scalar = typename E::Scalar;
  using Pool = PoolLane<E, POOL, DP, FULL>;
  using Words = typename Pool::Words;
  constexpr bool E4 = POOL == kPoolE4m3, F4 = POOL == kPoolFp4;
  constexpr int KS = Pool::KS, kCodes = F4 ? Pool::kScales : 1;
  const AttendLaunch& a = w.attend;
  const BatchView& b = a.batch;
  for (int s = threadIdx.x; s < b.sequences; s += kAttendThreads) {
    sums[s] = WeighSteps(LoadWeighKeys(w, s));
  }
  BlockSums(sums, b.sequences, a.most_few);
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const int all = one(sums[b.sequences - 1]);
  if (all == 0) return;
  const Axis axis = FewAxis(a, all);
  const int lane = threadIdx.x % 64;
  const int worker = group * kWaves + one(threadIdx.x / 64);
  if (worker >= axis.workers) return;
  const int x_end = axis.Start(worker + 1);
  const int in16 = lane % 16, quarter = lane / 16;
  const int G = a.q_heads / a.k_heads;
  const float c = a.scale * kLog2e;

  for (int x = axis.Start(worker); x < x_end;) {
    const int s = one(FirstAbove(sums, b.sequences, x / a.k_heads));
    const int before = s > 0 ? one(sums[s - 1]) : 0;
    const int steps = one(sums[s]) - before;
    const int off = x - before * a.k_heads;
    const int h = off / steps, step0 = off - h * steps;
    const int step1 = min(steps, step0 + (x_end - x));
    const WeighKeys k = LoadWeighKeys(w, s);
    const int begin = one(k.begin), end = one(k.end), rows = one(k.rows);
    const SequenceSpan span = {one(k.q.first), one(k.q.count), one(k.q.length)};
    const int held_end = one(k.held);

    // Queries: row l % 16 of each row tile; and of the rows that this lane gets
    // scores of, 4 (l / 16) + i, the log of their sums and the tokens that they see.
    u32x4 q[RT][KS];
    float base[RT][4];
    int seen[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = rt * 16 + in16, t = FastDivI(a.group_div, r);
      const int64_t token = span.first + t;
      const Scalar* p = static_cast<const Scalar*>(a.q) + token * a.q_token +
                        (h * G + (r - t * G)) * a.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = Pool::DimOf(quarter, ks);
        q[rt][ks] = u32x4{0, 0, 0, 0};
        if (r < rows && (FULL || d < a.head_dim)) {
          q[rt][ks] = *reinterpret_cast<const Bytes16*>(p + d);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = rt * 16 + quarter * 4 + i, at = FastDivI(a.group_div, row);
        base[rt][i] = 0.0f;
        seen[rt][i] = 0;
        if (row < rows) {
          base[rt][i] = w.lse[(span.first + at) * static_cast<int64_t>(a.q_heads) + h * G +
                              (row - at * G)] * kLog2e;
          seen[rt][i] = Visible(a, span, span.first + at);
        }
      }
    }

    const Pool pool(lane, h, a);
    const int32_t* table = b.tables + s * b.table_stride;
    const auto find = [&](int step, int (&id)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = begin + step * kFewStep + u * 16 + in16;
        id[u] = -1;
        if (step < step1 && p < end) id[u] = table[FastDivI(a.block_div, p)];
      }
    };
    int64_t at[2];
    // The weight of the lane's own token: 16 (l / 16) + l % 16 of the step, l < 32. The
    // load needs no branch: what has no weight yet reads some, and does not use it.
    int64_t mine = 0;
    bool writes = false, adds = false;
    float held = 0.0f;
    const auto place = [&](int step, const int (&id)[2]) {
      int64_t to[2];
      bool has[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = begin + step * kFewStep + u * 16 + in16;
        const int slot = p - FastDivI(a.block_div, p) * b.block_tokens;
        has[u] = id[u] >= 0 && id[u] < b.num_blocks;
        at[u] = pool.At(id[u], slot, has[u]);
        to[u] = has[u] ? (static_cast<int64_t>(id[u]) * a.k_heads + h) * b.block_tokens + slot : 0;
      }
      mine = quarter == 1 ? to[1] : to[0];
      writes = quarter < 2 && (quarter == 1 ? has[1] : has[0]);
      adds = w.decay != 0.0f && begin + step * kFewStep + quarter * 16 + in16 < held_end;
      held = w.weights[mine];
    };
    Words kw[2][KS];
    float kf[2] = {1, 1};
    [[maybe_unused]] uint32_t kc[2][kCodes];
    int id[2], id_now[2];
    const auto load = [&](const int (&of)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        pool.Load(a.k_pool, at[u], kw[u]);
        if constexpr (E4) {
          const bool has = of[u] >= 0 && of[u] < b.num_blocks;
          kf[u] = static_cast<const float*>(
              a.k_scales)[(has ? static_cast<int64_t>(of[u]) : 0) * a.k_heads + h];
        }
        if constexpr (F4) pool.LoadScales(a.k_scales, at[u], kc[u]);
      }
    };
    find(step0, id_now);
    find(step0 + 1, id);
    place(step0, id_now);
    load(id_now);
    for (int step = step0; step < step1; ++step) {
      const int p0 = begin + step * kFewStep;
      f32x4 sc[RT][2];
      float factor[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        factor[u] = E4 ? c * kf[u] : c;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt][u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 key;
          if constexpr (E4) {
            key = Widen<E>(kw[u][ks]);
          } else if constexpr (F4) {
            key = pool.FromCodes(kw[u][ks], kc[u], ks);
          } else {
            key = kw[u][ks];
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt][u] = Mma16<E>(q[rt][ks], key, sc[rt][u]);
        }
      }
      const int64_t to = mine;
      const bool writes_now = writes;
      const float was = adds ? held : 0.0f;
      id_now[0] = id[0];
      id_now[1] = id[1];
      place(step + 1, id_now);
      find(step + 2, id);
      load(id_now);
      float got[2] = {0, 0};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = p0 + u * 16 + in16;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(fmaf(sc[rt][u][i], factor[u], -base[rt][i]));
            got[u] += p < seen[rt][i] ? e : 0.0f;
          }
        }
        got[u] = Plus32(Plus16(got[u]));
      }
      if (writes_now) w.weights[to] = fmaf(w.decay, was, quarter == 0 ? got[0] : got[1]);
    }
    x += step1 - step0;
  }
}

// -- Many rows: tiles of WeighTile tokens of the sequences with more than kFewRows rows,
// each of as many stages of kWeighRows rows as see it.

struct WeighUnit {
  int rows;
  int begin, end;  // tokens
  int old_end;     // tokens that are not the call's own
  int held;        // tokens that hold a weight
  int tiles;
  // Tiles that all rows see, of `stages` each; the others have `less` stages less each
  // than the one before, the first of them `later`.
  int full, stages, later, less;
};

__device__ __forceinline__ WeighUnit LoadWeighUnit(const WeighLaunch& w, int s) {
  const WeighKeys k = LoadWeighKeys(w, s);
  const int G = w.attend.q_heads / w.attend.k_heads, tile = WeighTile(w.attend.padded_dim);
  WeighUnit u;
  u.less = tile / kWeighRows * G;
  u.rows = k.rows;
  u.begin = k.begin;
  u.end = k.end;
  u.old_end = k.q.length - k.q.count;
  u.held = k.held;
  u.tiles = k.rows > kFewRows ? (k.end - k.begin + tile - 1) / tile : 0;
  u.stages = (k.rows + kWeighRows - 1) / kWeighRows;
  u.full = u.tiles;
  u.later = 0;
  if (w.attend.causal) {
    u.full = u.old_end < u.begin ? 0 : min((u.old_end - u.begin) / tile + 1, u.tiles);
    // The first token of the next tile is so many behind the first of the call's own.
    const int behind = u.begin + u.full * tile - u.old_end;
    u.later = u.full < u.tiles ? u.stages - behind * G / kWeighRows : 0;
  }
  return u;
}

// Where tile i starts on its sequence's and head's axis.
__device__ __forceinline__ int WeighCost(const WeighUnit& u, int i) {
  if (i <= u.full) return i * u.stages;
  const int n = i - u.full;
  return u.full * u.stages + n * u.later - n * (n - 1) / 2 * u.less;
}

// The tile that holds `at`.
__device__ __forceinline__ int WeighTileAt(const WeighUnit& u, int at) {
  if (at < u.full * u.stages) return at / u.stages;
  int tile = u.full, tiles = u.tiles;
  while (tiles - tile > 1) {
    const int mid = (tile + tiles) / 2;
    if (WeighCost(u, mid) <= at) {
      tile = mid;
    } else {
      tiles = mid;
    }
  }
  return tile;
}

// Sums of all sequences' costs into LDS.
__device__ __forceinline__ void WeighSums(const WeighLaunch& w, int* sums) {
  for (int s = threadIdx.x; s < w.attend.batch.sequences; s += kAttendThreads) {
    const WeighUnit u = LoadWeighUnit(w, s);
    sums[s] = WeighCost(u, u.tiles);
  }
  BlockSums(sums, w.attend.batch.sequences, w.attend.most_many);
}

__device__ __forceinline__ Axis WeighAxis(const WeighLaunch& w, int work) {
  return Axis(work * w.attend.k_heads, w.attend.many_grid);
}

constexpr int kAhead = 4;  // products that operands are read ahead
constexpr int WeighGroups(int padded_dim) { return padded_dim <= 64 ? 3 : 2; }  // of a CU

template <class E, int POOL, int DP>
__device__ __forceinline__ void WeighMany(const WeighLaunch& w, char* lds, int place) {
  using Scalar = typename E::Scalar;
  constexpr bool E4 = POOL == kPoolE4m3, F4 = POOL == kPoolFp4;
  constexpr int KS = DP / 16, kRow = 2 * DP, kTile = WeighTile(DP);
  constexpr int CT = kTile / 128;    // 32s of tokens of a wave
  constexpr int kChunks = DP / 32;  // of a thread: every fourth of a row
  static_assert(kWeighRows * 4 == kAttendThreads);
  struct Rows {
    float base[kWeighRows];
    int seen[kWeighRows];
  };
  Rows* row_data = reinterpret_cast<Rows*>(lds + 2 * kWeighRows * kRow);
  int* sums = reinterpret_cast<int*>(row_data + 2);  // [sequences]
  const AttendLaunch& a = w.attend;
  const BatchView& b = a.batch;
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  WeighSums(w, sums);
  const int work = one(sums[b.sequences - 1]);
  if (work == 0) return;
  const Axis axis = WeighAxis(w, work);
  // The workgroups of one XCD take neighbouring parts, so its L2 serves a head's rows to
  // all of them.
  const int worker = WorkerAt(place, axis.workers);
  if (worker < 0) return;
  const int x_end = axis.Start(worker + 1);
  const int lane = threadIdx.x % 64, wave = one(threadIdx.x / 64);
  const int in32 = lane % 32, half = lane / 32;
  const int G = a.q_heads / a.k_heads;
  const float c = a.scale * kLog2e;
  // Where the lane's part of a row's operands is in a stage.
  int row_at[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    row_at[ks] = in32 * kRow + KeyChunk<DP>(in32, ks * 2 + half) * 16;
  }

  for (int x = axis.Start(worker); x < x_end;) {
    const int s = one(FirstAbove(sums, b.sequences, x / a.k_heads));
    const int before = s > 0 ? one(sums[s - 1]) : 0;
    const int per_head = one(sums[s]) - before;
    const int h = (x - before * a.k_heads) / per_head;
    const int at_unit = x - before * a.k_heads - h * per_head;
    const WeighUnit u = LoadWeighUnit(w, s);
    const int tile = one(WeighTileAt(u, at_unit));
    const int tile_at = one(WeighCost(u, tile));
    const int stages = one(WeighCost(u, tile + 1)) - tile_at;
    // The part's stages: the last of them end with the last row.
    const int stage0 = at_unit - tile_at, stage1 = min(stages, stage0 + (x_end - x));
    const int end = one(u.end), held_end = one(u.held);
    const int row0 = (one(u.stages) - stages + stage0) * kWeighRows;
    const int rows = min(one(u.rows), row0 + (stage1 - stage0) * kWeighRows);
    const SequenceSpan span = LoadSequence(b, s);
    const int j0 = one(u.begin) + tile * kTile + wave * (CT * 32);  // the wave's

    // Keys: token l % 32 of each of the wave's 32s, as an operand.
    u32x4 key[CT][KS];
    float factor[CT];
    float* mine[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int p = j0 + ct * 32 + in32;
      const int at = FastDivI(a.block_div, p), slot = p - at * b.block_tokens;
      const int id = p < end ? b.tables[s * b.table_stride + at] : -1;
      const bool has = id >= 0 && id < b.num_blocks;
      const int64_t of_block = static_cast<int64_t>(has ? id : 0);
      // Places in layouts with a head's tokens together, and with a token's heads.
      const int64_t by_head = (of_block * a.k_heads + h) * b.block_tokens + (has ? slot : 0);
      const int64_t by_token = (of_block * b.block_tokens + (has ? slot : 0)) * a.k_heads + h;
      mine[ct] = has ? w.weights + by_head : nullptr;
      factor[ct] = c;
      if constexpr (E4) {
        factor[ct] *= static_cast<const float*>(a.k_scales)[of_block * a.k_heads + h];
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = ks * 16 + half * 8;
        key[ct][ks] = u32x4{0, 0, 0, 0};
        if (!has || d >= a.head_dim) continue;
        if constexpr (F4) {
          const uint32_t code = static_cast<const uint8_t*>(
              a.k_scales)[by_head * (a.head_dim / kFp4Group) + d / kFp4Group];
          key[ct][ks] = FromFp4<E>(
              *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.k_pool) +
                                                 by_head * (a.head_dim / 2) + d / 2),
              Fp4Scale<E>(code));
        } else if constexpr (E4) {
          key[ct][ks] = Widen<E>(*reinterpret_cast<const Bytes8*>(
              static_cast<const uint8_t*>(a.k_pool) + by_token * a.head_dim + d));
        } else {
          key[ct][ks] = *reinterpret_cast<const Bytes16*>(static_cast<const Scalar*>(a.k_pool) +
                                                          by_token * a.head_dim + d);
        }
      }
    }

    // Four threads load a row of every stage, and step from one to the next without a
    // division.
    const int step_tokens = kWeighRows / G, step_heads = kWeighRows - step_tokens * G;
    const int my_row = threadIdx.x / 4, my_chunk = threadIdx.x % 4;
    int t = FastDivI(a.group_div, row0 + my_row), of_token = row0 + my_row - t * G;
    const Scalar* from = static_cast<const Scalar*>(a.q) +
                         static_cast<int64_t>(span.first + t) * a.q_token +
                         (h * G + of_token) * a.q_head + my_chunk * 8;
    u32x4 hold[kChunks];
    float hold_base = 0.0f;
    int hold_seen = 0;
    const auto load = [&](int r0) {
      const bool has = r0 + my_row < rows;
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        hold[n] = u32x4{0, 0, 0, 0};
        if (has && (my_chunk + n * 4) * 8 < a.head_dim) {
          hold[n] = *reinterpret_cast<const Bytes16*>(from + n * 32);
        }
      }
      hold_base = 0.0f;
      hold_seen = 0;
      if (has && my_chunk == 0) {
        hold_base = w.lse[(span.first + t) * static_cast<int64_t>(a.q_heads) + h * G + of_token] *
                    kLog2e;
        hold_seen = Visible(a, span, span.first + t);
      }
      t += step_tokens;
      of_token += step_heads;
      from += step_tokens * a.q_token + step_heads * a.q_head;
      if (of_token >= G) {  // from a token's heads to the next one's
        ++t;
        of_token -= G;
        from += a.q_token - G * a.q_head;
      }
    };
    const auto store = [&](auto buffer) {
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        *reinterpret_cast<u32x4*>(lds + buffer() * (kWeighRows * kRow) + my_row * kRow +
                                  KeyChunk<DP>(my_row, my_chunk + n * 4) * 16) = hold[n];
      }
      if (my_chunk == 0) {
        row_data[buffer()].base[my_row] = hold_base;
        row_data[buffer()].seen[my_row] = hold_seen;
      }
    };

    float got[CT] = {};
    // The last token of the wave that counts: rows that see it see all of them.
    const int last = min(j0 + CT * 32, end);
    // 32 rows of a stage. Lane: token l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4.
    const auto tile_of = [&](auto buffer, int rt, bool plain) {
      const char* at = lds + buffer() * (kWeighRows * kRow) + rt * 32 * kRow;
      const Rows& here = row_data[buffer()];
      const int r = rt * 32 + half * 4;
      f32x16 sc[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) sc[ct] = f32x16(0.0f);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 row = *reinterpret_cast<const u32x4*>(at + row_at[ks]);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sc[ct] = Mma32<E>(row, key[ct][ks], sc[ct]);
      }
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 base = *reinterpret_cast<const f32x4*>(&here.base[r + i * 2]);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sc[ct][i + j] = __builtin_amdgcn_exp2f(fmaf(sc[ct][i + j], factor[ct], -base[j]));
          }
        }
      }
      // Operands are read ahead of their products.
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int n = 0; n < KS; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x8, CT, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      if (!plain) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int seen = here.seen[r + i / 4 * 8 + i % 4];
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            if (j0 + ct * 32 + in32 >= seen) sc[ct][i] = 0.0f;
          }
        }
      }
      // Sums of 16 first: thousands of rows lose less so.
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float some[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          some[j] = (sc[ct][j] + sc[ct][4 + j]) + (sc[ct][8 + j] + sc[ct][12 + j]);
        }
        got[ct] += (some[0] + some[1]) + (some[2] + some[3]);
      }
    };
    const auto stage = [&](int r0, auto buffer) {
      store(buffer);
      __syncthreads();
      if (r0 + kWeighRows < rows) load(r0 + kWeighRows);
      const bool plain = r0 + kWeighRows <= rows &&
                         Visible(a, span, span.first + FastDivI(a.group_div, r0)) >= last;
#pragma unroll
      for (int rt = 0; rt < kWeighRows / 32; ++rt) tile_of(buffer, rt, plain);
    };
    load(row0);
    // (A buffer's readers are past the barrier of the stage in between.)
    for (int r0 = row0; r0 < rows; r0 += 2 * kWeighRows) {
      stage(r0, std::integral_constant<int, 0>{});
      if (r0 + kWeighRows < rows) stage(r0 + kWeighRows, std::integral_constant<int, 1>{});
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float sum = Plus32(got[ct]);
      if (half != 0) continue;
      if (stage0 > 0 || stage1 < stages) {
        w.parts[axis.Slot(worker, x) * kTile + (wave * CT + ct) * 32 + in32] = sum;
      } else if (mine[ct] != nullptr) {
        const float was =
            j0 + ct * 32 + in32 < held_end && w.decay != 0.0f ? *mine[ct] : 0.0f;
        *mine[ct] = fmaf(w.decay, was, sum);
      }
    }
    x += stage1 - stage0;
    __syncthreads();  // the next tile's rows take this one's place in LDS
  }
}

// Adds up the parts of tiles that were cut, in order: a workgroup takes the tile that a
// worker's start is in, if it is the first one in it.
__global__ __launch_bounds__(kAttendThreads) void weigh_join_kernel(const WeighLaunch w) {
  extern __shared__ int sums[];  // [sequences]
  const AttendLaunch& a = w.attend;
  const BatchView& b = a.batch;
  WeighSums(w, sums);
  const int work = sums[b.sequences - 1];
  if (work == 0) return;
  const Axis axis = WeighAxis(w, work);
  const int tokens = WeighTile(a.padded_dim), in_tile = threadIdx.x;
  const int cut = static_cast<int>(blockIdx.x) + 1;
  if (cut >= axis.workers || in_tile >= tokens) return;
  const int x = axis.Start(cut);
  const int s = FirstAbove(sums, b.sequences, x / a.k_heads);
  const int before = s > 0 ? sums[s - 1] : 0, per_head = sums[s] - before;
  const int h = (x - before * a.k_heads) / per_head;
  const int unit = before * a.k_heads + h * per_head;
  const WeighUnit u = LoadWeighUnit(w, s);
  const int tile = WeighTileAt(u, x - unit);
  const int first = unit + WeighCost(u, tile), last = unit + WeighCost(u, tile + 1);
  if (x == first || x - axis.each > first) return;
  float sum = 0.0f;
  for (int n = axis.Owner(first); n <= axis.Owner(last - 1); ++n) {
    const int slot = n < cut ? axis.Slot(n, first) : 2 * n;
    sum += w.parts[slot * tokens + in_tile];
  }
  const int p = u.begin + tile * tokens + in_tile;
  if (p >= u.end) return;
  const int at = FastDivI(a.block_div, p), id = b.tables[s * b.table_stride + at];
  if (id < 0 || id >= b.num_blocks) return;
  float* mine = w.weights + (static_cast<int64_t>(id) * a.k_heads + h) * b.block_tokens +
                (p - at * b.block_tokens);
  *mine = fmaf(w.decay, p < u.held && w.decay != 0.0f ? *mine : 0.0f, sum);
}

template <class E, int POOL, int DP, int RT, bool FULL>
__global__ __launch_bounds__(kAttendThreads, WeighFewGroups(DP, RT, FULL)) void weigh_few_kernel(
    const WeighLaunch w) {
  extern __shared__ int sums[];
  WeighFew<E, POOL, DP, RT, FULL>(w, sums, blockIdx.x);
}

// Places that WorkerAt needs for the workers of a grid.
__host__ __device__ inline int Places(int grid) { return (grid + kXcds - 1) / kXcds * kXcds; }

// Chunks, and what few rows there are beside them.
template <class E, int POOL, int DP, bool FULL>
__global__ __launch_bounds__(kAttendThreads, WeighGroups(DP)) void weigh_mixed_kernel(
    const WeighLaunch w) {
  extern __shared__ __align__(16) char lds[];
  const int place = static_cast<int>(blockIdx.x), many = Places(w.attend.many_grid);
  if (place < many) {
    WeighMany<E, POOL, DP>(w, lds, place);
  } else {
    WeighFew<E, POOL, DP, 2, FULL>(w, reinterpret_cast<int*>(lds), place - many);
  }
}

template <class E, int POOL, int DP, int RT, bool FULL>
hipError_t Few(const WeighLaunch& l, hipStream_t stream) {
  const size_t lds = static_cast<size_t>(l.attend.batch.sequences) * sizeof(int);
  hipLaunchKernelGGL((weigh_few_kernel<E, POOL, DP, RT, FULL>), dim3(l.attend.few_grid),
                     dim3(kAttendThreads), lds, stream, l);
  return hipGetLastError();
}

template <class E, int POOL, int DP, bool FULL>
hipError_t Mixed(const WeighLaunch& l, hipStream_t stream) {
  const AttendLaunch& a = l.attend;
  const size_t lds = 2 * kWeighRows * (2 * DP + 8) +
                     static_cast<size_t>(a.batch.sequences) * sizeof(int);
  constexpr auto kernel = weigh_mixed_kernel<E, POOL, DP, FULL>;
  hipError_t e = AllowDynamicLds<kernel>(lds + 1024);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3(Places(a.many_grid) + a.few_grid), dim3(kAttendThreads), lds, stream, l);
  e = hipGetLastError();
  if (e != hipSuccess || a.many_grid == 1) return e;  // one worker cuts nothing
  hipLaunchKernelGGL(weigh_join_kernel, dim3(a.many_grid - 1), dim3(kAttendThreads),
                     static_cast<size_t>(a.batch.sequences) * sizeof(int), stream, l);
  return hipGetLastError();
}

template <class E, int POOL, int DP>
hipError_t Both(const WeighLaunch& l, hipStream_t stream) {
  const AttendLaunch& a = l.attend;
  const bool full = a.head_dim == DP;
  if (a.many_grid > 0) {
    return full ? Mixed<E, POOL, DP, true>(l, stream) : Mixed<E, POOL, DP, false>(l, stream);
  }
  if (!full) return Few<E, POOL, DP, 2, false>(l, stream);
  return a.few_rows <= 16 ? Few<E, POOL, DP, 1, true>(l, stream)
                          : Few<E, POOL, DP, 2, true>(l, stream);
}

template <class E, int POOL>
hipError_t PickDim(const WeighLaunch& l, hipStream_t stream) {
  switch (l.attend.padded_dim) {
    case 64:
      return Both<E, POOL, 64>(l, stream);
    case 96:
      return Both<E, POOL, 96>(l, stream);
    case 128:
      return Both<E, POOL, 128>(l, stream);
    default:
      return Both<E, POOL, 256>(l, stream);
  }
}

template <class E>
hipError_t PickPool(const WeighLaunch& l, hipStream_t stream) {
  switch (l.attend.pool) {
    case kPoolE4m3:
      return PickDim<E, kPoolE4m3>(l, stream);
    case kPoolFp4:
      return PickDim<E, kPoolFp4>(l, stream);
    default:
      return PickDim<E, kPoolSame>(l, stream);
  }
}

}  // namespace

int64_t PlanWeigh(WeighLaunch* l) {
  AttendLaunch& a = l->attend;
  const int64_t G = a.q_heads / a.k_heads, T = a.batch.tokens, S = a.batch.sequences;
  const int64_t capacity = std::max(a.batch.capacity, 1);
  const bool single = a.batch.starts == nullptr;
  a.padded_dim = PaddedDim(a.head_dim);
  constexpr int kCus = 256;
  a.few_grid = a.few_rows = a.many_grid = 0;
  if (G <= kFewRows) {
    a.few_rows = static_cast<int>(single ? G : std::min<int64_t>(T * G, kFewRows));
    const int64_t steps = S * a.k_heads * ((capacity + kFewStep - 1) / kFewStep);
    const int resident = kCus * WeighFewGroups(a.padded_dim, a.few_rows <= 16 ? 1 : 2,
                                               a.head_dim == a.padded_dim);
    a.few_grid = static_cast<int>(std::min<int64_t>(resident, (steps + kWaves - 1) / kWaves));
  }
  if (single ? G > kFewRows : T * G > kFewRows) {
    const int tile = WeighTile(a.padded_dim);
    // Stages of the sequences with more than kFewRows rows (at most T * G / kFewRows).
    const int64_t units = std::min(S, T * G / kFewRows);
    const int64_t stages = (T * G + kWeighRows - 1) / kWeighRows + units;
    const int64_t work = stages * a.k_heads * ((capacity + tile - 1) / tile);
    a.many_grid =
        static_cast<int>(std::min<int64_t>(WeighGroups(a.padded_dim) * kCus, work));
  }
  return 2ll * a.many_grid * WeighTile(a.padded_dim) * static_cast<int64_t>(sizeof(float));
}

hipError_t LaunchWeigh(const WeighLaunch& l, hipStream_t stream) {
  return l.attend.type == kBf16 ? PickPool<Bf16>(l, stream) : PickPool<F16>(l, stream);
}

}  // namespace kvx
