// Paged attention of sequences with few rows a key head: single tokens, a few
// drafted ones.
//
// For rows q of one sequence and key head, over its tokens j in any order:
//   s_j = scale q.k_j,  m = max s_j,  l = sum e^{s_j - m},  o = sum e^{s_j - m} v_j
// in one pass, (m, l, o) rescaled when m grows. Every key and value is read
// once and meets 1 to 32 rows, so the time is that of reading the pool.
//
// Layout. All products are 16 x 16 x 32 matrix instructions with the tokens in
// the place of the output's rows: S^T = K Q^T needs K's rows as they lie in the
// pool (a lane's 16 bytes are 8 dimensions of one token), so keys go from
// memory straight into operands, no LDS. Lane l then holds scores of row l % 16
// and tokens 4 (l / 16).. of each half tile: maxima and sums stay in a lane but
// for two swaps, and the packed exponentials are the operand of O^T = V^T P^T
// as they stand. Only V needs its transpose: it passes through LDS, each wave's
// tile its own, and comes back by transposing reads; no barrier in the loop.
//
// Work. The steps (32 tokens) of all sequences and key heads form one axis, cut
// into equal parts, one a wave: long and short sequences load the GPU alike, and
// no wave waits for another. What a part cuts is at its two ends and goes to
// slots 2w and 2w + 1 of `parts`; what it holds whole goes straight to the
// output, or, where a group's prefix comes on top, to its own row of `parts`.
// 64 sequences of 65 to 8192 tokens, 32 heads on 8, D = 128, bf16: 210 us for 1.09
// GB (5.2 TB/s; 256-byte rows of one head at random 16-token blocks are read at 5.6
// to 6.0 by a kernel that does nothing else), in e4m3 on one key head 46 us for 266
// MB (5.7 TB/s). Three waves a SIMD instead of two: the same, e4m3 4 % slower.
#ifndef KVX_KERNELS_ATTEND_FEW_H_
#define KVX_KERNELS_ATTEND_FEW_H_

#include "attend_plan.h"

namespace kvx {

// Bytes of a token's values in LDS: an odd multiple of 32, so that the rows
// of a transposing read fall on different banks.
constexpr int FewValueStride(int dp) { return dp * 2 + 32; }

constexpr size_t FewLds(const AttendLaunch& l, int dp) {
  return kWaves * 32 * FewValueStride(dp) +
         (l.groups > 0 ? 3 : 2) * sizeof(int) * static_cast<size_t>(l.batch.sequences);
}

template <class E, bool E4, int DP, int RT, bool FULL>
__device__ __forceinline__ void AttendFew(const AttendLaunch& a, char* lds, int workgroup) {
  using Scalar = typename E::Scalar;
  constexpr int KS = DP / 32, DT = DP / 16, VST = FewValueStride(DP);
  // The order in which a product goes through the dimensions is free: a lane
  // takes 16 e4m3 ones in a row for two products where they come in pairs. 128
  // sequences of 8 query heads on one, 300 to 16384 tokens, D = 128: 56 us (4.7
  // TB/s); with 8 in a row 76 us.
  constexpr bool kWide = E4 && FULL && KS % 2 == 0;
  const BatchView& b = a.batch;
  int* sums = reinterpret_cast<int*>(lds + kWaves * 32 * VST);  // [sequences]
  int* lengths = sums + b.sequences;
  int* begins = lengths + b.sequences;  // with groups: 2 * begin + grouped
  for (int s = threadIdx.x; s < b.sequences; s += kAttendThreads) {
    const OwnKeys k = LoadOwnKeys(a, s);
    sums[s] = FewSteps(k);
    lengths[s] = k.q.length;
    if (a.groups > 0) begins[s] = 2 * k.begin + (k.grouped ? 1 : 0);
  }
  BlockSums(sums, b.sequences, a.most_few);
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const int all = one(sums[b.sequences - 1]);
  if (all == 0) return;
  const Axis axis = FewAxis(a, all);
  const int lane = threadIdx.x % 64, wave = one(threadIdx.x / 64);
  const int worker = workgroup * kWaves + wave;
  if (worker >= axis.workers) return;
  const int x_first = axis.Start(worker), x_end = axis.Start(worker + 1);

  const int in16 = lane % 16, quarter = lane / 16;
  const auto dim_of = [&](int ks) {
    return kWide ? ks / 2 * 64 + quarter * 16 + ks % 2 * 8 : ks * 32 + quarter * 8;
  };
  char* mine = lds + wave * 32 * VST;
  const int G = a.q_heads / a.k_heads;
  const int64_t row_stride = static_cast<int64_t>(a.k_heads) * a.head_dim;
  const float c = a.scale * kLog2e;

  for (int x = x_first; x < x_end;) {
    const int s = one(FirstAbove(sums, b.sequences, x / a.k_heads));
    const int before = s > 0 ? one(sums[s - 1]) : 0;
    const int steps = one(sums[s]) - before;
    const int off = x - before * a.k_heads;
    const int h = off / steps, step0 = off - h * steps;
    const int step1 = min(steps, step0 + (x_end - x));
    SequenceSpan span = {s, 1, one(lengths[s])};
    if (b.starts != nullptr) {
      span.first = one(min(max(b.starts[s], 0), b.tokens));
      span.count = one(min(max(b.starts[s + 1], span.first), b.tokens)) - span.first;
    }
    const int rows = span.count * G, end = min(span.length, b.capacity);
    const int word = a.groups > 0 ? one(begins[s]) : 0;
    const int begin = word >> 1;
    const bool grouped = (word & 1) != 0;
    const int seen_by_all = Visible(a, span, span.first);

    // Queries: row l % 16 of each row tile, the dimensions of a key operand.
    u32x4 q[RT][KS];
    int seen[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = rt * 16 + in16, t = FastDivI(a.group_div, r);
      const int64_t token = span.first + t;
      const Scalar* p = static_cast<const Scalar*>(a.q) + token * a.q_token +
                        (h * G + (r - t * G)) * a.q_head;
      seen[rt] = r < rows ? Visible(a, span, span.first + t) : INT_MAX;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[rt][ks] = u32x4{0, 0, 0, 0};
        if (r < rows && (FULL || dim_of(ks) < a.head_dim)) {
          q[rt][ks] = *reinterpret_cast<const Bytes16*>(p + dim_of(ks));
        }
      }
    }

    f32x4 o[RT][DT];
    float top[RT], sum[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      top[rt] = -__builtin_inff();
      sum[rt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0, 0, 0, 0};
    }

    // Tokens of a step: lane l loads token l % 16 of both halves, eight
    // dimensions in each group of 32.
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
    bool has[2];
    const auto place = [&](int step, const int (&id)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = begin + step * kFewStep + u * 16 + in16;
        const int slot = p - FastDivI(a.block_div, p) * b.block_tokens;
        has[u] = id[u] >= 0 && id[u] < b.num_blocks;
        // A token without a place reads the pool's first row (it is masked, and
        // its values are cleared), so that loads need no branch.
        const int64_t row = static_cast<int64_t>(id[u]) * b.block_tokens + slot;
        at[u] = (has[u] ? row : 0) * row_stride + h * a.head_dim + quarter * (kWide ? 16 : 8);
      }
    };
    constexpr int W = E4 ? 2 : 4;
    using Words = __attribute__((ext_vector_type(W))) uint32_t;
    const auto load = [&](const void* pool, Words (&w)[2][KS]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (kWide) {
#pragma unroll
          for (int ks = 0; ks < KS; ks += 2) {
            using Wide = u32x4 __attribute__((aligned(1)));
            const u32x4 x = *reinterpret_cast<const Wide*>(static_cast<const uint8_t*>(pool) +
                                                           at[u] + ks * 32);
            w[u][ks] = Words{x[0], x[1]};
            w[u][ks + 1] = Words{x[2], x[3]};
          }
          continue;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if constexpr (!FULL) w[u][ks] = Words(0);
          if (FULL || ks * 32 + quarter * 8 < a.head_dim) {
            if constexpr (E4) {
              w[u][ks] = *reinterpret_cast<const Bytes8*>(static_cast<const uint8_t*>(pool) +
                                                          at[u] + ks * 32);
            } else {
              w[u][ks] = *reinterpret_cast<const Bytes16*>(static_cast<const Scalar*>(pool) +
                                                           at[u] + ks * 32);
            }
          }
        }
      }
    };
    const auto scales_of = [&](const float* scales, const int (&id)[2], float (&f)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f[u] = scales[(has[u] ? static_cast<int64_t>(id[u]) : 0) * a.k_heads + h];
      }
    };

    Words kw[2][KS], vw[2][KS];
    float kf[2] = {1, 1}, vf[2] = {1, 1};
    uint32_t valid[2], valid_next[2];
    int id[2], id_first[2];
    const auto note = [&](uint32_t (&v)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = static_cast<uint32_t>(__ballot(has[u])) & 0xffffu;
    };
    // Loads return in order, so what a step needs first is issued first: its
    // block ids a whole step before its keys, its scales, its values.
    find(step0, id_first);
    find(step0 + 1, id);
    place(step0, id_first);
    note(valid);
    load(a.k_pool, kw);
    if constexpr (E4) {
      scales_of(a.k_scales, id_first, kf);
      scales_of(a.v_scales, id_first, vf);
    }
    load(a.v_pool, vw);

    for (int step = step0; step < step1; ++step) {
      const int p0 = begin + step * kFewStep;
      f32x4 sc[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt][0] = sc[rt][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 key;
          if constexpr (E4) {
            key = Widen<E>(kw[u][ks]);
          } else {
            key = kw[u][ks];
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt][u] = Mma16<E>(key, q[rt][ks], sc[rt][u]);
        }
      }
      float vs[8];  // scales, or their rests, of the values of the lane's tokens
      float power[2] = {1, 1};  // and powers of those that it loads
      if constexpr (E4) {
        const float rest[2] = {ValueRest<E>(vf[0]), ValueRest<E>(vf[1])};
        power[0] = ValuePower<E>(vf[0]);
        power[1] = ValuePower<E>(vf[1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = __shfl(kf[i / 4], quarter * 4 + i % 4);
          vs[i] = __shfl(rest[i / 4], quarter * 4 + i % 4);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt][i / 4][i % 4] *= f;
        }
      }
      // The next step's keys, while this one's scores are worked on.
      place(step + 1, id);
      note(valid_next);
      if constexpr (E4) {
        const int now[2] = {id[0], id[1]};
        find(step + 2, id);
        load(a.k_pool, kw);
        scales_of(a.k_scales, now, kf);
        scales_of(a.v_scales, now, vf);
      } else {
        find(step + 2, id);
        load(a.k_pool, kw);
      }
      if (p0 + 32 > seen_by_all || (valid[0] & valid[1]) != 0xffffu) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t there = valid[u] >> (quarter * 4);
          const int from = p0 + u * 16 + quarter * 4;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const int behind = seen[rt] - from;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i >= behind || (there & (1u << i)) == 0) sc[rt][u][i] = -__builtin_inff();
            }
          }
        }
      }
      u32x4 pw[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float most = sc[rt][0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, sc[rt][i / 4][i % 4]);
        most = Across32(Across16(most)) * c;
        // The maximum is only moved when it falls behind by 2^8: exponentials
        // up to there lose nothing in either type.
        if (__any(most > top[rt] + 8.0f)) {
          const float now = fmaxf(top[rt], most);
          const float back = now == -__builtin_inff() ? 0.0f : now;
          const float shrink = __builtin_amdgcn_exp2f(top[rt] - back);
          top[rt] = now;
          sum[rt] *= shrink;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= shrink;
        }
        const float base = top[rt] == -__builtin_inff() ? 0.0f : top[rt];
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(sc[rt][i / 4][i % 4], c, -base));
          sum[rt] += e[i];
        }
        if constexpr (E4) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // A hidden token's scale may be anything.
            e[i] = e[i] == 0.0f ? 0.0f : e[i] * vs[i];
          }
        }
        // The matrix instructions take 16-bit operands: each exponential is off by
        // half a step, in fp16 by up to 2^-25 of the largest, while the sum takes it
        // whole. In bf16 that makes 2.3e-3 of error against 64 bits where rounding
        // the result alone makes 1.7e-3; two operands for its two halves would
        // double the second product.
        pw[rt] = u32x4{Pack2<E>(e[0], e[1]), Pack2<E>(e[2], e[3]), Pack2<E>(e[4], e[5]),
                       Pack2<E>(e[6], e[7])};
      }
      if ((valid[0] & valid[1]) != 0xffffu) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if ((valid[u] >> in16 & 1) == 0) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) vw[u][ks] = Words(0);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 value;
          if constexpr (E4) {
            value = Widen<E>(vw[u][ks], power[u]);
          } else {
            value = vw[u][ks];
          }
          *reinterpret_cast<u32x4*>(mine + (u * 16 + in16) * VST + dim_of(ks) * 2) = value;
        }
      }
      load(a.v_pool, vw);
      valid[0] = valid_next[0];
      valid[1] = valid_next[1];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const char* p = mine + (quarter * 4 + in16 / 4) * VST + dt * 32 + (in16 % 4) * 8;
        const u32x2 lo = ReadTransposed(p), hi = ReadTransposed(p + 16 * VST);
        const u32x4 value = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = Mma16<E>(value, pw[rt], o[rt][dt]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }

    // Lane: row l % 16 of each row tile, dimensions 16 dt + 4 (l / 16)...
    const bool whole = step0 == 0 && step1 == steps;
    const int slot = axis.Slot(worker, x);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float l = sum[rt];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      const int row = rt * 16 + in16, t = FastDivI(a.group_div, row);
      const int64_t token = span.first + t;
      const int head = h * G + (row - t * G);
      if (row < rows) {
        if (whole && !grouped) {
          const float inverse = InverseSum(l);
          Scalar* out = static_cast<Scalar*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const int d = dt * 16 + quarter * 4;
            using Pair = u32x2 __attribute__((aligned(2)));
            const f32x4 v = Seen(o[rt][dt], l) * inverse;
            if (FULL || d < a.head_dim) {
              *reinterpret_cast<Pair*>(out + d) = u32x2{Pack2<E>(v[0], v[1]), Pack2<E>(v[2], v[3])};
            }
          }
          if (a.lse != nullptr && quarter == 0) {
            a.lse[token * a.q_heads + head] = (top[rt] + log2f(l)) / kLog2e;
          }
        } else {
          const int64_t to = whole ? WholeRow(a, false, token, head) : FewSlotRow(a, slot) + row;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            *reinterpret_cast<f32x4*>(a.parts + to * DP + dt * 16 + quarter * 4) =
                Seen(o[rt][dt], l);
          }
          if (quarter == 0) PartStats(a)[to] = f32x2{top[rt], l};
        }
      }
    }
    x += step1 - step0;
  }
}

}  // namespace kvx

#endif  // KVX_KERNELS_ATTEND_FEW_H_
