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
// Work. The steps (128 tokens, 32 a wave) of all sequences and key heads form
// one axis, cut into equal parts, one a workgroup: long and short sequences
// load the GPU alike. What a part cuts is at its two ends and goes to slots 2w
// and 2w + 1 of `parts`; what it holds whole goes straight to the output, or,
// where a group's prefix comes on top, to its own row of `parts`.
#include "attend_plan.h"

namespace kvx {
namespace {

using Bytes16 = u32x4 __attribute__((aligned(2)));
using Bytes8 = u32x2 __attribute__((aligned(1)));

constexpr int Waves() { return kAttendThreads / 64; }
// Bytes of a token's values in LDS: an odd multiple of 32, so that the rows
// of a transposing read fall on different banks.
constexpr int ValueStride(int dp) { return dp * 2 + 32; }

template <class E, bool E4, int DP, int RT, bool FULL>
__global__ __launch_bounds__(kAttendThreads, DP <= 128 ? (RT == 1 ? 3 : 2) : 1) void
attend_few_kernel(const AttendLaunch a) {
  using P = std::conditional_t<E4, Bf16, E>;  // of the second product
  using Scalar = typename E::Scalar;
  constexpr int KS = DP / 32, DT = DP / 16, VST = ValueStride(DP);
  extern __shared__ __align__(16) char lds[];
  f32x2* stats = reinterpret_cast<f32x2*>(lds + Waves() * 32 * VST);  // [waves][RT * 16]
  int* sums = reinterpret_cast<int*>(stats + Waves() * RT * 16);      // [sequences]
  const BatchView& b = a.batch;
  for (int s = threadIdx.x; s < b.sequences; s += kAttendThreads) {
    sums[s] = FewSteps(LoadOwnKeys(a, s));
  }
  BlockSums(sums, b.sequences);
  const int all = __builtin_amdgcn_readfirstlane(sums[b.sequences - 1]);
  if (all == 0) return;
  const FewAxis axis(a, all);
  if (static_cast<int>(blockIdx.x) >= axis.workers) return;
  const int x_first = axis.Start(blockIdx.x), x_end = axis.Start(blockIdx.x + 1);

  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int in16 = lane % 16, quarter = lane / 16;
  char* mine = lds + wave * 32 * VST;
  const int G = a.q_heads / a.k_heads;
  const int64_t row_stride = static_cast<int64_t>(a.k_heads) * a.head_dim;
  const float c = a.scale * kLog2e;
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };

  for (int x = x_first; x < x_end;) {
    const int s = one(FirstAbove(sums, b.sequences, x / a.k_heads));
    const int before = s > 0 ? one(sums[s - 1]) : 0;
    const int steps = one(sums[s]) - before;
    const int off = x - before * a.k_heads;
    const int h = off / steps, step0 = off - h * steps;
    const int step1 = min(steps, step0 + (x_end - x));
    const OwnKeys k = LoadOwnKeys(a, s);
    const int rows = one(k.rows), begin = one(k.begin), end = one(k.end);
    const int seen_by_all = one(Visible(a, k.q, k.q.first));

    // Queries: row l % 16 of each row tile, the dimensions of a key operand.
    u32x4 q[RT][KS];
    int seen[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = rt * 16 + in16, t = FastDivI(a.group_div, r);
      const int64_t token = k.q.first + t;
      const Scalar* p = static_cast<const Scalar*>(a.q) + token * a.q_token +
                        (h * G + (r - t * G)) * a.q_head + quarter * 8;
      seen[rt] = r < rows ? Visible(a, k.q, k.q.first + t) : INT_MAX;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[rt][ks] = u32x4{0, 0, 0, 0};
        if (r < rows && (FULL || ks * 32 + quarter * 8 < a.head_dim)) {
          q[rt][ks] = *reinterpret_cast<const Bytes16*>(p + ks * 32);
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

    // Tokens of a step: lane l loads token l % 16 of both halves of its
    // wave's 32, eight dimensions in each group of 32.
    const int32_t* table = b.tables + s * b.table_stride;
    const auto find = [&](int step, int (&id)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = begin + step * kFewStep + wave * 32 + u * 16 + in16;
        id[u] = -1;
        if (step < step1 && p < end) id[u] = table[FastDivI(a.block_div, p)];
      }
    };
    int64_t at[2];
    bool has[2];
    const auto place = [&](int step, const int (&id)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = begin + step * kFewStep + wave * 32 + u * 16 + in16;
        const int slot = p - FastDivI(a.block_div, p) * b.block_tokens;
        has[u] = id[u] >= 0 && id[u] < b.num_blocks;
        at[u] = (static_cast<int64_t>(id[u]) * b.block_tokens + slot) * row_stride +
                h * a.head_dim + quarter * 8;
      }
    };
    constexpr int W = E4 ? 2 : 4;
    using Words = __attribute__((ext_vector_type(W))) uint32_t;
    const auto load = [&](const void* pool, Words (&w)[2][KS]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          w[u][ks] = Words(0);
          if (has[u] && (FULL || ks * 32 + quarter * 8 < a.head_dim)) {
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
        f[u] = has[u] ? scales[static_cast<int64_t>(id[u]) * a.k_heads + h] : 0.0f;
      }
    };

    Words kw[2][KS], vw[2][KS];
    float kf[2] = {1, 1}, vf[2] = {1, 1}, kf_next[2] = {1, 1}, vf_next[2] = {1, 1};
    uint32_t valid[2], valid_next[2];
    int id[2];
    const auto note = [&](uint32_t (&v)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = static_cast<uint32_t>(__ballot(has[u])) & 0xffffu;
    };
    find(step0, id);
    place(step0, id);
    note(valid);
    load(a.k_pool, kw);
    load(a.v_pool, vw);
    if constexpr (E4) {
      scales_of(a.k_scales, id, kf);
      scales_of(a.v_scales, id, vf);
    }
    find(step0 + 1, id);

    for (int step = step0; step < step1; ++step) {
      const int p0 = begin + step * kFewStep + wave * 32;
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
      // The next step's keys, while this one's scores are worked on.
      place(step + 1, id);
      note(valid_next);
      load(a.k_pool, kw);
      if constexpr (E4) {
        scales_of(a.k_scales, id, kf_next);
        scales_of(a.v_scales, id, vf_next);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f = __shfl(kf[u], quarter * 4 + i);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][u][i] *= f;
          }
        }
      }
      if (p0 + 32 > seen_by_all || (valid[0] & valid[1]) != 0xffffu) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = quarter * 4 + i;
            const bool is = (valid[u] >> j & 1) != 0;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              if (!is || p0 + u * 16 + j >= seen[rt]) sc[rt][u][i] = -__builtin_inff();
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
          for (int i = 0; i < 8; ++i) e[i] *= __shfl(vf[i / 4], quarter * 4 + i % 4);
        }
        pw[rt] = u32x4{Pack2<P>(e[0], e[1]), Pack2<P>(e[2], e[3]), Pack2<P>(e[4], e[5]),
                       Pack2<P>(e[6], e[7])};
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 value;
          if constexpr (E4) {
            value = Widen<P>(vw[u][ks]);
          } else {
            value = vw[u][ks];
          }
          *reinterpret_cast<u32x4*>(mine + (u * 16 + in16) * VST + ks * 64 + quarter * 16) = value;
        }
      }
      load(a.v_pool, vw);
      find(step + 2, id);
      if constexpr (E4) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          kf[u] = kf_next[u];
          vf[u] = vf_next[u];
        }
      }
      valid[0] = valid_next[0];
      valid[1] = valid_next[1];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const char* p = mine + (quarter * 4 + in16 / 4) * VST + dt * 32 + (in16 % 4) * 8;
        const u32x2 lo = ReadTransposed(p), hi = ReadTransposed(p + 16 * VST);
        const u32x4 value = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = Mma16<P>(value, pw[rt], o[rt][dt]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }

    // The waves' parts of the keys, joined.
    const bool whole = step0 == 0 && step1 == steps;
    const int slot = x == x_first ? 2 * blockIdx.x : 2 * blockIdx.x + 1;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float l = sum[rt];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      if (quarter == 0) stats[wave * RT * 16 + rt * 16 + in16] = f32x2{top[rt], l};
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (rt * 16 >= rows) break;
      float most = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < Waves(); ++w) most = fmaxf(most, stats[(w * RT + rt) * 16 + in16][0]);
      const float back = most == -__builtin_inff() ? 0.0f : most;
      const float shrink = __builtin_amdgcn_exp2f(top[rt] - back);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        *reinterpret_cast<f32x4*>(mine + (in16 * DP + dt * 16 + quarter * 4) * 4) =
            o[rt][dt] * shrink;
      }
      __syncthreads();
      const int here = min(16, rows - rt * 16);
      for (int i = threadIdx.x; i < here * (DP / 4); i += kAttendThreads) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        f32x4 v = {0, 0, 0, 0};
        float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int w = 0; w < Waves(); ++w) {
          v += *reinterpret_cast<const f32x4*>(lds + w * 32 * VST + (r * DP + d) * 4);
          m = fmaxf(m, stats[(w * RT + rt) * 16 + r][0]);
        }
        const float m0 = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < Waves(); ++w) {
          const f32x2 st = stats[(w * RT + rt) * 16 + r];
          l += st[1] * __builtin_amdgcn_exp2f(st[0] - m0);
        }
        const int row = rt * 16 + r, t = FastDivI(a.group_div, row);
        const int64_t token = k.q.first + t;
        const int head = h * G + (row - t * G);
        if (whole && !k.grouped) {
          if (FULL || d < a.head_dim) {
            const float inverse = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
            using Pair = u32x2 __attribute__((aligned(2)));
            *reinterpret_cast<Pair*>(static_cast<Scalar*>(a.out) + token * a.out_token +
                                     head * a.out_head + d) =
                u32x2{Pack2<E>(v[0] * inverse, v[1] * inverse),
                      Pack2<E>(v[2] * inverse, v[3] * inverse)};
          }
          if (a.lse != nullptr && d == 0) {
            a.lse[token * a.q_heads + head] = (m + log2f(l)) / kLog2e;
          }
        } else {
          const int64_t to = whole ? WholeRow(a, token, head) : FewSlotRow(a, slot) + row;
          *reinterpret_cast<f32x4*>(a.parts + to * DP + d) = v;
          if (d == 0) PartStats(a)[to] = f32x2{m, l};
        }
      }
      __syncthreads();
    }
    x += step1 - step0;
  }
}

template <class E, bool E4, int DP, int RT, bool FULL>
hipError_t Launch(const AttendLaunch& l, hipStream_t stream) {
  const size_t lds = Waves() * 32 * ValueStride(DP) + Waves() * RT * 16 * sizeof(f32x2) +
                     static_cast<size_t>(l.batch.sequences) * sizeof(int);
  const auto kernel = attend_few_kernel<E, E4, DP, RT, FULL>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(lds));
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, dim3(l.few_grid), dim3(kAttendThreads), lds, stream, l);
  return hipGetLastError();
}

template <class E, bool E4, int DP>
hipError_t PickRows(const AttendLaunch& l, hipStream_t stream) {
  if (l.head_dim != DP) return Launch<E, E4, DP, 2, false>(l, stream);
  return l.few_rows == 16 ? Launch<E, E4, DP, 1, true>(l, stream)
                          : Launch<E, E4, DP, 2, true>(l, stream);
}

template <class E, bool E4>
hipError_t Pick(const AttendLaunch& l, hipStream_t stream) {
  switch (l.padded_dim) {
    case 64:
      return PickRows<E, E4, 64>(l, stream);
    case 96:
      return PickRows<E, E4, 96>(l, stream);
    case 128:
      return PickRows<E, E4, 128>(l, stream);
    default:
      return PickRows<E, E4, 256>(l, stream);
  }
}

}  // namespace

hipError_t LaunchAttendFew(const AttendLaunch& l, hipStream_t stream) {
  if (l.type == kBf16) return l.e4m3 ? Pick<Bf16, true>(l, stream) : Pick<Bf16, false>(l, stream);
  return l.e4m3 ? Pick<F16, true>(l, stream) : Pick<F16, false>(l, stream);
}

}  // namespace kvx
