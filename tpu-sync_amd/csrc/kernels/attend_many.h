// Paged attention of many rows a key head: chunks of new tokens, and all rows
// of sequences that share a prefix against that prefix.
//
// A workgroup takes a tile of 128 rows, 32 a wave, and steps through its keys
// 64 at a time; K and V of a step lie in LDS for all four waves. Matrix
// instructions bound it, so the layout keeps everything between the two products
// in place: S^T = K Q^T in 32 x 32 x 16 products leaves lane l with the scores of
// row l % 32, so a row's maximum takes one swap between the wave's halves, and
// the packed exponentials are the operand of O^T = V^T P^T as they stand (the
// contraction runs over tokens in the order that the scores lie in). V is
// transposed by the LDS reads.
//
// A wave works in halves of a step: the scores of the next 32 tokens are on the
// matrix cores while the exponentials of these are taken, and their operands are
// read four products ahead. Tokens go from memory straight into LDS, each storage
// refilled as soon as its last reader is past a barrier: keys run two steps
// ahead, values one, so K and V need two buffers each and no registers. (e4m3
// tokens are widened on the way, in registers.) 4099 new tokens of 5 sequences of
// 2000 to 12000, 32 heads on 8, D = 128, bf16: 730 us with tokens passing through
// registers and a wave's products and exponentials in turn, 676 us without, 655 us
// with operands read ahead and products given priority, 626 to 639 us with the
// places of tokens kept as byte offsets (back to back, 37 us of joining among them:
// 845 to 862 TFLOP/s, where an 8192^3 product of the library reaches 1211). Matrix
// cores are busy for 46 % of the CUs' cycles and other vector instructions for
// 51 %, so the two hardly overlap.
//
// Work. The tiles of all groups and sequences make one axis, weighed by the
// keys they see, and every workgroup gets an equal part of it: no tail of late
// tiles. What a part cuts is at its two ends and goes to slots 2w and 2w + 1 of
// `parts`; whole tiles go straight to the output, or, where a row has a group's
// part and one of its own, to its row of `parts`. The workgroups of one XCD take
// neighbouring parts, so its L2 serves a key head's tokens to all of them.
#ifndef KVX_KERNELS_ATTEND_MANY_H_
#define KVX_KERNELS_ATTEND_MANY_H_

#include "attend_plan.h"

namespace kvx {

// A token's row in LDS is its 2 DP bytes, in 16-byte chunks that are exchanged
// within the row so that the rows of one read fall on different banks (256
// bytes apart in 16ths): `chunk` of row `r` lies at chunk KeyChunk or ValueChunk.
// Keys are read 16 bytes of 16 neighbouring rows at a time, values 64 bytes of
// four neighbouring rows.
template <int DP>
__device__ __forceinline__ int KeyChunk(int r, int chunk) {
  if constexpr (DP == 64) return chunk ^ (r / 2 % 8);   // two rows in 256 bytes
  if constexpr (DP == 96) return chunk ^ (r / 4 % 4);   // rows 192 bytes apart
  return chunk ^ (r % 16);
}
template <int DP>
__device__ __forceinline__ int ValueChunk(int r, int chunk) {
  if constexpr (DP == 64) return chunk ^ (r / 2 % 2 * 4);
  if constexpr (DP == 96) return chunk;
  return chunk ^ (r % 4 * 4);
}

__device__ __forceinline__ uint32_t LdsAddress(char* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)p));
}
// Loads 16 bytes a lane straight into LDS, lane l's to address `to` + 16 l, which
// is taken from m0 (the compiler's to write, a wait state ahead). The compiler
// does not know of the loads: LdsArrived waits for all but the last N.
__device__ __forceinline__ void ToLds16(const void* from, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "{m0}"(to) : "memory");
}
template <int N>
__device__ __forceinline__ void LdsArrived() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Places of a step's tokens: looked up three steps ahead, their scales two.
struct Places {
  int64_t at[kManyStep];  // byte offset of the token's row; without one, of the first
  int32_t id[kManyStep];  // its block, or -1
  float k_scale[kManyStep], v_scale[kManyStep];
  uint64_t present;  // one bit a token
};

constexpr size_t ManyLds(const AttendLaunch& l, int dp) {
  return 2 * kManyStep * 4 * dp + 4 * sizeof(Places) +
         static_cast<size_t>(l.groups + l.batch.sequences) * sizeof(int);
}

template <class E, bool E4, int DP>
__device__ __forceinline__ void AttendMany(const AttendLaunch& a, char* lds, int place) {
  using Scalar = typename E::Scalar;
  constexpr int KS = DP / 16, DT = DP / 32, kRow = 2 * DP;  // bytes of a token's row
  constexpr int kChunks = kManyStep * (DP / 8) / kAttendThreads;  // of a thread
  constexpr int kTile = 2 * kManyStep * kRow;  // keys, then values
  Places* places = reinterpret_cast<Places*>(lds + 2 * kTile);
  int* sums = reinterpret_cast<int*>(places + 4);  // [groups + sequences]
  const BatchView& b = a.batch;
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  using Words = u32x2;  // e4m3 values of a chunk
  const uint32_t lds_at = one(LdsAddress(lds));

  // Dimensions behind the last one are never written.
  if (!E4 && a.head_dim < DP) {
    for (int i = threadIdx.x; i < 2 * kTile / 16; i += kAttendThreads) {
      reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    }
  }
  const int units = a.groups + b.sequences;
  for (int i = threadIdx.x; i < units; i += kAttendThreads) {
    sums[i] = ManyWork(a, i, LoadManyUnit(a, i));
  }
  BlockSums(sums, units, a.most_many);
  const int work = one(sums[units - 1]);
  if (work == 0) return;
  const Axis axis = ManyAxis(a, work);
  const int worker = WorkerAt(place, axis.workers);
  if (worker < 0) return;
  const int x_start = axis.Start(worker), x_end = axis.Start(worker + 1);
  const int G = a.q_heads / a.k_heads;
  const int lane = threadIdx.x % 64, wave = one(threadIdx.x / 64);
  const int in32 = lane % 32, half = lane / 32;

  // The end of a tile that the part starts with comes last, after the start of
  // the one that it ends with: workgroups with equal tiles then read the same
  // tokens at the same time.
  int limit = x_end, put_off = 0;
  for (int x = x_start; x < limit;) {
    const int i = one(FirstAbove(sums, units, x / a.k_heads));
    const int before = i > 0 ? one(sums[i - 1]) : 0;
    const int per_head = one(sums[i]) - before;
    const int h = (x - before * a.k_heads) / per_head;
    const int at_unit = x - before * a.k_heads - h * per_head;
    const ManyUnit u = LoadManyUnit(a, i);
    const int rows = one(u.rows), begin = one(u.begin), end = one(u.end), first = one(u.first);
    const int base = one(u.base);
    const bool group = i < a.groups;
    const int tile = one(TileAt(a, group, base, ManyTiles(u), at_unit));
    const int tile_at = ManyCost(a, group, base, tile);
    const int cost = ManyCost(a, group, base, tile + 1) - tile_at;
    const int from = at_unit - tile_at, to = min(cost, from + (limit - x));
    if (x == x_start && put_off == 0 && from > 0 && x + to - from < x_end) {
      put_off = x + to - from;
      x = put_off;
      continue;
    }
    const int sequence = group ? min(max(one(a.group_starts[i]), 0), b.sequences - 1)
                               : i - a.groups;
    const SequenceSpan span = LoadSequence(b, sequence);
    const bool grouped = group || LoadOwnKeys(a, sequence).grouped;
    // Steps that the tile's rows see, and this part's share of them.
    int steps = (end - begin + kManyStep - 1) / kManyStep;
    if (!group && a.causal) {
      const int last = min(rows, (tile + 1) * kManyRows) - 1;
      const int seen = Visible(a, span, first + FastDivI(a.group_div, last));
      steps = min(steps, (max(seen - begin, 0) + kManyStep - 1) / kManyStep);
    }
    steps = one(steps);
    const int step0 = static_cast<int>(static_cast<int64_t>(from) * steps / cost);
    const int step1 = static_cast<int>(static_cast<int64_t>(to) * steps / cost);

    // Queries: row l % 32 of the wave's 32, as an operand.
    const int row = tile * kManyRows + wave * 32 + in32;
    const int t = FastDivI(a.group_div, row);
    const int64_t token = first + t;
    const int head = h * G + (row - t * G);
    int seen = INT_MAX;
    if (row < rows) {
      if (!group) {
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
    // One wave looks up a step's 64 tokens, another one their scales. Loads
    // return in order, so a lookup is issued before the step's tokens and put
    // into LDS after its products: nobody waits for it.
    int found = -1;
    float found_k = 0.0f, found_v = 0.0f;
    const auto find = [&](int step) {
      const int p = begin + step * kManyStep + lane;
      found = step < step1 && p < end ? table[FastDivI(a.block_div, p)] : -1;
    };
    const auto keep = [&](int step) {
      Places& to = places[step & 3];
      const int p = begin + step * kManyStep + lane;
      const bool is = found >= 0 && found < b.num_blocks;
      const int slot = p - FastDivI(a.block_div, p) * b.block_tokens;
      const int64_t row = is ? static_cast<int64_t>(found) * b.block_tokens + slot : 0;
      to.at[lane] = (row * row_stride + h * a.head_dim) * (E4 ? 1 : 2);
      to.id[lane] = is ? found : -1;
      const uint64_t present = __ballot(is);
      if (lane == 0) to.present = present;
    };
    const auto find_scales = [&](int step) {
      const int id = places[step & 3].id[lane];
      const int64_t at = static_cast<int64_t>(max(id, 0)) * a.k_heads + h;
      found_k = a.k_scales[at];
      found_v = a.v_scales[at];
    };
    const auto keep_scales = [&](int step) {
      places[step & 3].k_scale[lane] = found_k;
      places[step & 3].v_scale[lane] = found_v;
    };
    // Tokens of a step on their way into LDS: e4m3 ones widened in registers,
    // others straight from memory, a wave's 64 chunks at a time. A token without
    // a place reads the pool's first row, so that this needs no branch.
    Words w[kChunks];
    const auto load = [&](int step, const void* pool) {
      const Places& held = places[step & 3];
      int64_t at[kChunks];
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        const int chunk = threadIdx.x + n * kAttendThreads;
        const int d = chunk % (DP / 8) * 8;
        at[n] = held.at[chunk / (DP / 8)] + (d < a.head_dim ? d : 0);
      }
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        w[n] = *reinterpret_cast<const Bytes8*>(static_cast<const uint8_t*>(pool) + at[n]);
      }
    };
    const auto store = [&](int step, auto is_key) {
      char* to = lds + (is_key() ? 0 : kTile) + (step & 1) * (kTile / 2);
      const Places& held = places[step & 3];
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        const int chunk = threadIdx.x + n * kAttendThreads;
        const int tok = chunk / (DP / 8), d = chunk % (DP / 8) * 8;
        const int at = is_key() ? KeyChunk<DP>(tok, d / 8) : ValueChunk<DP>(tok, d / 8);
        const bool is = (held.present >> tok & 1) != 0 && d < a.head_dim;
        *reinterpret_cast<u32x4*>(to + tok * kRow + at * 16) =
            Widen<E>(is ? w[n] : Words(0), is_key() ? 1.0f : ValuePower<E>(held.v_scale[tok]));
      }
    };
    const auto fetch = [&](int step, const void* pool, auto is_key) {
      const Places& held = places[step & 3];
      const uint32_t to = lds_at + (is_key() ? 0 : kTile) + (step & 1) * (kTile / 2) + wave * 1024;
      const auto from = [&](int n, int& d) {
        const int chunk = threadIdx.x + n * kAttendThreads;
        const int tok = chunk / (DP / 8), c = chunk % (DP / 8);
        d = (is_key() ? KeyChunk<DP>(tok, c) : ValueChunk<DP>(tok, c)) * 8;
        return static_cast<const char*>(pool) + d * 2 + held.at[tok];
      };
      const char* at[kChunks];
      int d[kChunks];
#pragma unroll
      for (int n = 0; n < kChunks; ++n) at[n] = from(n, d[n]);
      if (a.head_dim == DP) {
#pragma unroll
        for (int n = 0; n < kChunks; ++n) ToLds16(at[n], to + n * kAttendThreads * 16);
      } else {
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
          if (d[n] < a.head_dim) ToLds16(at[n], to + n * kAttendThreads * 16);
        }
      }
    };
    // Values of tokens without a place are cleared once they are there (their
    // scores are masked, whatever their keys are).
    const auto clear = [&](int step) {
      const Places& held = places[step & 3];
      if (held.present == ~uint64_t{0}) return;
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        const int chunk = threadIdx.x + n * kAttendThreads;
        if ((held.present >> (chunk / (DP / 8)) & 1) == 0) {
          *reinterpret_cast<u32x4*>(lds + kTile + (step & 1) * (kTile / 2) + chunk * 16) =
              u32x4{0, 0, 0, 0};
        }
      }
    };
    constexpr std::true_type kKeys{};
    constexpr std::false_type kValues{};

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16(0.0f);
    float top = -__builtin_inff(), sum = 0.0f;
    const float c = a.scale * kLog2e;
    // Scores of half a step. Lane: row l % 32, tokens 8 (i / 4) + 4 (l / 32) + i % 4.
    const auto scores = [&](int step, int u) {
      const char* keys = lds + (step & 1) * (kTile / 2);
      f32x16 sc = f32x16(0.0f);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 key = *reinterpret_cast<const u32x4*>(
            keys + (u * 32 + in32) * kRow + KeyChunk<DP>(u * 32 + in32, ks * 2 + half) * 16);
        sc = Mma32<E>(key, q[ks], sc);
      }
      return sc;
    };
    // Scales and masks them, and moves the maximum.
    const auto settle = [&](int step, int u, f32x16& sc) {
      const Places& here = places[step & 3];
      if constexpr (E4) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const f32x4 f = *reinterpret_cast<const f32x4*>(&here.k_scale[u * 32 + i * 2 + half * 4]);
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[i + j] *= f[j];
        }
      }
      const int p0 = begin + step * kManyStep + u * 32;
      const uint32_t present = static_cast<uint32_t>(here.present >> (u * 32));
      if (p0 + 32 > least || present != ~uint32_t{0}) {
        // Token n of the half is number n + 4 half of its lane's.
        const int behind = seen - p0 - half * 4;
        const uint32_t there = present >> (half * 4);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int n = (i / 4) * 8 + i % 4;
          if (n >= behind || (there & (1u << n)) == 0) sc[i] = -__builtin_inff();
        }
      }
      float most = sc[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) most = fmaxf(most, sc[i]);
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
    };
    f32x16 sc;
    if (step0 < step1) {
      if (wave < 3) {
        find(step0 + wave);
        keep(step0 + wave);
      }
      if constexpr (E4) {
        if (wave < 2) {
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          find_scales(step0 + wave);
          keep_scales(step0 + wave);
        }
      }
      __syncthreads();
      if constexpr (E4) {
        load(step0, a.k_pool);
        store(step0, kKeys);
        load(step0 + 1, a.k_pool);
        store(step0 + 1, kKeys);
        load(step0, a.v_pool);
        store(step0, kValues);
      } else {
        fetch(step0, a.k_pool, kKeys);
        fetch(step0, a.v_pool, kValues);
        fetch(step0 + 1, a.k_pool, kKeys);
        LdsArrived<0>();
        clear(step0);
      }
      __syncthreads();
      sc = scores(step0, 0);
      settle(step0, 0, sc);
      for (int step = step0; step < step1; ++step) {
        if (step > step0) __syncthreads();
        const bool finds = wave == (step & 3), finds_scales = E4 && wave == ((step + 1) & 3);
        if (finds) find(step + 3);
        if (finds_scales) find_scales(step + 2);
        // Keys two steps ahead and values one: the keys of this step go when the
        // scores of its second half are there, the values at its end.
        if constexpr (E4) {
          load(step + 2, a.k_pool);
        } else {
          fetch(step + 1, a.v_pool, kValues);
        }
        const Places& here = places[step & 3];
        const char* values = lds + kTile + (step & 1) * (kTile / 2);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // Exponentials and values of this half, while the matrix cores work on
          // the next one's scores.
          if (begin + step * kManyStep + u * 32 < most_seen) {
            const float base = top == -__builtin_inff() ? 0.0f : top;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            f32x16 next = scores(step + u, 1 - u);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              sc[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], c, -base));
              sum += sc[i];
            }
            if constexpr (E4) {
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const f32x4 f =
                    *reinterpret_cast<const f32x4*>(&here.v_scale[u * 32 + i * 2 + half * 4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  // A hidden token's scale may be anything.
                  sc[i + j] = sc[i + j] == 0.0f ? 0.0f : sc[i + j] * ValueRest<E>(f[j]);
                }
              }
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
              const int i = kk * 8;
              // Rounded to operands, as in attend_few.h.
              const u32x4 p = {Pack2<E>(sc[i], sc[i + 1]), Pack2<E>(sc[i + 2], sc[i + 3]),
                               Pack2<E>(sc[i + 4], sc[i + 5]), Pack2<E>(sc[i + 6], sc[i + 7])};
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) {
                // Row 4 half + l % 16 / 4 of 8, 8 bytes l % 4 of the 32 of l / 16 % 2.
                const int r = u * 32 + kk * 16 + half * 4 + lane % 16 / 4;
                const int chunk = dt * 4 + lane / 16 % 2 * 2 + lane % 4 / 2;
                const char* v = values + r * kRow + ValueChunk<DP>(r, chunk) * 16 + lane % 2 * 8;
                const u32x2 lo = ReadTransposed(v), hi = ReadTransposed(v + 8 * kRow);
                o[dt] = Mma32<E>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p, o[dt]);
              }
            }
            // Operands are read four products ahead.
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int n = 0; n < KS - 4; ++n) {
              __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
#pragma unroll
            for (int n = 0; n < DT * 2; ++n) {
              __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
            __builtin_amdgcn_s_setprio(0);
            sc = next;
            if (step + u < step1 && begin + step * kManyStep + u * 32 + 32 < most_seen) {
              settle(step + u, 1 - u, sc);
            }
          }
          if (u == 0) {
            if constexpr (!E4) {
              if (finds) keep(step + 3);
              LdsArrived<kChunks>();  // all but the values: the next step's keys
            }
            __syncthreads();
            if constexpr (E4) {
              store(step + 2, kKeys);
              load(step + 1, a.v_pool);
            } else {
              fetch(step + 2, a.k_pool, kKeys);
            }
          }
        }
        if constexpr (E4) {
          store(step + 1, kValues);
          if (finds) keep(step + 3);
          if (finds_scales) keep_scales(step + 2);
        } else {
          LdsArrived<kChunks>();  // all but the keys: the next step's values
          clear(step + 1);
        }
      }
      if constexpr (!E4) LdsArrived<0>();
    }

    // Lane: row l % 32, dimensions 32 dt + 8 (i / 4) + 4 (l / 32) + i % 4.
    sum += __shfl_xor(sum, 32);
    const bool whole = from == 0 && to == cost;
    if (row < rows) {
      if (whole && !grouped) {
        const float inverse = InverseSum(sum);
        Scalar* out = static_cast<Scalar*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int d = dt * 32 + i * 2 + half * 4;
            using Pair = u32x2 __attribute__((aligned(2)));
            if (d < a.head_dim) {
              const f32x4 v =
                  Seen(f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]}, sum) * inverse;
              *reinterpret_cast<Pair*>(out + d) = u32x2{Pack2<E>(v[0], v[1]), Pack2<E>(v[2], v[3])};
            }
          }
        }
        if (a.lse != nullptr && half == 0) {
          a.lse[token * a.q_heads + head] = (top + log2f(sum)) / kLog2e;
        }
      } else {
        const int64_t to_row = whole ? WholeRow(a, group, token, head)
                                     : ManySlotRow(a, axis.Slot(worker, x)) + wave * 32 + in32;
        if (half == 0) PartStats(a)[to_row] = f32x2{top, sum};
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            *reinterpret_cast<f32x4*>(a.parts + to_row * DP + dt * 32 + i * 2 + half * 4) =
                Seen(f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]}, sum);
          }
        }
      }
    }
    x += to - from;
    if (x == x_end && put_off > 0) {
      x = x_start;
      limit = put_off;
    }
    __syncthreads();  // the next piece's tokens take this one's place in LDS
  }
}

}  // namespace kvx

#endif  // KVX_KERNELS_ATTEND_MANY_H_
