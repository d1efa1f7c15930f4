// The kept tokens of each sequence and key head to the front of the sequence, in place:
// place i gets the key, the value (their scales) and the weight of token kept[i], kept
// ascending, so kept[i] >= i.
//
// In place without a copy: a workgroup goes through the places of one sequence and key
// head, K or V, in ascending rounds. A round reads all of its rows into registers,
// waits for every wave, and writes them; what it writes is below every row that a later
// round reads. Rows of the next round are on their way while this one's are written.
// Where there are few sequences and heads, several workgroups take a part of every
// row's bytes each. Rows that stay at their place are neither read nor written. 64
// sequences cut to 2048 tokens, 8 heads x 128, bf16: 192 us for 849 MB (4.4 TB/s, reads
// of scattered 256-byte rows and writes; torch's copy of 1 GiB reaches 5.1); one such
// sequence 18 us. In 4 bits 85 us for 232 MB: rows of 64 bytes, and their scales, which a
// thread a row moves byte by byte.
//
// e4m3 (compact_e4m3_kernel): rows that meet in a block come from blocks with scales of
// their own, so the block gets the largest of them, and codes are stored again as
// e4m3(code * old / new), which rounds those of smaller scales once. A block's scale is
// replaced when all of its rows are there; later rounds read later blocks. What a round
// needs is looked up two rounds ahead and decided on one ahead, by a thread a row. 24
// sequences cut to 3000 tokens, 8 heads x 128: 94 us for 301 MB; with three waits a round
// of 128 rows and a division a piece 155 us; lookups in three steps over rounds, a load
// each, 97 us. 384 workgroups of 8 waves leave the GPU's memory idle between their
// rounds: a block's scale ties its rows to one workgroup.
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

__device__ __forceinline__ uint32_t Rescaled(uint32_t w, float ratio) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  int q = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * ratio, lo[1] * ratio, 0, false);
  q = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * ratio, hi[1] * ratio, q, true);
  return static_cast<uint32_t>(q);
}

// WIDE: rows are whole 16 bytes. THREADS: of a workgroup, and rows of a round.
template <int DP, bool WIDE, int THREADS>
__global__ __launch_bounds__(THREADS, 2) void compact_e4m3_kernel(
    const CompactLaunch a) {
  // Rounds in turn, four at a time. Of a row: where it is and goes, its scale, its place
  // in `largest`. Of a block: the new scale's bits, and whether one of its rows moves.
  constexpr int kSlots = 4;
  using Piece = std::conditional_t<WIDE, u32x4, u32x2>;
  using Bytes = Piece __attribute__((aligned(1)));
  constexpr int kPiece = sizeof(Piece);
  __shared__ int64_t from[kSlots][THREADS], to[kSlots][THREADS];
  __shared__ float factors[2][THREADS];  // what a row's codes are multiplied with, 0: stays
  __shared__ float old_scale[kSlots][THREADS];
  __shared__ uint32_t largest[kSlots][THREADS];
  __shared__ int moves[kSlots][THREADS];
  constexpr int kPieces = DP / kPiece;  // of a thread
  const int s = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const bool key = blockIdx.y == 0;
  uint8_t* pool = static_cast<uint8_t*>(key ? a.k_pool : a.v_pool);
  float* scales = static_cast<float*>(key ? a.k_scales : a.v_scales);
  const int32_t* table = a.batch.tables + s * a.batch.table_stride;
  const int32_t* kept = a.kept + s * a.kept_sequence + h * a.kept_head;
  const int B = a.batch.block_tokens, pieces = a.head_dim / kPiece;
  const int me = static_cast<int>(threadIdx.x);
  // Threads of a row, a power of two, and where this one is in its rows.
  const int shift = 32 - __clz(pieces - 1 > 0 ? pieces - 1 : 0);
  const int my_row = me >> shift, my_piece = me & ((1 << shift) - 1), rows_apart = THREADS >> shift;
  const int passes = my_piece < pieces ? 1 << shift : 0;
  const bool takes_weight = a.weights != nullptr && key;
  // A round: as many whole blocks as it has rows for, or a part of one block.
  const int of_round = B <= THREADS ? THREADS / B : 1;
  const int parts = B <= THREADS ? 1 : (B + THREADS - 1) / THREADS;
  const int last = min(a.budget, a.batch.capacity);
  const int rounds =
      static_cast<int>((last + static_cast<int64_t>(of_round) * B - 1) / (of_round * B)) * parts;
  // First place of a round's blocks and of the round, and the end of the latter.
  const auto begin_of = [&](int r) { return r / parts * static_cast<int64_t>(of_round) * B; };
  const auto first_of = [&](int r) { return begin_of(r) + r % parts * THREADS; };
  const auto end_of = [&](int r) {
    const int64_t all = min(begin_of(r) + static_cast<int64_t>(of_round) * B, static_cast<int64_t>(last));
    return static_cast<int>(parts == 1 ? all : min(all, first_of(r) + THREADS));
  };
  const auto block_of = [&](int p) {  // block id, or -1
    if (p < 0 || p >= a.batch.capacity) return -1;
    const int id = table[FastDivI(a.block_div, p)];
    return id >= 0 && id < a.batch.num_blocks ? id : -1;
  };
  const auto scale_of = [&](int id) {
    const float f = scales[static_cast<int64_t>(id) * a.heads + h];
    return f > 0.0f ? f : 0.0f;
  };
  const auto row = [&](int id, int p) {
    const int slot = p - FastDivI(a.block_div, p) * B;
    return (static_cast<int64_t>(id) * B + slot) * a.heads + h;
  };
  // A block of several rounds keeps its scale in the slot of its own number.
  const auto slot_of = [&](int r) { return r / parts % kSlots; };
  const auto note = [&](int r, int g, int i, int p, float scale) {
    atomicMax(&largest[slot_of(r)][g], __builtin_bit_cast(uint32_t, scale));
    if (p != i) atomicOr(&moves[slot_of(r)][g], 1);
  };
  int place = 0, position = -1, next_place = 0, next_position = -1;
  // Thread t looks up row t of round r.
  const auto look = [&](int r) {
    int64_t x = -1, y = -1;
    float scale = 0.0f;
    next_position = -1;
    if (r < rounds) {
      const int begin = static_cast<int>(begin_of(r));
      const int64_t i64 = first_of(r) + me;
      if (i64 < end_of(r)) {
        const int i = static_cast<int>(i64), p = kept[i * a.kept_place];
        const int id = block_of(p), into = block_of(i);
        next_place = i;
        next_position = p;
        if (id >= 0) {
          scale = scale_of(id);
          if (parts == 1) note(r, FastDivI(a.block_div, i - begin), i, p, scale);
          // (Where a block's last row stays, all of them do.)
          const int end = min(i + B - (i - FastDivI(a.block_div, i) * B), last) - 1;
          if (into >= 0 && (p != i || kept[end * a.kept_place] != end)) {
            x = row(id, p);
            y = row(into, i);
          }
        }
      }
      if (parts > 1 && r % parts == 0) {
        const int end = min(begin + B, last);
        for (int i = begin + me; i < end; i += THREADS) {
          const int p = kept[i * a.kept_place], id = block_of(p);
          if (id >= 0) note(r, 0, i, p, scale_of(id));
        }
      }
    }
    from[r % kSlots][me] = x;
    to[r % kSlots][me] = y;
    old_scale[r % kSlots][me] = scale;
  };
  const auto clear = [&](int slot) {
    largest[slot][me] = 0;
    moves[slot][me] = 0;
  };
  // Thread t decides on row t of round r.
  const auto decide = [&](int r) {
    float f = 0.0f;
    const int64_t x = from[r % kSlots][me];
    const int g = parts == 1 ? FastDivI(a.block_div, me) : 0;
    if (x >= 0 && moves[slot_of(r)][g] != 0) {
      const float now = __builtin_bit_cast(float, largest[slot_of(r)][g]), old = old_scale[r % kSlots][me];
      if (old == now) {
        f = x == to[r % kSlots][me] ? 0.0f : 1.0f;
      } else {
        f = old / now;
        if (f == 0.0f) f = -1.0f;  // all codes become 0
      }
    }
    factors[r & 1][me] = f;
  };
  Piece held[kPieces];
  float weight = 0.0f;
  int64_t weight_to = -1;
  const auto load = [&](int r) {
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      held[n] = Piece(0);
      if (n < passes) {
        const int64_t x = from[r % kSlots][my_row + n * rows_apart];
        if (x >= 0) {
          held[n] = *reinterpret_cast<const Bytes*>(pool + x * a.head_dim + my_piece * kPiece);
        }
      }
    }
    place = next_place;
    position = next_position;
    weight_to = -1;
    if (takes_weight && position != place && from[r % kSlots][me] >= 0) {
      weight = a.weights[WeightAt<false>(a, h, from[r % kSlots][me], position)];
      weight_to = WeightAt<false>(a, h, to[r % kSlots][me], place);
    }
  };
  for (int n = 0; n < kSlots; ++n) clear(n);
  __syncthreads();
  look(0);
  __syncthreads();
  decide(0);
  load(0);
  look(1);
  for (int r = 0; r < rounds; ++r) {
    // Every wave has this round's rows before one of them is written over.
#pragma unroll
    for (int n = 0; n < kPieces; ++n) asm volatile("" : : "v"(held[n]));
    asm volatile("" : : "v"(weight));
    __syncthreads();
    Piece now[kPieces];
#pragma unroll
    for (int n = 0; n < kPieces; ++n) now[n] = held[n];
    const float now_weight = weight;
    const int64_t now_to = weight_to;
    decide(r + 1);
    load(r + 1);
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      if (n >= passes) continue;
      const int row_of = my_row + n * rows_apart;
      const float f = factors[r & 1][row_of];
      if (f == 0.0f) continue;
      if (f != 1.0f) {
        const float ratio = f < 0.0f ? 0.0f : f;
#pragma unroll
        for (int i = 0; i < kPiece / 4; ++i) now[n][i] = Rescaled(now[n][i], ratio);
      }
      *reinterpret_cast<Bytes*>(pool + to[r % kSlots][row_of] * a.head_dim + my_piece * kPiece) =
          now[n];
    }
    if (now_to >= 0) a.weights[now_to] = now_weight;
    // The scales of blocks that are whole now: nothing reads the old ones any more.
    if (me < of_round && r % parts == parts - 1 && moves[slot_of(r)][me] != 0) {
      const int64_t at = begin_of(r) + static_cast<int64_t>(me) * B;
      const int into = at < last ? block_of(static_cast<int>(at)) : -1;
      if (into >= 0) {
        scales[static_cast<int64_t>(into) * a.heads + h] =
            __builtin_bit_cast(float, largest[slot_of(r)][me]);
      }
    }
    // For the round after the next two, whose rows are looked up behind the next barrier.
    if (r % parts == 0) clear((slot_of(r) + kSlots - 1) % kSlots);
    look(r + 2);
  }
}

}  // namespace

hipError_t LaunchCompact(const CompactLaunch& l, hipStream_t stream) {
  const unsigned rows = static_cast<unsigned>(l.batch.sequences) * l.heads;
  if (l.pool == kPoolE4m3) {
    const bool wide = l.head_dim % 16 == 0;
    // Twice the threads, and half as many rounds, while the GPU holds all workgroups at
    // once: one sequence of 8 heads cut to 3000 tokens 51 to 31 us, 24 of them 97 to 94,
    // but 64 of them 199 to 208. (At D = 256 a CU would hold one of them.)
    const bool big = l.head_dim <= 128 && rows * 2ull <= 512;
    const unsigned threads = big ? 512 : 256;
    const auto kernel =
        big ? (wide ? compact_e4m3_kernel<128, true, 512> : compact_e4m3_kernel<128, false, 512>)
        : l.head_dim <= 128
            ? (wide ? compact_e4m3_kernel<128, true, 256> : compact_e4m3_kernel<128, false, 256>)
            : (wide ? compact_e4m3_kernel<256, true, 256> : compact_e4m3_kernel<256, false, 256>);
    hipLaunchKernelGGL(kernel, dim3(rows, 2), dim3(threads), 0, stream, l);
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
