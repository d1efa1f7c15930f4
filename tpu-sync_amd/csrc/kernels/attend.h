// Host-side interface of the paged attention kernels (gfx950).
//
// Rows. A query row is one head of one token; the Hq / Hk rows of a token that
// share a key head stand next to each other. Row at position p = length -
// count + i sees tokens 0..p of its sequence (causal) or all of them.
//
// Kernels.
//  * attend_few: every sequence has up to kFewRows rows a key head (single
//    tokens, a few drafted ones). One wave holds them; the key axis is split.
//  * attend_mixed: longer runs of queries too, in tiles of kManyRows rows, and
//    shared prefixes: all rows of a group's sequences against the prefix.
//  * attend_join: merges the parts of rows that were split.
//
// Which part of the work a workgroup takes is computed from the lengths on the
// device, by the same arithmetic in every kernel, so a call needs no plan, and
// a captured call follows lengths that change between replays.
#ifndef KVX_KERNELS_ATTEND_H_
#define KVX_KERNELS_ATTEND_H_

#include <hip/hip_runtime_api.h>

#include <cstdint>

#include "kv_element.h"
#include "tiled_copy.h"

namespace kvx {

// Rows a key head up to which a wave works alone on a part of the keys. 64
// sequences of 3000 to 4000 tokens, 32 query heads on one, D = 128: 40 us, as
// tiles of 128 rows 69 us; 24 heads on one over 100 to 200 tokens: 18 and 37 us;
// 4 new tokens of 32 heads on 4: 149 and 141 us.
constexpr int kFewRows = 32;
constexpr int kFewStep = 32;    // tokens of one step of a wave
constexpr int kManyRows = 128;  // rows of one tile
constexpr int kManyStep = 64;   // tokens of one step
constexpr int kMaxSequences = 4096;
constexpr int kMaxGroups = 256;
constexpr int kMaxHeadDim = 256;

// The worker at a place of a grid whose places go to the XCDs in turn, or -1:
// an XCD's workers are neighbours, and every XCD has its share of them, however
// many the lengths leave of the grid that the table's width allows. (Shared out
// over that grid, a prompt of 128 tokens, 32 heads on 8, in a table of 8192 had two
// XCDs: 31.3 us, here 24.2.)
constexpr int kXcds = 8;
constexpr int WorkerAt(int place, int workers) {
  const int each = (workers + kXcds - 1) / kXcds;
  const int at = place / kXcds, worker = place % kXcds * each + at;
  return at < each && worker < workers ? worker : -1;
}

struct AttendLaunch {
  BatchView batch;
  FastDivU32 block_div;  // by batch.block_tokens
  FastDivU32 group_div;  // by q_heads / k_heads
  const void* q = nullptr;  // [tokens][q_heads][head_dim]
  void* out = nullptr;
  float* lse = nullptr;  // [tokens][q_heads] or null
  int64_t q_token = 0, q_head = 0, out_token = 0, out_head = 0;
  const void* k_pool = nullptr;  // [num_blocks][block_tokens][k_heads][head_dim]
  const void* v_pool = nullptr;
  const float* k_scales = nullptr;  // e4m3: [num_blocks][k_heads]
  const float* v_scales = nullptr;
  int32_t most_few = 0, most_many = 0;  // steps of a key head that the sizes allow
  // Groups of sequences [group_starts[g], group_starts[g + 1]) whose first
  // prefix_lengths[g] tokens are in the same blocks.
  const int32_t* group_starts = nullptr;
  const int32_t* prefix_lengths = nullptr;
  int32_t groups = 0;
  int32_t q_heads = 0, k_heads = 0, head_dim = 0;
  int32_t type = kBf16;  // of q and out
  bool e4m3 = false;
  bool causal = true;
  float scale = 1.0f;
  // Parts of split rows, part_rows rows of padded_dim floats relative to their
  // maximum; then the (maximum in powers of two, sum) of each; then the plan
  // that attend_join reads (attend_plan.h).
  float* parts = nullptr;
  // Filled by PlanAttend.
  int32_t padded_dim = 0;
  int32_t few_grid = 0;   // workgroups for few rows
  int32_t few_rows = 0;   // most rows of such a sequence
  int32_t many_grid = 0;  // workgroups for many rows and groups, 0: attend_few alone
  int64_t part_rows = 0;
  int32_t join_grid = 0;  // workgroups of attend_join, 0: no row can be split
  int32_t join_rows = 0;  // rows that one of them joins at once
};

// Sizes of the launches of a call (from its shapes only). Returns the bytes of
// `parts`.
int64_t PlanAttend(AttendLaunch* l);

// Every address range must have been checked and PlanAttend called.
hipError_t LaunchAttend(const AttendLaunch& l, hipStream_t stream);

// The parts, by translation unit.
hipError_t LaunchAttendFew(const AttendLaunch& l, hipStream_t stream);
hipError_t LaunchAttendMixed(const AttendLaunch& l, hipStream_t stream);
hipError_t LaunchAttendJoin(const AttendLaunch& l, hipStream_t stream);

}  // namespace kvx

#endif  // KVX_KERNELS_ATTEND_H_
