// Host-side interface of the paged attention kernels (gfx950).
//
// Rows. A query row is one head of one token; the Hq / Hk rows of a token that
// share a key head stand next to each other. Row at position p = length -
// count + i sees tokens 0..p of its sequence (causal) or all of them.
//
// Kernels.
//  * attend_few: sequences of up to kFewRows rows a key head (single tokens, a
//    few drafted ones). One wave holds all their rows; the key axis is split.
//  * attend_many: longer runs of queries, in tiles of kManyRows rows, and the
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

constexpr int kFewRows = 32;
constexpr int kFewStep = 128;   // tokens of one step of a workgroup
constexpr int kManyRows = 128;  // rows of one tile
constexpr int kManyStep = 64;   // tokens of one step
constexpr int kMaxSequences = 4096;
constexpr int kMaxGroups = 256;
constexpr int kMaxHeadDim = 256;

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
  // Parts of split rows, each row padded_dim floats relative to its maximum:
  // two slots of few_rows rows a workgroup of attend_few, many_parts slots of
  // kManyRows rows, and with groups a row for every (token, head), for what
  // attend_few did not cut; then the (maximum in powers of two, sum) of each.
  float* parts = nullptr;
  // Filled by PlanAttend.
  int32_t padded_dim = 0;
  int32_t few_grid = 0;    // workgroups of attend_few, 0: not launched
  int32_t few_rows = 0;    // rows of its slots (16 or 32)
  int32_t many_grid = 0;   // workgroups of attend_many, 0: not launched
  int32_t many_target = 0; // items that attend_many is split into where rows are few
  int32_t many_parts = 0;
  int64_t part_rows = 0;
  bool join = false;
};

// Sizes of the launches of a call (from its shapes only). Returns the bytes of
// `parts`.
int64_t PlanAttend(AttendLaunch* l);

// Every address range must have been checked and PlanAttend called.
hipError_t LaunchAttend(const AttendLaunch& l, hipStream_t stream);

// The parts, by translation unit.
hipError_t LaunchAttendFew(const AttendLaunch& l, hipStream_t stream);
hipError_t LaunchAttendMany(const AttendLaunch& l, hipStream_t stream);
hipError_t LaunchAttendJoin(const AttendLaunch& l, hipStream_t stream);

}  // namespace kvx

#endif  // KVX_KERNELS_ATTEND_H_
