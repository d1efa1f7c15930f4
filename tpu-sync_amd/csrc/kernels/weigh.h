// Host-side interface of the kernels that add up what attention each cached token
// got (gfx950).
#ifndef KVX_KERNELS_WEIGH_H_
#define KVX_KERNELS_WEIGH_H_

#include "attend.h"

namespace kvx {

struct WeighLaunch {
  // Queries, keys, batch, scale and types (no values, no groups, no results).
  AttendLaunch attend;
  const float* lse = nullptr;       // [tokens][q_heads]
  float* weights = nullptr;         // [num_blocks][k_heads][block_tokens]
  const int32_t* begins = nullptr;  // [sequences]: first token weighed, or null: 0
  const int32_t* weighed = nullptr;  // [sequences]: tokens that hold a weight, or null: all
  float decay = 1.0f;
  // Sums of cut tiles: two slots of WeighTile floats a worker.
  float* parts = nullptr;
};

// Tokens of a tile of the kernel for many rows: 64 for every wave, whose keys fill half
// of its registers.
constexpr int WeighTile(int padded_dim) { return padded_dim <= 128 ? 256 : 128; }
constexpr int kWeighRows = 64;   // rows that they meet at once

// Sizes of the launches of a call (from its shapes only). Returns the bytes of `parts`.
int64_t PlanWeigh(WeighLaunch* l);

// Every address range must have been checked and PlanWeigh called.
hipError_t LaunchWeigh(const WeighLaunch& l, hipStream_t stream);

}  // namespace kvx

#endif  // KVX_KERNELS_WEIGH_H_
