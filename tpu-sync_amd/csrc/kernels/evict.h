// Host-side interface of the kernels that choose the tokens of a cache to keep and
// move them to the front of their sequences (gfx950).
#ifndef KVX_KERNELS_EVICT_H_
#define KVX_KERNELS_EVICT_H_

#include <hip/hip_runtime_api.h>

#include <cstdint>

#include "kv_element.h"
#include "tiled_copy.h"

namespace kvx {

struct ChooseLaunch {
  BatchView batch;       // starts and tokens are not used
  FastDivU32 block_div;  // by batch.block_tokens
  const float* weights = nullptr;   // [num_blocks][heads][block_tokens]
  const int32_t* begins = nullptr;  // [sequences] or null: 0
  int32_t* kept = nullptr;          // [sequences][heads][budget]
  int32_t* new_lengths = nullptr;   // [sequences] or null
  int32_t heads = 0, budget = 0, recent = 0;
};

hipError_t LaunchChooseKept(const ChooseLaunch& l, hipStream_t stream);

struct CompactLaunch {
  BatchView batch;  // tables alone
  FastDivU32 block_div;
  const int32_t* kept = nullptr;  // [sequences][heads][budget]
  int64_t kept_sequence = 0, kept_head = 0, kept_place = 0;  // its strides
  int32_t budget = 0;
  // Storages and their scales, laid out as PoolKind says.
  void* k_pool = nullptr;
  void* v_pool = nullptr;
  void* k_scales = nullptr;
  void* v_scales = nullptr;
  float* weights = nullptr;  // [num_blocks][heads][block_tokens] or null
  int32_t heads = 0, head_dim = 0;
  int32_t pool = kPoolSame;  // PoolKind
};

hipError_t LaunchCompact(const CompactLaunch& l, hipStream_t stream);

// Threads of a workgroup, one for every (sequence, head) and more.
constexpr int kChooseThreads = 1024;
constexpr int kCompactThreads = 256;

}  // namespace kvx

#endif  // KVX_KERNELS_EVICT_H_
