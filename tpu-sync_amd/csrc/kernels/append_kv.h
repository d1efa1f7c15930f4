// Host-side interface of the kernels that store new keys and values into the
// paged pool (gfx950).
#ifndef KVX_KERNELS_APPEND_KV_H_
#define KVX_KERNELS_APPEND_KV_H_

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstdint>

#include "kv_element.h"
#include "tiled_copy.h"

namespace kvx {

struct AppendLaunch {
  BatchView batch;
  FastDivU32 block_div;  // by batch.block_tokens
  // [tokens][heads][head_dim], the last dimension contiguous.
  const void* k = nullptr;
  const void* v = nullptr;
  int64_t k_token = 0, k_head = 0, v_token = 0, v_head = 0;
  // Storages [num_blocks][block_tokens][heads][head_dim]; in e4m3 with scales
  // [num_blocks][heads].
  void* k_pool = nullptr;
  void* v_pool = nullptr;
  float* k_scales = nullptr;
  float* v_scales = nullptr;
  const void* k_weight = nullptr;   // [head_dim], or null: no norm
  const void* positions = nullptr;  // of the rotation; null: the places in the cache
  const float* inv_freq = nullptr;  // [rotary_dim / 2]
  int32_t heads = 0;
  int32_t head_dim = 0;
  int32_t rotary_dim = 0;
  int32_t type = kBf16;  // of k and v (and of the pool unless it is e4m3)
  bool e4m3 = false;
  bool weight_f32 = false;
  bool positions_64 = false;
  bool interleaved = false;
  float eps = 0;
};

// The e4m3 kernel's workgroups, one for every block that the tokens can touch
// (whole ones, and a first and a last part of each sequence), and its threads.
inline int64_t MostBlocks(const AppendLaunch& l) {
  const int64_t tokens = l.batch.tokens, sequences = l.batch.sequences;
  return l.batch.starts == nullptr
             ? sequences
             : std::min(tokens, tokens / l.batch.block_tokens + 2 * sequences);
}
inline int BlockThreads(const AppendLaunch& l) { return 64 * std::min(l.heads, kRowThreads / 64); }

// Every address range must have been checked.
hipError_t LaunchAppendKv(const AppendLaunch& l, hipStream_t stream);

}  // namespace kvx

#endif  // KVX_KERNELS_APPEND_KV_H_
