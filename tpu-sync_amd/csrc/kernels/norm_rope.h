// Host-side interface of the norm + rotation kernel (gfx950).
#ifndef KVX_KERNELS_NORM_ROPE_H_
#define KVX_KERNELS_NORM_ROPE_H_

#include <hip/hip_runtime_api.h>

#include <cstdint>

#include "kv_element.h"

namespace kvx {

// Heads of one kind: [tokens][heads][head_dim], each dimension at a stride
// of its own (in elements), the last one contiguous.
struct HeadRows {
  const void* in = nullptr;
  void* out = nullptr;
  const void* weight = nullptr;  // [head_dim], or null: no norm
  int64_t in_token = 0, in_head = 0, out_token = 0, out_head = 0;
  int32_t heads = 0;
};

struct NormRopeLaunch {
  HeadRows q, k;  // k.heads may be 0
  const void* positions = nullptr;
  const float* inv_freq = nullptr;  // [rotary_dim / 2]
  int32_t tokens = 0;
  int32_t head_dim = 0;    // 1..256
  int32_t rotary_dim = 0;  // even, 0..head_dim
  int32_t type = kBf16;    // of in and out
  bool weight_f32 = false;
  bool positions_64 = false;
  bool interleaved = false;
  float eps = 0;
};

// Every address range must have been checked.
hipError_t LaunchNormRope(const NormRopeLaunch& l, hipStream_t stream);

}  // namespace kvx

#endif  // KVX_KERNELS_NORM_ROPE_H_
