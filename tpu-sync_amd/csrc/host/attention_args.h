// Checks of the arguments of the operators that fill and read the paged pool,
// and their translation into kernel launches. Every argument is checked before
// anything is issued; the contents of device arrays (lengths, starts, tables)
// are bounded by the kernels.
#ifndef KVX_HOST_ATTENTION_ARGS_H_
#define KVX_HOST_ATTENTION_ARGS_H_

#include <cstdint>

#include "../../../include/kvx.h"
#include "../kernels/append_kv.h"
#include "../kernels/attend.h"
#include "../kernels/norm_rope.h"
#include "status.h"

namespace kvx {

// One storage of a pool.
struct PoolStorage {
  uint64_t base = 0;
  int64_t bytes = 0;
  int64_t block_bytes = 0;
};

// The pool that a call names storages of; `find` returns false for a layer or
// shard that it does not have.
struct PoolSource {
  int device = 0;
  bool device_backed = true;
  const void* context = nullptr;
  bool (*find)(const void* context, int64_t layer, int64_t shard, PoolStorage* out) = nullptr;
};

// *launch->tokens == 0 on success: nothing to do.
Status CheckNormRope(const kvx_norm_rope_args& a, NormRopeLaunch* out);
Status CheckAppendKv(const PoolSource& pool, const kvx_append_kv_args& a, AppendLaunch* out);
// With `workspace_bytes`, sizes the workspace and leaves addresses unchecked.
Status CheckAttend(const PoolSource& pool, const kvx_attend_args& a, AttendLaunch* out,
                   int64_t* workspace_bytes);

}  // namespace kvx

#endif  // KVX_HOST_ATTENTION_ARGS_H_
