// What the entry points of the operators on the paged pool share: a manager's pool
// as the checks see it, and a launch on its device.
#ifndef KVX_CAPI_POOL_SOURCE_H_
#define KVX_CAPI_POOL_SOURCE_H_

#include "../host/attention_args.h"
#include "../host/hip_util.h"
#include "capi_internal.h"

namespace kvx_capi {

inline bool FindStorage(const void* context, int64_t layer, int64_t shard, kvx::PoolStorage* out) {
  const auto* m = static_cast<const kvx::KVCacheManager*>(context);
  if (layer < 0 || shard < 0) return false;
  out->block_bytes = 0;
  if (!m->DeviceStorage(static_cast<size_t>(layer), static_cast<size_t>(shard), &out->base,
                        &out->bytes)) {
    return false;
  }
  out->block_bytes = m->LayerBlockByteSize(static_cast<size_t>(layer));
  return out->block_bytes > 0;
}

inline kvx::PoolSource Source(const kvx_manager* m) {
  kvx::PoolSource p;
  p.device = m->impl->device();
  p.device_backed = m->impl->device_backed();
  p.context = m->impl.get();
  p.find = FindStorage;
  return p;
}

// Runs `launch` with `device` current.
template <class F>
int OnDevice(int device, F launch) {
  kvx::DeviceGuard dg(device);
  if (!dg.ok()) return Fail(KVX_INTERNAL, "hipSetDevice failed");
  return Done(kvx::HipStatus(launch(), "kernel launch"));
}

}  // namespace kvx_capi

#endif  // KVX_CAPI_POOL_SOURCE_H_
