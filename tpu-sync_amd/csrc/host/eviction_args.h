// Checks of the arguments of the operators that weigh, choose and move the tokens of
// the paged pool, and their translation into kernel launches (as attention_args.h).
#ifndef KVX_HOST_EVICTION_ARGS_H_
#define KVX_HOST_EVICTION_ARGS_H_

#include "../kernels/evict.h"
#include "../kernels/weigh.h"
#include "attention_args.h"

namespace kvx {

// attend.batch.tokens == 0 on success: nothing to do.
// With `workspace_bytes`, sizes the workspace and leaves addresses unchecked.
Status CheckWeigh(const PoolSource& pool, const kvx_weigh_args& a, WeighLaunch* out,
                  int64_t* workspace_bytes);
// batch.sequences == 0 on success: nothing to do.
Status CheckChooseKept(const kvx_choose_kept_args& a, ChooseLaunch* out);
Status CheckCompact(const PoolSource& pool, const kvx_compact_args& a, CompactLaunch* out);

}  // namespace kvx

#endif  // KVX_HOST_EVICTION_ARGS_H_
