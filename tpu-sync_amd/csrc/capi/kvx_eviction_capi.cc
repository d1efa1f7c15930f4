// extern "C" entry points of the operators that weigh, choose and move the tokens of
// the paged pool: checks (host/eviction_args.cc), then launches on the caller's stream.
#include "../host/eviction_args.h"
#include "pool_source.h"

namespace {

using kvx_capi::Fail;
using kvx_capi::OnDevice;
using kvx_capi::Source;

}  // namespace

extern "C" {

int kvx_manager_weigh_workspace(kvx_manager* m, const kvx_weigh_args* args, int64_t* bytes) {
  if (m == nullptr || args == nullptr || bytes == nullptr) {
    return Fail(KVX_INVALID_ARGUMENT, "null manager, arguments or output");
  }
  kvx::WeighLaunch l;
  return kvx_capi::Done(kvx::CheckWeigh(Source(m), *args, &l, bytes));
}

int kvx_manager_weigh(kvx_manager* m, const kvx_weigh_args* args, void* stream) {
  if (m == nullptr || args == nullptr) {
    return Fail(KVX_INVALID_ARGUMENT, "null manager or arguments");
  }
  kvx::WeighLaunch l;
  const kvx::Status st = kvx::CheckWeigh(Source(m), *args, &l, nullptr);
  if (!st.ok()) return Fail(st);
  if (l.attend.batch.tokens == 0) return KVX_OK;
  return OnDevice(m->impl->device(),
                  [&] { return kvx::LaunchWeigh(l, static_cast<hipStream_t>(stream)); });
}

int kvx_choose_kept(const kvx_choose_kept_args* args, void* stream) {
  if (args == nullptr) return Fail(KVX_INVALID_ARGUMENT, "null arguments");
  kvx::ChooseLaunch l;
  const kvx::Status st = kvx::CheckChooseKept(*args, &l);
  if (!st.ok()) return Fail(st);
  if (l.batch.sequences == 0) return KVX_OK;
  return OnDevice(args->device,
                  [&] { return kvx::LaunchChooseKept(l, static_cast<hipStream_t>(stream)); });
}

int kvx_manager_compact(kvx_manager* m, const kvx_compact_args* args, void* stream) {
  if (m == nullptr || args == nullptr) {
    return Fail(KVX_INVALID_ARGUMENT, "null manager or arguments");
  }
  kvx::CompactLaunch l;
  const kvx::Status st = kvx::CheckCompact(Source(m), *args, &l);
  if (!st.ok()) return Fail(st);
  if (l.batch.sequences == 0) return KVX_OK;
  return OnDevice(m->impl->device(),
                  [&] { return kvx::LaunchCompact(l, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
