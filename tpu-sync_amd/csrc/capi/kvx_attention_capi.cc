// extern "C" entry points of the operators that fill and read the paged pool:
// checks (host/attention_args.cc), then launches on the caller's stream.
#include "pool_source.h"

namespace {

using kvx_capi::Done;
using kvx_capi::Fail;
using kvx_capi::OnDevice;
using kvx_capi::Source;

}  // namespace

extern "C" {

int kvx_norm_rope(const kvx_norm_rope_args* args, void* stream) {
  if (args == nullptr) return Fail(KVX_INVALID_ARGUMENT, "null arguments");
  kvx::NormRopeLaunch l;
  const kvx::Status st = kvx::CheckNormRope(*args, &l);
  if (!st.ok()) return Fail(st);
  if (l.tokens == 0) return KVX_OK;
  return OnDevice(args->device,
                  [&] { return kvx::LaunchNormRope(l, static_cast<hipStream_t>(stream)); });
}

int kvx_manager_append_kv(kvx_manager* m, const kvx_append_kv_args* args, void* stream) {
  if (m == nullptr || args == nullptr) {
    return Fail(KVX_INVALID_ARGUMENT, "null manager or arguments");
  }
  kvx::AppendLaunch l;
  const kvx::Status st = kvx::CheckAppendKv(Source(m), *args, &l);
  if (!st.ok()) return Fail(st);
  if (l.batch.tokens == 0) return KVX_OK;
  return OnDevice(m->impl->device(),
                  [&] { return kvx::LaunchAppendKv(l, static_cast<hipStream_t>(stream)); });
}

int kvx_manager_attend_workspace(kvx_manager* m, const kvx_attend_args* args, int64_t* bytes) {
  if (m == nullptr || args == nullptr || bytes == nullptr) {
    return Fail(KVX_INVALID_ARGUMENT, "null manager, arguments or output");
  }
  kvx::AttendLaunch l;
  return Done(kvx::CheckAttend(Source(m), *args, &l, bytes));
}

int kvx_manager_attend(kvx_manager* m, const kvx_attend_args* args, void* stream) {
  if (m == nullptr || args == nullptr) {
    return Fail(KVX_INVALID_ARGUMENT, "null manager or arguments");
  }
  kvx::AttendLaunch l;
  const kvx::Status st = kvx::CheckAttend(Source(m), *args, &l, nullptr);
  if (!st.ok()) return Fail(st);
  if (l.batch.tokens == 0) return KVX_OK;
  return OnDevice(m->impl->device(),
                  [&] { return kvx::LaunchAttend(l, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
