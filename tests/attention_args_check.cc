// Checks of the arguments of the paged-attention operators on the CPU, no GPU
// calls: a pool and an address map of their own making stand in for the
// manager and the HIP runtime, and every bad argument must be refused with
// INVALID_ARGUMENT (or the code given) and a message that names it. Good ones
// pass the checks and give the launch's sizes; nothing is launched.
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>

#include "attention_args.h"
#include "device_memory.h"
#include "kvx.h"

namespace {

constexpr uint64_t kDev = 0x7f0000000000ull;  // device 0, 4 GiB
constexpr uint64_t kDevSize = 4ull << 30;
constexpr uint64_t kDev1 = 0x7e0000000000ull;  // device 1
constexpr uint64_t kHost = 0x600000000000ull;

kvx::AddressInfo FakeQuery(uint64_t a) {
  kvx::AddressInfo i;
  if (a >= kDev && a < kDev + kDevSize) {
    i = {kvx::MemKind::kDevice, 0, kDev, kDevSize};
  } else if (a >= kDev1 && a < kDev1 + (1ull << 30)) {
    i = {kvx::MemKind::kDevice, 1, kDev1, 1ull << 30};
  } else if (a >= kHost && a < kHost + (1ull << 30)) {
    i = {kvx::MemKind::kHost, 0, 0, 0};
  }
  return i;
}

int failures = 0;

void Refused(const kvx::Status& s, const char* needle, const char* what, int code = 3) {
  if (static_cast<int>(s.code()) != code || s.message().find(needle) == std::string::npos) {
    std::printf("FAIL %s: code %d, message '%s' (want %d with '%s')\n", what,
                static_cast<int>(s.code()), s.message().c_str(), code, needle);
    ++failures;
  }
}

void Passes(const kvx::Status& s, const char* what) {
  if (!s.ok()) {
    std::printf("FAIL %s: '%s'\n", what, s.message().c_str());
    ++failures;
  }
}

// 100 blocks of [16][2][64]: layers 0, 1 bf16; 2, 3 e4m3; 4, 5 their scales.
bool Find(const void*, int64_t layer, int64_t shard, kvx::PoolStorage* out) {
  if (layer < 0 || layer > 5 || shard != 0) return false;
  const int64_t block[] = {4096, 4096, 2048, 2048, 8, 8};
  *out = {kDev + (2ull << 30) + static_cast<uint64_t>(layer) * (1 << 20), block[layer] * 100,
          block[layer]};
  return true;
}

kvx::PoolSource Pool() {
  kvx::PoolSource p;
  p.find = Find;
  return p;
}

uint64_t At(int64_t mib) { return kDev + static_cast<uint64_t>(mib) * (1 << 20); }

kvx_norm_rope_args GoodNorm() {
  kvx_norm_rope_args a;
  std::memset(&a, 0, sizeof(a));
  a.dtype = KVX_BF16;
  a.tokens = 10;
  a.q_heads = 8;
  a.k_heads = 2;
  a.head_dim = 64;
  a.rotary_dim = 64;
  a.q = At(1);
  a.k = a.q + 8 * 64 * 2;  // q, k, v side by side
  a.q_token_stride = a.k_token_stride = 12 * 64;
  a.q_head_stride = a.k_head_stride = a.q_out_head_stride = a.k_out_head_stride = 64;
  a.q_out = At(2);
  a.k_out = At(3);
  a.q_out_token_stride = 8 * 64;
  a.k_out_token_stride = 2 * 64;
  a.positions = At(4);
  a.inv_freq = At(5);
  a.eps = 1e-6f;
  return a;
}

kvx_paged_cache GoodCache() {
  kvx_paged_cache c;
  std::memset(&c, 0, sizeof(c));
  c.v_layer = 1;
  c.dtype = KVX_BF16;
  c.block_tokens = 16;
  c.heads = 2;
  c.head_dim = 64;
  return c;
}

kvx_paged_batch GoodBatch() {
  kvx_paged_batch b;
  std::memset(&b, 0, sizeof(b));
  b.tables = At(10);
  b.table_stride = b.table_width = 6;
  b.lengths = At(11);
  b.starts = At(12);
  b.sequences = 3;
  return b;
}

kvx_append_kv_args GoodAppend() {
  kvx_append_kv_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = GoodCache();
  a.batch = GoodBatch();
  a.tokens = 10;
  a.dtype = KVX_BF16;
  a.rotary_dim = 64;
  a.k = At(1);
  a.v = At(2);
  a.k_token_stride = a.v_token_stride = 128;
  a.k_head_stride = a.v_head_stride = 64;
  a.inv_freq = At(5);
  return a;
}

kvx_attend_args GoodAttend() {
  kvx_attend_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = GoodCache();
  a.batch = GoodBatch();
  a.batch.table_stride = a.batch.table_width = 20;  // more than one step of tokens
  a.tokens = 10;
  a.dtype = KVX_BF16;
  a.q_heads = 8;
  a.q = At(1);
  a.out = At(2);
  a.q_token_stride = a.out_token_stride = 512;
  a.q_head_stride = a.out_head_stride = 64;
  a.scale = 0.125f;
  a.workspace = At(100);
  a.workspace_bytes = 512 << 20;
  return a;
}

kvx::Status Norm(const std::function<void(kvx_norm_rope_args&)>& change) {
  kvx_norm_rope_args a = GoodNorm();
  change(a);
  kvx::NormRopeLaunch l;
  return kvx::CheckNormRope(a, &l);
}

kvx::Status Append(const std::function<void(kvx_append_kv_args&)>& change) {
  kvx_append_kv_args a = GoodAppend();
  change(a);
  kvx::AppendLaunch l;
  return kvx::CheckAppendKv(Pool(), a, &l);
}

kvx::Status Attend(const std::function<void(kvx_attend_args&)>& change) {
  kvx_attend_args a = GoodAttend();
  change(a);
  kvx::AttendLaunch l;
  return kvx::CheckAttend(Pool(), a, &l, nullptr);
}

void NormRope() {
  using A = kvx_norm_rope_args;
  Passes(Norm([](A&) {}), "norm");
  Passes(Norm([](A& a) { a.q_out = a.q; a.q_out_token_stride = a.q_token_stride; }), "q in place");
  Passes(Norm([](A& a) {
           a.q_out = a.q;
           a.k_out = a.k;
           a.q_out_token_stride = a.k_out_token_stride = a.q_token_stride;
         }),
         "fused in place");
  Passes(Norm([](A& a) { a.tokens = 0; a.q = a.k = a.q_out = a.k_out = a.positions = 0; }),
         "no tokens");
  Passes(Norm([](A& a) { a.k_heads = 0; a.k = a.k_out = 0; }), "no keys");
  Passes(Norm([](A& a) { a.q_head_stride = 0; }), "expanded input");
  Refused(Norm([](A& a) { a.dtype = KVX_E4M3; }), "dtype", "norm: e4m3");
  Refused(Norm([](A& a) { a.tokens = -1; }), "tokens", "norm: negative tokens");
  Refused(Norm([](A& a) { a.q_heads = -1; }), "heads", "norm: negative heads");
  Refused(Norm([](A& a) { a.head_dim = 257; }), "head_dim", "norm: wide head");
  Refused(Norm([](A& a) { a.head_dim = 0; }), "head_dim", "norm: no head");
  Refused(Norm([](A& a) { a.rotary_dim = 66; }), "rotary_dim", "norm: rotary over head_dim");
  Refused(Norm([](A& a) { a.rotary_dim = 7; }), "rotary_dim", "norm: odd rotary");
  Refused(Norm([](A& a) { a.positions = 0; }), "positions", "norm: no positions");
  Refused(Norm([](A& a) { a.positions_64 = 1; a.positions += 4; }), "positions", "norm: odd int64");
  Refused(Norm([](A& a) { a.inv_freq = 0; }), "inv_freq", "norm: no frequencies");
  Refused(Norm([](A& a) { a.q = kHost; }), "q: host", "norm: host q");
  Refused(Norm([](A& a) { a.k_out = kDev1; }), "device 1", "norm: other device");
  Refused(Norm([](A& a) { a.q_out = kDev + kDevSize - 64; }), "past the end", "norm: overrun");
  Refused(Norm([](A& a) { a.q_token_stride = -1; }), "stride", "norm: negative stride");
  Refused(Norm([](A& a) { a.q_token_stride = INT64_MAX / 2; }), "overflow", "norm: huge stride");
  Refused(Norm([](A& a) { a.q += 1; }), "multiple", "norm: half an element off");
  Refused(Norm([](A& a) { a.q_out = a.q + 128; a.q_out_token_stride = a.q_token_stride; }),
          "overlaps", "norm: shifted onto the input");
  Refused(Norm([](A& a) { a.q_out = a.q; }), "overlaps", "norm: in place, other strides");
  Refused(Norm([](A& a) { a.q_out_token_stride = 64; }), "rows overlap", "norm: rows overlap");
  Refused(Norm([](A& a) { a.q_out_head_stride = 0; }), "rows overlap", "norm: expanded output");
  Refused(Norm([](A& a) { a.k_out = a.q_out + 1024; }), "overlaps", "norm: outputs overlap");
  Refused(Norm([](A& a) { a.k_out = a.q; a.k_out_token_stride = a.q_token_stride; }), "overlaps q",
          "norm: k onto q");
  Refused(Norm([](A& a) { a.q_weight = At(6); a.weight_dtype = KVX_F16; }), "q_weight",
          "norm: weight type");
  Refused(Norm([](A& a) { a.k_weight = kHost; }), "k_weight: host", "norm: host weight");
  Refused(Norm([](A& a) { a.q_weight = At(6); a.eps = NAN; }), "eps", "norm: eps");
  Refused(Norm([](A& a) { a.q_weight = At(6); a.eps = -1; }), "eps", "norm: negative eps");
  Refused(Norm([](A& a) { a.tokens = 1 << 28; }), "2^29", "norm: too many rows");
}

void AppendKv() {
  using A = kvx_append_kv_args;
  const auto e4m3 = [](A& a) {
    a.cache.k_layer = 2;
    a.cache.v_layer = 3;
    a.cache.k_scale_layer = 4;
    a.cache.v_scale_layer = 5;
    a.cache.dtype = KVX_E4M3;
  };
  Passes(Append([](A&) {}), "append");
  Passes(Append(e4m3), "append e4m3");
  Passes(Append([](A& a) { a.batch.starts = 0; a.tokens = 3; }), "append: single tokens");
  Passes(Append([](A& a) { a.batch.sequences = 0; a.batch.tables = a.batch.lengths = 0; }),
         "append: no sequences");
  Refused(Append([](A& a) { a.batch.starts = 0; }), "starts", "append: tokens without starts");
  Refused(Append([](A& a) { a.dtype = KVX_F32; }), "dtype", "append: fp32");
  Refused(Append([](A& a) { a.dtype = KVX_F16; }), "cache", "append: other 16-bit cache");
  Refused(Append([](A& a) { a.cache.v_layer = 9; }), "layer", "append: layer", 11);
  Refused(Append([](A& a) { a.cache.shard = 1; }), "shard", "append: shard", 11);
  Refused(Append([](A& a) { a.cache.v_layer = 0; }), "of their own", "append: K on V");
  Refused(Append([](A& a) { a.cache.heads = 4; }), "bytes", "append: block shape");
  Refused(Append([](A& a) { a.cache.v_layer = 2; }), "bytes", "append: other block size");
  Refused(Append([](A& a) { a.cache.heads = 0; }), "heads", "append: no heads");
  Refused(Append([](A& a) { a.cache.block_tokens = 0; }), "block_tokens", "append: no slots");
  Refused(Append([&](A& a) { e4m3(a); a.cache.v_scale_layer = 4; }), "of their own",
          "append: one scale table");
  Refused(Append([&](A& a) { e4m3(a); a.cache.k_scale_layer = 0; }), "scale tables",
          "append: scales of another size");
  Refused(Append([&](A& a) { e4m3(a); a.cache.k_scale_layer = -1; }), "scale layer",
          "append: no scales", 11);
  Refused(Append([](A& a) { a.k = kHost; }), "k: host", "append: host k");
  Refused(Append([](A& a) { a.v = 0; }), "v: null", "append: null v");
  Refused(Append([](A& a) { a.k = At(2048); }), "overlaps the cache", "append: from the cache");
  Refused(Append([](A& a) { a.batch.tables = kHost; }), "tables: host", "append: host tables");
  Refused(Append([](A& a) { a.batch.tables = kDev + kDevSize - 16; }), "past the end",
          "append: tables overrun");
  Refused(Append([](A& a) { a.batch.lengths += 2; }), "lengths: unaligned", "append: lengths");
  Refused(Append([](A& a) { a.batch.sequences = 4097; }), "sequences", "append: sequences");
  Refused(Append([](A& a) { a.batch.table_width = 1 << 27; }), "2^30", "append: table too wide");
  Refused(Append([](A& a) { a.batch.table_stride = -1; }), "stride", "append: table stride");
  Refused(Append([](A& a) { a.positions = kHost; }), "positions: host", "append: host positions");
  Refused(Append([](A& a) { a.rotary_dim = 66; }), "rotary_dim", "append: rotary");
  kvx::PoolSource host = Pool();
  host.device_backed = false;
  kvx::AppendLaunch l;
  Refused(kvx::CheckAppendKv(host, GoodAppend(), &l), "device-backed", "append: host manager", 9);
}

void AttendArgs() {
  using A = kvx_attend_args;
  Passes(Attend([](A&) {}), "attend");
  Passes(Attend([](A& a) { a.out = a.q; }), "attend: in place");
  Passes(Attend([](A& a) { a.groups = 2; a.group_starts = At(20); a.prefix_lengths = At(21); }),
         "attend: groups");
  Refused(Attend([](A& a) { a.q_heads = 7; }), "q_heads", "attend: heads");
  Refused(Attend([](A& a) { a.q_heads = 0; }), "q_heads", "attend: no heads");
  Refused(Attend([](A& a) { a.scale = 0; }), "scale", "attend: zero scale");
  Refused(Attend([](A& a) { a.scale = -1; }), "scale", "attend: negative scale");
  Refused(Attend([](A& a) { a.scale = INFINITY; }), "scale", "attend: infinite scale");
  Refused(Attend([](A& a) { a.cache.head_dim = 4; a.cache.heads = 32; a.q_heads = 32; }),
          "multiple of 8", "attend: head_dim");
  Refused(Attend([](A& a) { a.groups = 257; }), "groups", "attend: groups");
  Refused(Attend([](A& a) { a.groups = 1; a.prefix_lengths = At(21); }), "group_starts",
          "attend: no group starts");
  Refused(Attend([](A& a) { a.out = a.q + 1024; }), "overlaps q", "attend: shifted onto q");
  Refused(Attend([](A& a) { a.out_token_stride = 64; }), "rows overlap", "attend: output rows");
  Refused(Attend([](A& a) { a.lse = a.out + 64; }), "lse: overlaps", "attend: lse on out");
  Refused(Attend([](A& a) { a.workspace_bytes = 100; }), "workspace", "attend: small workspace");
  Refused(Attend([](A& a) { a.workspace += 4; }), "aligned", "attend: unaligned workspace");
  Refused(Attend([](A& a) { a.workspace = kHost; }), "workspace: host", "attend: host workspace");
  Refused(Attend([](A& a) { a.out = kDev1; }), "device 1", "attend: out on device 1");

  // Storages that do not start on 16 bytes: attend reads them in such pieces.
  kvx::PoolSource odd;
  odd.find = [](const void* c, int64_t layer, int64_t shard, kvx::PoolStorage* out) {
    const bool found = Find(c, layer, shard, out);
    out->base += 8;
    out->bytes -= out->block_bytes;
    return found;
  };
  {
    const kvx_attend_args good = GoodAttend();
    kvx::AttendLaunch launch;
    Refused(kvx::CheckAttend(odd, good, &launch, nullptr), "aligned to 16", "attend: odd storages");
  }

  // The workspace's size is the same with and without addresses, and nothing
  // is needed where no row can be cut.
  kvx_attend_args a = GoodAttend();
  kvx::AttendLaunch l, m;
  int64_t bytes = -1, bare = -1;
  a.batch.table_width = 600;
  a.batch.table_stride = 600;
  Passes(kvx::CheckAttend(Pool(), a, &l, &bytes), "attend: workspace");
  Passes(kvx::CheckAttend(Pool(), a, &m, nullptr), "attend: launch");
  a.q = a.out = a.batch.tables = a.batch.lengths = a.workspace = 0;
  a.batch.starts = 1;
  Passes(kvx::CheckAttend(Pool(), a, &l, &bare), "attend: workspace, no addresses");
  if (bytes <= 0 || bytes != bare || l.few_grid != m.few_grid || l.many_grid != m.many_grid ||
      l.part_rows != m.part_rows) {
    std::printf("FAIL attend: workspace of %lld and %lld bytes\n", static_cast<long long>(bytes),
                static_cast<long long>(bare));
    ++failures;
  }
  a.batch.table_width = 2;  // 32 tokens
  a.batch.starts = 0;
  a.tokens = 3;
  Passes(kvx::CheckAttend(Pool(), a, &l, &bytes), "attend: one step");
  if (bytes != 0 || l.join_grid != 0) {
    std::printf("FAIL attend: one step needs %lld bytes\n", static_cast<long long>(bytes));
    ++failures;
  }
  a.batch.table_width = 1 << 26;
  a.tokens = 1 << 24;
  a.batch.starts = 1;
  Refused(kvx::CheckAttend(Pool(), a, &l, &bytes), "too large", "attend: too large");
}

}  // namespace

int main() {
  kvx::SetAddressQueryForTesting(FakeQuery);
  NormRope();
  AppendKv();
  AttendArgs();
  kvx::SetAddressQueryForTesting(nullptr);
  if (failures == 0) std::printf("attention argument checks: all passed\n");
  return failures == 0 ? 0 : 1;
}
