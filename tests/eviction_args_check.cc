// Checks of the arguments of weigh, choose_kept and compact, and of 4-bit caches, on the
// CPU, no GPU calls (as attention_args_check.cc).
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>

#include "attention_args.h"
#include "device_memory.h"
#include "eviction_args.h"
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

// 100 blocks of 16 tokens, 2 heads of 64: layers 0, 1 bf16; 2, 3 e4m3 with scales 4, 5; 6, 7
// in 4 bits with scales 8, 9; 10 in 4 bits, 8 bytes off.
bool Find(const void*, int64_t layer, int64_t shard, kvx::PoolStorage* out) {
  if (layer < 0 || layer > 10 || shard != 0) return false;
  const int64_t block[] = {4096, 4096, 2048, 2048, 8, 8, 1024, 1024, 64, 64, 1024};
  *out = {kDev + (2ull << 30) + static_cast<uint64_t>(layer) * (1 << 20) + (layer == 10 ? 8 : 0),
          block[layer] * 100, block[layer]};
  return true;
}

kvx::PoolSource Pool() {
  kvx::PoolSource p;
  p.find = Find;
  return p;
}

uint64_t At(int64_t mib) { return kDev + static_cast<uint64_t>(mib) * (1 << 20); }

kvx_paged_cache Cache(int32_t type) {
  kvx_paged_cache c;
  std::memset(&c, 0, sizeof(c));
  c.k_layer = type == KVX_FP4 ? 6 : type == KVX_E4M3 ? 2 : 0;
  c.v_layer = c.k_layer + 1;
  c.k_scale_layer = type == KVX_FP4 ? 8 : 4;
  c.v_scale_layer = c.k_scale_layer + 1;
  c.dtype = type;
  c.block_tokens = 16;
  c.heads = 2;
  c.head_dim = 64;
  return c;
}

kvx_paged_batch Batch() {
  kvx_paged_batch b;
  std::memset(&b, 0, sizeof(b));
  b.tables = At(10);
  b.table_stride = b.table_width = 20;
  b.lengths = At(11);
  b.starts = At(12);
  b.sequences = 3;
  return b;
}

kvx_weigh_args GoodWeigh(int32_t type) {
  kvx_weigh_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = Cache(type);
  a.batch = Batch();
  a.tokens = 40;
  a.dtype = KVX_BF16;
  a.q_heads = 8;
  a.q = At(1);
  a.q_token_stride = 512;
  a.q_head_stride = 64;
  a.lse = At(2);
  a.weights = At(3);
  a.blocks = 100;
  a.begins = At(13);
  a.scale = 0.125f;
  a.decay = 0.9f;
  a.workspace = At(100);
  a.workspace_bytes = 64 << 20;
  return a;
}

kvx::Status Weigh(int32_t type, const std::function<void(kvx_weigh_args&)>& change) {
  kvx_weigh_args a = GoodWeigh(type);
  change(a);
  kvx::WeighLaunch l;
  return kvx::CheckWeigh(Pool(), a, &l, nullptr);
}

void WeighArgs() {
  using A = kvx_weigh_args;
  for (int32_t type : {KVX_BF16, KVX_E4M3, KVX_FP4}) {
    const auto run = [&](const std::function<void(A&)>& f) { return Weigh(type, f); };
    Passes(run([](A&) {}), "weigh");
    Passes(run([](A& a) { a.begins = 0; }), "weigh: no begins");
    Passes(run([](A& a) { a.blocks = 101; }), "weigh: a larger table");
    Passes(run([](A& a) { a.cache.v_layer = a.cache.v_scale_layer = -1; }), "weigh: keys alone");
    Passes(run([](A& a) { a.batch.sequences = 0; a.batch.tables = a.batch.lengths = 0; }),
           "weigh: no sequences");
    Refused(run([](A& a) { a.blocks = 99; }), "fewer blocks", "weigh: a smaller table");
    Refused(run([](A& a) { a.blocks = 0; }), "blocks", "weigh: no table");
    Refused(run([](A& a) { a.blocks = INT64_MAX; }), "blocks", "weigh: endless table");
    Refused(run([](A& a) { a.weights = 0; }), "weights: null", "weigh: null table");
    Refused(run([](A& a) { a.weights = kHost; }), "weights: host", "weigh: host table");
    Refused(run([](A& a) { a.weights = kDev1; }), "weights", "weigh: table elsewhere");
    Refused(run([](A& a) { a.weights += 2; }), "weights: unaligned", "weigh: odd table");
    Refused(run([](A& a) { a.weights = a.q + 64; }), "overlaps q", "weigh: table on q");
    Refused(run([](A& a) { a.weights = a.lse + 4; }), "overlaps lse", "weigh: table on lse");
    Refused(run([](A& a) { a.weights = a.begins - 8; }), "overlaps begins", "weigh: on begins");
    Refused(run([](A& a) { a.weights = kDev + (2ull << 30) + a.cache.k_layer * (1 << 20); }),
            "overlaps the cache", "weigh: table on the cache");
    Refused(run([](A& a) { a.lse = 0; }), "lse: null", "weigh: null lse");
    Refused(run([](A& a) { a.lse = kHost; }), "lse: host", "weigh: host lse");
    Refused(run([](A& a) { a.begins = kHost; }), "begins: host", "weigh: host begins");
    Refused(run([](A& a) { a.q = kHost; }), "q: host", "weigh: host q");
    Refused(run([](A& a) { a.q_heads = 7; }), "multiple", "weigh: heads");
    Refused(run([](A& a) { a.scale = 0; }), "scale", "weigh: scale");
    Refused(run([](A& a) { a.scale = NAN; }), "scale", "weigh: NaN scale");
    Refused(run([](A& a) { a.decay = -0.1f; }), "decay", "weigh: decay");
    Refused(run([](A& a) { a.decay = NAN; }), "decay", "weigh: NaN decay");
    Refused(run([](A& a) { a.decay = 1.5f; }), "decay", "weigh: growth");
    Refused(run([](A& a) { a.dtype = KVX_F32; }), "dtype", "weigh: fp32");
    Refused(run([](A& a) { a.cache.k_layer = 77; }), "layer", "weigh: layer", 11);
    Refused(run([](A& a) { a.batch.starts = 0; }), "starts", "weigh: tokens without starts");
    Refused(run([](A& a) { a.batch.sequences = 4097; }), "sequences", "weigh: sequences");
    Refused(run([](A& a) { a.workspace_bytes = 4; }), "are needed", "weigh: workspace");
    Refused(run([](A& a) { a.workspace += 8; }), "aligned", "weigh: odd workspace");
    Refused(run([](A& a) { a.workspace = kHost; }), "workspace: host", "weigh: host workspace");
    Refused(run([](A& a) { a.workspace = a.weights; }), "overlaps", "weigh: workspace on the table");
    Refused(run([](A& a) { a.workspace = a.q - 16; }), "overlaps q", "weigh: workspace on q");
  }
  // The workspace's size needs no addresses, and single tokens none of it.
  A a = GoodWeigh(KVX_BF16);
  kvx::WeighLaunch l;
  int64_t bytes = -1;
  a.q = a.lse = a.weights = a.begins = a.workspace = a.batch.tables = a.batch.lengths = 0;
  Passes(kvx::CheckWeigh(Pool(), a, &l, &bytes), "weigh workspace");
  if (bytes <= 0) {
    std::printf("FAIL weigh workspace: %lld bytes\n", static_cast<long long>(bytes));
    ++failures;
  }
  a.batch.starts = 0;
  a.tokens = 3;
  Passes(kvx::CheckWeigh(Pool(), a, &l, &bytes), "weigh workspace of single tokens");
  if (bytes != 0 || l.attend.many_grid != 0) {
    std::printf("FAIL weigh workspace of single tokens: %lld bytes\n",
                static_cast<long long>(bytes));
    ++failures;
  }
  a.batch.table_width = 1 << 26;
  a.tokens = 1 << 25;
  a.batch.starts = 1;
  Refused(kvx::CheckWeigh(Pool(), a, &l, &bytes), "too large", "weigh: too large");
}

void ChooseArgs() {
  using A = kvx_choose_kept_args;
  const auto run = [](const std::function<void(A&)>& change) {
    A a;
    std::memset(&a, 0, sizeof(a));
    a.heads = 2;
    a.block_tokens = 16;
    a.blocks = 100;
    a.weights = At(3);
    a.batch = Batch();
    a.batch.starts = 0;
    a.begins = At(13);
    a.kept = At(20);
    a.new_lengths = At(21);
    a.budget = 50;
    a.recent = 10;
    change(a);
    kvx::ChooseLaunch l;
    return kvx::CheckChooseKept(a, &l);
  };
  Passes(run([](A&) {}), "choose");
  Passes(run([](A& a) { a.begins = a.new_lengths = 0; }), "choose: least arguments");
  Passes(run([](A& a) { a.budget = 0; a.kept = 0; }), "choose: nothing stays");
  Passes(run([](A& a) { a.recent = INT64_MAX; }), "choose: all recent");
  Passes(run([](A& a) { a.batch.sequences = 0; a.batch.tables = a.batch.lengths = a.kept = 0; }),
         "choose: no sequences");
  Refused(run([](A& a) { a.batch.starts = At(12); }), "starts", "choose: starts");
  Refused(run([](A& a) { a.budget = -1; }), "budget", "choose: budget");
  Refused(run([](A& a) { a.budget = 1ll << 31; }), "budget", "choose: endless budget");
  Refused(run([](A& a) { a.recent = -1; }), "recent", "choose: recent");
  Refused(run([](A& a) { a.heads = 0; }), "heads", "choose: heads");
  Refused(run([](A& a) { a.heads = 1025; }), "heads", "choose: many heads");
  Refused(run([](A& a) { a.block_tokens = 0; }), "block_tokens", "choose: blocks");
  Refused(run([](A& a) { a.blocks = 0; }), "blocks", "choose: no blocks");
  Refused(run([](A& a) { a.weights = 0; }), "weights: null", "choose: null table");
  Refused(run([](A& a) { a.weights = kHost; }), "weights: host", "choose: host table");
  Refused(run([](A& a) { a.kept = kHost; }), "kept: host", "choose: host kept");
  Refused(run([](A& a) { a.kept = 0; }), "kept: null", "choose: null kept");
  Refused(run([](A& a) { a.kept = kDev + kDevSize - 8; }), "past the end", "choose: kept overruns");
  Refused(run([](A& a) { a.kept += 1; }), "kept: unaligned", "choose: odd kept");
  Refused(run([](A& a) { a.kept = a.weights; }), "overlaps weights", "choose: kept on weights");
  Refused(run([](A& a) { a.kept = a.batch.tables; }), "overlaps tables", "choose: kept on tables");
  Refused(run([](A& a) { a.kept = a.batch.lengths; }), "overlaps lengths", "choose: kept on lengths");
  Refused(run([](A& a) { a.new_lengths = a.batch.lengths; }), "overlaps lengths",
          "choose: lengths in place");
  Refused(run([](A& a) { a.new_lengths = a.kept + 16; }), "overlaps kept", "choose: lengths on kept");
  Refused(run([](A& a) { a.new_lengths = kHost; }), "new_lengths: host", "choose: host lengths");
  Refused(run([](A& a) { a.begins = kHost; }), "begins: host", "choose: host begins");
  Refused(run([](A& a) { a.batch.lengths = 0; }), "lengths: null", "choose: null lengths");
  Refused(run([](A& a) { a.batch.sequences = 4097; }), "sequences", "choose: sequences");
  Refused(run([](A& a) { a.device = 1; }), "device", "choose: another device");
}

void CompactArgs() {
  using A = kvx_compact_args;
  for (int32_t type : {KVX_BF16, KVX_E4M3, KVX_FP4}) {
    const auto run = [&](const std::function<void(A&)>& change) {
      A a;
      std::memset(&a, 0, sizeof(a));
      a.cache = Cache(type);
      a.tables = At(10);
      a.table_stride = a.table_width = 20;
      a.sequences = 3;
      a.kept = At(20);
      a.kept_sequence_stride = 100;
      a.kept_head_stride = 50;
      a.kept_place_stride = 1;
      a.budget = 50;
      a.weights = At(3);
      a.blocks = 100;
      change(a);
      kvx::CompactLaunch l;
      return kvx::CheckCompact(Pool(), a, &l);
    };
    Passes(run([](A&) {}), "compact");
    Passes(run([](A& a) { a.weights = 0; a.blocks = 0; }), "compact: no weights");
    Passes(run([](A& a) { a.budget = 0; a.kept = 0; }), "compact: nothing");
    Passes(run([](A& a) { a.sequences = 0; a.kept = a.tables = 0; }), "compact: no sequences");
    Passes(run([](A& a) { a.table_width = 0; a.tables = 0; }), "compact: no tables");
    Passes(run([](A& a) { a.kept_head_stride = 1; a.kept_place_stride = 2; }), "compact: strides");
    Refused(run([](A& a) { a.kept_place_stride = -1; }), "stride", "compact: negative stride");
    Refused(run([](A& a) { a.kept_place_stride = INT64_MAX / 4; }), "overflow", "compact: stride");
    Refused(run([](A& a) { a.kept_sequence_stride = 1ll << 30; }), "past the end",
            "compact: kept overruns");
    Refused(run([](A& a) { a.budget = -1; }), "budget", "compact: budget");
    Refused(run([](A& a) { a.sequences = -1; }), "sequences", "compact: sequences");
    Refused(run([](A& a) { a.kept = 0; }), "kept: null", "compact: null kept");
    Refused(run([](A& a) { a.kept = kHost; }), "kept: host", "compact: host kept");
    Refused(run([](A& a) { a.tables = kHost; }), "tables: host", "compact: host tables");
    Refused(run([](A& a) { a.blocks = 99; }), "fewer blocks", "compact: a smaller table");
    Refused(run([](A& a) { a.weights = kHost; }), "weights: host", "compact: host weights");
    Refused(run([](A& a) { a.weights = a.kept; }), "overlaps", "compact: weights on kept");
    Refused(run([](A& a) { a.weights = a.tables; }), "overlaps", "compact: weights on tables");
    const auto in = [](int64_t layer) { return kDev + (2ull << 30) + layer * (1 << 20); };
    Refused(run([&](A& a) { a.kept = in(a.cache.v_layer); }), "overlaps the cache",
            "compact: kept in the cache");
    Refused(run([&](A& a) { a.weights = in(a.cache.k_layer); }), "overlaps the cache",
            "compact: weights on the cache");
    Refused(run([&](A& a) { a.tables = in(a.cache.k_layer) + 16; }), "overlaps the cache",
            "compact: tables in the cache");
    if (type != KVX_BF16) {
      Refused(run([&](A& a) { a.kept = in(a.cache.v_scale_layer); }), "overlaps the cache's scales",
              "compact: kept in the scales");
    }
    Refused(run([](A& a) { a.cache.v_layer = a.cache.k_layer; }), "of their own",
            "compact: K on V");
    Refused(run([](A& a) { a.cache.dtype = KVX_F32; }), "cache", "compact: fp32");
  }
}

void Fp4Cache() {
  kvx_append_kv_args a;
  std::memset(&a, 0, sizeof(a));
  a.batch = Batch();
  a.tokens = 10;
  a.dtype = KVX_F16;
  a.k = At(1);
  a.v = At(2);
  a.k_token_stride = a.v_token_stride = 128;
  a.k_head_stride = a.v_head_stride = 64;
  const auto append = [&](const std::function<void(kvx_paged_cache&)>& change) {
    kvx_append_kv_args b = a;
    b.cache = Cache(KVX_FP4);
    change(b.cache);
    kvx::AppendLaunch l;
    return kvx::CheckAppendKv(Pool(), b, &l);
  };
  using C = kvx_paged_cache;
  Passes(append([](C&) {}), "fp4 append");
  Refused(append([](C& c) { c.k_scale_layer = 4; }), "one byte for 32", "fp4: e4m3's scales");
  Refused(append([](C& c) { c.v_scale_layer = -1; }), "scale layer", "fp4: no scales", 11);
  Refused(append([](C& c) { c.v_scale_layer = 8; }), "of their own", "fp4: one scale table");
  Refused(append([](C& c) { c.k_layer = 0; }), "bytes", "fp4: a 16-bit storage");
  Refused(append([](C& c) { c.k_layer = 10; }), "aligned to 16", "fp4: storage 8 bytes off");
  Refused(append([](C& c) { c.head_dim = 48; }), "multiple of 32", "fp4: head width");
}

}  // namespace

int main() {
  kvx::SetAddressQueryForTesting(FakeQuery);
  WeighArgs();
  ChooseArgs();
  CompactArgs();
  Fp4Cache();
  kvx::SetAddressQueryForTesting(nullptr);
  if (failures == 0) std::printf("eviction argument checks: all passed\n");
  return failures == 0 ? 0 : 1;
}
