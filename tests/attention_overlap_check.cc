// Which of the paged operators' arguments may lie in one buffer, be empty or be
// too many, on the CPU, no GPU calls: a pool and an address map of their own
// making stand in for the manager and the HIP runtime. Arguments that share no
// element pass, however they are interleaved; a result on anything else that the
// call reads or writes is refused with INVALID_ARGUMENT and a message that names
// both.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <set>
#include <string>

#include "attention_args.h"
#include "device_memory.h"
#include "kvx.h"

namespace {

constexpr uint64_t kDev = 0x7f0000000000ull;  // device 0, 4 GiB

kvx::AddressInfo FakeQuery(uint64_t a) {
  kvx::AddressInfo i;
  if (a >= kDev && a < kDev + (4ull << 30)) i = {kvx::MemKind::kDevice, 0, kDev, 4ull << 30};
  return i;
}

uint64_t At(int64_t mib) { return kDev + static_cast<uint64_t>(mib) * (1 << 20); }

int failures = 0;

void Refused(const kvx::Status& s, const char* needle, const char* what) {
  if (static_cast<int>(s.code()) != 3 || s.message().find(needle) == std::string::npos) {
    std::printf("FAIL %s: code %d, message '%s' (want 3 with '%s')\n", what,
                static_cast<int>(s.code()), s.message().c_str(), needle);
    ++failures;
  }
}

void Passes(const kvx::Status& s, const char* what) {
  if (!s.ok()) {
    std::printf("FAIL %s: '%s'\n", what, s.message().c_str());
    ++failures;
  }
}

// 10 tokens of 8 query and 8 key heads of 64, results apart.
kvx_norm_rope_args GoodNorm() {
  kvx_norm_rope_args a;
  std::memset(&a, 0, sizeof(a));
  a.dtype = KVX_BF16;
  a.tokens = 10;
  a.q_heads = a.k_heads = 8;
  a.head_dim = a.rotary_dim = 64;
  a.q = At(1);
  a.k = At(2);
  a.q_out = At(3);
  a.k_out = At(4);
  a.q_token_stride = a.k_token_stride = a.q_out_token_stride = a.k_out_token_stride = 512;
  a.q_head_stride = a.k_head_stride = a.q_out_head_stride = a.k_out_head_stride = 64;
  a.positions = At(5);
  a.inv_freq = At(6);
  return a;
}

kvx::Status Norm(const std::function<void(kvx_norm_rope_args&)>& change) {
  kvx_norm_rope_args a = GoodNorm();
  change(a);
  kvx::NormRopeLaunch l;
  return kvx::CheckNormRope(a, &l);
}

// q and k in one buffer, in place, at the given strides and `gap` elements apart.
kvx::Status Fused(int64_t token, int64_t head, int64_t gap, int64_t tokens = 10,
                  int32_t q_heads = 8, int32_t k_heads = 8) {
  return Norm([&](kvx_norm_rope_args& a) {
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.k_heads = k_heads;
    a.q_out = a.q;
    a.k = a.k_out = a.q + static_cast<uint64_t>(gap) * 2;
    a.q_token_stride = a.k_token_stride = a.q_out_token_stride = a.k_out_token_stride = token;
    a.q_head_stride = a.k_head_stride = a.q_out_head_stride = a.k_out_head_stride = head;
  });
}

// Whether the rows of Fused share an element, row by row.
bool Shares(int64_t token, int64_t head, int64_t gap, int64_t tokens, int32_t q_heads,
            int32_t k_heads) {
  std::set<int64_t> q;
  for (int64_t t = 0; t < tokens; ++t) {
    for (int64_t h = 0; h < q_heads; ++h) {
      for (int64_t d = 0; d < 64; ++d) q.insert(t * token + h * head + d);
    }
  }
  for (int64_t t = 0; t < tokens; ++t) {
    for (int64_t h = 0; h < k_heads; ++h) {
      for (int64_t d = 0; d < 64; ++d) {
        if (q.count(gap + t * token + h * head + d) != 0) return true;
      }
    }
  }
  return false;
}

void FusedProjections() {
  Passes(Fused(24 * 64, 64, 8 * 64), "q, k, v side by side");
  Passes(Fused(24 * 64, 3 * 64, 64), "q, k, v of every head");
  Passes(Fused(24 * 64, 3 * 64, 128), "q, v, k of every head");
  Passes(Fused(64, 30 * 64, 10 * 64), "[head][q, k, v][token]");
  Passes(Fused(3 * 64, 30 * 64, 64), "[head][token][q, k, v]");
  Passes(Fused(24 * 64, 3 * 64, 64, 1), "one token");
  Passes(Fused(24 * 64, 3 * 64, 64, 10, 8, 1), "one key head");
  Passes(Fused(24 * 64, 3 * 64, 64, 10, 1, 8), "one query head");
  Refused(Fused(24 * 64, 3 * 64, 32), "overlaps", "half a row off");
  Refused(Fused(24 * 64, 3 * 64, 160), "overlaps", "into the next head");
  Refused(Fused(24 * 64, 3 * 64, 24 * 64), "overlaps", "a token later");
  Refused(Fused(24 * 64, 3 * 64, 3 * 64), "overlaps", "a head later");
  // Never passed where an element is shared.
  int passed = 0;
  for (int64_t tokens : {1, 2, 3}) {
    for (int32_t qh : {1, 2, 3}) {
      for (int32_t kh : {1, 3}) {
        for (int64_t token : {64, 96, 192, 256, 576, 640}) {
          for (int64_t head : {64, 128, 192, 256, 576}) {
            for (int64_t gap = 32; gap <= 1600; gap += 32) {
              if (!Fused(token, head, gap, tokens, qh, kh).ok()) continue;
              ++passed;
              if (Shares(token, head, gap, tokens, qh, kh)) {
                std::printf("FAIL shared elements pass: strides %d %d gap %d, %d x (%d, %d)\n",
                            static_cast<int>(token), static_cast<int>(head),
                            static_cast<int>(gap), static_cast<int>(tokens), qh, kh);
                ++failures;
              }
            }
          }
        }
      }
    }
  }
  if (passed < 1000) {
    std::printf("FAIL only %d layouts pass\n", passed);
    ++failures;
  }
}

void NormInputs() {
  using A = kvx_norm_rope_args;
  const auto weighted = [](const std::function<void(A&)>& change) {
    return Norm([&](A& a) {
      a.q_weight = At(7);
      a.k_weight = At(8);
      a.weight_dtype = KVX_F32;
      change(a);
    });
  };
  Passes(weighted([](A&) {}), "norm");
  // Rows of 512 elements 1024 apart: the weights between the first two.
  Passes(weighted([](A& a) {
           a.q_out_token_stride = 1024;
           a.q_weight = a.q_out + 512 * 2;
         }),
         "a weight between rows");
  for (uint64_t off : {0, 9 * 512 * 2 + 510 * 2}) {
    for (bool q : {true, false}) {
      const char* name = q ? "q_out" : "k_out";
      const auto on = [&](uint64_t A::*input, const char* what) {
        const std::string message = std::string(name) + ": overlaps " + what;
        Refused(weighted([&](A& a) { a.*input = (q ? a.q_out : a.k_out) + off; }), message.c_str(),
                "norm onto its inputs");
      };
      on(&A::q_weight, "q_weight");
      on(&A::k_weight, "k_weight");
      on(&A::inv_freq, "inv_freq");
      on(&A::positions, "positions");
    }
  }
  Passes(weighted([](A& a) {
           a.rotary_dim = 0;
           a.positions = a.inv_freq = a.q_out;
         }),
         "nothing rotated");
}

// 100 blocks of [16][2][64]: layers 0, 1 bf16; 2, 3 e4m3; 4, 5 their scales.
bool Find(const void*, int64_t layer, int64_t shard, kvx::PoolStorage* out) {
  if (layer < 0 || layer > 5 || shard != 0) return false;
  const int64_t block[] = {4096, 4096, 2048, 2048, 8, 8};
  *out = {At(2048 + layer), block[layer] * 100, block[layer]};
  return true;
}

kvx::PoolSource Pool() {
  kvx::PoolSource p;
  p.find = Find;
  return p;
}

kvx_paged_cache GoodCache(bool e4m3) {
  kvx_paged_cache c;
  std::memset(&c, 0, sizeof(c));
  c.k_layer = e4m3 ? 2 : 0;
  c.v_layer = e4m3 ? 3 : 1;
  c.k_scale_layer = 4;
  c.v_scale_layer = 5;
  c.dtype = e4m3 ? KVX_E4M3 : KVX_BF16;
  c.block_tokens = 16;
  c.heads = 2;
  c.head_dim = 64;
  return c;
}

kvx_paged_batch GoodBatch() {
  kvx_paged_batch b;
  std::memset(&b, 0, sizeof(b));
  b.tables = At(10);
  b.table_stride = 64;
  b.table_width = 20;
  b.lengths = At(11);
  b.starts = At(12);
  b.sequences = 3;
  return b;
}

kvx::Status Attend(bool e4m3, const std::function<void(kvx_attend_args&)>& change) {
  kvx_attend_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = GoodCache(e4m3);
  a.batch = GoodBatch();
  a.tokens = 10;
  a.dtype = KVX_BF16;
  a.q_heads = 8;
  a.q = At(1);
  a.out = At(2);
  a.lse = At(3);
  a.q_token_stride = a.out_token_stride = 512;
  a.q_head_stride = a.out_head_stride = 64;
  a.group_starts = At(20);
  a.prefix_lengths = At(21);
  a.groups = 2;
  a.scale = 0.125f;
  a.workspace = At(100);
  a.workspace_bytes = 512 << 20;
  change(a);
  kvx::AttendLaunch l;
  return kvx::CheckAttend(Pool(), a, &l, nullptr);
}

void AttendResults() {
  using A = kvx_attend_args;
  for (bool e4m3 : {false, true}) {
    const auto run = [&](const std::function<void(A&)>& f) { return Attend(e4m3, f); };
    Passes(run([](A&) {}), "attend");
    Passes(run([](A& a) { a.out = a.q; }), "attend in place");
    Passes(run([](A& a) { a.workspace = At(2048) - (512 << 20); }), "a workspace before the cache");
    Passes(run([](A& a) { a.lse = a.out + 10 * 512 * 2; }), "lse behind out");
    const uint64_t k = e4m3 ? At(2050) : At(2048), v = k + (1 << 20);
    const uint64_t last = 100 * (e4m3 ? 2048 : 4096) - 16;
    struct {
      uint64_t at;
      const char* name;
    } others[] = {{k, "the cache"},        {v, "the cache"},          {k + last, "the cache"},
                  {v + last, "the cache"}, {At(10), "tables"},        {At(10) + 512 + 64, "tables"},
                  {At(11), "lengths"},     {At(12), "starts"},        {At(20), "group_starts"},
                  {At(21), "prefix_lengths"}};
    for (const auto& o : others) {
      Refused(run([&](A& a) { a.out = o.at; }), (std::string("out: overlaps ") + o.name).c_str(),
              "out");
      Refused(run([&](A& a) { a.lse = o.at; }), (std::string("lse: overlaps ") + o.name).c_str(),
              "lse");
      Refused(run([&](A& a) { a.workspace = o.at; }),
              (std::string("workspace: overlaps ") + o.name).c_str(), "workspace");
    }
    Refused(run([](A& a) { a.lse = a.out + 64; }), "lse: overlaps out", "lse on out");
    Refused(run([](A& a) { a.lse = a.q + 64; }), "lse: overlaps q", "lse on q");
    Refused(run([](A& a) { a.workspace = a.out + 64; }), "workspace: overlaps out", "parts on out");
    Refused(run([](A& a) { a.workspace = a.q + 64; }), "workspace: overlaps", "parts on q");
    Refused(run([](A& a) { a.workspace = a.lse; }), "workspace: overlaps lse", "parts on lse");
  }
  for (uint64_t at : {At(2052), At(2053) + 796}) {
    Refused(Attend(true, [&](kvx_attend_args& a) { a.lse = at; }), "the cache's scales",
            "lse on scales");
    Passes(Attend(false, [&](kvx_attend_args& a) { a.lse = at; }), "no scales in use");
  }
}

kvx::Status Append(bool e4m3, const std::function<void(kvx_append_kv_args&)>& change) {
  kvx_append_kv_args a;
  std::memset(&a, 0, sizeof(a));
  a.cache = GoodCache(e4m3);
  a.batch = GoodBatch();
  a.tokens = 10;
  a.dtype = KVX_BF16;
  a.rotary_dim = 64;
  a.k = At(1);
  a.v = At(2);
  a.k_token_stride = a.v_token_stride = 128;
  a.k_head_stride = a.v_head_stride = 64;
  a.k_weight = At(3);
  a.weight_dtype = KVX_F32;
  a.inv_freq = At(4);
  a.positions = At(5);
  a.positions_64 = 1;
  change(a);
  kvx::AppendLaunch l;
  return kvx::CheckAppendKv(Pool(), a, &l);
}

void AppendInputs() {
  using A = kvx_append_kv_args;
  struct {
    const char* name;
    std::function<void(A&, uint64_t)> put;
  } const inputs[] = {
      {"k", [](A& a, uint64_t at) { a.k = at; }},
      {"v", [](A& a, uint64_t at) { a.v = at; }},
      {"tables", [](A& a, uint64_t at) { a.batch.tables = at; }},
      {"lengths", [](A& a, uint64_t at) { a.batch.lengths = at; }},
      {"starts", [](A& a, uint64_t at) { a.batch.starts = at; }},
      {"k_weight", [](A& a, uint64_t at) { a.k_weight = at; }},
      {"inv_freq", [](A& a, uint64_t at) { a.inv_freq = at; }},
      {"positions", [](A& a, uint64_t at) { a.positions = at; }},
  };
  for (bool e4m3 : {false, true}) {
    Passes(Append(e4m3, [](A&) {}), "append");
    const uint64_t k = e4m3 ? At(2050) : At(2048), v = k + (1 << 20);
    const uint64_t last = 100 * (e4m3 ? 2048 : 4096) - 8;
    for (const auto& in : inputs) {
      const std::string on = std::string(in.name) + ": overlaps the cache";
      for (uint64_t at : {k, v, k + last, v + last}) {
        Refused(Append(e4m3, [&](A& a) { in.put(a, at); }), on.c_str(), "append from the cache");
      }
      for (uint64_t at : {At(2052), At(2053), At(2053) + 792}) {
        if (e4m3) {
          Refused(Append(true, [&](A& a) { in.put(a, at); }), (on + "'s scales").c_str(),
                  "append from the scales");
        } else {
          Passes(Append(false, [&](A& a) { in.put(a, at); }), "no scales in use");
        }
      }
    }
  }
}

// A table without a column, as torch makes it: no address, a stride of 1.
void NoTable() {
  for (int64_t sequences : {1, 3}) {
    const auto change = [&](auto& a) {
      a.batch.sequences = sequences;
      a.batch.tables = 0;
      a.batch.table_width = 0;
      a.batch.table_stride = 1;
    };
    for (bool e4m3 : {false, true}) {
      Passes(Append(e4m3, change), "append without a table");
      Passes(Attend(e4m3, change), "attend without a table");
    }
  }
}

// Grids of 2^32 threads and more, which no launch takes, are refused before it.
void LargestGrids() {
  const auto norm = [](int64_t tokens) {
    return Norm([&](kvx_norm_rope_args& a) {
      a.tokens = tokens;
      a.q_heads = 1;
      a.k_heads = 0;
      a.k = a.k_out = 0;
      a.head_dim = 1;
      a.rotary_dim = 0;
      a.q = At(0);
      a.q_out = At(1536);
      a.q_token_stride = a.q_out_token_stride = a.q_head_stride = a.q_out_head_stride = 1;
    });
  };
  Passes(norm((1ll << 29) - 32), "norm of 2^29 - 32 rows");
  Refused(norm((1ll << 29) - 31), "too many tokens", "norm of 2^29 - 31 rows");
  // Blocks of one slot [1][1][1], e4m3: a workgroup of 64 threads each.
  kvx::PoolSource pool;
  pool.find = [](const void*, int64_t layer, int64_t, kvx::PoolStorage* out) {
    const int64_t block = layer < 4 ? 1 : 4;
    *out = {At(2048 + layer * 16), block * 1000, block};
    return true;
  };
  const auto append = [&](int64_t tokens, int32_t type) {
    kvx_append_kv_args a;
    std::memset(&a, 0, sizeof(a));
    a.cache = GoodCache(true);
    a.cache.block_tokens = a.cache.heads = a.cache.head_dim = 1;
    a.batch = GoodBatch();
    a.tokens = tokens;
    a.dtype = type;
    a.k = At(0);
    a.v = At(1024);
    a.k_token_stride = a.v_token_stride = a.k_head_stride = a.v_head_stride = 1;
    a.batch.tables = At(4000);
    a.batch.lengths = At(4001);
    a.batch.starts = At(4002);
    kvx::AppendLaunch l;
    return kvx::CheckAppendKv(pool, a, &l);
  };
  Passes(append((1ll << 26) - 1, KVX_BF16), "append to 2^26 - 1 blocks");
  Refused(append(1ll << 26, KVX_F16), "too many tokens", "append to 2^26 blocks");
}

}  // namespace

int main() {
  kvx::SetAddressQueryForTesting(FakeQuery);
  FusedProjections();
  NormInputs();
  AttendResults();
  AppendInputs();
  NoTable();
  LargestGrids();
  kvx::SetAddressQueryForTesting(nullptr);
  if (failures == 0) std::printf("attention overlap checks: all passed\n");
  return failures == 0 ? 0 : 1;
}
