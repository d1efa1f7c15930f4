// Which of the paged operators' arguments may lie in one buffer, on the CPU, no
// GPU calls: a pool and an address map of their own making stand in for the
// manager and the HIP runtime. Arguments that share no element pass, however
// they are interleaved; a result on anything else that the call reads or writes
// is refused with INVALID_ARGUMENT and a message that names both.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <set>

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

}  // namespace

int main() {
  kvx::SetAddressQueryForTesting(FakeQuery);
  FusedProjections();
  kvx::SetAddressQueryForTesting(nullptr);
  if (failures == 0) std::printf("attention overlap checks: all passed\n");
  return failures == 0 ? 0 : 1;
}
