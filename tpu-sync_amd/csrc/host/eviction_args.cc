#include "eviction_args.h"

#include <algorithm>

#include <climits>
#include <utility>
#include <cmath>

#include "paged_args.h"

namespace kvx {
namespace {

using namespace paged;

constexpr int64_t kMostBudget = int64_t{1} << 30;

// A table of weights fp32 [blocks][heads][block_tokens].
Status CheckTable(DeviceRangeChecker* ranges, uint64_t at, int64_t blocks, int64_t heads,
                  int64_t block_tokens, Rows* out) {
  if (blocks < 1 || blocks > INT32_MAX) return Bad("weights: blocks must be 1..2^31 - 1");
  int64_t bytes = 0;
  if (__builtin_mul_overflow(blocks, heads * block_tokens * 4, &bytes)) {
    return Bad("weights: size overflows");
  }
  KVX_RETURN_IF_ERROR(CheckWords(ranges, at, bytes / 4, "weights"));
  *out = Whole(at, bytes);
  return OkStatus();
}

}  // namespace

Status CheckWeigh(const PoolSource& pool, const kvx_weigh_args& a, WeighLaunch* out,
                  int64_t* workspace_bytes) {
  Cache cache;
  KVX_RETURN_IF_ERROR(FindCache(pool, a.cache, a.dtype, &cache, false));
  const kvx_paged_cache& c = a.cache;
  KVX_RETURN_IF_ERROR(CheckTokens(a.tokens, a.q_heads, c.head_dim));
  if (c.head_dim % 8 != 0) return Bad("head_dim must be a multiple of 8");
  if (a.q_heads < 1 || a.q_heads % c.heads != 0) {
    return Bad("q_heads must be a multiple of the cache's heads");
  }
  if (!std::isfinite(a.scale) || a.scale <= 0) return Bad("scale must be finite and positive");
  if (!(a.decay >= 0 && a.decay <= 1)) return Bad("decay must be 0..1");
  DeviceRangeChecker ranges(pool.device);
  const Rows q = {a.q, a.q_token_stride, a.q_head_stride, a.tokens, a.q_heads, c.head_dim, 2};
  Rows table = Whole(0, 0);
  *out = WeighLaunch{};
  AttendLaunch& l = out->attend;
  l.pool = KindOf(c.dtype);
  if (workspace_bytes == nullptr) {
    KVX_RETURN_IF_ERROR(CheckRows(&ranges, q, "q"));
    KVX_RETURN_IF_ERROR(CheckBatch(&ranges, a.batch, a.tokens, c.block_tokens, cache.num_blocks,
                                   &l.batch));
    if (a.tokens > 0) {
      KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.lse, a.tokens * a.q_heads, "lse"));
    }
    if (a.begins != 0 && a.batch.sequences > 0) {
      KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.begins, a.batch.sequences, "begins"));
    }
    if (a.weighed != 0 && a.batch.sequences > 0) {
      KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.weighed, a.batch.sequences, "weighed"));
    }
    KVX_RETURN_IF_ERROR(CheckTable(&ranges, a.weights, a.blocks, c.heads, c.block_tokens, &table));
    if (a.blocks < cache.num_blocks) return Bad("weights: fewer blocks than the cache's");
    if (l.pool == kPoolSame && cache.k.base % 16 != 0) {
      return Bad("cache storages: must be aligned to 16 bytes");
    }
  } else {
    KVX_RETURN_IF_ERROR(CheckSizes(a.batch, a.tokens, c.block_tokens, &l.batch));
  }
  // Work is counted in 32 bits, for every head: steps of 32 tokens, and tiles by
  // stages of 64 rows.
  const int64_t G = a.q_heads / c.heads;
  const int64_t few = a.batch.sequences * (l.batch.capacity / kFewStep + 1);
  const int64_t tiles = l.batch.capacity / WeighTile(PaddedDim(c.head_dim)) + 1;
  const int64_t stages = a.tokens * G / kWeighRows + 1 + a.batch.sequences;
  if (few > INT32_MAX / 2 / c.heads || stages > INT32_MAX / 2 / c.heads / tiles) {
    return Bad("tokens * table_width is too large for one call");
  }
  l.most_few = static_cast<int32_t>(few);
  l.most_many = static_cast<int32_t>(tiles * stages);
  if (a.batch.sequences == 0) l.batch.tokens = 0;
  l.block_div = MakeFastDivU32(static_cast<uint32_t>(c.block_tokens));
  l.group_div = MakeFastDivU32(static_cast<uint32_t>(G));
  l.q = reinterpret_cast<const void*>(a.q);
  l.q_token = a.q_token_stride;
  l.q_head = a.q_head_stride;
  l.k_pool = reinterpret_cast<const void*>(cache.k.base);
  l.k_scales = reinterpret_cast<const void*>(cache.k_scales.base);
  l.q_heads = a.q_heads;
  l.k_heads = c.heads;
  l.head_dim = c.head_dim;
  l.type = a.dtype;
  l.causal = a.non_causal == 0;
  l.scale = a.scale;
  out->lse = reinterpret_cast<const float*>(a.lse);
  out->weights = reinterpret_cast<float*>(a.weights);
  out->begins = reinterpret_cast<const int32_t*>(a.begins);
  out->weighed = reinterpret_cast<const int32_t*>(a.weighed);
  out->decay = a.decay;
  const int64_t need = l.batch.tokens == 0 ? 0 : PlanWeigh(out);
  if (workspace_bytes != nullptr) {
    *workspace_bytes = need;
    return OkStatus();
  }
  if (need > 0) {
    if (a.workspace_bytes < need) {
      return Bad("workspace: " + std::to_string(need) + " bytes are needed");
    }
    if (a.workspace % 16 != 0) return Bad("workspace: must be aligned to 16 bytes");
    KVX_RETURN_IF_ERROR(ranges.Check(a.workspace, static_cast<uint64_t>(need), "workspace"));
    out->parts = reinterpret_cast<float*>(a.workspace);
  }
  const Named weights = {table, "weights"}, workspace = {Whole(a.workspace, need), "workspace"};
  for (const Named* written : {&weights, &workspace}) {
    KVX_RETURN_IF_ERROR(CheckApart(
        *written, {{q, "q"},
                   {Whole(cache.k), "the cache"},
                   {Whole(cache.k_scales), "the cache's scales"},
                   {Tables(a.batch), "tables"},
                   {Lengths(a.batch), "lengths"},
                   {Starts(a.batch), "starts"},
                   {Whole(a.lse, a.tokens * a.q_heads * 4), "lse"},
                   {Whole(a.begins, a.begins != 0 ? a.batch.sequences * 4 : 0), "begins"},
                   {Whole(a.weighed, a.weighed != 0 ? a.batch.sequences * 4 : 0), "weighed"}}));
  }
  return CheckApart(workspace, {weights});
}

Status CheckChooseKept(const kvx_choose_kept_args& a, ChooseLaunch* out) {
  if (a.heads < 1 || a.heads > 1024) return Bad("heads must be 1..1024");
  if (a.block_tokens < 1 || a.block_tokens > (1 << 20)) return Bad("block_tokens must be 1..2^20");
  if (a.budget < 0 || a.budget > kMostBudget) return Bad("budget must be 0..2^30");
  if (a.recent < 0) return Bad("recent must not be negative");
  if (a.batch.starts != 0) return Bad("starts: not used here");
  DeviceRangeChecker ranges(a.device);
  Rows table;
  KVX_RETURN_IF_ERROR(CheckTable(&ranges, a.weights, a.blocks, a.heads, a.block_tokens, &table));
  *out = ChooseLaunch{};
  KVX_RETURN_IF_ERROR(CheckBatch(&ranges, a.batch, a.batch.sequences, a.block_tokens, a.blocks,
                                 &out->batch));
  const int64_t S = a.batch.sequences, words = S * a.heads * a.budget;
  if (S > 0 && a.begins != 0) KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.begins, S, "begins"));
  if (words > 0) KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.kept, words, "kept"));
  if (S > 0 && a.new_lengths != 0) {
    KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.new_lengths, S, "new_lengths"));
  }
  KVX_RETURN_IF_ERROR(CheckGrid(S * a.heads, kChooseThreads));
  const Named kept = {Whole(a.kept, words * 4), "kept"};
  const Named cut = {Whole(a.new_lengths, a.new_lengths != 0 ? S * 4 : 0), "new_lengths"};
  for (const Named* written : {&kept, &cut}) {
    KVX_RETURN_IF_ERROR(CheckApart(
        *written, {{table, "weights"},
                   {Tables(a.batch), "tables"},
                   {Lengths(a.batch), "lengths"},
                   {Whole(a.begins, a.begins != 0 ? S * 4 : 0), "begins"}}));
  }
  KVX_RETURN_IF_ERROR(CheckApart(cut, {kept}));
  out->block_div = MakeFastDivU32(static_cast<uint32_t>(a.block_tokens));
  out->weights = reinterpret_cast<const float*>(a.weights);
  out->begins = reinterpret_cast<const int32_t*>(a.begins);
  out->kept = reinterpret_cast<int32_t*>(a.kept);
  out->new_lengths = reinterpret_cast<int32_t*>(a.new_lengths);
  out->heads = a.heads;
  out->budget = static_cast<int32_t>(a.budget);
  out->recent = static_cast<int32_t>(std::min(a.recent, kMostBudget));
  return OkStatus();
}

Status CheckCompact(const PoolSource& pool, const kvx_compact_args& a, CompactLaunch* out) {
  Cache cache;
  const kvx_paged_cache& c = a.cache;
  KVX_RETURN_IF_ERROR(FindCache(pool, c, Is16Bit(c.dtype) ? c.dtype : kBf16, &cache));
  if (c.head_dim % 8 != 0) return Bad("head_dim must be a multiple of 8");
  if (a.budget < 0 || a.budget > kMostBudget) return Bad("budget must be 0..2^30");
  if (KindOf(c.dtype) == kPoolSame && (cache.k.base | cache.v.base) % 16 != 0) {
    return Bad("cache storages: must be aligned to 16 bytes");
  }
  DeviceRangeChecker ranges(pool.device);
  *out = CompactLaunch{};
  if (a.sequences < 0 || a.sequences > kMaxSequences) return Bad("sequences must be 0..4096");
  if (a.kept_sequence_stride < 0 || a.kept_head_stride < 0 || a.kept_place_stride < 0) {
    return Bad("kept: negative stride");
  }
  if (a.sequences == 0 || a.budget == 0) return OkStatus();
  int64_t words = 1;
  for (const auto& [n, stride] : {std::pair<int64_t, int64_t>{a.sequences, a.kept_sequence_stride},
                                  {c.heads, a.kept_head_stride},
                                  {a.budget, a.kept_place_stride}}) {
    int64_t more = 0;
    if (__builtin_mul_overflow(n - 1, stride, &more) ||
        __builtin_add_overflow(words, more, &words) || words > INT64_MAX / 4) {
      return Bad("kept: size overflows");
    }
  }
  KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.kept, words, "kept"));
  const kvx_paged_batch batch = {a.tables, a.table_stride, a.table_width, 0, 0, a.sequences};
  KVX_RETURN_IF_ERROR(CheckTables(&ranges, batch, c.block_tokens, cache.num_blocks, &out->batch));
  KVX_RETURN_IF_ERROR(CheckGrid(a.sequences * c.heads, kCompactThreads));
  Rows table = Whole(0, 0);
  if (a.weights != 0) {
    KVX_RETURN_IF_ERROR(CheckTable(&ranges, a.weights, a.blocks, c.heads, c.block_tokens, &table));
    if (a.blocks < cache.num_blocks) return Bad("weights: fewer blocks than the cache's");
  }
  const Named weights = {table, "the weights"};
  for (const Named& read : {Named(Tables(batch), "tables"), Named(Whole(a.kept, words * 4), "kept"),
                            weights}) {
    KVX_RETURN_IF_ERROR(CheckApart(read, {{Whole(cache.k), "the cache"},
                                          {Whole(cache.v), "the cache"},
                                          {Whole(cache.k_scales), "the cache's scales"},
                                          {Whole(cache.v_scales), "the cache's scales"}}));
  }
  KVX_RETURN_IF_ERROR(CheckApart(weights, {{Tables(batch), "tables"},
                                           {Whole(a.kept, words * 4), "kept"}}));
  out->block_div = MakeFastDivU32(static_cast<uint32_t>(c.block_tokens));
  out->kept = reinterpret_cast<const int32_t*>(a.kept);
  out->kept_sequence = a.kept_sequence_stride;
  out->kept_head = a.kept_head_stride;
  out->kept_place = a.kept_place_stride;
  out->budget = static_cast<int32_t>(a.budget);
  out->k_pool = reinterpret_cast<void*>(cache.k.base);
  out->v_pool = reinterpret_cast<void*>(cache.v.base);
  out->k_scales = reinterpret_cast<void*>(cache.k_scales.base);
  out->v_scales = reinterpret_cast<void*>(cache.v_scales.base);
  out->weights = reinterpret_cast<float*>(a.weights);
  out->heads = c.heads;
  out->head_dim = c.head_dim;
  out->pool = KindOf(c.dtype);
  return OkStatus();
}

}  // namespace kvx
