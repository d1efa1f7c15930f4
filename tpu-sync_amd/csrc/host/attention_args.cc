#include "attention_args.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <string>

#include "paged_args.h"

namespace kvx {
namespace {

using namespace paged;

Status CheckRowGrid(int64_t tokens) {
  return CheckGrid((tokens + kMostRowTokens - 1) / kMostRowTokens, kRowThreads);
}

Status CheckRotation(DeviceRangeChecker* ranges, int64_t rotary, int64_t dim, uint64_t inv_freq,
                     uint64_t positions, bool positions_64, int64_t tokens) {
  if (rotary < 0 || rotary % 2 != 0 || rotary > dim) {
    return Bad("rotary_dim must be even and at most head_dim");
  }
  if (rotary == 0 || tokens == 0) return OkStatus();
  KVX_RETURN_IF_ERROR(ranges->Check(inv_freq, static_cast<uint64_t>(rotary / 2) * 4, "inv_freq"));
  if (positions != 0) {
    if (positions % (positions_64 ? 8 : 4) != 0) return Bad("positions: unaligned address");
    KVX_RETURN_IF_ERROR(
        ranges->Check(positions, static_cast<uint64_t>(tokens) * (positions_64 ? 8 : 4),
                      "positions"));
  }
  return OkStatus();
}

Status CheckWeight(DeviceRangeChecker* ranges, uint64_t at, int32_t type, int32_t row_type,
                   int64_t dim, float eps, const char* what) {
  if (at == 0) return OkStatus();
  if (type != row_type && type != kF32) {
    return Bad(std::string(what) + ": must be of the rows' type or fp32");
  }
  if (!std::isfinite(eps) || eps < 0) return Bad("eps must be finite and not negative");
  if (at % static_cast<uint64_t>(ElementBytes(type)) != 0) {
    return Bad(std::string(what) + ": unaligned address");
  }
  return ranges->Check(at, static_cast<uint64_t>(dim * ElementBytes(type)), what);
}

}  // namespace

Status CheckNormRope(const kvx_norm_rope_args& a, NormRopeLaunch* out) {
  if (a.dtype != kBf16 && a.dtype != kF16 && a.dtype != kF32) {
    return Bad("dtype must be KVX_BF16, KVX_F16 or KVX_F32");
  }
  KVX_RETURN_IF_ERROR(CheckTokens(a.tokens, static_cast<int64_t>(a.q_heads) + a.k_heads,
                                  a.head_dim));
  if (a.q_heads < 0 || a.k_heads < 0) return Bad("negative number of heads");
  KVX_RETURN_IF_ERROR(CheckRowGrid(a.tokens));
  DeviceRangeChecker ranges(a.device);
  const int64_t item = ElementBytes(a.dtype);
  const Rows q = {a.q, a.q_token_stride, a.q_head_stride, a.tokens, a.q_heads, a.head_dim, item};
  const Rows k = {a.k, a.k_token_stride, a.k_head_stride, a.tokens, a.k_heads, a.head_dim, item};
  const Rows qo = {a.q_out, a.q_out_token_stride, a.q_out_head_stride, a.tokens, a.q_heads,
                   a.head_dim, item};
  const Rows ko = {a.k_out, a.k_out_token_stride, a.k_out_head_stride, a.tokens, a.k_heads,
                   a.head_dim, item};
  KVX_RETURN_IF_ERROR(CheckRows(&ranges, q, "q"));
  KVX_RETURN_IF_ERROR(CheckRows(&ranges, k, "k"));
  KVX_RETURN_IF_ERROR(CheckRows(&ranges, qo, "q_out"));
  KVX_RETURN_IF_ERROR(CheckRows(&ranges, ko, "k_out"));
  KVX_RETURN_IF_ERROR(CheckInPlace(q, qo, "q", "q_out"));
  KVX_RETURN_IF_ERROR(CheckInPlace(k, ko, "k", "k_out"));
  if (Meet(k, qo) || Meet(qo, ko)) return Bad("q_out: overlaps k or k_out");
  if (Meet(q, ko)) return Bad("k_out: overlaps q");
  if (a.rotary_dim > 0 && a.tokens > 0 && a.positions == 0) return Bad("positions: null");
  KVX_RETURN_IF_ERROR(CheckRotation(&ranges, a.rotary_dim, a.head_dim, a.inv_freq, a.positions,
                                    a.positions_64 != 0, a.tokens));
  KVX_RETURN_IF_ERROR(CheckWeight(&ranges, a.q_weight, a.weight_dtype, a.dtype, a.head_dim, a.eps,
                                  "q_weight"));
  KVX_RETURN_IF_ERROR(CheckWeight(&ranges, a.k_weight, a.weight_dtype, a.dtype, a.head_dim, a.eps,
                                  "k_weight"));
  const int64_t weight_bytes = a.head_dim * ElementBytes(a.weight_dtype);
  const int64_t rotated = a.rotary_dim > 0 ? a.tokens : 0;
  for (const Named& written : {Named(qo, "q_out"), Named(ko, "k_out")}) {
    KVX_RETURN_IF_ERROR(CheckApart(
        written, {{Whole(a.q_weight, a.q_weight != 0 ? weight_bytes : 0), "q_weight"},
                  {Whole(a.k_weight, a.k_weight != 0 ? weight_bytes : 0), "k_weight"},
                  {Whole(a.inv_freq, a.tokens > 0 ? a.rotary_dim * 2 : 0), "inv_freq"},
                  {Whole(a.positions, rotated * (a.positions_64 != 0 ? 8 : 4)), "positions"}}));
  }
  const auto rows = [](const Rows& in, const Rows& o, uint64_t weight) {
    HeadRows r;
    r.in = reinterpret_cast<const void*>(in.at);
    r.out = reinterpret_cast<void*>(o.at);
    r.weight = reinterpret_cast<const void*>(weight);
    r.in_token = in.token_stride;
    r.in_head = in.head_stride;
    r.out_token = o.token_stride;
    r.out_head = o.head_stride;
    r.heads = static_cast<int32_t>(in.heads);
    return r;
  };
  *out = NormRopeLaunch{};
  out->q = rows(q, qo, a.q_weight);
  out->k = rows(k, ko, a.k_weight);
  out->positions = reinterpret_cast<const void*>(a.positions);
  out->inv_freq = reinterpret_cast<const float*>(a.inv_freq);
  out->tokens = a.q_heads + a.k_heads > 0 ? static_cast<int32_t>(a.tokens) : 0;
  out->head_dim = a.head_dim;
  out->rotary_dim = a.rotary_dim;
  out->type = a.dtype;
  out->weight_f32 = a.weight_dtype == kF32;
  out->positions_64 = a.positions_64 != 0;
  out->interleaved = a.interleaved != 0;
  out->eps = a.eps;
  return OkStatus();
}

Status CheckAppendKv(const PoolSource& pool, const kvx_append_kv_args& a, AppendLaunch* out) {
  Cache cache;
  KVX_RETURN_IF_ERROR(FindCache(pool, a.cache, a.dtype, &cache));
  const kvx_paged_cache& c = a.cache;
  KVX_RETURN_IF_ERROR(CheckTokens(a.tokens, c.heads, c.head_dim));
  DeviceRangeChecker ranges(pool.device);
  const Rows k = {a.k, a.k_token_stride, a.k_head_stride, a.tokens, c.heads, c.head_dim, 2};
  const Rows v = {a.v, a.v_token_stride, a.v_head_stride, a.tokens, c.heads, c.head_dim, 2};
  KVX_RETURN_IF_ERROR(CheckRows(&ranges, k, "k"));
  KVX_RETURN_IF_ERROR(CheckRows(&ranges, v, "v"));
  *out = AppendLaunch{};
  KVX_RETURN_IF_ERROR(CheckBatch(&ranges, a.batch, a.tokens, c.block_tokens, cache.num_blocks,
                                 &out->batch));
  KVX_RETURN_IF_ERROR(CheckRotation(&ranges, a.rotary_dim, c.head_dim, a.inv_freq, a.positions,
                                    a.positions_64 != 0, a.tokens));
  KVX_RETURN_IF_ERROR(CheckWeight(&ranges, a.k_weight, a.weight_dtype, a.dtype, c.head_dim, a.eps,
                                  "k_weight"));
  // What is written may meet nothing that is read.
  const std::initializer_list<Named> read = {
      {k, "k"},
      {v, "v"},
      {Tables(a.batch), "tables"},
      {Lengths(a.batch), "lengths"},
      {Starts(a.batch), "starts"},
      {Whole(a.k_weight, a.k_weight != 0 ? c.head_dim * ElementBytes(a.weight_dtype) : 0),
       "k_weight"},
      {Whole(a.inv_freq, a.tokens > 0 ? a.rotary_dim * 2 : 0), "inv_freq"},
      {Whole(a.positions,
             a.rotary_dim > 0 && a.positions != 0 ? a.tokens * (a.positions_64 != 0 ? 8 : 4) : 0),
       "positions"}};
  for (const Named& r : read) {
    KVX_RETURN_IF_ERROR(CheckApart(r, {{Whole(cache.k), "the cache"},
                                       {Whole(cache.v), "the cache"},
                                       {Whole(cache.k_scales), "the cache's scales"},
                                       {Whole(cache.v_scales), "the cache's scales"}}));
  }
  if (a.batch.sequences == 0) out->batch.tokens = 0;
  out->block_div = MakeFastDivU32(static_cast<uint32_t>(c.block_tokens));
  out->k = reinterpret_cast<const void*>(a.k);
  out->v = reinterpret_cast<const void*>(a.v);
  out->k_token = a.k_token_stride;
  out->k_head = a.k_head_stride;
  out->v_token = a.v_token_stride;
  out->v_head = a.v_head_stride;
  out->k_pool = reinterpret_cast<void*>(cache.k.base);
  out->v_pool = reinterpret_cast<void*>(cache.v.base);
  out->k_scales = reinterpret_cast<void*>(cache.k_scales.base);
  out->v_scales = reinterpret_cast<void*>(cache.v_scales.base);
  out->k_weight = reinterpret_cast<const void*>(a.k_weight);
  out->positions = reinterpret_cast<const void*>(a.positions);
  out->inv_freq = reinterpret_cast<const float*>(a.inv_freq);
  out->heads = c.heads;
  out->head_dim = c.head_dim;
  out->rotary_dim = a.rotary_dim;
  out->type = a.dtype;
  out->pool = KindOf(c.dtype);
  out->weight_f32 = a.weight_dtype == kF32;
  out->positions_64 = a.positions_64 != 0;
  out->interleaved = a.interleaved != 0;
  out->eps = a.eps;
  return out->pool == kPoolE4m3 ? CheckGrid(MostBlocks(*out), BlockThreads(*out)) : CheckRowGrid(a.tokens);
}

Status CheckAttend(const PoolSource& pool, const kvx_attend_args& a, AttendLaunch* out,
                   int64_t* workspace_bytes) {
  Cache cache;
  KVX_RETURN_IF_ERROR(FindCache(pool, a.cache, a.dtype, &cache));
  const kvx_paged_cache& c = a.cache;
  KVX_RETURN_IF_ERROR(CheckTokens(a.tokens, a.q_heads, c.head_dim));
  if (c.head_dim % 8 != 0) return Bad("head_dim must be a multiple of 8");
  if (a.q_heads < 1 || a.q_heads % c.heads != 0) {
    return Bad("q_heads must be a multiple of the cache's heads");
  }
  if (!std::isfinite(a.scale) || a.scale <= 0) return Bad("scale must be finite and positive");
  if (a.groups < 0 || a.groups > kMaxGroups) return Bad("groups must be 0..256");
  DeviceRangeChecker ranges(pool.device);
  const Rows q = {a.q, a.q_token_stride, a.q_head_stride, a.tokens, a.q_heads, c.head_dim, 2};
  const Rows o = {a.out, a.out_token_stride, a.out_head_stride, a.tokens, a.q_heads, c.head_dim,
                  2};
  *out = AttendLaunch{};
  if (workspace_bytes == nullptr) {
    KVX_RETURN_IF_ERROR(CheckRows(&ranges, q, "q"));
    KVX_RETURN_IF_ERROR(CheckRows(&ranges, o, "out"));
    KVX_RETURN_IF_ERROR(CheckInPlace(q, o, "q", "out"));
    KVX_RETURN_IF_ERROR(CheckBatch(&ranges, a.batch, a.tokens, c.block_tokens, cache.num_blocks,
                                   &out->batch));
    if (a.groups > 0 && a.batch.sequences > 0) {
      KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.group_starts, a.groups + 1, "group_starts"));
      KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.prefix_lengths, a.groups, "prefix_lengths"));
    }
    if (a.lse != 0) {
      KVX_RETURN_IF_ERROR(CheckWords(&ranges, a.lse, a.tokens * a.q_heads, "lse"));
    }
  } else {
    KVX_RETURN_IF_ERROR(CheckSizes(a.batch, a.tokens, c.block_tokens, &out->batch));
  }
  const int64_t G = a.q_heads / c.heads;
  // Work is counted in 32 bits: tiles by steps of 64 tokens, sequences by steps
  // of 32, each for every key head, and squares of tiles.
  const int64_t tiles = 2 * (a.tokens * G / kManyRows + 1) + a.batch.sequences + a.groups;
  const int64_t steps = out->batch.capacity / kManyStep + 3 + a.tokens / kManyStep;
  const int64_t few = a.batch.sequences * (out->batch.capacity / kFewStep + 1);
  if (tiles > 65536 || tiles > INT32_MAX / 2 / c.heads / steps || few > INT32_MAX / 2 / c.heads) {
    return Bad("tokens * table_width is too large for one call");
  }
  out->most_few = static_cast<int32_t>(few);
  out->most_many = static_cast<int32_t>(tiles * steps);
  if (a.batch.sequences == 0) out->batch.tokens = 0;
  out->block_div = MakeFastDivU32(static_cast<uint32_t>(c.block_tokens));
  out->group_div = MakeFastDivU32(static_cast<uint32_t>(G));
  out->q = reinterpret_cast<const void*>(a.q);
  out->out = reinterpret_cast<void*>(a.out);
  out->lse = reinterpret_cast<float*>(a.lse);
  out->q_token = a.q_token_stride;
  out->q_head = a.q_head_stride;
  out->out_token = a.out_token_stride;
  out->out_head = a.out_head_stride;
  out->k_pool = reinterpret_cast<const void*>(cache.k.base);
  out->v_pool = reinterpret_cast<const void*>(cache.v.base);
  out->k_scales = reinterpret_cast<const void*>(cache.k_scales.base);
  out->v_scales = reinterpret_cast<const void*>(cache.v_scales.base);
  out->group_starts = reinterpret_cast<const int32_t*>(a.group_starts);
  out->prefix_lengths = reinterpret_cast<const int32_t*>(a.prefix_lengths);
  out->groups = a.groups;
  out->q_heads = a.q_heads;
  out->k_heads = c.heads;
  out->head_dim = c.head_dim;
  out->type = a.dtype;
  out->pool = KindOf(c.dtype);
  out->causal = a.non_causal == 0;
  out->scale = a.scale;
  const int64_t need = out->batch.tokens == 0 ? 0 : PlanAttend(out);
  if (workspace_bytes != nullptr) {
    *workspace_bytes = need;
    return OkStatus();
  }
  if (out->pool == kPoolSame && (reinterpret_cast<uintptr_t>(out->k_pool) |
                     reinterpret_cast<uintptr_t>(out->v_pool)) % 16 != 0) {
    return Bad("cache storages: must be aligned to 16 bytes");
  }
  if (need > 0) {
    if (a.workspace_bytes < need) {
      return Bad("workspace: " + std::to_string(need) + " bytes are needed");
    }
    if (a.workspace % 16 != 0) return Bad("workspace: must be aligned to 16 bytes");
    KVX_RETURN_IF_ERROR(ranges.Check(a.workspace, static_cast<uint64_t>(need), "workspace"));
    out->parts = reinterpret_cast<float*>(a.workspace);
  }
  // What is written may meet nothing else (`out` may be q).
  const Named results = {o, "out"}, queries = {q, "q"};
  const Named lse = {Whole(a.lse, a.lse != 0 ? a.tokens * a.q_heads * 4 : 0), "lse"};
  const Named workspace = {Whole(a.workspace, need), "workspace"};
  const int64_t groups = a.batch.sequences > 0 ? a.groups : 0;
  const std::initializer_list<Named> others = {
      {Whole(cache.k), "the cache"},
      {Whole(cache.v), "the cache"},
      {Whole(cache.k_scales), "the cache's scales"},
      {Whole(cache.v_scales), "the cache's scales"},
      {Tables(a.batch), "tables"},
      {Lengths(a.batch), "lengths"},
      {Starts(a.batch), "starts"},
      {Whole(a.group_starts, groups > 0 ? (groups + 1) * 4 : 0), "group_starts"},
      {Whole(a.prefix_lengths, groups * 4), "prefix_lengths"}};
  for (const Named* written : {&results, &lse, &workspace}) {
    KVX_RETURN_IF_ERROR(CheckApart(*written, others));
  }
  KVX_RETURN_IF_ERROR(CheckApart(lse, {results, queries}));
  return CheckApart(workspace, {results, queries, lse});
}

}  // namespace kvx
