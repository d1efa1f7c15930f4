#include "attention_args.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <string>

#include "device_memory.h"

namespace kvx {
namespace {

constexpr int64_t kMostTokens = int64_t{1} << 30;  // of a call and of a table row

Status Bad(const std::string& what) { return InvalidArgumentError(what); }

// Rows [tokens][heads][dim] at strides in elements.
struct Rows {
  uint64_t at;
  int64_t token_stride, head_stride;
  int64_t tokens, heads, dim, item;

  bool empty() const { return tokens == 0 || heads == 0 || dim == 0; }
  // Bytes from the first to behind the last element; false on overflow.
  bool Extent(uint64_t* bytes) const {
    int64_t t = 0, h = 0, n = 0;
    if (__builtin_mul_overflow(tokens - 1, token_stride, &t) ||
        __builtin_mul_overflow(heads - 1, head_stride, &h) || __builtin_add_overflow(t, h, &n) ||
        __builtin_add_overflow(n, dim, &n) || __builtin_mul_overflow(n, item, &n)) {
      return false;
    }
    *bytes = static_cast<uint64_t>(n);
    return true;
  }
  // Whether two rows share elements.
  bool SelfOverlaps() const {
    const int64_t t = tokens > 1 ? token_stride : INT64_MAX;
    const int64_t h = heads > 1 ? head_stride : INT64_MAX;
    if (t >= h) return h < dim || (tokens > 1 && (heads - 1) * h + dim > t);
    return t < dim || (heads > 1 && (tokens - 1) * t + dim > h);
  }
  bool Same(const Rows& o) const {
    return at == o.at && (tokens == 1 || token_stride == o.token_stride) &&
           (heads == 1 || head_stride == o.head_stride);
  }
};

Status CheckRows(DeviceRangeChecker* ranges, const Rows& r, const char* what) {
  if (r.token_stride < 0 || r.head_stride < 0) return Bad(std::string(what) + ": negative stride");
  if (r.empty()) return OkStatus();
  uint64_t bytes = 0;
  if (!r.Extent(&bytes)) return Bad(std::string(what) + ": size overflows");
  if (r.at % static_cast<uint64_t>(r.item) != 0) {
    return Bad(std::string(what) + ": address is not a multiple of the element size");
  }
  return ranges->Check(r.at, bytes, what);
}

bool Meet(uint64_t a, uint64_t a_bytes, uint64_t b, uint64_t b_bytes) {
  return a_bytes > 0 && b_bytes > 0 && a < b + b_bytes && b < a + a_bytes;
}

// Rows in bytes: `blocks` of them `period` apart, each of `rows` of `width`
// bytes `step` apart (a stride of one row or block is 0).
struct Lattice {
  int64_t blocks = 1, period = 0, rows = 1, step = 0, width = 0;

  explicit Lattice(const Rows& r) : width(r.dim * r.item) {
    const int64_t t = r.tokens > 1 ? r.token_stride * r.item : 0;
    const int64_t h = r.heads > 1 ? r.head_stride * r.item : 0;
    const bool tokens_outside = t >= h;
    blocks = tokens_outside ? r.tokens : r.heads;
    period = tokens_outside ? t : h;
    rows = tokens_outside ? r.heads : r.tokens;
    step = tokens_outside ? h : t;
  }
  int64_t span() const { return (rows - 1) * step + width; }  // of a block
};

// Whether pieces of `a` and `b` bytes, each repeated `period` apart and the
// latter `gap` behind the former, stay apart.
bool Apart(int64_t a, int64_t b, int64_t period, int64_t gap) {
  if (period <= 0) return false;
  const int64_t at = (gap % period + period) % period;
  return a <= at && at + b <= period;
}

bool Meet(const Rows& a, const Rows& b) {
  uint64_t x = 0, y = 0;
  if (a.empty() || b.empty() || !a.Extent(&x) || !b.Extent(&y)) return false;
  if (!Meet(a.at, x, b.at, y)) return false;
  // Parts of one wider row (a fused projection): apart if no block of one
  // reaches into a block of the other, or, with heads side by side ([q, k, v] of
  // each), no row into a row.
  const Lattice l(a), m(b);
  const int64_t gap = static_cast<int64_t>(b.at - a.at);
  const auto common = [](int64_t s, int64_t n, int64_t t, int64_t k) {
    return n == 1 ? t : k == 1 || s == t ? s : 0;
  };
  const int64_t period = common(l.period, l.blocks, m.period, m.blocks);
  if (Apart(l.span(), m.span(), period, gap)) return false;
  const int64_t step = common(l.step, l.rows, m.step, m.rows);
  return step <= 0 || l.period % step != 0 || m.period % step != 0 ||
         !Apart(l.width, m.width, step, gap);
}

// An argument, with its extent.
struct Named {
  Rows rows;
  const char* name;
  uint64_t bytes = 0;

  Named(const Rows& r, const char* n) : rows(r), name(n) {
    if (r.empty() || !r.Extent(&bytes)) bytes = 0;
  }
};

// `bytes` bytes at an address, without gaps.
Rows Whole(uint64_t at, int64_t bytes) { return {at, 0, 0, bytes > 0 ? 1 : 0, 1, bytes, 1}; }

Status CheckApart(const Named& a, std::initializer_list<Named> others) {
  for (const Named& o : others) {
    if (Meet(a.rows.at, a.bytes, o.rows.at, o.bytes) && Meet(a.rows, o.rows)) {
      return Bad(std::string(a.name) + ": overlaps " + o.name);
    }
  }
  return OkStatus();
}

// Results may take the place of what they are computed from, row for row;
// any other overlap would be read after it is written.
Status CheckInPlace(const Rows& in, const Rows& out, const char* in_name, const char* out_name) {
  if (out.empty()) return OkStatus();
  if (out.SelfOverlaps()) return Bad(std::string(out_name) + ": rows overlap");
  if (!in.Same(out) && Meet(in, out)) {
    return Bad(std::string(out_name) + ": overlaps " + in_name +
               " (in place it has to have the same address and strides)");
  }
  return OkStatus();
}

Status CheckTokens(int64_t tokens, int64_t heads, int64_t dim) {
  if (tokens < 0 || tokens > kMostTokens) return Bad("tokens must be 0..2^30");
  if (heads < 0 || heads > 1024) return Bad("heads must be at most 1024");
  if (dim < 1 || dim > kMaxHeadDim) return Bad("head_dim must be 1..256");
  if (tokens * heads > INT32_MAX / 4) return Bad("tokens * heads must be below 2^29");
  return OkStatus();
}

Status CheckGrid(int64_t workgroups, int64_t threads) {
  return GridFits(workgroups, threads) ? OkStatus() : Bad("too many tokens for one call");
}
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

Status CheckWords(DeviceRangeChecker* ranges, uint64_t at, int64_t n, const char* what) {
  if (at % 4 != 0) return Bad(std::string(what) + ": unaligned address");
  return ranges->Check(at, static_cast<uint64_t>(n) * 4, what);
}

Status CheckBatch(DeviceRangeChecker* ranges, const kvx_paged_batch& b, int64_t tokens,
                  int64_t block_tokens, int64_t num_blocks, BatchView* out) {
  if (b.sequences < 0 || b.sequences > kMaxSequences) return Bad("sequences must be 0..4096");
  if (b.starts == 0 && tokens != b.sequences) {
    return Bad("without starts there is one token a sequence: tokens must equal sequences");
  }
  if (b.table_width < 0 || b.table_stride < 0) return Bad("negative table width or stride");
  if (block_tokens < 1) return Bad("block_tokens must be positive");
  if (b.table_width > kMostTokens / block_tokens) {
    return Bad("table_width * block_tokens must be at most 2^30");
  }
  if (b.sequences > 0) {
    int64_t words = 0;
    if (__builtin_mul_overflow(b.sequences - 1, b.table_stride, &words) ||
        __builtin_add_overflow(words, b.table_width, &words) || words > INT64_MAX / 4) {
      return Bad("tables: size overflows");
    }
    if (b.table_width > 0) KVX_RETURN_IF_ERROR(CheckWords(ranges, b.tables, words, "tables"));
    KVX_RETURN_IF_ERROR(CheckWords(ranges, b.lengths, b.sequences, "lengths"));
    if (b.starts != 0) {
      KVX_RETURN_IF_ERROR(CheckWords(ranges, b.starts, b.sequences + 1, "starts"));
    }
  }
  out->tables = reinterpret_cast<const int32_t*>(b.tables);
  out->lengths = reinterpret_cast<const int32_t*>(b.lengths);
  out->starts = reinterpret_cast<const int32_t*>(b.starts);
  out->table_stride = b.table_stride;
  out->table_width = static_cast<int32_t>(b.table_width);
  out->sequences = static_cast<int32_t>(b.sequences);
  out->tokens = static_cast<int32_t>(tokens);
  out->block_tokens = static_cast<int32_t>(block_tokens);
  out->capacity = static_cast<int32_t>(b.table_width * block_tokens);
  out->num_blocks = static_cast<int32_t>(num_blocks);
  return OkStatus();
}

// The arrays of a batch, checked before.
Rows Tables(const kvx_paged_batch& b) {
  return {b.tables, b.table_stride, 0, b.sequences, 1, b.table_width, 4};
}
Rows Lengths(const kvx_paged_batch& b) { return Whole(b.lengths, b.sequences * 4); }
Rows Starts(const kvx_paged_batch& b) {
  return Whole(b.starts, b.starts != 0 ? (b.sequences + 1) * 4 : 0);
}

struct Cache {
  PoolStorage k, v;
  PoolStorage k_scales, v_scales;  // e4m3
  int64_t num_blocks = 0;
};

Rows Whole(const PoolStorage& s) { return Whole(s.base, s.bytes); }

Status FindCache(const PoolSource& pool, const kvx_paged_cache& c, int32_t type, Cache* out) {
  if (!pool.device_backed) {
    return FailedPreconditionError("needs a device-backed KVCacheManagerBase");
  }
  if (!Is16Bit(type)) return Bad("dtype must be KVX_BF16 or KVX_F16");
  if (c.dtype != type && c.dtype != kE4m3) {
    return Bad("the cache must be of the tensors' type or KVX_E4M3");
  }
  if (c.heads < 1 || c.heads > 1024) return Bad("heads must be 1..1024");
  if (c.head_dim < 1 || c.head_dim > kMaxHeadDim) return Bad("head_dim must be 1..256");
  if (c.block_tokens < 1 || c.block_tokens > (1 << 20)) return Bad("block_tokens must be 1..2^20");
  if (!pool.find(pool.context, c.k_layer, c.shard, &out->k) ||
      !pool.find(pool.context, c.v_layer, c.shard, &out->v)) {
    return OutOfRangeError("layer or shard index out of range");
  }
  const int64_t block = static_cast<int64_t>(c.block_tokens) * c.heads * c.head_dim *
                        ElementBytes(c.dtype);
  if (out->k.block_bytes != block || out->v.block_bytes != block) {
    return Bad("blocks of " + std::to_string(out->k.block_bytes) + " and " +
               std::to_string(out->v.block_bytes) + " bytes do not hold [" +
               std::to_string(c.block_tokens) + ", " + std::to_string(c.heads) + ", " +
               std::to_string(c.head_dim) + "] of " + std::to_string(ElementBytes(c.dtype)) +
               " bytes");
  }
  int64_t blocks = std::min(out->k.bytes, out->v.bytes) / block;
  if (c.dtype == kE4m3) {
    PoolStorage s[2];
    if (!pool.find(pool.context, c.k_scale_layer, c.shard, &s[0]) ||
        !pool.find(pool.context, c.v_scale_layer, c.shard, &s[1])) {
      return OutOfRangeError("scale layer or shard index out of range");
    }
    for (const PoolStorage& t : s) {
      if (t.block_bytes != static_cast<int64_t>(c.heads) * 4) {
        return Bad("scale tables must hold one fp32 a (block, head): " +
                   std::to_string(c.heads * 4) + " bytes a block, not " +
                   std::to_string(t.block_bytes));
      }
      if (t.base % 4 != 0) return Bad("scale tables: unaligned address");
      blocks = std::min(blocks, t.bytes / t.block_bytes);
    }
    if (s[0].base == s[1].base) return Bad("keys and values need scale tables of their own");
    out->k_scales = s[0];
    out->v_scales = s[1];
  } else if ((out->k.base | out->v.base) % 2 != 0) {
    return Bad("cache storages: unaligned address");
  }
  if (out->k.base == out->v.base) return Bad("keys and values need storages of their own");
  if (blocks < 1) return Bad("the cache has no blocks");
  out->num_blocks = std::min<int64_t>(blocks, INT32_MAX);
  return OkStatus();
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
  out->k_scales = reinterpret_cast<float*>(cache.k_scales.base);
  out->v_scales = reinterpret_cast<float*>(cache.v_scales.base);
  out->k_weight = reinterpret_cast<const void*>(a.k_weight);
  out->positions = reinterpret_cast<const void*>(a.positions);
  out->inv_freq = reinterpret_cast<const float*>(a.inv_freq);
  out->heads = c.heads;
  out->head_dim = c.head_dim;
  out->rotary_dim = a.rotary_dim;
  out->type = a.dtype;
  out->e4m3 = c.dtype == kE4m3;
  out->weight_f32 = a.weight_dtype == kF32;
  out->positions_64 = a.positions_64 != 0;
  out->interleaved = a.interleaved != 0;
  out->eps = a.eps;
  return out->e4m3 ? CheckGrid(MostBlocks(*out), BlockThreads(*out)) : CheckRowGrid(a.tokens);
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
    // Sizes only: the address arguments may still be unset.
    if (a.batch.sequences < 0 || a.batch.sequences > kMaxSequences) {
      return Bad("sequences must be 0..4096");
    }
    if (a.batch.table_width < 0 || a.batch.table_width > kMostTokens / c.block_tokens) {
      return Bad("table_width * block_tokens must be at most 2^30");
    }
    out->batch.starts = reinterpret_cast<const int32_t*>(a.batch.starts);
    out->batch.sequences = static_cast<int32_t>(a.batch.sequences);
    out->batch.tokens = static_cast<int32_t>(a.tokens);
    out->batch.capacity = static_cast<int32_t>(a.batch.table_width * c.block_tokens);
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
  out->k_scales = reinterpret_cast<const float*>(cache.k_scales.base);
  out->v_scales = reinterpret_cast<const float*>(cache.v_scales.base);
  out->group_starts = reinterpret_cast<const int32_t*>(a.group_starts);
  out->prefix_lengths = reinterpret_cast<const int32_t*>(a.prefix_lengths);
  out->groups = a.groups;
  out->q_heads = a.q_heads;
  out->k_heads = c.heads;
  out->head_dim = c.head_dim;
  out->type = a.dtype;
  out->e4m3 = c.dtype == kE4m3;
  out->causal = a.non_causal == 0;
  out->scale = a.scale;
  const int64_t need = out->batch.tokens == 0 ? 0 : PlanAttend(out);
  if (workspace_bytes != nullptr) {
    *workspace_bytes = need;
    return OkStatus();
  }
  if (!out->e4m3 && (reinterpret_cast<uintptr_t>(out->k_pool) |
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
