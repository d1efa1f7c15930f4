#include "paged_args.h"

#include <algorithm>

namespace kvx {
namespace paged {
namespace {

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

}  // namespace

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

Status CheckApart(const Named& a, std::initializer_list<Named> others) {
  for (const Named& o : others) {
    if (Meet(a.rows.at, a.bytes, o.rows.at, o.bytes) && Meet(a.rows, o.rows)) {
      return Bad(std::string(a.name) + ": overlaps " + o.name);
    }
  }
  return OkStatus();
}

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
Status CheckWords(DeviceRangeChecker* ranges, uint64_t at, int64_t n, const char* what) {
  if (at % 4 != 0) return Bad(std::string(what) + ": unaligned address");
  return ranges->Check(at, static_cast<uint64_t>(n) * 4, what);
}

Status CheckSizes(const kvx_paged_batch& b, int64_t tokens, int64_t block_tokens, BatchView* out) {
  if (b.sequences < 0 || b.sequences > kMaxSequences) return Bad("sequences must be 0..4096");
  if (b.table_width < 0 || b.table_width > kMostTokens / block_tokens) {
    return Bad("table_width * block_tokens must be at most 2^30");
  }
  out->starts = reinterpret_cast<const int32_t*>(b.starts);
  out->sequences = static_cast<int32_t>(b.sequences);
  out->tokens = static_cast<int32_t>(tokens);
  out->capacity = static_cast<int32_t>(b.table_width * block_tokens);
  return OkStatus();
}

Status CheckTables(DeviceRangeChecker* ranges, const kvx_paged_batch& b, int64_t block_tokens,
                   int64_t num_blocks, BatchView* out) {
  if (b.sequences < 0 || b.sequences > kMaxSequences) return Bad("sequences must be 0..4096");
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
  }
  out->tables = reinterpret_cast<const int32_t*>(b.tables);
  out->table_stride = b.table_stride;
  out->table_width = static_cast<int32_t>(b.table_width);
  out->sequences = static_cast<int32_t>(b.sequences);
  out->block_tokens = static_cast<int32_t>(block_tokens);
  out->capacity = static_cast<int32_t>(b.table_width * block_tokens);
  out->num_blocks = static_cast<int32_t>(num_blocks);
  return OkStatus();
}

Status CheckBatch(DeviceRangeChecker* ranges, const kvx_paged_batch& b, int64_t tokens,
                  int64_t block_tokens, int64_t num_blocks, BatchView* out) {
  if (b.sequences < 0 || b.sequences > kMaxSequences) return Bad("sequences must be 0..4096");
  if (b.starts == 0 && tokens != b.sequences) {
    return Bad("without starts there is one token a sequence: tokens must equal sequences");
  }
  KVX_RETURN_IF_ERROR(CheckTables(ranges, b, block_tokens, num_blocks, out));
  if (b.sequences > 0) {
    KVX_RETURN_IF_ERROR(CheckWords(ranges, b.lengths, b.sequences, "lengths"));
    if (b.starts != 0) {
      KVX_RETURN_IF_ERROR(CheckWords(ranges, b.starts, b.sequences + 1, "starts"));
    }
  }
  out->lengths = reinterpret_cast<const int32_t*>(b.lengths);
  out->starts = reinterpret_cast<const int32_t*>(b.starts);
  out->tokens = static_cast<int32_t>(tokens);
  return OkStatus();
}

Rows Tables(const kvx_paged_batch& b) {
  return {b.tables, b.table_stride, 0, b.sequences, 1, b.table_width, 4};
}

Status FindCache(const PoolSource& pool, const kvx_paged_cache& c, int32_t type, Cache* out,
                 bool with_values) {
  if (!pool.device_backed) {
    return FailedPreconditionError("needs a device-backed KVCacheManagerBase");
  }
  if (!Is16Bit(type)) return Bad("dtype must be KVX_BF16 or KVX_F16");
  if (c.dtype != type && c.dtype != kE4m3 && c.dtype != kFp4) {
    return Bad("the cache must be of the tensors' type, KVX_E4M3 or KVX_FP4");
  }
  if (c.heads < 1 || c.heads > 1024) return Bad("heads must be 1..1024");
  if (c.head_dim < 1 || c.head_dim > kMaxHeadDim) return Bad("head_dim must be 1..256");
  if (c.block_tokens < 1 || c.block_tokens > (1 << 20)) return Bad("block_tokens must be 1..2^20");
  if (!pool.find(pool.context, c.k_layer, c.shard, &out->k) ||
      (with_values && !pool.find(pool.context, c.v_layer, c.shard, &out->v))) {
    return OutOfRangeError("layer or shard index out of range");
  }
  if (!with_values) out->v = out->k;
  const bool fp4 = c.dtype == kFp4;
  if (fp4 && c.head_dim % kFp4Group != 0) {
    return Bad("head_dim must be a multiple of 32 in a KVX_FP4 cache");
  }
  const int64_t values = static_cast<int64_t>(c.block_tokens) * c.heads * c.head_dim;
  const int64_t block = fp4 ? values / 2 : values * ElementBytes(c.dtype);
  if (out->k.block_bytes != block || out->v.block_bytes != block) {
    return Bad("blocks of " + std::to_string(out->k.block_bytes) + " and " +
               std::to_string(out->v.block_bytes) + " bytes do not hold [" +
               std::to_string(c.block_tokens) + ", " + std::to_string(c.heads) + ", " +
               std::to_string(c.head_dim) + "] of " +
               (fp4 ? "4 bits" : std::to_string(ElementBytes(c.dtype)) + " bytes"));
  }
  int64_t blocks = std::min(out->k.bytes, out->v.bytes) / block;
  if (c.dtype == kE4m3 || fp4) {
    PoolStorage s[2];
    if (!pool.find(pool.context, c.k_scale_layer, c.shard, &s[0]) ||
        (with_values && !pool.find(pool.context, c.v_scale_layer, c.shard, &s[1]))) {
      return OutOfRangeError("scale layer or shard index out of range");
    }
    if (!with_values) s[1] = s[0];
    for (const PoolStorage& t : s) {
      if (fp4 && t.block_bytes != values / kFp4Group) {
        return Bad("scale tables must hold one byte for 32 values: " +
                   std::to_string(values / kFp4Group) + " bytes a block, not " +
                   std::to_string(t.block_bytes));
      }
      if (!fp4 && t.block_bytes != static_cast<int64_t>(c.heads) * 4) {
        return Bad("scale tables must hold one fp32 a (block, head): " +
                   std::to_string(c.heads * 4) + " bytes a block, not " +
                   std::to_string(t.block_bytes));
      }
      if (!fp4 && t.base % 4 != 0) return Bad("scale tables: unaligned address");
      blocks = std::min(blocks, t.bytes / t.block_bytes);
    }
    if (with_values && s[0].base == s[1].base) return Bad("keys and values need scale tables of their own");
    out->k_scales = s[0];
    out->v_scales = s[1];
    if (fp4 && (out->k.base | out->v.base) % 16 != 0) {
      return Bad("cache storages: must be aligned to 16 bytes");
    }
  } else if ((out->k.base | out->v.base) % 2 != 0) {
    return Bad("cache storages: unaligned address");
  }
  if (with_values && out->k.base == out->v.base) return Bad("keys and values need storages of their own");
  if (blocks < 1) return Bad("the cache has no blocks");
  out->num_blocks = std::min<int64_t>(blocks, INT32_MAX);
  return OkStatus();
}

}  // namespace paged
}  // namespace kvx
