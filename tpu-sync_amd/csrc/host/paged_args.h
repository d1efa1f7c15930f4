// Checks that the operators on the paged pool share: addresses, strides,
// overlaps, a call's sequences and the storages of a layer.
#ifndef KVX_HOST_PAGED_ARGS_H_
#define KVX_HOST_PAGED_ARGS_H_

#include <climits>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../../include/kvx.h"
#include "../kernels/attend.h"
#include "../kernels/kv_element.h"
#include "attention_args.h"
#include "device_memory.h"
#include "status.h"

namespace kvx {
namespace paged {

constexpr int64_t kMostTokens = int64_t{1} << 30;  // of a call and of a table row

inline Status Bad(const std::string& what) { return InvalidArgumentError(what); }

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

Status CheckRows(DeviceRangeChecker* ranges, const Rows& r, const char* what);

// Whether two arguments share bytes.
bool Meet(const Rows& a, const Rows& b);

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
inline Rows Whole(uint64_t at, int64_t bytes) {
  return {at, 0, 0, bytes > 0 ? 1 : 0, 1, bytes, 1};
}
inline Rows Whole(const PoolStorage& s) { return Whole(s.base, s.bytes); }

Status CheckApart(const Named& a, std::initializer_list<Named> others);

// Results may take the place of what they are computed from, row for row;
// any other overlap would be read after it is written.
Status CheckInPlace(const Rows& in, const Rows& out, const char* in_name, const char* out_name);

Status CheckTokens(int64_t tokens, int64_t heads, int64_t dim);
Status CheckGrid(int64_t workgroups, int64_t threads);
Status CheckWords(DeviceRangeChecker* ranges, uint64_t at, int64_t n, const char* what);

// A batch's sizes alone: the addresses may still be unset.
Status CheckSizes(const kvx_paged_batch& b, int64_t tokens, int64_t block_tokens, BatchView* out);
// The tables of a batch alone, and all of it.
Status CheckTables(DeviceRangeChecker* ranges, const kvx_paged_batch& b, int64_t block_tokens,
                   int64_t num_blocks, BatchView* out);
Status CheckBatch(DeviceRangeChecker* ranges, const kvx_paged_batch& b, int64_t tokens,
                  int64_t block_tokens, int64_t num_blocks, BatchView* out);
// The arrays of a batch, checked before.
Rows Tables(const kvx_paged_batch& b);
inline Rows Lengths(const kvx_paged_batch& b) { return Whole(b.lengths, b.sequences * 4); }
inline Rows Starts(const kvx_paged_batch& b) {
  return Whole(b.starts, b.starts != 0 ? (b.sequences + 1) * 4 : 0);
}

struct Cache {
  PoolStorage k, v;
  PoolStorage k_scales, v_scales;  // e4m3 and 4 bits
  int64_t num_blocks = 0;
};

inline int32_t KindOf(int32_t cache_type) {
  return cache_type == kE4m3 ? kPoolE4m3 : cache_type == kFp4 ? kPoolFp4 : kPoolSame;
}

// The storages of a layer; without `values`, its keys alone.
Status FindCache(const PoolSource& pool, const kvx_paged_cache& c, int32_t type, Cache* out,
                 bool values = true);

}  // namespace paged
}  // namespace kvx

#endif  // KVX_HOST_PAGED_ARGS_H_
