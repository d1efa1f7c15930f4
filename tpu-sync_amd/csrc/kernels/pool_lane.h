// How a wave takes 16 tokens of a pool as an operand of the matrix instructions:
// lane l holds token l % 16 and, for each product of 32 dimensions, eight of them
// that l / 16 chooses. The order in which a product goes through the dimensions is
// free as long as the queries follow it, so a lane takes as many in a row as make a
// load of 16 bytes: 8 of a 16-bit pool, 16 in e4m3 where they come in pairs of
// products, 32 in 4 bits, which at 64 and 128 dimensions have one scale.
#ifndef KVX_KERNELS_POOL_LANE_H_
#define KVX_KERNELS_POOL_LANE_H_

#include "attend_plan.h"

namespace kvx {

template <class E, int POOL, int DP, bool FULL>
struct PoolLane {
  using Scalar = typename E::Scalar;
  static constexpr int KS = DP / 32;  // products
  static constexpr bool E4 = POOL == kPoolE4m3, F4 = POOL == kPoolFp4;
  // 128 sequences of 8 query heads on one e4m3 head, 300 to 16384 tokens, D = 128:
  // 56 us (4.7 TB/s); with 8 dimensions in a row 76 us.
  static constexpr bool kWide = E4 && FULL && KS % 2 == 0;
  static constexpr int kRun = KS < 4 ? KS : 4;  // chunks in a row in 4 bits
  // Scales that a lane's dimensions have in 4 bits.
  static constexpr int kScales = !F4 ? 0 : KS == 3 || KS == 8 ? 2 : 1;
  // Eight dimensions as they lie in the pool.
  using Words = std::conditional_t<F4, uint32_t,
                                   __attribute__((ext_vector_type(E4 ? 2 : 4))) uint32_t>;

  int quarter, h, head_dim, heads, block_tokens;

  __device__ PoolLane(int lane, int head, const AttendLaunch& a)
      : quarter(lane / 16),
        h(head),
        head_dim(FULL ? DP : a.head_dim),
        heads(a.k_heads),
        block_tokens(a.batch.block_tokens) {}

  // First dimension of a lane's chunk.
  static __device__ __forceinline__ int DimOf(int quarter, int ks) {
    if constexpr (F4) return ks / 4 * 128 + quarter * (kRun * 8) + ks % 4 * 8;
    return kWide ? ks / 2 * 64 + quarter * 16 + ks % 2 * 8 : ks * 32 + quarter * 8;
  }
  __device__ __forceinline__ int Dim(int ks) const { return DimOf(quarter, ks); }

  // Where the lane's part of a token starts: in elements, in 4 bits the token's row.
  __device__ __forceinline__ int64_t At(int id, int slot, bool has) const {
    if constexpr (F4) {
      return (static_cast<int64_t>(has ? id : 0) * heads + h) * block_tokens + (has ? slot : 0);
    }
    const int64_t row = static_cast<int64_t>(id) * block_tokens + slot;
    return (has ? row : 0) * (static_cast<int64_t>(heads) * head_dim) + h * head_dim +
           quarter * (kWide ? 16 : 8);
  }

  __device__ __forceinline__ void Load(const void* pool, int64_t at, Words (&w)[KS]) const {
    if constexpr (F4) {
      const uint8_t* p = static_cast<const uint8_t*>(pool) + at * (head_dim / 2);
      if constexpr (FULL) {
        using Run = __attribute__((ext_vector_type(kRun))) uint32_t;
        using Unaligned = Run __attribute__((aligned(4)));
#pragma unroll
        for (int ks = 0; ks < KS; ks += kRun) {
          const Run x = *reinterpret_cast<const Unaligned*>(p + Dim(ks) / 2);
#pragma unroll
          for (int i = 0; i < kRun; ++i) w[ks + i] = x[i];
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          w[ks] = 0;
          if (Dim(ks) < head_dim) w[ks] = *reinterpret_cast<const uint32_t*>(p + Dim(ks) / 2);
        }
      }
      return;
    } else if constexpr (kWide) {
#pragma unroll
      for (int ks = 0; ks < KS; ks += 2) {
        using Wide = u32x4 __attribute__((aligned(1)));
        const u32x4 x =
            *reinterpret_cast<const Wide*>(static_cast<const uint8_t*>(pool) + at + ks * 32);
        w[ks] = Words{x[0], x[1]};
        w[ks + 1] = Words{x[2], x[3]};
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (!FULL) w[ks] = Words(0);
        if (FULL || ks * 32 + quarter * 8 < head_dim) {
          if constexpr (E4) {
            w[ks] = *reinterpret_cast<const Bytes8*>(static_cast<const uint8_t*>(pool) + at + ks * 32);
          } else {
            w[ks] = *reinterpret_cast<const Bytes16*>(static_cast<const Scalar*>(pool) + at + ks * 32);
          }
        }
      }
    }
  }

  // Scale of chunk ks, of those that LoadScales reads.
  __device__ __forceinline__ int ScaleOf(int ks) const {
    if constexpr (KS == 3) return Dim(ks) / kFp4Group != Dim(0) / kFp4Group ? 1 : 0;
    return KS == 8 ? ks / 4 : 0;
  }
  // e8m0 codes of a token's scales.
  __device__ __forceinline__ void LoadScales(const void* scales, int64_t at,
                                             uint32_t (&f)[kScales > 0 ? kScales : 1]) const {
    const int groups = head_dim / kFp4Group;
    const uint8_t* p = static_cast<const uint8_t*>(scales) + at * groups;
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      f[i] = p[min(Dim(i * (KS == 3 ? 2 : 4)) / kFp4Group, groups - 1)];
    }
  }
  // A chunk of a 4-bit pool as an operand.
  __device__ __forceinline__ u32x4 FromCodes(uint32_t w, const uint32_t (&f)[kScales > 0 ? kScales : 1],
                                             int ks) const {
    uint32_t code = f[0];
    if constexpr (kScales > 1) code = ScaleOf(ks) == 0 ? f[0] : f[1];
    return FromFp4<E>(w, Fp4Scale<E>(code));
  }
};

}  // namespace kvx

#endif  // KVX_KERNELS_POOL_LANE_H_
