// Device code of one head's row: RMS norm and position rotation, shared by
// the kernels that do it on the way to another place.
//
// A row of D elements lies across a team of LPR lanes, lane l holding the chunks
// l + LPR * n of VEC elements. The sum of squares is taken over the lanes; the
// other half of a rotated pair is read again from the row (the line is in the
// cache) instead of being moved between lanes, so any rotated width fits. VEC is
// 16 bytes where addresses and widths allow it, else 1.
//
// With x the row, o its pairs' other halves (o negated where it is subtracted)
// and r = 1 / sqrt(mean(x^2) + eps), the result is r (x A + o B) with
//   A = w cos, B = w' sin   (w' the weight at the other half),
// and A, B are the same for every head of a token: a team takes one token's
// heads in turn and multiplies weights and angles once.
#ifndef KVX_KERNELS_HEAD_ROW_H_
#define KVX_KERNELS_HEAD_ROW_H_

#include <type_traits>

#include "kv_element.h"

#ifdef __HIPCC__
namespace kvx {

// A chunk as it lies in memory.
template <class E, int VEC>
struct Chunk {
  using Raw = std::conditional_t<VEC == 1, typename E::Scalar,
                                 std::conditional_t<VEC == 8, u32x4, f32x4>>;
  Raw raw;

  __device__ __forceinline__ void Load(const typename E::Scalar* p) {
    raw = *reinterpret_cast<const Raw*>(p);
  }
  __device__ __forceinline__ void Store(typename E::Scalar* p) const {
    *reinterpret_cast<Raw*>(p) = raw;
  }
  __device__ __forceinline__ void Clear() { raw = Raw(0); }
  __device__ __forceinline__ void To(float* x) const {
    if constexpr (VEC == 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2 f = Unpack2<E>(raw[j]);
        x[2 * j] = f[0];
        x[2 * j + 1] = f[1];
      }
    } else if constexpr (VEC == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = raw[j];
    } else {
      x[0] = static_cast<float>(raw);
    }
  }
  __device__ __forceinline__ void From(const float* x) {
    if constexpr (VEC == 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j] = Pack2<E>(x[2 * j], x[2 * j + 1]);
    } else if constexpr (VEC == 4) {
      raw = f32x4{x[0], x[1], x[2], x[3]};
    } else {
      raw = static_cast<typename E::Scalar>(x[0]);
    }
  }
  // -x where `negative` (all of the lane's).
  __device__ __forceinline__ void Negate(bool negative) {
    if constexpr (VEC == 8) {
      const uint32_t sign = negative ? 0x80008000u : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j] ^= sign;
    } else {
      if (negative) raw = -raw;
    }
  }
};

// Sum over the LPR lanes of a team, in each of them.
template <int LPR>
__device__ __forceinline__ float TeamSum(float x) {
  const auto add = [&x](auto control) {
    x += __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(control)::value,
                                           0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xb1>{});   // lanes 1 0 3 2
  add(std::integral_constant<int, 0x4e>{});   // lanes 2 3 0 1
  add(std::integral_constant<int, 0x141>{});  // halves of eight, mirrored
  if constexpr (LPR >= 16) add(std::integral_constant<int, 0x140>{});  // sixteen, mirrored
  if constexpr (LPR >= 32) x += __shfl_xor(x, 16);
  if constexpr (LPR >= 64) x += __shfl_xor(x, 32);
  return x;
}

// Chunk of a norm's weight, of the row's type or fp32, as floats.
template <class E, int VEC>
__device__ __forceinline__ void LoadWeight(const void* w, bool f32, int d, float* x) {
  if (f32) {
    using Four = f32x4 __attribute__((aligned(4)));
    const float* p = static_cast<const float*>(w) + d;
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const f32x4 f = *reinterpret_cast<const Four*>(p + j);
        x[j] = f[0];
        x[j + 1] = f[1];
        x[j + 2] = f[2];
        x[j + 3] = f[3];
      }
    } else {
      x[0] = *p;
    }
    return;
  }
  const auto* p = static_cast<const typename E::Scalar*>(w) + d;
  if constexpr (VEC == 8) {
    using Eight = u32x4 __attribute__((aligned(2)));
    Chunk<E, VEC> c;
    c.raw = *reinterpret_cast<const Eight*>(p);
    c.To(x);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = static_cast<float>(p[j]);
  }
}

// What a lane needs to know of its chunks, fixed for all rows of one kind.
template <class E, int VEC, int LPR>
struct RowLane {
  static constexpr int kChunks = VEC == 1 ? 4 : 1;  // 256 / 64
  int dim, rotary;
  bool interleaved;
  int lane;  // in its row

  __device__ RowLane(int head_dim, int rotary_dim, bool inter)
      : dim(head_dim), rotary(rotary_dim), interleaved(inter), lane(threadIdx.x % LPR) {}

  __device__ __forceinline__ int Dim(int n) const { return (lane + LPR * n) * VEC; }
  __device__ __forceinline__ bool Has(int n) const { return Dim(n) < dim; }
  __device__ __forceinline__ bool Rotated(int n) const { return Dim(n) < rotary; }
  // Whether the pairs' other halves are in another chunk, and where.
  __device__ __forceinline__ bool Apart() const { return VEC == 1 || !interleaved; }
  __device__ __forceinline__ int Other(int n) const {
    const int d = Dim(n), half = rotary / 2;
    if (interleaved) return d ^ 1;
    return d < half ? d + half : d - half;
  }
  // Whether chunk n's results subtract the other halves.
  __device__ __forceinline__ bool First(int n) const {
    return interleaved ? (Dim(n) & 1) == 0 : Dim(n) < rotary / 2;
  }
  // Pair of element j of chunk n: index into its token's cos and sin.
  __device__ __forceinline__ int Pair(int n, int j) const {
    const int d = Dim(n), half = rotary / 2;
    if (interleaved) return (d + j) / 2;
    return (d < half ? d : d - half) + j;
  }
};

// One row's chunks and, where they are rotated, the chunks of their pairs'
// other halves, as loaded.
template <class E, int VEC, int LPR>
struct RawRow {
  using Lane = RowLane<E, VEC, LPR>;
  Chunk<E, VEC> x[Lane::kChunks], o[Lane::kChunks];

  __device__ __forceinline__ void Load(const Lane& l, const typename E::Scalar* p,
                                       bool with_pairs) {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
      x[n].Clear();
      o[n].Clear();
      if (l.Has(n)) {
        x[n].Load(p + l.Dim(n));
        if (with_pairs && l.Rotated(n) && l.Apart()) o[n].Load(p + l.Other(n));
      }
    }
  }
  __device__ __forceinline__ void Store(const Lane& l, typename E::Scalar* p) const {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
      if (l.Has(n)) x[n].Store(p + l.Dim(n));
    }
  }
};

// A lane's weights, and those at the other halves of its pairs; 1 without a norm.
template <class E, int VEC, int LPR>
struct Weights {
  using Lane = RowLane<E, VEC, LPR>;
  float w[Lane::kChunks][VEC], o[Lane::kChunks][VEC];

  __device__ __forceinline__ void Load(const Lane& l, const void* weight, bool f32) {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[n][j] = o[n][j] = 1.0f;
      if (weight == nullptr || !l.Has(n)) continue;
      LoadWeight<E, VEC>(weight, f32, l.Dim(n), w[n]);
      if (!l.Rotated(n)) continue;
      if (l.Apart()) {
        LoadWeight<E, VEC>(weight, f32, l.Other(n), o[n]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[n][j] = w[n][VEC > 1 ? j ^ 1 : j];
      }
    }
  }
};

// A and B of one token for a lane's chunks.
template <class E, int VEC, int LPR>
struct Factors {
  using Lane = RowLane<E, VEC, LPR>;
  float a[Lane::kChunks][VEC], b[Lane::kChunks][VEC];

  // cs: (cos, sin) of the token, one of each pair.
  __device__ __forceinline__ Factors(const Lane& l, const f32x2* cs,
                                     const Weights<E, VEC, LPR>& weights) {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        a[n][j] = weights.w[n][j];
        b[n][j] = 0.0f;
        if (l.Rotated(n)) {
          const f32x2 t = cs[l.Pair(n, j)];
          a[n][j] *= t[0];
          b[n][j] = weights.o[n][j] * t[1];
        }
      }
    }
  }
};

// A row in fp32.
template <class E, int VEC, int LPR>
struct Row {
  using Lane = RowLane<E, VEC, LPR>;
  float x[Lane::kChunks][VEC];

  // r (x A + o B), r = 1 without a norm.
  __device__ __forceinline__ Row(const Lane& l, RawRow<E, VEC, LPR>& raw,
                                 const Factors<E, VEC, LPR>& f, bool norm, float eps) {
    float o[Lane::kChunks][VEC];
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
      raw.x[n].To(x[n]);
      if (l.Apart()) {
        raw.o[n].Negate(l.First(n));
        raw.o[n].To(o[n]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float other = x[n][VEC > 1 ? j ^ 1 : j];
          o[n][j] = !l.Rotated(n) ? 0.0f : j % 2 == 0 ? -other : other;
        }
      }
    }
    float r = 1.0f;
    if (norm) {
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < Lane::kChunks; ++n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum += x[n][j] * x[n][j];
      }
      r = rsqrtf(TeamSum<LPR>(sum) / static_cast<float>(l.dim) + eps);
    }
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        x[n][j] = fmaf(o[n][j], f.b[n][j], x[n][j] * f.a[n][j]);
        if (norm) x[n][j] *= r;
      }
    }
  }
  // As loaded.
  __device__ __forceinline__ explicit Row(const RawRow<E, VEC, LPR>& raw) {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) raw.x[n].To(x[n]);
  }

  __device__ __forceinline__ void Store(const Lane& l, typename E::Scalar* p) const {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
      if (!l.Has(n)) continue;
      Chunk<E, VEC> c;
      c.From(x[n]);
      c.Store(p + l.Dim(n));
    }
  }
};

// Teams that take one token's heads in turn: as many as there are heads, at
// most a wave's.
constexpr int TeamsOfToken(int heads, int lpr) {
  int n = 1;
  while (n < heads && n < 64 / lpr) n *= 2;
  return n;
}

// Whether rows can move in 16-byte chunks of `vec` elements: every stride,
// the width and the rotated half are whole chunks and every address is aligned.
inline bool ChunksFit(int vec, int dim, int rotary, bool interleaved) {
  return dim % vec == 0 && rotary % (interleaved ? vec : 2 * vec) == 0;
}

}  // namespace kvx
#endif  // __HIPCC__

#endif  // KVX_KERNELS_HEAD_ROW_H_
