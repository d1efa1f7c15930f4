// Device code of one head's row: RMS norm and position rotation, shared by
// the kernels that do it on the way to another place.
//
// A row of D elements lies across LPR lanes, lane l holding the chunks
// l + LPR * n of VEC elements. The sum of squares is taken over the lanes with
// shuffles; the other half of a rotated pair is read again from the row (the
// line is in the cache) instead of being moved between lanes, so any rotated
// width fits. VEC is 16 bytes where addresses and widths allow it, else 1.
#ifndef KVX_KERNELS_HEAD_ROW_H_
#define KVX_KERNELS_HEAD_ROW_H_

#include "kv_element.h"

#ifdef __HIPCC__
namespace kvx {

template <class E, int VEC>
__device__ __forceinline__ void LoadChunk(const typename E::Scalar* p, float* x) {
  if constexpr (VEC == 8) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 f = Unpack2<E>(w[j]);
      x[2 * j] = f[0];
      x[2 * j + 1] = f[1];
    }
  } else if constexpr (VEC == 4) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = w[j];
  } else {
    x[0] = static_cast<float>(*p);
  }
}

template <class E, int VEC>
__device__ __forceinline__ void StoreChunk(typename E::Scalar* p, const float* x) {
  if constexpr (VEC == 8) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = Pack2<E>(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<u32x4*>(p) = w;
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
  } else {
    *p = static_cast<typename E::Scalar>(x[0]);
  }
}

// Chunk of a norm's weight, of the row's type or fp32, as floats.
template <class E, int VEC>
__device__ __forceinline__ void LoadWeight(const void* w, bool f32, int d, float* x) {
  if (f32) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = static_cast<const float*>(w)[d + j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[j] = static_cast<float>(static_cast<const typename E::Scalar*>(w)[d + j]);
    }
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
  // First dimension of the chunk that holds the pairs' other halves.
  __device__ __forceinline__ int Other(int n) const {
    const int d = Dim(n), half = rotary / 2;
    if (interleaved) return VEC == 1 ? (d ^ 1) : d;
    return d < half ? d + half : d - half;
  }
  // First pair of chunk n: index into the row's cos and sin.
  __device__ __forceinline__ int Pair(int n) const {
    const int d = Dim(n), half = rotary / 2;
    if (interleaved) return d / 2;
    return d < half ? d : d - half;
  }
};

// One row's chunks and, where they are rotated, the chunks of their pairs'
// other halves.
template <class E, int VEC, int LPR>
struct Row {
  using Lane = RowLane<E, VEC, LPR>;
  float x[Lane::kChunks][VEC];
  float o[Lane::kChunks][VEC];

  __device__ __forceinline__ void Load(const Lane& l, const typename E::Scalar* p) {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[n][j] = o[n][j] = 0.0f;
      if (l.Has(n)) {
        LoadChunk<E, VEC>(p + l.Dim(n), x[n]);
        if (l.Rotated(n) && (VEC == 1 || !l.interleaved)) {
          LoadChunk<E, VEC>(p + l.Other(n), o[n]);
        }
      }
    }
  }

  // x * weight / sqrt(mean(x^2) + eps), the mean over the row's lanes.
  __device__ __forceinline__ void Norm(const Lane& l, const float (&w)[Lane::kChunks][VEC],
                                       const float (&wo)[Lane::kChunks][VEC], float eps) {
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum += x[n][j] * x[n][j];
    }
#pragma unroll
    for (int m = LPR / 2; m > 0; m /= 2) sum += __shfl_xor(sum, m);
    const float r = 1.0f / sqrtf(sum / static_cast<float>(l.dim) + eps);
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        x[n][j] *= r * w[n][j];
        o[n][j] *= r * wo[n][j];
      }
    }
  }

  // cs: (cos, sin) of the row's token, one of each pair.
  __device__ __forceinline__ void Rotate(const Lane& l, const f32x2* cs) {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
      if (!l.Rotated(n)) continue;
      const f32x2* c = cs + l.Pair(n);
      if (l.interleaved && VEC > 1) {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          const f32x2 t = c[j / 2];
          const float u = x[n][j], v = x[n][VEC > 1 ? j + 1 : j];
          x[n][j] = u * t[0] - v * t[1];
          x[n][VEC > 1 ? j + 1 : j] = v * t[0] + u * t[1];
        }
      } else {
        const int d = l.Dim(n);
        const bool first = l.interleaved ? (d & 1) == 0 : d < l.rotary / 2;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const f32x2 t = c[j];
          x[n][j] = first ? x[n][j] * t[0] - o[n][j] * t[1] : x[n][j] * t[0] + o[n][j] * t[1];
        }
      }
    }
  }

  __device__ __forceinline__ void Store(const Lane& l, typename E::Scalar* p) const {
#pragma unroll
    for (int n = 0; n < Lane::kChunks; ++n) {
      if (l.Has(n)) StoreChunk<E, VEC>(p + l.Dim(n), x[n]);
    }
  }
};

// Weight chunks of a lane (own and the other halves'), 1 without a norm.
template <class E, int VEC, int LPR>
__device__ __forceinline__ void LoadWeights(const RowLane<E, VEC, LPR>& l, const void* w, bool f32,
                                            float (&own)[RowLane<E, VEC, LPR>::kChunks][VEC],
                                            float (&other)[RowLane<E, VEC, LPR>::kChunks][VEC]) {
#pragma unroll
  for (int n = 0; n < RowLane<E, VEC, LPR>::kChunks; ++n) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) own[n][j] = other[n][j] = 1.0f;
    if (w != nullptr && l.Has(n)) {
      LoadWeight<E, VEC>(w, f32, l.Dim(n), own[n]);
      if (l.Rotated(n)) LoadWeight<E, VEC>(w, f32, l.Other(n), other[n]);
    }
  }
}

// Whether rows can move in 16-byte chunks of `vec` elements: every stride,
// the width and the rotated half are whole chunks and every address is aligned.
inline bool ChunksFit(int vec, int dim, int rotary, bool interleaved) {
  return dim % vec == 0 && rotary % (interleaved ? vec : 2 * vec) == 0;
}

}  // namespace kvx
#endif  // __HIPCC__

#endif  // KVX_KERNELS_HEAD_ROW_H_
