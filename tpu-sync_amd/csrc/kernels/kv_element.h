// Element types of the operators that fill and read the paged KV pool, and
// what their kernels share on the device.
#ifndef KVX_KERNELS_KV_ELEMENT_H_
#define KVX_KERNELS_KV_ELEMENT_H_

#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace kvx {

enum ElementType : int32_t {
  kBf16 = 0,
  kF16 = 1,
  kF32 = 2,
  kE4m3 = 3,  // OCP e4m3 (no infinities, largest value 448)
  kFp4 = 4,   // OCP e2m1 with one e8m0 scale for 32 neighbouring values
};

constexpr bool Is16Bit(int32_t t) { return t == kBf16 || t == kF16; }
constexpr int64_t ElementBytes(int32_t t) { return t == kF32 ? 4 : t == kE4m3 ? 1 : 2; }  // not kFp4
constexpr float kE4m3Max = 448.0f;
constexpr int kFp4Group = 32;  // values that share a scale

// How a pool is held, next to tensors of a 16-bit type.
enum PoolKind : int {
  kPoolSame = 0,  // [blocks][tokens][heads][dim] of the tensors' type
  kPoolE4m3 = 1,  // the same in e4m3, scales [blocks][heads] fp32
  // e2m1 codes [blocks][heads][tokens][dim / 2] and e8m0 scales [blocks][heads]
  // [tokens][dim / 32]. A head's tokens of a block lie together: a row is 64 bytes at
  // 128 dimensions, half a cache line, which heads side by side would each read whole.
  kPoolFp4 = 2,
};

// A launch counts the threads of a grid's dimension in 32 bits.
constexpr bool GridFits(int64_t workgroups, int64_t threads) {
  return workgroups <= UINT32_MAX / threads;
}
// Of the kernels that take up to so many tokens a workgroup of so many threads.
constexpr int kRowThreads = 256;
constexpr int kMostRowTokens = 32;

// x + y, but at most `most`, for x and y of [0, most]. Work is summed up so
// where it comes from device arrays: a valid call's sums stay below `most`, and
// starts that are out of order, whose tokens count for many sequences, can
// neither make more work nor wrap around to places that others have.
constexpr int AddUpTo(int x, int y, int most) {
  const uint32_t sum = static_cast<uint32_t>(x) + static_cast<uint32_t>(y);
  return sum < static_cast<uint32_t>(most) ? static_cast<int>(sum) : most;
}

// The sequences of a call. Sequence s owns the new tokens [starts[s],
// starts[s + 1]) (starts null: token s) and holds lengths[s] tokens with them,
// token p in slot p % block_tokens of block tables[s][p / block_tokens]. The
// arrays are device memory, so kernels bound what they read: a start to [0,
// tokens] and from below by its predecessor, a length from below by 0; a
// position from capacity on and a block id outside the pool have no block.
struct BatchView {
  const int32_t* tables = nullptr;
  const int32_t* lengths = nullptr;
  const int32_t* starts = nullptr;
  int64_t table_stride = 0;
  int32_t table_width = 0;
  int32_t sequences = 0;
  int32_t tokens = 0;
  int32_t block_tokens = 0;
  int32_t capacity = 0;    // table_width * block_tokens
  int32_t num_blocks = 0;  // blocks of the pool
};

}  // namespace kvx

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

namespace kvx {

using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

// Element type tags: `Scalar` in memory, `V8` as an operand of the matrix
// instructions (8 values along the contraction).
struct Bf16 {
  using Scalar = __bf16;
  using V2 = bf16x2;
  using V8 = bf16x8;
};
struct F16 {
  using Scalar = _Float16;
  using V2 = f16x2;
  using V8 = f16x8;
};
struct F32 {
  using Scalar = float;
};

// Two values rounded to nearest even, in one word.
template <class E>
__device__ __forceinline__ uint32_t Pack2(float a, float b) {
  const f32x2 f = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, typename E::V2));
}

template <class E>
__device__ __forceinline__ f32x2 Unpack2(uint32_t w) {
  return __builtin_convertvector(__builtin_bit_cast(typename E::V2, w), f32x2);
}

// The two e4m3 values in half `hi` of w, times a power of two: exact in either
// 16-bit type for powers from 2^-15 to 2^7.
template <class E>
__device__ __forceinline__ uint32_t FromE4m3(uint32_t w, bool hi, float power) {
  if constexpr (std::is_same_v<E, F16>) {
    return hi ? __builtin_bit_cast(uint32_t,
                                   __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, true))
              : __builtin_bit_cast(uint32_t,
                                   __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, false));
  } else {
    return hi ? __builtin_bit_cast(uint32_t,
                                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, true))
              : __builtin_bit_cast(uint32_t,
                                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, false));
  }
}

// Eight e2m1 values times a scale, given as the bits of a float whose exponent is
// the e8m0 code (255 makes NaN of all): exact in bf16, and in fp16 for scales of
// 2^-23 to 2^13.
template <class E>
__device__ __forceinline__ u32x4 FromFp4(uint32_t w, uint32_t scale) {
  const float f = __builtin_bit_cast(float, scale);
  if constexpr (std::is_same_v<E, F16>) {
    return u32x4{
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 3))};
  } else {
    return u32x4{
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3))};
  }
}

// The scale of an e8m0 code for FromFp4. In fp16 a scale above 2^13, whose values
// could leave the type's range, counts as 2^13; append_kv stores none from fp16.
constexpr uint32_t kFp4MostF16 = 127 + 13, kFp4Most = 127 + 125, kFp4Least = 127 - 125;
template <class E>
__device__ __forceinline__ uint32_t Fp4Scale(uint32_t code) {
  if constexpr (std::is_same_v<E, F16>) {
    code = code > kFp4MostF16 && code != 255 ? kFp4MostF16 : code;
  }
  return code << 23;
}

struct SequenceSpan {
  int32_t first;   // its first new token
  int32_t count;   // its new tokens
  int32_t length;  // its tokens with them
};

__device__ __forceinline__ SequenceSpan LoadSequence(const BatchView& b, int32_t s) {
  SequenceSpan r;
  if (b.starts != nullptr) {
    r.first = min(max(b.starts[s], 0), b.tokens);
    r.count = min(max(b.starts[s + 1], r.first), b.tokens) - r.first;
  } else {
    r.first = s;
    r.count = 1;
  }
  r.length = max(b.lengths[s], 0);
  return r;
}

// cos and sin of position * inv_freq. The product and its turns are taken in
// two 64-bit words (each error term exact by a fused multiply-add) and reduced
// there, so any position up to 2^53 keeps its angle; cos and sin get the nearest
// 32-bit one, and what that leaves, up to 2^-26 turns, turns their result.
__device__ __forceinline__ f32x2 Turn(int64_t position, float inv_freq) {
// A product fused into the difference would bring its error term in twice.
#pragma clang fp contract(off)
  constexpr double kTurn = 0x1.45f306dc9c883p-3;        // 1 / (2 pi), and
  constexpr double kTurnRest = -0x1.6b01ec5417056p-57;  // what it leaves
  const double p = static_cast<double>(position), f = static_cast<double>(inv_freq);
  const double angle = p * f, angle_rest = fma(p, f, -angle);
  const double turns = angle * kTurn;
  const double rest = fma(angle, kTurn, -turns) + angle * kTurnRest + angle_rest * kTurn;
  const double within = (turns - rint(turns)) + rest;
  const float part = static_cast<float>(within);
  const float left = static_cast<float>(within - part) * 6.2831853f;
  float s, c;
  sincospif(2.0f * part, &s, &c);
  return f32x2{__builtin_fmaf(-left, s, c), __builtin_fmaf(left, c, s)};
}

}  // namespace kvx
#endif  // __HIPCC__

#endif  // KVX_KERNELS_KV_ELEMENT_H_
