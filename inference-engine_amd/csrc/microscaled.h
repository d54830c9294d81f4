// Microscaled cache elements, as microscaled.hip writes them and attention reads them.
//
// 32 dimensions of a head (the last group of a head may have fewer) share a power of two 2^e;
// an element x is held as c = x / 2^e rounded to nearest even in 8 bits (e4m3, integers) or 4
// (e2m1). e is the smallest from kLeastExponent on with which the group's largest magnitude is
// within the type's: nothing saturates, and x / 2^e is exact in 32 bits, so that rounding to
// the type is the only one. A head's record is its elements' bytes and then one word, byte g of
// it group g's e + 127. A group that held a NaN or an infinity has the byte 255 and is NaN.
//
// c 2^e is exact in float32 and, e4m3's and e2m1's few bits and 8-bit integers alike, in
// bfloat16; gfx950 converts the two floating types with their scale in one operation, two
// elements at a time.
#ifndef IEKV_MICROSCALED_H_
#define IEKV_MICROSCALED_H_

#include <type_traits>

#include "ops_common.h"

namespace iekv_ops {

struct Mxfp8 {
  uint8_t bits;   // e4m3
};
struct Mxint8 {
  int8_t value;   // -127 .. 127
};
struct Mxfp4 {
  uint8_t pair;   // e2m1: the even dimension in the low half
};

template <typename C>
constexpr bool kScaled =
    std::is_same_v<C, Mxfp8> || std::is_same_v<C, Mxint8> || std::is_same_v<C, Mxfp4>;
template <typename C>
constexpr int kBits = std::is_same_v<C, Mxfp4> ? 4 : 8 * int(sizeof(C));

constexpr int kGroup = 32;
constexpr int kScaleBytes = 4;          // a byte for each group of the largest head
constexpr int kLeastExponent = -100;    // far from where 2^e or an element is no normal number
static_assert(IEKV_ATTENTION_MAX_DIM <= kGroup * kScaleBytes);

// Bytes of `d` dimensions of a head in the cache (d a multiple of 8), without and with its scales.
template <typename C>
__host__ __device__ constexpr int32_t code_bytes(int32_t d) {
  return d * kBits<C> / 8;
}
template <typename C>
__host__ __device__ constexpr int32_t head_bytes(int32_t d) {
  return code_bytes<C>(d) + (kScaled<C> ? kScaleBytes : 0);
}

// 2^e of a record's word: `shift` is eight times the group. 255 gives infinity, which is NaN to
// the conversions and times an integer's zero.
__device__ __forceinline__ float scale_of(uint32_t scales, int32_t shift) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ubfe(scales, shift, 8) << 23);
}

template <int N>
struct Words {
  uint32_t w[N];
};

// BYTES from any address (caches and queries may begin at any element).
template <int BYTES>
__device__ __forceinline__ Words<(BYTES + 3) / 4> load_bytes(const void* p) {
  Words<(BYTES + 3) / 4> r;
  r.w[(BYTES - 1) / 4] = 0;
  __builtin_memcpy(&r, p, BYTES);
  return r;
}

// The same of a stream that is read once.
template <int BYTES>
__device__ __forceinline__ Words<(BYTES + 3) / 4> stream_bytes(const void* p) {
  // (Vectors of three are loaded as four.)
  if constexpr (BYTES % 4 || BYTES == 12) {
    return load_bytes<BYTES>(p);
  } else {
    typedef uint32_t Vec __attribute__((ext_vector_type(BYTES / 4), aligned(1)));
    return __builtin_bit_cast(Words<BYTES / 4>,
                              __builtin_nontemporal_load(static_cast<const Vec*>(p)));
  }
}

// BYTES (a multiple of 4) to any address, of a stream that nothing here reads again.
template <int BYTES>
__device__ __forceinline__ void stream_out(void* p, const Words<BYTES / 4>& x) {
  typedef uint32_t Vec __attribute__((ext_vector_type(BYTES / 4), aligned(1)));
  __builtin_nontemporal_store(__builtin_bit_cast(Vec, x), static_cast<Vec*>(p));
}

// Two elements of the compute type in a word, rounded to nearest even.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<Bf16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
}
template <>
__device__ __forceinline__ uint32_t pack2<_Float16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}

// Elements 2 `i` and 2 `i` + 1 of `x` times `scale`, as T rounded to nearest even: two floats, or
// a word of two. `i` is known when compiled.
template <typename T, typename C>
__device__ __forceinline__ Words<2 * sizeof(T) / 4> pair_of(const uint32_t* x, int i,
                                                            float scale) {
  using R = Words<2 * sizeof(T) / 4>;
  if constexpr (std::is_same_v<C, Mxint8>) {
    const uint32_t w = x[i / 2] >> i % 2 * 16;
    const float a = static_cast<float>(static_cast<int8_t>(w)) * scale;
    const float b = static_cast<float>(static_cast<int8_t>(w >> 8)) * scale;
    if constexpr (sizeof(T) == 4)
      return R{{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)}};
    else
      return R{{pack2<T>(a, b)}};
  } else if constexpr (std::is_same_v<C, Mxfp8>) {
    const uint32_t w = x[i / 2];
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(R, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false));
    else if constexpr (std::is_same_v<T, Bf16>)
      return __builtin_bit_cast(R, i % 2
                                       ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)
                                       : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
    else
      return __builtin_bit_cast(R, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
  } else {
    static_assert(std::is_same_v<C, Mxfp4>);
    const uint32_t w = x[i / 4];
    const auto at = [&](auto byte) {
      constexpr int B = decltype(byte)::value;
      if constexpr (sizeof(T) == 4)
        return __builtin_bit_cast(R, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, B));
      else if constexpr (std::is_same_v<T, Bf16>)
        return __builtin_bit_cast(R, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
      else
        return __builtin_bit_cast(R, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, B));
    };
    switch (i % 4) {
      case 0: return at(std::integral_constant<int, 0>{});
      case 1: return at(std::integral_constant<int, 1>{});
      case 2: return at(std::integral_constant<int, 2>{});
      default: return at(std::integral_constant<int, 3>{});
    }
  }
}

// N elements (2 or more) of a group as T.
template <typename T, typename C, int N>
__device__ __forceinline__ Words<N * sizeof(T) / 4> scaled(
    const Words<(N * kBits<C> / 8 + 3) / 4>& x, float scale) {
  Words<N * sizeof(T) / 4> r;
  constexpr int each = 2 * sizeof(T) / 4;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const auto p = pair_of<T, C>(x.w, i, scale);
#pragma unroll
    for (int e = 0; e < each; ++e) r.w[i * each + e] = p.w[e];
  }
  return r;
}

}  // namespace iekv_ops

#endif  // IEKV_MICROSCALED_H_
