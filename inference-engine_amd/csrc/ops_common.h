// What the operator sources (attention.hip, logprobs.hip) share: the thread's error message,
// the HIP status check and the element types.
#ifndef IEKV_OPS_COMMON_H_
#define IEKV_OPS_COMMON_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "iekv_ops.h"

namespace iekv_ops {

// Records the message iekv_ops_last_error returns and gives `code` back.
int set_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

#define IEKV_OPS_HIP(expr)                                                                 \
  do {                                                                                     \
    hipError_t err_ = (expr);                                                              \
    if (err_ != hipSuccess) {                                                              \
      (void)hipGetLastError();                                                             \
      return iekv_ops::set_error(IEKV_ERR_HIP, "%s: %s", #expr, hipGetErrorString(err_));  \
    }                                                                                      \
  } while (0)

// Element types as they lie in memory.
struct E4m3 {
  uint8_t bits;
};
struct Bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(_Float16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_float(Bf16 x) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(x.bits) << 16);
}
__device__ __forceinline__ float to_float(E4m3 x) {
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(x.bits), 0);
}

// Rounded to nearest even.
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ _Float16 from_float<_Float16>(float x) {
  return static_cast<_Float16>(x);
}
template <>
__device__ __forceinline__ Bf16 from_float<Bf16>(float x) {
  return {__builtin_bit_cast(uint16_t, static_cast<__bf16>(x))};
}

}  // namespace iekv_ops

#endif  // IEKV_OPS_COMMON_H_
