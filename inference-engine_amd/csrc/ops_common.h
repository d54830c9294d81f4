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

// A dispatch counts its work-items in 32 bits: workgroups of 256 threads that one launch may
// have. What needs more is launched in several.
constexpr int64_t kMaxGrid = static_cast<int64_t>(UINT32_MAX) / 256;

// Makes a device current for a call that launches on it, and the caller's again after.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    error_ = hipGetDevice(&before_);
    if (error_ == hipSuccess && before_ != device) {
      error_ = hipSetDevice(device);
      switched_ = error_ == hipSuccess;
    }
    if (error_ != hipSuccess) (void)hipGetLastError();
  }
  ~DeviceGuard() {
    if (switched_) (void)hipSetDevice(before_);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  hipError_t error() const { return error_; }

 private:
  int before_ = 0;
  hipError_t error_;
  bool switched_ = false;
};

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

// --- lanes of a wave ------------------------------------------------------------------------
//
// By the vector unit's own lane moves: an LDS shuffle takes some 100 cycles, and there are six
// to a reduction and 21 to a sort, each waiting for the one before it.

template <int CTRL>
__device__ __forceinline__ uint32_t lane_move(uint32_t x) {
  return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false);
}
constexpr int kQuad1 = 0xb1, kQuad2 = 0x4e, kQuad3 = 0x1b;   // lane ^ 1, ^ 2, ^ 3
constexpr int kMirror8 = 0x141, kMirror16 = 0x140;           // lane ^ 7, ^ 15

// The word of lane ^ M.
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  if constexpr (M == 1) return lane_move<kQuad1>(x);
  if constexpr (M == 2) return lane_move<kQuad2>(x);
  if constexpr (M == 4) return lane_move<kQuad3>(lane_move<kMirror8>(x));
  if constexpr (M == 8) return lane_move<kMirror8>(lane_move<kMirror16>(x));
  // Swaps rows of 16 (32) lanes of two operands: the even rows of the first and of the second.
  // (Their halves are named: a bit cast of a vector's element takes its first.)
  if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t even = r[0], odd = r[1];
    return threadIdx.x & 16 ? even : odd;
  }
  if constexpr (M == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const uint32_t even = r[0], odd = r[1];
    return threadIdx.x & 32 ? even : odd;
  }
}
template <int M>
__device__ __forceinline__ float lane_xor(float x) {
  return __builtin_bit_cast(float, lane_xor<M>(__builtin_bit_cast(uint32_t, x)));
}
template <int M>
__device__ __forceinline__ uint64_t lane_xor(uint64_t x) {
  return static_cast<uint64_t>(lane_xor<M>(static_cast<uint32_t>(x >> 32))) << 32 |
         lane_xor<M>(static_cast<uint32_t>(x));
}

// op over the lanes, the same in each of them. `op` takes its operands in either order.
template <typename V, typename Op>
__device__ __forceinline__ V wave_all(V x, Op op) {
  x = op(x, lane_xor<1>(x));
  x = op(x, lane_xor<2>(x));
  x = op(x, lane_xor<4>(x));
  x = op(x, lane_xor<8>(x));
  x = op(x, lane_xor<16>(x));
  return op(x, lane_xor<32>(x));
}
__device__ __forceinline__ float wave_max(float x) {
  return wave_all(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
  return wave_all(x, [](float a, float b) { return a + b; });
}

}  // namespace iekv_ops

#endif  // IEKV_OPS_COMMON_H_
