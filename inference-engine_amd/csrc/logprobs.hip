// Log probabilities of given tokens, entropy and the most likely alternatives of rows of
// logits (C-ABI in iekv_ops.h).
//
// For a row x with m = max x, s = sum e^(x - m), w = sum e^(x - m) (x - m):
//   logprob(t) = (x_t - m) - ln s,  entropy = -sum p ln p = ln s - w / s.
// (x_t - (m + ln s) would lose ln s next to a type's lowest value, a usual mask.)
// The alternatives are ordered by a 64-bit key: the logit as a whole number that orders as
// the values do (NaN above all), then the index, smaller first, so that no two are alike.
#include "ops_common.h"

#include <cmath>

using namespace iekv_ops;

namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;

// A logit as an unsigned number of the same order; NaN is the largest. Zeros of both signs
// are equal.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  if (x != x) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  return static_cast<uint64_t>(ordered(x)) << 32 | (0xffffffffu - index);
}

__device__ __forceinline__ uint64_t wave_top(uint64_t k) {
  for (int s = 32; s; s >>= 1) {
    const uint64_t other = __shfl_xor(static_cast<unsigned long long>(k), s);
    k = other > k ? other : k;
  }
  return k;
}

// Sums of a part of a row: m, s and w above.
struct Sums {
  float m, s, w;
};

__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = a.m > b.m || a.m != a.m ? a.m : b.m;      // a NaN stays
  const float base = m == -INFINITY ? 0.f : m;
  const float da = a.m - base, db = b.m - base;
  const float ea = expf(da), eb = expf(db);
  // e^(x - m) (x - m) = e^(m_a - m) (e^(x - m_a) (x - m_a) + e^(x - m_a) (m_a - m))
  const float wa = ea > 0.f ? ea * fmaf(a.s, da, a.w) : 0.f;
  const float wb = eb > 0.f ? eb * fmaf(b.s, db, b.w) : 0.f;
  return {m, fmaf(a.s, ea, b.s * eb), wa + wb};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void score_rows(const T* logits, int64_t stride,
                                                       int32_t vocab, const int64_t* tokens,
                                                       int32_t top, float* logprobs,
                                                       float* entropy, float* top_logprobs,
                                                       int64_t* top_ids) {
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  __shared__ Sums sums[kThreads];
  __shared__ uint64_t best[kThreads / kWave];
  Sums mine{-INFINITY, 0.f, 0.f};
  for (int32_t i = threadIdx.x; i < vocab; i += kThreads)
    mine = join(mine, {to_float(x[i]), 1.f, 0.f});
  sums[threadIdx.x] = mine;
  __syncthreads();
  for (int n = kThreads / 2; n; n >>= 1) {
    if (threadIdx.x < n) sums[threadIdx.x] = join(sums[threadIdx.x], sums[threadIdx.x + n]);
    __syncthreads();
  }
  const Sums all = sums[0];
  const float log_s = logf(all.s);
  if (threadIdx.x == 0) {
    const int64_t t = tokens[row];
    const bool none = all.m == -INFINITY;
    logprobs[row] = t < 0 || t >= vocab ? NAN : none ? -INFINITY : (to_float(x[t]) - all.m) - log_s;
    entropy[row] = none ? 0.f : log_s - all.w / all.s;
  }
  uint64_t below = ~uint64_t(0);
  for (int32_t k = 0; k < top; ++k) {
    uint64_t key = 0;
    for (int32_t i = threadIdx.x; i < vocab; i += kThreads) {
      const uint64_t c = key_of(to_float(x[i]), i);
      key = c < below && c > key ? c : key;
    }
    key = wave_top(key);
    if (threadIdx.x % kWave == 0) best[threadIdx.x / kWave] = key;
    __syncthreads();
    for (int w = 0; w < kThreads / kWave; ++w) key = best[w] > key ? best[w] : key;
    below = key;
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t id = 0xffffffffu - static_cast<uint32_t>(key);
      const float v = to_float(x[id]);
      top_logprobs[row * top + k] = all.m == -INFINITY ? -INFINITY : (v - all.m) - log_s;
      top_ids[row * top + k] = id;
    }
  }
}

template <typename T>
int launch(const void* logits, int64_t stride, int64_t n_rows, int64_t vocab,
           const int64_t* tokens, int32_t top, float* logprobs, float* entropy,
           float* top_logprobs, int64_t* top_ids, hipStream_t stream) {
  hipLaunchKernelGGL((score_rows<T>), dim3(n_rows), dim3(kThreads), 0, stream,
                     static_cast<const T*>(logits), stride, static_cast<int32_t>(vocab), tokens,
                     top, logprobs, entropy, top_logprobs, top_ids);
  IEKV_OPS_HIP(hipGetLastError());
  return IEKV_OK;
}

}  // namespace

extern "C" {

int64_t iekv_logprobs_workspace(int32_t, int64_t, int64_t, int32_t) { return 0; }

int iekv_logprobs(int32_t type, const void* logits, int64_t row_stride, int64_t n_rows,
                  int64_t vocab, const int64_t* tokens, int32_t top, float* logprobs,
                  float* entropy, float* top_logprobs, int64_t* top_ids, void* workspace,
                  int64_t workspace_bytes, hipStream_t stream) {
  if (n_rows < 0 || n_rows > INT32_MAX)
    return set_error(IEKV_ERR_INVALID, "n_rows %lld out of range", static_cast<long long>(n_rows));
  if (vocab < 1 || vocab > INT32_MAX)
    return set_error(IEKV_ERR_INVALID, "vocab %lld out of range", static_cast<long long>(vocab));
  if (top < 0 || top > IEKV_LOGPROBS_MAX_TOP || top > vocab)
    return set_error(IEKV_ERR_INVALID, "top %d out of range for a vocabulary of %lld (at most %d)",
                     top, static_cast<long long>(vocab), IEKV_LOGPROBS_MAX_TOP);
  if (row_stride < 0)
    return set_error(IEKV_ERR_INVALID, "row_stride %lld is negative",
                     static_cast<long long>(row_stride));
  if (type != IEKV_TYPE_F32 && type != IEKV_TYPE_F16 && type != IEKV_TYPE_BF16)
    return set_error(IEKV_ERR_INVALID, "logits of type %d", type);
  if (!n_rows) return IEKV_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top && (!top_logprobs || !top_ids)))
    return set_error(IEKV_ERR_INVALID, "null argument");
  const int64_t need = iekv_logprobs_workspace(type, n_rows, vocab, top);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(IEKV_ERR_CAPACITY, "workspace of %lld bytes, %lld are needed",
                     static_cast<long long>(workspace ? workspace_bytes : 0),
                     static_cast<long long>(need));
  switch (type) {
    case IEKV_TYPE_F32:
      return launch<float>(logits, row_stride, n_rows, vocab, tokens, top, logprobs, entropy,
                           top_logprobs, top_ids, stream);
    case IEKV_TYPE_F16:
      return launch<_Float16>(logits, row_stride, n_rows, vocab, tokens, top, logprobs, entropy,
                              top_logprobs, top_ids, stream);
    default:
      return launch<Bf16>(logits, row_stride, n_rows, vocab, tokens, top, logprobs, entropy,
                          top_logprobs, top_ids, stream);
  }
}

}  // extern "C"
