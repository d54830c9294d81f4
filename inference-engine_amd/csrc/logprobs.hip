// Log probabilities of given tokens, entropy and the most likely alternatives of rows of
// logits (C-ABI in iekv_ops.h).
//
// For a row x with m = max x, s = sum e^(x - m), w = sum e^(x - m) (x - m):
//   logprob(t) = (x_t - m) - ln s,  entropy = -sum p ln p = ln s - w / s.
// (x_t - (m + ln s) would lose ln s next to a type's lowest value, a usual mask.)
// The alternatives are ordered by a 64-bit key: the logit as a whole number that orders as
// the values do (NaN above all), then the index, smaller first, so that no two are alike.
//
// The logits are read once: a row is cut into parts of at most 8,192, each held whole in the
// registers of a workgroup, which leaves m, s, w and its part's alternatives to a second
// launch that joins a row's parts in their order. Rows of one part are done in one launch.
// How a row is cut depends on the vocabulary alone, so a row's result does not depend on the
// rows beside it. Bound by the stream of logits where there are many (2,001 rows of 100,003 in
// fp32: 117 us, 6.8 TB/s), by the two launches otherwise (64 rows of 128,000 in bf16 with 20
// alternatives: 12 us for the parts, whose sums and alternatives follow one another, 7 to join).
#include "ops_common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace iekv_ops;

namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr int kWaves = kThreads / kWave;
constexpr int kCandidates = 512;   // of a row's parts that are ranked at once
constexpr int kEach = 128;         // and of a wave's share of a part
constexpr int kOneByOne = 5;       // largest lanes that are found by so many reductions
constexpr int kSmall = 8, kLarge = 32;  // logits a thread holds
constexpr int64_t kCacheBytes = 256 << 20;  // of the last-level cache

// A logit as an unsigned number of the same order; NaN is the largest. Zeros of both signs
// are equal.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  if (x != x) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Keys of logits are above 0.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  return static_cast<uint64_t>(ordered(x)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) {
  return 0xffffffffu - static_cast<uint32_t>(key);
}

__device__ __forceinline__ uint64_t wave_top(uint64_t k) {
  return wave_all(k, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}

// The lanes' values in falling order (Batcher's bitonic network: runs of SIZE, compared at
// distance STEP).
template <int SIZE = 2, int STEP = 1>
__device__ __forceinline__ float wave_sorted(float x) {
  const float other = lane_xor<STEP>(x);
  const bool first = !(threadIdx.x & STEP), falling = !(threadIdx.x & SIZE) || SIZE == kWave;
  x = first == falling ? fmaxf(x, other) : fminf(x, other);
  if constexpr (STEP > 1) return wave_sorted<SIZE, STEP / 2>(x);
  else if constexpr (SIZE < kWave) return wave_sorted<SIZE * 2, SIZE>(x);
  else return x;
}

// Sums of a part of a row: m, s and w above.
struct Sums {
  float m, s, w;
};

// e^d for d <= 0, flushed to zero where e^d is no normal number.
__device__ __forceinline__ float exponential(float d) {
  return __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
}

// The part's sums as they count next to a maximum m of all parts.
__device__ __forceinline__ Sums moved(Sums a, float m) {
  const float d = a.m == -INFINITY ? 0.f : a.m - m;
  const float e = exponential(d);
  // e^(x - m) (x - m) = e^(a.m - m) (e^(x - a.m) (x - a.m) + e^(x - a.m) (a.m - m))
  return {m, a.s * e, e > 0.f ? e * fmaf(a.s, d, a.w) : 0.f};
}

// What a row's results are written from.
struct Scores {
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  int32_t vocab, top;
};

// A row of nothing but -inf has no sum.
__device__ __forceinline__ float logprob_of(float x, const Sums& a, float log_s) {
  return a.s == 0.f ? -INFINITY : (x - a.m) - log_s;
}

// The logit of the row's token, NaN for one outside the vocabulary. Read before the sums, so
// that nothing waits for it.
template <typename T>
__device__ __forceinline__ float given_of(const Scores& out, const T* x, int64_t row) {
  const int64_t t = out.tokens[row];
  return t < 0 || t >= out.vocab ? NAN : to_float(x[t]);
}

__device__ __forceinline__ void write_row(const Scores& out, float given, int64_t row,
                                          const Sums& a, float log_s) {
  out.logprobs[row] = given != given ? NAN : logprob_of(given, a, log_s);
  out.entropy[row] = a.s == 0.f ? 0.f : log_s - a.w / a.s;
}

__device__ __forceinline__ void write_top(const Scores& out, int64_t row, int32_t rank,
                                          uint64_t key, const Sums& a, float log_s) {
  out.top_logprobs[row * out.top + rank] = logprob_of(logit_of(key), a, log_s);
  out.top_ids[row * out.top + rank] = index_of(key);
}

// Parts of rows in the workspace: their sums, then the keys of their alternatives.
struct Parts {
  Sums* sums;        // [rows][parts]
  uint64_t* keys;    // [rows][parts][top], falling; 0 past the part's logits
  int32_t parts, size;
};

// How many keys of a list are larger. The list goes on for `kPad` zeros: eight keys are read
// at a time, or each would be waited for.
constexpr int kPad = 8;
__device__ __forceinline__ int32_t rank_of(uint64_t key, const uint64_t* list, int32_t count) {
  int32_t rank = 0;
  for (int32_t j = 0; j < count; j += kPad)
#pragma unroll
    for (int i = 0; i < kPad; ++i) rank += list[j + i] > key;
  return rank;
}

// One part of a row by one workgroup.
//
// The alternatives: a lower bound of the part's k-th largest logit is found from the lanes'
// own largest ones. Each wave sorts its 64: if every wave has ceil(k / 4) lanes of at least
// b, or one wave has k, there are k logits of at least b. What reaches the bound, a few more
// than k as a rule, is put on the waves' lists in LDS and ranked by counting the larger keys.
// Where more reach it than a list holds (rows of equal logits, all but barred rows) or the
// part holds a NaN, the largest key is taken k times instead.
//
// STREAM reads past the caches: logits that no cache holds come 13% faster so (2,001 rows of
// 100,003 in fp32 117 us against 132), those that one may hold 10% slower (512 rows of 128,000
// in bf16 57 us against 51).
template <typename T, int HELD, bool STREAM>
__global__ __launch_bounds__(kThreads) void score_part(const T* logits, int64_t stride, Scores out,
                                                       Parts parts) {
  constexpr int VEC = 16 / sizeof(T), LOADS = HELD / VEC;
  const int64_t row = blockIdx.x / parts.parts;
  const int32_t part = blockIdx.x % parts.parts, tid = threadIdx.x;
  const int wave = tid / kWave, lane = tid % kWave;
  const int32_t first = part * parts.size;
  const int32_t n = parts.size < out.vocab - first ? parts.size : out.vocab - first;
  const T* x = logits + row * stride;
  __shared__ float most[kWaves];
  __shared__ float2 sums[kWaves], bounds[kWaves];
  __shared__ uint64_t lists[kWaves][kEach + kPad];
  __shared__ int32_t listed[kWaves];

  // Logit v (of this thread's `HELD`) is number (v / VEC * kThreads + tid) * VEC + v % VEC.
  float held[HELD];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int32_t at = (i * kThreads + tid) * VEC;
    T e[VEC];
    if (at + VEC <= n) {
      typedef uint32_t Chunk __attribute__((ext_vector_type(4), aligned(2)));
      const Chunk* from = reinterpret_cast<const Chunk*>(x + first + at);
      const Chunk chunk = STREAM ? __builtin_nontemporal_load(from) : *from;
      __builtin_memcpy(e, &chunk, sizeof(e));
#pragma unroll
      for (int j = 0; j < VEC; ++j) held[i * VEC + j] = to_float(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        held[i * VEC + j] = at + j < n ? to_float(x[first + at + j]) : -INFINITY;
    }
  }
  const bool whole = parts.parts == 1;
  const float given = whole ? given_of(out, x, row) : 0.f;
  const auto index = [&](int v) { return (v / VEC * kThreads + tid) * VEC + v % VEC; };

  constexpr int GROUP = 8;
  float of_group[HELD / GROUP], mine = -INFINITY;
#pragma unroll
  for (int g = 0; g < HELD / GROUP; ++g) {
    of_group[g] = -INFINITY;
#pragma unroll
    for (int v = 0; v < GROUP; ++v) of_group[g] = fmaxf(of_group[g], held[g * GROUP + v]);
    mine = fmaxf(mine, of_group[g]);
  }
  const float of_wave = wave_max(mine);
  if (lane == 0) most[wave] = of_wave;
  __syncthreads();
  Sums all;
  all.m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  const float base = all.m == -INFINITY ? 0.f : all.m;
  float s = 0.f, w = 0.f;
#pragma unroll
  for (int v = 0; v < HELD; ++v) {
    const float d = held[v] - base, e = exponential(d);
    s += e;
    // e is 0 from -104 on, and 0 * -inf would be NaN.
    w = fmaf(e, __builtin_amdgcn_fmed3f(d, -200.f, 0.f), w);
  }
  s = wave_sum(s);
  w = wave_sum(w);
  if (lane == 0) sums[wave] = {s, w};
  const int32_t top = out.top;
  if (top) {
    // The wave's ceil(k / 4)-th largest lane, and where some wave has few lanes with logits its
    // k-th. Few are found one by one, more by a sort.
    const int32_t share = (top + kWaves - 1) / kWaves;
    float each = of_wave, alone = top == 1 ? of_wave : -INFINITY;
    if (top > 1 && (n < kThreads * VEC || share > kOneByOne)) {
      const float sorted = wave_sorted(mine);
      each = __shfl(sorted, share - 1);
      alone = __shfl(sorted, top - 1);
    } else {
      float left = mine;
      for (int32_t i = 1; i < share; ++i) {
        const uint64_t who = __ballot(left == each);
        if (lane == __ffsll(static_cast<unsigned long long>(who)) - 1) left = -INFINITY;
        each = wave_max(left);
      }
    }
    if (lane == 0) bounds[wave] = {each, alone};
  }
  __syncthreads();
  all.s = (sums[0].x + sums[1].x) + (sums[2].x + sums[3].x);
  all.w = (sums[0].y + sums[1].y) + (sums[2].y + sums[3].y);
  const float log_s = logf(all.s);
  if (tid == 0) {
    if (whole)
      write_row(out, given, row, all, log_s);
    else
      parts.sums[blockIdx.x] = all;
  }
  if (!top) return;

  const auto put = [&](int32_t rank, uint64_t key) {
    if (whole)
      write_top(out, row, rank, key, all, log_s);
    else
      parts.keys[static_cast<int64_t>(blockIdx.x) * top + rank] = key;
  };
  const float bound =
      fmaxf(fminf(fminf(bounds[0].x, bounds[1].x), fminf(bounds[2].x, bounds[3].x)),
            fmaxf(fmaxf(bounds[0].y, bounds[1].y), fmaxf(bounds[2].y, bounds[3].y)));
  // Each wave lists its own. Only where nothing bounds them could what fills the part up, -inf,
  // be among them.
  uint64_t* list = lists[wave];
  int32_t own = 0;
  const auto collect = [&](auto unbounded) {
#pragma unroll
    for (int g = 0; g < HELD / GROUP; ++g) {
      if (!__any(of_group[g] >= bound)) continue;
#pragma unroll
      for (int v = g * GROUP; v < (g + 1) * GROUP; ++v) {
        const bool in = held[v] >= bound && (!unbounded || index(v) < n);
        const uint64_t who = __ballot(in);
        if (!who) continue;
        const int32_t at = own + __popcll(who & ((uint64_t(1) << lane) - 1));
        if (in && at < kEach) list[at] = key_of(held[v], first + index(v));
        own += __popcll(who);
      }
    }
  };
  if (bound == -INFINITY)
    collect(std::true_type{});
  else if (__any(mine >= bound))
    collect(std::false_type{});
  if (lane < kPad && own <= kEach) list[own + lane] = 0;
  if (lane == 0) listed[wave] = own;
  __syncthreads();
  int32_t count = 0;
  bool fits = all.s == all.s;
  for (int w = 0; w < kWaves; ++w) {
    count += listed[w];
    fits = fits && listed[w] <= kEach;
  }
  if (fits) {
    for (int32_t i = lane; i < own; i += kWave) {
      const uint64_t key = list[i];
      int32_t rank = 0;
      for (int w = 0; w < kWaves; ++w) rank += rank_of(key, lists[w], listed[w]);
      if (rank < top) put(rank, key);
    }
    // A part of fewer logits than alternatives (of a row of several parts).
    for (int32_t rank = count + tid; rank < top; rank += kThreads) put(rank, 0);
    return;
  }
  uint64_t below = ~uint64_t(0);
  for (int32_t rank = 0; rank < top; ++rank) {
    uint64_t key = 0;
#pragma unroll
    for (int v = 0; v < HELD; ++v) {
      const uint64_t k = index(v) < n ? key_of(held[v], first + index(v)) : 0;
      key = k < below && k > key ? k : key;
    }
    key = wave_top(key);
    __syncthreads();
    if (lane == 0) lists[0][wave] = key;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) key = lists[0][i] > key ? lists[0][i] : key;
    below = key;
    if (tid == 0) put(rank, key);
  }
}

// A row's parts, by one wave. Bounds of the row's k-th largest key, as above: any part's
// k-th, and the least of the parts' ceil(k / parts)-th.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_rows(const T* logits, int64_t stride,
                                                      int64_t n_rows, Scores out, Parts parts) {
  __shared__ uint64_t lists[kWaves][kCandidates + kPad];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  if (row >= n_rows) return;
  const Sums* sums = parts.sums + row * parts.parts;
  const int32_t n = parts.parts, top = out.top;
  const uint64_t* keys = parts.keys + row * n * top;
  const float given = given_of(out, logits + row * stride, row);
  uint64_t any = 0, least = ~uint64_t(0);
  const int32_t each = (top + n - 1) / n;
  float m = -INFINITY;
  for (int32_t p = lane; p < n; p += kWave) {
    m = fmaxf(m, sums[p].m);
    if (top) {
      const uint64_t last = keys[static_cast<int64_t>(p) * top + top - 1];
      const uint64_t share = keys[static_cast<int64_t>(p) * top + each - 1];
      any = last > any ? last : any;
      least = share < least ? share : least;
    }
  }
  Sums all{wave_max(m), 0.f, 0.f};
  for (int32_t p = lane; p < n; p += kWave) {
    const Sums a = moved(sums[p], all.m);
    all.s += a.s;
    all.w += a.w;
  }
  all.s = wave_sum(all.s);
  all.w = wave_sum(all.w);
  const float log_s = logf(all.s);
  if (lane == 0) write_row(out, given, row, all, log_s);
  if (!top) return;

  any = wave_top(any);
  least = ~wave_top(~least);
  const uint64_t bound = any > least ? any : least;
  uint64_t* list = lists[wave];
  int32_t count = 0;
  const int32_t total = n * top;
  constexpr int kAtOnce = 8;                  // loads on their way
  for (int32_t i0 = 0; i0 < total && count <= kCandidates; i0 += kAtOnce * kWave) {
    uint64_t key[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int32_t at = i0 + i * kWave + lane;
      key[i] = keys[at < total ? at : total - 1];
      if (at >= total) key[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const bool in = key[i] && key[i] >= bound;
      const uint64_t who = __ballot(in);
      const int32_t at = count + __popcll(who & ((uint64_t(1) << lane) - 1));
      if (in && at < kCandidates) list[at] = key[i];
      count += __popcll(who);
    }
  }
  if (lane < kPad && count <= kCandidates) list[count + lane] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (count <= kCandidates) {
    for (int32_t i = lane; i < count; i += kWave) {
      const uint64_t key = list[i];
      const int32_t rank = rank_of(key, list, count);
      if (rank < top) write_top(out, row, rank, key, all, log_s);
    }
    return;
  }
  uint64_t below = ~uint64_t(0);
  for (int32_t rank = 0; rank < top; ++rank) {
    uint64_t key = 0;
    for (int32_t i = lane; i < total; i += kWave)
      key = keys[i] < below && keys[i] > key ? keys[i] : key;
    below = wave_top(key);
    if (lane == 0) write_top(out, row, rank, below, all, log_s);
  }
}

// How rows are cut: parts of equal size (a multiple of 8) that a workgroup can hold.
struct Cut {
  int32_t held, parts, size;
};

Cut cut_of(int64_t vocab) {
  const int held = vocab <= kSmall * kThreads ? kSmall : kLarge;
  const int64_t most = int64_t(held) * kThreads, parts = (vocab + most - 1) / most;
  return {held, static_cast<int32_t>(parts),
          static_cast<int32_t>(((vocab + parts - 1) / parts + 7) / 8 * 8)};
}

template <typename T>
int launch(const Cut& cut, const T* logits, int64_t stride, int64_t n_rows, const Scores& out,
           void* workspace, hipStream_t stream) {
  // Parts of the rounded size may be one fewer.
  const int32_t count = (out.vocab + cut.size - 1) / cut.size;
  auto* keys = static_cast<uint64_t*>(workspace);
  auto* sums = reinterpret_cast<Sums*>(keys + n_rows * count * out.top);
  const bool stream_past = n_rows * out.vocab * int64_t(sizeof(T)) > kCacheBytes;
  const auto kernel = cut.held == kSmall ? score_part<T, kSmall, false>
                      : stream_past      ? score_part<T, kLarge, true>
                                         : score_part<T, kLarge, false>;
  for (int64_t first = 0; first < n_rows; first += kMaxGrid / count) {
    const int64_t rows = std::min(n_rows - first, kMaxGrid / count);
    const T* x = logits + first * stride;
    const Scores to{out.tokens + first, out.logprobs + first, out.entropy + first,
                    out.top_logprobs + first * out.top, out.top_ids + first * out.top,
                    out.vocab, out.top};
    const Parts parts{sums + first * count, keys + first * count * out.top, count, cut.size};
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(rows * count)), dim3(kThreads), 0, stream,
                       x, stride, to, parts);
    IEKV_OPS_HIP(hipGetLastError());
    if (count > 1) {
      hipLaunchKernelGGL((join_rows<T>), dim3(static_cast<uint32_t>((rows + kWaves - 1) / kWaves)),
                         dim3(kThreads), 0, stream, x, stride, rows, to, parts);
      IEKV_OPS_HIP(hipGetLastError());
    }
  }
  return IEKV_OK;
}

}  // namespace

extern "C" {

int64_t iekv_logprobs_workspace(int32_t, int64_t n_rows, int64_t vocab, int32_t top) {
  if (n_rows < 1 || vocab < 1 || vocab > INT32_MAX || top < 0) return 0;
  const Cut cut = cut_of(vocab);
  return cut.parts == 1 ? 0 : n_rows * cut.parts * int64_t(sizeof(Sums) + top * sizeof(uint64_t));
}

int iekv_logprobs(int32_t type, const void* logits, int64_t row_stride, int64_t n_rows,
                  int64_t vocab, const int64_t* tokens, int32_t top, float* logprobs,
                  float* entropy, float* top_logprobs, int64_t* top_ids, void* workspace,
                  int64_t workspace_bytes, hipStream_t stream) {
  if (n_rows < 0 || n_rows > INT32_MAX)
    return set_error(IEKV_ERR_INVALID, "n_rows %lld out of range", static_cast<long long>(n_rows));
  if (vocab < 1 || vocab > INT32_MAX - 8 * kThreads * kLarge)
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
  const Cut cut = cut_of(vocab);
  const int64_t need = iekv_logprobs_workspace(type, n_rows, vocab, top);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(IEKV_ERR_CAPACITY, "workspace of %lld bytes, %lld are needed",
                     static_cast<long long>(workspace ? workspace_bytes : 0),
                     static_cast<long long>(need));
  if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(IEKV_ERR_INVALID, "workspace is not aligned to 16 bytes");
  const Scores out{tokens,       logprobs, entropy, top_logprobs, top_ids,
                   static_cast<int32_t>(vocab), top};
  switch (type) {
    case IEKV_TYPE_F32:
      return launch(cut, static_cast<const float*>(logits), row_stride, n_rows, out, workspace,
                    stream);
    case IEKV_TYPE_F16:
      return launch(cut, static_cast<const _Float16*>(logits), row_stride, n_rows, out, workspace,
                    stream);
    default:
      return launch(cut, static_cast<const Bf16*>(logits), row_stride, n_rows, out, workspace,
                    stream);
  }
}

}  // extern "C"
