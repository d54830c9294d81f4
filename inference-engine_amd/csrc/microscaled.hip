// Writing rows into a microscaled cache and reading them back (C-ABI in iekv_ops.h, the format
// in microscaled.h).
#include "microscaled.h"

#include <algorithm>

namespace iekv_ops {
namespace {

constexpr int kThreads = 256;
// Dimensions a lane takes: 16 bytes of rows or of values, so that a wave's are on end; and the
// lanes of a group.
template <typename T>
constexpr int kEach = 16 / int(sizeof(T));
template <typename T>
constexpr int kLanes = kGroup / kEach<T>;

struct Fp8Limits {
  static constexpr int kPower = 8;             // the largest element is 1.75 2^8,
  static constexpr uint32_t kPart = 0x600000;  // its part after the leading one in 23 bits
};
struct Int8Limits {
  static constexpr int kPower = 6;
  static constexpr uint32_t kPart = 0x7e0000;  // 127 = 1.984375 2^6
};
struct Fp4Limits {
  static constexpr int kPower = 2;
  static constexpr uint32_t kPart = 0x400000;  // 6 = 1.5 2^2
};
template <typename C>
using Limits = std::conditional_t<std::is_same_v<C, Mxfp8>, Fp8Limits,
                                  std::conditional_t<std::is_same_v<C, Mxint8>, Int8Limits,
                                                     Fp4Limits>>;

// e + 127 of a group whose largest magnitude has these bits: its own exponent less the largest
// element's, and one more where its part is the larger (the sum carries into the exponent).
template <typename C>
__device__ __forceinline__ uint32_t exponent_byte(uint32_t largest) {
  if (largest >= 0x7f800000u) return 255;      // an infinity or a NaN
  const int32_t e = static_cast<int32_t>((largest + (0x7fffffu - Limits<C>::kPart)) >> 23) -
                    Limits<C>::kPower;
  return max(e, kLeastExponent + 127);
}

// N elements as codes.
template <typename C, int N>
__device__ __forceinline__ Words<(N * kBits<C> + 31) / 32> encode(const float (&x)[N],
                                                                   uint32_t byte) {
  Words<(N * kBits<C> + 31) / 32> r{};
  if (byte == 255) return r;
  if constexpr (std::is_same_v<C, Mxint8>) {
    const float inverse = __builtin_bit_cast(float, (254 - byte) << 23);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int32_t c = static_cast<int32_t>(rintf(x[i] * inverse));
      r.w[i / 4] |= (static_cast<uint32_t>(c) & 255u) << i % 4 * 8;
    }
  } else if constexpr (std::is_same_v<C, Mxfp8>) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const float scale = __builtin_bit_cast(float, byte << 23);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      s16x2 w{};
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i], x[4 * i + 1], scale, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i + 2], x[4 * i + 3], scale, true);
      r.w[i] = __builtin_bit_cast(uint32_t, w);
    }
  } else {
    const float scale = __builtin_bit_cast(float, byte << 23);
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    if constexpr (N == 8) {
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    }
    r.w[0] = w;
  }
  return r;
}

// n / d by a product (Granlund and Montgomery), for any n of 32 bits and d up to 2^31.
struct Divisor {
  uint32_t d, magic, shift;
};
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor& by) {
  return static_cast<uint32_t>((static_cast<uint64_t>(__umulhi(n, by.magic)) + n) >> by.shift);
}

// Two arrays at a time of those at even distances: their loads are on their way together, and
// what finds a lane's place is paid once.
constexpr int kAtOnce = 2;

// Slots or block ids: in device memory, or in a launch's own arguments, where no upload has to
// come before it (a call with a list of 37 slots 12.6 us of the host against 24.9).
template <typename I, int N>
struct Ids {
  I id[N];
  __device__ __forceinline__ I operator[](uint32_t i) const { return id[i]; }
};
template <typename I>
struct Ids<I, 0> {
  const I* id;
  __device__ __forceinline__ I operator[](uint32_t i) const { return id[i]; }
};

struct WriteArgs {
  uint64_t k_cache, v_cache;                   // of the first layer
  int64_t k_cache_stride, v_cache_stride;      // bytes from one layer's to the next
  const void* k;
  const void* v;
  int64_t k_layer, k_token, k_head, v_layer, v_token, v_head;   // strides in elements
  int64_t n_slots;
  uint32_t n;                                  // tokens
  int32_t layers, heads, head_dim;
  Divisor lanes, row_lanes;                    // of a head (a multiple of kLanes), of a token
};

// Bound by memory: a lane brings 16 bytes of K and of V of one token's head, the lanes of a
// group find its largest magnitude, and each writes its codes. The rows are read past the
// caches, which leaves room there for the codes' lines to be filled: 32 layers of 2,001 tokens
// of eight bf16 heads of 128 to mxfp8 63 us (6.3 TB/s), 74 with ordinary loads; one layer at a
// time 86, four at a time 75 (of those).
template <typename T, typename C, int N>
__global__ __launch_bounds__(kThreads) void write_rows(WriteArgs a, Ids<int64_t, N> slots) {
  constexpr int EACH = kEach<T>, LANES = kLanes<T>;
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t t = quotient(at, a.row_lanes), in_row = at - t * a.row_lanes.d;
  if (t >= a.n) return;                        // whole groups of lanes
  const uint32_t head = quotient(in_row, a.lanes), lane = in_row - head * a.lanes.d;
  const int32_t d0 = lane * EACH, layer0 = blockIdx.y * kAtOnce;
  const bool in = d0 < a.head_dim;
  Words<4> raw[kAtOnce][2];
#pragma unroll
  for (int l = 0; l < kAtOnce; ++l)
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int64_t layer = min(layer0 + l, a.layers - 1);
      const T* from = static_cast<const T*>(o ? a.v : a.k) +
                      layer * (o ? a.v_layer : a.k_layer) + t * (o ? a.v_token : a.k_token) +
                      head * (o ? a.v_head : a.k_head);
      raw[l][o] = stream_bytes<16>(from + (in ? d0 : 0));
    }
  const int64_t slot = slots[t];
  const int32_t codes = code_bytes<C>(a.head_dim), record = head_bytes<C>(a.head_dim);
#pragma unroll
  for (int l = 0; l < kAtOnce; ++l)
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      T row[EACH];
      __builtin_memcpy(row, &raw[l][o], 16);
      // Magnitudes as integers: a NaN is the largest of all.
      float x[EACH];
      uint32_t largest = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        x[i] = in ? to_float(row[i]) : 0.f;
        largest = max(largest, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
      }
      largest = max(largest, lane_xor<1>(largest));
      largest = max(largest, lane_xor<2>(largest));
      if constexpr (LANES == 8) largest = max(largest, lane_xor<4>(largest));
      const uint32_t byte = exponent_byte<C>(largest);
      const auto code = encode<C>(x, byte);
      if (static_cast<uint64_t>(slot) >= static_cast<uint64_t>(a.n_slots) ||
          layer0 + l >= a.layers)
        continue;
      char* to = reinterpret_cast<char*>((o ? a.v_cache : a.k_cache) +
                                         (layer0 + l) * (o ? a.v_cache_stride : a.k_cache_stride)) +
                 (slot * a.heads + head) * record;
      if (in) __builtin_memcpy(to + code_bytes<C>(d0), &code, code_bytes<C>(EACH));
      if (lane % LANES == 0) to[codes + lane / LANES] = static_cast<char>(byte);
      // Bytes past the last group.
      if (lane == 0)
        for (int32_t g = a.lanes.d / LANES; g < kScaleBytes; ++g) to[codes + g] = 0;
    }
}

struct ReadArgs {
  uint64_t cache;                              // the first array
  int64_t cache_stride;
  void* out;                                   // [arrays][n][heads][head_dim]
  int64_t out_stride;                          // elements from one array's values to the next
  uint32_t n;                                  // rows
  int32_t arrays, heads, head_dim;
  int64_t num_blocks;
  Divisor lanes, row_lanes, block_size;        // lanes: of a head, and of a row
};

// Bound by memory: a lane makes 16 bytes of values, of several arrays. The values pass the
// caches by, the records stay in them where a write has just left them there: 64 arrays of 6,000
// rows of eight heads of 128 from mxfp8 to bf16 190 us (6.3 TB/s), 204 with ordinary stores and
// 230 with loads past the caches; one array at a time 234, four 204. (Stores past the caches pay
// only where a wave's are on end: with 32 bytes a lane 285.)
template <typename T, typename C, int N>
__global__ __launch_bounds__(kThreads) void read_rows(ReadArgs a, Ids<int32_t, N> table) {
  constexpr int EACH = kEach<T>;
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t j = quotient(at, a.row_lanes), in_row = at - j * a.row_lanes.d;
  if (j >= a.n) return;
  const uint32_t head = quotient(in_row, a.lanes), b = quotient(j, a.block_size);
  const int32_t d0 = (in_row - head * a.lanes.d) * EACH, array0 = blockIdx.y * kAtOnce;
  const int32_t block = table[b];
  if (block < 0 || block >= a.num_blocks) return;
  const int64_t row = static_cast<int64_t>(block) * a.block_size.d + (j - b * a.block_size.d);
  const char* from = reinterpret_cast<const char*>(a.cache) +
                     (row * a.heads + head) * head_bytes<C>(a.head_dim);
  Words<(EACH * kBits<C> + 31) / 32> code[kAtOnce];
  uint32_t scales[kAtOnce];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    const char* of = from + min(array0 + i, a.arrays - 1) * a.cache_stride;
    code[i] = load_bytes<code_bytes<C>(EACH)>(of + code_bytes<C>(d0));
    scales[i] = load_bytes<kScaleBytes>(of + code_bytes<C>(a.head_dim)).w[0];
  }
  const int64_t in_array = (static_cast<int64_t>(j) * a.heads + head) * a.head_dim + d0;
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    if (array0 + i >= a.arrays) break;
    T* to = static_cast<T*>(a.out) +
            static_cast<int64_t>(array0 + i) * a.out_stride + in_array;
    stream_out<16>(to, scaled<T, C, EACH>(code[i], scale_of(scales[i], d0 / kGroup * 8)));
  }
}

Divisor divisor(uint32_t d) {
  Divisor r{d, 0, 0};
  while ((uint64_t(1) << r.shift) < d) ++r.shift;
  r.magic = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << r.shift) - d)) / d + 1);
  return r;
}

int check_cache(const iekv_mx_cache* c) {
  if (!c) return set_error(IEKV_ERR_INVALID, "cache is null");
  if (c->cache_type < IEKV_TYPE_MXFP8 || c->cache_type > IEKV_TYPE_MXFP4)
    return set_error(IEKV_ERR_INVALID, "%d is no microscaled type", c->cache_type);
  if (c->num_kv_heads < 1 || c->num_kv_heads > 4096)
    return set_error(IEKV_ERR_INVALID, "num_kv_heads %d out of range", c->num_kv_heads);
  if (c->head_dim < 8 || c->head_dim > IEKV_ATTENTION_MAX_DIM || c->head_dim % 8)
    return set_error(IEKV_ERR_INVALID, "head_dim %d is not a multiple of 8 up to %d", c->head_dim,
                     IEKV_ATTENTION_MAX_DIM);
  if (c->block_size < 1 || c->block_size > (1 << 20))
    return set_error(IEKV_ERR_INVALID, "block_size %d out of range", c->block_size);
  if (c->num_blocks < 1 || c->num_blocks > INT32_MAX)
    return set_error(IEKV_ERR_INVALID, "num_blocks %lld out of range",
                     static_cast<long long>(c->num_blocks));
  return IEKV_OK;
}

bool is_float(int32_t type) { return type >= IEKV_TYPE_F32 && type <= IEKV_TYPE_BF16; }

// How many of the arrays from `first` on lie at even distances, and that distance: all of a
// pool's that one allocation holds, two at least of others.
int32_t run_of(const uint64_t* arrays, int32_t first, int32_t n, int64_t* stride) {
  *stride = first + 1 < n ? static_cast<int64_t>(arrays[first + 1] - arrays[first]) : 0;
  int32_t last = first;
  while (last + 1 < n && static_cast<int64_t>(arrays[last + 1] - arrays[last]) == *stride) ++last;
  return last - first + 1;
}

// Calls f with a row type and a cache type.
template <typename F>
void with_types(int32_t row, int32_t cache, F f) {
  const auto with_cache = [&](auto t) {
    switch (cache) {
      case IEKV_TYPE_MXFP8: return f(t, Mxfp8{});
      case IEKV_TYPE_MXINT8: return f(t, Mxint8{});
      default: return f(t, Mxfp4{});
    }
  };
  switch (row) {
    case IEKV_TYPE_F32: return with_cache(float{});
    case IEKV_TYPE_F16: return with_cache(_Float16{});
    default: return with_cache(Bf16{});
  }
}

constexpr int32_t kMostLayers = 65535;         // of a launch: its grid's second dimension
constexpr int32_t kSlots = IEKV_MX_INLINE_SLOTS, kBlocks = IEKV_MX_INLINE_BLOCKS;

// N: slots on the host that a launch carries, 0 for those on the device.
template <int N>
int write(const iekv_mx_cache* cache, const uint64_t* k_arrays, const uint64_t* v_arrays,
          int32_t n_layers, int32_t row_type, const void* k, const int64_t* k_strides,
          const void* v, const int64_t* v_strides, const int64_t* slots, int64_t n_tokens,
          hipStream_t stream) {
  if (const int rc = check_cache(cache)) return rc;
  if (!is_float(row_type)) return set_error(IEKV_ERR_INVALID, "rows of type %d", row_type);
  if (n_layers < 0 || n_tokens < 0)
    return set_error(IEKV_ERR_INVALID, "%d layers of %lld tokens", n_layers,
                     static_cast<long long>(n_tokens));
  if (!n_layers || !n_tokens) return IEKV_OK;
  if (!k_arrays || !v_arrays || !k || !k_strides || !v || !v_strides || !slots)
    return set_error(IEKV_ERR_INVALID, "null argument");
  const int64_t size = row_type == IEKV_TYPE_F32 ? 4 : 2;
  const int64_t n_slots = cache->num_blocks * cache->block_size;
  for (int64_t t = 0; N && t < n_tokens; ++t)
    if (slots[t] < 0 || slots[t] >= n_slots)
      return set_error(IEKV_ERR_RANGE, "slot %lld out of range for a pool of %lld slots",
                       static_cast<long long>(slots[t]), static_cast<long long>(n_slots));
  const int32_t lanes = (cache->head_dim + kGroup - 1) / kGroup *
                        (row_type == IEKV_TYPE_F32 ? kLanes<float> : kLanes<Bf16>);
  // Tokens of a launch.
  const int64_t most = N ? N : kMaxGrid * kThreads / (cache->num_kv_heads * lanes);
  for (int32_t l = 0; l < n_layers;) {
    WriteArgs a{};
    const int32_t run = std::min(std::min(run_of(k_arrays, l, n_layers, &a.k_cache_stride),
                                          run_of(v_arrays, l, n_layers, &a.v_cache_stride)),
                                 kMostLayers);
    a.k_cache = k_arrays[l];
    a.v_cache = v_arrays[l];
    a.k_layer = k_strides[0], a.k_token = k_strides[1], a.k_head = k_strides[2];
    a.v_layer = v_strides[0], a.v_token = v_strides[1], a.v_head = v_strides[2];
    a.n_slots = n_slots;
    a.layers = run;
    a.heads = cache->num_kv_heads;
    a.head_dim = cache->head_dim;
    a.lanes = divisor(lanes);
    a.row_lanes = divisor(a.heads * lanes);
    for (int64_t t = 0; t < n_tokens; t += most) {
      a.k = static_cast<const char*>(k) + (l * a.k_layer + t * a.k_token) * size;
      a.v = static_cast<const char*>(v) + (l * a.v_layer + t * a.v_token) * size;
      a.n = static_cast<uint32_t>(std::min(most, n_tokens - t));
      Ids<int64_t, N> ids;
      if constexpr (N)
        std::copy_n(slots + t, a.n, ids.id);
      else
        ids.id = slots + t;
      const int64_t threads = static_cast<int64_t>(a.n) * a.heads * lanes;
      const dim3 grid((threads + kThreads - 1) / kThreads, (run + kAtOnce - 1) / kAtOnce);
      with_types(row_type, cache->cache_type, [&](auto row, auto code) {
        hipLaunchKernelGGL((write_rows<decltype(row), decltype(code), N>), grid, dim3(kThreads), 0,
                           stream, a, ids);
      });
      IEKV_OPS_HIP(hipGetLastError());
    }
    l += run;
  }
  return IEKV_OK;
}

template <int N>
int read(const iekv_mx_cache* cache, const uint64_t* arrays, int32_t n_arrays,
         const int32_t* table, int64_t context_len, int32_t out_type, void* out,
         hipStream_t stream) {
  if (const int rc = check_cache(cache)) return rc;
  if (!is_float(out_type)) return set_error(IEKV_ERR_INVALID, "values of type %d", out_type);
  if (n_arrays < 0 || context_len < 0 || context_len > IEKV_ATTENTION_MAX_CONTEXT)
    return set_error(IEKV_ERR_INVALID, "%d arrays of a context of %lld", n_arrays,
                     static_cast<long long>(context_len));
  if (!n_arrays || !context_len) return IEKV_OK;
  if (!arrays || !table || !out) return set_error(IEKV_ERR_INVALID, "null argument");
  const int64_t size = out_type == IEKV_TYPE_F32 ? 4 : 2, bs = cache->block_size;
  const int64_t used = (context_len + bs - 1) / bs;
  for (int64_t b = 0; N && b < used; ++b)
    if (table[b] < 0 || table[b] >= cache->num_blocks)
      return set_error(IEKV_ERR_RANGE, "block id %d out of range for a pool of %lld blocks",
                       table[b], static_cast<long long>(cache->num_blocks));
  const int32_t lanes = cache->head_dim * static_cast<int32_t>(size) / 16;
  const int64_t row = static_cast<int64_t>(cache->num_kv_heads) * cache->head_dim;
  // Blocks of a launch.
  const int64_t fit = kMaxGrid * kThreads / (cache->num_kv_heads * lanes) / bs;
  const int64_t most = N ? std::min<int64_t>(N, fit) : fit;
  if (!most)
    return set_error(IEKV_ERR_INVALID, "blocks of %lld rows of %d heads are too large",
                     static_cast<long long>(bs), cache->num_kv_heads);
  for (int32_t i = 0; i < n_arrays;) {
    ReadArgs a{};
    const int32_t run = std::min(run_of(arrays, i, n_arrays, &a.cache_stride), kMostLayers);
    a.cache = arrays[i];
    a.out_stride = context_len * row;
    a.arrays = run;
    a.heads = cache->num_kv_heads;
    a.head_dim = cache->head_dim;
    a.lanes = divisor(lanes);
    a.row_lanes = divisor(a.heads * lanes);
    a.block_size = divisor(cache->block_size);
    a.num_blocks = cache->num_blocks;
    for (int64_t b = 0; b < used; b += most) {
      a.n = static_cast<uint32_t>(std::min(most * bs, context_len - b * bs));
      a.out = static_cast<char*>(out) + (i * context_len + b * bs) * row * size;
      Ids<int32_t, N> ids;
      if constexpr (N)
        std::copy_n(table + b, std::min(most, used - b), ids.id);
      else
        ids.id = table + b;
      const int64_t threads = a.n * static_cast<int64_t>(a.heads) * lanes;
      const dim3 grid((threads + kThreads - 1) / kThreads, (run + kAtOnce - 1) / kAtOnce);
      with_types(out_type, cache->cache_type, [&](auto value, auto code) {
        hipLaunchKernelGGL((read_rows<decltype(value), decltype(code), N>), grid, dim3(kThreads),
                           0, stream, a, ids);
      });
      IEKV_OPS_HIP(hipGetLastError());
    }
    i += run;
  }
  return IEKV_OK;
}

}  // namespace
}  // namespace iekv_ops

using namespace iekv_ops;

extern "C" {

int64_t iekv_mx_head_bytes(int32_t cache_type, int32_t head_dim) {
  if (cache_type < IEKV_TYPE_MXFP8 || cache_type > IEKV_TYPE_MXFP4 || head_dim < 8 ||
      head_dim > IEKV_ATTENTION_MAX_DIM || head_dim % 8)
    return 0;
  return cache_type == IEKV_TYPE_MXFP4 ? head_bytes<Mxfp4>(head_dim) : head_bytes<Mxfp8>(head_dim);
}

int iekv_mx_write_slots(const iekv_mx_cache* cache, const uint64_t* k_arrays,
                        const uint64_t* v_arrays, int32_t n_layers, int32_t row_type,
                        const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, const int64_t* slots, int64_t n_tokens,
                        hipStream_t stream) {
  return write<0>(cache, k_arrays, v_arrays, n_layers, row_type, k, k_strides, v, v_strides, slots,
                  n_tokens, stream);
}

int iekv_mx_write_slots_ids(const iekv_mx_cache* cache, const uint64_t* k_arrays,
                            const uint64_t* v_arrays, int32_t n_layers, int32_t row_type,
                            const void* k, const int64_t* k_strides, const void* v,
                            const int64_t* v_strides, const int64_t* slots, int64_t n_tokens,
                            hipStream_t stream) {
  return write<kSlots>(cache, k_arrays, v_arrays, n_layers, row_type, k, k_strides, v, v_strides,
                       slots, n_tokens, stream);
}

int iekv_mx_read_rows(const iekv_mx_cache* cache, const uint64_t* arrays, int32_t n_arrays,
                      const int32_t* table, int64_t context_len, int32_t out_type, void* out,
                      hipStream_t stream) {
  return read<0>(cache, arrays, n_arrays, table, context_len, out_type, out, stream);
}

int iekv_mx_read_rows_ids(const iekv_mx_cache* cache, const uint64_t* arrays, int32_t n_arrays,
                          const int32_t* table, int64_t context_len, int32_t out_type, void* out,
                          hipStream_t stream) {
  return read<kBlocks>(cache, arrays, n_arrays, table, context_len, out_type, out, stream);
}

}  // extern "C"
