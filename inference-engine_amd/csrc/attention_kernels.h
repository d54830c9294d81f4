// Device code of attention over the paged cache: the rows of a work item (attention_plan.h)
// against its keys. `narrow` holds up to 16 rows and streams the cache, a wave to itself;
// `wide` holds many rows, whose waves share tiles of keys; `join` puts parts together.
//
// Both compute S^T = K Q^T and then O^T = V^T P^T. A matrix instruction returns a column of
// S^T per lane, four (or eight) of its keys at a time, which is also how it takes a column of
// P^T: the weights go from one product into the other without leaving their lane, and a
// row's maximum, sum and rescaling are that lane's own. Which key sits at which place of the
// contraction is free as long as V^T is given in the same order; the key orders below make
// the two fit.
#ifndef IEKV_ATTENTION_KERNELS_H_
#define IEKV_ATTENTION_KERNELS_H_

#include <type_traits>

#include "attention_plan.h"
#include "microscaled.h"
#include "ops_common.h"

namespace iekv_ops {

using iekv_attention::Item;

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr int kWaves = kThreads / kWave;

struct Args {
  const int32_t* words;       // the plan's words: its items first
  const void* k;
  const void* v;
  const void* q;
  void* out;
  float* part_o;              // [slots][kv_heads][head_dim]: sums of e^(s - m) v
  float2* part_ml;            // [slots][kv_heads]: m (base 2) and the sum of e^(s - m)
  int64_t positions_at, tables_at;
  int64_t q_token_stride, q_head_stride;
  int32_t window, sinks;      // window: INT32_MAX for all keys
  int32_t kv_heads, group, head_dim, block_size;
  int32_t together;           // KV heads of a narrow item that a workgroup takes: 1, 2 or 4
  uint32_t block_magic, block_shift;  // j / block_size = (mulhi(j, magic) + j) >> shift
  uint32_t q_sign;            // flips the sign of q (in each half for 16 bits): scale >= 0
  float scale;                // |scale| log2(e)
};

// --- elements ----------------------------------------------------------------------------

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// N elements of type C as elements of the compute type T (exact: T holds every value of C).
template <typename T, typename C, int N>
struct Convert {                                 // T == C
  static __device__ __forceinline__ Words<N * sizeof(T) / 4> of(
      const Words<(N * sizeof(C) + 3) / 4>& x) {
    return x;
  }
};
template <int N>
struct Convert<Bf16, E4m3, N> {
  static __device__ __forceinline__ Words<N / 2> of(const Words<(N + 3) / 4>& x) {
    Words<N / 2> r;
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      r.w[i] = __builtin_bit_cast(
          uint32_t, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w[i / 2], 1.f, true)
                          : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w[i / 2], 1.f, false));
    return r;
  }
};
template <int N>
struct Convert<_Float16, E4m3, N> {
  static __device__ __forceinline__ Words<N / 2> of(const Words<(N + 3) / 4>& x) {
    Words<N / 2> r;
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      r.w[i] = __builtin_bit_cast(
          uint32_t, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.w[i / 2], 1.f, true)
                          : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.w[i / 2], 1.f, false));
    return r;
  }
};
template <int N>
struct Convert<float, E4m3, N> {
  static __device__ __forceinline__ Words<N> of(const Words<(N + 3) / 4>& x) {
    Words<N> r;
#pragma unroll
    for (int i = 0; i < N; ++i)
      r.w[i] = __builtin_bit_cast(
          uint32_t, to_float(E4m3{static_cast<uint8_t>(x.w[i / 4] >> (i % 4 * 8))}));
    return r;
  }
};
template <int N>
struct Convert<float, Bf16, N> {
  static __device__ __forceinline__ Words<N> of(const Words<N / 2>& x) {
    Words<N> r;
#pragma unroll
    for (int i = 0; i < N; ++i)
      r.w[i] = i % 2 ? x.w[i / 2] & 0xffff0000u : x.w[i / 2] << 16;
    return r;
  }
};
template <int N>
struct Convert<float, _Float16, N> {
  static __device__ __forceinline__ Words<N> of(const Words<N / 2>& x) {
    Words<N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint16_t h = static_cast<uint16_t>(x.w[i / 2] >> (i % 2 * 16));
      r.w[i] = __builtin_bit_cast(uint32_t, static_cast<float>(__builtin_bit_cast(_Float16, h)));
    }
    return r;
  }
};

// c += A B with 16 rows and columns over the lane's elements of A and B: eight of 16 bits
// (32 in all), or four of 32 bits (16 in all).
__device__ __forceinline__ f32x4 mma16(const Words<4>& a, const Words<4>& b, f32x4 c, Bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const Words<4>& a, const Words<4>& b, f32x4 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const Words<4>& a, const Words<4>& b, f32x4 c, float) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, a.w[e]),
                                             __builtin_bit_cast(float, b.w[e]), c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x16 mma32(const Words<4>& a, const Words<4>& b, f32x16 c, Bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(const Words<4>& a, const Words<4>& b, f32x16 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// --- keys --------------------------------------------------------------------------------

__device__ __forceinline__ Item item_of(const Args& a, int32_t i) {
  return reinterpret_cast<const Item*>(a.words)[i];
}

// Key number `v` of the item's ranges laid end to end.
__device__ __forceinline__ int32_t key_at(const Item& it, int32_t v) {
  const int32_t na = it.a1 - it.a0;
  return v < na ? it.a0 + v : it.b0 + (v - na);
}

__device__ __forceinline__ bool sees(const Args& a, int32_t position, int32_t key) {
  return (key <= position) & ((key > position - a.window) | (key < a.sinks));
}

// Every position of the item sees every one of its keys v0 .. v1 - 1.
__device__ __forceinline__ bool all_see(const Args& a, const Item& it, int32_t v0, int32_t v1) {
  if (it.low == it.high) return true;            // its ranges are what the position sees
  const int32_t first = key_at(it, v0), last = key_at(it, v1 - 1);
  return last - first == v1 - 1 - v0 && last <= it.low &&
         (first > it.high - a.window || last < a.sinks);
}

// A key's place in the pool: its block's entry in the tables, and its row there.
struct Place {
  int32_t block, within;
};
__device__ __forceinline__ Place place_of(const Args& a, const Item& it, int32_t j) {
  const uint32_t b = (__umulhi(j, a.block_magic) + j) >> a.block_shift;
  return {a.words[a.tables_at + it.table + b],
          static_cast<int32_t>(j - b * static_cast<uint32_t>(a.block_size))};
}
__device__ __forceinline__ uint32_t row_of(const Args& a, Place p) {
  return static_cast<uint32_t>(p.block) * static_cast<uint32_t>(a.block_size) + p.within;
}

// What rounding to T leaves of two weights that it made `w`.
template <typename T>
__device__ __forceinline__ uint32_t rest2(float p0, float p1, uint32_t w) {
  const Words<2> held = Convert<float, T, 2>::of(Words<1>{{w}});
  return pack2<T>(p0 - __builtin_bit_cast(float, held.w[0]),
                  p1 - __builtin_bit_cast(float, held.w[1]));
}

__device__ __forceinline__ float power2(float x) { return __builtin_amdgcn_exp2f(x); }

// float16 ends at 2^-25: of weights relative to a largest one of about 1, a long flat tail beside
// a single high key would be lost from O while their sum holds it. So m is held that many powers
// of two below the maximum, and the weights as many above, up to 2^15: O and the sum carry the
// factor alike. What is lost then is less than 2^-39 (narrow) and 2^-32 (wide, where the maximum
// may be 2^8 more) of the largest weight. The other types reach as far down as the power does.
template <typename T>
constexpr float lift(float narrow_or_wide) {
  return std::is_same_v<T, _Float16> ? narrow_or_wide : 0.f;
}

// --- one row key by key ------------------------------------------------------------------

// The matrix kernels take s - m of a score that is not rounded first (one operation less a
// key), where m is: off by half a step of m, which past this many powers of two would leave a
// row's largest weight far above or below 1, in the end infinite or zero.
constexpr float kFar = 1 << 20;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > kFar && fabsf(m) < INFINITY; }

// Dimension `i` of a head of `d` in the cache, as T holds it.
template <typename T, typename C>
__device__ __forceinline__ float cached(const char* head, int32_t d, int32_t i) {
  if constexpr (!kScaled<C>) {
    return to_float(reinterpret_cast<const C*>(head)[i]);
  } else {
    const uint8_t code = head[code_bytes<C>(i)];
    const uint32_t w = kBits<C> == 4 ? code >> i % 2 * 4 : code;
    const float scale = scale_of(static_cast<uint8_t>(head[code_bytes<C>(d) + i / kGroup]), 0);
    const float x = __builtin_bit_cast(float, pair_of<float, C>(&w, 0, scale).w[0]);
    return to_float(from_float<T>(x));
  }
}

// One query row by one wave: a lane scores a key of each 64, then holds two dimensions of
// the output. A key the row does not see is not read for it at all, so that whatever the
// cache holds there (infinities, NaN) stays out. The matrix kernels multiply such a V by a
// weight of zero; where that, or anything else, leaves a NaN in their output, or where a row's
// maximum is far, they come here for the item's rows, at a hundredth of their speed.
template <typename T, typename C>
__device__ void attend_row(const Args& a, const Item& it, int32_t kv_head, int32_t row, int lane) {
  const int32_t token = it.token0 + row / a.group, in_group = row % a.group;
  const int32_t position = a.words[a.positions_at + token];
  const int32_t d = a.head_dim;
  const int32_t size = head_bytes<C>(d);
  const int64_t row_bytes = static_cast<int64_t>(a.kv_heads) * size;
  const int64_t head = static_cast<int64_t>(kv_head) * a.group + in_group;
  const T* q = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride;
  const char* kc = static_cast<const char*>(a.k) + static_cast<int64_t>(kv_head) * size;
  const char* vc = static_cast<const char*>(a.v) + static_cast<int64_t>(kv_head) * size;
  const float scale = a.q_sign ? -a.scale : a.scale;
  const int32_t n = (it.a1 - it.a0) + (it.b1 - it.b0);
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int32_t v0 = 0; v0 < n; v0 += kWave) {
    const bool in = v0 + lane < n;
    const int32_t j = key_at(it, in ? v0 + lane : n - 1);
    const int64_t at = row_of(a, place_of(a, it, j)) * row_bytes;
    const bool seen = in && sees(a, position, j);
    float s = -INFINITY;
    if (seen) {
      float dot = 0.f;
      for (int32_t i = 0; i < d; ++i) dot = fmaf(to_float(q[i]), cached<T, C>(kc + at, d, i), dot);
      s = dot * scale;
    }
    // A score that is NaN stays in the sum, and the row is NaN as it has to be.
    const float top = fmaxf(m, wave_max(s));
    const float base = top == -INFINITY ? 0.f : top;
    const float fade = exp2f(m - base);
    const float p = seen ? exp2f(s - base) : 0.f;
    m = top;
    l = l * fade + wave_sum(p);
    o0 *= fade;
    o1 *= fade;
    uint64_t left = __ballot(seen);
    while (left) {
      const int i = __ffsll(static_cast<unsigned long long>(left)) - 1;
      left &= left - 1;
      const float pi = __shfl(p, i);
      const int64_t ai = __shfl(at, i);
      if (lane < d) o0 = fmaf(pi, cached<T, C>(vc + ai, d, lane), o0);
      if (lane + kWave < d) o1 = fmaf(pi, cached<T, C>(vc + ai, d, lane + kWave), o1);
    }
  }
  if (it.slot >= 0) {
    const int64_t slot = static_cast<int64_t>(it.slot + row) * a.kv_heads + kv_head;
    if (lane < d) a.part_o[slot * d + lane] = o0;
    if (lane + kWave < d) a.part_o[slot * d + lane + kWave] = o1;
    if (lane == 0) a.part_ml[slot] = {m, l};
    return;
  }
  T* out = static_cast<T*>(a.out) + (token * static_cast<int64_t>(a.kv_heads) * a.group + head) * d;
  if (lane < d) out[lane] = from_float<T>(o0 / l);
  if (lane + kWave < d) out[lane + kWave] = from_float<T>(o1 / l);
}

// --- narrow: up to 16 rows ---------------------------------------------------------------

// N floats of a row's output, as T.
template <typename T, int N>
__device__ __forceinline__ void store_out(T* out, const float* x) {
  if constexpr (sizeof(T) == 4) {
    __builtin_memcpy(out, x, N * 4);
  } else {
    Words<N / 2> w;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w.w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    __builtin_memcpy(out, &w, N * 2);
  }
}

// 16 bytes of each lane into LDS, the wave's in a row from `to` on; past the caches if STREAM.
template <bool STREAM = false>
__device__ __forceinline__ void bring16(const char* from, u32x4* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) uint32_t*)reinterpret_cast<uintptr_t>(from),
      (__attribute__((address_space(3))) uint32_t*)to, 16, 0, STREAM ? 2 : 0);
}

// A barrier that the wave's loads into LDS have ended at, too.
__device__ __forceinline__ void arrive() {
  __builtin_amdgcn_s_waitcnt(0xf70);      // vmcnt 0; the other counters are not waited for
  __syncthreads();
}

// The records of a step of a microscaled cache, on their way through LDS into the products'
// operands. Records begin at any multiple of 4, and as operands sixteen lanes would take from
// sixteen of them: what bounds such loads is the first cache, a line at a time. So a wave brings
// the 64 records in chunks of 16 bytes laid end to end (of 32 dimensions 4), the last of each the
// one that ends with the scales, and every lane's load is full. 48 sequences of 6,000 tokens of
// eight mxfp8 heads of 128 120 us, against 137 where lanes load their operands' records (and 183
// past the caches: neighbouring records share their lines, which are then brought twice).
template <typename C, int DP>
struct Staged {
  static constexpr int KEYS = 64;
  static constexpr int CODES = DP * kBits<C> / 8;            // bytes of a key; its scales' chunk
  static constexpr int W = DP == 32 ? 4 : 16;                // follows them
  static constexpr int CHUNKS = CODES / W + 1;               // and loads of a wave
  // Reads of neighbouring keys meet in no bank.
  static constexpr int PITCH = CODES + W + (CODES == 48 ? 16 : 0);
  alignas(16) char bytes[kScaled<C> ? KEYS * PITCH : 16];

  using Chunk = Words<W / 4>;
  // What a lane brings with each of its loads: chunk 64 n + lane of all. The key, the bytes into
  // its record, and its place here.
  struct Lane {
    int32_t key[CHUNKS], from[CHUNKS], to[CHUNKS];
  };

  // Key 32 p + 8 a + 4 b + e lies at 32 p + 16 b + 4 a + e: in the order in which the lanes of
  // two tiles of scores take them.
  static __device__ __forceinline__ int32_t placed(int32_t key) {
    return (key & 32) | (key & 4) << 2 | (key & 24) >> 1 | (key & 3);
  }
  static __device__ __forceinline__ Lane lane_of(int lane, int32_t d) {
    Lane r;
#pragma unroll
    for (int n = 0; n < CHUNKS; ++n) {
      const int32_t at = n * kWave + lane, key = at / CHUNKS, chunk = at % CHUNKS;
      const int32_t codes = code_bytes<C>(d);
      // The last of the codes begins sooner where it would end behind them.
      const int32_t begin = chunk * W < codes - W ? chunk * W : codes - W;
      const bool scales = chunk == CHUNKS - 1;
      r.key[n] = key;
      r.from[n] = scales ? codes + kScaleBytes - W : begin;
      r.to[n] = placed(key) * PITCH + (scales ? CODES : begin);
    }
    return r;
  }
  // Zeros behind the dimensions, where nothing is brought.
  __device__ __forceinline__ void clear(int lane) {
    for (int32_t i = lane * 4; i < KEYS * PITCH; i += kWave * 4)
      __builtin_memset(__builtin_assume_aligned(bytes + i, 4), 0, 4);
  }
  static __device__ __forceinline__ void load(Chunk (&x)[CHUNKS], const Lane& lane,
                                              const char* head, const int64_t* rows) {
#pragma unroll
    for (int n = 0; n < CHUNKS; ++n) x[n] = load_bytes<W>(head + rows[lane.key[n]] + lane.from[n]);
  }
  __device__ __forceinline__ void put(const Chunk (&x)[CHUNKS], const Lane& lane, int32_t d) {
    if (code_bytes<C>(d) % W == 0) {
#pragma unroll
      for (int n = 0; n < CHUNKS; ++n)
        __builtin_memcpy(__builtin_assume_aligned(bytes + lane.to[n], W), &x[n], W);
    } else {
#pragma unroll
      for (int n = 0; n < CHUNKS; ++n)
        __builtin_memcpy(__builtin_assume_aligned(bytes + lane.to[n], 4), &x[n], W);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // BYTES of the codes of the key at a place, from dimension `d0` on; and 2^e of its group.
  template <int BYTES>
  __device__ __forceinline__ Words<(BYTES + 3) / 4> codes(int32_t place, int32_t d0) const {
    constexpr int align = BYTES % 16 == 0 && PITCH % 16 == 0  ? 16
                          : BYTES % 8 == 0 && PITCH % 8 == 0 ? 8
                          : BYTES % 4 == 0                   ? 4
                                                             : BYTES;
    Words<(BYTES + 3) / 4> r;
    r.w[(BYTES - 1) / 4] = 0;
    __builtin_memcpy(&r, __builtin_assume_aligned(bytes + place * PITCH + code_bytes<C>(d0), align),
                     BYTES);
    return r;
  }
  __device__ __forceinline__ float scale(int32_t place, int32_t d0) const {
    return scale_of(static_cast<uint8_t>(bytes[place * PITCH + CODES + W - kScaleBytes +
                                               d0 / kGroup]), 0);
  }
};

// The same of the four neighbouring heads that a workgroup takes: their records lie on end, and
// of whole groups of 32 dimensions four are a multiple of 16 bytes. The workgroup brings them as
// they lie, straight into LDS and each line once; a wave reads its own head's out of them. Two
// tiles in turn, so that a step's loads are on their way while the one before is worked on and a
// step has one barrier: 48 sequences of 6,000 tokens of eight mxfp8 heads of 128 107 us a call
// with its joins, 128 of 4,200 in mxfp4 115; through registers and one tile 112 and 127, each
// wave with its own head's records (Staged) 131 and 144. 32 keys at a time and two workgroups to a
// compute unit (short records three): what is on its way then stays in L2 until the workgroup of
// the next four heads has taken its part of the lines that they share. Past the caches, or 117
// and 116.
template <typename C, int DP>
struct Together {
  static constexpr int KEYS = 32, HEADS = 4;
  static constexpr int CODES = DP * kBits<C> / 8, RECORD = head_bytes<C>(DP);
  static constexpr int PITCH = HEADS * RECORD;
  // Chunks of 16 bytes of a key, as many loads as K's and V's of a step are (of 64 chunks each),
  // and what a wave has of these.
  static constexpr int OF_KEY = PITCH / 16, LOADS = (OF_KEY + kWaves - 1) / kWaves;
  static_assert(!kScaled<C> || PITCH % 16 == 0);
  struct Tile {
    alignas(16) char k[KEYS * PITCH], v[KEYS * PITCH];
  };
  struct Lane {
    const char* from[LOADS];
    int32_t key[LOADS];
  };
  // Chunks lie in LDS in the order of the lanes that bring them, so a lane finds its key from
  // the place: the inverse of Staged's.
  static __device__ __forceinline__ Lane lane_of(const char* k, const char* v, int wave, int lane) {
    Lane r;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int32_t at = (wave + i * kWaves) * kWave + lane, place = at / OF_KEY % KEYS;
      r.key[i] = (place & 16) >> 2 | (place & 12) << 1 | (place & 3);
      r.from[i] = (at < KEYS * OF_KEY ? k : v) + at % OF_KEY * 16;
    }
    return r;
  }
  static __device__ __forceinline__ void bring(Tile& tile, const Lane& lane, int wave,
                                               const int64_t* rows) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int n = wave + i * kWaves;
      if ((i + 1) * kWaves > OF_KEY && n >= OF_KEY) break;   // the same for a whole wave
      bring16<true>(lane.from[i] + rows[lane.key[i]],
                    reinterpret_cast<u32x4*>(tile.k) + n * kWave);
    }
  }
  // As Staged's, of a head.
  template <int BYTES>
  static __device__ __forceinline__ Words<(BYTES + 3) / 4> codes(const char* tile, int32_t place,
                                                                 int32_t head, int32_t d0) {
    Words<(BYTES + 3) / 4> r;
    r.w[(BYTES - 1) / 4] = 0;
    __builtin_memcpy(&r, __builtin_assume_aligned(tile + place * PITCH + head * RECORD +
                                                  code_bytes<C>(d0), BYTES < 4 ? BYTES : 4), BYTES);
    return r;
  }
  static __device__ __forceinline__ float scale(const char* tile, int32_t place, int32_t head,
                                                int32_t d0) {
    return scale_of(static_cast<uint8_t>(tile[place * PITCH + head * RECORD + CODES +
                                              d0 / kGroup]), 0);
  }
};

// What bounds it is the cache's stream: each wave has a step's K or V (64 keys; 32 of 32-bit
// caches) in flight at any time, straight into the registers the products read, and nothing
// but block ids passes through LDS (of microscaled caches the records do, see above). A
// workgroup takes 1, 2 or 4 neighbouring KV heads: its waves go through the same keys, whose
// rows are neighbours in memory, and waves of the same head take steps in turn and join at the
// end. 64 sequences of 16,000 tokens of eight bf16 heads of 128: 5.45 TB/s with four waves on
// one head, 5.95 with one on each of four, 6.3 with loads that pass the caches by besides (an
// 8-bit cache 4.7, 5.0 and 5.7). Of a pair of key tiles (32 keys), lane group g = lane / 16
// holds the weights of keys 8 g .. 8 g + 7: a lane loads those keys' V, EV dimensions each,
// and turns them in its own registers into the EV operands of V^T (dimension c EV + t at place
// c of tile t).
//
// 16-bit operands hold a weight as two, its value rounded to the type and what that leaves:
// together off by 2^-16 (bf16) of it, as good as 32 bits beside V's own. The second product is
// hidden behind the stream: 48 sequences of about 6,000 tokens of eight bf16 heads, in a window
// of 4,096, 129.9 us against 130.1 with the rounded weights alone, one of 16,384 on an 8-bit
// cache, in one of 12,000, 16.0 against 15.7.
template <typename T, typename C, int DP>
struct Narrow {
  static constexpr int EK = sizeof(T) == 4 ? 4 : 8;       // K elements a lane feeds at a time
  // and brings at a time: 16 bytes, so that the four lanes of a key read 64 bytes on end
  static constexpr int EL = 128 / kBits<C> * 4 <= DP ? 128 / kBits<C> : DP / 4;
  static constexpr int NL = (DP + 4 * EL - 1) / (4 * EL), MF = EL / EK, NK = NL * MF;
  static constexpr int EV = DP <= 32 ? 2 : DP <= 64 ? 4 : 8;
  static constexpr int KT = kBits<C> == 32 ? 2 : 4;       // key tiles of 16 in a step
  static constexpr int KS = 16 * KT;
  static constexpr float LIFT = lift<T>(14.f);
  using RawK = Words<EL * kBits<C> / 32>;
  using RawV = Words<(EV * kBits<C> / 8 + 3) / 4>;
  static constexpr int LDO = DP + 4;                      // floats of a row of o in LDS
  struct Lds {
    alignas(16) int64_t rows[kWaves][2][KS];              // bytes to the keys' rows
    float2 ml[kWaves][16];
    union {
      alignas(16) float o[kWaves][16][LDO];
      Staged<C, DP> staged[kScaled<C> ? kWaves : 1];      // until the last step
    };
    int32_t redo[kWaves];
  };
  struct Rows {                                           // of heads taken together
    int64_t rows[kWaves][2][Together<C, DP>::KEYS];
  };
};

// The rows of a head that a wave has to itself: a lane holds EV dimensions on end of row c at a
// time (of `o`: dimension (4 g + r) EV + t at o[t][r]).
template <typename T, typename C, int DP>
__device__ __forceinline__ void write_head(const Args& a, const Item& it, int32_t kv_head,
                                           int32_t head0, int32_t heads, int32_t rows,
                                           const f32x4 (&o)[Narrow<T, C, DP>::EV], float m, float l,
                                           int lane) {
  constexpr int EV = Narrow<T, C, DP>::EV;
  const int32_t g = lane / 16, c = lane % 16;
  bool odd = l != l || is_far(m);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < EV; ++t) odd = odd || ((g * 4 + r) * EV < DP && o[t][r] != o[t][r]);
  // Nothing is written where rows are done again: the output may lie where their queries do.
  if (__any(odd && c < rows)) {
    for (int32_t r = 0; r < rows; ++r)
      attend_row<T, C>(a, it, kv_head, r / heads * a.group + head0 + r % heads, lane);
    return;
  }
  if (c >= rows) return;
  const int32_t token = c / heads, in_group = head0 + c % heads;
  const int64_t slot =
      static_cast<int64_t>(it.slot + token * a.group + in_group) * a.kv_heads + kv_head;
  const int64_t at = (it.token0 + token) * static_cast<int64_t>(a.kv_heads) * a.group +
                     static_cast<int64_t>(kv_head) * a.group + in_group;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int32_t d0 = (g * 4 + r) * EV;
    if (d0 >= DP) break;
    float x[EV];
#pragma unroll
    for (int t = 0; t < EV; ++t) x[t] = it.slot >= 0 ? o[t][r] : o[t][r] / l;
    if (it.slot >= 0)
      __builtin_memcpy(a.part_o + slot * DP + d0, x, EV * 4);
    else
      store_out<T, EV>(static_cast<T*>(a.out) + at * DP + d0, x);
  }
  if (it.slot >= 0 && g == 0) a.part_ml[slot] = {m, l};
}

// A group of more than 16 heads takes several workgroups for each of its tokens, `head0` on.
// TOGETHER: four KV heads of a microscaled cache, of DP dimensions each; their records come into
// two `tiles`.
template <typename T, typename C, int DP, bool TOGETHER, typename Lds>
__device__ __forceinline__ void narrow_item(Lds& lds, typename Together<C, DP>::Tile* tiles,
                                            const Args& a, int32_t item, int32_t kv_head0,
                                            int32_t head0) {
  using N = Narrow<T, C, DP>;
  constexpr int EK = N::EK, EL = N::EL, NL = N::NL, MF = N::MF, NK = N::NK;
  constexpr int EV = N::EV, KS = TOGETHER ? Together<C, DP>::KEYS : N::KS, KT = KS / 16;
  const Item it = item_of(a, item);
  const int32_t heads = a.group - head0 < 16 ? a.group - head0 : 16;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, g = lane / 16, c = lane % 16;
  const int32_t together = TOGETHER ? kWaves : a.together, turns = kWaves / together;
  const int32_t kv_head = kv_head0 + wave % together, turn = wave / together;
  const int32_t d = a.head_dim, rows = it.tokens * heads;
  const int32_t n = (it.a1 - it.a0) + (it.b1 - it.b0), steps = (n + KS - 1) / KS;
  const int32_t size = head_bytes<C>(d);
  const int64_t row_bytes = static_cast<int64_t>(a.kv_heads) * size;
  if constexpr (!TOGETHER) {
    if (threadIdx.x < kWaves) lds.redo[threadIdx.x] = 0;
  }

  // Q^T: row c, zeros past the rows and past the dimensions.
  Words<4> q[NK];
  int32_t position;
  {
    const int32_t row = c < rows ? c : 0, token = it.token0 + row / heads;
    const int64_t head = static_cast<int64_t>(kv_head) * a.group + head0 + row % heads;
    position = a.words[a.positions_at + token];
    const T* at = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int32_t d0 = (4 * (i / MF) + g) * EL + i % MF * EK;
      const bool in = c < rows && d0 < d;
      q[i] = load_bytes<EK * sizeof(T)>(at + (d0 < d ? d0 : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) q[i].w[e] = (q[i].w[e] ^ a.q_sign) & (in ? ~0u : 0u);
    }
  }
  const char* kc = static_cast<const char*>(a.k) + static_cast<int64_t>(kv_head) * size;
  const char* vh = static_cast<const char*>(a.v) + static_cast<int64_t>(kv_head) * size;
  const char* vc = vh + code_bytes<C>(c * EV < d ? c * EV : 0);

  const auto place = [&](int32_t s) {
    const int32_t v = s * KS + lane % KS;
    return place_of(a, it, key_at(it, v < n ? v : n - 1));
  };
  const auto keep = [&](int half, Place p) {
    if (lane < KS) lds.rows[wave][half][lane] = row_of(a, p) * row_bytes;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  typename N::RawK k[kScaled<C> ? 1 : KT][NL];
  // Of microscaled caches: what a lane brings of a step's records, K's and V's.
  using G = Together<C, DP>;
  using S = Staged<C, DP>;
  static_assert(!kScaled<C> || KS == (TOGETHER ? G::KEYS : S::KEYS));
  typename G::Lane brings_all;
  typename S::Lane brings;
  typename S::Chunk k_chunks[kScaled<C> ? S::CHUNKS : 1], v_chunks[kScaled<C> ? S::CHUNKS : 1];
  if constexpr (TOGETHER) {
    brings_all = G::lane_of(kc - wave * size, vh - wave * size, wave, lane);
  } else if constexpr (kScaled<C>) {
    brings = S::lane_of(lane, d);
    if (d < DP) lds.staged[wave].clear(lane);
  }
  const auto load_k = [&](int half) {
    if constexpr (kScaled<C>) {
      S::load(k_chunks, brings, kc, lds.rows[wave][half]);
    } else {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const char* at =
            kc + lds.rows[wave][half][t / 2 * 32 + (c >> 2) * 8 + t % 2 * 4 + (c & 3)];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int32_t d0 = (4 * i + g) * EL;
          // 16 elements past the head's end would be past the cache's at its last row.
          const int32_t from = d0 >= d ? 0 : EL == 16 && d0 + 8 == d ? d0 - 8 : d0;
          k[t][i] = stream_bytes<code_bytes<C>(EL)>(at + code_bytes<C>(from));
        }
      }
    }
  };
  // Loads end behind 96 dimensions.
  const auto within = [](int32_t d0) { return d0 < DP ? d0 : 0; };
  using Tile = typename G::Tile;
  const auto k_of = [&](const Tile* tile, int t, int i) {
    const int32_t d0 = within((4 * i + g) * EL);
    if constexpr (TOGETHER)
      return G::template codes<code_bytes<C>(EL)>(tile->k, t * 16 + c, wave, d0);
    else if constexpr (kScaled<C>)
      return lds.staged[wave].template codes<code_bytes<C>(EL)>(t * 16 + c, d0);
    else
      return k[t][i];
  };
  const auto k_scale = [&](const Tile* tile, int t, int32_t d0) {
    if constexpr (TOGETHER)
      return G::scale(tile->k, t * 16 + c, wave, d0);
    else
      return lds.staged[wave].scale(t * 16 + c, d0);
  };

  // The elements of feed `e` of a load; zeros past the head's dimensions. Not where they are
  // loaded, or they would be waited for there.
  constexpr int KW = (EK * kBits<C> / 8 + 3) / 4;
  const auto feed = [&](const typename N::RawK& x, int i, int e) {
    Words<KW> r;
    if constexpr (kScaled<C>) {
#pragma unroll
      for (int w = 0; w < KW; ++w) r.w[w] = x.w[e * EK * kBits<C> / 32 + w];
      if (EK * kBits<C> < 32) r.w[0] >>= e * EK * kBits<C> % 32;
      return r;
    }
    const int32_t d0 = (4 * i + g) * EL + e * EK;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      r.w[w] = x.w[e * KW + w];
      if ((i + 1) * 4 * EL > DP - 32) {
        if (EL == 16 && e * EK < 8 && d0 - e * EK + 8 == d) r.w[w] = x.w[(e * EK + 8) / 4 + w];
        r.w[w] &= d0 < d ? ~0u : 0u;
      }
    }
    return r;
  };

  f32x4 o[EV];
#pragma unroll
  for (int t = 0; t < EV; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;                 // l: of the lane's own keys

  Place next{0, 0};
  if (turn < steps) {
    const Place now = place(turn);
    next = place(turn + turns);                 // before K's loads: see below
    keep(0, now);
    if constexpr (TOGETHER) {
      G::bring(tiles[0], brings_all, wave, lds.rows[wave][0]);
      arrive();
    } else {
      load_k(0);
    }
  }
  // Step s, whose rows are in `half`. Of heads taken together its records are in `tile`, and the
  // next one's go to `after`, which the compiler has to know to be another: it would wait for
  // loads into LDS before it reads there.
  const auto step = [&](int32_t s, int half, const Tile* __restrict tile, Tile* __restrict after) {
    keep(half ^ 1, next);
    typename N::RawV v[KT / 2][kScaled<C> ? 1 : 8];
    if constexpr (TOGETHER) {
      next = place(s + 2);
      if (s + 1 < steps) G::bring(*after, brings_all, wave, lds.rows[wave][half ^ 1]);
    } else if constexpr (kScaled<C>) {
      S::load(v_chunks, brings, vh, lds.rows[wave][half]);
      __builtin_amdgcn_sched_barrier(0);
      lds.staged[wave].put(k_chunks, brings, d);
    } else {
#pragma unroll
      for (int p = 0; p < KT / 2; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[p][e] = stream_bytes<EV * kBits<C> / 8>(vc + lds.rows[wave][half][p * 32 + g * 8 + e]);
    }
    __builtin_amdgcn_sched_barrier(0);          // no wait for K's before V's are on their way
    f32x4 sc[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const typename N::RawK whole = k_of(tile, t, i);
#pragma unroll
        for (int e = 0; e < MF; ++e) {
          const auto raw = feed(whole, i, e);
          if constexpr (kScaled<C>)
            sc[t] = mma16(
                scaled<T, C, EK>(raw, k_scale(tile, t, within((4 * i + g) * EL) + e * EK)),
                q[i * MF + e], sc[t], T{});
          else
            sc[t] = mma16(Convert<T, C, EK>::of(raw), q[i * MF + e], sc[t], T{});
        }
      }
    }
    // In this order: loads return in theirs, and the block's id is what is needed first. Past
    // the last step these read the last key: a branch would make the next wait one for all.
    if constexpr (!TOGETHER) {
      next = place(s + 2 * turns);
      load_k(half ^ 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    // V of key `e` of the lane's eight of pair `p`, as the type of `as`.
    const auto v_of = [&](auto as, int p, int e) {
      if constexpr (kScaled<C>) {
        const int32_t at = p * 32 + e / 4 * 16 + g * 4 + e % 4, d0 = within(c * EV);
        if constexpr (TOGETHER)
          return scaled<decltype(as), C, EV>(
              G::template codes<EV * kBits<C> / 8>(tile->v, at, wave, d0),
              G::scale(tile->v, at, wave, d0));
        else
          return scaled<decltype(as), C, EV>(
              lds.staged[wave].template codes<EV * kBits<C> / 8>(at, d0),
              lds.staged[wave].scale(at, d0));
      } else {
        return Convert<T, C, EV>::of(v[p][e]);
      }
    };

    const int32_t v0 = s * KS;
    if (v0 + KS > n || !all_see(a, it, v0, v0 + KS)) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int32_t at = v0 + t / 2 * 32 + g * 8 + t % 2 * 4 + r;
          if (at >= n || !sees(a, position, key_at(it, at))) sc[t][r] = -INFINITY;
        }
    }
    float top = m;
    {
      float x = -INFINITY;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) x = fmaxf(x, sc[t][r]);
      x = fmaxf(x, lane_xor<16>(x));
      x = fmaxf(x, lane_xor<32>(x));
      top = fmaxf(m, x * a.scale - N::LIFT);
    }
    const float base = top == -INFINITY ? 0.f : top;
    if (__any(top > m)) {
      const float fade = power2(m - base);
      l *= fade;
#pragma unroll
      for (int t = 0; t < EV; ++t) o[t] *= fade;
      m = top;
    }
    float p[KT][4];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[t][r] = power2(fmaf(sc[t][r], a.scale, -base));
        l += p[t][r];
      }
    if constexpr (kScaled<C> && !TOGETHER) lds.staged[wave].put(v_chunks, brings, d);
#pragma unroll
    for (int pr = 0; pr < KT / 2; ++pr) {
      if constexpr (sizeof(T) == 4) {
        Words<EV> x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v_of(T{}, pr, e);
#pragma unroll
        for (int t = 0; t < EV; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x[e].w[t]),
                                                        p[2 * pr + e / 4][e % 4], o[t], 0, 0, 0);
      } else {
        // Integers become floats first, which two keys at a time are rounded to where V^T has them;
        // the others come as words of two dimensions, which change places with another key's.
        constexpr bool BY_KEY = std::is_same_v<C, Mxint8>;
        Words<4> by_key[BY_KEY ? EV : 1];
        Words<EV / 2> x[BY_KEY ? 1 : 8];
        if constexpr (BY_KEY) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const Words<EV> v0 = v_of(0.f, pr, 2 * i), v1 = v_of(0.f, pr, 2 * i + 1);
#pragma unroll
            for (int t = 0; t < EV; ++t)
              by_key[t].w[i] = pack2<T>(__builtin_bit_cast(float, v0.w[t]),
                                        __builtin_bit_cast(float, v1.w[t]));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = v_of(T{}, pr, e);
        }
        Words<4> w, rest;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = p[2 * pr + i / 2][i % 2 * 2], p1 = p[2 * pr + i / 2][i % 2 * 2 + 1];
          w.w[i] = pack2<T>(p0, p1);
          rest.w[i] = rest2<T>(p0, p1, w.w[i]);
        }
#pragma unroll
        for (int t = 0; t < EV; ++t) {
          Words<4> vt;                          // dimension c EV + t of keys 8 g ..
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if constexpr (BY_KEY)
              vt.w[i] = by_key[t].w[i];
            else
              vt.w[i] = __builtin_amdgcn_perm(x[2 * i + 1].w[t / 2], x[2 * i].w[t / 2],
                                              t % 2 ? 0x07060302u : 0x05040100u);
          o[t] = mma16(vt, rest, mma16(vt, w, o[t], T{}), T{});
        }
      }
    }
    if constexpr (TOGETHER) arrive();
  };
  int half = 0;
  for (int32_t s = turn; s < steps; s += turns, half ^= 1)
    step(s, half, TOGETHER ? tiles + half : nullptr, TOGETHER ? tiles + (half ^ 1) : nullptr);

  l += lane_xor<16>(l);
  l += lane_xor<32>(l);
  if constexpr (TOGETHER) {
    write_head<T, C, DP>(a, it, kv_head, head0, heads, rows, o, m, l, lane);
  } else {
    if (lane < 16) lds.ml[wave][lane] = {m, l};
    __syncthreads();
    float all = -INFINITY;
    for (int w = wave % together; w < kWaves; w += together) all = fmaxf(all, lds.ml[w][c].x);
    const float fade = power2(m - (all == -INFINITY ? 0.f : all));
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < EV; ++t)
        if ((g * 4 + r) * EV + t < DP) lds.o[wave][c][(g * 4 + r) * EV + t] = o[t][r] * fade;
    __syncthreads();
    // Eight dimensions of a row a thread, of each head.
    const int32_t row = threadIdx.x / 16, d0 = threadIdx.x % 16 * 8;
    const int32_t in_group = head0 + row % heads, token = row / heads;
    const bool mine = row < rows && d0 < d;
    float x[kWaves][8];
    float2 ml[kWaves];
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      if (!mine || k >= together) break;
      float total = 0.f, most = -INFINITY;
      for (int w = k; w < kWaves; w += together) most = fmaxf(most, lds.ml[w][row].x);
      const float from = most == -INFINITY ? 0.f : most;
      for (int w = k; w < kWaves; w += together)
        total = fmaf(lds.ml[w][row].y, power2(lds.ml[w][row].x - from), total);
      ml[k] = {most, total};
      bool odd = total != total || is_far(most);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k][i] = lds.o[k][row][d0 + i];
      for (int w = k + together; w < kWaves; w += together)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] += lds.o[w][row][d0 + i];
#pragma unroll
      for (int i = 0; i < 8; ++i) odd = odd || x[k][i] != x[k][i];
      if (odd) lds.redo[k] = 1;
    }
    __syncthreads();
    // Nothing is written of a head whose rows are done again: the output may lie where their
    // queries do.
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      if (!mine || k >= together) break;
      if (lds.redo[k]) continue;
      const int64_t kv = kv_head0 + k;
      if (it.slot >= 0) {
        const int64_t slot =
            static_cast<int64_t>(it.slot + token * a.group + in_group) * a.kv_heads + kv;
        __builtin_memcpy(a.part_o + slot * d + d0, x[k], 32);
        if (d0 == 0) a.part_ml[slot] = ml[k];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] /= ml[k].y;
        const int64_t at = (it.token0 + token) * static_cast<int64_t>(a.kv_heads) * a.group +
                           kv * a.group + in_group;
        store_out<T, 8>(static_cast<T*>(a.out) + at * d + d0, x[k]);
      }
    }
    for (int k = 0; k < together; ++k) {
      if (!lds.redo[k]) continue;
      for (int32_t r = wave; r < rows; r += kWaves)
        attend_row<T, C>(a, it, kv_head0 + k, r / heads * a.group + head0 + r % heads, lane);
    }
  }
}

// --- wide: many rows ---------------------------------------------------------------------

// Four waves, 32 rows each, share tiles of 64 keys in LDS, two tiles in turn: a tile's
// loads are issued before the products of the one before it. V^T is read from V's rows by the
// transposing LDS load (a group of 16 lanes reads 4 keys of 16 dimensions, and each lane gets
// one dimension of the four). A tile lies in LDS without gaps, so that the loads can go there
// directly (DIRECT; 8-bit caches are converted on their way, and caches that begin at any
// element are copied through registers); its rows' 16-byte chunks change places by key, so
// that the 256 bytes that are read at a time lie in different banks: a chunk of K of 16 keys
// each, four chunks of V of four keys each. A prompt of 7,777 tokens in a window of 4,096, 32
// bf16 heads of 128: 398-406 us by the box, 950-965 TFLOP/s, the matrix units busy for 46% of the
// cycles and the vector units for 48%: two waves to a SIMD, one with its products and one with
// its weights. Scoring a tile while the one before is weighted in the same wave was 3-12% slower.
//
// Weights are rounded to the queries' type, by at most half a step of it each: an output is off
// by no more than that of the mean of |v|, as it is by its own rounding. The remainders' product
// that narrow items add is not hidden here: that prompt took 519 us with it, 398 without, three
// chunks of 555 fp16 tokens 16.2 against 14.4. Over microscaled caches it is added all the same,
// so that a chunk is as near to 64 bits as single tokens are and as weights of 32 bits would be:
// 2,048 tokens at the end of 7,777 off by 0.0017 of the output in bf16, 0.0023 with the rounded
// weights alone, and 330 us against 256 (mxfp8, the same box).
template <typename T, int DP>
struct Wide {
  static constexpr int KS = 64;
  static constexpr int CHUNKS = DP / 8;                      // of eight elements, a row's
  // Dimensions that a thread brings at a time, and how often for a tile.
  template <typename C>
  static constexpr int EACH = kScaled<C> && DP > 32 ? 16 : 8;
  template <typename C>
  static constexpr int LOADS = (KS * DP / EACH<C> + kThreads - 1) / kThreads;
  static constexpr float LIFT = lift<T>(7.f);
  // The place of a chunk, and the chunk at a place.
  static __device__ __forceinline__ int place_k(int key, int chunk) {
    return chunk ^ (DP == 128 ? key & 15 : DP == 64 ? key >> 1 & 7 : key >> 2 & 3);
  }
  static __device__ __forceinline__ int place_v(int key, int chunk) {
    return chunk ^ (DP == 128 ? (key & 3) * 4 : DP == 64 ? (key >> 1 & 1) * 4 : 0);
  }
  using Tile = u32x4[KS * CHUNKS];
  using Rows = int64_t[2][KS];                               // bytes to the keys' rows
  struct Lds {
    Tile k[2], v[2];
    Rows rows;
    int32_t redo;
  };
};

__device__ __forceinline__ Words<2> transposed(const char* lds) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      Words<2>, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4*)const_cast<char*>(lds)));
}

// K's and V's buffers are arguments of their own: the compiler then knows that a load into one
// leaves the others alone, and does not wait for it before it reads them.
template <typename T, typename C, int DP, bool DIRECT>
__device__ __forceinline__ void wide_item(typename Wide<T, DP>::Tile& k0,
                                          typename Wide<T, DP>::Tile& k1,
                                          typename Wide<T, DP>::Tile& v0,
                                          typename Wide<T, DP>::Tile& v1,
                                          typename Wide<T, DP>::Rows& lds_rows, int32_t& redo,
                                          const Args& a, int32_t item, int32_t kv_head) {
  using W = Wide<T, DP>;
  constexpr int KS = W::KS, CHUNKS = W::CHUNKS;
  constexpr int NQ = DP / 16, ND = DP / 32;
  const Item it = item_of(a, item);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, h = lane / 32, c = lane % 32;
  const int32_t d = a.head_dim, rows = it.tokens * a.group;
  const int32_t n = (it.a1 - it.a0) + (it.b1 - it.b0), steps = (n + KS - 1) / KS;
  if (threadIdx.x == 0) redo = 0;

  // Q^T: row `mine`, zeros past the rows and past the dimensions.
  const int32_t mine = wave * 32 + c;
  Words<4> q[NQ];
  int32_t position;
  {
    const int32_t row = mine < rows ? mine : 0, token = it.token0 + row / a.group;
    const int64_t head = static_cast<int64_t>(kv_head) * a.group + row % a.group;
    position = a.words[a.positions_at + token];
    const T* at = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int32_t d0 = i * 16 + h * 8;
      const bool in = mine < rows && d0 < d;
      q[i] = load_bytes<16>(at + (d0 < d ? d0 : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) q[i].w[e] = (q[i].w[e] ^ a.q_sign) & (in ? ~0u : 0u);
    }
  }

  const int32_t size = head_bytes<C>(d);
  const int64_t row_bytes = static_cast<int64_t>(a.kv_heads) * size;
  const char* kc = static_cast<const char*>(a.k) + static_cast<int64_t>(kv_head) * size;
  const char* vc = static_cast<const char*>(a.v) + static_cast<int64_t>(kv_head) * size;
  const auto place = [&](int32_t s) {
    const int32_t v = s * KS + lane;
    return place_of(a, it, key_at(it, v < n ? v : n - 1));
  };
  // The thread's chunks of a tile. Chunks past the head's dimensions hold its first ones: Q is
  // zero there, and nothing of V there is written.
  using Raw = Words<W::template EACH<C> * kBits<C> / 32>;
  constexpr int EACH = W::template EACH<C>, LOADS = W::template LOADS<C>;
  struct Held {
    Raw k[LOADS], v[LOADS];
    uint32_t k_scales[LOADS], v_scales[LOADS];   // of microscaled caches
  };
  // Of microscaled caches 16 dimensions at a time, for the places of the dimensions from `to` on.
  // Where only eight are left, those and the eight before them: they change places, so that the
  // place behind them holds the latter.
  struct Part {
    int32_t key, from, to;
    bool turned;
  };
  const auto part = [&](int i) {
    constexpr int all = KS * DP / EACH;
    const int32_t n = threadIdx.x + i * kThreads, at = n < all ? n : all - 1;
    const int32_t d0 = at % (DP / EACH) * EACH;
    const bool turned = d0 < d && d < d0 + EACH;
    return Part{at / (DP / EACH), turned ? d - EACH : d0 < d ? d0 : 0, d0, turned};
  };
  const auto load = [&](int64_t (&row)[KS], typename W::Tile& kt, typename W::Tile& vt, Held& x) {
    if constexpr (kScaled<C>) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const Part p = part(i);
        const int64_t from = row[p.key];
        x.k[i] = load_bytes<code_bytes<C>(EACH)>(kc + from + code_bytes<C>(p.from));
        x.v[i] = load_bytes<code_bytes<C>(EACH)>(vc + from + code_bytes<C>(p.from));
        x.k_scales[i] = load_bytes<kScaleBytes>(kc + from + code_bytes<C>(d)).w[0];
        x.v_scales[i] = load_bytes<kScaleBytes>(vc + from + code_bytes<C>(d)).w[0];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int32_t at = threadIdx.x + i * kThreads, key = at / CHUNKS, to = at % CHUNKS;
      const int32_t dk = W::place_k(key, to) * 8, dv = W::place_v(key, to) * 8;
      const int64_t from = row[key];
      const char* ks = kc + from + (dk < d ? dk : 0) * sizeof(C);
      const char* vs = vc + from + (dv < d ? dv : 0) * sizeof(C);
      if constexpr (DIRECT) {
        const int32_t first = wave * kWave + i * kThreads;       // lane l's goes l places on
        bring16(ks, &kt[first]);
        bring16(vs, &vt[first]);
      } else if constexpr (!kScaled<C>) {
        x.k[i] = load_bytes<8 * sizeof(C)>(ks);
        x.v[i] = load_bytes<8 * sizeof(C)>(vs);
      }
    }
  };
  const auto store = [&](const Held& x, typename W::Tile& kt, typename W::Tile& vt) {
    if constexpr (kScaled<C>) {
      using Eight = Words<kBits<C> / 4>;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const Part p = part(i);
#pragma unroll
        for (int e = 0; e < EACH; e += 8) {
          Eight k8, v8;
          __builtin_memcpy(&k8, &x.k[i].w[e * kBits<C> / 32], sizeof(Eight));
          __builtin_memcpy(&v8, &x.v[i].w[e * kBits<C> / 32], sizeof(Eight));
          const int32_t shift = (p.from + e) / kGroup * 8;
          const int32_t chunk = (p.to + (p.turned ? EACH - 8 - e : e)) / 8;
          kt[p.key * CHUNKS + W::place_k(p.key, chunk)] = __builtin_bit_cast(
              u32x4, scaled<T, C, 8>(k8, scale_of(x.k_scales[i], shift)));
          vt[p.key * CHUNKS + W::place_v(p.key, chunk)] = __builtin_bit_cast(
              u32x4, scaled<T, C, 8>(v8, scale_of(x.v_scales[i], shift)));
        }
      }
    } else if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int32_t at = threadIdx.x + i * kThreads;
        kt[at] = __builtin_bit_cast(u32x4, Convert<T, C, 8>::of(x.k[i]));
        vt[at] = __builtin_bit_cast(u32x4, Convert<T, C, 8>::of(x.v[i]));
      }
    }
  };

  f32x16 o[ND];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;

  if (wave < 2) lds_rows[wave][lane] = row_of(a, place(wave)) * row_bytes;
  __syncthreads();
  {
    Held x;
    load(lds_rows[0], k0, v0, x);
    store(x, k0, v0);
  }
  arrive();
  // Tile s, in `kt` and `vt`; the next one goes to `kn` and `vn`.
  const auto step = [&](int32_t s, int half, typename W::Tile& kt, typename W::Tile& vt,
                        typename W::Tile& kn, typename W::Tile& vn) {
    // No branch around these loads, or every wait after them would be one for all: past the
    // last step they read the last key.
    const Place next = place(s + 2);
    Held held;
    load(lds_rows[half ^ 1], kn, vn, held);
    __builtin_amdgcn_sched_barrier(0);

    f32x16 sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[t][r] = 0.f;
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Words<4> k = __builtin_bit_cast(
            Words<4>, kt[(t * 32 + c) * CHUNKS + W::place_k(c, i * 2 + h)]);
        sc[t] = mma32(k, q[i], sc[t], T{});
      }
    // Half of K's reads at once, then one behind each product: left to itself the compiler
    // waits for every read before its product.
    constexpr int kDsRead = 0x100, kMfma = 0x8;
    __builtin_amdgcn_sched_group_barrier(kDsRead, NQ, 0);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMfma, NQ, 0);

    const int32_t first = s * KS;
    if (first + KS > n || !all_see(a, it, first, first + KS)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t at = first + t * 32 + r / 4 * 8 + h * 4 + r % 4;
          const bool seen = (at < n) & sees(a, position, key_at(it, at));
          sc[t][r] = seen ? sc[t][r] : -INFINITY;
        }
    }
    float x = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) x = fmaxf(x, sc[t][r]);
    // The maximum that weights are taken relative to follows only when a row's has grown by a
    // factor of 2^8: weights, their sum and O are floating point and as exact relative to any
    // of them, and of 32 rows one or another would grow at almost every tile.
    const float top = fmaxf(x, lane_xor<32>(x)) * a.scale - W::LIFT;
    if (__any(top > m + 8.f)) {
      const float to = fmaxf(m, top), fade = to == -INFINITY ? 1.f : power2(m - to);
      l *= fade;
#pragma unroll
      for (int t = 0; t < ND; ++t) o[t] *= fade;
      m = to;
    }
    const float base = m == -INFINITY ? 0.f : m;
    Words<4> p[4], rest[kScaled<C> ? 4 : 1];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = power2(fmaf(sc[t][r], a.scale, -base));
        const float p1 = power2(fmaf(sc[t][r + 1], a.scale, -base));
        l += p0 + p1;
        const uint32_t w = pack2<T>(p0, p1);
        p[t * 2 + r / 8].w[r % 8 / 2] = w;
        if constexpr (kScaled<C>) rest[t * 2 + r / 8].w[r % 8 / 2] = rest2<T>(p0, p1, w);
      }
    // Of 16 keys, half h holds the weights of 4 h .. 4 h + 3 and 8 + 4 h ..
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        const int key = i * 16 + h * 4 + c % 16 / 4, chunk = t * 4 + c / 16 * 2 + c % 4 / 2;
        const char* at = reinterpret_cast<const char*>(&vt[key * CHUNKS + W::place_v(key, chunk)]) +
                         c % 2 * 8;
        const Words<2> lo = transposed(at), hi = transposed(at + 8 * CHUNKS * 16);
        const Words<4> vt{{lo.w[0], lo.w[1], hi.w[0], hi.w[1]}};
        if constexpr (kScaled<C>) o[t] = mma32(vt, rest[i], o[t], T{});
        o[t] = mma32(vt, p[i], o[t], T{});
      }
    __builtin_amdgcn_sched_barrier(0);
    store(held, kn, vn);
    if (wave == 0) lds_rows[half][lane] = row_of(a, next) * row_bytes;
    arrive();
  };
  for (int32_t s = 0;;) {
    step(s, 0, k0, v0, k1, v1);
    if (++s >= steps) break;
    step(s, 1, k1, v1, k0, v0);
    if (++s >= steps) break;
  }

  l += lane_xor<32>(l);
  bool odd = l != l || is_far(m);
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = odd || (t * 32 + r / 4 * 8 < d && o[t][r] != o[t][r]);
  if (odd && mine < rows) redo = 1;
  __syncthreads();
  if (redo) {
    for (int32_t r = wave; r < rows; r += kWaves) attend_row<T, C>(a, it, kv_head, r, lane);
    return;
  }
  if (mine >= rows) return;
  const int64_t token = it.token0 + mine / a.group;
  const int64_t head = static_cast<int64_t>(kv_head) * a.group + mine % a.group;
  const int64_t slot = static_cast<int64_t>(it.slot + mine) * a.kv_heads + kv_head;
  T* out = static_cast<T*>(a.out) + (token * static_cast<int64_t>(a.kv_heads) * a.group + head) * d;
  const float inverse = 1.f / l;
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int32_t d0 = t * 32 + r * 2 + h * 4;
      if (d0 >= d) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = it.slot >= 0 ? o[t][r + e] : o[t][r + e] * inverse;
      if (it.slot >= 0)
        __builtin_memcpy(a.part_o + slot * d + d0, x, 16);
      else
        store_out<T, 4>(out + d0, x);
    }
  if (it.slot >= 0 && h == 0) a.part_ml[slot] = {m, l};
}

// --- kernels -----------------------------------------------------------------------------

// A block is one or more KV heads of an item. Blocks go to the XCDs in turn: the ones of a
// narrow item, which read neighbouring rows of the cache, go to the same one.
template <typename T, typename C, int DP, bool TOGETHER>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && DP > 64 ? 1 : 2) void attend_narrow(
    Args a, int32_t first, int32_t n) {
  using N = Narrow<T, C, DP>;
  constexpr int kXcds = 8;
  const int32_t each = a.kv_heads / a.together, b = blockIdx.x;
  const bool whole = b < n / kXcds * kXcds * each;
  const int32_t item = whole ? b / kXcds / each * kXcds + b % kXcds : b / each;
  const int32_t part = whole ? b / kXcds % each : b % each;
  const int32_t kv_head0 = part * a.together, head0 = blockIdx.y * 16;
  if constexpr (TOGETHER) {
    __shared__ typename Together<C, DP>::Tile tiles[2];
    __shared__ typename N::Rows rows;
    narrow_item<T, C, DP, true>(rows, tiles, a, first + item, kv_head0, head0);
  } else {
    extern __shared__ __attribute__((aligned(16))) char shared[];
    narrow_item<T, C, DP, false>(*reinterpret_cast<typename N::Lds*>(shared), nullptr, a,
                                 first + item, kv_head0, head0);
  }
}

constexpr int kWideRows = kWaves * 32;

// Wide items from `wide` on, of 16-bit caches at 16-byte addresses, whose tiles come into LDS
// directly, and of microscaled ones. Neighbouring blocks are the
// heads of an item, and where there are eight, all blocks of an XCD are of one head, whose
// keys the items share in its L2.
template <typename T, typename C, int DP>
__global__ __launch_bounds__(kThreads, 2) void attend_wide(Args a, int32_t wide) {
  using W = Wide<T, DP>;
  __shared__ typename W::Tile k0, k1, v0, v1;
  __shared__ typename W::Rows rows;
  __shared__ int32_t redo;
  wide_item<T, C, DP, !kScaled<C>>(k0, k1, v0, v1, rows, redo, a, wide + blockIdx.x / a.kv_heads,
                                   blockIdx.x % a.kv_heads);
}

// `n_wide` wide items from `wide` on and `n_narrow` narrow ones from `narrow` on in one launch:
// the matrix units work on the former while the latter wait for memory.
template <typename T, typename C, int DP>
__global__ __launch_bounds__(kThreads, 2) void attend_both(
    Args a, int32_t wide, int32_t n_wide, int32_t narrow, int32_t n_narrow) {
  extern __shared__ __attribute__((aligned(16))) char shared[];
  auto& of_wide = *reinterpret_cast<typename Wide<T, DP>::Lds*>(shared);
  // Runs of as many blocks as a narrow item has; a wide item is `together` such runs. Those
  // of the wide items come at even distances among the first three quarters.
  const uint32_t each = a.kv_heads / a.together, run = blockIdx.x / each, part = blockIdx.x % each;
  const uint32_t wides = n_wide * a.together, runs = wides + n_narrow;
  const uint32_t span = wides > runs - runs / 4 ? wides : runs - runs / 4;
  const uint32_t before = run < span ? uint64_t(run) * wides / span : wides;
  const uint32_t after = run < span ? uint64_t(run + 1) * wides / span : wides;
  if (after > before)
    wide_item<T, C, DP, false>(of_wide.k[0], of_wide.k[1], of_wide.v[0], of_wide.v[1],
                                           of_wide.rows, of_wide.redo, a,
                                           wide + before / a.together,
                                           before % a.together * each + part);
  else
    narrow_item<T, C, DP, false>(*reinterpret_cast<typename Narrow<T, C, DP>::Lds*>(shared),
                                 nullptr, a, narrow + run - before, part * a.together, 0);
}

// Joins the parts of a (token, head): o = sum_i e^(m_i - m) o_i / sum_i e^(m_i - m) l_i, W
// waves a row. The loads of a row's parts are what takes time, so they are independent of one
// another: a lane holds 4 dimensions of every 64 / lanes-th part (of each 64, whose maxima
// and sums the lanes hold), and the waves take turns. The order of the sums is fixed. The
// launch's workgroups are the `first` one and on.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void join_parts(Args a, const int32_t* tokens,
                                                       const int32_t* starts,
                                                       const int32_t* parts, int32_t n,
                                                       int64_t first) {
  __shared__ float sums[kWaves][IEKV_ATTENTION_MAX_DIM];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, turn = wave % W;
  const int32_t heads = a.kv_heads * a.group, d = a.head_dim;
  const int64_t row = (first + blockIdx.x) * (kWaves / W) + wave / W;
  const bool real = row < static_cast<int64_t>(n) * heads;
  const int32_t entry = real ? static_cast<int32_t>(row / heads) : 0;
  const int32_t head = real ? static_cast<int32_t>(row % heads) : 0;
  const int32_t kv_head = head / a.group, in_group = head % a.group;
  const int32_t p0 = starts[entry], p1 = starts[entry + 1];
  const int32_t lanes = d <= 32 ? 8 : d <= 64 ? 16 : 32, each = kWave / lanes;
  const int32_t which = lane / lanes, d0 = lane % lanes * 4;
  const auto slot_of = [&](int32_t p) {
    return static_cast<int64_t>(parts[p] + in_group) * a.kv_heads + kv_head;
  };
  float m = -INFINITY, l = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  for (int32_t q0 = p0; q0 < p1; q0 += kWave) {
    const int32_t count = p1 - q0 < kWave ? p1 - q0 : kWave;
    const int64_t slot = slot_of(q0 + (lane < count ? lane : 0));
    const float2 ml = a.part_ml[slot];
    // The first parts' sums are on their way while the maximum is found.
    constexpr int kAtOnce = 4;
    f32x4 x[kAtOnce];
    const auto load = [&](int32_t q) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int32_t mine = q + i * W * each + which;
        const int64_t at = __shfl(slot, mine < count ? mine : 0) * d + (d0 < d ? d0 : 0);
        __builtin_memcpy(&x[i], a.part_o + at, 16);
      }
    };
    load(turn * each);
    const float top = fmaxf(m, wave_max(lane < count ? ml.x : -INFINITY));
    const float base = top == -INFINITY ? 0.f : top, fade = power2(m - base);
    m = top;
    l *= fade;
    o *= fade;
    const float weight = power2(ml.x - base);
    if (lane < count) l = fmaf(weight, ml.y, l);
    for (int32_t q = turn * each; q < count; q += kAtOnce * W * each) {
      if (q != turn * each) load(q);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int32_t mine = q + i * W * each + which;
        const float w = __shfl(weight, mine < count ? mine : 0);
        if (mine < count) o += x[i] * w;
      }
    }
  }
  l = wave_sum(l);
  for (int s = lanes; s < kWave; s *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], s);
  if constexpr (W > 1) {
    if (which == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][d0 + i] = o[i];
    __syncthreads();
    if (turn == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        for (int w = 1; w < W; ++w) o[i] += sums[wave + w][d0 + i];
  }
  if (!real || turn || which || d0 >= d) return;
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = o[i] / l;
  store_out<T, 4>(static_cast<T*>(a.out) +
                      (static_cast<int64_t>(tokens[entry]) * heads + head) * d + d0, x);
}

}  // namespace iekv_ops

#endif  // IEKV_ATTENTION_KERNELS_H_
