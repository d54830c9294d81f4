// Attention over the paged KV cache (C-ABI in iekv_ops.h, work items in attention_plan.h).
//
// For a query row q at position p and the keys j it sees (j <= p, and j > p - window or
// j < sinks): o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q.k_j, m = max s_j.
// Powers are taken to base 2: scores are scaled by scale * log2(e).
#include "ops_common.h"

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <string>
#include <vector>

#include "attention_kernels.h"

namespace iekv_ops {

thread_local std::string g_error;

int set_error(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_error = buf;
  return code;
}

}  // namespace iekv_ops

using namespace iekv_ops;
using iekv_attention::Launch;

struct iekv_attention_plan {
  iekv_attention_shape shape;
  int device;                    // whose arrays it is for
  Launch narrow, wide;
  bool streams;                  // the narrow items are a long stream
  int32_t together;              // KV heads a workgroup of the narrow kernel takes
  int32_t joined;                // tokens with several parts
  int64_t tokens, slots;
  int64_t positions_at, join_tokens_at, join_starts_at, join_parts_at, tables_at;  // words
  std::vector<int32_t> words;
};

namespace {

constexpr int64_t kJoinFew = 2048;  // rows that are joined by four waves each

int current_device() {
  int device = 0;
  if (hipGetDevice(&device) == hipSuccess) return device;
  (void)hipGetLastError();
  return 0;         // no GPU in sight: a plan made to be looked at
}

int compute_units(int device) {
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) == hipSuccess &&
      n > 0)
    return n;
  (void)hipGetLastError();
  return 256;
}

// More LDS than a kernel may have without asking: asked for once on each device.
template <typename K>
hipError_t allow_lds(K kernel, int bytes, int device, std::atomic<uint64_t>* asked) {
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (asked->load() & bit) return hipSuccess;
  const hipError_t error = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (error == hipSuccess) asked->fetch_or(bit);
  return error;
}

int32_t bytes_of(int32_t type) {
  return type == IEKV_TYPE_F32 ? 4 : type == IEKV_TYPE_E4M3 ? 1 : 2;
}

// Bytes of a head of a key in the cache.
int32_t head_bytes_of(const iekv_attention_shape& s) {
  return s.cache_type >= IEKV_TYPE_MXFP8
             ? static_cast<int32_t>(iekv_mx_head_bytes(s.cache_type, s.head_dim))
             : s.head_dim * bytes_of(s.cache_type);
}

// Whether narrow items of four KV heads are taken together: see Together.
bool together_fits(const iekv_attention_shape& s) {
  return s.cache_type >= IEKV_TYPE_MXFP8 && s.num_kv_heads % kWaves == 0 &&
         s.head_dim % kGroup == 0;
}

// Workgroups that a long stream is cut into for each compute unit. Of four heads' long records two
// keep the memory busy (and have LDS for two), and more drive each other's lines out of L2: 48
// sequences of 6,000 tokens of eight mxfp8 heads of 128 107 us with two, 127 with three, of 96 86
// and 94. Short records take more work for their bytes: 128 sequences of 4,200 tokens in mxfp4 115
// us with three, 126 with two, 143 with four, in mxfp8 heads of 64 107 and 116. So do integers: in
// mxint8 heads of 96 182 us with three and 201 with two, of 128 252 and 225.
int32_t streams_at_once(const iekv_attention_shape& s) {
  const int32_t is_long = s.cache_type == IEKV_TYPE_MXINT8 ? 500 : 400;
  return together_fits(s) && head_bytes_of(s) * kWaves >= is_long ? 2 : 3;
}

// And few items: twice the steps for a wave of microscaled caches take less than twice the parts do,
// the joins' reads included. One sequence of 16,384 tokens of eight heads of 128 in mxint8 17.0 us
// with one, 18.6 with two; two of them in mxfp8 22.2 and 23.8. (Of eight sequences of unlike
// lengths and more, two are better balanced: 16 of 6,000 50 us, with one 55.)
int32_t few_at_once(const iekv_attention_shape& s) { return s.cache_type >= IEKV_TYPE_MXFP8 ? 1 : 2; }

// And what a long stream is: four heads' records come together sooner than other caches' rows pay
// for their parts. 16 sequences of 6,000 tokens of eight mxfp8 heads of 128 42 us together, 50 each
// head by itself, 8 of 8,000 31.5 and 36 (in mxfp4 32 and 35, 24 and 27; in mxint8 51 and 52, 36
// and 39, though 8 of 6,000 34 and 32). A chunk beside them is then in a launch of its own: with
// the last 2,048 of 7,777 tokens 8 of 6,000 360 us, in one launch 450, but with a prompt of 2,048
// 100 and 85 (in the caches of a card that holds many layers, as all of these).
int32_t stream_steps(const iekv_attention_shape& s) { return together_fits(s) ? 1 : 4; }

template <typename T, typename C, int DP>
int launch_dim(const iekv_attention_plan& plan, const Args& a, hipStream_t stream) {
  const int32_t wide = plan.wide.n, narrow = plan.narrow.n;
  const int64_t each = a.kv_heads / a.together;     // workgroups of a narrow item
  const int64_t blocks = wide * int64_t(a.kv_heads) + narrow * each;
  // Both kinds in one launch where the narrow ones are soon done (24 sequences of two KV heads
  // behind 512 tokens: 12.4 us against 18.4 in two); a long stream of them is better alone on
  // the card (128 sequences of the 8B shape: 206 us in two launches, 246 in one).
  const bool both = wide && narrow && !plan.streams && blocks <= kMaxGrid;
  // As many of n items at a time as a launch has workgroups for.
  const auto in_launches = [](int64_t n, int64_t blocks_each, const auto& run) {
    const int64_t most = kMaxGrid / blocks_each;
    for (int64_t first = 0; first < n; first += most) {
      run(first, std::min(most, n - first));
      IEKV_OPS_HIP(hipGetLastError());
    }
    return int(IEKV_OK);
  };
  if constexpr (sizeof(T) == 2) {
    bool done = !wide;
    if constexpr (std::is_same_v<T, C> || kScaled<C>) {
      const auto aligned = [](const void* p) {
        return kScaled<C> || reinterpret_cast<uintptr_t>(p) % 16 == 0;
      };
      if (wide && !both && aligned(a.k) && aligned(a.v)) {
        if (const int rc = in_launches(wide, a.kv_heads, [&](int64_t first, int64_t n) {
              hipLaunchKernelGGL((attend_wide<T, C, DP>), dim3(n * a.kv_heads), dim3(kThreads), 0,
                                 stream, a, static_cast<int32_t>(plan.wide.first + first));
            }))
          return rc;
        done = true;
      }
    }
    if (!done) {
      constexpr int bytes = std::max<int>(sizeof(typename Wide<T, DP>::Lds),
                                          sizeof(typename Narrow<T, C, DP>::Lds));
      static std::atomic<uint64_t> asked{0};
      IEKV_OPS_HIP(allow_lds(attend_both<T, C, DP>, bytes, plan.device, &asked));
      if (const int rc = in_launches(wide, a.kv_heads, [&](int64_t first, int64_t n) {
            hipLaunchKernelGGL((attend_both<T, C, DP>),
                               dim3(both ? blocks : n * a.kv_heads), dim3(kThreads), bytes, stream,
                               a, static_cast<int32_t>(plan.wide.first + first),
                               static_cast<int32_t>(n), plan.narrow.first, both ? narrow : 0);
          }))
        return rc;
    }
  }
  if (narrow && !both) {
    // Only 32-bit queries have narrow items of more than 16 heads.
    const auto run = [&](auto kernel, size_t bytes) {
      return in_launches(narrow, each, [&](int64_t first, int64_t n) {
        hipLaunchKernelGGL(kernel, dim3(n * each, (a.group + 15) / 16), dim3(kThreads), bytes,
                           stream, a, static_cast<int32_t>(plan.narrow.first + first),
                           static_cast<int32_t>(n));
      });
    };
    using N = Narrow<T, C, DP>;
    constexpr size_t kUnasked = 64 << 10;           // of LDS for a workgroup
    static_assert(sizeof(typename N::Lds) <= kUnasked);
    bool done = false;
    if constexpr (kScaled<C>) {
      // Chunks of 16 bytes come into LDS directly.
      const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
      if (a.together == kWaves && together_fits(plan.shape) && aligned(a.k) && aligned(a.v)) {
        if (const int rc = run(attend_narrow<T, C, DP, true>, 0)) return rc;
        done = true;
      }
    }
    if (!done) {
      if (const int rc = run(attend_narrow<T, C, DP, false>, sizeof(typename N::Lds))) return rc;
    }
  }
  if (plan.joined) {
    // Few rows have many parts each: their loads are spread over four waves.
    const int64_t rows = int64_t(plan.joined) * a.kv_heads * a.group;
    const int32_t* w = a.words;
    const bool few = rows <= kJoinFew;
    if (const int rc = in_launches(few ? rows : (rows + kWaves - 1) / kWaves, 1,
                                   [&](int64_t first, int64_t n) {
          hipLaunchKernelGGL((few ? join_parts<T, kWaves> : join_parts<T, 1>), dim3(n),
                             dim3(kThreads), 0, stream, a, w + plan.join_tokens_at,
                             w + plan.join_starts_at, w + plan.join_parts_at, plan.joined, first);
        }))
      return rc;
  }
  return IEKV_OK;
}

template <typename T, typename C>
int launch(const iekv_attention_plan& plan, const Args& a, hipStream_t stream) {
  switch ((a.head_dim + 31) / 32) {
    case 1: return launch_dim<T, C, 32>(plan, a, stream);
    case 2: return launch_dim<T, C, 64>(plan, a, stream);
    case 3: return launch_dim<T, C, 96>(plan, a, stream);
    default: return launch_dim<T, C, 128>(plan, a, stream);
  }
}

// Whether the output lies over queries of other rows: a workgroup writes its rows when it has
// read their queries, and not when others have read theirs.
bool overlaps(const iekv_attention_plan& plan, const void* q, int64_t token_stride,
              int64_t head_stride, const void* out) {
  const iekv_attention_shape& s = plan.shape;
  const int64_t tokens = plan.tokens, heads = s.num_heads, size = bytes_of(s.query_type);
  const int64_t row = s.head_dim * size, bytes = tokens * heads * row;
  const auto at = [](const void* p) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); };
  const int64_t q0 = at(q), out0 = at(out);
  const int64_t along = (tokens - 1) * token_stride * size, across = (heads - 1) * head_stride * size;
  const int64_t lo = q0 + std::min<int64_t>(along, 0) + std::min<int64_t>(across, 0);
  const int64_t hi = q0 + std::max<int64_t>(along, 0) + std::max<int64_t>(across, 0) + row;
  if (hi <= out0 || out0 + bytes <= lo) return false;
  if (q0 == out0 && (tokens == 1 || token_stride == heads * s.head_dim) &&
      (heads == 1 || head_stride == s.head_dim))
    return false;                    // row over row
  for (int64_t t = 0; t < tokens; ++t)
    for (int64_t h = 0; h < heads; ++h) {
      const int64_t first = q0 + (t * token_stride + h * head_stride) * size;
      if (first < out0 + bytes && out0 < first + row) return true;
    }
  return false;
}

int64_t workspace_bytes_of(const iekv_attention_plan& p) {
  return p.slots * p.shape.num_kv_heads * (p.shape.head_dim + 2) * int64_t(sizeof(float));
}

bool known_types(int32_t query, int32_t cache) {
  if (query == IEKV_TYPE_F32) return cache >= IEKV_TYPE_F32 && cache <= IEKV_TYPE_MXFP4;
  return (query == IEKV_TYPE_F16 || query == IEKV_TYPE_BF16) &&
         (cache == query || (cache >= IEKV_TYPE_E4M3 && cache <= IEKV_TYPE_MXFP4));
}

int check_shape(const iekv_attention_shape& s) {
  const auto bad = [](const char* what, int64_t v) {
    return set_error(IEKV_ERR_INVALID, "%s %lld out of range", what, static_cast<long long>(v));
  };
  if (s.num_kv_heads < 1 || s.num_kv_heads > 4096) return bad("num_kv_heads", s.num_kv_heads);
  if (s.num_heads < 1 || s.num_heads % s.num_kv_heads)
    return set_error(IEKV_ERR_INVALID, "%d query heads for %d KV heads", s.num_heads,
                     s.num_kv_heads);
  if (s.num_heads / s.num_kv_heads > IEKV_ATTENTION_MAX_GROUP)
    return set_error(IEKV_ERR_INVALID, "%d query heads per KV head, at most %d are taken",
                     s.num_heads / s.num_kv_heads, IEKV_ATTENTION_MAX_GROUP);
  if (s.head_dim < 8 || s.head_dim > IEKV_ATTENTION_MAX_DIM || s.head_dim % 8)
    return set_error(IEKV_ERR_INVALID, "head_dim %d is not a multiple of 8 up to %d", s.head_dim,
                     IEKV_ATTENTION_MAX_DIM);
  if (s.block_size < 1 || s.block_size > (1 << 20)) return bad("block_size", s.block_size);
  if (s.num_blocks < 1 || s.num_blocks > INT32_MAX) return bad("num_blocks", s.num_blocks);
  if (s.num_blocks * s.block_size > UINT32_MAX)
    return set_error(IEKV_ERR_INVALID, "%lld blocks of %d rows: more than 2^32 rows",
                     static_cast<long long>(s.num_blocks), s.block_size);
  if (!known_types(s.query_type, s.cache_type))
    return set_error(IEKV_ERR_INVALID, "queries of type %d on a cache of type %d", s.query_type,
                     s.cache_type);
  if (s.window < 0) return bad("window", s.window);
  if (s.sinks < 0) return bad("sinks", s.sinks);
  if (s.shared_blocks < 0 || s.shared_blocks > IEKV_ATTENTION_MAX_CONTEXT / s.block_size)
    return bad("shared_blocks", s.shared_blocks);
  return IEKV_OK;
}

// Keys that one workgroup takes for less than the parts and their join cost: four steps of its
// four waves, or what a compute unit's loads bring in that time (one sequence of 700 tokens of
// eight bf16 heads of 128, 350 KB a workgroup: 13.5 us against 15.8 in parts; of 1,000 tokens
// 19 against 14, and of 1,000 on an 8-bit cache 16.7 against 19.2).
int32_t few_keys(const iekv_attention_shape& s) {
  return std::min(s.cache_type == IEKV_TYPE_F32 ? 512 : 1024, (384 << 10) / (2 * head_bytes_of(s)));
}

int make(const iekv_attention_shape& shape, int32_t n_seqs, const int32_t* context_lens,
         const int32_t* query_lens, const int32_t* tables, const int64_t* starts,
         iekv_attention_plan** out) {
  const int64_t bs = shape.block_size;
  std::vector<iekv_attention::Sequence> seqs(n_seqs);
  std::vector<int32_t> entries;
  int64_t tokens = 0;
  const int32_t* leading = nullptr;
  for (int32_t s = 0; s < n_seqs; ++s) {
    const int64_t context = context_lens[s], queries = query_lens[s];
    if (context < 0 || context > IEKV_ATTENTION_MAX_CONTEXT || queries < 0 || queries > context)
      return set_error(IEKV_ERR_INVALID, "sequence %d: %lld queries in a context of %lld", s,
                       static_cast<long long>(queries), static_cast<long long>(context));
    const int64_t used = (context + bs - 1) / bs, held = starts[s + 1] - starts[s];
    if (starts[s] < 0 || held < used)
      return set_error(IEKV_ERR_RANGE, "sequence %d: context of %lld needs %lld blocks, table has %lld",
                       s, static_cast<long long>(context), static_cast<long long>(used),
                       static_cast<long long>(held));
    if (!tables && (used || held)) return set_error(IEKV_ERR_INVALID, "tables is null");
    const int32_t* table = tables + starts[s];
    for (int64_t b = 0; b < used; ++b)
      if (table[b] < 0 || table[b] >= shape.num_blocks)
        return set_error(IEKV_ERR_RANGE, "sequence %d: block id %d out of range for a pool of %lld blocks",
                         s, table[b], static_cast<long long>(shape.num_blocks));
    if (shape.shared_blocks && queries) {
      if (context < shape.shared_blocks * bs)
        return set_error(IEKV_ERR_IDS, "sequence %d: a context of %lld does not fill %lld shared blocks",
                         s, static_cast<long long>(context),
                         static_cast<long long>(shape.shared_blocks));
      if (!leading) leading = table;
      if (!std::equal(leading, leading + shape.shared_blocks, table))
        return set_error(IEKV_ERR_IDS, "sequence %d does not begin with the %lld shared blocks", s,
                         static_cast<long long>(shape.shared_blocks));
    }
    if (tokens + queries > INT32_MAX / 2 / shape.num_heads ||
        static_cast<int64_t>(entries.size()) + used > INT32_MAX)
      return set_error(IEKV_ERR_INVALID, "too many query rows or blocks in one step");
    seqs[s] = {static_cast<int32_t>(context), static_cast<int32_t>(queries),
               static_cast<int32_t>(tokens), static_cast<int32_t>(entries.size())};
    if (queries) entries.insert(entries.end(), table, table + used);
    tokens += queries;
  }
  iekv_attention::Shape sh{shape.num_heads / shape.num_kv_heads, shape.num_kv_heads,
                           shape.block_size, shape.window, shape.sinks,
                           static_cast<int32_t>(shape.shared_blocks * bs),
                           shape.query_type == IEKV_TYPE_F32 ? 0 : kWideRows,
                           few_keys(shape), 2 * head_bytes_of(shape),
                           streams_at_once(shape), few_at_once(shape),
                           stream_steps(shape)};
  const int device = current_device();
  iekv_attention::Plan made = iekv_attention::make_plan(sh, seqs, compute_units(device));
  if (static_cast<int64_t>(made.items.size()) * shape.num_kv_heads > INT32_MAX ||
      made.slots > INT32_MAX)
    return set_error(IEKV_ERR_INVALID, "too many work items in one step");
  auto plan = new iekv_attention_plan{};
  plan->shape = shape;
  plan->device = device;
  plan->narrow = made.narrow;
  plan->wide = made.wide;
  plan->streams = made.streams;
  plan->together = made.together;
  plan->joined = static_cast<int32_t>(made.join_tokens.size());
  plan->tokens = tokens;
  plan->slots = made.slots;
  std::vector<int32_t>& w = plan->words;
  const auto* items = reinterpret_cast<const int32_t*>(made.items.data());
  w.assign(items, items + made.items.size() * iekv_attention::kItemWords);
  const auto append = [&w](const std::vector<int32_t>& x) {
    const int64_t at = static_cast<int64_t>(w.size());
    w.insert(w.end(), x.begin(), x.end());
    return at;
  };
  plan->positions_at = append(made.positions);
  plan->join_tokens_at = append(made.join_tokens);
  plan->join_starts_at = append(made.join_starts);
  plan->join_parts_at = append(made.join_parts);
  plan->tables_at = append(entries);
  *out = plan;
  return IEKV_OK;
}

}  // namespace

extern "C" {

int iekv_ops_abi_version(void) { return IEKV_OPS_ABI_VERSION; }

const char* iekv_ops_last_error(void) { return g_error.c_str(); }

int iekv_attention_plan_create(const iekv_attention_shape* shape, int32_t n_seqs,
                               const int32_t* context_lens, const int32_t* query_lens,
                               const int32_t* tables, const int64_t* table_starts,
                               iekv_attention_plan** out) {
  if (!out) return set_error(IEKV_ERR_INVALID, "out is null");
  *out = nullptr;
  if (!shape) return set_error(IEKV_ERR_INVALID, "shape is null");
  if (n_seqs < 0) return set_error(IEKV_ERR_INVALID, "n_seqs %d is negative", n_seqs);
  if (n_seqs && (!context_lens || !query_lens || !table_starts))
    return set_error(IEKV_ERR_INVALID, "context_lens, query_lens or table_starts is null");
  if (const int rc = check_shape(*shape)) return rc;
  try {
    return make(*shape, n_seqs, context_lens, query_lens, tables, table_starts, out);
  } catch (const std::bad_alloc&) {
    return set_error(IEKV_ERR_CAPACITY, "out of host memory for a plan of %d sequences", n_seqs);
  }
}

int iekv_attention_plan_destroy(iekv_attention_plan* plan) {
  delete plan;
  return IEKV_OK;
}

int iekv_attention_plan_info(const iekv_attention_plan* plan, const int32_t** words,
                             int64_t* n_words, int64_t* tokens, int64_t* workspace_bytes) {
  if (!plan || !words || !n_words || !tokens || !workspace_bytes)
    return set_error(IEKV_ERR_INVALID, "null argument");
  *words = plan->words.data();
  *n_words = static_cast<int64_t>(plan->words.size());
  *tokens = plan->tokens;
  *workspace_bytes = workspace_bytes_of(*plan);
  return IEKV_OK;
}

int iekv_attend(const iekv_attention_plan* plan, const int32_t* words, const void* k,
                const void* v, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                float scale, void* out, void* workspace, int64_t workspace_bytes,
                hipStream_t stream) {
  if (!plan) return set_error(IEKV_ERR_INVALID, "plan is null");
  if (!plan->tokens) return IEKV_OK;
  if (!words || !k || !v || !q || !out)
    return set_error(IEKV_ERR_INVALID, "words, k, v, q or out is null");
  if (reinterpret_cast<uintptr_t>(words) % 16)
    return set_error(IEKV_ERR_INVALID, "words is not aligned to 16 bytes");
  if (!std::isfinite(scale)) return set_error(IEKV_ERR_INVALID, "scale is not finite");
  const int64_t need = workspace_bytes_of(*plan);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(IEKV_ERR_CAPACITY, "workspace of %lld bytes, %lld are needed",
                     static_cast<long long>(workspace ? workspace_bytes : 0),
                     static_cast<long long>(need));
  if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(IEKV_ERR_INVALID, "workspace is not aligned to 16 bytes");
  if (overlaps(*plan, q, q_token_stride, q_head_stride, out))
    return set_error(IEKV_ERR_INVALID, "out overlaps q without being in its place");
  const iekv_attention_shape& s = plan->shape;
  Args a{};
  a.words = words;
  a.k = k;
  a.v = v;
  a.q = q;
  a.out = out;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + plan->slots * s.num_kv_heads * s.head_dim);
  a.positions_at = plan->positions_at;
  a.tables_at = plan->tables_at;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.window = static_cast<int32_t>(std::min<int64_t>(s.window ? s.window : INT32_MAX, INT32_MAX));
  a.sinks = static_cast<int32_t>(std::min<int64_t>(s.sinks, INT32_MAX));
  a.kv_heads = s.num_kv_heads;
  a.group = s.num_heads / s.num_kv_heads;
  a.head_dim = s.head_dim;
  a.block_size = s.block_size;
  a.together = plan->together;
  // Division by a constant as a product (Granlund and Montgomery), for numerators below 2^31.
  while ((uint64_t(1) << a.block_shift) < static_cast<uint64_t>(s.block_size)) ++a.block_shift;
  a.block_magic = static_cast<uint32_t>(
      ((uint64_t(1) << 32) * ((uint64_t(1) << a.block_shift) - s.block_size)) / s.block_size + 1);
  // The kernels take the maximum before they scale, so the sign goes to q; a scale of zero
  // is held above it, so that it leaves the -inf of a hidden key alone.
  a.q_sign = !std::signbit(scale) ? 0 : s.query_type == IEKV_TYPE_F32 ? 0x80000000u : 0x80008000u;
  a.scale = std::max(std::fabs(scale) * 1.4426950408889634f, FLT_MIN);
  const DeviceGuard guard(plan->device);
  IEKV_OPS_HIP(guard.error());
  switch (s.query_type * 8 + s.cache_type) {
    case IEKV_TYPE_F32 * 8 + IEKV_TYPE_F32: return launch<float, float>(*plan, a, stream);
    case IEKV_TYPE_F32 * 8 + IEKV_TYPE_F16: return launch<float, _Float16>(*plan, a, stream);
    case IEKV_TYPE_F32 * 8 + IEKV_TYPE_BF16: return launch<float, Bf16>(*plan, a, stream);
    case IEKV_TYPE_F32 * 8 + IEKV_TYPE_E4M3: return launch<float, E4m3>(*plan, a, stream);
    case IEKV_TYPE_F16 * 8 + IEKV_TYPE_F16: return launch<_Float16, _Float16>(*plan, a, stream);
    case IEKV_TYPE_F16 * 8 + IEKV_TYPE_E4M3: return launch<_Float16, E4m3>(*plan, a, stream);
    case IEKV_TYPE_BF16 * 8 + IEKV_TYPE_BF16: return launch<Bf16, Bf16>(*plan, a, stream);
    case IEKV_TYPE_BF16 * 8 + IEKV_TYPE_E4M3: return launch<Bf16, E4m3>(*plan, a, stream);
    case IEKV_TYPE_F32 * 8 + IEKV_TYPE_MXFP8: return launch<float, Mxfp8>(*plan, a, stream);
    case IEKV_TYPE_F32 * 8 + IEKV_TYPE_MXINT8: return launch<float, Mxint8>(*plan, a, stream);
    case IEKV_TYPE_F32 * 8 + IEKV_TYPE_MXFP4: return launch<float, Mxfp4>(*plan, a, stream);
    case IEKV_TYPE_F16 * 8 + IEKV_TYPE_MXFP8: return launch<_Float16, Mxfp8>(*plan, a, stream);
    case IEKV_TYPE_F16 * 8 + IEKV_TYPE_MXINT8: return launch<_Float16, Mxint8>(*plan, a, stream);
    case IEKV_TYPE_F16 * 8 + IEKV_TYPE_MXFP4: return launch<_Float16, Mxfp4>(*plan, a, stream);
    case IEKV_TYPE_BF16 * 8 + IEKV_TYPE_MXFP8: return launch<Bf16, Mxfp8>(*plan, a, stream);
    case IEKV_TYPE_BF16 * 8 + IEKV_TYPE_MXINT8: return launch<Bf16, Mxint8>(*plan, a, stream);
    default: return launch<Bf16, Mxfp4>(*plan, a, stream);
  }
}

}  // extern "C"
