// How a step's attention is cut into work items: host code, no GPU (checked on the CPU by
// tests/attention_plan_check.cpp).
//
// A query row is (token, head). The rows of one KV head that read the same keys go
// together: an item is a run of tokens, all `group` heads of each, over a set of keys of
// one block table. The keys are two ranges: [a0, a1), of the sink tokens, then [b0, b1).
// An item whose rows see other keys in other items leaves partial results (the sum of
// e^(s - m) v, m and the sum of e^(s - m)) for a second launch that joins them.
#ifndef IEKV_ATTENTION_PLAN_H_
#define IEKV_ATTENTION_PLAN_H_

#include <algorithm>
#include <cstdint>
#include <vector>

namespace iekv_attention {

struct Item {
  int32_t token0, tokens;  // rows: tokens token0 .. token0 + tokens - 1, every head of the group
  int32_t table;           // first entry of the block table among the plan's tables
  int32_t a0, a1, b0, b1;  // keys
  int32_t slot;            // first partial slot, or -1: the item alone makes its rows
  int32_t low, high;       // smallest and largest position of its tokens
  int32_t pad[2];
};
static_assert(sizeof(Item) == 48, "items are read as 12 words");
constexpr int kItemWords = 12;

struct Shape {
  int32_t group, kv_heads, block_size;
  int64_t window, sinks;  // window 0: every key up to the query's own
  int32_t shared;         // keys of the shared blocks (0: none)
  int32_t wide_rows;      // rows an item of the wide kernel holds at most (0: there is none)
  int32_t few_keys = 1024;  // that a narrow workgroup takes whole rather than leave parts
  int32_t key_bytes = 512;  // K and V of a key in one KV head
};

struct Sequence {
  int32_t context, queries, token0, table;
};

// What one launch runs: `n` items from item `first` on.
struct Launch {
  int32_t first = 0, n = 0;
};

struct Plan {
  std::vector<Item> items;
  Launch narrow, wide;
  bool streams = false;                // the narrow items keep the card's memory busy for long
  int32_t together = 1;                // KV heads a workgroup of the narrow kernel takes
  std::vector<int32_t> positions;      // per token
  std::vector<int32_t> join_tokens;    // tokens with several parts
  std::vector<int32_t> join_starts;    // n + 1: where each one's parts begin
  std::vector<int32_t> join_parts;     // first slot of the token in each part
  int64_t slots = 0;                   // partial slots per KV head
};

constexpr int kNarrowRows = 16;
constexpr int kNarrowWaves = 4;
constexpr int64_t kSharedBytes = 256 << 10;  // of shared keys in a KV head that are worth a join
constexpr int64_t kSavedBytes = 8 << 20;     // and of reads that sharing them saves

// Keys of [lo, hi) that any of positions low..high sees.
inline void visible(const Shape& sh, int64_t low, int64_t high, int64_t lo, int64_t hi, Item* it) {
  hi = std::min(hi, high + 1);
  const int64_t window = sh.window > 0 ? sh.window : int64_t(1) << 40;
  const int64_t a1 = std::max(lo, std::min(sh.sinks, hi));
  const int64_t b0 = std::max(a1, low - window + 1);
  it->a0 = static_cast<int32_t>(lo);
  it->a1 = static_cast<int32_t>(a1);
  it->b0 = static_cast<int32_t>(std::min(b0, std::max(hi, a1)));
  it->b1 = static_cast<int32_t>(std::max<int64_t>(hi, it->b0));
  if (it->b0 == it->a1) {  // one range
    it->b0 = it->a0;
    it->a1 = it->a0;
  }
}

inline int32_t keys_of(const Item& it) { return (it.a1 - it.a0) + (it.b1 - it.b0); }

// Keys v0 .. v1 - 1 of the item's ranges laid end to end.
inline Item cut(const Item& it, int32_t v0, int32_t v1) {
  const int32_t na = it.a1 - it.a0;
  Item out = it;
  out.a0 = it.a0 + std::min(v0, na);
  out.a1 = it.a0 + std::min(v1, na);
  out.b0 = it.b0 + std::max(v0 - na, 0);
  out.b1 = it.b0 + std::max(v1 - na, 0);
  return out;
}

// Items of a run of tokens over keys [lo, hi) of a table, at most `rows` rows each.
inline void add_tiles(const Shape& sh, const std::vector<int32_t>& positions, int32_t token0,
                      int32_t tokens, int32_t table, int64_t lo, int64_t hi, int32_t rows,
                      std::vector<Item>* out) {
  const int32_t per = std::max(1, rows / sh.group);
  for (int32_t t = 0; t < tokens; t += per) {
    Item it{};
    it.token0 = token0 + t;
    it.tokens = std::min(per, tokens - t);
    it.table = table;
    const auto first = positions.begin() + it.token0;
    it.low = *std::min_element(first, first + it.tokens);
    it.high = *std::max_element(first, first + it.tokens);
    visible(sh, it.low, it.high, lo, hi, &it);
    if (keys_of(it)) out->push_back(it);
  }
}

// Splits items into parts of at most `each` keys, the smallest such number (a multiple of
// `step`, `least` or more, and no less than a workgroup's share of them all) that keeps to
// `want` workgroups, so that they run at once and none is much longer than another. Where
// there are more items than that, half as many again are allowed: one long sequence among
// many short ones is cut all the same.
inline std::vector<Item> split(const std::vector<Item>& in, int64_t blocks_per_item, int64_t want,
                               int64_t least, int64_t step) {
  int64_t longest = 0, keys = 0;
  for (const Item& it : in) {
    longest = std::max<int64_t>(longest, keys_of(it));
    keys += keys_of(it);
  }
  const int64_t items = static_cast<int64_t>(in.size());
  const int64_t share = std::max<int64_t>(1, want / blocks_per_item);
  const int64_t most = std::max(share, items + items / 2);
  least = (std::max(least, keys / share) + step - 1) / step * step;
  const auto parts = [](const Item& it, int64_t each) { return (keys_of(it) + each - 1) / each; };
  // In steps: too small, and large enough.
  int64_t low = least / step - 1, high = std::max((longest + step - 1) / step, least / step);
  while (high - low > 1) {
    const int64_t middle = (low + high) / 2;
    int64_t total = 0;
    for (const Item& it : in) total += parts(it, middle * step);
    (total <= most ? high : low) = middle;
  }
  std::vector<Item> out;
  for (const Item& it : in) {
    const int64_t n = keys_of(it), count = parts(it, high * step);
    const int64_t size = ((n + count - 1) / count + step - 1) / step * step;
    for (int64_t v = 0; v < n; v += size)
      out.push_back(cut(it, static_cast<int32_t>(v), static_cast<int32_t>(std::min(n, v + size))));
  }
  return out;
}

inline Plan make_plan(const Shape& sh, const std::vector<Sequence>& seqs, int32_t compute_units) {
  Plan plan;
  int32_t tokens = 0;
  for (const Sequence& s : seqs)
    for (int32_t i = 0; i < s.queries; ++i, ++tokens)
      plan.positions.push_back(s.context - s.queries + i);
  std::vector<Item> narrow, wide;
  auto add = [&](int32_t token0, int32_t n, int32_t table, int64_t lo, int64_t hi) {
    const bool is_wide = sh.wide_rows > 0 && int64_t(n) * sh.group > kNarrowRows;
    add_tiles(sh, plan.positions, token0, n, table, lo, hi,
              is_wide ? sh.wide_rows : kNarrowRows, is_wide ? &wide : &narrow);
  };
  // Sequences whose own rows fill a tile gain nothing from a tile shared with others: they
  // read the shared keys with their own, and leave no partial results. The rest are taken in
  // runs.
  const auto could = [&](const Sequence& s) {
    return sh.shared && s.queries &&
           int64_t(s.queries) * sh.group < (sh.wide_rows ? sh.wide_rows : kNarrowRows);
  };
  // Nor do short prefixes, or those of few sequences, where what is read again for each is less
  // than the parts of every row, their join and a second launch take. Of eight bf16 heads of 128
  // alone and shared: 96 sequences of 1,200 tokens behind 16 of them 85 us and 94, behind 512 76
  // and 70, behind 1,024 68 and 32; eight of 612 behind 512 16.9 and 12.0, four 11.7 and 11.7.
  // 8-bit keys pay from twice as many on: 64 sequences of 612 behind 512 17 us and 23, 128 of
  // 1,124 behind 1,024 50 and 38. Between, some gain a tenth and some lose one.
  // What counts is what the sequences see: a window may have left most of the prefix behind.
  int64_t seen = 0, longest = 0;
  for (const Sequence& s : seqs) {
    if (!could(s)) continue;
    Item it{};
    visible(sh, s.context - s.queries, s.context - 1, 0, sh.shared, &it);
    seen += keys_of(it);
    longest = std::max<int64_t>(longest, keys_of(it));
  }
  const bool worth = longest * sh.key_bytes >= kSharedBytes &&
                     (seen - longest) * sh.key_bytes * sh.kv_heads >= kSavedBytes;
  const auto shares = [&](const Sequence& s) { return worth && could(s); };
  int32_t leading = -1, run0 = 0, run = 0;
  for (const Sequence& s : seqs) {
    if (!s.queries) continue;
    if (leading < 0) leading = s.table;
    if (shares(s)) {
      if (!run) run0 = s.token0;
      run += s.queries;
    } else if (run) {
      add(run0, run, leading, 0, sh.shared);
      run = 0;
    }
    add(s.token0, s.queries, s.table, shares(s) ? sh.shared : 0, s.context);
  }
  if (run) add(run0, run, leading, 0, sh.shared);
  // A workgroup of several heads reads longer runs of the cache, and each of its waves leaves
  // a part of its own: worth it where a wave has steps enough to outweigh the part.
  int64_t narrow_keys = 0;
  for (const Item& it : narrow) narrow_keys += keys_of(it);
  plan.streams = narrow_keys * sh.kv_heads >= int64_t(4) * compute_units * kNarrowWaves * 256;
  if (plan.streams)
    plan.together = sh.kv_heads % 4 == 0 ? 4 : sh.kv_heads % 2 == 0 ? 2 : 1;
  // Few keys take less time in turn than a join does, if there is none yet.
  int32_t longest_item = 0;
  for (const Item& it : narrow) longest_item = std::max(longest_item, keys_of(it));
  const bool whole = longest_item <= sh.few_keys && !worth;
  // Two workgroups fit a compute unit. Long streams are cut for half as many again: 128
  // sequences of unlike lengths 182 us against 191 with two, of one length 175 against 173.
  if (!whole)
    narrow = split(narrow, sh.kv_heads / plan.together, (plan.streams ? 3 : 2) * compute_units, 256,
                   64);
  const int64_t narrow_blocks = int64_t(narrow.size()) * sh.kv_heads / plan.together;
  // Parts of wide items are 64 times as many rows to write and join as those of narrow ones
  // are: they are cut only where more than half of the compute units would have none, and so
  // that those of a step run at once, two to a compute unit.
  if (int64_t(wide.size()) * sh.kv_heads * 2 < compute_units)
    wide = split(wide, sh.kv_heads,
                 std::max<int64_t>(compute_units, 2 * compute_units - narrow_blocks), 128, 64);
  // The longest first: the last workgroups to start are short ones.
  auto longer = [](const Item& x, const Item& y) { return keys_of(x) > keys_of(y); };
  std::stable_sort(narrow.begin(), narrow.end(), longer);
  std::stable_sort(wide.begin(), wide.end(), longer);
  plan.narrow = {0, static_cast<int32_t>(narrow.size())};
  plan.wide = {plan.narrow.n, static_cast<int32_t>(wide.size())};
  plan.items = std::move(narrow);
  plan.items.insert(plan.items.end(), wide.begin(), wide.end());

  // A token is joined unless one item makes its rows, and those of the item's other tokens,
  // alone.
  std::vector<int32_t> parts(tokens, 0);
  std::vector<char> joined(tokens, 0);
  for (const Item& it : plan.items)
    for (int32_t t = 0; t < it.tokens; ++t) ++parts[it.token0 + t];
  for (Item& it : plan.items) {
    bool alone = true;
    for (int32_t t = 0; t < it.tokens; ++t) alone = alone && parts[it.token0 + t] == 1;
    it.slot = alone ? -1 : 0;
    for (int32_t t = 0; t < it.tokens && !alone; ++t) joined[it.token0 + t] = 1;
  }
  std::vector<int32_t> at(tokens, -1);
  plan.join_starts.push_back(0);
  for (int32_t t = 0; t < tokens; ++t) {
    if (!joined[t]) continue;
    at[t] = plan.join_starts.back();
    plan.join_tokens.push_back(t);
    plan.join_starts.push_back(plan.join_starts.back() + parts[t]);
  }
  plan.join_parts.resize(plan.join_starts.back());
  for (Item& it : plan.items) {
    if (it.slot < 0) continue;
    it.slot = static_cast<int32_t>(plan.slots);
    for (int32_t t = 0; t < it.tokens; ++t)
      plan.join_parts[at[it.token0 + t]++] = it.slot + t * sh.group;
    plan.slots += int64_t(it.tokens) * sh.group;
  }
  return plan;
}

}  // namespace iekv_attention

#endif  // IEKV_ATTENTION_PLAN_H_
