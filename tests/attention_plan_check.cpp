// Checks attention_plan.h on the CPU: for every step read from stdin, each (token, key) that
// the mask lets through is in exactly one item, no item has a key that none of its tokens
// sees beyond what its ranges need, and the parts of a token are the slots of its items.
//
// Input, one step a line: group kv_heads block window sinks shared wide_rows units n, then n times
// context queries. Prints "ok" and the number of items, or what is wrong.
#include <cstdio>
#include <iostream>
#include <map>
#include <set>
#include <sstream>
#include <string>

#include "attention_plan.h"

using namespace iekv_attention;

static std::string check(const Shape& sh, const std::vector<Sequence>& seqs, int units) {
  const Plan plan = make_plan(sh, seqs, units);
  std::vector<std::pair<int, int>> where;   // sequence, position of each token
  for (size_t s = 0; s < seqs.size(); ++s)
    for (int i = 0; i < seqs[s].queries; ++i)
      where.push_back({static_cast<int>(s), seqs[s].context - seqs[s].queries + i});
  if (plan.positions.size() != where.size()) return "positions";
  if (plan.narrow.first != 0 || plan.wide.first != plan.narrow.n ||
      plan.narrow.n + plan.wide.n != static_cast<int>(plan.items.size()))
    return "launches";
  std::vector<std::map<int, int>> seen(where.size());
  std::vector<std::multiset<int>> slots(where.size());
  std::vector<bool> direct(where.size(), false);
  int64_t used = 0;
  int leading = -1;
  for (const Sequence& s : seqs)
    if (s.queries && leading < 0) leading = s.table;
  for (size_t i = 0; i < plan.items.size(); ++i) {
    const Item& it = plan.items[i];
    const int most = static_cast<int>(i) < plan.narrow.n ? kNarrowRows : sh.wide_rows;
    if (it.tokens < 1 || (it.tokens > 1 && it.tokens * sh.group > most)) return "rows";
    if (it.a0 > it.a1 || it.b0 > it.b1 || (it.a1 > it.a0 && it.b1 > it.b0 && it.b0 < it.a1))
      return "ranges";
    if (!keys_of(it)) return "empty item";
    if (it.slot >= 0) {
      if (it.slot != used) return "slots overlap";
      used += int64_t(it.tokens) * sh.group;
    }
    for (int t = it.token0; t < it.token0 + it.tokens; ++t) {
      const auto& [s, p] = where[t];
      if (p != plan.positions[t] || p < it.low || p > it.high) return "position";
      const bool prefix = it.table == leading && it.b1 <= sh.shared && sh.shared;
      if (!prefix && it.table != seqs[s].table) return "table";
      if (it.slot >= 0) slots[t].insert(it.slot + (t - it.token0) * sh.group);
      else if (direct[t]) return "two items write a row";
      else direct[t] = true;
      for (int v = 0; v < keys_of(it); ++v) {
        const int j = v < it.a1 - it.a0 ? it.a0 + v : it.b0 + (v - (it.a1 - it.a0));
        if (j < 0 || j >= seqs[s].context) return "key outside the context";
        if (j <= p && (!sh.window || j > p - sh.window || j < sh.sinks)) ++seen[t][j];
      }
    }
  }
  if (used != plan.slots) return "slot count";
  for (size_t t = 0; t < where.size(); ++t) {
    const int p = where[t].second;
    int want = 0;
    for (int j = 0; j <= p; ++j)
      if (!sh.window || j > p - sh.window || j < sh.sinks) {
        ++want;
        const auto f = seen[t].find(j);
        if (f == seen[t].end() || f->second != 1) return "a key is not read once";
      }
    if (want != static_cast<int>(seen[t].size())) return "other keys";
    if (direct[t] == !slots[t].empty()) return "a row is written directly and joined, or neither";
  }
  std::vector<bool> joined(where.size(), false);
  if (plan.join_starts.size() != plan.join_tokens.size() + 1) return "join starts";
  for (size_t e = 0; e < plan.join_tokens.size(); ++e) {
    const int t = plan.join_tokens[e];
    if (joined[t]) return "joined twice";
    joined[t] = true;
    std::multiset<int> got(plan.join_parts.begin() + plan.join_starts[e],
                           plan.join_parts.begin() + plan.join_starts[e + 1]);
    if (got != slots[t]) return "parts";
  }
  for (size_t t = 0; t < where.size(); ++t)
    if (joined[t] == direct[t]) return "join list";
  return "ok " + std::to_string(plan.items.size());
}

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    Shape sh{};
    int units, n;
    in >> sh.group >> sh.kv_heads >> sh.block_size >> sh.window >> sh.sinks >> sh.shared >>
        sh.wide_rows >> units >> n;
    std::vector<Sequence> seqs(n);
    int tokens = 0, table = 0;
    for (Sequence& s : seqs) {
      in >> s.context >> s.queries;
      s.token0 = tokens;
      s.table = table;
      tokens += s.queries;
      table += (s.context + sh.block_size - 1) / sh.block_size;
    }
    std::cout << check(sh, seqs, units) << std::endl;
  }
}
