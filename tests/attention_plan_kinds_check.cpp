// The checks of attention_plan_check.cpp for steps of every kind: input lines begin with few_keys
// and key_bytes, then go on as there. Prints "ok", the number of items and which kinds the step
// has: shared (items of leading blocks), narrow-parts and wide-parts (keys of a sequence's own cut
// up), mixed (a token of shared keys and of its own), streams, together (KV heads a workgroup
// takes).
#pragma GCC diagnostic push
#pragma GCC diagnostic ignored "-Wreturn-type"
#define main old_main
#include "attention_plan_check.cpp"
#undef main
#pragma GCC diagnostic pop

static std::string kinds(const Shape& sh, const std::vector<Sequence>& seqs, int units) {
  const Plan plan = make_plan(sh, seqs, units);
  std::vector<int> sequence;
  for (size_t s = 0; s < seqs.size(); ++s)
    sequence.insert(sequence.end(), seqs[s].queries, static_cast<int>(s));
  std::set<std::string> has;
  std::map<std::pair<int, bool>, int> own;   // items of a token's own keys
  std::set<int> in_shared;
  for (size_t i = 0; i < plan.items.size(); ++i) {
    const Item& it = plan.items[i];
    const bool narrow = static_cast<int>(i) < plan.narrow.n;
    const int first = it.a1 > it.a0 ? it.a0 : it.b0;
    bool several = false;
    for (int t = it.token0; t < it.token0 + it.tokens; ++t)
      several = several || sequence[t] != sequence[it.token0];
    const bool shared = sh.shared && it.b1 <= sh.shared && first < sh.shared &&
                        (several || it.table != seqs[sequence[it.token0]].table);
    if (shared) has.insert("shared");
    for (int t = it.token0; t < it.token0 + it.tokens; ++t) {
      if (shared) in_shared.insert(t);
      else if (++own[{t, narrow}] > 1) has.insert(narrow ? "narrow-parts" : "wide-parts");
    }
  }
  for (const auto& [key, n] : own)
    if (in_shared.count(key.first)) has.insert("mixed");
  if (plan.streams) has.insert("streams");
  has.insert("together-" + std::to_string(plan.together));
  std::string out;
  for (const std::string& k : has) out += " " + k;
  return out;
}

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    Shape sh{};
    int units, n;
    in >> sh.few_keys >> sh.key_bytes >> sh.group >> sh.kv_heads >> sh.block_size >> sh.window >>
        sh.sinks >> sh.shared >> sh.wide_rows >> units >> n;
    std::vector<Sequence> seqs(n);
    int tokens = 0, table = 0;
    for (Sequence& s : seqs) {
      in >> s.context >> s.queries;
      s.token0 = tokens;
      s.table = table;
      tokens += s.queries;
      table += (s.context + sh.block_size - 1) / sh.block_size;
    }
    std::cout << check(sh, seqs, units) << kinds(sh, seqs, units) << std::endl;
  }
  return 0;
}
