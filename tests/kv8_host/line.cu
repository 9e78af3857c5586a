// Walks the line of work of the 8-bit cache's attention on the host, worker by worker, as the kernels' warps
// do. Calls whose sums are in order: every tile of every (sequence, kv head, row block) is in one piece, a
// block that is cut has one Cut and its parts are where the merge looks for them. Sums that go back and
// forth: nothing leaves the tensors. Exit code 0: all of it holds.
#include <cstdio>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "kv8_attn.cuh"

using namespace fa2kv;

struct Call {
  std::vector<int> cu, lens;
  AttnArgs a{};
  int err = 0;
  std::vector<Cut> cuts;
  // As the entry point does. `rows`: the largest of a sequence.
  void finish(int group, int heads_kv, int n_q, int total_q, int max_k, int causal, int bottom_right, int workers) {
    const int64_t rows = static_cast<int64_t>(n_q) * group;
    a.lens = lens.data();
    a.cu_q = cu.empty() ? nullptr : cu.data();
    a.err = &err;
    a.batch = static_cast<int>(lens.size());
    a.group = group;
    a.by_group = divisor(group);
    a.heads_kv = heads_kv;
    a.n_q = n_q;
    a.total_q = total_q;
    a.max_k = max_k;
    a.causal = causal;
    a.bottom_right = causal && bottom_right;
    a.c.page_size = 128;
    a.pages_per_seq = (max_k + 127) / 128;
    a.block = rows <= 8 ? 8 : rows <= 16 ? 16 : 256;
    a.workers = workers;
    cuts.assign(workers, Cut{-7});
    a.cuts = cuts.data();
  }
};

// find_share for all lanes, and the result for worker w; false where the line is refused.
struct Lanes {
  Run run[32];
  int sum[32], sum_blocks[32];
  explicit Lanes(const AttnArgs& a) {
    int s = 0, n = 0;
    for (int i = 0; i < 32; ++i) {
      run[i] = run_of(a, i);
      s = sum[i] = line_sum(s, run[i].cost);
      n = sum_blocks[i] = line_sum(n, run[i].blocks);
    }
  }
  bool find(const AttnArgs& a, int w, Share& r, bool& held) const {
    if (!share_of(a, w, sum[31], sum_blocks[31], r)) return false;
    held = r.p0 >= r.p1;  // an empty share needs none
    r.b = run[0].b0;
    for (int i = 31; i >= 0; --i) {
      const int own = run[i].cost + r.block_cost * run[i].blocks, before = sum[i] + r.block_cost * sum_blocks[i] - own;
      if (before <= r.p0 && r.p0 < before + own) {
        r.b = run[i].b0;
        r.start_b = before;
        held = true;
      }
    }
    return true;
  }
};

#define CHECK(x)                                   \
  do {                                             \
    if (!(x)) {                                    \
      std::printf("line %d: %s\n", __LINE__, #x);  \
      return false;                                \
    }                                              \
  } while (0)

static bool walk(Call& c, bool in_order) {
  AttnArgs& a = c.a;
  const Lanes lanes(a);
  struct Part {
    int worker, t0, tiles, slot;
  };
  std::map<std::tuple<int, int, int>, std::vector<Part>> got;
  for (int w = 0; w < a.workers; ++w) {
    Pieces p{};
    bool held = false;
    if (!lanes.find(a, w, p.s, held)) {
      CHECK(!in_order);
      continue;
    }
    CHECK(p.s.p0 >= 0 && p.s.p1 >= p.s.p0 && p.s.p1 <= p.s.total && held);
    p.p = p.s.p0;
    p.w = w;
    if (p.s.p0 >= p.s.p1) a.cuts[w].n_parts = 0;
    Piece o;
    while (p.next(a, o)) {
      CHECK(o.b >= 0 && o.b < a.batch && o.h >= 0 && o.h < a.heads_kv && o.rb >= 0);
      CHECK(o.rb * a.block < o.sq.n_q * a.group);
      CHECK(o.t0 >= 0 && o.tiles > 0 && o.t0 + o.tiles <= Line::tiles(a, o.sq, o.rb));
      CHECK(o.sq.q0 >= 0 && o.sq.len >= 0 && o.sq.len <= a.max_k && o.slot < 2 * a.workers);
      CHECK(a.cu_q == nullptr || o.sq.q0 + o.sq.n_q <= a.total_q);
      CHECK((o.tiles == Line::tiles(a, o.sq, o.rb)) == (o.slot < 0));
      if (in_order) got[{o.b, o.h, o.rb}].push_back({w, o.t0, o.tiles, o.slot});
    }
  }
  if (!in_order) return true;
  CHECK(c.err == 0);
  std::map<std::tuple<int, int, int>, int> cut_by;
  for (int w = 0; w < a.workers; ++w) {
    CHECK(a.cuts[w].n_parts >= 0);  // (written)
    if (a.cuts[w].n_parts > 0) {
      CHECK(w > 0 && cut_by.emplace(std::make_tuple(a.cuts[w].b, a.cuts[w].h, a.cuts[w].row0 / a.block), w).second);
    }
  }
  size_t cut_blocks = 0;
  for (int b = 0; b < a.batch; ++b) {
    const Seq s = sequence(a, b);
    for (int rb = 0; rb < Line::blocks(a, s); ++rb) {
      for (int h = 0; h < a.heads_kv; ++h) {
        const int tiles = Line::tiles(a, s, rb);
        const auto it = got.find({b, h, rb});
        CHECK((it != got.end()) == (tiles > 0));
        if (tiles == 0) continue;
        int next = 0;
        for (const Part& p : it->second) {
          CHECK(p.t0 == next);
          next += p.tiles;
        }
        CHECK(next == tiles);
        if (it->second.size() == 1) continue;
        ++cut_blocks;
        const auto at = cut_by.find({b, h, rb});
        CHECK(at != cut_by.end());
        const int w = at->second;
        const Cut& cut = a.cuts[w];
        CHECK(cut.n_parts == static_cast<int>(it->second.size()) && cut.q0 == s.q0 && cut.n_q == s.n_q);
        for (int i = 0; i < cut.n_parts; ++i) {
          CHECK(it->second[i].slot == (i == 0 ? cut.first_slot : 2 * (w - 1 + i)));
          CHECK(it->second[i].worker == w - 1 + i);
        }
      }
    }
  }
  CHECK(cut_blocks == cut_by.size());
  return true;
}

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); };
  int bad = 0;
  for (int i = 0; i < 3000; ++i) {
    Call c;
    const int batch = pick(0, 3) ? pick(1, 12) : pick(30, 200), group = pick(1, 20), n_q = pick(0, 2) ? pick(1, 20) : pick(1, 200);
    const int max_k = pick(0, 1) ? pick(1, 700) : pick(1, 6000);
    const bool packed = pick(0, 1), back = packed && pick(0, 3) == 0;
    int total = 0;
    if (packed) {
      c.cu.push_back(0);
      for (int b = 0; b < batch; ++b) c.cu.push_back(total += pick(0, 3) ? pick(0, n_q) : 0);
      if (back) {
        for (int k = 0; k < 3; ++k) c.cu[pick(0, batch)] = pick(-2, total + 2);
      }
    }
    for (int b = 0; b < batch; ++b) c.lens.push_back(pick(0, 3) ? pick(0, max_k) : 0);
    const int workers = pick(0, 2) ? pick(1, 2) * 148 : pick(1, 2368);
    c.finish(group, pick(1, 8), n_q, total, max_k, pick(0, 1), pick(0, 1), workers);
    if (!walk(c, !back)) {
      std::printf("call %d\n", i);
      ++bad;
    }
  }
  // Queries counted thousands of times: the tiles alone stay below the limit, the blocks' own cost does not.
  struct {
    int batch, top, group, heads, keys;
  } const falling[] = {{6000, 131072, 8, 8, 256}, {1 << 16, 1 << 20, 1, 1, 128}, {1 << 16, 1 << 20, 1, 4, 1024}};
  for (const auto& f : falling) {
    Call c;
    for (int b = 0; b <= f.batch; ++b) c.cu.push_back(b % 2 ? f.top : 0);
    c.lens.assign(f.batch, f.keys);
    c.finish(f.group, f.heads, f.top, f.top, f.keys, 0, 0, 148);
    if (!walk(c, false)) {
      std::printf("%d sequences, %d queries again and again\n", f.batch, f.top);
      ++bad;
    }
  }
  // The longest sequence: its tiles, as many as there are, in shares that lie in order.
  for (const int n_q : {1, 100}) {
    Call c;
    c.lens = {MAX_KEYS, 5};
    c.finish(4, 1, n_q, 0, MAX_KEYS, 1, 1, 296);
    if (!walk(c, true) || Line::tiles(c.a, sequence(c.a, 0), 0) != (1 << 24) - 8) {
      std::printf("%d keys, %d queries\n", MAX_KEYS, n_q);
      ++bad;
    }
    c.lens[0] = MAX_KEYS + 1;
    if (sequence(c.a, 0).len != 0 || c.err != FA2_ERR_SHAPE) {
      std::printf("a longer one is not refused\n");
      ++bad;
    }
  }
  return bad ? 1 : 0;
}
