// The tile arithmetic of the tensor-core linear layers on the host, built with the sanitizer of
// undefined behaviour: every row of every expert meets every weight block once, no tile leaves
// its expert's rows, and offsets that name the same rows over and over do not wrap the counts.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "linear_tiles.cuh"

using namespace qg::lin;

#define CHECK(c)                                              \
  do {                                                        \
    if (!(c)) {                                               \
      std::printf("line %d: %s\n", __LINE__, #c);             \
      std::exit(1);                                           \
    }                                                         \
  } while (0)

struct Host {
  std::vector<int> row0, cnt, pref;
  Table t;
  bool bad = false;
};

// The table as the kernels' fill_table leaves it, one expert after the other.
static void fill(const Schedule& p, const std::vector<int>& off, Host& h) {
  h.row0.resize(p.E);
  h.cnt.resize(p.E);
  h.pref.resize(p.E + 1);
  std::vector<int> tiles(p.E);
  long long all = 0;
  for (int e = 0; e < p.E; ++e) {
    int o0, o1;
    if (!expert_rows(p, off.data(), e, o0, o1)) h.bad = true;
    h.row0[e] = o0;
    h.cnt[e] = o1 - o0;
    tiles[e] = blocks_of(p, o1 - o0) * p.num_w_blocks;
    all += tiles[e];
  }
  if (all > kMostTiles) h.bad = true;
  long long run = 0;
  for (int e = 0; e < p.E; ++e) {
    h.pref[e] = tiles_before(run, all);
    run += tiles[e];
  }
  h.pref[p.E] = tiles_before(all, all);
  h.t = {h.row0.data(), h.cnt.data(), h.pref.data()};
}

static void inside(const Schedule& p, const Host& h, const Tile& t) {
  CHECK(t.e >= 0 && t.e < p.E && t.wb >= 0 && t.wb < p.num_w_blocks);
  CHECK(t.n >= 0 && t.n <= p.tok_max);
  CHECK(t.n == 0 || (t.t0 >= h.row0[t.e] && t.t0 + t.n <= h.row0[t.e] + h.cnt[t.e]));
}

static void cover(const Schedule& p, const std::vector<int>& off, int npairs) {
  Host h;
  fill(p, off, h);
  const int T = h.pref[p.E];
  std::vector<std::vector<int>> by_tile(p.E), by_pair(p.E);
  for (int e = 0; e < p.E; ++e) {
    by_tile[e].assign((size_t)h.cnt[e] * p.num_w_blocks, 0);
    by_pair[e] = by_tile[e];
  }
  auto add = [&](std::vector<std::vector<int>>& to, const Tile& t) {
    inside(p, h, t);
    for (int i = 0; i < t.n; ++i)
      ++to[t.e][(size_t)(t.t0 - h.row0[t.e] + i) * p.num_w_blocks + t.wb];
  };
  for (int t = 0; t < T; ++t) {
    const Tile r = tile_of(p, h.t, t, p.band);
    CHECK(r.n > 0);
    add(by_tile, r);
  }
  for (int pid = 0; pid < npairs; ++pid) {
    Tile r;
    for (int i = 0; pair_item(p, h.t, pid, npairs, i, r); ++i) add(by_pair, r);
  }
  for (int e = 0; e < p.E; ++e)
    for (size_t i = 0; i < by_tile[e].size(); ++i) CHECK(by_tile[e][i] == 1 && by_pair[e][i] == 1);
}

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const int toks[] = {16, 32, 48, 64, 80, 96, 128, 256};
  for (int c = 0; c < 3000; ++c) {
    Schedule p;
    p.E = pick(1, 4) == 1 ? 1 : pick(2, 40);
    p.M = pick(0, 700);
    p.tok_max = toks[pick(0, 7)];
    p.tok_round = p.tok_max >= 128 ? 32 : 16;
    p.num_w_blocks = pick(1, 9);
    p.band = pick(0, 1) ? 1 << 20 : pick(1, 5);
    std::vector<int> off(p.E + 1);
    for (int& o : off) o = pick(0, p.M);
    // sorted: what routing makes; as drawn: skipped and overlapping experts
    if (pick(0, 3)) std::sort(off.begin(), off.end());
    cover(p, off, pick(0, 1) ? 74 : pick(1, 80));
  }
  // counts near their limits: 2^30 rows, in one expert and spread
  for (int E : {1, 7, 1024}) {
    Schedule p = {E, 1 << 30, 96, 16, 16, 1 << 20};
    std::vector<int> off(E + 1);
    for (int e = 0; e <= E; ++e) off[e] = (int)((long long)p.M * e / E);
    Host h;
    fill(p, off, h);
    CHECK(!h.bad);
    const int T = h.pref[E];
    for (int i = 0; i < 20000; ++i) {
      const int t = i < 100 ? i : i < 200 ? T - 1 - (i - 100) : pick(0, T - 1);
      inside(p, h, tile_of(p, h.t, t, p.band));
    }
  }
  // every other expert names all rows: 512 x 43691 x 96 tiles are past 2^31
  Schedule p = {1024, 1 << 22, 96, 16, 96, 1 << 20};
  std::vector<int> off(p.E + 1);
  for (int e = 0; e <= p.E; ++e) off[e] = e % 2 ? p.M : 0;
  Host h;
  fill(p, off, h);
  CHECK(h.bad);
  const int T = h.pref[p.E];
  CHECK(T >= 0);
  for (int i = 0; i < 20000 && T > 0; ++i) {
    const int t = i < 100 ? i : pick(0, T - 1);
    inside(p, h, tile_of(p, h.t, t, p.band));
  }
  std::printf("ok\n");
  return 0;
}
