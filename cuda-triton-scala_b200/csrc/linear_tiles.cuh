// linear_tiles.cuh -- how the tensor-core linear layers cut their work into tiles: plain integer
// arithmetic that the kernels share, and that compiles for the host as well.
#pragma once

#include <algorithm>

#ifdef __CUDACC__
#define QG_HD __host__ __device__ __forceinline__
#else
#define QG_HD inline
#endif

namespace qg {
namespace lin {

#ifndef __CUDACC__
using std::max;
using std::min;
#endif

struct Schedule {
  int E, M;         // experts, rows of x and out
  int tok_max;      // tokens of a tile at most
  int tok_round;    // tokens of a tile are a multiple of this (MMA N)
  int num_w_blocks; // weight blocks of an expert
  int band;         // token blocks of a band of the schedule
};

// The experts' rows and tiles, in shared memory.
struct Table {
  int* row0;  // [E] first row
  int* cnt;   // [E] rows (0 where the offsets are not usable)
  int* pref;  // [E + 1] tiles before the expert
};

struct Tile {
  int e, wb;   // expert, weight block
  int t0, n;   // first row of x / out, rows
};

QG_HD int blocks_of(const Schedule& p, int cnt) {
  return (cnt + p.tok_max - 1) / p.tok_max;
}

// Rows o0 .. o1 of expert e.  Offsets that are not 0 <= o[e] <= o[e+1] <= M name no rows: false,
// and none.
QG_HD bool expert_rows(const Schedule& p, const int* offsets, int e, int& o0, int& o1) {
  o0 = offsets[e];
  o1 = offsets[e + 1];
  if (o0 >= 0 && o1 >= o0 && o1 <= p.M) return true;
  o0 = o1 = 0;
  return false;
}

// Tiles at most.  Experts that share no rows stay below (the host refuses sizes that could pass
// it); offsets that fall and rise again can name the same rows for every other expert, and 512
// times the tiles of M rows would wrap an int.  Such offsets name no rows at all.
constexpr long long kMostTiles = 1ll << 30;

// Tiles before an expert (or of all), as the table has them.
QG_HD int tiles_before(long long before, long long all) {
  return all <= kMostTiles ? (int)before : 0;
}

// Tile `t` of the schedule.  An expert's rows are cut into blocks of equal size (rounded up
// to tok_round).  Order inside an expert: bands of `band` token blocks; in a band the token
// block runs fastest, so CTAs that work at the same time share weights and tokens in L2.
QG_HD Tile tile_of(const Schedule& p, const Table& tb, int t, int band) {
  int e = 0;
  if (p.E > 1) {  // the last expert whose first tile is <= t (experts without rows have none)
    int lo = 0, hi = p.E;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (tb.pref[mid] <= t) lo = mid; else hi = mid;
    }
    e = lo;
  }
  const int idx = t - tb.pref[e], cnt = tb.cnt[e];
  const int nblk = blocks_of(p, cnt);
  const int blk = (((cnt + nblk - 1) / nblk) + p.tok_round - 1) / p.tok_round * p.tok_round;
  band = min(band, nblk);
  const int per_band = band * p.num_w_blocks;
  const int b = idx / per_band, in = idx - b * per_band;
  const int rows = min(nblk - b * band, band);
  Tile r;
  r.e = e;
  r.wb = in / rows;
  const int first = (b * band + in % rows) * blk;
  r.t0 = tb.row0[e] + first;
  r.n = max(0, min(blk, cnt - first));
  return r;
}

// Item i of pair `pid`: a whole tile in the full rounds; in the last round the `rest` tiles
// that are left are cut along their tokens into up to four parts, one a pair, so that the
// round takes a part's time.  Returns false when there is none; an item may have no tokens.
QG_HD bool pair_item(const Schedule& p, const Table& tb, int pid, int npairs, int i, Tile& r) {
  const int T = tb.pref[p.E];
  const int rounds = T / npairs, rest = T - rounds * npairs;
  if (i < rounds) {
    r = tile_of(p, tb, pid + i * npairs, p.band);
    return true;
  }
  if (i > rounds || rest == 0) return false;
  const int parts = min(4, npairs / rest);
  if (pid >= rest * parts) return false;
  r = tile_of(p, tb, rounds * npairs + pid / parts, p.band);
  if (parts > 1) {
    const int w = ((r.n + parts - 1) / parts + p.tok_round - 1) / p.tok_round * p.tok_round;
    const int first = (pid % parts) * w;
    r.n = max(0, min(w, r.n - first));
    r.t0 += first;
  }
  return true;
}

}  // namespace lin
}  // namespace qg
