// Plan of an orthogonalisation: how the matrices of a call are padded, grouped by shape, cut into
// batches that share one piece of scratch, and where each of their operands lies.  Host arithmetic.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

namespace kfac {

// The iteration runs on matrices of r rows and c >= r columns (a taller matrix is read and written
// transposed).  Matrices of one shape, with their sides padded by zeros to whole tiles: R, C.
// Offsets are in halves from the start of the operands; of matrix k of the group
//   x[p] + k * 2RC   X, row-major [R][C]: the high halves, then the low ones (two of them: a step
//                    reads one and writes the other)
//   a    + k * 2RR   A = X X^T, in the same form
//   b    + k * 2RR   B = aI + bA + cAA
struct OrthGroup {
  int R, C, r, c;
  int count, first;      // matrices, and the first of them in the table
  int tile;              // side of the tiles its products are computed in
  int tile0, tiles;      // of the launch: first workgroup, and workgroups with a tile
  long x[2], a, b;
};

struct OrthBatch {
  int tile;
  std::vector<OrthGroup> groups;
  long halves;           // scratch for the operands
  int first, count;      // matrices of the table
};

struct OrthPlan {
  std::vector<int> order;          // table position -> matrix of the call
  std::vector<OrthBatch> batches;
  long halves = 0;                 // of the largest batch
};

constexpr int ORTH_MAX_SIDE = 16384;
constexpr int ORTH_GROUPS = 24;                  // shapes of a batch (they travel as kernel arguments)
constexpr long ORTH_BATCH_HALVES = 1L << 29;     // a batch is closed when it needs more: 1 GiB

inline int orth_pad(int n, int tile) { return (n + tile - 1) / tile * tile; }

// sides are padded to multiples of 64, 128 or 256 by the smaller of them
constexpr int ORTH_SMALL_SIDE = 128, ORTH_MID_SIDE = 512;
inline int orth_tile(int r) { return r <= ORTH_SMALL_SIDE ? 64 : r <= ORTH_MID_SIDE ? 128 : 256; }

inline OrthPlan orth_plan(int count, const int* rows, const int* cols) {
  OrthPlan p;
  for (int i = 0; i < count; ++i)
    if (rows[i] > 0 && cols[i] > 0) p.order.push_back(i);
  const auto lo = [&](int i) { return std::min(rows[i], cols[i]); };
  const auto hi = [&](int i) { return std::max(rows[i], cols[i]); };
  // longest reductions first, so that a launch does not end with them; equal shapes side by side
  std::stable_sort(p.order.begin(), p.order.end(), [&](int i, int j) {
    const int ti = orth_tile(lo(i)), tj = orth_tile(lo(j));
    if (ti != tj) return ti > tj;
    if (hi(i) != hi(j)) return hi(i) > hi(j);
    return lo(i) > lo(j);
  });
  for (size_t at = 0; at < p.order.size(); ++at) {
    const int i = p.order[at], r = lo(i), c = hi(i), tile = orth_tile(r);
    const long R = orth_pad(r, tile), C = orth_pad(c, tile), need = 4 * R * C + 4 * R * R;
    OrthBatch* b = p.batches.empty() ? nullptr : &p.batches.back();
    const bool same = b && !b->groups.empty() && b->tile == tile && b->groups.back().r == r &&
                      b->groups.back().c == c;
    if (!b || b->tile != tile || b->halves + need > ORTH_BATCH_HALVES ||
        (!same && (int)b->groups.size() == ORTH_GROUPS)) {
      p.batches.push_back(OrthBatch{tile, {}, 0, (int)at, 0});
      b = &p.batches.back();
    }
    if (b->groups.empty() || b->groups.back().r != r || b->groups.back().c != c)
      b->groups.push_back(OrthGroup{(int)R, (int)C, r, c, 0, (int)at, tile, 0, 0, {0, 0}, 0, 0});
    b->groups.back().count++;
    b->halves += need;
    b->count++;
  }
  for (OrthBatch& b : p.batches) {
    long at = 0;
    for (OrthGroup& g : b.groups) {
      const long x = 2L * g.R * g.C * g.count, a = 2L * g.R * g.R * g.count;
      g.x[0] = at;
      g.x[1] = at + x;
      g.a = at + 2 * x;
      g.b = at + 2 * x + a;
      at += 2 * x + 2 * a;
    }
    p.halves = std::max(p.halves, at);
  }
  return p;
}

// Tiles of one matrix: of a symmetric product those on and below the diagonal, or all of B X.
inline long orth_tiles(const OrthGroup& g, int tile, bool symmetric) {
  const long t = g.R / tile;
  return symmetric ? t * (t + 1) / 2 : t * (g.C / tile);
}

// Workgroups of a launch over the groups; sets their tile0 and tiles.  Workgroups go to the eight
// dies in turn, and a group starts at a multiple of eight.
inline int orth_launch(std::vector<OrthGroup>& groups, int tile, bool symmetric) {
  int at = 0;
  for (OrthGroup& g : groups) {
    g.tile0 = at;
    g.tiles = (int)(g.count * orth_tiles(g, tile, symmetric));
    at += (g.tiles + 7) / 8 * 8;
  }
  return at;
}

// The tiles that a product of the batch is computed in: 256 wide, one workgroup to a compute unit; 128
// wide, two to a unit or, where there are not as many tiles, one with more stages in flight; 64 wide.
enum { ORTH_LARGE, ORTH_MID, ORTH_DEEP, ORTH_SMALL };
constexpr long ORTH_UNITS = 256;
inline int orth_pick_tile(const OrthBatch& b, bool symmetric) {
  const auto tiles = [&](int tile) {
    long n = 0;
    for (const OrthGroup& g : b.groups) n += g.count * orth_tiles(g, tile, symmetric);
    return n;
  };
  if (b.tile == 64) return ORTH_SMALL;
  if (b.tile == 256 && tiles(256) >= ORTH_UNITS / 2) return ORTH_LARGE;
  const long n = tiles(128);
  return n > ORTH_UNITS ? ORTH_MID : n > ORTH_UNITS / 2 ? ORTH_DEEP : ORTH_SMALL;
}

}  // namespace kfac
