// Plan of an orthogonalisation: how the matrices of a call are padded, grouped by shape, cut into
// batches that share one piece of scratch, and where each of their operands lies.  Host arithmetic.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <vector>

namespace kfac {

// The iteration runs on matrices of r rows and c >= r columns (a taller matrix is read and written
// transposed).  Matrices of one shape, with their sides padded by zeros to whole tiles: R, C.
// Offsets are in halves from the start of the operands; of matrix k of the group
//   x[p] + k * 2RC   X, [R][C], room for two parts (two of them: a step reads one and writes the other)
//   a    + k * 2RR   A = X X^T, in the same form
//   b    + k * 2RR   B = aI + bA + cAA
struct OrthGroup {
  int R, C, r, c;
  int count, first;      // matrices, and the first of them in the table
  int pad;               // R and C are multiples of it
  long x[2], a, b;
};

struct OrthBatch {
  int pad;               // of its largest matrices
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

// Sides are padded to multiples of 64 where the smaller one is at most this, else of 128, or of 256
// where the smaller one is more than ORTH_MID_SIDE and such matrices hold as many 256-wide tiles as
// half of the chip takes (they are in batches of their own then).
constexpr int ORTH_SMALL_SIDE = 64, ORTH_MID_SIDE = 512;
constexpr long ORTH_UNITS = 256;           // compute units

// tiles on and below the diagonal
inline long orth_triangle(long t) { return t * (t + 1) / 2; }

// Matrices that a workgroup iterates on by itself, in LDS, with sides padded to multiples of 32.  64 x 64 takes
// 27 us and 16 x 20 15, where the seventeen launches of the others take about 90 even with next to nothing to
// do.  Larger ones (64 x 256 50 us) are left to those launches, in which they cost nothing beside others.
constexpr int ORTH_TINY_SIDE = 64, ORTH_TINY_SIZE = 4096;
constexpr int ORTH_MAX_STEPS = 64;               // of an iteration (their coefficients travel as kernel arguments)
// A schedule whose operands fit fp16 numbers times 2^13, up to 7.99: with |X| = t in the spectral norm at most
// `bound` in front of a step, A has t^2, B |a + b t^2 + c t^4| and the next X |a t + b t^3 + c t^5|.  (Two per
// cent for what the products round.)  growth: so many bits at most X gains in each step.
constexpr double ORTH_OPERAND_BOUND = 7.9;
inline bool orth_schedule_ok(int steps, const float* coeffs, int* growth = nullptr) {
  double bound = 1.;
  if (steps < 1 || steps > ORTH_MAX_STEPS) return false;
  for (int k = 0; k < steps; ++k) {
    const double a = coeffs[3 * k], b = coeffs[3 * k + 1], c = coeffs[3 * k + 2], end = bound * bound;
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
    double value = 0., factor = 0.;
    // at s = t^2: the ends, and where the derivatives of the two vanish
    const auto look = [&](double s) {
      if (!(s >= 0. && s <= end)) return;
      const double f = std::fabs(a + (b + c * s) * s);
      factor = std::max(factor, f);
      value = std::max(value, f * std::sqrt(s));
    };
    look(0.);
    look(end);
    if (c == 0.) {
      if (b != 0.) look(-a / (3. * b));
    } else {
      look(-b / (2. * c));
      const double d = 9. * b * b - 20. * a * c;
      if (d >= 0.)
        for (double root : {std::sqrt(d), -std::sqrt(d)}) look((-3. * b + root) / (10. * c));
    }
    bound = value;
    // (the caller's coefficients may have been rounded to float32)
    if (!(1.02 * std::max(bound, std::max(bound * bound, factor)) <= ORTH_OPERAND_BOUND * (1. + 1e-5))) return false;
    if (growth) growth[k] = std::max(0, (int)std::ceil(std::log2(std::max(1.02 * factor, 0.5))));
  }
  return true;
}

inline bool orth_tiny(int rows, int cols) {
  const int R = orth_pad(std::min(rows, cols), 32), C = orth_pad(std::max(rows, cols), 32);
  return R <= ORTH_TINY_SIDE && R * C <= ORTH_TINY_SIZE;
}

// without_tiny: those are left out
inline OrthPlan orth_plan(int count, const int* rows, const int* cols, bool without_tiny = false) {
  OrthPlan p;
  for (int i = 0; i < count; ++i)
    if (rows[i] > 0 && cols[i] > 0 && !(without_tiny && orth_tiny(rows[i], cols[i]))) p.order.push_back(i);
  const auto lo = [&](int i) { return std::min(rows[i], cols[i]); };
  const auto hi = [&](int i) { return std::max(rows[i], cols[i]); };
  long large = 0;
  for (int i : p.order)
    if (lo(i) > ORTH_MID_SIDE) large += orth_triangle(orth_pad(lo(i), 256) / 256);
  const auto pad = [&](int i) {
    const int r = lo(i);
    return r <= ORTH_SMALL_SIDE ? 64 : r <= ORTH_MID_SIDE || large < ORTH_UNITS / 2 ? 128 : 256;
  };
  // longest reductions first, so that a launch does not end with them; equal shapes side by side
  std::stable_sort(p.order.begin(), p.order.end(), [&](int i, int j) {
    const bool li = pad(i) == 256, lj = pad(j) == 256;
    if (li != lj) return li;
    if (hi(i) != hi(j)) return hi(i) > hi(j);
    return lo(i) > lo(j);
  });
  for (size_t at = 0; at < p.order.size(); ++at) {
    const int i = p.order[at], r = lo(i), c = hi(i), side = pad(i);
    const bool is_large = side == 256;
    const long R = orth_pad(r, side), C = orth_pad(c, side), need = 4 * R * C + 4 * R * R;
    OrthBatch* b = p.batches.empty() ? nullptr : &p.batches.back();
    const bool same = b && b->groups.back().r == r && b->groups.back().c == c;
    if (!b || (b->pad == 256) != is_large || b->halves + need > ORTH_BATCH_HALVES ||
        (!same && (int)b->groups.size() == ORTH_GROUPS)) {
      p.batches.push_back(OrthBatch{0, {}, 0, (int)at, 0});
      b = &p.batches.back();
    }
    if (b->groups.empty() || b->groups.back().r != r || b->groups.back().c != c)
      b->groups.push_back(OrthGroup{(int)R, (int)C, r, c, 0, (int)at, side, {0, 0}, 0, 0});
    b->pad = std::max(b->pad, side);
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

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------

// The kernels' tiles: 256 wide, one workgroup to a compute unit; 128 wide, two to a unit (in such a launch
// matrices padded to 64 have 64-wide tiles); 64 wide, one to a unit with more stages of its operands in
// flight (DEEP), or two.
enum { ORTH_LARGE, ORTH_MID, ORTH_DEEP, ORTH_SMALL, ORTH_KINDS };
struct OrthKind {
  int tile, slots;       // workgroups at a time
  float unit, ends, poly_ends;   // us for 64 reduction steps of a tile, in two parts, and to start and end it
                                 // (of B, which reads A and is written twice), with all slots taken
};
// From 16 matrices of 1024 x 2752, 8 of 2048^2 and of 512 x 2048, a ResNet-50's, 784-1000-1000-10 and AlexNet's
// layers, each in all kinds that the padding allows (large / mid / deep / small), us with the second launch for pieces:
//   A  200 218 - - - 570 / 169 208 30 64 21 640 / 232 333 31 69 14 1031 / 207 291 25 60 16 974
//   B  98 228 - - - 351 / 82 219 19 36 23 382 / 114 349 17 36 14 668 / 98 291 12 27 17 633
//   BX 249 313 - - - 948 / 293 369 28 86 27 1118 / 543 721 52 158 21 2079 / 445 598 39 112 17 1918
constexpr OrthKind ORTH_KIND[ORTH_KINDS] = {{256, 256, 4.3f, 11.f, 20.f},
                                            {128, 512, 2.7f, 6.5f, 6.5f},
                                            {64, 256, 0.63f, 4.5f, 4.5f},
                                            {64, 512, 1.f, 3.f, 3.f}};

enum { ORTH_GRAM, ORTH_POLY, ORTH_APPLY };

// What a launch does for a group.  Of its tiles the first `whole` are a workgroup each, from workgroup
// tile0 on; every other one is cut along the reduction into `cuts` pieces of `len` (in units of 64
// steps; the last may be shorter), a workgroup each from piece0 on, whose sums a second launch adds up.
struct OrthSlice {
  int tile, tiles, whole, cuts, len, tile0, piece0, fix0;
};
struct OrthLaunch {
  int kind = 0;
  std::vector<OrthSlice> slices;
  int pieces0 = 0, blocks = 0, fixes = 0;      // first piece, all workgroups, cut tiles
};

inline long orth_tiles(const OrthGroup& g, int tile, int product) {
  const long t = g.R / tile;
  return g.count * (product == ORTH_APPLY ? t * (g.C / tile) : orth_triangle(t));
}
inline int orth_length(const OrthGroup& g, int product) { return (product == ORTH_GRAM ? g.C : g.R) / 64; }

// When the last of the items is done, each taken by the slot that is free first, in order.
struct OrthClock {
  std::vector<std::pair<float, long>> free;     // (time, slots), earliest first
  float end = 0.f;
  explicit OrthClock(long slots) { free.push_back({0.f, slots}); }
  // items that a slot can end by `until`; the rest is not taken
  long take(float length, long n, float until = 1e30f) {
    long taken = 0;
    while (taken < n) {
      const float t = free.front().first + length;
      if (t > until) break;
      const long k = std::min(n - taken, free.front().second);
      if ((free.front().second -= k) == 0) free.erase(free.begin());
      const auto at = std::lower_bound(free.begin(), free.end(), t,
                                       [](const std::pair<float, long>& f, float v) { return f.first < v; });
      if (at != free.end() && at->first == t) at->second += k;
      else free.insert(at, {t, k});
      end = std::max(end, t);
      taken += k;
    }
    return taken;
  }
};

constexpr int ORTH_MIN_PIECE = 4;                 // a shorter one writes its sums for too little work
constexpr long ORTH_PARTIAL_BYTES = 64L << 20;    // of all pieces

// Room for the pieces of a batch's launches, which no schedule exceeds.  A piece is a sixteenth or more of the
// longest tile's length, in which ORTH_NARROW of a narrow tile's reduction count, and ORTH_MIN_PIECE or more.
constexpr float ORTH_NARROW = 0.6f;
inline long orth_partial_bytes(const OrthBatch& b) {
  long most = 0;
  for (int product : {ORTH_GRAM, ORTH_POLY, ORTH_APPLY})
    for (const OrthKind& K : ORTH_KIND) {
      if (K.tile > b.pad) continue;
      long pieces = 0;
      for (const OrthGroup& g : b.groups) {
        const int all = orth_length(g, product), tile = std::min(K.tile, g.pad);
        const long c = std::min((int)((tile < K.tile ? 16.f / ORTH_NARROW : 16.f) + 1.f),
                                (all + ORTH_MIN_PIECE - 1) / ORTH_MIN_PIECE);
        if (c > 1) pieces += orth_tiles(g, tile, product) * c;
      }
      most = std::max(most, pieces * K.tile * K.tile * 4);
    }
  return std::min(most, ORTH_PARTIAL_BYTES);
}

// The schedule of one kind, and its time: whole tiles as long as they keep all slots busy, the rest cut
// if that gains more than the second launch and the pieces' sums cost.
inline float orth_schedule(const OrthBatch& b, int product, int kind, OrthLaunch& out) {
  const OrthKind& K = ORTH_KIND[kind];
  const int n = (int)b.groups.size();
  out.kind = kind;
  out.slices.assign(n, OrthSlice{});
  std::vector<float> length(n);                   // of a tile, in this kind's units
  std::vector<int> order(n);
  const float ends = (product == ORTH_POLY ? K.poly_ends : K.ends) / K.unit;
  double work = 0.;
  float longest = 0.f;
  for (int i = 0; i < n; ++i) {
    const OrthGroup& g = b.groups[i];
    OrthSlice& s = out.slices[i];
    s.tile = std::min(K.tile, g.pad);
    s.tiles = s.whole = (int)orth_tiles(g, s.tile, product);
    length[i] = orth_length(g, product) * (s.tile < K.tile ? ORTH_NARROW : 1.f) + ends;
    work += (double)length[i] * s.tiles;
    longest = std::max(longest, length[i]);
    order[i] = i;
  }
  std::stable_sort(order.begin(), order.end(), [&](int i, int j) { return length[i] > length[j]; });
  OrthClock plain(K.slots);
  for (int i : order) plain.take(length[i], out.slices[i].tiles);
  const float even = (float)(work / K.slots);
  float best = plain.end * K.unit;
  if (plain.end > 1.1f * even && plain.end * K.unit > 8.f) {
    OrthClock full(K.slots);
    std::vector<long> whole(n, 0);
    for (int i : order) {
      whole[i] = full.take(length[i], out.slices[i].tiles, 1.02f * even);
      if (whole[i] < out.slices[i].tiles) break;
    }
    int last = 0;
    for (int d : {2, 3, 4, 6, 8, 12, 16}) {
      const int piece = std::max(ORTH_MIN_PIECE, (int)((longest + d - 1) / d));
      if (piece == last) continue;
      last = piece;
      OrthClock clock = full;
      long pieces = 0;
      std::vector<OrthSlice> cut = out.slices;
      for (int i : order) {
        OrthSlice& s = cut[i];
        const int all = orth_length(b.groups[i], product), c = (all + piece - 1) / piece;
        s.cuts = 0;
        s.whole = s.tiles;
        if (whole[i] == s.tiles) continue;
        if (c < 2) {
          clock.take(length[i], s.tiles - whole[i]);
          continue;
        }
        s.whole = (int)whole[i];
        s.cuts = c;
        s.len = (all + c - 1) / c;
        const long m = (long)(s.tiles - s.whole) * c;
        clock.take((length[i] - ends) * s.len / all + ends, m);
        pieces += m;
      }
      const long bytes = pieces * K.tile * K.tile * 4;
      const float t = clock.end * K.unit + 5.f + 2.f * bytes / 3.5e6f;
      if (t < best - 10.f && bytes <= orth_partial_bytes(b)) {
        best = t;
        out.slices = cut;
      }
    }
  }
  // workgroups: whole tiles from multiples of eight on (workgroups go to the eight dies in turn), then
  // the pieces, longest first throughout
  int at = 0, fixes = 0;
  for (int i : order) {
    OrthSlice& s = out.slices[i];
    s.tile0 = at;
    at += (s.whole + 7) / 8 * 8;
  }
  out.pieces0 = at;
  for (int i : order) {
    OrthSlice& s = out.slices[i];
    s.piece0 = at;
    s.fix0 = fixes;
    if (s.cuts > 0) {
      // (a last piece without anything to do is left out)
      s.cuts = (orth_length(b.groups[i], product) + s.len - 1) / s.len;
      at += (s.tiles - s.whole) * s.cuts;
      fixes += s.tiles - s.whole;
    }
  }
  out.blocks = at;
  out.fixes = fixes;
  return best;
}

inline OrthLaunch orth_launch(const OrthBatch& b, int product) {
  OrthLaunch best;
  float time = 1e30f;
  for (int kind = b.pad == 256 ? ORTH_LARGE : b.pad == 128 ? ORTH_MID : ORTH_DEEP; kind < ORTH_KINDS; ++kind) {
    OrthLaunch l;
    const float t = orth_schedule(b, product, kind, l);
    if (t < time) {
      time = t;
      best = l;
    }
  }
  return best;
}

}  // namespace kfac
