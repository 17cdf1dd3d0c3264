// Newton-Schulz orthogonalisation of lists of matrices, and Muon's update with it.
//
//   X = G / (|G| + eps);   every step:  A = X X^T,  B = a I + b A + c A A,  X = B X
//
// A matrix whose norm is small beside eps would leave the lower end of what its operands hold (2^-38): it is
// iterated on as X 2^lift, with b 2^-2lift and c 2^-4lift, and in every step that X may gain g bits the lift
// falls by g, until it is 0.
//
// G: the matrix itself, or the direction that momentum makes of a gradient.  A pass over the inputs
// renews the momentum and sums the squares, a second one normalises and writes the operands; then
// three launches a step, each over the tiles of all matrices.  The last one writes the result in
// its own type, or decays and updates the parameters.
#include "element_types.h"
#include "orth_core.h"
#include "orth_plan.h"

#include <limits.h>
#include <string.h>

#include <exception>
#include <type_traits>

namespace kfac {
namespace {

// one matrix of the table
struct OrthMat {
  const void* in;        // gradient
  void* out;             // result or parameter
  float* buf;            // momentum, or NULL
  long numel;
  int rows, cols;
  int group, index;      // of its batch
  int sum0, sums;        // its partial sums, and the workgroups that make them
  int pack0;             // first workgroup of the second pass (within the batch)
  float step, keep;      // parameter = keep * parameter - step * result
  int aligned;           // in and buf can be read 8 elements at a time from their start
  int vec;               // ... and from the start of every row
  int wide;              // out can be written 4 elements at a time
};

constexpr int SUM_ELEMS = 4096;                  // a workgroup of the first pass
constexpr int SUM_MAX = 1024;                    // ... at most as many for a matrix
constexpr int PACK_R = 64, PACK_C = 128;         // a workgroup of the second pass

struct Momentum {
  float mu;
  int nesterov;
};

// sum over the workgroup, the same in every thread
__device__ __forceinline__ double block_sum(double v, double* tmp) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  const double s = (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
  __syncthreads();
  return s;
}

// What normalises and scales an element, in two factors: of numbers close to the ends of float32's range the
// product of the two lies outside it (a matrix of zeros would be 0 * inf).
struct OrthNorm {
  float first, second;
  int lift;              // |X| 2^lift is at least 1/2, or lift 0
};
__device__ __forceinline__ OrthNorm orth_norm(double squares, float eps) {
  const double norm = sqrt(squares), all = norm + (double)eps, share = norm / all;
  const int lift = share > 0. && share < 0.5 ? -ilogb(share) - 1 : 0;
  const double v = ldexp((double)ORTH_SCALE / all, lift);
  const double first = v > 0x1p100 ? 0x1p100 : v < 0x1p-100 ? 0x1p-60 : 1.;
  return OrthNorm{(float)first, (float)(v / first), lift};
}

// First pass: momentum, and the sum of squares in 64 bits (the squares of float32 numbers neither
// overflow nor vanish there).  Bound by memory: 58.6 million float32 elements in 54 us, 4.3 TB/s; 177
// million bfloat16 ones with their momentum, in three launches, 293 us, 6.0 TB/s of the 10 bytes each (part
// of which the caches hold).
template <class V, bool MUON>
__global__ __launch_bounds__(256) void orth_sum_kernel(const OrthMat* mats, int n, Momentum mom, double* sums) {
  __shared__ double tmp[4];
  int j = 0, end = n;
  while (end - j > 1) {
    const int mid = (j + end) >> 1;
    if (mats[mid].sum0 <= (int)blockIdx.x) j = mid; else end = mid;
  }
  const OrthMat m = mats[j];
  const int local = blockIdx.x - m.sum0;
  const V* const in = (const V*)m.in;
  double s = 0.;
  constexpr int N = 8;
  const long whole = m.aligned ? m.numel / N * N : 0;
  for (long i = ((long)local * 256 + threadIdx.x) * N; i < whole; i += (long)m.sums * 256 * N) {
    const Pack<V, N> g = *(const Pack<V, N>*)(in + i);
    float b[N];
    if (MUON) {
      Pack<float, 4>* const at = (Pack<float, 4>*)(m.buf + i);
      Pack<float, 4> b0 = at[0], b1 = at[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        b[e] = b0.v[e] = fmaf(mom.mu, b0.v[e], Element<V>::get(g.v[e]));
        b[e + 4] = b1.v[e] = fmaf(mom.mu, b1.v[e], Element<V>::get(g.v[e + 4]));
      }
      at[0] = b0;
      at[1] = b1;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float u = Element<V>::get(g.v[e]);
      if (MUON) u = mom.nesterov ? fmaf(mom.mu, b[e], u) : b[e];
      s = fma((double)u, (double)u, s);
    }
  }
  // the rest, or all where the addresses do not allow that
  const long step = (long)m.sums * 256;
  for (long i0 = whole + (long)local * 256 + threadIdx.x; i0 < m.numel; i0 += N * step) {
    float u[N], b[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const long i = i0 + e * step;
      u[e] = b[e] = 0.f;
      if (i < m.numel) {
        u[e] = Element<V>::get(in[i]);
        if (MUON) b[e] = m.buf[i];
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const long i = i0 + e * step;
      if (i >= m.numel) break;
      if (MUON) {
        m.buf[i] = b[e] = fmaf(mom.mu, b[e], u[e]);
        u[e] = mom.nesterov ? fmaf(mom.mu, b[e], u[e]) : b[e];
      }
      s = fma((double)u[e], (double)u[e], s);
    }
  }
  s = block_sum(s, tmp);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

struct OrthGroups {
  OrthGroup g[ORTH_GROUPS];
};

// Second pass: X, normalised, scaled and in halves, zeros in the padding.  Bound by memory: the matrices
// above 94 us, 5.0 TB/s, and 389 us, 4.6 TB/s, of 8 and 10 bytes an element.  A matrix stored transposed goes
// through LDS, read in runs of 8 where its rows allow that (element by element the second figure is 527 us).
template <class V, bool MUON>
__global__ __launch_bounds__(256) void orth_pack_kernel(const OrthMat* mats, int n, Momentum mom, const double* sums,
                                                        float eps, half_t* base, int* lifts, OrthGroups groups,
                                                        int low) {
  __shared__ double tmp[4];
  __shared__ float tile[PACK_R][PACK_C + 1];
  int j = 0, end = n;
  while (end - j > 1) {
    const int mid = (j + end) >> 1;
    if (mats[mid].pack0 <= (int)blockIdx.x) j = mid; else end = mid;
  }
  const OrthMat m = mats[j];
  const OrthGroup& g = groups.g[m.group];
  double s = 0.;
  for (int i = threadIdx.x; i < m.sums; i += 256) s += sums[m.sum0 + i];
  s = block_sum(s, tmp);
  const OrthNorm norm = orth_norm(s, eps);
  const int across = (g.C + PACK_C - 1) / PACK_C, local = blockIdx.x - m.pack0;
  if (local == 0 && threadIdx.x == 0) lifts[j] = norm.lift;
  const int r0 = local / across * PACK_R, c0 = local % across * PACK_C;
  const int R = g.R, C = g.C;
  const V* const in = (const V*)m.in;
  const auto value = [&](long i) {
    float u = Element<V>::get(in[i]);
    if (MUON) {
      const float b = m.buf[i];
      u = mom.nesterov ? fmaf(mom.mu, b, u) : b;
    }
    return u * norm.first * norm.second;
  };
  // 8 of them that lie side by side
  const auto run = [&](long at, float (&v)[8]) {
    const Pack<V, 8> p = *(const Pack<V, 8>*)(in + at);
    float b[8];
    if (MUON) {
      *(Pack<float, 4>*)b = *(const Pack<float, 4>*)(m.buf + at);
      *(Pack<float, 4>*)(b + 4) = *(const Pack<float, 4>*)(m.buf + at + 4);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float u = Element<V>::get(p.v[e]);
      if (MUON) u = mom.nesterov ? fmaf(mom.mu, b[e], u) : b[e];
      v[e] = u * norm.first * norm.second;
    }
  };
  const bool tall = m.rows > m.cols;
  if (tall) {
    // in: rows of g.r values, as many as g.c
    if (m.vec) {
      // (a run of 8 is inside the matrix or outside; a wave's 64 runs are stored to different banks)
#pragma unroll
      for (int t = 0; t < PACK_R * PACK_C / 8 / 256; ++t) {
        const int i = threadIdx.x + t * 256, r = i % (PACK_R / 8) * 8, c = i / (PACK_R / 8);
        const bool inside = r0 + r < g.r && c0 + c < g.c;
        float v[8];
        run((long)min(c0 + c, g.c - 1) * g.r + min(r0 + r, g.r - 8), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) tile[r + e][c] = inside ? v[e] : 0.f;
      }
    } else {
      for (int i0 = threadIdx.x; i0 < PACK_R * PACK_C; i0 += 8 * 256) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // (a load under a condition would wait for the one before it)
          const int i = i0 + e * 256, r = min(r0 + i % PACK_R, g.r - 1), c = min(c0 + i / PACK_R, g.c - 1);
          v[e] = value((long)c * g.r + r);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = i0 + e * 256, r = i % PACK_R, c = i / PACK_R;
          tile[r][c] = r0 + r < g.r && c0 + c < g.c ? v[e] : 0.f;
        }
      }
    }
    __syncthreads();
  }
  half_t* const x = base + g.x[0] + (long)m.index * 2 * R * C;
  for (int i = threadIdx.x; i < PACK_R * PACK_C / 8; i += 256) {
    const int r = i / (PACK_C / 8), c = i % (PACK_C / 8) * 8;
    if (r0 + r >= R || c0 + c >= C) continue;
    float v[8];
    const long at = (long)(r0 + r) * g.c + c0 + c;
    if (tall) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile[r][c + e];
    } else if (r0 + r >= g.r) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    } else if (m.vec && c0 + c + 8 <= g.c) {
      run(at, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = value((long)(r0 + r) * g.c + min(c0 + c + e, g.c - 1));
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c0 + c + e < g.c ? v[e] : 0.f;
    }
    h8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = (half_t)v[e];
      l[e] = (half_t)(v[e] - (float)h[e]);
    }
    half_t* const to = x + orth_at(r0 + r, c0 + c, C, low);
    *(h8*)to = h;
    if (low) *(h8*)(to + 32) = l;
  }
}

enum { GRAM = ORTH_GRAM, POLY = ORTH_POLY, APPLY = ORTH_APPLY, LAST };

struct OrthProduct {
  half_t* base;
  float* partial;        // sums of the pieces, a tile each
  const OrthMat* mats;
  const int* lifts;
  float ca, cb, cc;      // of this step
  int fallen, growth;    // the lifts have fallen by so much before this step, and fall by this behind it
  int from;              // which X is read (the other one is written)
  int low;               // APPLY: the next step reads X in two parts
  int type, update;      // LAST: type of the result; parameters are updated with it
  int pieces0;
  int tile0[ORTH_GROUPS], piece0[ORTH_GROUPS], fix0[ORTH_GROUPS];     // (beyond any workgroup: no group)
  OrthGroup g[ORTH_GROUPS];
  OrthSlice s[ORTH_GROUPS];
};
static_assert(sizeof(OrthProduct) <= 4096, "kernel arguments");

// the last group that starts at or before `at` (the starts grow)
__device__ __forceinline__ int orth_find(const int (&starts)[ORTH_GROUPS], int at) {
  int gi = -1;
#pragma unroll
  for (int i = 0; i < ORTH_GROUPS; ++i) gi += starts[i] <= at;
  return __builtin_amdgcn_readfirstlane(gi);
}

// Four elements of a result, columns c ... c + 3 of row r of the matrix as it is stored.
template <class V>
__device__ __forceinline__ void orth_store(const OrthMat& mat, int r, int c, f4 v, int update) {
  if (r >= mat.rows || c >= mat.cols) return;
  V* const out = (V*)mat.out + (long)r * mat.cols + c;
  if (mat.wide) {
    Pack<V, 4> o;
    if (update) o = *(const Pack<V, 4>*)out;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o.v[e] = Element<V>::put(update ? mat.keep * Element<V>::get(o.v[e]) - mat.step * v[e] : v[e]);
    *(Pack<V, 4>*)out = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < mat.cols)
      out[e] = Element<V>::put(update ? mat.keep * Element<V>::get(out[e]) - mat.step * v[e] : v[e]);
}

typedef OrthTile<64, 64, 2, 2, 2, false, 2> SmallTile;
typedef OrthTile<64, 64, 2, 2, 4, false, 2> DeepTile;
typedef OrthTile<128, 128, 2, 4, 2, true> MidTile;
typedef OrthTile<256, 256, 2, 4, 2, true> LargeTile;

// A tile of a group: of matrix k, rows tm of P and tn of Q.
template <int MODE>
__device__ __forceinline__ void orth_place(const OrthGroup& g, int tile, int t, int& k, int& tm, int& tn) {
  const int rt = g.R / tile;
  if (MODE == GRAM || MODE == POLY) {
    const int per = rt * (rt + 1) / 2, u = t % per;
    k = t / per;
    tm = (int)((sqrtf(8.f * u + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > u) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= u) ++tm;
    tn = u - tm * (tm + 1) / 2;
  } else {
    const int per = rt * (g.C / tile), u = t % per;
    k = t / per;
    tm = u / rt;
    tn = u % rt;
  }
}

// The coefficients of matrices that are lifted, and the factor of BX: to the next step's lift, or to none.
struct OrthFactors {
  float b, c, x;
};
template <int MODE>
__device__ __forceinline__ OrthFactors orth_factors(const OrthProduct& p, int lift) {
  constexpr float INV = 1.f / ORTH_SCALE;
  const int now = max(0, lift - p.fallen), next = MODE == LAST ? 0 : max(0, now - p.growth);
  return OrthFactors{ldexpf(p.cb, -2 * now), ldexpf(p.cc, -4 * now), ldexpf(MODE == LAST ? INV * INV : INV, next - now)};
}

// What a product's sums become: B = aI + bA + cAA, or they are it.  Elements D[m ... m + 3][n].
template <int MODE, bool SPLIT>
__device__ __forceinline__ f4 orth_value(const OrthProduct& p, const OrthFactors& f, const OrthGroup& g, int k, int m, int n,
                                         f4 v) {
  constexpr float INV = 1.f / ORTH_SCALE;
  if (MODE == APPLY || MODE == LAST) return v * f.x;
  v *= INV;
  if (MODE == POLY) {
    const half_t* const from = p.base + g.a + (long)k * 2 * g.R * g.R + orth_at(n, m, g.R, SPLIT);
    const h4 ah = *(const h4*)from;
    h4 al = {0, 0, 0, 0};
    if (SPLIT) al = *(const h4*)(from + 32);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = fmaf(f.c, v[e], f.b * ((float)ah[e] + (float)al[e]));
      if (m + e == n) v[e] += p.ca * ORTH_SCALE;
    }
  }
  return v;
}

// Where a product goes, its rows' length, and whether in two parts.
template <int MODE, bool SPLIT>
__device__ __forceinline__ half_t* orth_target(const OrthProduct& p, const OrthGroup& g, int k, int& ld, bool& low) {
  constexpr bool SYM = MODE == GRAM || MODE == POLY;
  ld = SYM ? g.R : g.C;
  low = SYM ? SPLIT : p.low;
  return p.base + (MODE == GRAM ? g.a : MODE == POLY ? g.b : g.x[1 - p.from]) + (long)k * 2 * g.R * ld;
}

// Writes the elements of a wave, FM x FN blocks from D[m0][n0] on: D[m][n] to row n, and for a symmetric
// product also to row m (`mirror`).  A lane holds pieces of four along m of 16 rows n, which would reach
// memory 32 bytes at a time (two, of the mirror image): they go through LDS, sixteen rows at a time, and
// leave it as whole rows of the wave's part.  Without that a product of 16 matrices of 1024^2 spends 40 of
// 113 us on writing.
template <class TILE, bool SPLIT, int MODE>
__device__ __forceinline__ void orth_write(const OrthProduct& p, const OrthFactors& factors, const OrthGroup& g,
                                           const OrthMat& mat, int k, int m0, int n0, bool mirror,
                                           f4 (&acc)[TILE::FM][TILE::FN], lds_char* lds, int lane) {
  constexpr int FM = TILE::FM, FN = TILE::FN;
  typedef __attribute__((address_space(3))) half_t lds_half;
  typedef __attribute__((address_space(3))) h4 lds_h4;
  typedef __attribute__((address_space(3))) f4 lds_f4;
  typedef __attribute__((address_space(3))) float lds_float;
  int ld = 0;
  bool low = false;
  half_t* const out = MODE == LAST ? nullptr : orth_target<MODE, SPLIT>(p, g, k, ld, low);
  // 16 rows from `row0` on of W elements from column `col0` on, from LDS to memory
  const auto rows_out = [&](auto width, int pitch, int row0, int col0) {
    constexpr int W = decltype(width)::value;
    asm volatile("" : "+v"(lane));     // (addresses are formed here, or all of a tile's would be kept in registers)
    // (rolled up: the code of a whole tile has to stay in the instruction cache)
    if (MODE == LAST) {
#pragma unroll 1
      for (int t = 0; t < W / 16; ++t) {
        const int at = t * 64 + lane, row = at / (W / 4), c = at % (W / 4) * 4;
        const f4 v = *(lds_f4*)(lds + row * pitch + c * 4);
        if (p.type == TYPE_F32) orth_store<float>(mat, row0 + row, col0 + c, v, p.update);
        else if (p.type == TYPE_BF16) orth_store<__hip_bfloat16>(mat, row0 + row, col0 + c, v, p.update);
        else orth_store<half_t>(mat, row0 + row, col0 + c, v, p.update);
      }
    } else if (low) {
#pragma unroll 2
      for (int t = 0; t < W / 16; ++t) {
        const int at = t * 64 + lane, row = at / (W / 4), c = at % (W / 4) * 16;
        *(f4*)((char*)(out + orth_at(row0 + row, col0, ld, true)) + c) = *(lds_f4*)(lds + row * pitch + c);
      }
    } else {
#pragma unroll 2
      for (int t = 0; t < W / 32; ++t) {
        const int at = t * 64 + lane, row = at / (W / 8), c = at % (W / 8) * 16;
        *(f4*)((char*)(out + orth_at(row0 + row, col0, ld, false)) + c) = *(lds_f4*)(lds + row * pitch + c);
      }
    }
  };
  // (a result whose matrix is stored transposed has m down its rows)
  const bool tall = MODE == LAST && mat.rows > mat.cols;
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    asm volatile("" : "+v"(lane));
    const int nl = lane & 15, ml = 4 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      acc[i][j] = orth_value<MODE, SPLIT>(p, factors, g, k, m0 + 16 * i + ml, n0 + 16 * j + nl, acc[i][j]);
      if (tall) continue;
      lds_char* const row = lds + nl * TILE::M_PITCH;
      const int c = 16 * i + ml;
      if (MODE == LAST) {
        *(lds_f4*)(row + c * 4) = acc[i][j];
      } else {
        h4 h, l;
        split4(acc[i][j], h, l);
        lds_h4* const to = (lds_h4*)(row + 2 * (int)orth_at(0, c, 0, low));
        *to = h;
        if (low) to[8] = l;
      }
    }
    if (tall) continue;
    wave_fence();
    rows_out(std::integral_constant<int, FM * 16>(), TILE::M_PITCH, n0 + 16 * j, m0);
    wave_fence();
  }
  if (!mirror && !tall) return;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    asm volatile("" : "+v"(lane));
    const int nl = lane & 15, ml = 4 * (lane >> 4);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int c = 16 * j + nl;
      h4 h, l;
      asm volatile("" : "+v"(acc[i][j]));     // (or the parts of the whole tile would be kept from above)
      split4(acc[i][j], h, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lds_char* const row = lds + (ml + e) * TILE::N_PITCH;
        if (MODE == LAST) {
          *(lds_float*)(row + c * 4) = acc[i][j][e];
        } else {
          lds_half* const to = (lds_half*)row + orth_at(0, c, 0, low);
          *to = h[e];
          if (low) to[32] = l[e];
        }
      }
    }
    wave_fence();
    rows_out(std::integral_constant<int, FN * 16>(), TILE::N_PITCH, m0 + 16 * i, n0);
    wave_fence();
  }
}

template <class TILE, bool SPLIT, int MODE>
__device__ __forceinline__ void orth_item(const OrthProduct& p, const OrthGroup& g, const OrthSlice& s, int t, int piece,
                                          long partial, lds_char* lds) {
  constexpr bool SYM = MODE == GRAM || MODE == POLY;
  constexpr int T = TILE::TM, FM = TILE::FM, FN = TILE::FN, UNIT = SPLIT ? 2 : 1;    // stages of 64 steps
  static_assert(TILE::TM == TILE::TN, "symmetric products");
  int k, tm, tn;
  orth_place<MODE>(g, T, t, k, tm, tn);
  // (divisions leave them in vector registers)
  k = __builtin_amdgcn_readfirstlane(k);
  tm = __builtin_amdgcn_readfirstlane(tm);
  tn = __builtin_amdgcn_readfirstlane(tn);
  piece = __builtin_amdgcn_readfirstlane(piece);
  const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = all % TILE::WAVES, team = all / TILE::WAVES;
  const int wm = wave / TILE::WN, wn = wave % TILE::WN, R = g.R, C = g.C;
  const long XS = (long)R * C, AS = (long)R * R;
  const half_t* const x = p.base + g.x[p.from] + k * 2 * XS;
  const half_t* const a = p.base + g.a + k * 2 * AS;
  const half_t* const b = p.base + g.b + k * 2 * AS;
  OrthOperand<TILE::TM, TILE::WAVES, FM, !SYM, SPLIT> P;   // (columns of X, or rows of X or A)
  OrthOperand<TILE::TN, TILE::WAVES, FN, false, SPLIT> Q;
  if (MODE == POLY) P.init(a, R, tm * T, wm, wave, lane);
  else P.init(x, C, tm * T, wm, wave, lane);
  if (MODE == GRAM) Q.init(x, C, tn * T, wn, wave, lane);
  else Q.init(MODE == POLY ? a : b, R, tn * T, wn, wave, lane);
  int steps = (MODE == GRAM ? C : R) / 64;
  if (piece >= 0) {
    const int from = piece * s.len;
    P.base += from * UNIT * P.step;
    Q.base += from * UNIT * Q.step;
    steps = min(s.len, steps - from);
  }
  steps *= UNIT;
  const int lift = MODE == GRAM ? 0 : p.lifts[g.first + k];
  f4 acc[FM][FN];
  if constexpr (TILE::PAIR) orth_pair_product<TILE, SPLIT>(P, Q, steps, lds, wave, acc);
  else orth_product<TILE, SPLIT>(P, Q, steps, lds, wave, team, acc);
  if (team > 0) return;
  if (piece >= 0) {
    f4* const to = (f4*)(p.partial + partial * T * T) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) to[(i * FN + j) * TILE::TEAM] = acc[i][j];
    return;
  }
  OrthMat mat;
  if (MODE == LAST) mat = p.mats[g.first + k];
  const OrthFactors factors = orth_factors<MODE>(p, lift);
  orth_write<TILE, SPLIT, MODE>(p, factors, g, mat, k, tm * T + wm * FM * 16, tn * T + wn * FN * 16, SYM && tm != tn,
                                acc, lds + TILE::SUMS + wave * TILE::WRITE, lane);
}

// One launch: the tiles of all groups, or pieces of them.  256-wide tiles run at 1390 TFLOP/s of fp16 products
// (BX of AlexNet's layers, three products a number: 463 of float32 quality; the matrix cores busy 81 % of the
// cycles at the 1.6 GHz that the power leaves), 1200 where a launch is one round of tiles and its tail; 128-wide
// ones, two workgroups to a unit, at 1140 (A of 16 matrices of 1024 x 2752), both near what the library's own
// fp16 product of 8192^3 reaches, 1250.  64-wide ones wait for their loads: at 660 (A of a ResNet-50's matrices)
// they ask the dies' caches for 13 TB/s, of which 36 % miss and come from the last cache at 4.8 TB/s (which of
// the two is the limit was not measured); but they fill the chip where there are few tiles.
template <class TILE, bool SPLIT, int MODE>
__global__ __launch_bounds__(TILE::THREADS, TILE::LDS > 80 * 1024 ? 2 : 4) void orth_product_kernel(const OrthProduct p) {
  extern __shared__ __align__(16) char smem[];
  lds_char* const lds = (lds_char*)smem;
  const int block = blockIdx.x;
  int t, piece = -1, gi;
  long partial = 0;
  if (block < p.pieces0) {
    gi = orth_find(p.tile0, block);
    const int whole = p.s[gi].whole, local = block - p.tile0[gi], each = (whole + 7) / 8;
    t = (local & 7) * each + (local >> 3);     // neighbours in the tile order share a die's cache
    if (t >= whole) return;
  } else {
    gi = orth_find(p.piece0, block);
    const int local = block - p.piece0[gi], cuts = p.s[gi].cuts;
    t = p.s[gi].whole + local / cuts;
    piece = local % cuts;
    partial = block - p.pieces0;
  }
  const OrthGroup& g = p.g[gi];
  const OrthSlice& s = p.s[gi];
  if constexpr (TILE::TM == 128) {
    if (s.tile == 64) {
      orth_item<SmallTile, SPLIT, MODE>(p, g, s, t, piece, partial * 4, lds);
      return;
    }
  }
  orth_item<TILE, SPLIT, MODE>(p, g, s, t, piece, partial, lds);
}

// Adds up the pieces of cut tiles, in order; a workgroup takes two rows of fragments of a tile (32 rows of
// each wave's part, a whole piece of the operands' layout).  7 to 16 us.  The last piece to end adding up
// the others instead, in the products' launch, needs fences between the dies' caches that cost more: 17 -> 78 us
// for A of 517 x 301, 1263 x 517 and 37 x 1263.
template <class TILE, bool SPLIT, int MODE>
__device__ __forceinline__ void orth_fix_item(const OrthProduct& p, int gi, int local, int i, int scale,
                                              lds_char* lds) {
  constexpr int T = TILE::TM, FM = TILE::FM, FN = TILE::FN;
  const OrthGroup& g = p.g[gi];
  const OrthSlice& s = p.s[gi];
  i *= 2;
  if (i >= FM || threadIdx.x >= TILE::TEAM) return;
  int k, tm, tn;
  orth_place<MODE>(g, T, s.whole + local, k, tm, tn);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / TILE::WN, wn = wave % TILE::WN;
  const long first = (long)(s.piece0 - p.pieces0 + local * s.cuts) * scale;
  typedef OrthTile<32 * TILE::WM, TILE::TN, TILE::WM, TILE::WN, TILE::STAGES> Rows;
  f4 sum[2][FN];
#pragma unroll
  for (int j = 0; j < 2 * FN; ++j) sum[j / FN][j % FN] = f4{0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < s.cuts; ++c) {
    const f4* const from = (const f4*)(p.partial + (first + (long)c * scale) * T * T) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < 2 * FN; ++j) sum[j / FN][j % FN] += from[(i * FN + j) * TILE::TEAM];
  }
  const int m = tm * T + wm * FM * 16 + 16 * i, n0 = tn * T + wn * FN * 16;
  OrthMat mat;
  if (MODE == LAST) mat = p.mats[g.first + k];
  const OrthFactors factors = orth_factors<MODE>(p, MODE == GRAM ? 0 : p.lifts[g.first + k]);
  orth_write<Rows, SPLIT, MODE>(p, factors, g, mat, k, m, n0, MODE != LAST && MODE != APPLY && tm != tn, sum,
                                lds + wave * Rows::WRITE, lane);
}

template <class TILE, bool SPLIT, int MODE>
__global__ __launch_bounds__(TILE::TEAM) void orth_fix_kernel(const OrthProduct p) {
  constexpr int PITCH = 64 * (TILE::FN > 2 ? TILE::FN : 2) + 16;
  __shared__ __align__(16) char smem[TILE::WAVES * 16 * PITCH];
  lds_char* const lds = (lds_char*)smem;
  const int cut = blockIdx.x / (TILE::FM / 2), i = blockIdx.x % (TILE::FM / 2), gi = orth_find(p.fix0, cut);
  const int local = cut - p.fix0[gi];
  if constexpr (TILE::TM == 128) {
    if (p.s[gi].tile == 64) {
      orth_fix_item<SmallTile, SPLIT, MODE>(p, gi, local, i, 4, lds);
      return;
    }
  }
  orth_fix_item<TILE, SPLIT, MODE>(p, gi, local, i, 1, lds);
}

template <class TILE, bool SPLIT, int MODE>
bool launch_tiles(const OrthProduct& p, const OrthLaunch& l, hipStream_t stream) {
  const auto kernel = orth_product_kernel<TILE, SPLIT, MODE>;
  if (!enable_large_lds((const void*)kernel, TILE::LDS)) return false;
  hipLaunchKernelGGL(kernel, dim3(l.blocks), dim3(TILE::THREADS), TILE::LDS, stream, p);
  if (l.fixes > 0)
    hipLaunchKernelGGL((orth_fix_kernel<TILE, SPLIT, MODE>), dim3(l.fixes * (TILE::FM / 2)), dim3(TILE::TEAM), 0, stream,
                       p);
  return true;
}

template <class TILE, int MODE>
bool launch_parts(const OrthProduct& p, const OrthLaunch& l, bool split, hipStream_t stream) {
  return split ? launch_tiles<TILE, true, MODE>(p, l, stream) : launch_tiles<TILE, false, MODE>(p, l, stream);
}

template <int MODE>
bool launch_product(OrthProduct& p, const OrthBatch& b, const OrthLaunch& l, bool split, hipStream_t stream) {
  // groups by their first whole tile, piece or cut tile: the same order for all three; those without one
  // of a sort share its start with the group behind them, which is found
  std::vector<int> order(b.groups.size());
  for (size_t i = 0; i < order.size(); ++i) order[i] = (int)i;
  std::stable_sort(order.begin(), order.end(), [&](int i, int j) {
    const OrthSlice &u = l.slices[i], &v = l.slices[j];
    if (u.tile0 != v.tile0) return u.tile0 < v.tile0;
    return u.piece0 < v.piece0;
  });
  p.pieces0 = l.pieces0;
  for (int i = 0; i < ORTH_GROUPS; ++i) {
    const bool is = i < (int)order.size();
    if (is) {
      p.g[i] = b.groups[order[i]];
      p.s[i] = l.slices[order[i]];
    }
    p.tile0[i] = is ? p.s[i].tile0 : INT_MAX;
    p.piece0[i] = is ? p.s[i].piece0 : INT_MAX;
    p.fix0[i] = is ? p.s[i].fix0 : INT_MAX;
  }
  switch (l.kind) {
    case ORTH_SMALL: return launch_parts<SmallTile, MODE>(p, l, split, stream);
    case ORTH_DEEP: return launch_parts<DeepTile, MODE>(p, l, split, stream);
    case ORTH_MID: return launch_parts<MidTile, MODE>(p, l, split, stream);
    default: return launch_parts<LargeTile, MODE>(p, l, split, stream);
  }
}

bool launch_step(OrthProduct& p, const OrthBatch& b, const OrthLaunch (&l)[3], const float* coeffs, bool split,
                 bool next_split, bool last, hipStream_t stream) {
  p.ca = coeffs[0];
  p.cb = coeffs[1];
  p.cc = coeffs[2];
  if (!launch_product<GRAM>(p, b, l[ORTH_GRAM], split, stream) ||
      !launch_product<POLY>(p, b, l[ORTH_POLY], split, stream))
    return false;
  p.low = next_split;
  return last ? launch_product<LAST>(p, b, l[ORTH_APPLY], split, stream)
              : launch_product<APPLY>(p, b, l[ORTH_APPLY], split, stream);
}

template <class V, bool MUON>
void launch_passes(const OrthMat* mats, const OrthBatch& b, Momentum mom, double* sums, int sum_blocks,
                   int pack_blocks, float eps, half_t* base, int* lifts, bool low, hipStream_t stream) {
  hipLaunchKernelGGL((orth_sum_kernel<V, MUON>), dim3(sum_blocks), dim3(256), 0, stream, mats, b.count, mom, sums);
  OrthGroups groups;
  std::copy(b.groups.begin(), b.groups.end(), groups.g);
  hipLaunchKernelGGL((orth_pack_kernel<V, MUON>), dim3(pack_blocks), dim3(256), 0, stream, mats, b.count, mom,
                     (const double*)sums, eps, base, lifts, groups, (int)low);
}

// ---------------------------------------------------------------------------------------
// small matrices
// ---------------------------------------------------------------------------------------

template <int N>
struct TinyArgs {
  OrthMat m[N];
  float coeffs[3 * ORTH_MAX_STEPS];
  unsigned char growth[ORTH_MAX_STEPS];
  int steps, update;
  Momentum mom;
  float eps;
};
static_assert(sizeof(TinyArgs<32>) <= 4096, "kernel arguments");

constexpr int TINY_THREADS = 512, TINY_WAVES = 8;
// halves between rows in LDS of n elements: 16 bytes more, so that rows begin in different banks
__host__ __device__ constexpr int tiny_pitch(int n) { return n + 8; }
constexpr int tiny_lds(int R, int C) { return 4 * R * tiny_pitch(C) + 8 * R * tiny_pitch(R); }
// of 64 x 64, which needs most: rows cost more than columns
constexpr int TINY_LDS = tiny_lds(ORTH_TINY_SIDE, ORTH_TINY_SIZE / ORTH_TINY_SIDE);
static_assert(TINY_LDS >= tiny_lds(32, ORTH_TINY_SIZE / 32) && TINY_LDS <= 150 * 1024, "LDS of a small matrix");

// The fragments of 32 reduction steps: of rows row0 ... row0 + 15 with k along them, or of columns.
__device__ __forceinline__ h8 tiny_rows(lds_char* at, int pitch, int row0, int k0, int lane) {
  return *(__attribute__((address_space(3))) h8*)(at + 2 * ((row0 + (lane & 15)) * pitch + k0 + 8 * (lane >> 4)));
}
__device__ __forceinline__ h8 tiny_columns(lds_char* at, int pitch, int col0, int k0, int lane) {
  lds_char* const p = at + 2 * ((k0 + 8 * (lane >> 4) + ((lane & 15) >> 2)) * pitch + col0 + 4 * (lane & 3));
  const h4s u = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4s*)p);
  const h4s v = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4s*)(p + 8 * pitch));
  return __builtin_bit_cast(h8, (h8s)__builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A workgroup does all of one matrix: X, A and B in LDS in two parts, one launch for a list.  What bounds it
// are latencies: of the instructions, which no workgroup before this one has fetched, and of a chain of short
// phases.  So loops are rolled up, and where a product has fewer blocks than there are waves, these share its
// reduction.
template <class V, bool MUON, int N>
__global__ __launch_bounds__(TINY_THREADS) void orth_tiny_kernel(const TinyArgs<N> a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ double sums[TINY_WAVES];
  __shared__ f4 shares[TINY_WAVES][64];
  typedef __attribute__((address_space(3))) half_t lds_half;
  typedef __attribute__((address_space(3))) h4 lds_h4;
  typedef __attribute__((address_space(3))) h8 lds_h8;
  const OrthMat& m = a.m[blockIdx.x];
  const bool tall = m.rows > m.cols;
  const int cols = m.cols, numel = m.rows * cols;
  const int r = tall ? cols : m.rows, c = tall ? m.rows : cols;
  const int R = (r + 31) / 32 * 32, C = (c + 31) / 32 * 32, px = tiny_pitch(C), pa = tiny_pitch(R);
  lds_char* const x = (lds_char*)smem;               // two planes of R rows each
  lds_char* const A = x + 4 * R * px;
  lds_char* const B = A + 4 * R * pa;
  const int xs = 2 * R * px, as = 2 * R * pa;        // bytes to the low plane
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const V* const in = (const V*)m.in;
  for (int i = threadIdx.x; i < (4 * R * px + 8 * R * pa) / 16; i += TINY_THREADS)
    ((lds_h8*)x)[i] = h8{0, 0, 0, 0, 0, 0, 0, 0};
  // the direction, and with it the sum of squares, then the operand: a thread meets the same elements again
  // and reads the momentum that it wrote
  constexpr int K = 4;
  double s = 0.;
  OrthNorm norm{0.f, 0.f, 0};
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    for (int i0 = threadIdx.x; i0 < numel; i0 += K * TINY_THREADS) {
      float u[K], b[K];
#pragma unroll
      for (int e = 0; e < K; ++e) {
        const int i = i0 + e * TINY_THREADS;
        u[e] = b[e] = 0.f;
        if (i < numel) {
          u[e] = Element<V>::get(in[i]);
          if (MUON) b[e] = m.buf[i];
        }
      }
#pragma unroll
      for (int e = 0; e < K; ++e) {
        const int i = i0 + e * TINY_THREADS;
        if (i >= numel) break;
        if (MUON) {
          if (pass == 0) m.buf[i] = b[e] = fmaf(a.mom.mu, b[e], u[e]);
          u[e] = a.mom.nesterov ? fmaf(a.mom.mu, b[e], u[e]) : b[e];
        }
        if (pass == 0) {
          s = fma((double)u[e], (double)u[e], s);
        } else {
          const int p = i / cols, q = i - p * cols;
          lds_half* const to = (lds_half*)x + (tall ? q * px + p : p * px + q);
          const float v = u[e] * norm.first * norm.second;
          const half_t h = (half_t)v;
          *to = h;
          to[xs / 2] = (half_t)(v - (float)h);
        }
      }
    }
    if (pass == 0) {
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
      if (lane == 0) sums[wave] = s;
    }
    __syncthreads();
    if (pass == 0) {
      s = 0.;
      for (int w = 0; w < TINY_WAVES; ++w) s += sums[w];
      norm = orth_norm(s, a.eps);
    }
  }
  constexpr float INV = 1.f / ORTH_SCALE;
  const int nb = (r + 15) / 16, blocks = nb * (nb + 1) / 2, nl = lane & 15, ml = 4 * (lane >> 4);
  const int share = blocks <= TINY_WAVES / 2 ? TINY_WAVES / blocks : 1;      // waves to a block
  int lift = norm.lift;
  for (int step = 0; step < a.steps; ++step) {
    const float ca = a.coeffs[3 * step], cb = ldexpf(a.coeffs[3 * step + 1], -2 * lift),
                cc = ldexpf(a.coeffs[3 * step + 2], -4 * lift);
    const int next = max(0, lift - (int)a.growth[step]);
    const float to_next = ldexpf(INV, next - lift);
    lift = next;
    // A = X X^T, then B = aI + bA + cAA: the blocks on and below the diagonal
#pragma unroll 1
    for (int poly = 0; poly < 2; ++poly) {
      lds_char* const src = poly ? A : x;
      lds_char* const dst = poly ? B : A;
      const int pitch = poly ? pa : px, second = poly ? as : xs, K = poly ? R : C;
      for (int b0 = 0; b0 < blocks; b0 += TINY_WAVES / share) {
        const int b = b0 + wave / share;
        int i = 0;
        while ((i + 1) * (i + 2) / 2 <= b) ++i;
        const int j = b - i * (i + 1) / 2;
        f4 d0 = {0.f, 0.f, 0.f, 0.f}, d1 = d0, d2 = d0;
        if (b < blocks && wave < blocks * share) {
          for (int k = 32 * (wave % share); k < K; k += 32 * share) {
            const h8 ph = tiny_rows(src, pitch, 16 * i, k, lane), pl = tiny_rows(src + second, pitch, 16 * i, k, lane);
            const h8 qh = tiny_rows(src, pitch, 16 * j, k, lane), ql = tiny_rows(src + second, pitch, 16 * j, k, lane);
            d0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, d0, 0, 0, 0);
            d1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, d1, 0, 0, 0);
            d2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, d2, 0, 0, 0);
          }
        }
        f4 d = (d0 + d1) + d2;
        if (share > 1) {
          shares[wave][lane] = d;
          __syncthreads();
          if (wave % share == 0)
            for (int w = 1; w < share; ++w) d += shares[wave + w][lane];
        }
        if (b >= blocks || wave >= blocks * share || wave % share != 0) continue;
        d *= INV;
        const int mm = 16 * i + ml, n = 16 * j + nl;
        if (poly) {
          const h4 ah = *(lds_h4*)(A + 2 * (n * pa + mm)), al = *(lds_h4*)(A + as + 2 * (n * pa + mm));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[e] = fmaf(cc, d[e], cb * ((float)ah[e] + (float)al[e]));
            if (mm + e == n) d[e] += ca * ORTH_SCALE;
          }
        }
        h4 h, l;
        split4(d, h, l);
        *(lds_h4*)(dst + 2 * (n * pa + mm)) = h;
        *(lds_h4*)(dst + as + 2 * (n * pa + mm)) = l;
        if (i != j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            lds_half* const to = (lds_half*)dst + (mm + e) * pa + n;
            *to = h[e];
            to[as / 2] = l[e];
          }
        }
      }
      __syncthreads();
    }
    // X = B X in place: a wave reads 16 columns whole and writes them
    for (int col = 16 * wave; col < C; col += 16 * TINY_WAVES) {
      constexpr int NB = ORTH_TINY_SIDE / 16;
      f4 d[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) d[n] = f4{0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < R; k += 32) {
        const h8 ph = tiny_columns(x, px, col, k, lane), pl = tiny_columns(x + xs, px, col, k, lane);
        h8 qh[NB], ql[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          if (n >= nb) continue;
          qh[n] = tiny_rows(B, pa, 16 * n, k, lane);
          ql[n] = tiny_rows(B + as, pa, 16 * n, k, lane);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
          if (n < nb) d[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh[n], d[n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NB; ++n)
          if (n < nb) d[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql[n], d[n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NB; ++n)
          if (n < nb) d[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh[n], d[n], 0, 0, 0);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if (n >= nb) continue;
        h4 h, l;
        split4(d[n] * to_next, h, l);
        lds_char* const to = x + 2 * ((16 * n + nl) * px + col + ml);
        *(lds_h4*)to = h;
        *(lds_h4*)(to + xs) = l;
      }
    }
    __syncthreads();
  }
  const float to_result = ldexpf(INV, -lift);
#pragma unroll 2
  for (int i = threadIdx.x; i < numel; i += TINY_THREADS) {
    const int p = i / cols, q = i - p * cols;
    const lds_half* const from = (const lds_half*)x + (tall ? q * px + p : p * px + q);
    const float o = ((float)from[0] + (float)from[xs / 2]) * to_result;
    V* const to = (V*)m.out + i;
    *to = Element<V>::put(a.update ? m.keep * Element<V>::get(*to) - m.step * o : o);
  }
}

struct Layout {
  size_t table, sums, lifts, partials, operands, bytes;
};
Layout layout(const OrthPlan& plan) {
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Layout l{0, 0, 0, 0, 0, 256};
  if (plan.order.empty()) return l;        // small matrices alone
  l.sums = up(plan.order.size() * sizeof(OrthMat));
  long sums = 0, count = 0, partials = 0;
  for (const OrthBatch& b : plan.batches) {
    sums = std::max(sums, (long)b.count * SUM_MAX);
    count = std::max(count, (long)b.count);
    partials = std::max(partials, orth_partial_bytes(b));
  }
  l.lifts = l.sums + up((size_t)sums * sizeof(double));
  l.partials = l.lifts + up((size_t)count * sizeof(int));
  l.operands = l.partials + up((size_t)partials);
  l.bytes = l.operands + (size_t)plan.halves * sizeof(half_t);
  return l;
}

bool sizes_ok(int count, const int* rows, const int* cols) {
  if (count < 0 || (count > 0 && (!rows || !cols))) return false;
  for (int i = 0; i < count; ++i)
    if (rows[i] < 0 || cols[i] < 0 || rows[i] > ORTH_MAX_SIDE || cols[i] > ORTH_MAX_SIDE) return false;
  return true;
}

struct Call {
  int count;
  const int *rows, *cols;
  int type;
  const void* const* in;
  void* const* out;
  float* const* buf;                 // NULL: no momentum
  const float *step, *keep;          // NULL: the result itself is written
  Momentum mom;
  int steps;
  const float* coeffs;
  float eps;
  int late;                          // steps at the end with single products
  int growth[ORTH_MAX_STEPS];        // bits that X may gain in a step
};

template <class V, bool MUON, int N>
bool launch_tiny(const Call& c, const std::vector<int>& which, size_t first, hipStream_t stream) {
  TinyArgs<N> a;
  memset(&a, 0, sizeof(a));
  const int n = (int)std::min(which.size() - first, (size_t)N);
  int lds = 0;
  for (int k = 0; k < n; ++k) {
    const int i = which[first + k];
    OrthMat& m = a.m[k];
    m.in = c.in[i];
    m.out = c.out[i];
    m.buf = c.buf ? c.buf[i] : nullptr;
    m.rows = c.rows[i];
    m.cols = c.cols[i];
    m.step = c.step ? c.step[i] : 0.f;
    m.keep = c.keep ? c.keep[i] : 0.f;
    lds = std::max(lds, tiny_lds(orth_pad(std::min(m.rows, m.cols), 32), orth_pad(std::max(m.rows, m.cols), 32)));
  }
  std::copy(c.coeffs, c.coeffs + 3 * c.steps, a.coeffs);
  std::copy(c.growth, c.growth + c.steps, a.growth);
  a.steps = c.steps;
  a.update = c.step != nullptr;
  a.mom = c.mom;
  a.eps = c.eps;
  const auto kernel = orth_tiny_kernel<V, MUON, N>;
  if (!enable_large_lds((const void*)kernel, TINY_LDS)) return false;
  hipLaunchKernelGGL(kernel, dim3(n), dim3(TINY_THREADS), lds, stream, a);
  return true;
}

// (short lists have short arguments: they cost host time)
template <class V, bool MUON>
bool launch_tiny_list(const Call& c, const std::vector<int>& which, hipStream_t stream) {
  for (size_t first = 0; first < which.size(); first += 32)
    if (!(which.size() <= 4 ? launch_tiny<V, MUON, 4>(c, which, first, stream)
                            : launch_tiny<V, MUON, 32>(c, which, first, stream)))
      return false;
  return true;
}
template <class V>
bool launch_tiny_type(const Call& c, const std::vector<int>& which, hipStream_t stream) {
  return c.buf ? launch_tiny_list<V, true>(c, which, stream) : launch_tiny_list<V, false>(c, which, stream);
}

int run(Call& c, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (!sizes_ok(c.count, c.rows, c.cols)) return KFAC_ERR_ARG;
  if (c.count == 0) return KFAC_OK;
  if (!c.in || !c.out || !c.coeffs || !orth_schedule_ok(c.steps, c.coeffs, c.growth) || c.late < 0 || c.type < TYPE_F32 ||
      c.type > TYPE_F16 || !(c.eps > 0.f && c.eps < INFINITY))
    return KFAC_ERR_ARG;
  std::vector<int> tiny;
  for (int i = 0; i < c.count; ++i) {
    if (c.rows[i] == 0 || c.cols[i] == 0) continue;
    if (!c.in[i] || !c.out[i] || (c.buf && !c.buf[i])) return KFAC_ERR_ARG;
    if (orth_tiny(c.rows[i], c.cols[i])) tiny.push_back(i);
  }
  OrthPlan plan = orth_plan(c.count, c.rows, c.cols, true);
  if (plan.order.empty() && tiny.empty()) return KFAC_OK;
  const Layout l = layout(plan);
  if (!workspace || workspace_bytes < l.bytes) return KFAC_ERR_WORKSPACE;
  if (!tiny.empty() && !(c.type == TYPE_F32    ? launch_tiny_type<float>(c, tiny, stream)
                         : c.type == TYPE_BF16 ? launch_tiny_type<__hip_bfloat16>(c, tiny, stream)
                                               : launch_tiny_type<half_t>(c, tiny, stream)))
    return KFAC_ERR_LAUNCH;
  if (plan.order.empty()) return launch_status();
  std::vector<OrthMat> table(plan.order.size());
  std::vector<int> sum_blocks, pack_blocks;
  const size_t size = type_size(c.type);
  for (OrthBatch& b : plan.batches) {
    int sum0 = 0, pack0 = 0, gi = 0, index = 0;
    for (int at = b.first; at < b.first + b.count; ++at) {
      if (index == b.groups[gi].count) {
        ++gi;
        index = 0;
      }
      const OrthGroup& g = b.groups[gi];
      const int i = plan.order[at];
      OrthMat& m = table[at];
      m.in = c.in[i];
      m.out = c.out[i];
      m.buf = c.buf ? c.buf[i] : nullptr;
      m.rows = c.rows[i];
      m.cols = c.cols[i];
      m.numel = (long)m.rows * m.cols;
      m.group = gi;
      m.index = index++;
      m.sum0 = sum0;
      m.sums = (int)std::min((m.numel + SUM_ELEMS - 1) / SUM_ELEMS, (long)SUM_MAX);
      m.pack0 = pack0;
      m.step = c.step ? c.step[i] : 0.f;
      m.keep = c.keep ? c.keep[i] : 0.f;
      m.aligned = (uintptr_t)m.in % (8 * size) == 0 && ((uintptr_t)m.buf & 15) == 0;
      m.vec = m.aligned && m.cols % 8 == 0;
      m.wide = m.cols % 4 == 0 && (uintptr_t)m.out % (4 * size) == 0;
      sum0 += m.sums;
      pack0 += cdiv(g.R, PACK_R) * cdiv(g.C, PACK_C);
    }
    sum_blocks.push_back(sum0);
    pack_blocks.push_back(pack0);
  }
  char* const ws = (char*)workspace;
  upload_table(table.data(), table.size() * sizeof(OrthMat), ws + l.table, stream);
  double* const sums = (double*)(ws + l.sums);
  int* const lifts = (int*)(ws + l.lifts);
  half_t* const base = (half_t*)(ws + l.operands);
  for (size_t bi = 0; bi < plan.batches.size(); ++bi) {
    OrthBatch& b = plan.batches[bi];
    const OrthMat* const mats = (const OrthMat*)(ws + l.table) + b.first;
    for (OrthGroup& g : b.groups) g.first -= b.first;
    const bool low = c.steps > c.late;
    const auto passes = [&](auto* v) {
      using V = std::remove_pointer_t<decltype(v)>;
      if (c.buf) launch_passes<V, true>(mats, b, c.mom, sums, sum_blocks[bi], pack_blocks[bi], c.eps, base, lifts, low, stream);
      else launch_passes<V, false>(mats, b, c.mom, sums, sum_blocks[bi], pack_blocks[bi], c.eps, base, lifts, low, stream);
    };
    if (c.type == TYPE_F32) passes((float*)nullptr);
    else if (c.type == TYPE_BF16) passes((__hip_bfloat16*)nullptr);
    else passes((half_t*)nullptr);
    OrthProduct p;
    memset(&p, 0, sizeof(p));
    const OrthLaunch launches[3] = {orth_launch(b, ORTH_GRAM), orth_launch(b, ORTH_POLY), orth_launch(b, ORTH_APPLY)};
    p.base = base;
    p.partial = (float*)(ws + l.partials);
    p.mats = mats;
    p.lifts = lifts;
    p.type = c.type;
    p.update = c.step != nullptr;
    for (int k = 0; k < c.steps; ++k) {
      const bool split = c.steps - k > c.late, next = c.steps - k - 1 > c.late, last = k + 1 == c.steps;
      p.from = k & 1;
      p.growth = c.growth[k];
      if (!launch_step(p, b, launches, c.coeffs + 3 * k, split, next, last, stream)) return KFAC_ERR_LAUNCH;
      p.fallen += p.growth;
    }
  }
  return launch_status();
}

}  // namespace
}  // namespace kfac

extern "C" {

size_t kfac_orthogonalize_workspace_bytes(int count, const int* rows, const int* cols) {
  try {
    if (!kfac::sizes_ok(count, rows, cols) || count == 0) return 0;
    return kfac::layout(kfac::orth_plan(count, rows, cols, true)).bytes;
  } catch (const std::exception&) {
    return 0;
  }
}

int kfac_orthogonalize_batched(int count, const int* rows, const int* cols, int type, const void* const* in,
                               void* const* out, int steps, const float* coefficients, float eps, int late_steps,
                               void* workspace, size_t workspace_bytes, void* stream) {
  try {
    kfac::Call c{count, rows, cols, type, in, out, nullptr, nullptr, nullptr, {0.f, 0},
                 steps, coefficients, eps, late_steps, {}};
    return kfac::run(c, workspace, workspace_bytes, (hipStream_t)stream);
  } catch (const std::exception&) {
    return KFAC_ERR_TOO_LARGE;
  }
}

int kfac_muon_update_batched(int count, const int* rows, const int* cols, int type, void* const* params,
                             const void* const* grads, float* const* buffers, const float* step, const float* keep,
                             float momentum, int nesterov, int steps, const float* coefficients, float eps,
                             int late_steps, void* workspace, size_t workspace_bytes, void* stream) {
  try {
    if (count > 0 && (!buffers || !step || !keep)) return KFAC_ERR_ARG;
    kfac::Call c{count, rows, cols, type, grads, params, buffers, step, keep, {momentum, nesterov},
                 steps, coefficients, eps, late_steps, {}};
    return kfac::run(c, workspace, workspace_bytes, (hipStream_t)stream);
  } catch (const std::exception&) {
    return KFAC_ERR_TOO_LARGE;
  }
}

}  // extern "C"
