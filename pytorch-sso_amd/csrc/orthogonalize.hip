// Newton-Schulz orthogonalisation of lists of matrices, and Muon's update with it.
//
//   X = G / (|G| + eps);   every step:  A = X X^T,  B = a I + b A + c A A,  X = B X
//
// G: the matrix itself, or the direction that momentum makes of a gradient.  A pass over the inputs
// renews the momentum and sums the squares, a second one normalises and writes the operands; then
// three launches a step, each over the tiles of all matrices.  The last one writes the result in
// its own type, or decays and updates the parameters.
#include "element_types.h"
#include "orth_core.h"
#include "orth_plan.h"

#include <string.h>

#include <exception>

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
  int vec;               // in, out and buf are 16-byte aligned, and so are all rows
};

constexpr int SUM_ELEMS = 16384;                 // a workgroup of the first pass
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

// First pass: momentum, and the sum of squares in 64 bits (the squares of float32 numbers neither
// overflow nor vanish there).
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
  if (m.vec) {
    for (long i = ((long)local * 256 + threadIdx.x) * N; i < m.numel; i += (long)m.sums * 256 * N) {
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
  } else {
    for (long i = (long)local * 256 + threadIdx.x; i < m.numel; i += (long)m.sums * 256) {
      float u = Element<V>::get(in[i]);
      if (MUON) {
        const float b = fmaf(mom.mu, m.buf[i], u);
        m.buf[i] = b;
        u = mom.nesterov ? fmaf(mom.mu, b, u) : b;
      }
      s = fma((double)u, (double)u, s);
    }
  }
  s = block_sum(s, tmp);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

struct OrthGroups {
  OrthGroup g[ORTH_GROUPS];
  int n;
};

// Second pass: X, normalised, scaled and in halves, zeros in the padding.
template <class V, bool MUON>
__global__ __launch_bounds__(256) void orth_pack_kernel(const OrthMat* mats, int n, Momentum mom, const double* sums,
                                                        float eps, half_t* base, OrthGroups groups, int low) {
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
  const float scale = (float)((double)ORTH_SCALE / (sqrt(s) + (double)eps));
  const int across = (g.C + PACK_C - 1) / PACK_C, local = blockIdx.x - m.pack0;
  const int r0 = local / across * PACK_R, c0 = local % across * PACK_C;
  const int R = g.R, C = g.C;
  const V* const in = (const V*)m.in;
  const auto value = [&](long i) {
    float u = Element<V>::get(in[i]);
    if (MUON) u = mom.nesterov ? fmaf(mom.mu, m.buf[i], u) : m.buf[i];
    return u * scale;
  };
  const bool tall = m.rows > m.cols;
  if (tall) {
    // in: rows of g.r values, as many as g.c
    for (int i = threadIdx.x; i < PACK_R * PACK_C; i += 256) {
      const int r = i % PACK_R, c = i / PACK_R;
      tile[r][c] = r0 + r < g.r && c0 + c < g.c ? value((long)(c0 + c) * g.r + r0 + r) : 0.f;
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
        v[e] = u * scale;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c0 + c + e < g.c ? value(at + e) : 0.f;
    }
    h8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = (half_t)v[e];
      l[e] = (half_t)(v[e] - (float)h[e]);
    }
    half_t* const to = x + (long)(r0 + r) * C + c0 + c;
    *(h8*)to = h;
    if (low) *(h8*)(to + (long)R * C) = l;
  }
}

enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };

struct OrthProduct {
  half_t* base;
  const OrthMat* mats;
  float ca, cb, cc;      // of this step
  int from;              // which X is read (the other one is written)
  int low;               // the low halves of the result are wanted
  int type, update;      // LAST: type of the result; parameters are updated with it
  int n;
  OrthGroup g[ORTH_GROUPS];
};
static_assert(sizeof(OrthProduct) <= 4096, "kernel arguments");

template <class V>
__device__ __forceinline__ void orth_store(const OrthMat& m, long at, float o, int update) {
  V* const out = (V*)m.out;
  if (update) o = m.keep * Element<V>::get(out[at]) - m.step * o;
  out[at] = Element<V>::put(o);
}

typedef OrthTile<64, 64, 2, 2, 4> SmallTile;
typedef OrthTile<128, 128, 2, 2, 2> MidTile;
typedef OrthTile<128, 128, 2, 2, 4> DeepTile;
typedef OrthTile<256, 256, 2, 4, 2, true> LargeTile;

template <class TILE, bool SPLIT, int MODE>
__global__ __launch_bounds__(TILE::THREADS, 2) void orth_product_kernel(const OrthProduct p) {
  extern __shared__ __align__(16) char smem[];
  constexpr int T = TILE::TM, FM = TILE::FM, FN = TILE::FN;
  static_assert(TILE::TM == TILE::TN, "symmetric products");
  constexpr bool SYM = MODE == GRAM || MODE == POLY;
  int gi = 0;
  while (gi + 1 < p.n && p.g[gi + 1].tile0 <= (int)blockIdx.x) ++gi;
  const OrthGroup& g = p.g[gi];
  const int local = blockIdx.x - g.tile0, each = (g.tiles + 7) / 8;
  const int t = (local & 7) * each + (local >> 3);     // neighbours in the tile order share a die's cache
  if (t >= g.tiles) return;
  const int R = g.R, C = g.C, rt = R / T, ct = C / T;
  int tm, tn, k;
  if (SYM) {
    const int per = rt * (rt + 1) / 2, u = t % per;
    k = t / per;
    tm = (int)((sqrtf(8.f * u + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > u) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= u) ++tm;
    tn = u - tm * (tm + 1) / 2;
  } else {
    const int per = rt * ct, u = t % per;
    k = t / per;
    tm = u / rt;
    tn = u % rt;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / TILE::WN, wn = wave % TILE::WN;
  const long XS = (long)R * C, AS = (long)R * R;
  half_t* const x = p.base + g.x[p.from] + k * 2 * XS;
  half_t* const a = p.base + g.a + k * 2 * AS;
  half_t* const b = p.base + g.b + k * 2 * AS;
  OrthOperand<TILE::TM, TILE::WAVES, FM, !SYM> P;
  OrthOperand<TILE::TN, TILE::WAVES, FN, false> Q;
  int steps;
  if (MODE == GRAM) {
    P.init(x, SPLIT ? XS : 0, C, tm * T, wm, wave, lane);
    Q.init(x, SPLIT ? XS : 0, C, tn * T, wn, wave, lane);
    steps = C;
  } else if (MODE == POLY) {
    P.init(a, SPLIT ? AS : 0, R, tm * T, wm, wave, lane);
    Q.init(a, SPLIT ? AS : 0, R, tn * T, wn, wave, lane);
    steps = R;
  } else {
    P.init(x, SPLIT ? XS : 0, C, tm * T, wm, wave, lane);          // (columns of X)
    Q.init(b, SPLIT ? AS : 0, R, tn * T, wn, wave, lane);
    steps = R;
  }
  steps /= SPLIT ? ORTH_BK : 2 * ORTH_BK;
  lds_char* const lds = (lds_char*)smem;
  f4 acc[FM][FN];
  if constexpr (TILE::PAIR) orth_pair_product<TILE, SPLIT>(P, Q, steps, lds, wave, acc);
  else orth_product<TILE, SPLIT>(P, Q, steps, lds, wave, acc);

  constexpr float INV = 1.f / ORTH_SCALE;
  const int m0 = tm * T + wm * FM * 16 + 4 * (lane >> 4), n0 = tn * T + wn * FN * 16 + (lane & 15);
  if (MODE == LAST) {
    const OrthMat m = p.mats[g.first + k];
    const bool tall = m.rows > m.cols;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = n0 + 16 * j, col = m0 + 16 * i + e;
          if (row >= g.r || col >= g.c) continue;
          const long at = tall ? (long)col * g.r + row : (long)row * g.c + col;
          const float o = acc[i][j][e] * (INV * INV);
          if (p.type == TYPE_F32) orth_store<float>(m, at, o, p.update);
          else if (p.type == TYPE_BF16) orth_store<__hip_bfloat16>(m, at, o, p.update);
          else orth_store<half_t>(m, at, o, p.update);
        }
    return;
  }
  // D[m][n] to row n: four values of a lane side by side
  const long S = SYM ? AS : XS;
  const int ld = SYM ? R : C;
  half_t* const out = MODE == GRAM ? a : MODE == POLY ? b : p.base + g.x[1 - p.from] + k * 2 * XS;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int m = m0 + 16 * i, n = n0 + 16 * j;
      f4 v = acc[i][j] * INV;
      if (MODE == POLY) {
        const h4 ah = *(const h4*)(a + (long)n * R + m);
        h4 al = {0, 0, 0, 0};
        if (SPLIT) al = *(const h4*)(a + AS + (long)n * R + m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = fmaf(p.cc, v[e], p.cb * ((float)ah[e] + (float)al[e]));
          if (m + e == n) v[e] += p.ca * ORTH_SCALE;
        }
      }
      h4 h, l;
      split4(v, h, l);
      half_t* const to = out + (long)n * ld + m;
      *(h4*)to = h;
      if (p.low) *(h4*)(to + S) = l;
      if (SYM && tm != tn) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          half_t* const mirror = out + (long)(m + e) * ld + n;
          *mirror = h[e];
          if (p.low) mirror[S] = l[e];
        }
      }
    }
}

template <class TILE, bool SPLIT, int MODE>
bool launch_tiles(OrthProduct& p, OrthBatch& b, hipStream_t stream) {
  const int grid = orth_launch(b.groups, TILE::TM, MODE == GRAM || MODE == POLY);
  p.n = (int)b.groups.size();
  std::copy(b.groups.begin(), b.groups.end(), p.g);
  constexpr int lds = TILE::LDS;
  const auto kernel = orth_product_kernel<TILE, SPLIT, MODE>;
  if (!enable_large_lds((const void*)kernel, lds)) return false;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(TILE::THREADS), lds, stream, p);
  return true;
}

template <class TILE, int MODE>
bool launch_parts(OrthProduct& p, OrthBatch& b, bool split, hipStream_t stream) {
  return split ? launch_tiles<TILE, true, MODE>(p, b, stream) : launch_tiles<TILE, false, MODE>(p, b, stream);
}

template <int MODE>
bool launch_product(OrthProduct& p, OrthBatch& b, bool split, hipStream_t stream) {
  switch (orth_pick_tile(b, MODE == GRAM || MODE == POLY)) {
    case ORTH_SMALL: return launch_parts<SmallTile, MODE>(p, b, split, stream);
    case ORTH_DEEP: return launch_parts<DeepTile, MODE>(p, b, split, stream);
    case ORTH_MID: return launch_parts<MidTile, MODE>(p, b, split, stream);
    default: return launch_parts<LargeTile, MODE>(p, b, split, stream);
  }
}

bool launch_step(OrthProduct& p, OrthBatch& b, const float* coeffs, bool split, bool next_split, bool last,
                 hipStream_t stream) {
  p.ca = coeffs[0];
  p.cb = coeffs[1];
  p.cc = coeffs[2];
  p.low = split;
  if (!launch_product<GRAM>(p, b, split, stream) || !launch_product<POLY>(p, b, split, stream)) return false;
  p.low = next_split;
  return last ? launch_product<LAST>(p, b, split, stream) : launch_product<APPLY>(p, b, split, stream);
}

template <class V, bool MUON>
void launch_passes(const OrthMat* mats, const OrthBatch& b, Momentum mom, double* sums, int sum_blocks,
                   int pack_blocks, float eps, half_t* base, bool low, hipStream_t stream) {
  hipLaunchKernelGGL((orth_sum_kernel<V, MUON>), dim3(sum_blocks), dim3(256), 0, stream, mats, b.count, mom, sums);
  OrthGroups groups;
  groups.n = (int)b.groups.size();
  std::copy(b.groups.begin(), b.groups.end(), groups.g);
  hipLaunchKernelGGL((orth_pack_kernel<V, MUON>), dim3(pack_blocks), dim3(256), 0, stream, mats, b.count, mom,
                     (const double*)sums, eps, base, groups, (int)low);
}

struct Layout {
  size_t table, sums, operands, bytes;
};
Layout layout(const OrthPlan& plan) {
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Layout l;
  l.table = 0;
  l.sums = up(plan.order.size() * sizeof(OrthMat));
  long sums = 0;
  for (const OrthBatch& b : plan.batches) sums = std::max(sums, (long)b.count * SUM_MAX);
  l.operands = l.sums + up((size_t)sums * sizeof(double));
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
};

int run(const Call& c, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (!sizes_ok(c.count, c.rows, c.cols)) return KFAC_ERR_ARG;
  if (c.count == 0) return KFAC_OK;
  if (!c.in || !c.out || !c.coeffs || c.steps < 1 || c.late < 0 || c.type < TYPE_F32 || c.type > TYPE_F16)
    return KFAC_ERR_ARG;
  OrthPlan plan = orth_plan(c.count, c.rows, c.cols);
  if (plan.order.empty()) return KFAC_OK;
  for (int i : plan.order)
    if (!c.in[i] || !c.out[i] || (c.buf && !c.buf[i])) return KFAC_ERR_ARG;
  const Layout l = layout(plan);
  if (!workspace || workspace_bytes < l.bytes) return KFAC_ERR_WORKSPACE;
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
      // rows of whole 8-element groups at aligned addresses
      m.vec = m.cols % 8 == 0 && ((uintptr_t)m.in % (8 * size)) == 0 && ((uintptr_t)m.buf & 15) == 0;
      sum0 += m.sums;
      pack0 += cdiv(g.R, PACK_R) * cdiv(g.C, PACK_C);
    }
    sum_blocks.push_back(sum0);
    pack_blocks.push_back(pack0);
  }
  char* const ws = (char*)workspace;
  upload_table(table.data(), table.size() * sizeof(OrthMat), ws + l.table, stream);
  double* const sums = (double*)(ws + l.sums);
  half_t* const base = (half_t*)(ws + l.operands);
  for (size_t bi = 0; bi < plan.batches.size(); ++bi) {
    OrthBatch& b = plan.batches[bi];
    const OrthMat* const mats = (const OrthMat*)(ws + l.table) + b.first;
    for (OrthGroup& g : b.groups) g.first -= b.first;
    const bool low = c.steps > c.late;
    const auto passes = [&](auto* v) {
      using V = std::remove_pointer_t<decltype(v)>;
      if (c.buf) launch_passes<V, true>(mats, b, c.mom, sums, sum_blocks[bi], pack_blocks[bi], c.eps, base, low, stream);
      else launch_passes<V, false>(mats, b, c.mom, sums, sum_blocks[bi], pack_blocks[bi], c.eps, base, low, stream);
    };
    if (c.type == TYPE_F32) passes((float*)nullptr);
    else if (c.type == TYPE_BF16) passes((__hip_bfloat16*)nullptr);
    else passes((half_t*)nullptr);
    OrthProduct p;
    memset(&p, 0, sizeof(p));
    p.base = base;
    p.mats = mats;
    p.type = c.type;
    p.update = c.step != nullptr;
    for (int k = 0; k < c.steps; ++k) {
      const bool split = c.steps - k > c.late, next = c.steps - k - 1 > c.late, last = k + 1 == c.steps;
      p.from = k & 1;
      if (!launch_step(p, b, c.coeffs + 3 * k, split, next, last, stream)) return KFAC_ERR_LAUNCH;
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
    return kfac::layout(kfac::orth_plan(count, rows, cols)).bytes;
  } catch (const std::exception&) {
    return 0;
  }
}

int kfac_orthogonalize_batched(int count, const int* rows, const int* cols, int type, const void* const* in,
                               void* const* out, int steps, const float* coefficients, float eps, int late_steps,
                               void* workspace, size_t workspace_bytes, void* stream) {
  try {
    kfac::Call c{count, rows, cols, type, in, out, nullptr, nullptr, nullptr, {0.f, 0},
                 steps, coefficients, eps, late_steps};
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
                 steps, coefficients, eps, late_steps};
    return kfac::run(c, workspace, workspace_bytes, (hipStream_t)stream);
  } catch (const std::exception&) {
    return KFAC_ERR_TOO_LARGE;
  }
}

}  // extern "C"
