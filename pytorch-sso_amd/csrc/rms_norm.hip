// Root-mean-square norm with the residual's addition in front of it, its backward pass, and the
// diagonal curvature of its gain.
//
//   h = x + residual (rounded to its type)       r = 1 / sqrt(mean(h^2) + eps)
//   y = h r w                                    (8 bits: y / scale, scale = max |y| / 448 of the row)
//   dx = dh + r (w dy - h r^2 mean(w dy h))
//   s_n = sum over the rows of sample n of dy h r      dw = sum_n s_n      curvature = N sum_n s_n^2
//
// All of it is bound by memory.  A row stays in the registers of the threads that read it, a wave
// or a workgroup, so every stream passes once; the backward pass forms its two sums over a row
// (h^2 and w dy h) together, so that nothing but h is kept for it.  The sums over rows stay in
// registers over the rows of a unit (a wave or a workgroup), whose partial sums a second launch
// adds up in order.
#include <exception>

#include "common.h"
#include "element_types.h"
#include "norm_rows.h"

namespace kfac {
namespace {

constexpr float LARGEST_8 = 448.f;        // of the 8-bit type (4 exponent bits, 3 of the significand)

struct NormArgs {
  const void *x, *residual, *w;
  void *y, *h;
  float* scale;                           // 8 bits out
  long rows, ldx, ldr;
  int dim, w_f32;
  float eps;
};

template <class V, int N>
__device__ __forceinline__ void load(const V* p, float (&v)[N]) {
  if constexpr (N * sizeof(V) > 16) {
    const Pack<V, N / 2> a = *(const Pack<V, N / 2>*)p, b = *(const Pack<V, N / 2>*)(p + N / 2);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      v[e] = Element<V>::get(a.v[e]);
      v[e + N / 2] = Element<V>::get(b.v[e]);
    }
  } else {
    const Pack<V, N> a = *(const Pack<V, N>*)p;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = Element<V>::get(a.v[e]);
  }
}
template <class V, int N>
__device__ __forceinline__ void store(V* p, const float (&v)[N]) {
  Pack<V, N> a;
#pragma unroll
  for (int e = 0; e < N; ++e) a.v[e] = Element<V>::put(v[e]);
  *(Pack<V, N>*)p = a;
}

// 16 bytes of a stream.  ONCE: of more bytes in all than the last cache holds, which are not to displace one
// another there: 16384 rows of 4096 in bfloat16 forward and backward 219 us without that, 206 with it, 8193
// rows of 5120 to 8 bits 64 and 56.  Where the caches hold them for the kernels in front and behind it costs
// (4096 rows of 4096 between two other operations on them: forward 48 us without and 51 with it, backward 55
// and 66).
typedef unsigned u4 __attribute__((ext_vector_type(4)));
constexpr long LAST_CACHE = 256L << 20;
template <bool ONCE, class V, int N>
__device__ __forceinline__ Pack<V, N> stream_load(const V* p) {
  if constexpr (ONCE) return __builtin_bit_cast(Pack<V, N>, __builtin_nontemporal_load((const u4*)p));
  else return *(const Pack<V, N>*)p;
}
template <bool ONCE, class V, int N>
__device__ __forceinline__ void stream_load(const V* p, float (&v)[N]) {
  const Pack<V, N> a = stream_load<ONCE, V, N>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = Element<V>::get(a.v[e]);
}
template <bool ONCE, class V, int N>
__device__ __forceinline__ void stream_store(V* p, const float (&v)[N]) {
  Pack<V, N> a;
#pragma unroll
  for (int e = 0; e < N; ++e) a.v[e] = Element<V>::put(v[e]);
  if constexpr (ONCE) __builtin_nontemporal_store(__builtin_bit_cast(u4, a), (u4*)p);
  else *(Pack<V, N>*)p = a;
}
template <class V, int N>
__device__ __forceinline__ void load_gain(const void* w, int w_f32, int c, float (&v)[N]) {
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = 1.f;
  } else if (w_f32) {
    load<float, N>((const float*)w + c, v);
  } else {
    load<V, N>((const V*)w + c, v);
  }
}

// N values divided by `scale` in 8 bits
template <int N>
__device__ __forceinline__ void store8(unsigned char* p, const float (&v)[N], float scale) {
  if constexpr (N == 1) {
    *p = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(v[0] / scale, 0.f, 0, false);
  } else {
    unsigned q[N / 4];
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[e] / scale, v[e + 1] / scale, 0, false);
      q[e / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(v[e + 2] / scale, v[e + 3] / scale, low, true);
    }
    if constexpr (N == 8) *(uint2*)p = make_uint2(q[0], q[1]);
    else *(unsigned*)p = q[0];
  }
}

struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Max {
  static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

// Over the threads of a unit, the same in each: a wave, or a workgroup of T threads (`tmp`: room for
// 2 K T / 64 floats, `turn` alternates so that one barrier is enough).
template <class OP, int T, int K>
__device__ __forceinline__ void unit_reduce(float (&v)[K], float* tmp, int& turn) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = OP::of(v[k], __shfl_xor(v[k], o));
  if constexpr (T > 64) {
    constexpr int W = T / 64;
    float* const at = tmp + turn * K * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) at[k * W + (threadIdx.x >> 6)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = at[k * W];
#pragma unroll
      for (int i = 1; i < W; ++i) v[k] = OP::of(v[k], at[k * W + i]);
    }
  }
}

constexpr int block_threads(int T) { return T < 256 ? 256 : T; }

// T threads a row, N accesses of E elements each.  8193 rows of 5120 in bfloat16 with their residual, 8 bits
// out: 56 us, 5.2 TB/s, a copy's rate; 16384 rows of 4096 with their residual 91 us, 5.9 TB/s.
template <class V, int E, int T, int N, bool ONCE>
__global__ __launch_bounds__(block_threads(T)) void norm_kernel(const NormArgs a) {
  __shared__ float tmp[T > 64 ? 2 * T / 64 : 1];
  const int t = threadIdx.x % T;
  const long row = (long)blockIdx.x * (block_threads(T) / T) + threadIdx.x / T;
  if (row >= a.rows) return;               // (a whole unit)
  const V* const x = (const V*)a.x + row * a.ldx;
  const V* const res = a.residual ? (const V*)a.residual + row * a.ldr : nullptr;
  V* const hout = a.h ? (V*)a.h + row * a.dim : nullptr;
  float h[N][E];
  float s[1] = {0.f};
  int turn = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * T + t) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) h[n][e] = 0.f;
    if (c >= a.dim) continue;
    stream_load<ONCE, V, E>(x + c, h[n]);
    if (res) {
      float b[E];
      stream_load<ONCE, V, E>(res + c, b);
#pragma unroll
      for (int e = 0; e < E; ++e) h[n][e] = Element<V>::get(Element<V>::put(h[n][e] + b[e]));
    }
  }
  if (hout) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * T + t) * E;
      if (c < a.dim) stream_store<ONCE, V, E>(hout + c, h[n]);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] = fmaf(h[n][e], h[n][e], s[0]);
  unit_reduce<Sum, T, 1>(s, tmp, turn);
  const float r = rsqrtf(s[0] / (float)a.dim + a.eps);
  float top[1] = {0.f};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * T + t) * E;
    if (c >= a.dim) continue;
    float w[E];
    load_gain<V, E>(a.w, a.w_f32, c, w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[n][e] = h[n][e] * r * w[e];
      top[0] = fmaxf(top[0], fabsf(h[n][e]));
    }
    if (!a.scale) stream_store<ONCE, V, E>((V*)a.y + row * a.dim + c, h[n]);
  }
  if (!a.scale) return;
  unit_reduce<Max, T, 1>(top, tmp, turn);
  const float scale = top[0] > 0.f ? top[0] / LARGEST_8 : 1.f;
  if (t == 0) a.scale[row] = scale;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * T + t) * E;
    if (c < a.dim) store8<E>((unsigned char*)a.y + row * a.dim + c, h[n], scale);
  }
}

// Rows that do not fit registers: three passes over the row, from cache as a rule.
template <class V>
__global__ __launch_bounds__(1024) void norm_long_kernel(const NormArgs a) {
  __shared__ float tmp[2 * 16];
  const long row = blockIdx.x;
  const V* const x = (const V*)a.x + row * a.ldx;
  const V* const res = a.residual ? (const V*)a.residual + row * a.ldr : nullptr;
  const auto value = [&](int c) {
    float v[1];
    load<V, 1>(x + c, v);
    if (res) v[0] = Element<V>::get(Element<V>::put(v[0] + Element<V>::get(res[c])));
    return v[0];
  };
  float s[1] = {0.f};
  int turn = 0;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float v = value(c);
    if (a.h) ((V*)a.h)[row * a.dim + c] = Element<V>::put(v);
    s[0] = fmaf(v, v, s[0]);
  }
  unit_reduce<Sum, 1024, 1>(s, tmp, turn);
  const float r = rsqrtf(s[0] / (float)a.dim + a.eps);
  const auto result = [&](int c) {
    float w[1];
    load_gain<V, 1>(a.w, a.w_f32, c, w);
    return value(c) * r * w[0];
  };
  float top[1] = {0.f};
  if (a.scale) {
    for (int c = threadIdx.x; c < a.dim; c += 1024) top[0] = fmaxf(top[0], fabsf(result(c)));
    unit_reduce<Max, 1024, 1>(top, tmp, turn);
  }
  const float scale = top[0] > 0.f ? top[0] / LARGEST_8 : 1.f;
  if (a.scale && threadIdx.x == 0) a.scale[row] = scale;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float v[1] = {result(c)};
    if (a.scale) store8<1>((unsigned char*)a.y + row * a.dim + c, v, scale);
    else store<V, 1>((V*)a.y + row * a.dim + c, v);
  }
}

// ---------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------

// How the rows are dealt to units.  parts > 0: a unit takes one of `parts` pieces (of `rows` rows)
// of a sample, and leaves its part of s_n; parts == 0: it takes `rows` / tokens whole samples, or
// just rows where no curvature is wanted, and leaves its part of dw and of sum s_n^2.
struct Deal {
  int units, parts, samples;
  long tokens, rows;
  int whole;                              // squares are formed in the units
};

struct BackArgs {
  const void *dy, *dh, *h, *w;
  void* dx;
  float* partial;                         // [units][dim] s or dw, then (whole) [units][dim] sum s^2
  long rows, lddy, lddh, ldh;
  int dim, w_f32;
  float eps;
  Deal deal;
};

__device__ __forceinline__ void unit_rows(const Deal& d, long all, int unit, long& first, long& last) {
  if (d.parts > 0) {
    const long n = unit / d.parts, part = unit % d.parts;
    first = n * d.tokens + part * d.rows;
    last = n * d.tokens + min(d.tokens, (part + 1) * d.rows);
  } else {
    first = unit * d.rows;
    last = min(all, first + d.rows);
  }
}

template <class V, int E, int T, int N, bool WHOLE, bool ONCE>
__global__ __launch_bounds__(block_threads(T)) void norm_backward_kernel(const BackArgs a) {
  __shared__ float tmp[T > 64 ? 4 * T / 64 : 1];
  const int t = threadIdx.x % T;
  const int unit = blockIdx.x * (block_threads(T) / T) + threadIdx.x / T;
  if (unit >= a.deal.units) return;
  long row, last;
  unit_rows(a.deal, a.rows, unit, row, last);
  float s[N][E], sum[WHOLE ? N : 1][E], sq[WHOLE ? N : 1][E];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < E; ++e) s[n][e] = 0.f;
  if (WHOLE)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < E; ++e) sum[n][e] = sq[n][e] = 0.f;
  int turn = 0;
  const float inv_dim = 1.f / (float)a.dim;
  long token = 0;
  for (; row < last; ++row) {
    const V* const dy = (const V*)a.dy + row * a.lddy;
    const V* const h = (const V*)a.h + row * a.ldh;
    float g[N][E], v[N][E];
    Pack<V, E> dh[N];
    float two[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * T + t) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) g[n][e] = v[n][e] = 0.f;
      if (c >= a.dim) continue;
      stream_load<ONCE, V, E>(dy + c, g[n]);
      stream_load<ONCE, V, E>(h + c, v[n]);
      if (a.dh) dh[n] = stream_load<ONCE, V, E>((const V*)a.dh + row * a.lddh + c);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * T + t) * E;
      float w[E];
      if (c < a.dim) load_gain<V, E>(a.w, a.w_f32, c, w);
      else
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        two[0] = fmaf(v[n][e], v[n][e], two[0]);
        two[1] = fmaf(w[e] * g[n][e], v[n][e], two[1]);
      }
    }
    unit_reduce<Sum, T, 2>(two, tmp, turn);
    const float r = rsqrtf(two[0] * inv_dim + a.eps), k = r * r * two[1] * inv_dim;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * T + t) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) s[n][e] = fmaf(g[n][e] * r, v[n][e], s[n][e]);
      if (a.dx && c < a.dim) {
        float w[E], d[E];
        load_gain<V, E>(a.w, a.w_f32, c, w);
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = r * (w[e] * g[n][e] - v[n][e] * k);
        if (a.dh)
#pragma unroll
          for (int e = 0; e < E; ++e) d[e] += Element<V>::get(dh[n].v[e]);
        stream_store<ONCE, V, E>((V*)a.dx + row * a.dim + c, d);
      }
    }
    if (WHOLE && ++token == a.deal.tokens) {
      token = 0;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          sum[n][e] += s[n][e];
          sq[n][e] = fmaf(s[n][e], s[n][e], sq[n][e]);
          s[n][e] = 0.f;
        }
    }
  }
  if (!a.partial) return;
  float* const to = a.partial + (long)unit * a.dim;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * T + t) * E;
    if (c >= a.dim) continue;
    if (WHOLE) {
      store<float, E>(to + c, sum[n]);
      store<float, E>(to + (long)a.deal.units * a.dim + c, sq[n]);
    } else {
      store<float, E>(to + c, s[n]);
    }
  }
}

// Rows that do not fit registers: the sums of a unit stay in its partial sums in memory (every
// column is the same thread's throughout).  With squares, a third row of them holds s_n.
template <class V>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(const BackArgs a, float* current) {
  __shared__ float tmp[4 * 16];
  long row, last;
  unit_rows(a.deal, a.rows, blockIdx.x, row, last);
  float* const to = a.partial ? a.partial + (long)blockIdx.x * a.dim : nullptr;
  float* const sq = to + (long)a.deal.units * a.dim;
  float* const cur = a.deal.whole ? current + (long)blockIdx.x * a.dim : to;
  if (to)
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      to[c] = 0.f;
      if (a.deal.whole) sq[c] = cur[c] = 0.f;
    }
  int turn = 0;
  long token = 0;
  for (; row < last; ++row) {
    const V* const dy = (const V*)a.dy + row * a.lddy;
    const V* const h = (const V*)a.h + row * a.ldh;
    float two[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      float w[1];
      load_gain<V, 1>(a.w, a.w_f32, c, w);
      const float v = Element<V>::get(h[c]), g = Element<V>::get(dy[c]);
      two[0] = fmaf(v, v, two[0]);
      two[1] = fmaf(w[0] * g, v, two[1]);
    }
    unit_reduce<Sum, 1024, 2>(two, tmp, turn);
    const float r = rsqrtf(two[0] / (float)a.dim + a.eps), k = r * r * two[1] / (float)a.dim;
    const bool ends = a.deal.whole && ++token == a.deal.tokens;
    if (ends) token = 0;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      const float v = Element<V>::get(h[c]), g = Element<V>::get(dy[c]);
      if (to) {
        float s = fmaf(g * r, v, cur[c]);
        if (ends) {
          to[c] += s;
          sq[c] = fmaf(s, s, sq[c]);
          s = 0.f;
        }
        cur[c] = s;
      }
      if (a.dx) {
        float w[1];
        load_gain<V, 1>(a.w, a.w_f32, c, w);
        float d = r * (w[0] * g - v * k);
        if (a.dh) d += Element<V>::get(((const V*)a.dh)[row * a.lddh + c]);
        ((V*)a.dx)[row * a.dim + c] = Element<V>::put(d);
      }
    }
  }
}

// The partial sums of the units, added up in 64 bits (rounded once on the way, a group's sum) and in an order
// that depends on their number alone.  A workgroup
// takes 32 columns, E of them to a thread, in G groups of threads over the units (1024 units of 4096 columns,
// a sample each 6.4 us, of 8 samples 7.0; in 24 with 16 groups of a column to a thread).
constexpr int REDUCE_COLUMNS = 32, REDUCE_THREADS = 1024;
template <int E>
__global__ __launch_bounds__(REDUCE_THREADS) void norm_reduce_kernel(const float* partial, Deal d, int dim, void* dw,
                                                                     int w_type, float* curvature) {
  constexpr int LANES = REDUCE_COLUMNS / E, G = REDUCE_THREADS / LANES, TEAMS = REDUCE_THREADS / REDUCE_COLUMNS;
  __shared__ float part[2][G][REDUCE_COLUMNS + 1];
  __shared__ double sums[2][TEAMS][REDUCE_COLUMNS];
  const int group = threadIdx.x / LANES, column = threadIdx.x % LANES * E, c = blockIdx.x * REDUCE_COLUMNS + column;
  double sum[E], sq[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = sq[e] = 0.;
  const bool squares = curvature != nullptr;
  // to = sum over `count` units from `first` on, `step` apart, several in flight; squared: sq, of their squares
  const auto add = [&](long first, long step, int count, double (&to)[E], bool squared = false) {
    if (c >= dim) return;
    const float* at = partial + first * dim + c;
    constexpr int K = 8;
    for (int i = 0; i < count; i += K) {
      float v[K][E];
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[k][e] = 0.f;
        if (i + k < count) load<float, E>(at + (long)(i + k) * step * dim, v[k]);
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) to[e] += (double)v[k][e];
      if (squared)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) sq[e] = fma((double)v[k][e], (double)v[k][e], sq[e]);
    }
  };
  // few samples in many parts: several groups a sample
  const int share = d.parts > 1 && d.samples < G ? G / d.samples : 1;
  if (d.parts == 1) {
    add(group, G, group < d.samples ? (d.samples - group + G - 1) / G : 0, sum, true);
  } else if (d.parts > 1) {
    for (int n = group / share; n < d.samples; n += G / share) {
      double s[E];
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] = 0.;
      const int p = group % share;
      add((long)n * d.parts + p, share, p < d.parts ? (d.parts - p + share - 1) / share : 0, s);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sum[e] += s[e];
        if (share == 1) sq[e] = fma(s[e], s[e], sq[e]);
      }
    }
  } else {
    const int count = group < d.units ? (d.units - group + G - 1) / G : 0;
    add(group, G, count, sum);
    if (squares) add((long)group + d.units, G, count, sq);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    part[0][group][column + e] = (float)sum[e];
    part[1][group][column + e] = (float)sq[e];
  }
  __syncthreads();
  // the groups' sums, or with several groups a sample the samples': dealt to 32 threads a column, then added up
  const int mine = threadIdx.x % REDUCE_COLUMNS, team = threadIdx.x / REDUCE_COLUMNS;
  double total = 0., square = 0.;
  if (share > 1) {
    for (int n = team; n < d.samples; n += TEAMS) {
      double s = 0.;
      for (int i = 0; i < share; ++i) s += (double)part[0][n * share + i][mine];
      total += s;
      square = fma(s, s, square);
    }
  } else {
    for (int i = team; i < G; i += TEAMS) {
      total += (double)part[0][i][mine];
      square += (double)part[1][i][mine];
    }
  }
  sums[0][team][mine] = total;
  sums[1][team][mine] = square;
  __syncthreads();
  const int to = blockIdx.x * REDUCE_COLUMNS + mine;
  if (team > 1 || to >= dim) return;
  double t[4] = {0., 0., 0., 0.};          // (an addition in 64 bits waits for the one before it)
#pragma unroll
  for (int i = 0; i < TEAMS; ++i) t[i & 3] += sums[team][i][mine];
  const double all = (t[0] + t[1]) + (t[2] + t[3]);
  if (team == 1) {
    if (squares) curvature[to] = (float)((double)d.samples * all);
  } else if (dw) {
    if (w_type == TYPE_F32) ((float*)dw)[to] = (float)all;
    else if (w_type == TYPE_BF16) ((__hip_bfloat16*)dw)[to] = Element<__hip_bfloat16>::put((float)all);
    else ((_Float16*)dw)[to] = Element<_Float16>::put((float)all);
  }
}

// Threads a row and accesses of `e` elements a thread; 0: longer than the registers of 1024 threads.
struct Shape {
  int threads, accesses;
};
// forward: a wave up to four accesses (16 of single elements), then 256 threads, then 1024
Shape norm_shape(int dim, int e) {
  const int n = (dim + e - 1) / e, most = e == 1 ? 16 : 4;
  for (int t : {64, 256, 1024})
    for (int k : {most / 4, most / 2, most})
      if (n <= t * k) return Shape{t, k};
  return Shape{0, 0};
}
// backward, which holds three rows and the sums: at most two accesses a thread (16384 rows of 4096 in
// bfloat16: two on 256 threads 112 us, 4.8 TB/s; with cached streams 132, one on 512 142; asking for the next row before the sums of
// one are formed changes nothing)
constexpr Shape BACK_SHAPES[] = {{64, 1}, {64, 2}, {256, 1}, {256, 2}, {512, 2}, {1024, 2}};
Shape backward_shape(int dim, int e) {
  const int n = (dim + e - 1) / e, scale = e == 1 ? 8 : 1;
  for (const Shape& s : BACK_SHAPES)
    if (n <= s.threads * s.accesses * scale) return Shape{s.threads, s.accesses * scale};
  return Shape{0, 0};
}

Deal deal_rows(long rows, int samples, bool squares, int threads) {
  Deal d;
  const long target = threads == 64 ? 4096 : threads == 0 || threads == 1024 ? 512 : 1024;
  d.samples = samples;
  d.tokens = rows / samples;
  const long per = std::max(1L, (rows + target - 1) / target);       // rows of a unit
  d.whole = 0;
  if (squares && d.tokens >= per) {
    d.parts = (int)((d.tokens + per - 1) / per);
    d.rows = (d.tokens + d.parts - 1) / d.parts;
    d.units = d.parts * samples;
  } else {
    d.parts = 0;
    d.whole = squares;
    d.rows = squares ? per / d.tokens * d.tokens : per;
    d.units = (int)((rows + d.rows - 1) / d.rows);
  }
  return d;
}

// `n` rows of `a` from `first` on
template <class V>
NormArgs norm_rows(NormArgs a, long first, long n) {
  const auto ahead = [](const void* p, long elements, size_t size) { return p ? (const char*)p + elements * (long)size : nullptr; };
  a.x = ahead(a.x, first * a.ldx, sizeof(V));
  a.residual = ahead(a.residual, first * a.ldr, sizeof(V));
  a.y = (void*)ahead(a.y, first * a.dim, a.scale ? 1 : sizeof(V));
  a.h = (void*)ahead(a.h, first * a.dim, sizeof(V));
  a.scale = (float*)ahead(a.scale, first, sizeof(float));
  a.rows = n;
  return a;
}

template <class V, int E, bool ONCE = false>
bool launch_norm(const NormArgs& a, hipStream_t stream) {
  const long bytes = a.rows * a.dim * (long)((a.residual ? 3 : a.h ? 2 : 1) * sizeof(V) + (a.scale ? 1 : sizeof(V)));
  if constexpr (E > 1 && !ONCE)
    if (bytes > LAST_CACHE) return launch_norm<V, E, true>(a, stream);
  const Shape s = norm_shape(a.dim, E);
#define NORM_CASE(T, N)                                                                                   \
  if (s.threads == T && s.accesses == N) {                                                                \
    for_row_ranges(a.rows, block_threads(T), block_threads(T) / T, [&](long first, long n, unsigned blocks) { \
      hipLaunchKernelGGL((norm_kernel<V, E, T, N, ONCE>), dim3(blocks), dim3(block_threads(T)), 0, stream, \
                         norm_rows<V>(a, first, n));                                                      \
    });                                                                                                   \
    return true;                                                                                          \
  }
  constexpr int M = E == 1 ? 16 : 4;
  NORM_CASE(64, M / 4) NORM_CASE(64, M / 2) NORM_CASE(64, M)
  NORM_CASE(256, M / 4) NORM_CASE(256, M / 2) NORM_CASE(256, M)
  NORM_CASE(1024, M / 4) NORM_CASE(1024, M / 2) NORM_CASE(1024, M)
#undef NORM_CASE
  for_row_ranges(a.rows, 1024, 1, [&](long first, long n, unsigned blocks) {
    hipLaunchKernelGGL((norm_long_kernel<V>), dim3(blocks), dim3(1024), 0, stream, norm_rows<V>(a, first, n));
  });
  return true;
}

template <class V, int E, bool ONCE = false>
bool launch_backward(const BackArgs& a, float* current, hipStream_t stream) {
  const long bytes = a.rows * a.dim * (long)((2 + (a.dh != nullptr) + (a.dx != nullptr)) * sizeof(V));
  if constexpr (E > 1 && !ONCE)
    if (bytes > LAST_CACHE) return launch_backward<V, E, true>(a, current, stream);
  const Shape s = backward_shape(a.dim, E);
#define BACK_CASE(T, N)                                                                                   \
  if (s.threads == T && s.accesses == N) {                                                                \
    const int per = block_threads(T) / T;                                                                 \
    const dim3 grid(cdiv(a.deal.units, per)), block(block_threads(T));                                    \
    if (a.deal.whole)                                                                                     \
      hipLaunchKernelGGL((norm_backward_kernel<V, E, T, N, true, ONCE>), grid, block, 0, stream, a);      \
    else                                                                                                  \
      hipLaunchKernelGGL((norm_backward_kernel<V, E, T, N, false, ONCE>), grid, block, 0, stream, a);     \
    return true;                                                                                          \
  }
  constexpr int M = E == 1 ? 8 : 1;
  BACK_CASE(64, M) BACK_CASE(64, 2 * M) BACK_CASE(256, M) BACK_CASE(256, 2 * M) BACK_CASE(512, 2 * M) BACK_CASE(1024, 2 * M)
#undef BACK_CASE
  hipLaunchKernelGGL((norm_backward_long_kernel<V>), dim3(a.deal.units), dim3(1024), 0, stream, a, current);
  return true;
}

// All rows can be accessed 16 bytes at a time.
bool aligned(int dim, int e, std::initializer_list<std::pair<const void*, long>> rows, const void* w, int w_f32) {
  if (dim % e != 0) return false;
  for (const auto& r : rows)
    if (r.first && (((uintptr_t)r.first & 15) || r.second % e != 0)) return false;
  return ((uintptr_t)w & 15) == 0;
}

constexpr int NORM_MAX_DIM = 1 << 24;
bool norm_args_ok(int type, int w_f32, int64_t rows, int dim, float eps) {
  return type >= TYPE_F32 && type <= TYPE_F16 && (w_f32 == 0 || w_f32 == 1) && rows >= 0 && rows < (1LL << 31) &&
         dim > 0 && dim <= NORM_MAX_DIM && eps >= 0.f;
}

int run_norm(int type, const NormArgs& a, hipStream_t stream) {
  const int e = type == TYPE_F32 ? 4 : 8;
  const bool vec = aligned(a.dim, e, {{a.x, a.ldx}, {a.residual, a.ldr}, {a.y, a.dim}, {a.h, a.dim}}, a.w, a.w_f32);
  if (type == TYPE_F32) vec ? launch_norm<float, 4>(a, stream) : launch_norm<float, 1>(a, stream);
  else if (type == TYPE_BF16)
    vec ? launch_norm<__hip_bfloat16, 8>(a, stream) : launch_norm<__hip_bfloat16, 1>(a, stream);
  else vec ? launch_norm<_Float16, 8>(a, stream) : launch_norm<_Float16, 1>(a, stream);
  return launch_status();
}

// the deal must not depend on alignment (the caller asks for scratch by sizes alone)
int deal_threads(int type, int dim) { return backward_shape(dim, type == TYPE_F32 ? 4 : 8).threads; }

size_t backward_floats(const Deal& d, int dim) { return (size_t)d.units * dim * (d.whole ? 3 : 1); }

}  // namespace
}  // namespace kfac

using namespace kfac;

extern "C" {

int kfac_rms_norm(int type, int gain_is_float, int64_t rows, int dim, const void* x, int64_t ldx,
                  const void* residual, int64_t ldr, const void* gain, float eps, void* y, void* h, float* scale,
                  void* stream) {
  if (!norm_args_ok(type, gain_is_float, rows, dim, eps)) return KFAC_ERR_ARG;
  if (rows == 0) return KFAC_OK;
  if (!x || !y || (residual && !h) || ldx < 0 || ldr < 0) return KFAC_ERR_ARG;
  NormArgs a{x, residual, gain, y, h, scale, (long)rows, (long)ldx, (long)ldr, dim, gain_is_float, eps};
  return run_norm(type, a, (hipStream_t)stream);
}

size_t kfac_rms_norm_backward_workspace_bytes(int type, int64_t rows, int dim, int samples, int squares) {
  if (!norm_args_ok(type, 0, rows, dim, 0.f) || samples <= 0 || rows == 0 || rows % samples != 0) return 0;
  return sizeof(float) * backward_floats(deal_rows((long)rows, samples, squares != 0, deal_threads(type, dim)), dim);
}

int kfac_rms_norm_backward(int type, int gain_is_float, int64_t rows, int dim, int samples, const void* dy,
                           int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh, const void* gain,
                           float eps, void* dx, void* dgain, float* curvature, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (!norm_args_ok(type, gain_is_float, rows, dim, eps) || samples <= 0 || rows % samples != 0) return KFAC_ERR_ARG;
  if (rows == 0 || !dy || !h || lddy < 0 || lddh < 0 || ldh < 0 || (dh && !dx)) return KFAC_ERR_ARG;
  const bool sums = dgain || curvature;
  BackArgs a{dy, dh, h, gain, dx, nullptr, (long)rows, (long)lddy, (long)lddh, (long)ldh, dim, gain_is_float, eps, {}};
  a.deal = deal_rows((long)rows, samples, curvature != nullptr, deal_threads(type, dim));
  float* current = nullptr;
  if (sums) {
    if (!workspace || workspace_bytes < sizeof(float) * backward_floats(a.deal, dim)) return KFAC_ERR_WORKSPACE;
    a.partial = (float*)workspace;
    current = a.partial + 2 * (size_t)a.deal.units * dim;
  }
  const int e = type == TYPE_F32 ? 4 : 8;
  const bool vec = aligned(dim, e, {{dy, a.lddy}, {dh, a.lddh}, {h, a.ldh}, {dx, dim}, {a.partial, dim}}, gain,
                           gain_is_float);
  const hipStream_t s = (hipStream_t)stream;
  if (type == TYPE_F32) vec ? launch_backward<float, 4>(a, current, s) : launch_backward<float, 1>(a, current, s);
  else if (type == TYPE_BF16)
    vec ? launch_backward<__hip_bfloat16, 8>(a, current, s) : launch_backward<__hip_bfloat16, 1>(a, current, s);
  else vec ? launch_backward<_Float16, 8>(a, current, s) : launch_backward<_Float16, 1>(a, current, s);
  if (sums)
    hipLaunchKernelGGL((dim % 4 == 0 && ((uintptr_t)a.partial & 15) == 0 ? norm_reduce_kernel<4> : norm_reduce_kernel<1>),
                       dim3(cdiv(dim, REDUCE_COLUMNS)), dim3(REDUCE_THREADS), 0, s, a.partial, a.deal, dim, dgain,
                       gain_is_float ? TYPE_F32 : type, curvature);
  return launch_status();
}

}  // extern "C"
