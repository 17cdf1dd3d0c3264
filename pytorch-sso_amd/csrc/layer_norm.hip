// Layer norm with the residual's addition in front of it, its backward pass, and the diagonal curvature of its
// gain and bias.
//
//   h = x + residual (rounded to its type)       r = 1 / sqrt(var(h) + eps)      xh = (h - mean(h)) r
//   y = xh w + b                                 (8 bits: y / scale, scale = max |y| / 448 of the row)
//   dx = dh + r (w dy - mean(w dy) - xh mean(w dy xh))
//   s_n = sum over the rows of sample n of (dy xh | dy)      (dw | db) = sum_n s_n      curvature = N sum_n s_n^2
//
// All of it is bound by memory.  A row stays in the registers of the threads that read it, a wave or a workgroup,
// so every stream passes once.  A row's mean is formed in two steps that cost the two sums over the row which the
// variance needs in any case: m, a float32 sum over dim, then with d = h - m (exact, or small) the sums of d and d^2,
//   e = mean(d)      var = mean(d^2) - e^2      xh = (d - e) r
// so that rows far off zero keep their digits: e takes what rounding has lost of m.  A forward pass with a backward
// pass behind it keeps (m, e, r) of each row, 12 bytes, which spares that pass its first two sums.  The sums over
// rows stay in registers over the rows of a unit (a wave or a workgroup), whose partial sums a second launch adds up
// in order; of rows that leave no registers for them a pass of its own forms them, a thread its columns.
//
// Rows of any length and alignment are accessed 16 bytes at a time; only the last elements of a ragged row are by themselves.
#include "norm_core.h"

// Products are fused with sums where that is written, and nowhere else: m fused into h - m would be another number than
// the rounded one that is kept of it, and each variant of a kernel would round in its own way.
#pragma clang fp contract(off)

namespace kfac {
namespace {

constexpr int STATS = 3;                  // numbers kept of a row: m, e, r

// Elements of an access
template <class V> constexpr int width() { return 16 / sizeof(V); }

// 16 bytes, or 8, at addresses that are multiples of an element's size only (loads and stores of that width all the same)
typedef unsigned loose4 __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef unsigned loose4_floats __attribute__((ext_vector_type(4), aligned(4), may_alias));
typedef unsigned loose1 __attribute__((aligned(1), may_alias));
typedef unsigned loose2 __attribute__((ext_vector_type(2), aligned(1), may_alias));
template <class V> struct Loose { typedef loose4 type; };
template <> struct Loose<float> { typedef loose4_floats type; };

// The columns of an access of N elements from `first` on.  RAGGED, rows of any length and alignment: the last access of a
// row ends where the row does, so that its first `skip` columns are those of the access in front of it as well.  They
// are left out of sums over the row; what is stored for them is the same twice.  `count`: N, but in rows of fewer.
template <bool RAGGED, int N>
struct Place {
  int c, skip, count;
  bool any;
  __device__ __forceinline__ Place(int first, int dim) : c(first), skip(0), count(N), any(first < dim) {
    if (RAGGED) {
      c = max(min(first, dim - N), 0);
      skip = first - c;
      count = min(dim, N);
    }
  }
  __device__ __forceinline__ bool of_row(int e) const { return !RAGGED || (e >= skip && e < count); }
};

template <bool RAGGED, bool ONCE, class V, int N>
__device__ __forceinline__ Pack<V, N> row_load(const V* p, const Place<RAGGED, N>& at) {
  p += at.c;
  if constexpr (!RAGGED) return stream_load<ONCE, V, N>(p);
  if (at.count == N) return __builtin_bit_cast(Pack<V, N>, (u4)*(const typename Loose<V>::type*)p);
  Pack<V, N> a;
#pragma unroll
  for (int e = 0; e < N; ++e) a.v[e] = e < at.count ? p[e] : Element<V>::put(0.f);
  return a;
}
template <bool RAGGED, bool ONCE, class V, int N>
__device__ __forceinline__ void row_load(const V* p, const Place<RAGGED, N>& at, float (&v)[N]) {
  const Pack<V, N> a = row_load<RAGGED, ONCE, V, N>(p, at);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = Element<V>::get(a.v[e]);
}
template <bool RAGGED, bool ONCE, class V, int N>
__device__ __forceinline__ void row_store(V* p, const Place<RAGGED, N>& at, const float (&v)[N]) {
  p += at.c;
  if constexpr (!RAGGED) {
    stream_store<ONCE, V, N>(p, v);
  } else if (at.count == N) {
    Pack<V, N> a;
#pragma unroll
    for (int e = 0; e < N; ++e) a.v[e] = Element<V>::put(v[e]);
    *(typename Loose<V>::type*)p = __builtin_bit_cast(u4, a);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < at.count) p[e] = Element<V>::put(v[e]);
  }
}
template <bool RAGGED, class V, int N>
__device__ __forceinline__ void row_gain(const void* w, int w_f32, const Place<RAGGED, N>& at, float (&v)[N]) {
  if (!RAGGED || w == nullptr) {
    load_gain<V, N>(w, w_f32, at.c, v);
  } else if (!w_f32) {
    row_load<RAGGED, false, V, N>((const V*)w, at, v);
  } else if (at.count == N) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u4 a = *(const loose4_floats*)((const float*)w + at.c + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i + e] = __uint_as_float(a[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < at.count ? ((const float*)w)[e] : 0.f;
  }
}
// ... in 8 bits, times the reciprocal of the row's scale (a division an element is a third of the pass's arithmetic: 8193
// rows of 5120 61 us, without it 57)
template <bool RAGGED, int N>
__device__ __forceinline__ void row_store8(unsigned char* p, const Place<RAGGED, N>& at, const float (&v)[N], float inverse) {
  p += at.c;
  unsigned q[N / 4];
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[e] * inverse, v[e + 1] * inverse, 0, false);
    q[e / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(v[e + 2] * inverse, v[e + 3] * inverse, low, true);
  }
  if (at.count == N) {
    if constexpr (N == 8) *(loose2*)p = loose2{q[0], q[1]};
    else *(loose1*)p = q[0];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < at.count) p[e] = (unsigned char)(q[e / 4] >> (8 * (e & 3)));
  }
}

struct LayerNormArgs {
  const void *x, *residual, *w, *b;
  void *y, *h;                            // (no y: the statistics alone)
  float *scale, *stats;                   // 8 bits out; of a row
  long rows, ldx, ldr;
  int dim, w_f32;
  float eps;
};

// r from mean(d^2) and mean(d)
__device__ __forceinline__ float row_scale(float squares, float mean, float eps) {
  return rsqrtf(fmaxf(fmaf(-mean, mean, squares), 0.f) + eps);
}

// Scale of a row whose largest |y| is `top`: not so small that its reciprocal would leave float32
__device__ __forceinline__ float eight_scale(float top) { return top > 0.f ? fmaxf(top / LARGEST_8, 0x1p-120f) : 1.f; }

// T threads a row, N accesses each.
template <class V, int T, int N, bool RAGGED, bool ONCE>
__global__ __launch_bounds__(block_threads(T)) void layer_norm_kernel(const LayerNormArgs a) {
  constexpr int E = width<V>();
  __shared__ float tmp[T > 64 ? 4 * T / 64 : 1];
  const int t = threadIdx.x % T;
  const long row = (long)blockIdx.x * (block_threads(T) / T) + threadIdx.x / T;
  if (row >= a.rows) return;               // (a whole unit)
  const V* const x = (const V*)a.x + row * a.ldx;
  const V* const res = a.residual ? (const V*)a.residual + row * a.ldr : nullptr;
  V* const hout = a.h ? (V*)a.h + row * a.dim : nullptr;
  float h[N][E];
  int turn = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + t) * E, a.dim);
#pragma unroll
    for (int e = 0; e < E; ++e) h[n][e] = 0.f;
    if (!at.any) continue;
    row_load<RAGGED, ONCE, V, E>(x, at, h[n]);
    if (res) {
      float b[E];
      row_load<RAGGED, ONCE, V, E>(res, at, b);
#pragma unroll
      for (int e = 0; e < E; ++e) h[n][e] = Element<V>::get(Element<V>::put(h[n][e] + b[e]));
    }
  }
  if (hout) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const Place<RAGGED, E> at((n * T + t) * E, a.dim);
      if (at.any) row_store<RAGGED, ONCE, V, E>(hout, at, h[n]);
    }
  }
  float s[1] = {0.f};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + t) * E, a.dim);
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += at.of_row(e) ? h[n][e] : 0.f;
  }
  unit_reduce<Sum, T, 1>(s, tmp, turn);
  const float inv_dim = 1.f / (float)a.dim, m = s[0] * inv_dim;
  float two[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + t) * E, a.dim);
    if (!at.any) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[n][e] -= m;
      const float d = at.of_row(e) ? h[n][e] : 0.f;
      two[0] += d;
      two[1] = fmaf(d, d, two[1]);
    }
  }
  // (two values at a time from here on, behind the one of the first sum: the other half of `tmp`)
  turn = 1;
  unit_reduce<Sum, T, 2>(two, tmp, turn);
  const float e0 = two[0] * inv_dim, r = row_scale(two[1] * inv_dim, e0, a.eps);
  if (a.stats && t == 0) {
    float* const to = a.stats + row * STATS;
    to[0] = m;
    to[1] = e0;
    to[2] = r;
  }
  if (!a.y) return;
  float top[1] = {0.f};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + t) * E, a.dim);
    if (!at.any) continue;
    float w[E], b[E];
    row_gain<RAGGED, V, E>(a.w, a.w_f32, at, w);
    if (a.b) row_gain<RAGGED, V, E>(a.b, a.w_f32, at, b);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float xh = (h[n][e] - e0) * r;
      h[n][e] = a.b ? fmaf(xh, w[e], b[e]) : xh * w[e];
      if (at.of_row(e)) top[0] = fmaxf(top[0], fabsf(h[n][e]));
    }
    if (!a.scale) row_store<RAGGED, ONCE, V, E>((V*)a.y + row * a.dim, at, h[n]);
  }
  if (!a.scale) return;
  turn = 0;
  unit_reduce<Max, T, 1>(top, tmp, turn);
  const float scale = eight_scale(top[0]), inverse = 1.f / scale;
  if (t == 0) a.scale[row] = scale;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + t) * E, a.dim);
    if (at.any) row_store8<RAGGED, E>((unsigned char*)a.y + row * a.dim, at, h[n], inverse);
  }
}

// Rows of more than four accesses a thread of 1024, which the kernel above does not hold as floats: three passes over the
// row, or four, from cache as a rule, 16 bytes an access wherever a row begins (1024 bfloat16 rows of 65536 with their residual:
// 167 us, one element an access 380; the streams alone 104).  Packed in their 16-bit type rows of up to 65536 elements would
// fit registers; that is not built.
template <class V>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(const LayerNormArgs a) {
  constexpr int E = width<V>(), STEP = 1024 * E;
  __shared__ float tmp[4 * 16];
  const long row = blockIdx.x;
  const V* const x = (const V*)a.x + row * a.ldx;
  const V* const res = a.residual ? (const V*)a.residual + row * a.ldr : nullptr;
  const int begin = (int)threadIdx.x * E;
  const auto values = [&](const Place<true, E>& at, float (&v)[E]) {
    row_load<true, false, V, E>(x, at, v);
    if (!res) return;
    float b[E];
    row_load<true, false, V, E>(res, at, b);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = Element<V>::get(Element<V>::put(v[e] + b[e]));
  };
  int turn = 0;
  float s[1] = {0.f};
  for (int c = begin; c < a.dim; c += STEP) {
    const Place<true, E> at(c, a.dim);
    float v[E];
    values(at, v);
    if (a.h) row_store<true, false, V, E>((V*)a.h + row * a.dim, at, v);
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += at.of_row(e) ? v[e] : 0.f;
  }
  unit_reduce<Sum, 1024, 1>(s, tmp, turn);
  const float inv_dim = 1.f / (float)a.dim, m = s[0] * inv_dim;
  float two[2] = {0.f, 0.f};
  for (int c = begin; c < a.dim; c += STEP) {
    const Place<true, E> at(c, a.dim);
    float v[E];
    values(at, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = at.of_row(e) ? v[e] - m : 0.f;
      two[0] += d;
      two[1] = fmaf(d, d, two[1]);
    }
  }
  turn = 1;
  unit_reduce<Sum, 1024, 2>(two, tmp, turn);
  const float e0 = two[0] * inv_dim, r = row_scale(two[1] * inv_dim, e0, a.eps);
  if (a.stats && threadIdx.x == 0) {
    float* const to = a.stats + row * STATS;
    to[0] = m;
    to[1] = e0;
    to[2] = r;
  }
  if (!a.y) return;
  const auto results = [&](const Place<true, E>& at, float (&v)[E]) {
    float w[E], b[E];
    values(at, v);
    row_gain<true, V, E>(a.w, a.w_f32, at, w);
    if (a.b) row_gain<true, V, E>(a.b, a.w_f32, at, b);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float xh = ((v[e] - m) - e0) * r;
      v[e] = a.b ? fmaf(xh, w[e], b[e]) : xh * w[e];
    }
  };
  float scale = 1.f, inverse = 1.f;
  if (a.scale) {
    float top[1] = {0.f};
    for (int c = begin; c < a.dim; c += STEP) {
      float v[E];
      results(Place<true, E>(c, a.dim), v);
#pragma unroll
      for (int e = 0; e < E; ++e) top[0] = fmaxf(top[0], fabsf(v[e]));
    }
    turn = 0;
    unit_reduce<Max, 1024, 1>(top, tmp, turn);
    scale = eight_scale(top[0]);
    inverse = 1.f / scale;
    if (threadIdx.x == 0) a.scale[row] = scale;
  }
  for (int c = begin; c < a.dim; c += STEP) {
    const Place<true, E> at(c, a.dim);
    float v[E];
    results(at, v);
    if (a.scale) row_store8<true, E>((unsigned char*)a.y + row * a.dim, at, v, inverse);
    else row_store<true, false, V, E>((V*)a.y + row * a.dim, at, v);
  }
}

// ---------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------

struct LayerBackArgs {
  const void *dy, *dh, *h, *w;
  const float* stats;
  void* dx;
  float* partial;                         // [units][vectors][dim] s or its sum, then (whole) the same of s^2
  long rows, lddy, lddh, ldh;
  int dim, w_f32, vectors;                // vectors 2: the sums of dy beside those of dy xh
  Deal deal;
};

// The sums of a thread's columns: of the sample at hand, and (WHOLE) over the samples before
template <int E, bool WHOLE>
struct ColumnSums {
  float s[2][E], sum[2][WHOLE ? E : 1], sq[2][WHOLE ? E : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[k][e] = 0.f;
        if (WHOLE) sum[k][e] = sq[k][e] = 0.f;
      }
  }
  __device__ __forceinline__ void add(int e, float dy, float xh) {
    s[0][e] = fmaf(dy, xh, s[0][e]);
    s[1][e] += dy;
  }
  __device__ __forceinline__ void end_sample() {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sum[k][e] += s[k][e];
        sq[k][e] = fmaf(s[k][e], s[k][e], sq[k][e]);
        s[k][e] = 0.f;
      }
  }
  template <bool RAGGED>
  __device__ __forceinline__ void leave(const LayerBackArgs& a, int unit, const Place<RAGGED, E>& at) const {
    if (!at.any) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == a.vectors) break;
      float* const to = a.partial + ((long)unit * a.vectors + k) * a.dim + at.c;
      if constexpr (WHOLE) {
        store(to, at.count, sum[k]);
        store(to + (long)a.deal.units * a.vectors * a.dim, at.count, sq[k]);
      } else {
        store(to, at.count, s[k]);
      }
    }
  }

 private:
  static __device__ __forceinline__ void store(float* to, int count, const float (&x)[E]) {
    if (count == E) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *(loose4_floats*)(to + e) = u4{__float_as_uint(x[e]), __float_as_uint(x[e + 1]), __float_as_uint(x[e + 2]), __float_as_uint(x[e + 3])};
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < count) to[e] = x[e];
    }
  }
};

// Gradient and sums of rows that T threads hold, N accesses each
template <class V, int T, int N, bool WHOLE, bool RAGGED, bool ONCE>
__global__ __launch_bounds__(block_threads(T)) void layer_norm_backward_kernel(const LayerBackArgs a) {
  constexpr int E = width<V>();
  __shared__ float tmp[T > 64 ? 4 * T / 64 : 1];
  const int t = threadIdx.x % T;
  const int unit = blockIdx.x * (block_threads(T) / T) + threadIdx.x / T;
  if (unit >= a.deal.units) return;
  long row, last;
  unit_rows(a.deal, a.rows, unit, row, last);
  ColumnSums<E, WHOLE> sums[N];
#pragma unroll
  for (int n = 0; n < N; ++n) sums[n].clear();
  int turn = 0;
  const float inv_dim = 1.f / (float)a.dim;
  long token = 0;
  for (; row < last; ++row) {
    const float *const of = a.stats + row * STATS, m = of[0], e0 = of[1], r = of[2];
    float g[N][E], v[N][E], two[2] = {0.f, 0.f};
    Pack<V, E> dh[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const Place<RAGGED, E> at((n * T + t) * E, a.dim);
      if (!at.any) continue;
      row_load<RAGGED, ONCE, V, E>((const V*)a.dy + row * a.lddy, at, g[n]);
      row_load<RAGGED, ONCE, V, E>((const V*)a.h + row * a.ldh, at, v[n]);
      if (a.dh) dh[n] = row_load<RAGGED, ONCE, V, E>((const V*)a.dh + row * a.lddh, at);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const Place<RAGGED, E> at((n * T + t) * E, a.dim);
      if (!at.any) continue;
      float w[E];
      row_gain<RAGGED, V, E>(a.w, a.w_f32, at, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[n][e] = ((v[n][e] - m) - e0) * r;
        sums[n].add(e, g[n][e], v[n][e]);
        g[n][e] *= w[e];
        const float u = at.of_row(e) ? g[n][e] : 0.f;
        two[0] += u;
        two[1] = fmaf(u, v[n][e], two[1]);
      }
    }
    unit_reduce<Sum, T, 2>(two, tmp, turn);
    const float mean = two[0] * inv_dim, along = two[1] * inv_dim;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const Place<RAGGED, E> at((n * T + t) * E, a.dim);
      if (!at.any) continue;
      float d[E];
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = r * fmaf(-v[n][e], along, g[n][e] - mean);
      if (a.dh)
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] += Element<V>::get(dh[n].v[e]);
      row_store<RAGGED, ONCE, V, E>((V*)a.dx + row * a.dim, at, d);
    }
    if (WHOLE && ++token == a.deal.tokens) {
      token = 0;
#pragma unroll
      for (int n = 0; n < N; ++n) sums[n].end_sample();
    }
  }
  if (!a.partial) return;
#pragma unroll
  for (int n = 0; n < N; ++n) sums[n].template leave<RAGGED>(a, unit, Place<RAGGED, E>((n * T + t) * E, a.dim));
}

// The gradient alone of longer rows: N accesses each on 1024 threads
template <class V, int N, bool RAGGED, bool ONCE>
__global__ __launch_bounds__(1024) void layer_norm_dx_kernel(const LayerBackArgs a) {
  constexpr int E = width<V>(), T = 1024;
  __shared__ float tmp[4 * T / 64];
  const long row = blockIdx.x;
  const float *const of = a.stats + row * STATS, m = of[0], e0 = of[1], r = of[2];
  float g[N][E], v[N][E], two[2] = {0.f, 0.f};
  Pack<V, E> dh[N];
  int turn = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + (int)threadIdx.x) * E, a.dim);
    if (!at.any) continue;
    row_load<RAGGED, ONCE, V, E>((const V*)a.dy + row * a.lddy, at, g[n]);
    row_load<RAGGED, ONCE, V, E>((const V*)a.h + row * a.ldh, at, v[n]);
    if (a.dh) dh[n] = row_load<RAGGED, ONCE, V, E>((const V*)a.dh + row * a.lddh, at);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + (int)threadIdx.x) * E, a.dim);
    if (!at.any) continue;
    float w[E];
    row_gain<RAGGED, V, E>(a.w, a.w_f32, at, w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[n][e] = ((v[n][e] - m) - e0) * r;
      g[n][e] *= w[e];
      const float u = at.of_row(e) ? g[n][e] : 0.f;
      two[0] += u;
      two[1] = fmaf(u, v[n][e], two[1]);
    }
  }
  unit_reduce<Sum, T, 2>(two, tmp, turn);
  const float inv_dim = 1.f / (float)a.dim, mean = two[0] * inv_dim, along = two[1] * inv_dim;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const Place<RAGGED, E> at((n * T + (int)threadIdx.x) * E, a.dim);
    if (!at.any) continue;
    float d[E];
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = r * fmaf(-v[n][e], along, g[n][e] - mean);
    if (a.dh)
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] += Element<V>::get(dh[n].v[e]);
    row_store<RAGGED, ONCE, V, E>((V*)a.dx + row * a.dim, at, d);
  }
}

// ... of rows of more than four accesses a thread: two passes over the row, the second from cache as a rule (the backward pass
// of 1024 rows of 65536: 244 us with the sums over rows, one element an access 474; the streams alone 104)
template <class V>
__global__ __launch_bounds__(1024) void layer_norm_dx_long_kernel(const LayerBackArgs a) {
  constexpr int E = width<V>(), STEP = 1024 * E;
  __shared__ float tmp[4 * 16];
  const long row = blockIdx.x;
  const float *const of = a.stats + row * STATS, m = of[0], e0 = of[1], r = of[2];
  const int begin = (int)threadIdx.x * E;
  // u = gain dy and xh
  const auto terms = [&](const Place<true, E>& at, float (&u)[E], float (&xh)[E]) {
    float w[E];
    row_load<true, false, V, E>((const V*)a.dy + row * a.lddy, at, u);
    row_load<true, false, V, E>((const V*)a.h + row * a.ldh, at, xh);
    row_gain<true, V, E>(a.w, a.w_f32, at, w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      u[e] *= w[e];
      xh[e] = ((xh[e] - m) - e0) * r;
    }
  };
  float two[2] = {0.f, 0.f};
  int turn = 0;
  for (int c = begin; c < a.dim; c += STEP) {
    const Place<true, E> at(c, a.dim);
    float u[E], xh[E];
    terms(at, u, xh);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float one = at.of_row(e) ? u[e] : 0.f;
      two[0] += one;
      two[1] = fmaf(one, xh[e], two[1]);
    }
  }
  unit_reduce<Sum, 1024, 2>(two, tmp, turn);
  const float inv_dim = 1.f / (float)a.dim, mean = two[0] * inv_dim, along = two[1] * inv_dim;
  for (int c = begin; c < a.dim; c += STEP) {
    const Place<true, E> at(c, a.dim);
    float u[E], xh[E], d[E];
    terms(at, u, xh);
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = r * fmaf(-xh[e], along, u[e] - mean);
    if (a.dh) {
      float b[E];
      row_load<true, false, V, E>((const V*)a.dh + row * a.lddh, at, b);
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] += b[e];
    }
    row_store<true, false, V, E>((V*)a.dx + row * a.dim, at, d);
  }
}

// The sums alone: what they need of a row is kept, so a thread takes its columns down the rows of a unit.  `across`
// threads (a power of two) beside each other, the others of a workgroup on units of their own.
constexpr int COLUMN_THREADS = 256;
template <class V, bool WHOLE, bool RAGGED>
__global__ __launch_bounds__(COLUMN_THREADS) void layer_norm_columns_kernel(const LayerBackArgs a, int across) {
  constexpr int E = width<V>(), K = 4;                // rows in flight
  const Place<RAGGED, E> place((blockIdx.x * across + (threadIdx.x & (across - 1))) * E, a.dim);
  const int unit = blockIdx.y * (COLUMN_THREADS / across) + threadIdx.x / across;
  if (unit >= a.deal.units || !place.any) return;
  long row, last;
  unit_rows(a.deal, a.rows, unit, row, last);
  ColumnSums<E, WHOLE> sums;
  sums.clear();
  long token = 0;
  for (; row < last; row += K) {
    Pack<V, E> g[K], h[K];
    float stats[K][STATS];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long at = min(row + k, last - 1);
      g[k] = row_load<RAGGED, false, V, E>((const V*)a.dy + at * a.lddy, place);
      h[k] = row_load<RAGGED, false, V, E>((const V*)a.h + at * a.ldh, place);
#pragma unroll
      for (int i = 0; i < STATS; ++i) stats[k][i] = a.stats[at * STATS + i];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (row + k >= last) break;
#pragma unroll
      for (int e = 0; e < E; ++e)
        sums.add(e, Element<V>::get(g[k].v[e]), ((Element<V>::get(h[k].v[e]) - stats[k][0]) - stats[k][1]) * stats[k][2]);
      if (WHOLE && ++token == a.deal.tokens) {
        token = 0;
        sums.end_sample();
      }
    }
  }
  sums.template leave<RAGGED>(a, unit, place);
}

// Threads a row and accesses of a thread.  Forward: a wave with up to two accesses, then 128 threads with two, 256 and 1024
// with two to four.  (8193 rows of 5120 with their residual to 8 bits: three accesses on 256 threads 61 us, four of which a
// third is idle 65, ten on a wave 77; 16000 rows of 2048 with their residual: 128 threads 45, a wave with four accesses 52.)
constexpr Shape LAYER_SHAPES[] = {{64, 1}, {64, 2}, {128, 2}, {256, 2}, {256, 3}, {256, 4}, {1024, 2}, {1024, 3}, {1024, 4}};
Shape layer_norm_shape(int n) {
  for (const Shape& s : LAYER_SHAPES)
    if (n <= s.threads * s.accesses) return s;
  return Shape{0, 0};
}

// Backward, which holds three rows and the sums of two vectors: one access a thread, in as many units as are resident
// or a little more, so that each takes many rows and few partial sums are left.  In us with the curvature, in bfloat16:
//   16384 rows of 4096   512 threads, 512 units 108   1024 units 134   256 threads with two accesses, 1024 units 120
//   16000 rows of 2048   256, 768 units 62.5, 1024 units 64      8192 rows of 5120   768, 512 units 81; 512 with two accesses 92
//   4096 rows of 8192    1024, 256 units 68; 512 with two 84     16384 rows of 1024  128, 1280 units 41; 64 with two 51
//   16384 rows of 512    64, 2048 units 26; 4096 units 31        65536 rows of 64    64, 4096 units 40; 2048 units 43
// On 1024 threads a row may have two accesses where no squares are formed (2048 rows of 16384 79 us, the sums by themselves
// 105); beyond that, and with them (281 and 110), the sums are formed apart.
struct BackShape {
  int threads, units;
};
constexpr BackShape LAYER_BACK_SHAPES[] = {{64, 2048}, {128, 1280}, {256, 768}, {512, 512}, {768, 512}};
BackShape layer_backward_shape(int n) {
  if (n <= 16) return BackShape{64, 4096};
  for (const BackShape& s : LAYER_BACK_SHAPES)
    if (n <= s.threads) return s;
  // (rows whose sums are formed apart: fewer units for more columns, as the partial sums are a row each)
  return BackShape{1024, n <= 2048 ? 256 : std::max(8, (1 << 19) / n)};
}

// `n` rows of `a` from `first` on
template <class V>
LayerNormArgs layer_norm_rows(LayerNormArgs a, long first, long n) {
  const auto ahead = [](const void* p, long elements, size_t size) { return p ? (const char*)p + elements * (long)size : nullptr; };
  a.x = ahead(a.x, first * a.ldx, sizeof(V));
  a.residual = ahead(a.residual, first * a.ldr, sizeof(V));
  a.y = (void*)ahead(a.y, first * a.dim, a.scale ? 1 : sizeof(V));
  a.h = (void*)ahead(a.h, first * a.dim, sizeof(V));
  a.scale = (float*)ahead(a.scale, first, sizeof(float));
  a.stats = (float*)ahead(a.stats, first * STATS, sizeof(float));
  a.rows = n;
  return a;
}

template <class V>
int accesses(int dim) {
  return (dim + width<V>() - 1) / width<V>();
}

template <class V, bool RAGGED, bool ONCE>
void launch_layer_norm(const LayerNormArgs& a, hipStream_t stream) {
  const Shape s = layer_norm_shape(accesses<V>(a.dim));
#define NORM_CASE(T, N)                                                                                   \
  if (s.threads == T && s.accesses == N) {                                                                \
    for_row_ranges(a.rows, block_threads(T), block_threads(T) / T, [&](long first, long n, unsigned blocks) { \
      hipLaunchKernelGGL((layer_norm_kernel<V, T, N, RAGGED, ONCE>), dim3(blocks), dim3(block_threads(T)), 0, stream, \
                         layer_norm_rows<V>(a, first, n));                                                \
    });                                                                                                   \
    return;                                                                                               \
  }
  NORM_CASE(64, 1) NORM_CASE(64, 2) NORM_CASE(128, 2)
  NORM_CASE(256, 2) NORM_CASE(256, 3) NORM_CASE(256, 4)
  NORM_CASE(1024, 2) NORM_CASE(1024, 3) NORM_CASE(1024, 4)
#undef NORM_CASE
  for_row_ranges(a.rows, 1024, 1, [&](long first, long n, unsigned blocks) {
    hipLaunchKernelGGL((layer_norm_long_kernel<V>), dim3(blocks), dim3(1024), 0, stream, layer_norm_rows<V>(a, first, n));
  });
}
template <class V>
void launch_layer_norm(const LayerNormArgs& a, bool ragged, hipStream_t stream) {
  const long bytes = a.rows * a.dim * (long)((a.residual ? 3 : a.h ? 2 : 1) * sizeof(V) + (a.scale ? 1 : a.y ? sizeof(V) : 0));
  if (ragged) launch_layer_norm<V, true, false>(a, stream);
  else if (bytes > LAST_CACHE) launch_layer_norm<V, false, true>(a, stream);
  else launch_layer_norm<V, false, false>(a, stream);
}

// `n` rows from `first` on, for passes over single rows
template <class V>
LayerBackArgs layer_back_rows(LayerBackArgs a, long first, long n) {
  a.dy = (const V*)a.dy + first * a.lddy;
  if (a.dh) a.dh = (const V*)a.dh + first * a.lddh;
  a.h = (const V*)a.h + first * a.ldh;
  a.stats += first * STATS;
  a.dx = (V*)a.dx + first * a.dim;
  a.rows = n;
  return a;
}

template <class V, bool RAGGED>
void launch_columns(const LayerBackArgs& a, hipStream_t stream) {
  const int n = accesses<V>(a.dim);
  int across = 1;
  while (across < n && across < COLUMN_THREADS) across *= 2;
  // (rows of the grid are counted in 16 bits)
  const int per = COLUMN_THREADS / across, rows = cdiv(a.deal.units, per);
  const dim3 grid(cdiv(n, across), rows);
  if (a.deal.whole)
    hipLaunchKernelGGL((layer_norm_columns_kernel<V, true, RAGGED>), grid, dim3(COLUMN_THREADS), 0, stream, a, across);
  else
    hipLaunchKernelGGL((layer_norm_columns_kernel<V, false, RAGGED>), grid, dim3(COLUMN_THREADS), 0, stream, a, across);
}

template <class V, bool RAGGED, bool ONCE>
void launch_layer_backward(const LayerBackArgs& a, hipStream_t stream) {
  const int n = accesses<V>(a.dim);
  if (!a.dx) return launch_columns<V, RAGGED>(a, stream);
  const int threads = layer_backward_shape(n).threads;
#define BACK_CASE(T, N, WHOLE)                                                                            \
  if (n <= T * N && threads == T && (bool)a.deal.whole == WHOLE) {                                        \
    const dim3 grid(cdiv(a.deal.units, block_threads(T) / T)), block(block_threads(T));                   \
    hipLaunchKernelGGL((layer_norm_backward_kernel<V, T, N, WHOLE, RAGGED, ONCE>), grid, block, 0, stream, a); \
    return;                                                                                               \
  }
#define BACK_CASES(T) BACK_CASE(T, 1, false) BACK_CASE(T, 1, true)
  BACK_CASES(64) BACK_CASES(128) BACK_CASES(256) BACK_CASES(512) BACK_CASES(768) BACK_CASES(1024)
  BACK_CASE(1024, 2, false)
#undef BACK_CASES
#undef BACK_CASE
  if (a.partial) launch_columns<V, RAGGED>(a, stream);
  for_row_ranges(a.rows, 1024, 1, [&](long first, long rows, unsigned blocks) {
    const LayerBackArgs part = layer_back_rows<V>(a, first, rows);
    if (n <= 2 * 1024)
      hipLaunchKernelGGL((layer_norm_dx_kernel<V, 2, RAGGED, ONCE>), dim3(blocks), dim3(1024), 0, stream, part);
    else if (n <= 4 * 1024)
      hipLaunchKernelGGL((layer_norm_dx_kernel<V, 4, RAGGED, ONCE>), dim3(blocks), dim3(1024), 0, stream, part);
    else hipLaunchKernelGGL((layer_norm_dx_long_kernel<V>), dim3(blocks), dim3(1024), 0, stream, part);
  });
}
template <class V>
void launch_layer_backward(const LayerBackArgs& a, bool ragged, hipStream_t stream) {
  const long bytes = a.rows * a.dim * (long)((2 + (a.dh != nullptr) + (a.dx != nullptr)) * sizeof(V));
  if (ragged) launch_layer_backward<V, true, false>(a, stream);
  else if (bytes > LAST_CACHE) launch_layer_backward<V, false, true>(a, stream);
  else launch_layer_backward<V, false, false>(a, stream);
}

// (the deal must not depend on alignment or on what is wanted: the caller asks for scratch by sizes alone)
Deal layer_deal(int type, int64_t rows, int dim, int samples, bool squares) {
  const int e = type == TYPE_F32 ? 4 : 8;
  return deal_rows((long)rows, samples, squares, layer_backward_shape((dim + e - 1) / e).units);
}
size_t layer_backward_floats(const Deal& d, int dim, int vectors) { return (size_t)d.units * dim * vectors * (d.whole ? 2 : 1); }

}  // namespace
}  // namespace kfac

using namespace kfac;

extern "C" {

int kfac_layer_norm(int type, int gain_is_float, int64_t rows, int dim, const void* x, int64_t ldx,
                    const void* residual, int64_t ldr, const void* gain, const void* bias, float eps, void* y, void* h,
                    float* scale, float* stats, void* stream) {
  if (!norm_args_ok(type, gain_is_float, rows, dim, eps)) return KFAC_ERR_ARG;
  if (rows == 0) return KFAC_OK;
  if (!x || (!y && !stats) || (residual && !h) || (bias && !gain) || (scale && !y) || ldx < 0 || ldr < 0)
    return KFAC_ERR_ARG;
  const LayerNormArgs a{x, residual, gain, bias, y, h, scale, stats, (long)rows, (long)ldx, (long)ldr, dim, gain_is_float, eps};
  const int e = type == TYPE_F32 ? 4 : 8;
  const bool ragged = !aligned(dim, e, {{x, a.ldx}, {residual, a.ldr}, {y, dim}, {h, dim}, {bias, dim}}, gain, gain_is_float);
  const hipStream_t s = (hipStream_t)stream;
  if (type == TYPE_F32) launch_layer_norm<float>(a, ragged, s);
  else if (type == TYPE_BF16) launch_layer_norm<__hip_bfloat16>(a, ragged, s);
  else launch_layer_norm<_Float16>(a, ragged, s);
  return launch_status();
}

size_t kfac_layer_norm_backward_workspace_bytes(int type, int64_t rows, int dim, int samples, int vectors, int squares) {
  if (!norm_args_ok(type, 0, rows, dim, 0.f) || samples <= 0 || rows == 0 || rows % samples != 0 || vectors < 1 ||
      vectors > 2)
    return 0;
  return sizeof(float) * layer_backward_floats(layer_deal(type, rows, dim, samples, squares != 0), dim, vectors);
}

int kfac_layer_norm_backward(int type, int gain_is_float, int64_t rows, int dim, int samples, int vectors, const void* dy,
                             int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh, const float* stats,
                             const void* gain, void* dx, void* dgain, void* dbias, float* curvature, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (!norm_args_ok(type, gain_is_float, rows, dim, 0.f) || samples <= 0 || rows % samples != 0 || vectors < 1 || vectors > 2)
    return KFAC_ERR_ARG;
  if (rows == 0 || !dy || !h || !stats || lddy < 0 || lddh < 0 || ldh < 0 || (dh && !dx) || (dbias && vectors != 2))
    return KFAC_ERR_ARG;
  const bool sums = dgain || dbias || curvature;
  if (!sums && !dx) return KFAC_OK;
  LayerBackArgs a{dy, dh, h, gain, stats, dx, nullptr, (long)rows, (long)lddy, (long)lddh, (long)ldh, dim, gain_is_float, vectors, {}};
  a.deal = layer_deal(type, rows, dim, samples, curvature != nullptr);
  if (sums) {
    if (!workspace || workspace_bytes < sizeof(float) * layer_backward_floats(a.deal, dim, vectors)) return KFAC_ERR_WORKSPACE;
    a.partial = (float*)workspace;
  }
  const int e = type == TYPE_F32 ? 4 : 8;
  const bool ragged = !aligned(dim, e, {{dy, a.lddy}, {dh, a.lddh}, {h, a.ldh}, {dx, dim}, {a.partial, dim}}, gain, gain_is_float);
  const hipStream_t s = (hipStream_t)stream;
  if (type == TYPE_F32) launch_layer_backward<float>(a, ragged, s);
  else if (type == TYPE_BF16) launch_layer_backward<__hip_bfloat16>(a, ragged, s);
  else launch_layer_backward<_Float16>(a, ragged, s);
  if (sums)
    launch_reduce(a.partial, a.deal, vectors * dim, dim, dgain, dbias, gain_is_float ? TYPE_F32 : type, curvature, s);
  return launch_status();
}

}  // extern "C"
