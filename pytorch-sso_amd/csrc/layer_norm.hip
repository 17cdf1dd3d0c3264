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
// so that rows far off zero keep their digits: e takes what rounding has lost of m.  (m is a quotient: a product
// would be fused into the differences h - m, and what is kept of it, rounded, would be another number.)  A forward pass with a backward
// pass behind it keeps (m, e, r) of each row, 12 bytes, which spares that pass its first two sums.  The sums over
// rows stay in registers over the rows of a unit (a wave or a workgroup), whose partial sums a second launch adds up
// in order.
#include "norm_core.h"

namespace kfac {
namespace {

constexpr int STATS = 3;                  // numbers kept of a row: m, e, r

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

// T threads a row, N accesses of E elements each.
template <class V, int E, int T, int N, bool ONCE>
__global__ __launch_bounds__(block_threads(T)) void layer_norm_kernel(const LayerNormArgs a) {
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
  float s[1] = {0.f};
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += h[n][e];
  unit_reduce<Sum, T, 1>(s, tmp, turn);
  const float inv_dim = 1.f / (float)a.dim, m = s[0] / (float)a.dim;
  float two[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * T + t) * E;
    if (c >= a.dim) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[n][e] -= m;
      two[0] += h[n][e];
      two[1] = fmaf(h[n][e], h[n][e], two[1]);
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
    const int c = (n * T + t) * E;
    if (c >= a.dim) continue;
    float w[E], b[E];
    load_gain<V, E>(a.w, a.w_f32, c, w);
    if (a.b) load_gain<V, E>(a.b, a.w_f32, c, b);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float xh = (h[n][e] - e0) * r;
      h[n][e] = a.b ? fmaf(xh, w[e], b[e]) : xh * w[e];
      top[0] = fmaxf(top[0], fabsf(h[n][e]));
    }
    if (!a.scale) stream_store<ONCE, V, E>((V*)a.y + row * a.dim + c, h[n]);
  }
  if (!a.scale) return;
  turn = 0;
  unit_reduce<Max, T, 1>(top, tmp, turn);
  const float scale = top[0] > 0.f ? top[0] / LARGEST_8 : 1.f;
  if (t == 0) a.scale[row] = scale;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * T + t) * E;
    if (c < a.dim) store8<E>((unsigned char*)a.y + row * a.dim + c, h[n], scale);
  }
}

// Rows that do not fit registers: three passes over the row, or four, from cache as a rule.
template <class V>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(const LayerNormArgs a) {
  __shared__ float tmp[4 * 16];
  const long row = blockIdx.x;
  const V* const x = (const V*)a.x + row * a.ldx;
  const V* const res = a.residual ? (const V*)a.residual + row * a.ldr : nullptr;
  const auto value = [&](int c) {
    float v[1];
    load<V, 1>(x + c, v);
    if (res) v[0] = Element<V>::get(Element<V>::put(v[0] + Element<V>::get(res[c])));
    return v[0];
  };
  int turn = 0;
  float s[1] = {0.f};
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float v = value(c);
    if (a.h) ((V*)a.h)[row * a.dim + c] = Element<V>::put(v);
    s[0] += v;
  }
  unit_reduce<Sum, 1024, 1>(s, tmp, turn);
  const float inv_dim = 1.f / (float)a.dim, m = s[0] / (float)a.dim;
  float two[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float d = value(c) - m;
    two[0] += d;
    two[1] = fmaf(d, d, two[1]);
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
  const auto result = [&](int c) {
    float w[1], b[1] = {0.f};
    load_gain<V, 1>(a.w, a.w_f32, c, w);
    const float xh = ((value(c) - m) - e0) * r;
    if (!a.b) return xh * w[0];
    load_gain<V, 1>(a.b, a.w_f32, c, b);
    return fmaf(xh, w[0], b[0]);
  };
  float top[1] = {0.f};
  if (a.scale) {
    for (int c = threadIdx.x; c < a.dim; c += 1024) top[0] = fmaxf(top[0], fabsf(result(c)));
    turn = 0;
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

struct LayerBackArgs {
  const void *dy, *dh, *h, *w;
  const float* stats;
  void* dx;
  float* partial;                         // [units][vectors][dim] s or its sum, then (whole) the same of s^2
  long rows, lddy, lddh, ldh;
  int dim, w_f32;
  Deal deal;
};

// B: the sums of dy are formed beside those of dy xh.
template <class V, int E, int T, int N, bool B, bool WHOLE, bool ONCE>
__global__ __launch_bounds__(block_threads(T)) void layer_norm_backward_kernel(const LayerBackArgs a) {
  constexpr int K = B ? 2 : 1;
  __shared__ float tmp[T > 64 ? 4 * T / 64 : 1];
  const int t = threadIdx.x % T;
  const int unit = blockIdx.x * (block_threads(T) / T) + threadIdx.x / T;
  if (unit >= a.deal.units) return;
  long row, last;
  unit_rows(a.deal, a.rows, unit, row, last);
  float s[K][N][E], sum[K][WHOLE ? N : 1][E], sq[K][WHOLE ? N : 1][E];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[k][n][e] = 0.f;
        if (WHOLE) sum[k][n][e] = sq[k][n][e] = 0.f;
      }
  int turn = 0;
  const float inv_dim = 1.f / (float)a.dim;
  long token = 0;
  for (; row < last; ++row) {
    const V* const dy = (const V*)a.dy + row * a.lddy;
    const V* const h = (const V*)a.h + row * a.ldh;
    const float *const of = a.stats + row * STATS, m = of[0], e0 = of[1], r = of[2];
    float g[N][E], v[N][E];
    Pack<V, E> dh[N];
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
    float two[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * T + t) * E;
      if (c >= a.dim) continue;
      float w[E];
      load_gain<V, E>(a.w, a.w_f32, c, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[n][e] = ((v[n][e] - m) - e0) * r;
        s[0][n][e] = fmaf(g[n][e], v[n][e], s[0][n][e]);
        if (B) s[K - 1][n][e] += g[n][e];
        g[n][e] *= w[e];
        two[0] += g[n][e];
        two[1] = fmaf(g[n][e], v[n][e], two[1]);
      }
    }
    if (a.dx) {
      unit_reduce<Sum, T, 2>(two, tmp, turn);
      const float mean = two[0] * inv_dim, along = two[1] * inv_dim;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * T + t) * E;
        if (c >= a.dim) continue;
        float d[E];
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = r * ((g[n][e] - mean) - v[n][e] * along);
        if (a.dh)
#pragma unroll
          for (int e = 0; e < E; ++e) d[e] += Element<V>::get(dh[n].v[e]);
        stream_store<ONCE, V, E>((V*)a.dx + row * a.dim + c, d);
      }
    }
    if (WHOLE && ++token == a.deal.tokens) {
      token = 0;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            sum[k][n][e] += s[k][n][e];
            sq[k][n][e] = fmaf(s[k][n][e], s[k][n][e], sq[k][n][e]);
            s[k][n][e] = 0.f;
          }
    }
  }
  if (!a.partial) return;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float* const to = a.partial + ((long)unit * K + k) * a.dim;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * T + t) * E;
      if (c >= a.dim) continue;
      if (WHOLE) {
        store<float, E>(to + c, sum[k][n]);
        store<float, E>(to + (long)a.deal.units * K * a.dim + c, sq[k][n]);
      } else {
        store<float, E>(to + c, s[k][n]);
      }
    }
  }
}

// Rows that do not fit registers: the sums of a unit stay in its partial sums in memory (every column is the same
// thread's throughout).  With squares, a third row of them holds s_n.
template <class V>
__global__ __launch_bounds__(1024) void layer_norm_backward_long_kernel(const LayerBackArgs a, float* current, int vectors) {
  __shared__ float tmp[4 * 16];
  long row, last;
  unit_rows(a.deal, a.rows, blockIdx.x, row, last);
  const long at = (long)blockIdx.x * vectors * a.dim;
  float* const to = a.partial ? a.partial + at : nullptr;
  float* const sq = to + (long)a.deal.units * vectors * a.dim;
  float* const cur = a.deal.whole ? current + at : to;
  if (to)
    for (int k = 0; k < vectors; ++k)
      for (int c = threadIdx.x; c < a.dim; c += 1024) {
        const long i = (long)k * a.dim + c;
        to[i] = 0.f;
        if (a.deal.whole) sq[i] = cur[i] = 0.f;
      }
  int turn = 0;
  long token = 0;
  for (; row < last; ++row) {
    const V* const dy = (const V*)a.dy + row * a.lddy;
    const V* const h = (const V*)a.h + row * a.ldh;
    const float *const of = a.stats + row * STATS, m = of[0], e0 = of[1], r = of[2];
    float two[2] = {0.f, 0.f};
    if (a.dx) {
      for (int c = threadIdx.x; c < a.dim; c += 1024) {
        float w[1];
        load_gain<V, 1>(a.w, a.w_f32, c, w);
        const float xh = ((Element<V>::get(h[c]) - m) - e0) * r, u = w[0] * Element<V>::get(dy[c]);
        two[0] += u;
        two[1] = fmaf(u, xh, two[1]);
      }
      unit_reduce<Sum, 1024, 2>(two, tmp, turn);
    }
    const float mean = two[0] / (float)a.dim, along = two[1] / (float)a.dim;
    const bool ends = a.deal.whole && ++token == a.deal.tokens;
    if (ends) token = 0;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      const float xh = ((Element<V>::get(h[c]) - m) - e0) * r, g = Element<V>::get(dy[c]);
      if (to)
        for (int k = 0; k < vectors; ++k) {
          const long i = (long)k * a.dim + c;
          float s = k == 0 ? fmaf(g, xh, cur[i]) : cur[i] + g;
          if (ends) {
            to[i] += s;
            sq[i] = fmaf(s, s, sq[i]);
            s = 0.f;
          }
          cur[i] = s;
        }
      if (a.dx) {
        float w[1];
        load_gain<V, 1>(a.w, a.w_f32, c, w);
        float d = r * ((w[0] * g - mean) - xh * along);
        if (a.dh) d += Element<V>::get(((const V*)a.dh)[row * a.lddh + c]);
        ((V*)a.dx)[row * a.dim + c] = Element<V>::put(d);
      }
    }
  }
}

// backward, which holds three rows and the sums of two vectors: at most two accesses a thread
constexpr Shape LAYER_BACK_SHAPES[] = {{64, 1}, {64, 2}, {256, 1}, {256, 2}, {512, 2}, {1024, 2}};
Shape layer_backward_shape(int dim, int e) {
  const int n = (dim + e - 1) / e, scale = e == 1 ? 8 : 1;
  for (const Shape& s : LAYER_BACK_SHAPES)
    if (n <= s.threads * s.accesses * scale) return Shape{s.threads, s.accesses * scale};
  return Shape{0, 0};
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

template <class V, int E, bool ONCE = false>
void launch_layer_norm(const LayerNormArgs& a, hipStream_t stream) {
  const long bytes = a.rows * a.dim * (long)((a.residual ? 3 : a.h ? 2 : 1) * sizeof(V) + (a.scale ? 1 : a.y ? sizeof(V) : 0));
  if constexpr (E > 1 && !ONCE)
    if (bytes > LAST_CACHE) return launch_layer_norm<V, E, true>(a, stream);
  const Shape s = norm_shape(a.dim, E);
#define NORM_CASE(T, N)                                                                                   \
  if (s.threads == T && s.accesses == N) {                                                                \
    for_row_ranges(a.rows, block_threads(T), block_threads(T) / T, [&](long first, long n, unsigned blocks) { \
      hipLaunchKernelGGL((layer_norm_kernel<V, E, T, N, ONCE>), dim3(blocks), dim3(block_threads(T)), 0, stream, \
                         layer_norm_rows<V>(a, first, n));                                                \
    });                                                                                                   \
    return;                                                                                               \
  }
  constexpr int M = E == 1 ? 16 : 4;
  NORM_CASE(64, M / 4) NORM_CASE(64, M / 2) NORM_CASE(64, M)
  NORM_CASE(256, M / 4) NORM_CASE(256, M / 2) NORM_CASE(256, M)
  NORM_CASE(1024, M / 4) NORM_CASE(1024, M / 2) NORM_CASE(1024, M)
#undef NORM_CASE
  for_row_ranges(a.rows, 1024, 1, [&](long first, long n, unsigned blocks) {
    hipLaunchKernelGGL((layer_norm_long_kernel<V>), dim3(blocks), dim3(1024), 0, stream, layer_norm_rows<V>(a, first, n));
  });
}

template <class V, int E, bool ONCE = false>
void launch_layer_backward(const LayerBackArgs& a, float* current, int vectors, hipStream_t stream) {
  const long bytes = a.rows * a.dim * (long)((2 + (a.dh != nullptr) + (a.dx != nullptr)) * sizeof(V));
  if constexpr (E > 1 && !ONCE)
    if (bytes > LAST_CACHE) return launch_layer_backward<V, E, true>(a, current, vectors, stream);
  const Shape s = layer_backward_shape(a.dim, E);
#define BACK_LAUNCH(T, N, B, W) \
  hipLaunchKernelGGL((layer_norm_backward_kernel<V, E, T, N, B, W, ONCE>), grid, block, 0, stream, a)
#define BACK_CASE(T, N)                                                                                   \
  if (s.threads == T && s.accesses == N) {                                                                \
    const int per = block_threads(T) / T;                                                                 \
    const dim3 grid(cdiv(a.deal.units, per)), block(block_threads(T));                                    \
    if (vectors == 2) {                                                                                   \
      if (a.deal.whole) BACK_LAUNCH(T, N, true, true);                                                    \
      else BACK_LAUNCH(T, N, true, false);                                                                \
    } else {                                                                                              \
      if (a.deal.whole) BACK_LAUNCH(T, N, false, true);                                                   \
      else BACK_LAUNCH(T, N, false, false);                                                               \
    }                                                                                                     \
    return;                                                                                               \
  }
  constexpr int M = E == 1 ? 8 : 1;
  BACK_CASE(64, M) BACK_CASE(64, 2 * M) BACK_CASE(256, M) BACK_CASE(256, 2 * M) BACK_CASE(512, 2 * M) BACK_CASE(1024, 2 * M)
#undef BACK_CASE
#undef BACK_LAUNCH
  hipLaunchKernelGGL((layer_norm_backward_long_kernel<V>), dim3(a.deal.units), dim3(1024), 0, stream, a, current, vectors);
}

// (the deal must not depend on alignment: the caller asks for scratch by sizes alone)
Deal layer_deal(int type, int64_t rows, int dim, int samples, bool squares) {
  return deal_rows((long)rows, samples, squares, layer_backward_shape(dim, type == TYPE_F32 ? 4 : 8).threads);
}

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
  const bool vec = aligned(dim, e, {{x, a.ldx}, {residual, a.ldr}, {y, dim}, {h, dim}, {bias, dim}}, gain, gain_is_float);
  const hipStream_t s = (hipStream_t)stream;
  if (type == TYPE_F32) vec ? launch_layer_norm<float, 4>(a, s) : launch_layer_norm<float, 1>(a, s);
  else if (type == TYPE_BF16)
    vec ? launch_layer_norm<__hip_bfloat16, 8>(a, s) : launch_layer_norm<__hip_bfloat16, 1>(a, s);
  else vec ? launch_layer_norm<_Float16, 8>(a, s) : launch_layer_norm<_Float16, 1>(a, s);
  return launch_status();
}

size_t kfac_layer_norm_backward_workspace_bytes(int type, int64_t rows, int dim, int samples, int vectors, int squares) {
  if (!norm_args_ok(type, 0, rows, dim, 0.f) || samples <= 0 || rows == 0 || rows % samples != 0 || vectors < 1 ||
      vectors > 2)
    return 0;
  return sizeof(float) * vectors * backward_floats(layer_deal(type, rows, dim, samples, squares != 0), dim);
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
  LayerBackArgs a{dy, dh, h, gain, stats, dx, nullptr, (long)rows, (long)lddy, (long)lddh, (long)ldh, dim, gain_is_float, {}};
  a.deal = layer_deal(type, rows, dim, samples, curvature != nullptr);
  float* current = nullptr;
  if (sums) {
    if (!workspace || workspace_bytes < sizeof(float) * vectors * backward_floats(a.deal, dim)) return KFAC_ERR_WORKSPACE;
    a.partial = (float*)workspace;
    current = a.partial + 2 * (size_t)vectors * a.deal.units * dim;
  }
  const int e = type == TYPE_F32 ? 4 : 8;
  const bool vec = aligned(dim, e, {{dy, a.lddy}, {dh, a.lddh}, {h, a.ldh}, {dx, dim}, {a.partial, dim}}, gain, gain_is_float);
  const hipStream_t s = (hipStream_t)stream;
  if (type == TYPE_F32)
    vec ? launch_layer_backward<float, 4>(a, current, vectors, s) : launch_layer_backward<float, 1>(a, current, vectors, s);
  else if (type == TYPE_BF16)
    vec ? launch_layer_backward<__hip_bfloat16, 8>(a, current, vectors, s)
        : launch_layer_backward<__hip_bfloat16, 1>(a, current, vectors, s);
  else
    vec ? launch_layer_backward<_Float16, 8>(a, current, vectors, s) : launch_layer_backward<_Float16, 1>(a, current, vectors, s);
  if (sums)
    launch_reduce(a.partial, a.deal, vectors * dim, dim, dgain, dbias, gain_is_float ? TYPE_F32 : type, curvature, s);
  return launch_status();
}

}  // extern "C"
