// What the norms of rows have in common: access to rows, sums over a row, how rows are dealt to units in a
// backward pass, and the sum of what the units leave.
#pragma once
#include <utility>

#include "common.h"
#include "element_types.h"
#include "norm_rows.h"

namespace kfac {
namespace {

constexpr float LARGEST_8 = 448.f;        // of the 8-bit type (4 exponent bits, 3 of the significand)

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

// x of the lane that is O away (xor), in registers: lanes of 16 rotate (what is added or compared has come to
// repeat every 2 O lanes by then, so that a rotation by O is that), rows and halves are swapped.  In the caller's order
// 32, 16, 8, 4, 2, 1.
template <class OP, int O>
__device__ __forceinline__ float with_other(float x) {
  const unsigned u = __float_as_uint(x);
  if constexpr (O == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return OP::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  } else if constexpr (O == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return OP::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  } else {
    return OP::of(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, u, 0x120 + O, 0xf, 0xf, true)));
  }
}

// Over the threads of a unit, the same in each: a wave, or a workgroup of T threads (`tmp`: room for
// 2 K T / 64 floats, `turn` alternates so that one barrier is enough).
template <class OP, int T, int K>
__device__ __forceinline__ void unit_reduce(float (&v)[K], float* tmp, int& turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = with_other<OP, 32>(v[k]);
    v[k] = with_other<OP, 16>(v[k]);
    v[k] = with_other<OP, 8>(v[k]);
    v[k] = with_other<OP, 4>(v[k]);
    v[k] = with_other<OP, 2>(v[k]);
    v[k] = with_other<OP, 1>(v[k]);
  }
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

// threads of a workgroup of units of T threads: waves by fours, larger units by themselves
constexpr int block_threads(int T) { return T == 64 ? 256 : T; }

// How the rows are dealt to units.  parts > 0: a unit takes one of `parts` pieces (of `rows` rows)
// of a sample, and leaves its part of s_n; parts == 0: it takes `rows` / tokens whole samples, or
// just rows where no curvature is wanted, and leaves its part of dw and of sum s_n^2.
struct Deal {
  int units, parts, samples;
  long tokens, rows;
  int whole;                              // squares are formed in the units
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

// The partial sums of the units, added up in 64 bits (rounded once on the way, a group's sum) and in an order
// that depends on their number alone.  A workgroup
// takes 32 columns, E of them to a thread, in G groups of threads over the units (1024 units of 4096 columns,
// a sample each 6.4 us, of 8 samples 7.0; in 24 with 16 groups of a column to a thread).  The first `split`
// columns are those of dw, the others those of db.
constexpr int REDUCE_COLUMNS = 32, REDUCE_THREADS = 1024;
template <int E>
__global__ __launch_bounds__(REDUCE_THREADS) void norm_reduce_kernel(const float* partial, Deal d, int dim, int split,
                                                                     void* dw, void* db, int w_type, float* curvature) {
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
  } else if (void* const out = to < split ? dw : db) {
    const int at = to < split ? to : to - split;
    if (w_type == TYPE_F32) ((float*)out)[at] = (float)all;
    else if (w_type == TYPE_BF16) ((__hip_bfloat16*)out)[at] = Element<__hip_bfloat16>::put((float)all);
    else ((_Float16*)out)[at] = Element<_Float16>::put((float)all);
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
// to about `target` units
Deal deal_rows(long rows, int samples, bool squares, long target) {
  Deal d;
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

// (with squares the units leave those too, and a row that does not fit registers needs room for one more)
size_t backward_floats(const Deal& d, int dim) { return (size_t)d.units * dim * (d.whole ? 3 : 1); }

void launch_reduce(const float* partial, const Deal& d, int dim, int split, void* dw, void* db, int w_type,
                   float* curvature, hipStream_t stream) {
  hipLaunchKernelGGL((dim % 4 == 0 && ((uintptr_t)partial & 15) == 0 ? norm_reduce_kernel<4> : norm_reduce_kernel<1>),
                     dim3(cdiv(dim, REDUCE_COLUMNS)), dim3(REDUCE_THREADS), 0, stream, partial, d, dim, split, dw, db,
                     w_type, curvature);
}

}  // namespace
}  // namespace kfac
