// AdamW: one update of a list of tensors, with states in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2
//   p = (1 - lr wd) p - m / (root sqrt(v) + eps'),   root = 1 / (size sqrt(1 - b2^t)),  eps' = eps / size,
//                                                    size = lr / (1 - b1^t)
//
// In 8 bits a state is kept by blocks of 128 consecutive elements with a float32 scale each: m / scale in e4m3 with
// scale = max |m| / 448 of the block, v / scale in e5m2 with scale = max v / 57344.  Both are rounded at random to one of
// their two neighbours, so that what an update adds is kept on average: with b2 = 0.999 a v moves by a thousandth of
// (g^2 - v) an update, and rounding to the nearest number, at least a sixteenth away, would never move it.  e5m2 for v
// and not e4m3 for its root, which has the same steps: v's own mean is what rounding at random keeps.  A v above 0
// never becomes 0, whose root would stand alone with eps.  The update uses m and v as they are before they are rounded.
//
// Bound by memory: 3 s + 16 bytes an element with states in 32 bits (s: a parameter's), 3 s + 4.25 in 8.  A thread takes
// 8 consecutive elements, so 16 threads hold a block, and every stream is read and written once, 16 bytes at a time (8
// of an 8-bit state).  The list travels as a kernel argument, as that of the other element-wise passes (elementwise.hip).
// 244 million bfloat16 parameters: 991 us in 32 bits, 5.4 TB/s, and 388 in 8, 6.4, where a large copy reaches 5.2; a
// ResNet-50 in float32 142 us, 5.0 TB/s.  With twice and four times the elements to a workgroup the last takes 3 and 6 % longer.
#include <cmath>

#include "common.h"
#include "element_types.h"

namespace kfac {
namespace {

constexpr int ADAM_THREADS = 256, UNIT = 8, BLOCK = 128, LANES = BLOCK / UNIT;
constexpr long ADAM_GROUP = ADAM_THREADS * UNIT;     // elements of a workgroup
constexpr long ADAM_MOST_GROUPS = (1L << 32) / ADAM_THREADS - 1;      // a launch has fewer than 2^32 threads
constexpr float LARGEST_M = 448.f, LARGEST_V = 57344.f, LEAST_V = 0x1p-16f;
// A block whose largest number is below this is kept as zeros (its reciprocal scale would overflow).
constexpr float LEAST_TOP = 0x1p-100f;
constexpr unsigned INFINITE = 0x7f800000u;

// What depends on the number of the update
struct AdamScalars {
  float keep, root, eps;                  // 1 - lr wd, and what stands above
  unsigned key;                           // of its random numbers
};
struct AdamRates {
  float b1, c1, b2, c2;                   // c: 1 - b
};

template <int BITS> struct AdamTensor;
template <> struct AdamTensor<32> {
  void *p, *m, *v;
  const void* g;
  long n;
};
template <> struct AdamTensor<8> {
  void *p, *m, *v;
  const void* g;
  float *m_scale, *v_scale;
  long n;
};

// Tensors of a launch: as many as 4 KiB of arguments hold.  (A launch more costs 5 us and the end of another one: the 161 tensors
// of a ResNet-50 in launches of up to 86 142 us, 80 146, 48 151.)  The numbers of their updates are few as a rule, and
// are kept apart.
constexpr int ADAM_SHORT = 8, ADAM_SETS = 8;
template <int BITS> constexpr int adam_long() { return BITS == 32 ? 86 : 64; }
template <int BITS, int N>
struct AdamList {
  AdamTensor<BITS> d[N];
  int first[N + 1];                       // workgroup of each
  int n, index;                           // of the launch's first tensor in the call
  const AdamScalars* scalars;             // on the device, one for each tensor: in the place of the sets
  AdamScalars sets[ADAM_SETS];
  unsigned char set[N];
};
static_assert(sizeof(AdamList<8, adam_long<8>()>) + sizeof(AdamRates) <= 4096, "kernel arguments");
static_assert(sizeof(AdamList<32, adam_long<32>()>) + sizeof(AdamRates) <= 4096, "kernel arguments");

// ---- random numbers --------------------------------------------------------

// One 32-bit word a tensor and update, one for every 8 elements by mixing their index into it, and one an element by a
// step of Marsaglia's xorshift (13, 17, 5) each.  The factors are 2^32 over the golden ratio and 2^31.5, made odd.
__host__ __device__ inline unsigned mix(unsigned x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0xB504F333u;
  return x ^ (x >> 16);
}
__host__ __device__ inline unsigned update_key(unsigned seed, unsigned step) { return mix(mix(seed) + step); }
__device__ __forceinline__ unsigned next_word(unsigned x) {
  x ^= x << 13;
  x ^= x >> 17;
  return x ^ (x << 5);
}

// 8 and 16 bytes of elements of 1, 2 and 4 bytes that may begin anywhere (as parts of a buffer do): one access all the same
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned loose2 __attribute__((ext_vector_type(2), aligned(1), may_alias));
typedef unsigned loose4 __attribute__((ext_vector_type(4), aligned(2), may_alias));

// ---- 8-bit states ----------------------------------------------------------

// x to one of its two neighbours, four numbers into a word: the instructions add the upper 20 (e4m3) or 21 bits (e5m2) of
// a random word below the last bit that is kept, also among the numbers below the type's normal ones (all 2^16
// random numbers compared with that formula).  Of those the upper 16 are random and the others 0, so that a number some
// last bits above the largest one, as the reciprocal of the scale may make it, stays that.
template <int BYTE>
__device__ __forceinline__ int encode_m(float x, unsigned word, int into) {
  return __builtin_amdgcn_cvt_sr_fp8_f32(x, word & 0xffff0000u, into, BYTE);
}
template <int BYTE>
__device__ __forceinline__ int encode_v(float x, unsigned word, int into) {
  return __builtin_amdgcn_cvt_sr_bf8_f32(x, word << 16, into, BYTE);
}
template <int BYTE>
__device__ __forceinline__ void encode(const float (&m)[UNIT], const float (&v)[UNIT], int k, unsigned& word, int& mq, int& vq) {
  mq = encode_m<BYTE>(m[4 * k + BYTE], word, mq);
  vq = encode_v<BYTE>(v[4 * k + BYTE], word, vq);
  word = next_word(word);
}

__device__ __forceinline__ void decode_m(u2 q, float (&x)[UNIT]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int w = (int)q[k];
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[4 * k] = low[0], x[4 * k + 1] = low[1], x[4 * k + 2] = high[0], x[4 * k + 3] = high[1];
  }
}
__device__ __forceinline__ void decode_v(u2 q, float (&x)[UNIT]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int w = (int)q[k];
    const auto low = __builtin_amdgcn_cvt_pk_f32_bf8(w, false), high = __builtin_amdgcn_cvt_pk_f32_bf8(w, true);
    x[4 * k] = low[0], x[4 * k + 1] = low[1], x[4 * k + 2] = high[0], x[4 * k + 3] = high[1];
  }
}

// Largest of the 16 threads that hold a block, a row of the wave: rotated in registers
static_assert(LANES == 16, "a row of a wave");
__device__ __forceinline__ unsigned block_max(unsigned x) {
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true));
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, true));
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, true));
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, true));
}

// Scale and its reciprocal from the bits of the block's largest number (products with reciprocals that are rounded:
// three roundings of the scale's are no more than a thousandth of an 8-bit step)
__device__ __forceinline__ void block_scale(unsigned top_bits, float largest, float& scale, float& inverse) {
  const float top = __uint_as_float(top_bits);
  const bool some = top >= LEAST_TOP;
  scale = some ? top * (1.f / largest) : 0.f;
  inverse = some ? 1.f / top * largest : 0.f;
}

// ---- the update --------------------------------------------------------------

// ONCE: past the caches.  States in 8 bits of calls that access more than the last cache holds: 244 million bfloat16
// parameters 435 us without that, 390 with it.  (In 32 bits it costs: on one card 958 without and 977 with it.)
constexpr double LAST_CACHE = 256. * (1 << 20);
template <bool ONCE>
__device__ __forceinline__ u4 load16(const void* p) {
  return ONCE ? __builtin_nontemporal_load((const loose4*)p) : *(const loose4*)p;
}
template <bool ONCE>
__device__ __forceinline__ u2 load8(const void* p) {
  return ONCE ? __builtin_nontemporal_load((const loose2*)p) : *(const loose2*)p;
}
template <bool ONCE>
__device__ __forceinline__ void store16(void* p, u4 w) {
  if (ONCE) __builtin_nontemporal_store(w, (loose4*)p);
  else *(loose4*)p = w;
}
template <bool ONCE>
__device__ __forceinline__ void store8(void* p, u2 w) {
  if (ONCE) __builtin_nontemporal_store(w, (loose2*)p);
  else *(loose2*)p = w;
}
template <bool ONCE, class V>
__device__ __forceinline__ void load_unit(const V* p, float (&v)[UNIT]) {
  constexpr int E = 16 / sizeof(V);
#pragma unroll
  for (int i = 0; i < UNIT; i += E) {
    const Pack<V, E> a = __builtin_bit_cast(Pack<V, E>, load16<ONCE>(p + i));
#pragma unroll
    for (int e = 0; e < E; ++e) v[i + e] = Element<V>::get(a.v[e]);
  }
}
template <bool ONCE, class V>
__device__ __forceinline__ void store_unit(V* p, const float (&v)[UNIT]) {
  constexpr int E = 16 / sizeof(V);
#pragma unroll
  for (int i = 0; i < UNIT; i += E) {
    Pack<V, E> a;
#pragma unroll
    for (int e = 0; e < E; ++e) a.v[e] = Element<V>::put(v[i + e]);
    store16<ONCE>(p + i, __builtin_bit_cast(u4, a));
  }
}

// FAST: root and reciprocal by the instructions alone, 2^-23 off, of numbers that are not below 2^-126 where it matters
// (with states in 8 bits eps is at least 1e-12).
template <bool FAST>
__device__ __forceinline__ void update(const AdamRates& r, const AdamScalars& s, float g, float& p, float& m, float& v) {
  {
#pragma clang fp contract(off)
    m = r.b1 * m + r.c1 * g;
    v = r.b2 * v + r.c2 * g * g;
  }
  if (FAST) p = fmaf(-m, __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(v), s.root, s.eps)), p * s.keep);
  else p = fmaf(p, s.keep, -(m / fmaf(sqrtf(v), s.root, s.eps)));
}

// Elements i ... i + 7 of a tensor, or the `have` of them that there are
template <bool ONCE, class V>
__device__ __forceinline__ void update_unit(const AdamTensor<32>& t, const AdamScalars& s, const AdamRates& r, long i, int have) {
  const bool whole = have == UNIT;
  V* const pp = (V*)t.p + i;
  const V* const gp = (const V*)t.g + i;
  float *const mp = (float*)t.m + i, *const vp = (float*)t.v + i;
  if (whole) {
    float p[UNIT], g[UNIT], m[UNIT], v[UNIT];
    load_unit<ONCE>(gp, g);
    load_unit<ONCE>(pp, p);
    load_unit<ONCE>(mp, m);
    load_unit<ONCE>(vp, v);
#pragma unroll
    for (int e = 0; e < UNIT; ++e) update<false>(r, s, g[e], p[e], m[e], v[e]);
    store_unit<ONCE>(pp, p);
    store_unit<ONCE>(mp, m);
    store_unit<ONCE>(vp, v);
  } else {
    for (int e = 0; e < have; ++e) {
      float p = Element<V>::get(pp[e]), m = mp[e], v = vp[e];
      update<false>(r, s, Element<V>::get(gp[e]), p, m, v);
      pp[e] = Element<V>::put(p);
      mp[e] = m;
      vp[e] = v;
    }
  }
}

template <bool ONCE, class V>
__device__ __forceinline__ void update_unit(const AdamTensor<8>& t, const AdamScalars& s, const AdamRates& r, long i, int have) {
  const bool whole = have == UNIT;
  V* const pp = (V*)t.p + i;
  const V* const gp = (const V*)t.g + i;
  unsigned char *const mp = (unsigned char*)t.m + i, *const vp = (unsigned char*)t.v + i;
  float p[UNIT], g[UNIT], m[UNIT], v[UNIT];
  u2 mq = {0, 0}, vq = {0, 0};
  float m_scale = 0.f, v_scale = 0.f;
  if (have > 0) {
    m_scale = t.m_scale[i / BLOCK];
    v_scale = t.v_scale[i / BLOCK];
  }
  if (whole) {
    load_unit<ONCE>(gp, g);
    load_unit<ONCE>(pp, p);
    mq = load8<ONCE>(mp);
    vq = load8<ONCE>(vp);
  } else {
#pragma unroll
    for (int e = 0; e < UNIT; ++e) {
      p[e] = g[e] = 0.f;
      if (e < have) {
        p[e] = Element<V>::get(pp[e]);
        g[e] = Element<V>::get(gp[e]);
        mq[e / 4] |= (unsigned)mp[e] << (8 * (e & 3));
        vq[e / 4] |= (unsigned)vp[e] << (8 * (e & 3));
      }
    }
  }
  decode_m(mq, m);
  decode_v(vq, v);
  unsigned top_m = 0, top_v = 0;
#pragma unroll
  for (int e = 0; e < UNIT; ++e) {
    m[e] *= m_scale;
    v[e] *= v_scale;
    update<true>(r, s, g[e], p[e], m[e], v[e]);
    top_m = max(top_m, __float_as_uint(m[e]) & 0x7fffffffu);
    top_v = max(top_v, __float_as_uint(v[e]));
  }
  if (whole) {
    store_unit<ONCE>(pp, p);
  } else {
#pragma unroll
    for (int e = 0; e < UNIT; ++e)
      if (e < have) pp[e] = Element<V>::put(p[e]);
  }
  top_m = block_max(top_m);
  top_v = block_max(top_v);
  // (numbers that are not finite stay by themselves: the block's scale is that of the others)
  const bool odd = top_m >= INFINITE || top_v >= INFINITE;
  if (odd) {
    top_m = top_v = 0;
#pragma unroll
    for (int e = 0; e < UNIT; ++e) {
      const unsigned bm = __float_as_uint(m[e]) & 0x7fffffffu, bv = __float_as_uint(v[e]);
      if (bm < INFINITE) top_m = max(top_m, bm);
      if (bv < INFINITE) top_v = max(top_v, bv);
    }
    top_m = block_max(top_m);
    top_v = block_max(top_v);
  }
  float m_inverse, v_inverse;
  block_scale(top_m, LARGEST_M, m_scale, m_inverse);
  block_scale(top_v, LARGEST_V, v_scale, v_inverse);
  const float least = v_inverse > 0.f ? LEAST_V : 0.f;
  if (odd && v_scale == 0.f) {                       // (an infinite v stays one beside zeros)
    v_scale = 1.f;
    v_inverse = 0x1p-126f;
  }
  float scaled[UNIT], lowest = LARGEST_V;
#pragma unroll
  for (int e = 0; e < UNIT; ++e) {
    m[e] *= m_inverse;
    scaled[e] = v[e] * v_inverse;
    lowest = fminf(lowest, scaled[e]);
  }
  // a v above 0 is at least the smallest number (they are rarely below it: few threads come here)
  if (lowest < least) {
#pragma unroll
    for (int e = 0; e < UNIT; ++e)
      if (v[e] > 0.f) scaled[e] = fmaxf(scaled[e], least);
  }
  unsigned word = mix(s.key + (unsigned)(i / UNIT));
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int mw = 0, vw = 0;
    encode<0>(m, scaled, k, word, mw, vw);
    encode<1>(m, scaled, k, word, mw, vw);
    encode<2>(m, scaled, k, word, mw, vw);
    encode<3>(m, scaled, k, word, mw, vw);
    mq[k] = (unsigned)mw;
    vq[k] = (unsigned)vw;
  }
  if (whole) {
    store8<ONCE>(mp, mq);
    store8<ONCE>(vp, vq);
  } else {
#pragma unroll
    for (int e = 0; e < UNIT; ++e)
      if (e < have) {
        mp[e] = (unsigned char)(mq[e / 4] >> (8 * (e & 3)));
        vp[e] = (unsigned char)(vq[e / 4] >> (8 * (e & 3)));
      }
  }
  if (have > 0 && i % BLOCK == 0) {
    t.m_scale[i / BLOCK] = m_scale;
    t.v_scale[i / BLOCK] = v_scale;
  }
}

template <class V, int BITS, int N, bool ONCE>
__global__ __launch_bounds__(ADAM_THREADS) void adamw_kernel(const AdamList<BITS, N> list, const AdamRates r) {
  int j = 0, end = list.n;
  while (end - j > 1) {
    const int mid = (j + end) >> 1;
    if (list.first[mid] <= (int)blockIdx.x) j = mid; else end = mid;
  }
  const AdamTensor<BITS> t = list.d[j];
  AdamScalars s = list.scalars ? list.scalars[j] : list.sets[list.set[j]];
  if (BITS == 8) s.key = mix(s.key + (unsigned)(list.index + j));
  const long i = (long)((int)blockIdx.x - list.first[j]) * ADAM_GROUP + (long)threadIdx.x * UNIT;
  const int have = (int)min(max(t.n - i, 0L), (long)UNIT);
  // (in 8 bits a block's threads go on together)
  if (BITS == 32 ? have > 0 : i / BLOCK * BLOCK < t.n) update_unit<ONCE, V>(t, s, r, i, have);
}

// ---- numbers of the update on the device -----------------------------------------

// (an update by less than LEAST_SIZE is none: the quotients above would leave float32.  eps' is infinite then, and root 1: 0
// would make a number that is none of it where v has overflowed)
constexpr double LEAST_SIZE = 1e-30;
__host__ __device__ inline AdamScalars scalars_of(double t, unsigned step, double lr, double b1, double b2, double eps,
                                                  double decay, unsigned seed) {
  AdamScalars s;
  const double size = lr / (b1 > 0. ? -expm1(t * log(b1)) : 1.);
  const bool some = !(fabs(size) < LEAST_SIZE);
  s.keep = (float)(1. - lr * decay);
  s.root = some ? (float)(1. / (size * sqrt(b2 > 0. ? -expm1(t * log(b2)) : 1.))) : 1.f;
  s.eps = some ? (float)(eps / size) : INFINITY;
  s.key = update_key(seed, step);
  return s;
}

struct AdamCounters {
  int* step[256];
  int n;
};
__global__ __launch_bounds__(256) void adamw_scalars_kernel(const AdamCounters c, const float* lr_on_device, double lr, double b1,
                                                            double b2, double eps, double decay, unsigned seed, int first,
                                                            AdamScalars* out) {
  const int i = threadIdx.x;
  if (i >= c.n) return;
  const int t = *c.step[i] + 1;
  *c.step[i] = t;
  if (lr_on_device) lr = (double)*lr_on_device;
  out[first + i] = scalars_of((double)t, (unsigned)t, lr, b1, b2, eps, decay, seed);
}

long groups_of(int64_t elements) { return ((long)elements + ADAM_GROUP - 1) / ADAM_GROUP; }

struct AdamCall {
  int count;
  const int64_t *numel, *steps;
  void *const *params, *const *m, *const *v;
  const void* const* grads;
  float *const *m_scales, *const *v_scales;
  const AdamScalars* scalars;             // on the device, where there are no steps
  double lr, beta1, beta2, eps, decay;
  unsigned seed;
  AdamRates rates;
  bool once;
};

// The tensors from `first` on, as many as a launch takes; how many those are.
template <class V, int BITS, int N>
int launch_adamw(const AdamCall& c, int first, hipStream_t stream) {
  AdamList<BITS, N> list;
  list.n = list.first[0] = 0;
  list.index = first;
  list.scalars = c.scalars ? c.scalars + first : nullptr;
  int sets = 0;
  int64_t step[ADAM_SETS];
  for (int k = 0; k < N && first + k < c.count; ++k) {
    const int i = first + k;
    const long groups = groups_of(c.numel[i]);
    if (k > 0 && list.first[k] + groups > ADAM_MOST_GROUPS) break;
    if (c.steps) {
      int at = 0;
      while (at < sets && step[at] != c.steps[i]) ++at;
      if (at == ADAM_SETS) break;
      if (at == sets) {
        step[sets] = c.steps[i];
        list.sets[sets++] = scalars_of((double)c.steps[i], (unsigned)c.steps[i], c.lr, c.beta1, c.beta2, c.eps, c.decay, c.seed);
      }
      list.set[k] = (unsigned char)at;
    }
    AdamTensor<BITS>& t = list.d[k];
    t.p = c.params[i];
    t.g = c.grads[i];
    t.m = c.m[i];
    t.v = c.v[i];
    if constexpr (BITS == 8) {
      t.m_scale = c.m_scales[i];
      t.v_scale = c.v_scales[i];
    }
    t.n = (long)c.numel[i];
    list.first[k + 1] = list.first[k] + (int)groups;
    ++list.n;
  }
  const dim3 grid((unsigned)list.first[list.n]), block(ADAM_THREADS);
  if (grid.x > 0) {
    if (BITS == 8 && c.once) hipLaunchKernelGGL((adamw_kernel<V, BITS, N, BITS == 8>), grid, block, 0, stream, list, c.rates);
    else hipLaunchKernelGGL((adamw_kernel<V, BITS, N, false>), grid, block, 0, stream, list, c.rates);
  }
  return list.n;
}

template <class V, int BITS>
void launch_all(const AdamCall& c, hipStream_t stream) {
  for (int first = 0; first < c.count;)
    first += c.count - first <= ADAM_SHORT ? launch_adamw<V, BITS, ADAM_SHORT>(c, first, stream)
                                           : launch_adamw<V, BITS, adam_long<BITS>()>(c, first, stream);
}

}  // namespace
}  // namespace kfac

using namespace kfac;

extern "C" {

size_t kfac_adamw_workspace_bytes(int count, int counters_on_device) {
  return count > 0 && counters_on_device ? (size_t)count * sizeof(AdamScalars) : 0;
}

int kfac_adamw_batched(int count, const int64_t* numel, int type, int state_bits, void* const* params, const void* const* grads,
                       void* const* m, void* const* v, float* const* m_scales, float* const* v_scales, const int64_t* steps,
                       int* const* counters, double lr, const float* lr_on_device, double beta1, double beta2, double eps,
                       double weight_decay, unsigned seed, void* workspace, size_t workspace_bytes, void* stream) {
  if (count == 0) return KFAC_OK;
  if (count < 0 || type < TYPE_F32 || type > TYPE_F16 || (state_bits != 8 && state_bits != 32) || !numel || !params || !grads ||
      !m || !v || (state_bits == 8 && (!m_scales || !v_scales)) || !steps == !counters || (lr_on_device && !counters))
    return KFAC_ERR_ARG;
  if (!(lr >= 0.) || !(beta1 >= 0. && beta1 < 1.) || !(beta2 >= 0. && beta2 < 1.) || !(eps >= (state_bits == 8 ? 1e-12 : 0.)) ||
      !(weight_decay >= 0.))
    return KFAC_ERR_ARG;
  constexpr int64_t most = ADAM_MOST_GROUPS * ADAM_GROUP;
  bool some = counters != nullptr;
  double elements = 0.;
  for (int i = 0; i < count; ++i) {
    some = some || numel[i] > 0;
    elements += (double)numel[i];
    if (numel[i] < 0 || numel[i] > most || (steps && steps[i] < 1)) return KFAC_ERR_ARG;
    if (numel[i] > 0 && (!params[i] || !grads[i] || !m[i] || !v[i] || (state_bits == 8 && (!m_scales[i] || !v_scales[i]))))
      return KFAC_ERR_ARG;
    if (counters && !counters[i]) return KFAC_ERR_ARG;
  }
  if (!some) return KFAC_OK;
  if (counters && (!workspace || workspace_bytes < kfac_adamw_workspace_bytes(count, 1))) return KFAC_ERR_WORKSPACE;
  const hipStream_t s = (hipStream_t)stream;
  AdamScalars* const on_device = counters ? (AdamScalars*)workspace : nullptr;
  for (int first = 0; counters && first < count; first += 256) {
    AdamCounters c;
    c.n = std::min(256, count - first);
    for (int k = 0; k < c.n; ++k) c.step[k] = counters[first + k];
    hipLaunchKernelGGL(adamw_scalars_kernel, dim3(1), dim3(256), 0, s, c, lr_on_device, lr, beta1, beta2, eps, weight_decay, seed, first,
                       on_device);
  }
  const AdamCall c{count, numel, steps, params, m, v, grads, m_scales, v_scales, on_device, lr, beta1, beta2, eps, weight_decay, seed,
                   {(float)beta1, (float)(1. - beta1), (float)beta2, (float)(1. - beta2)},
                   elements * (3 * type_size(type) + 4) > LAST_CACHE};
  const bool wide = state_bits == 32;
  if (type == TYPE_F32) wide ? launch_all<float, 32>(c, s) : launch_all<float, 8>(c, s);
  else if (type == TYPE_BF16) wide ? launch_all<__hip_bfloat16, 32>(c, s) : launch_all<__hip_bfloat16, 8>(c, s);
  else wide ? launch_all<_Float16, 32>(c, s) : launch_all<_Float16, 8>(c, s);
  return launch_status();
}

}  // extern "C"
