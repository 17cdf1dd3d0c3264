// AdamW: one update of a list of tensors, with states in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2
//   p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
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
#include <cmath>

#include "common.h"
#include "element_types.h"

namespace kfac {
namespace {

constexpr int ADAM_THREADS = 256, UNIT = 8, BLOCK = 128, LANES = BLOCK / UNIT;
constexpr int ADAM_ROUND = ADAM_THREADS * UNIT;      // elements that a workgroup takes at a time
constexpr int ADAM_ROUNDS = 2;                       // ... how many times
constexpr long ADAM_GROUP = (long)ADAM_ROUND * ADAM_ROUNDS;
constexpr long ADAM_MOST_GROUPS = (1L << 32) / ADAM_THREADS - 1;      // a launch has fewer than 2^32 threads
constexpr float LARGEST_M = 448.f, LARGEST_V = 57344.f, LEAST_V = 0x1p-16f;
// A block whose largest number is below this is kept as zeros (its reciprocal scale would overflow).
constexpr float LEAST_TOP = 0x1p-100f;
constexpr unsigned INFINITE = 0x7f800000u;

// What depends on the number of the update
struct AdamScalars {
  float keep, size, root;                 // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  unsigned key;                           // of the tensor's random numbers
};
struct AdamRates {
  float b1, c1, b2, c2, eps;              // c: 1 - b
};

template <int BITS> struct AdamTensor;
template <> struct AdamTensor<32> {
  void *p, *m, *v;
  const void* g;
  long n;
  AdamScalars s;
};
template <> struct AdamTensor<8> {
  void *p, *m, *v;
  const void* g;
  float *m_scale, *v_scale;
  long n;
  AdamScalars s;
};

constexpr int ADAM_SHORT = 8, ADAM_LONG = 48;
template <int BITS, int N>
struct AdamList {
  AdamTensor<BITS> d[N];
  int first[N + 1];                       // workgroup of each
  int n;
  const AdamScalars* scalars;             // on the device: in the place of those above
};
static_assert(sizeof(AdamList<8, ADAM_LONG>) + sizeof(AdamRates) <= 4096, "kernel arguments");

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
__host__ __device__ inline unsigned tensor_key(unsigned seed, unsigned step, unsigned index) {
  return mix(mix(mix(seed) + step) + index);
}
__device__ __forceinline__ unsigned next_word(unsigned x) {
  x ^= x << 13;
  x ^= x >> 17;
  return x ^ (x << 5);
}

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

__device__ __forceinline__ void decode_m(uint2 q, float (&x)[UNIT]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int w = (int)(k ? q.y : q.x);
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[4 * k] = low[0], x[4 * k + 1] = low[1], x[4 * k + 2] = high[0], x[4 * k + 3] = high[1];
  }
}
__device__ __forceinline__ void decode_v(uint2 q, float (&x)[UNIT]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int w = (int)(k ? q.y : q.x);
    const auto low = __builtin_amdgcn_cvt_pk_f32_bf8(w, false), high = __builtin_amdgcn_cvt_pk_f32_bf8(w, true);
    x[4 * k] = low[0], x[4 * k + 1] = low[1], x[4 * k + 2] = high[0], x[4 * k + 3] = high[1];
  }
}

// Largest of the 16 threads that hold a block
__device__ __forceinline__ unsigned block_max(unsigned x) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) x = max(x, (unsigned)__shfl_xor((int)x, o));
  return x;
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

template <class V, int N>
__device__ __forceinline__ void load_all(const V* p, float (&v)[N]) {
  constexpr int E = 16 / sizeof(V) < N ? 16 / sizeof(V) : N;
#pragma unroll
  for (int i = 0; i < N; i += E) {
    const Pack<V, E> a = *(const Pack<V, E>*)(p + i);
#pragma unroll
    for (int e = 0; e < E; ++e) v[i + e] = Element<V>::get(a.v[e]);
  }
}
template <class V, int N>
__device__ __forceinline__ void store_all(V* p, const float (&v)[N]) {
  constexpr int E = 16 / sizeof(V) < N ? 16 / sizeof(V) : N;
#pragma unroll
  for (int i = 0; i < N; i += E) {
    Pack<V, E> a;
#pragma unroll
    for (int e = 0; e < E; ++e) a.v[e] = Element<V>::put(v[i + e]);
    *(Pack<V, E>*)(p + i) = a;
  }
}

// (m and v without fused products: an 8-bit state that is off by a bit before it is rounded may become another
// number, and this is the sequence that the formula has in float32 operations)
// FAST: root and reciprocal by the instructions alone, 2^-23 off, of numbers that are not below 2^-126 where it matters
// (with states in 8 bits eps is at least 1e-12).
template <bool FAST>
__device__ __forceinline__ void update(const AdamRates& r, const AdamScalars& s, float g, float& p, float& m, float& v) {
  {
#pragma clang fp contract(off)
    m = r.b1 * m + r.c1 * g;
    v = r.b2 * v + r.c2 * g * g;
  }
  if (FAST) p = fmaf(p, s.keep, -s.size * m * __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(v), s.root, r.eps)));
  else p = fmaf(p, s.keep, -s.size * (m / fmaf(sqrtf(v), s.root, r.eps)));
}

// Elements i ... i + 7 of a tensor, `have` of them (8 where all streams can be accessed 16 bytes at a time: whole).
template <class V>
__device__ __forceinline__ void update_unit(const AdamTensor<32>& t, const AdamScalars& s, const AdamRates& r, long i, int have,
                                            bool whole) {
  V* const pp = (V*)t.p + i;
  const V* const gp = (const V*)t.g + i;
  float *const mp = (float*)t.m + i, *const vp = (float*)t.v + i;
  if (whole) {
    float p[UNIT], g[UNIT], m[UNIT], v[UNIT];
    load_all<V, UNIT>(gp, g);
    load_all<V, UNIT>(pp, p);
    load_all<float, UNIT>(mp, m);
    load_all<float, UNIT>(vp, v);
#pragma unroll
    for (int e = 0; e < UNIT; ++e) update<false>(r, s, g[e], p[e], m[e], v[e]);
    store_all<V, UNIT>(pp, p);
    store_all<float, UNIT>(mp, m);
    store_all<float, UNIT>(vp, v);
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

template <class V>
__device__ __forceinline__ void update_unit(const AdamTensor<8>& t, const AdamScalars& s, const AdamRates& r, long i, int have,
                                            bool whole) {
  V* const pp = (V*)t.p + i;
  const V* const gp = (const V*)t.g + i;
  unsigned char *const mp = (unsigned char*)t.m + i, *const vp = (unsigned char*)t.v + i;
  float p[UNIT], g[UNIT], m[UNIT], v[UNIT];
  uint2 mq = make_uint2(0, 0), vq = make_uint2(0, 0);
  float m_scale = 0.f, v_scale = 0.f;
  if (have > 0) {
    m_scale = t.m_scale[i / BLOCK];
    v_scale = t.v_scale[i / BLOCK];
  }
  if (whole) {
    load_all<V, UNIT>(gp, g);
    load_all<V, UNIT>(pp, p);
    mq = *(const uint2*)mp;
    vq = *(const uint2*)vp;
  } else {
#pragma unroll
    for (int e = 0; e < UNIT; ++e) {
      p[e] = g[e] = 0.f;
      if (e < have) {
        p[e] = Element<V>::get(pp[e]);
        g[e] = Element<V>::get(gp[e]);
        (e < 4 ? mq.x : mq.y) |= (unsigned)mp[e] << (8 * (e & 3));
        (e < 4 ? vq.x : vq.y) |= (unsigned)vp[e] << (8 * (e & 3));
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
    store_all<V, UNIT>(pp, p);
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
  // a v above 0 is at least the smallest number
  const float least = v_inverse > 0.f ? LEAST_V : 0.f;
  if (odd && v_scale == 0.f) {                       // (an infinite v stays one beside zeros)
    v_scale = 1.f;
    v_inverse = 0x1p-126f;
  }
#pragma unroll
  for (int e = 0; e < UNIT; ++e) {
    m[e] *= m_inverse;
    v[e] = v[e] > 0.f ? fmaxf(v[e] * v_inverse, least) : v[e];
  }
  unsigned word = mix(s.key + (unsigned)(i / UNIT));
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int mw = 0, vw = 0;
    encode<0>(m, v, k, word, mw, vw);
    encode<1>(m, v, k, word, mw, vw);
    encode<2>(m, v, k, word, mw, vw);
    encode<3>(m, v, k, word, mw, vw);
    (k ? mq.y : mq.x) = (unsigned)mw;
    (k ? vq.y : vq.x) = (unsigned)vw;
  }
  if (whole) {
    *(uint2*)mp = mq;
    *(uint2*)vp = vq;
  } else {
#pragma unroll
    for (int e = 0; e < UNIT; ++e)
      if (e < have) {
        mp[e] = (unsigned char)((e < 4 ? mq.x : mq.y) >> (8 * (e & 3)));
        vp[e] = (unsigned char)((e < 4 ? vq.x : vq.y) >> (8 * (e & 3)));
      }
  }
  if (have > 0 && i % BLOCK == 0) {
    t.m_scale[i / BLOCK] = m_scale;
    t.v_scale[i / BLOCK] = v_scale;
  }
}

template <int BITS>
__device__ __forceinline__ bool accesses_whole(const AdamTensor<BITS>& t) {
  const uintptr_t wide = (uintptr_t)t.p | (uintptr_t)t.g, states = (uintptr_t)t.m | (uintptr_t)t.v;
  return ((wide | (BITS == 32 ? states : 0)) & 15) == 0 && (states & 7) == 0;
}

template <class V, int BITS, int N>
__global__ __launch_bounds__(ADAM_THREADS) void adamw_kernel(const AdamList<BITS, N> list, const AdamRates r) {
  int j = 0, end = list.n;
  while (end - j > 1) {
    const int mid = (j + end) >> 1;
    if (list.first[mid] <= (int)blockIdx.x) j = mid; else end = mid;
  }
  const AdamTensor<BITS> t = list.d[j];
  const AdamScalars s = list.scalars ? list.scalars[j] : t.s;
  const bool whole = accesses_whole<BITS>(t);
  const long from = (long)((int)blockIdx.x - list.first[j]) * ADAM_GROUP;
#pragma unroll
  for (int k = 0; k < ADAM_ROUNDS; ++k) {
    const long i = from + k * ADAM_ROUND + (long)threadIdx.x * UNIT;
    const int have = (int)min(max(t.n - i, 0L), (long)UNIT);
    // (in 8 bits a block's threads go on together)
    if (BITS == 32 ? have > 0 : i / BLOCK * BLOCK < t.n) update_unit<V>(t, s, r, i, have, whole && have == UNIT);
  }
}

// ---- numbers of the update on the device -----------------------------------------

struct AdamCounters {
  int* step[256];
  int n;
};
__global__ __launch_bounds__(256) void adamw_scalars_kernel(const AdamCounters c, const float* lr_on_device, double lr, double b1,
                                                            double b2, double decay, unsigned seed, int first,
                                                            AdamScalars* out) {
  const int i = threadIdx.x;
  if (i >= c.n) return;
  const int t = *c.step[i] + 1;
  *c.step[i] = t;
  if (lr_on_device) lr = (double)*lr_on_device;
  AdamScalars s;
  s.keep = (float)(1. - lr * decay);
  s.size = (float)(lr / (b1 > 0. ? -expm1((double)t * log(b1)) : 1.));
  s.root = (float)(1. / sqrt(b2 > 0. ? -expm1((double)t * log(b2)) : 1.));
  s.key = tensor_key(seed, (unsigned)t, (unsigned)(first + i));
  out[first + i] = s;
}

long groups_of(int64_t elements) { return ((long)elements + ADAM_GROUP - 1) / ADAM_GROUP; }

struct AdamCall {
  int count, type;
  const int64_t* numel;
  void *const *params, *const *m, *const *v;
  const void* const* grads;
  float *const *m_scales, *const *v_scales;
  AdamRates rates;
};

template <class V, int BITS, int N>
void launch_adamw(const AdamCall& c, int first, int count, const AdamScalars* scalars, const AdamScalars* on_device,
                  hipStream_t stream) {
  AdamList<BITS, N> list;
  list.n = count;
  list.first[0] = 0;
  list.scalars = on_device ? on_device + first : nullptr;
  for (int k = 0; k < count; ++k) {
    const int i = first + k;
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
    t.s = on_device ? AdamScalars{} : scalars[k];
    list.first[k + 1] = list.first[k] + (int)groups_of(t.n);
  }
  if (list.first[count] > 0)
    hipLaunchKernelGGL((adamw_kernel<V, BITS, N>), dim3((unsigned)list.first[count]), dim3(ADAM_THREADS), 0, stream, list, c.rates);
}

template <int BITS, int N>
void launch_adamw(const AdamCall& c, int first, int count, const AdamScalars* scalars, const AdamScalars* on_device,
                  hipStream_t stream) {
  if (c.type == TYPE_F32) launch_adamw<float, BITS, N>(c, first, count, scalars, on_device, stream);
  else if (c.type == TYPE_BF16) launch_adamw<__hip_bfloat16, BITS, N>(c, first, count, scalars, on_device, stream);
  else launch_adamw<_Float16, BITS, N>(c, first, count, scalars, on_device, stream);
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
  for (int i = 0; i < count; ++i) {
    some = some || numel[i] > 0;
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
    hipLaunchKernelGGL(adamw_scalars_kernel, dim3(1), dim3(256), 0, s, c, lr_on_device, lr, beta1, beta2, weight_decay, seed, first,
                       on_device);
  }
  const AdamCall c{count, type, numel, params, m, v, grads, m_scales, v_scales,
                   {(float)beta1, (float)(1. - beta1), (float)beta2, (float)(1. - beta2), (float)eps}};
  for (int first = 0, n; first < count; first += n) {
    long groups = groups_of(numel[first]);
    for (n = 1; n < ADAM_LONG && first + n < count; ++n)
      if ((groups += groups_of(numel[first + n])) > ADAM_MOST_GROUPS) break;
    AdamScalars scalars[ADAM_LONG];
    for (int k = 0; steps && k < n; ++k) {
      const int64_t t = steps[first + k];
      if (k > 0 && t == steps[first + k - 1]) {
        scalars[k] = scalars[k - 1];
      } else {
        scalars[k].keep = (float)(1. - lr * weight_decay);
        scalars[k].size = (float)(lr / (beta1 > 0. ? -std::expm1((double)t * std::log(beta1)) : 1.));
        scalars[k].root = (float)(1. / std::sqrt(beta2 > 0. ? -std::expm1((double)t * std::log(beta2)) : 1.));
      }
      scalars[k].key = tensor_key(seed, (unsigned)t, (unsigned)(first + k));
    }
    const bool few = n <= ADAM_SHORT;
    if (state_bits == 32) few ? launch_adamw<32, ADAM_SHORT>(c, first, n, scalars, on_device, s)
                              : launch_adamw<32, ADAM_LONG>(c, first, n, scalars, on_device, s);
    else few ? launch_adamw<8, ADAM_SHORT>(c, first, n, scalars, on_device, s)
             : launch_adamw<8, ADAM_LONG>(c, first, n, scalars, on_device, s);
  }
  return launch_status();
}

}  // extern "C"
