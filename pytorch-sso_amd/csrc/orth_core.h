// Products of the Newton-Schulz iteration on the fp16 matrix cores (gfx950, wave64).
//
// Every operand of the iteration is bounded: X, A = X X^T and B = aI + bA + cAA have entries of at
// most a few units once X is normalised.  Times 2^13 they are kept as fp16 numbers: in two parts,
// x = h + l with h = fp16(x), l = fp16(x - h), 22 bits and the sign of l, or h alone.  A product of
// two such numbers is
//     x y = h h' + h l' + l h' + [l l']
// where the bracket is at most 2^-24 of |x y|, as much as one float32 rounding, and is left out:
// three v_mfma_f32_16x16x32_f16 with exact products and float32 sums, where three bf16 parts, which
// hold any float32, take six.
//
// One workgroup of 256 threads (4 waves, 2 x 2) computes a T x T tile D[m][n] = sum_k P[m][k] Q[n][k].
// Operands go from memory to LDS directly (16 bytes a lane), 32 reduction steps a stage, two stages.
//   rows of an operand with k along them ("KC"): 64 bytes a row; the 16-byte groups of a row are
//     exchanged by (row / 4) % 4, so that the 16 rows that lanes read at once lie in different banks;
//   an operand with k down its rows ("KM"): T columns a row, read by the transposing LDS loads, 16
//     columns (32 bytes) of 4 rows at a time; the 32-byte groups of a row are exchanged by its number.
#pragma once
#include "common.h"

namespace kfac {

typedef _Float16 half_t;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __fp16 h4s __attribute__((ext_vector_type(4)));
typedef __fp16 h8s __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr float ORTH_SCALE = 8192.f;             // 2^13
constexpr int ORTH_THREADS = 256, ORTH_BK = 32;

template <int T>
struct OrthCfg {
  static constexpr int PLANE = T * ORTH_BK * 2;         // bytes of a stage of one plane
  static constexpr int LOADS = PLANE / 4096;            // 16-byte loads of a lane for it
  static constexpr int NF = T / 32;                     // 16-row fragments of a wave's half
  template <bool SPLIT>
  static constexpr int stage() { return (SPLIT ? 4 : 2) * PLANE; }
  template <bool SPLIT>
  static constexpr int lds() { return 2 * stage<SPLIT>(); }
};

// 64 lanes times 16 bytes from `base` + voff to LDS at `dst` (lane i at dst + 16 i).
__device__ __forceinline__ void lds_load(const char* base, unsigned voff, lds_char* dst) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(base + voff),
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
// This wave's loads into LDS have landed and its reads are done, and so it is with all others'.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// exchange of the 32-byte groups of row k of a KM stage: the 16 rows that a transposing load reads
// at once (k, k+8, k+16, k+24 for four successive k) fall on all banks evenly
template <int T>
__device__ __forceinline__ int km_swap(int k) {
  return T == 128 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
}

// What a lane needs to load and read one operand of a tile.
template <int T, bool KM>
struct OrthOperand {
  using Cfg = OrthCfg<T>;
  unsigned voff[Cfg::LOADS];       // byte offsets of its loads from the operand's corner
  const char* base;                // the corner, at the next stage
  long step;                       // bytes to the next stage
  long lo;                         // bytes from the high to the low plane
  unsigned frag[KM ? Cfg::NF : 1]; // LDS byte offsets of its fragments

  // rows [row0, row0 + T) (KM: columns) of a plane with row length ld; `side`: which half of them
  // this wave computes
  __device__ __forceinline__ void init(const half_t* plane, long lo_halves, int ld, int row0, int side, int wave,
                                       int lane) {
    lo = 2 * lo_halves;
#pragma unroll
    for (int j = 0; j < Cfg::LOADS; ++j) {
      const int i = wave * Cfg::LOADS + j;               // which KiB of the stage
      if (KM) {
        constexpr int LANES = T / 8, ROWS = 64 / LANES;  // lanes a row, rows a load
        const int k = i * ROWS + lane / LANES, slot = lane % LANES;
        voff[j] = (unsigned)k * ld * 2 + ((slot ^ (km_swap<T>(k) << 1)) << 4);
      } else {
        const int row = i * 16 + (lane >> 2), group = (lane & 3) ^ ((row >> 2) & 3);
        voff[j] = (unsigned)row * ld * 2 + (group << 4);
      }
    }
    if (KM) {
      base = (const char*)(plane + row0);
      step = (long)ORTH_BK * ld * 2;
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
      for (int f = 0; f < Cfg::NF; ++f)
        frag[f] = k * T * 2 + (((side * Cfg::NF + f) ^ km_swap<T>(k)) << 5) + ((lane & 3) << 3);
    } else {
      base = (const char*)(plane + (long)row0 * ld);
      step = ORTH_BK * 2;
      frag[0] = side * Cfg::NF * 1024 + (lane & 15) * 64 + (((lane >> 4) ^ ((lane >> 2) & 3)) << 4);
    }
  }

  template <bool SPLIT>
  __device__ __forceinline__ void load(lds_char* dst, int wave) {
#pragma unroll
    for (int p = 0; p < (SPLIT ? 2 : 1); ++p)
#pragma unroll
      for (int j = 0; j < Cfg::LOADS; ++j)
        lds_load(base + p * lo, voff[j], dst + p * Cfg::PLANE + (wave * Cfg::LOADS + j) * 1024);
    base += step;
  }

  __device__ __forceinline__ h8 read(lds_char* stage, int f) const {
    if (KM) {
      lds_char* const at = stage + frag[f];
      const h4s u = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4s*)at);
      const h4s v = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4s*)(at + 4 * T * 2));
      return __builtin_bit_cast(h8, (h8s)__builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *(__attribute__((address_space(3))) h8*)(stage + frag[0] + f * 1024);
  }
};

// acc[i][j]: 16 x 16 block of fragment i of P against fragment j of Q; of each block lane l holds
// D[4 (l / 16) + 0..3][l % 16].
template <int T, bool SPLIT, bool P_KM>
__device__ __forceinline__ void orth_tile_product(OrthOperand<T, P_KM>& P, OrthOperand<T, false>& Q, int steps,
                                                  lds_char* lds, int wave,
                                                  f4 (&acc)[OrthCfg<T>::NF][OrthCfg<T>::NF]) {
  using Cfg = OrthCfg<T>;
  constexpr int NF = Cfg::NF, STAGE = Cfg::template stage<SPLIT>(), Q_AT = (SPLIT ? 2 : 1) * Cfg::PLANE;
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  P.template load<SPLIT>(lds, wave);
  Q.template load<SPLIT>(lds + Q_AT, wave);
  stage_barrier();
  for (int s = 0; s < steps; ++s) {
    const int cur = (s & 1) * STAGE, next = STAGE - cur;
    lds_char* const ps = lds + cur;
    lds_char* const qs = ps + Q_AT;
    h8 ph[NF], pl[NF], qh[NF], ql[NF];
    // (P first: a transposing read behind a load into LDS would wait for it)
#pragma unroll
    for (int f = 0; f < NF; ++f) ph[f] = P.read(ps, f);
    if (SPLIT) {
#pragma unroll
      for (int f = 0; f < NF; ++f) pl[f] = P.read(ps + Cfg::PLANE, f);
    }
    if (s + 1 < steps) {
      P.template load<SPLIT>(lds + next, wave);
      Q.template load<SPLIT>(lds + next + Q_AT, wave);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) qh[f] = Q.read(qs, f);
    if (SPLIT) {
#pragma unroll
      for (int f = 0; f < NF; ++f) ql[f] = Q.read(qs + Cfg::PLANE, f);
    }
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        if (SPLIT) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[i], qh[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[i], ql[j], acc[i][j], 0, 0, 0);
        }
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[i], qh[j], acc[i][j], 0, 0, 0);
      }
    stage_barrier();
  }
}

// four scaled values -> their high halves, and the low ones
__device__ __forceinline__ void split4(f4 v, h4& h, h4& l) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = (half_t)v[i];
    l[i] = (half_t)(v[i] - (float)h[i]);
  }
}

}  // namespace kfac
