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
// A workgroup computes a tile D[m][n] = sum_k P[m][k] Q[n][k].  Operands go from memory to LDS
// directly (16 bytes a lane) in stages of two planes of 32 reduction steps: the high and the low parts
// of the same steps, or of operands in one part two successive pieces of 32.
//   rows of an operand with k along them ("KC"): 64 bytes a row; the 16-byte groups of a row are
//     exchanged by its number, so that the lanes that read at once fall on different banks (they are
//     0-3, 12-15, 20-27 and so on);
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
constexpr int ORTH_BK = 32;                      // reduction steps of a stage

// A TM x TN tile on WM x WN waves, STAGES of its operands in LDS.  PAIR: see orth_pair_product.
template <int TM_, int TN_, int WM_, int WN_, int STAGES_, bool PAIR_ = false>
struct OrthTile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int STAGES = STAGES_;
  static constexpr bool PAIR = PAIR_;
  static constexpr int FM = TM / WM / 16, FN = TN / WN / 16;        // 16-row fragments of a wave
  static constexpr int P_PLANE = TM * ORTH_BK * 2, Q_PLANE = TN * ORTH_BK * 2;
  static constexpr int Q_AT = 2 * P_PLANE, STAGE = Q_AT + 2 * Q_PLANE;            // bytes
  static constexpr int LDS = STAGES * STAGE;
};

// 64 lanes times 16 bytes from `base` + voff to LDS at `dst` (lane i at dst + 16 i).  M0 holds the
// LDS address and is written right in front of its use, here as in what the compiler makes of its
// builtin; the builtin itself would have every transposing read wait for all loads in flight.
__device__ __forceinline__ void lds_load(const char* base, unsigned voff, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(dst), "v"(voff), "s"(base) : "memory");
}
// Of this wave's loads into LDS all but the last N have landed, its reads are done, and so it is with
// all other waves.
template <int N>
__device__ __forceinline__ void stage_barrier() {
  static_assert(N < 64, "loads in flight");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory");
}

// exchange of the 32-byte groups of row k of a KM stage: the 16 rows that a transposing load reads
// at once (k, k+8, k+16, k+24 for four successive k) fall on all banks evenly
template <int T>
__device__ __forceinline__ int km_swap(int k) {
  return T >= 128 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
}

// What a lane needs to load and read one operand of a tile: T rows (KM: columns) of it, loaded by
// WAVES waves, F fragments of them read by each.
template <int T, int WAVES, int F, bool KM>
struct OrthOperand {
  static constexpr int PLANE = T * ORTH_BK * 2, LOADS = PLANE / (1024 * WAVES);
  static_assert(LOADS >= 1, "waves");
  unsigned voff[LOADS];            // byte offsets of its loads from the operand's corner
  const char* base;                // the corner, at the next stage
  long step;                       // bytes to the next stage
  long second;                     // bytes from the first to the second plane
  unsigned frag[KM ? F : 1];       // LDS byte offsets of its fragments

  // rows [row0, row0 + T) (KM: columns) of a matrix with row length ld, its low parts lo_halves behind
  // its high ones (0: it has one part); `side`: which F fragments of them this wave computes
  __device__ __forceinline__ void init(const half_t* plane, long lo_halves, int ld, int row0, int side, int wave,
                                       int lane) {
    const long piece = (long)ORTH_BK * 2 * (KM ? ld : 1);
    second = lo_halves ? 2 * lo_halves : piece;
    step = lo_halves ? piece : 2 * piece;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int i = wave * LOADS + j;               // which KiB of the stage
      if (KM) {
        constexpr int LANES = T / 8, ROWS = 64 / LANES;  // lanes a row, rows a load
        const int k = i * ROWS + lane / LANES, slot = lane % LANES;
        voff[j] = (unsigned)k * ld * 2 + ((slot ^ (km_swap<T>(k) << 1)) << 4);
      } else {
        const int row = i * 16 + (lane >> 2), group = (lane & 3) ^ (-(row >> 2) & 3);
        voff[j] = (unsigned)row * ld * 2 + (group << 4);
      }
    }
    if (KM) {
      base = (const char*)(plane + row0);
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
      for (int f = 0; f < F; ++f)
        frag[f] = k * T * 2 + (((side * F + f) ^ km_swap<T>(k)) << 5) + ((lane & 3) << 3);
    } else {
      base = (const char*)(plane + (long)row0 * ld);
      frag[0] = side * F * 1024 + (lane & 15) * 64 + (((lane >> 4) ^ (-(lane >> 2) & 3)) << 4);
    }
  }

  __device__ __forceinline__ void load(unsigned dst, int wave) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        lds_load(base + p * second, voff[j], dst + p * PLANE + (wave * LOADS + j) * 1024);
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

// The blocks of fragments i0 ... i0 + N - 1 of P against all of Q.
template <bool SPLIT, int N, int FM, int FN>
__device__ __forceinline__ void orth_mfma(const h8 (&p)[2][N], const h8 (&q)[2][FN], f4 (&acc)[FM][FN], int i0) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      f4& d = acc[i0 + i][j];
      if (SPLIT) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[1][i], q[0][j], d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[0][i], q[1][j], d, 0, 0, 0);
      } else {
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[1][i], q[1][j], d, 0, 0, 0);
      }
      d = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[0][i], q[0][j], d, 0, 0, 0);
    }
}

template <int N, class OP>
__device__ __forceinline__ void orth_read(const OP& op, lds_char* stage, int f0, h8 (&v)[2][N]) {
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int f = 0; f < N; ++f) v[p][f] = op.read(stage + p * OP::PLANE, f0 + f);
}

template <class TILE>
__device__ __forceinline__ void orth_clear(f4 (&acc)[TILE::FM][TILE::FN]) {
#pragma unroll
  for (int i = 0; i < TILE::FM; ++i)
#pragma unroll
    for (int j = 0; j < TILE::FN; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
}

// acc[i][j]: 16 x 16 block of fragment i of P against fragment j of Q over `steps` stages; of each
// block lane l holds D[4 (l / 16) + 0..3][l % 16].  One barrier a stage, behind which the stage that
// is STAGES - 1 ahead is asked for.
template <class TILE, bool SPLIT, class OP_P, class OP_Q>
__device__ __forceinline__ void orth_product(OP_P& P, OP_Q& Q, int steps, lds_char* lds, int wave,
                                             f4 (&acc)[TILE::FM][TILE::FN]) {
  constexpr int S = TILE::STAGES, LOADS = 2 * (OP_P::LOADS + OP_Q::LOADS);
  orth_clear<TILE>(acc);
  const unsigned at = (unsigned)(uintptr_t)lds;
  const auto load = [&](int stage) {
    P.load(at + stage * TILE::STAGE, wave);
    Q.load(at + stage * TILE::STAGE + TILE::Q_AT, wave);
  };
  int ahead = 0;                           // stages asked for
  for (; ahead < S - 1 && ahead < steps; ++ahead) load(ahead);
  int cur = 0, into = S - 1;
  for (int s = 0; s < steps; ++s) {
    if (ahead - s == S - 1) stage_barrier<(S - 2) * LOADS>();
    else stage_barrier<0>();
    if (ahead < steps) {
      load(into);
      ++ahead;
    }
    lds_char* const stage = lds + cur * TILE::STAGE;
    h8 p[2][TILE::FM], q[2][TILE::FN];
    orth_read(P, stage, 0, p);
    orth_read(Q, stage + TILE::Q_AT, 0, q);
    orth_mfma<SPLIT>(p, q, acc, 0);
    into = cur;
    cur = cur + 1 == S ? 0 : cur + 1;
  }
}

// The same for a workgroup of eight waves that has the compute unit to itself, two waves on every
// SIMD: while one reads its fragments of a stage, the other multiplies those that it has read, and
// they change places at a barrier.  Stage s is read by the first four waves in phase 2s and by the
// others in phase 2s + 1, so that its successor, in the other half of the LDS, may be asked for from
// phase 2s on and has to be there at the end of phase 2s + 1.
template <class TILE, bool SPLIT, class OP_P, class OP_Q>
__device__ __forceinline__ void orth_pair_product(OP_P& P, OP_Q& Q, int steps, lds_char* lds, int wave,
                                                  f4 (&acc)[TILE::FM][TILE::FN]) {
  static_assert(TILE::WAVES == 8 && TILE::STAGES == 2, "waves");
  orth_clear<TILE>(acc);
  const unsigned at = (unsigned)(uintptr_t)lds;
  const auto load = [&](int stage) {
    P.load(at + stage * TILE::STAGE, wave);
    Q.load(at + stage * TILE::STAGE + TILE::Q_AT, wave);
  };
  h8 p[2][TILE::FM], q[2][TILE::FN];
  const auto read = [&](int stage) {
    orth_read(P, lds + stage * TILE::STAGE, 0, p);
    orth_read(Q, lds + stage * TILE::STAGE + TILE::Q_AT, 0, q);
  };
  constexpr int LOADS = 2 * (OP_P::LOADS + OP_Q::LOADS);
  load(0);
  stage_barrier<0>();
  if (wave < 4) {
    for (int s = 0; s < steps; ++s) {
      read(s & 1);
      if (s + 1 < steps) load((s + 1) & 1);
      stage_barrier<LOADS>();
      __builtin_amdgcn_sched_barrier(0);
      orth_mfma<SPLIT>(p, q, acc, 0);
      __builtin_amdgcn_sched_barrier(0);
      stage_barrier<0>();
    }
  } else {
    if (steps > 1) load(1);
    stage_barrier<LOADS>();
    for (int s = 0; s < steps; ++s) {
      read(s & 1);
      stage_barrier<0>();
      if (s + 2 < steps) load(s & 1);
      __builtin_amdgcn_sched_barrier(0);
      orth_mfma<SPLIT>(p, q, acc, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (s + 1 < steps) stage_barrier<LOADS>();
    }
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
