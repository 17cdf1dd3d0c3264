// Products of the Newton-Schulz iteration on the fp16 matrix cores (gfx950, wave64).
//
// Every operand of the iteration is bounded: X, A = X X^T and B = aI + bA + cAA have entries of at
// most a few units once X is normalised.  Times 2^13 they are kept as fp16 numbers: in two parts,
// x = h + l with h = fp16(x), l = fp16(x - h), 22 bits and the sign of l, or h alone.  A product of
// two such numbers is
//     x y = h h' + h l' + l h' + [l l']
// where the bracket is at most 2^-22 of |x y|, on average (l is 2^-12.2 of x) 2^-24.5, about what rounding to
// float32 makes, and is left out: three v_mfma_f32_16x16x32_f16 with exact products and float32 sums, where
// three bf16 parts, which hold any float32, take six.
//
// In memory a row of a matrix in two parts is made of pieces of 32 elements, 64 bytes of high parts and
// 64 of low ones, so that what a tile reads of a row at a time, both parts of 32 elements, is one cache
// line; in one part it is just a row (a line is 64 elements).
//
// A workgroup computes a tile D[m][n] = sum_k P[m][k] Q[n][k].  Operands go from memory to LDS
// directly (16 bytes a lane, whole cache lines) in stages of two planes of 32 reduction steps: the high
// and the low parts of the same steps, or of operands in one part two successive pieces of 32.
//   rows of an operand with k along them ("KC"): 128 bytes a row, both planes; the 16-byte groups of a
//     row are exchanged by half its number, so that the lanes that read at once fall on different banks
//     (they are 0-3, 12-15, 20-27 and so on);
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

// A TM x TN tile on WM x WN waves, STAGES of its operands in LDS.  PAIR: see orth_pair_product.  WK: as
// many teams of WM x WN waves, each with stages of its own and every WK-th piece of the reduction.
template <int TM_, int TN_, int WM_, int WN_, int STAGES_, bool PAIR_ = false, int WK_ = 1>
struct OrthTile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, WK = WK_, WAVES = WM * WN, TEAM = 64 * WAVES, THREADS = TEAM * WK;
  static constexpr int STAGES = STAGES_;
  static constexpr bool PAIR = PAIR_;
  static constexpr int FM = TM / WM / 16, FN = TN / WN / 16;        // 16-row fragments of a wave
  static constexpr int P_PLANE = TM * ORTH_BK * 2, Q_PLANE = TN * ORTH_BK * 2;
  static constexpr int Q_AT = 2 * P_PLANE, STAGE = Q_AT + 2 * Q_PLANE;            // bytes
  static constexpr int LDS = WK * STAGES * STAGE;
  // behind the product: the sums of the other teams, then a piece for each wave that writes the tile
  static constexpr int SUMS = (WK - 1) * FM * FN * TEAM * 16;
  static constexpr int M_PITCH = FM * 64 + 16, N_PITCH = FN * 64 + 16;
  static constexpr int WRITE = 16 * (M_PITCH > N_PITCH ? M_PITCH : N_PITCH);
  static_assert(SUMS + WAVES * WRITE <= LDS, "room to write a tile");
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

// exchange of the 32-byte groups of row k of a KM stage of rows of BYTES: the 16 rows that a transposing
// load reads at once (k, k+8, k+16, k+24 for four successive k) fall on all banks evenly
template <int BYTES>
__device__ __forceinline__ int km_swap(int k) {
  return BYTES >= 256 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
}

// What a lane needs to load and read one operand of a tile: T rows (KM: columns) of it, loaded by
// WAVES waves, F fragments of them read by each.
template <int T, int WAVES, int F, bool KM, bool SPLIT>
struct OrthOperand {
  static constexpr int STAGE = T * ORTH_BK * 4, LOADS = STAGE / (1024 * WAVES);
  static_assert(LOADS >= 1, "waves");
  // KM: bytes of a row, which holds both parts (pieces of 32 columns of each in turn) or one
  static constexpr int ROW = T * (SPLIT ? 4 : 2);
  static constexpr int SECOND = KM ? (SPLIT ? 64 : ORTH_BK * ROW) : 64;      // from the first plane to the second
  unsigned voff[LOADS];            // byte offsets of its loads from the operand's corner
  const char* base;                // the corner, at the next stage
  long step;                       // bytes to the next stage
  unsigned frag[KM ? 2 * F : 2];   // LDS byte offsets of its fragments in the planes (KC: of the first ones)

  // rows [row0, row0 + T) (KM: columns) of a matrix of rows of `ld` elements; `side`: which F fragments
  // of them this wave computes
  __device__ __forceinline__ void init(const half_t* matrix, int ld, int row0, int side, int wave, int lane) {
    const int row_bytes = ld * (SPLIT ? 4 : 2);
    step = !KM ? 128 : (long)(SPLIT ? 1 : 2) * ORTH_BK * row_bytes;
    base = (const char*)matrix + (KM ? (long)row0 * (SPLIT ? 4 : 2) : (long)row0 * row_bytes);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int at = ((wave * LOADS + j) * 64 + lane) * 16;           // where this lane's bytes go
      constexpr int BYTES = KM ? ROW : 128;
      const int row = at / BYTES, group = at % BYTES / 16;
      voff[j] = (unsigned)row * row_bytes + 16 * (group ^ (KM ? km_swap<ROW>(row) << 1 : (row >> 1) & 7));
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (KM) {
        const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
        for (int f = 0; f < F; ++f) {
          const int c = side * F + f;                                 // which 16 columns
          const int group = SPLIT ? (c >> 1) * 4 + 2 * p + (c & 1) : c;
          frag[p * F + f] = (SPLIT ? 0 : p * SECOND) + k * ROW + ((group ^ km_swap<ROW>(k)) << 5) + ((lane & 3) << 3);
        }
      } else {
        const int row = lane & 15, group = 4 * p + (lane >> 4);
        frag[p] = side * F * 2048 + row * 128 + ((group ^ ((row >> 1) & 7)) << 4);
      }
    }
  }

  __device__ __forceinline__ void load(unsigned dst, int wave) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) lds_load(base, voff[j], dst + (wave * LOADS + j) * 1024);
    base += step;
  }

  __device__ __forceinline__ h8 read(lds_char* stage, int plane, int f) const {
    if (KM) {
      lds_char* const at = stage + frag[plane * F + f];
      const h4s u = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4s*)at);
      const h4s v = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4s*)(at + 4 * ROW));
      return __builtin_bit_cast(h8, (h8s)__builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *(__attribute__((address_space(3))) h8*)(stage + frag[plane] + f * 2048);
  }
};

// The blocks of fragments i0 ... i0 + N - 1 of P against all of Q, one of the partial products after
// the other: an instruction waits for the one before it that adds to the same block.
template <bool SPLIT, int N, int FM, int FN>
__device__ __forceinline__ void orth_mfma(const h8 (&p)[2][N], const h8 (&q)[2][FN], f4 (&acc)[FM][FN], int i0) {
  constexpr int TERMS = SPLIT ? 3 : 2;
  constexpr int PP[3] = {1, 0, 0}, QQ[3] = {SPLIT ? 0 : 1, SPLIT ? 1 : 0, 0};
#pragma unroll
  for (int t = 0; t < TERMS; ++t)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i0 + i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[PP[t]][i], q[QQ[t]][j], acc[i0 + i][j], 0, 0, 0);
}

template <int N, class OP>
__device__ __forceinline__ void orth_read(const OP& op, lds_char* stage, h8 (&v)[2][N]) {
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int f = 0; f < N; ++f) v[p][f] = op.read(stage, p, f);
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
// is STAGES - 1 ahead is asked for.  With several teams the first one ends up with the sum.
template <class TILE, bool SPLIT, class OP_P, class OP_Q>
__device__ __forceinline__ void orth_product(OP_P& P, OP_Q& Q, int steps, lds_char* lds, int wave, int team,
                                             f4 (&acc)[TILE::FM][TILE::FN]) {
  constexpr int S = TILE::STAGES, LOADS = OP_P::LOADS + OP_Q::LOADS, WK = TILE::WK;
  static_assert(WK > 1, "teams");
  orth_clear<TILE>(acc);
  lds_char* const mine = lds + team * S * TILE::STAGE;
  const unsigned at = (unsigned)(uintptr_t)mine;
  P.base += team * P.step;
  Q.base += team * Q.step;
  P.step *= WK;
  Q.step *= WK;
  const int own = (steps + WK - 1 - team) / WK, all = (steps + WK - 1) / WK;
  const auto load = [&](int stage) {
    P.load(at + stage * TILE::STAGE, wave);
    Q.load(at + stage * TILE::STAGE + TILE::Q_AT, wave);
  };
  int ahead = 0;                           // stages asked for
  for (; ahead < S - 1 && ahead < own; ++ahead) load(ahead);
  int cur = 0, into = S - 1;
  for (int s = 0; s < all; ++s) {
    if (ahead - s == S - 1) stage_barrier<(S - 2) * LOADS>();
    else stage_barrier<0>();
    if (ahead < own) {
      load(into);
      ++ahead;
    }
    if (s < own) {
      lds_char* const stage = mine + cur * TILE::STAGE;
      h8 p[2][TILE::FM], q[2][TILE::FN];
      orth_read(P, stage, p);
      orth_read(Q, stage + TILE::Q_AT, q);
      orth_mfma<SPLIT>(p, q, acc, 0);
    }
    into = cur;
    cur = cur + 1 == S ? 0 : cur + 1;
  }
  typedef __attribute__((address_space(3))) f4 lds_f4;
  constexpr int PER = TILE::FM * TILE::FN, TEAM = TILE::TEAM;
  stage_barrier<0>();
  lds_f4* const sums = (lds_f4*)lds + (threadIdx.x & (TEAM - 1));
  if (team > 0)
#pragma unroll
    for (int i = 0; i < PER; ++i) sums[((team - 1) * PER + i) * TEAM] = acc[i / TILE::FN][i % TILE::FN];
  stage_barrier<0>();
  if (team == 0)
#pragma unroll
    for (int w = 0; w < WK - 1; ++w)
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i / TILE::FN][i % TILE::FN] += sums[(w * PER + i) * TEAM];
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
    orth_read(P, lds + stage * TILE::STAGE, p);
    orth_read(Q, lds + stage * TILE::STAGE + TILE::Q_AT, q);
  };
  constexpr int LOADS = OP_P::LOADS + OP_Q::LOADS;
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

// Where element c of a row of `ld` elements lies (in halves, from the start of the matrix); its low part
// is 32 behind.
__device__ __forceinline__ long orth_at(int row, int c, int ld, bool split) {
  return split ? (long)row * 2 * ld + ((c >> 5) << 6) + (c & 31) : (long)row * ld + c;
}

// What this wave has written to LDS can be read by its other lanes, and the other way round.
__device__ __forceinline__ void wave_fence() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
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
