// tiles.hpp — one block's tile of C = A . B^T on the matrix cores, for operands
// whose rows lie along the sum: bytes (Int8Op) or bf16 (Bf16Op, A as a sum of
// P parts).  Internal to the library.
//
// A stage is 64 bytes of each of the tile's rows, copied from memory straight
// into LDS, a 16-byte chunk a lane; NBUF stages are under way at a time and a
// block has one barrier a stage.  Chunk c of row r lies at c ^ (r / 2 % 4): the
// copies stay whole 64-byte pieces of a row, and eight lanes that read the
// same chunk of neighbouring rows touch all of LDS's banks once.  Rows past an
// operand's last are the last one again, and their results are not stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wh {
namespace tiles {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Int8Op {
  using acc = i32x16;
  __device__ static inline acc mma(i32x4 a, i32x4 b, acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
};
struct Bf16Op {
  using acc = f32x16;
  __device__ static inline acc mma(i32x4 a, i32x4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};

constexpr int kStageBytes = 64;

struct Operands {
  const char *a;
  int64_t a_pitch, a_plane;  // bytes between rows, between parts
  int a_rows;
  int a_last;  // the last 16-byte chunk of a row of A; B's zeros cover what is taken past it
  const char *b;
  int64_t b_pitch;  // of whole stages
  int b_rows;
  int stages;
};

// WM x WN waves, each TM x TN products of 32 x 32.
template <class Op, int P, int WM, int WN, int TM, int TN, int NBUF>
struct Tile {
  static constexpr int kWaves = WM * WN, kRows = WM * TM * 32, kCols = WN * TN * 32;
  static constexpr int kStage = (P * kRows + kCols) * kStageBytes, kLds = NBUF * kStage;
  static constexpr int kLoads = (P * kRows + kCols) / 16 / kWaves;
  static_assert((P * kRows + kCols) % (16 * kWaves) == 0, "every wave copies whole pieces of 16 rows");
  static constexpr int kTM = TM, kTN = TN;
  using Acc = typename Op::acc;

  // at most `left` of this wave's loads still under way, and none of its LDS reads
  template <int LEFT>
  __device__ static inline void wait() {
    static_assert(LEFT < 64, "the counter's range");
    __builtin_amdgcn_s_waitcnt((LEFT & 15) | ((LEFT >> 4) << 14) | (7 << 4));
    asm volatile("" ::: "memory");
  }

  __device__ static inline void run(const Operands &o, int m0, int n0, Acc (&acc)[TM][TN], char *lds) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const char *from[kLoads];
    int last[kLoads];
    const int chunk = ((lane & 3) ^ ((lane >> 3) & 3)) * 16;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int piece = j * kWaves + wave;
      if (piece < P * (kRows / 16)) {
        const int part = piece / (kRows / 16), r = m0 + piece % (kRows / 16) * 16 + (lane >> 2);
        from[j] = o.a + part * o.a_plane + (int64_t)min(r, o.a_rows - 1) * o.a_pitch;
        last[j] = o.a_last;
      } else {
        const int r = n0 + (piece - P * (kRows / 16)) * 16 + (lane >> 2);
        from[j] = o.b + (int64_t)min(r, o.b_rows - 1) * o.b_pitch;
        last[j] = INT32_MAX;
      }
    }
    const auto load = [&](int stage, int buf) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int at = min(stage * kStageBytes + chunk, last[j]);
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)(from[j] + at),
            (__attribute__((address_space(3))) void *)(lds + buf * kStage + (j * kWaves + wave) * 1024), 16, 0, 0);
      }
    };
    // this lane's chunk of its first row of A and of B; the second half of a stage lies at ^ 32
    const int swz = (((lane >> 5) ^ ((lane >> 1) & 3)) * 16) + (lane & 31) * kStageBytes;
    const int a_at = wm * TM * 32 * kStageBytes + swz, b_at = (P * kRows + wn * TN * 32) * kStageBytes + swz;
#pragma unroll
    for (int s = 0; s < NBUF - 1; ++s)
      if (s < o.stages) load(s, s);
    int buf = 0, into = NBUF - 1;
    for (int s = 0; s < o.stages; ++s) {
      if (s + NBUF - 2 < o.stages) wait<(NBUF - 2) * kLoads>();
      else wait<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s + NBUF - 1 < o.stages) load(s + NBUF - 1, into);
      const char *at = lds + buf * kStage;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        i32x4 a[P][TM], b[TN];
#pragma unroll
        for (int u = 0; u < TN; ++u) b[u] = *(const i32x4 *)(at + ((b_at ^ (half * 32)) + u * 32 * kStageBytes));
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int t = 0; t < TM; ++t)
            a[p][t] = *(const i32x4 *)(at + ((a_at ^ (half * 32)) + (p * kRows + t * 32) * kStageBytes));
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int t = 0; t < TM; ++t)
#pragma unroll
            for (int u = 0; u < TN; ++u) acc[t][u] = Op::mma(a[p][t], b[u], acc[t][u]);
      }
      buf = buf + 1 == NBUF ? 0 : buf + 1;
      into = into + 1 == NBUF ? 0 : into + 1;
    }
  }
  // f(row, col, value) of this lane's results, row by row: 32 lanes take 32 neighbouring columns.
  template <class F>
  __device__ static inline void results(int m0, int n0, const Acc (&acc)[TM][TN], F &&f) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int u = 0; u < TN; ++u)
          f(m0 + (wm * TM + t) * 32 + (i >> 2) * 8 + (lane >> 5) * 4 + (i & 3), n0 + (wn * TN + u) * 32 + (lane & 31),
            acc[t][u][i]);
  }
};

// The tile of a block: blocks of one XCD (every eighth) take neighbouring
// tiles, so that its L2 holds their rows: columns by columns of eight rows.
struct Place {
  int m, n;
};
__device__ inline Place place(int tiles_m, int tiles_n) {
  const int all = tiles_m * tiles_n, per = all / 8, more = all % 8, xcd = blockIdx.x % 8;
  const int at = xcd * per + min(xcd, more) + (int)(blockIdx.x / 8);
  const int band = at / (8 * tiles_n), rows = min(8, tiles_m - band * 8), in = at - band * 8 * tiles_n;
  return {band * 8 + in % rows, in / rows};
}

}  // namespace tiles
}  // namespace wh
