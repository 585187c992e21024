// tiles.hpp — one block's tile of C = A . B^T on the matrix cores, for operands
// whose rows lie along the sum: bytes (Int8Op) or f16 (HalfOp, A as a sum of P
// parts).  Internal to the library.
//
// A stage is 128 bytes of each of the tile's rows, copied from memory straight
// into LDS, a 16-byte chunk a lane; A's stages take turns in three places, B's
// in two, so that a stage of A is still under way when a block meets at its one
// barrier a stage.  A's P parts are stages of their own over one of B.  Chunk c
// of row r lies at c ^ (r / 2 % 8): the copies stay whole 128-byte lines, and
// sixteen lanes that read the same chunk of neighbouring rows touch all of LDS's
// banks once.  A wave's chunks for one 32-byte slab of the sum are read while
// the slab before is multiplied.  Rows past an operand's last are the last one
// again, and their results are not stored.
//
// 256 x 256 is bound by the operands' way from the L2s (the copies alone, of
// 8192 x 11008 x 4096 bytes, take 205 us of 367, the products alone 280), at
// some 2.0 GHz.  Measured beside it (us; int8 8192 x 11008 x 4096, f16 8192 x
// 4096 x 11008, f16 of two parts 11008 x 4096 x 8192): 367, 611, 1256; four
// waves of 128 x 128 each 343, 630, 1284; 128 x 128 tiles, two blocks a CU, 369,
// 734; stages of 64 bytes, four places, 397, 754, 1514; two parts as twice the
// sum 1358; two places for both, loads issued after the barrier 367, 586, 1370
// (128 x 256); the barrier ahead of the last slab's products 376, 612, 1238.  With
// the waves' priority raised for a stage's products, in the layers' own calls (f16 int8
// 4096 -> 11008, dw of two parts and dx of one, 8192 rows): 478 -> 466, 1372 -> 1328, 697 ->
// 672; with the barrier ahead as well 470, 1301, 710.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "stages.hpp"

namespace wh {
namespace tiles {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Int8Op {
  using acc = i32x16;
  __device__ static inline acc mma(i32x4 a, i32x4 b, acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
};
struct HalfOp {
  using acc = f32x16;
  __device__ static inline acc mma(i32x4 a, i32x4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
};

constexpr int kStageBytes = 128;
// Bytes between rows of at least `bytes`: an odd multiple of the 256 bytes after
// which memory's channels change, so that a tile's rows, read at one place along
// them, lie in all of an L2's 16.
constexpr int64_t spread(int64_t bytes) { return ((bytes + 255) / 256 | 1) * 256; }

struct Operands {
  // the stages from `first` on, `count` of them
  __host__ __device__ Operands part(int first, int count) const {
    Operands o = *this;
    o.a += (int64_t)first * kStageBytes;
    o.b += (int64_t)first * kStageBytes;
    if (o.a_last != INT32_MAX) o.a_last -= first * kStageBytes;
    o.stages = count;
    return o;
  }
  const char *a;
  int64_t a_pitch, a_plane;  // bytes between rows, between parts
  int a_rows;
  int a_last;  // the last 16-byte chunk of a row of A; B's zeros cover what is taken past it
  const char *b;
  int64_t b_pitch;  // of whole stages
  int b_rows;
  int stages;
};

// WM x WN waves, each TM x TN products of 32 x 32.  SA and SB: the operands'
// places in LDS.  Three and two leave 128 x 128 tiles two blocks a CU; four of
// each keep three stages under way where there is one block a CU, or none.
template <class Op, int P, int WM, int WN, int TM, int TN, int SA = 3, int SB = 2>
struct Tile {
  static constexpr int kWaves = WM * WN, kRows = WM * TM * 32, kCols = WN * TN * 32;
  static constexpr int kA = kRows * kStageBytes, kB = kCols * kStageBytes, kLds = SA * kA + SB * kB;
  static constexpr int kLoadsA = kRows / 8 / kWaves, kLoadsB = kCols / 8 / kWaves;
  static constexpr int kTM = TM, kTN = TN, kParts = P;
  // of LDS after the products: the results' turning place, then the caller's
  static constexpr int kResults = kWaves * 32 * (TN * 32 + 4) * 4;
  static_assert(kRows % (8 * kWaves) == 0 && kCols % (8 * kWaves) == 0 && kWaves % 2 == 0,
                "every wave copies whole pieces of 8 rows, its chunks' places the same in all");
  static_assert(P == 1 || P == 2, "parts");
  static_assert((SA == 3 && SB == 2) || (SA == SB && SA >= 3), "the copies that may be left under way at a step");
  using Acc = typename Op::acc;
  // at most `left` of this wave's copies still under way, and none of its LDS reads
  template <int LEFT>
  __device__ static inline void wait() {
    static_assert(LEFT < 64, "the counter's range");
    __builtin_amdgcn_s_waitcnt((LEFT & 15) | ((LEFT >> 4) << 14) | (7 << 4));
    asm volatile("" ::: "memory");
  }
  // The tile at (m0, n0) into acc; B's rows are the instruction's first side, so a
  // lane's results are four neighbouring columns each time.
  __device__ static inline void run(const Operands &o, int m0, int n0, Acc (&acc)[TM][TN], char *lds) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const char *from_a[kLoadsA], *from_b[kLoadsB];
    const int chunk = ((lane & 7) ^ ((wave & 1) * 4 + (lane >> 4))) * 16;
    // how far the last stage's chunk lies past A's last one
    const int past = max((o.stages - 1) * kStageBytes + chunk - o.a_last, 0);
#pragma unroll
    for (int j = 0; j < kLoadsA; ++j)
      from_a[j] = o.a + (int64_t)min(m0 + (j * kWaves + wave) * 8 + (lane >> 3), o.a_rows - 1) * o.a_pitch + chunk;
#pragma unroll
    for (int j = 0; j < kLoadsB; ++j)
      from_b[j] = o.b + (int64_t)min(n0 + (j * kWaves + wave) * 8 + (lane >> 3), o.b_rows - 1) * o.b_pitch + chunk;
    const int steps = o.stages * P;
    constexpr Stages order{P, SA, SB};
    const auto copy = [&](const char *p, char *to) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)p,
                                       (__attribute__((address_space(3))) void *)to, 16, 0, 0);
    };
    const auto load_a = [&](int h, int part, char *to) {
      if (h >= steps - P && o.a_last != INT32_MAX && (P == 1 || part == 0)) {
#pragma unroll
        for (int j = 0; j < kLoadsA; ++j) from_a[j] -= past;
      }
#pragma unroll
      for (int j = 0; j < kLoadsA; ++j) {
        copy(P == 1 || part == 0 ? from_a[j] : from_a[j] + o.a_plane, to + (j * kWaves + wave) * 1024);
        if (part == P - 1) from_a[j] += kStageBytes;
      }
    };
    const auto load_b = [&](char *to) {
#pragma unroll
      for (int j = 0; j < kLoadsB; ++j) {
        copy(from_b[j], to + (j * kWaves + wave) * 1024);
        from_b[j] += kStageBytes;
      }
    };
    // this lane's chunk of its first rows; slab s lies at ^ 32 s
    const int swz = (((lane >> 5) ^ ((lane >> 1) & 7)) * 16) + (lane & 31) * kStageBytes;
    const int a_at = wm * TM * 32 * kStageBytes + swz, b_at = wn * TN * 32 * kStageBytes + swz;
    char *const lds_b = lds + SA * kA;
    i32x4 a[2][TM], b[2][TN];
    const auto fetch = [&](const char *at, const char *bt, int slab, int into) {
#pragma unroll
      for (int u = 0; u < TN; ++u) b[into][u] = *(const i32x4 *)(bt + ((b_at ^ (slab * 32)) + u * 32 * kStageBytes));
#pragma unroll
      for (int t = 0; t < TM; ++t) a[into][t] = *(const i32x4 *)(at + ((a_at ^ (slab * 32)) + t * 32 * kStageBytes));
    };
    constexpr int kReads = TN + TM, kMul = TM * TN;
    // A's steps and B's stages go out in the order in which they are needed; at step
    // h A has SA - 1 steps, B SB - 1 stages out ahead.
#pragma unroll
    for (int h = 0; h < SA - 1; ++h) {
      if (h % P == 0 && h / P < SB - 1 && h / P < o.stages) load_b(lds_b + h / P * kB);
      if (h < steps) load_a(h, h % P, lds + h * kA);
    }
#pragma unroll
    for (int s = (SA - 2) / P + 1; s < SB - 1; ++s)
      if (s < o.stages) load_b(lds_b + s * kB);
    int ia = 0, ib = 0;  // places of this step
    const auto step = [&](int h, auto part_) {
      constexpr int part = decltype(part_)::value;
      if (order.drains(h, steps)) wait<0>();
      else wait<order.left_a() * kLoadsA + order.left_b(part) * kLoadsB>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (part == 0 && order.sends_b(h, steps)) load_b(lds_b + (ib == 0 ? SB - 1 : ib - 1) * kB);
      if (order.sends_a(h, steps)) load_a(h + SA - 1, (part + SA - 1) % P, lds + (ia == 0 ? SA - 1 : ia - 1) * kA);
      const char *at = lds + ia * kA, *bt = lds_b + ib * kB;
      fetch(at, bt, 0, 0);
      __builtin_amdgcn_s_setprio(1);  // ahead of a wave that still waits or copies
#pragma unroll
      for (int slab = 0; slab < 4; ++slab) {
        if (slab < 3) fetch(at, bt, slab + 1, (slab + 1) & 1);
#pragma unroll
        for (int t = 0; t < TM; ++t)
#pragma unroll
          for (int u = 0; u < TN; ++u)
            acc[t][u] = Op::mma(b[slab & 1][u], a[slab & 1][t], acc[t][u]);
        // a read after each product, until they are all under way
        if (slab < 3) {
#pragma unroll
          for (int i = 0; i < kReads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          }
        }
        __builtin_amdgcn_sched_group_barrier(0x008, kMul, 0);
      }
      __builtin_amdgcn_s_setprio(0);
      ia = ia == SA - 1 ? 0 : ia + 1;
      if (part == P - 1) ib = ib == SB - 1 ? 0 : ib + 1;
    };
    for (int h = 0; h < steps; h += P) {
      step(h, std::integral_constant<int, 0>{});
      if constexpr (P == 2) step(h + 1, std::integral_constant<int, 1>{});
    }
  }
  // The first of the eight columns that `results` gives a lane.
  __device__ static inline int first_col(int n0) {
    return n0 + (int)(threadIdx.x >> 6) % WN * TN * 32 + (int)(threadIdx.x & 63) % (TN * 4) * 8;
  }
  // f(row, col, values) with W neighbouring columns of a row a lane, so that a store
  // of theirs is 16 bytes and a row's lie side by side: a wave turns its results 32 rows at a time in LDS, which
  // has to be left by the block's products (a barrier).
  using Value = std::remove_cv_t<std::remove_reference_t<decltype(std::declval<Acc>()[0])>>;
  template <int W, class F>
  __device__ static inline void results(int m0, int n0, const Acc (&acc)[TM][TN], char *lds, F &&f) {
    constexpr int kPitch = TN * 32 + 4, kAcross = TN * 32 / W;  // values, lanes a row
    static_assert(W == 4 || W == 8, "columns");
    static_assert(kWaves * 32 * kPitch * 4 <= kResults, "the results' place");
    typedef Value quad __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Value *mine = (Value *)lds + wave * 32 * kPitch;
    const int m = m0 + wave / WN * TM * 32 + lane / kAcross, n = n0 + wave % WN * TN * 32 + lane % kAcross * W;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int u = 0; u < TN; ++u)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(quad *)(mine + (lane & 31) * kPitch + u * 32 + i * 2 + (lane >> 5) * 4) =
              quad{acc[t][u][i], acc[t][u][i + 1], acc[t][u][i + 2], acc[t][u][i + 3]};
      asm volatile("" ::: "memory");
#pragma unroll 1
      for (int r = 0; r < 32; r += 64 / kAcross) {
        const quad *at = (const quad *)(mine + (r + lane / kAcross) * kPitch + lane % kAcross * W);
        Value v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = at[i / 4][i % 4];
        f(m + t * 32 + r, n, v);
      }
      asm volatile("" ::: "memory");
    }
  }
};

// Few tiles: the sum's stages in parts, a block each, whose results are joined
// in a launch of their own.  As many as give every CU a block, of eight stages and
// more, at most 16; in two parts sums of 40 steps and more, and those of 100 and more
// in three from 129 tiles to 170, two blocks a CU: below, the parts' way through memory
// takes more than they save (us, in parts and whole: int8 1024 -> 8192 of 256 rows, two
// of four stages, 29 / 15; 2048 -> 8192 of 200, two of eight, 30 / 19; 4096 -> 4096 of
// 512, two of sixteen, 34 / 31; 8192 -> 4096 45 / 50; 11008 -> 4096 53 / 64; 4096 ->
// 18432 of 128, three of eleven, 39 / 30; dx f32 8512 <- 9536 of 153, three of 50
// stages, 121 and 6 for the join / 182).
constexpr int kSplitRows = 128;  // of the largest tile that is split
struct Splits {
  int splits, each;      // parts, and the stages of one
  int64_t parts_values;  // of one's [rows][cols] results
  void *parts;
  Splits(int splits_, int64_t values, void *ws) : splits(splits_), each(0), parts_values(values), parts(ws) {}
  // steps: of the product a stage, A's parts
  Splits(int tiles_m, int tiles_n, const Operands &o, int tile_rows, int steps, void *ws)
      : splits(1), each(o.stages), parts_values((int64_t)o.a_rows * o.b_rows), parts(ws) {
    const int64_t tiles = (int64_t)tiles_m * tiles_n;
    if (tile_rows > kSplitRows || tiles > 170 || (!one_a_cu(tiles) && o.stages * steps < 100)) return;
    const int most = (int)std::min<int64_t>(16, std::min<int64_t>((one_a_cu(tiles) ? 256 : 512) / tiles, o.stages / 8));
    if (most < 2 || (most == 2 && o.stages * steps < 40)) return;
    each = (o.stages + most - 1) / most;
    splits = (o.stages + each - 1) / each;
  }
  static bool one_a_cu(int64_t tiles) { return tiles <= 128; }
};
// Their workspace for results of rows x cols: at most 512 tiles of 128 x 128; not
// less for more rows.
inline size_t parts_bytes(int64_t rows, int64_t cols) {
  return (size_t)std::min<int64_t>((int64_t)512 * kSplitRows * kSplitRows, 16 * rows * cols) * 4;
}

// The tile of a block: blocks of one XCD (every eighth) take neighbouring
// tiles, so that its L2 holds their rows: columns by columns of eight rows.
struct Place {
  int m, n;
};
__device__ inline Place place(int block, int tiles_m, int tiles_n) {
  const int all = tiles_m * tiles_n, per = all / 8, more = all % 8, xcd = block % 8;
  const int at = xcd * per + min(xcd, more) + block / 8;
  const int band = at / (8 * tiles_n), rows = min(8, tiles_m - band * 8), in = at - band * 8 * tiles_n;
  return {band * 8 + in % rows, in / rows};
}

}  // namespace tiles
}  // namespace wh
