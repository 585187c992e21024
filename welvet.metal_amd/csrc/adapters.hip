// adapters.hip — low-rank adapters of many requests beside one shared
// projection: adapter a holds a down factor [rank][in] and an up factor
// [rank][out], and every row of x names its own adapter (or none).
//   forward   h = x . down_a^T             y  = base + s_a h . up_a
//   backward  g = dy . up_a^T              dx = dx_base + s_a g . down_a
//             ddown_a = s_a sum_t g_t x_t  dup_a = s_a sum_t h_t dy_t
// Both factors keep the rank first, so the two directions are the same three
// products: rows by a factor over its width (down_row_kernel, slice_kernel),
// rank values spread over a width (spread_row, up_kernel), and sums over an
// adapter's rows (few_kernel, outer_kernel, and slice_kernel for dup, whose dy
// it reads anyway).  Products and sums are f32: activations are f32 and a
// 16-bit factor is exact in f32.
//
// Few rows go one by one in two launches, in their own order: latency and the
// factors' reads through the L2s bound them (f32 1001x777 rank 5 n3: 11.9 us;
// bf16 4096x11008 rank 16 n64: 11.6, 28 MB at 2.1 TB/s; backward, f32 2048x8192
// rank 8 n256: 16.3).  Many rows are sorted by their adapters (tokens.hpp), so
// that an adapter's rows pass a factor held in registers, and cost about the
// activations' bytes (bf16 4096x4096 rank 16 n8192 forward: 89 us, 403 MB at
// 4.5 TB/s; backward bf16 4096x11008 rank 32 n8192: 281 us, 787 MB at 2.8 TB/s,
// of which the matrix pipe would take 105 with f32 MFMAs alone).  Rows of
// different adapters never share a sum, so no value of another tenant's factor
// reaches a row, NaN or not.
#include <hip/hip_runtime.h>

#include "tokens.hpp"

namespace wh {
namespace {

using namespace tok;

using v4f = __attribute__((ext_vector_type(4))) float;
__device__ inline v4f mfma(float a, float b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

constexpr int kMaxRank = 256;

// The rows of a launch: position p -> row and adapter (count: none).
struct RowMap {
  const int32_t *key;    // adapter by position
  const int32_t *order;  // row by position; null: the row itself, unsorted
  int n, count;
  __device__ int row(int p) const { return order ? order[p] : p; }
  __device__ int adapter(int p) const {
    const uint32_t a = (uint32_t)key[p];
    return a < (uint32_t)count ? (int)a : count;
  }
};
struct Factor {
  const void *p;
  const int32_t *ranks;
  const float *scales;
  int rank, width;
  __device__ int rank_of(int a) const { return ranks ? min(max(ranks[a], 0), rank) : rank; }
  __device__ float scale_of(int a) const { return scales ? scales[a] : 1.0f; }
};
// Rows' products with a factor: [splits][n][rank], to be added up.
struct Hidden {
  float *p;
  int splits, n, rank;
  __device__ float at(int row, int j) const {
    const float *q = p + (int64_t)row * rank + j;
    const int64_t step = (int64_t)n * rank;
    float v = q[0];
    for (int s = 1; s < splits; s += 8) {  // eight loads in flight
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = q[min(s + i, splits - 1) * step];
#pragma unroll
      for (int i = 0; i < 8; ++i) v = s + i < splits ? v + w[i] : v;
    }
    return v;
  }
  // Four neighbouring ones, zeros past the rank.
  __device__ float4 at4(int row, int j) const {
    if (rank % 4 != 0) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = j + i < rank ? at(row, j + i) : 0.0f;
      return make_float4(v[0], v[1], v[2], v[3]);
    }
    if (j >= rank) return make_float4(0, 0, 0, 0);
    const float *q = p + (int64_t)row * rank + j;
    const int64_t step = (int64_t)n * rank;
    float4 v = load4(q, 0, 4);
    for (int s = 1; s < splits; s += 4) {
      float4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = load4(q + min(s + i, splits - 1) * step, 0, 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v = s + i < splits ? add4(v, w[i]) : v;
    }
    return v;
  }
};

// --------------------------------------------------------- rows by a factor
// hidden[split][row][j] = sum over the split's k of x[row][k] factor_a[j][k].
//
// Few rows: a block one row, R ranks and a split of the width.  What is read
// counts here, and every lane reads its own: four neighbouring k of x and of
// each rank row, 256 k a wave's step, the block's waves in turn with the next
// step's loads in flight.  (Lanes of an MFMA would share an x value sixteen
// times and load it as often: f32 2048x8192 rank 8 n256 17 us, so 6.8.)
// A rank's 64 lane sums are folded so that each exchange halves the values.
// Rank rows past the adapter's repeat its last one and are dropped at the end.
constexpr int kDownWaves = 4;
constexpr int kStep = 256;
template <class T, int R>
__global__ void __launch_bounds__(kDownWaves * 64) down_row_kernel(RowMap rows, Factor fac,
                                                                   const float *__restrict__ x, int64_t xstride,
                                                                   Hidden out, int split_len) {
  using raw = typename T::raw;
  __shared__ float red[kDownWaves][R];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x, j0 = blockIdx.z * R;
  const int kbegin = blockIdx.y * split_len, kend = min(kbegin + split_len, fac.width);
  const int first = kbegin + wave * kStep;
  const int full = first + kStep <= kend ? (kend - first - kStep) / (kDownWaves * kStep) + 1 : 0;  // whole steps
  const float *xrow = x + (int64_t)row * xstride;
  const int a = __builtin_amdgcn_readfirstlane(rows.adapter(row)), ra = a < rows.count ? fac.rank_of(a) : 0;
  if (ra > j0) {
    float acc[R] = {};
    const raw *f = (const raw *)fac.p + ((int64_t)a * fac.rank + j0) * fac.width;
    const int last = min(R, ra - j0) - 1;
    Quad<F32> xv[2];
    Quad<T> fv[2][R];
    const auto load = [&](int d, int step) {
      const int k = first + min(step, full - 1) * (kDownWaves * kStep) + 4 * lane;
      xv[d] = Quad<F32>::load((const uint32_t *)xrow + k);
#pragma unroll
      for (int j = 0; j < R; ++j) fv[d][j] = Quad<T>::load(f + (int64_t)min(j, last) * fac.width + k);
      issued();
    };
    const auto multiply = [&](int d) {
#pragma unroll
      for (int j = 0; j < R; ++j)
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[j] = fmaf(xv[d].get(m), fv[d][j].get(m), acc[j]);
    };
    if (full > 0) {
      // no condition between a load and its use: the compiler would move the
      // load past it
      load(0, 0);
      for (int step = 1; step < full; step += 2) {
        load(1, step);
        multiply(0);
        load(0, step + 1);
        multiply(1);
      }
      if (full & 1) multiply(0);
    }
    const int k = first + full * (kDownWaves * kStep);  // the rest of the width, one wave's
    if (k < kend) {
      const Quad<F32> xs = Quad<F32>::load((const uint32_t *)xrow, k + 4 * lane, kend);
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const Quad<T> fs = Quad<T>::load(f + (int64_t)min(j, last) * fac.width, k + 4 * lane, kend);
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[j] = fmaf(xs.get(m), fs.get(m), acc[j]);
      }
    }
    int own = 0;  // the rank whose sum the lane ends with
#pragma unroll
    for (int half = R / 2, mask = 32, bit = 1; half > 0; half /= 2, mask /= 2, bit *= 2) {
      const bool upper = lane & mask;
      own += upper ? bit : 0;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float mine = upper ? acc[2 * i + 1] : acc[2 * i], other = upper ? acc[2 * i] : acc[2 * i + 1];
        acc[i] = mine + __shfl_xor(other, mask);
      }
    }
    float sum = acc[0];
#pragma unroll
    for (int mask = 32 / R; mask > 0; mask /= 2) sum += __shfl_xor(sum, mask);
    if ((lane & (64 / R - 1)) == 0) red[wave][own] = sum;
  }
  __syncthreads();
  const int j = threadIdx.x;
  if (j < min(R, fac.rank - j0)) {
    float sum = 0.0f;
    if (j0 + j < ra)
#pragma unroll
      for (int w = 0; w < kDownWaves; ++w) sum += red[w][j];
    out.p[((int64_t)blockIdx.y * out.n + row) * out.rank + j0 + j] = sum;
  }
}

// An adapter's sums over a block's rows, D[i = rank][j = column]: into the
// gradient where all its rows lie in the block, else into the block's partial
// (slot 0: its rows began earlier, slot 1: they go on) for sum_kernel.
struct Sum {
  const float *hidden, *x;
  int64_t xstride;
  int width, chunk;  // chunk: rows of a block
  float *grad, *part;
};
template <bool ACC, int RT, bool NARROW>
__device__ inline void store_sums(const v4f (&acc)[RT][4], const Factor &fac, int a, int ra, int j0, int q,
                                  const Cols<NARROW> &cols, bool began, bool goes_on, const Sum &job) {
  const int64_t size = (int64_t)fac.rank * job.width;
  const float scale = fac.scale_of(a);
  const bool whole = began && !goes_on;
  float *to = whole ? job.grad + (int64_t)a * size : job.part + ((int64_t)blockIdx.y * 2 + (began ? 1 : 0)) * size;
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = j0 + 16 * t + 4 * q + r;
      if (j >= fac.rank || !cols.any()) continue;
      float4 v = j < ra ? make_float4(acc[t][0][r], acc[t][1][r], acc[t][2][r], acc[t][3][r])
                        : make_float4(0, 0, 0, 0);  // rank rows past the adapter's
      float *at = to + (int64_t)j * job.width;
      if (whole) {
        v = j < ra ? mul4(v, scale) : v;
        if constexpr (ACC) v = add4(cols.load(at), v);
      }
      cols.store(at, v);
    }
}

// f32 products at the bf16 MFMA's rate, for 16-bit factors: x is cut into
// three bf16 parts without rounding (8 + 8 + 8 significand bits), a bf16 value
// is one part and an f16 value (11 bits) two, so the part products are exact;
// of f16's six the smallest, below 2^-24 of the product, is left out.  The caller
// does again by f32 products
//   sums that come out as Inf or NaN: a part product can be one where the
//   product is not;
//   sums of values below 2^-110 with bits below 2^-133, where bf16 ends.  In 64
//   columns those come to less than 2^-127 of the largest factor value: half an
//   ulp of a sum of kSmallSum while that is below kLargeFactor.  So values are
//   looked at where a sum is smaller, or the factor has a larger one.
constexpr uint32_t kSmallSum = 47u << 23;           // 2^-80, as bits
constexpr uint32_t kLargeFactor = (127 + 23) << 7;  // 2^23, as bf16's
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ inline v4f mfma16(const uint4 &a, const uint4 &b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <class T>
constexpr int kParts = std::is_same_v<T, BF16> ? 1 : 2;
// the upper halves of two words, the first's below
__device__ inline uint32_t upper2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
// Eight values as bf16 parts, the next part's source left in v.
__device__ inline uint4 take_part(uint4 (&v)[2]) {
  const uint4 part = {upper2(v[0].x, v[0].y), upper2(v[0].z, v[0].w), upper2(v[1].x, v[1].y), upper2(v[1].z, v[1].w)};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[i].x = f2u(u2f(v[i].x) - u2f(v[i].x & 0xffff0000u));
    v[i].y = f2u(u2f(v[i].y) - u2f(v[i].y & 0xffff0000u));
    v[i].z = f2u(u2f(v[i].z) - u2f(v[i].z & 0xffff0000u));
    v[i].w = f2u(u2f(v[i].w) - u2f(v[i].w & 0xffff0000u));
  }
  return part;
}
__device__ inline void pin(uint4 &v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
// Whether two parts leave one of the eight values more than a third holds.
__device__ inline bool past_parts(const uint4 &a, const uint4 &b) {
  uint4 v[2] = {a, b};
  pin(v[0]);  // cut anew, rather than kept from the products
  pin(v[1]);
  take_part(v);
  take_part(v);
  return ((v[0].x | v[0].y | v[0].z | v[0].w | v[1].x | v[1].y | v[1].z | v[1].w) & 0xffff) != 0;
}
// Two quads of a 16-bit factor as parts.
template <class T>
__device__ inline void factor_parts(const Quad<T> &a, const Quad<T> &b, uint4 (&p)[2]) {
  if constexpr (kParts<T> == 1) {
    p[0] = {a.v.x, a.v.y, b.v.x, b.v.y};
  } else {
    uint4 v[2] = {{f2u(a.get(0)), f2u(a.get(1)), f2u(a.get(2)), f2u(a.get(3))},
                  {f2u(b.get(0)), f2u(b.get(1)), f2u(b.get(2)), f2u(b.get(3))}};
    p[0] = take_part(v);
    p[1] = take_part(v);
  }
}
// Value i of eight from its parts (exact).
template <class T>
__device__ inline float from_parts(const uint4 (&p)[2], int i) {
  const auto half = [&](const uint4 &w) {
    const uint32_t word = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
    return u2f(i & 1 ? word & 0xffff0000u : word << 16);
  };
  if constexpr (kParts<T> == 1) return half(p[0]);
  else return half(p[0]) + half(p[1]);
}

// Many rows, a block a slice of the width: the slice's factor
// values stay in registers while an adapter's rows pass, 16 at a time, the next
// 16 rows' loads in flight.  Every wave holds 64 columns, its products are
// added up across the block in LDS, and the slices' sums are left for
// fold_kernel: hidden[slice][row][j].  A lane's four 16-byte pieces of a row
// start at its wave's column + 16 m + 4 (l / 16).  A wave whose columns pass
// the row's end takes the row's last 64, the first `skip` of them (another
// wave's) as zeros; rows of fewer than 64 columns (NARROW) go value by value.
//
// SUMS: the rows also give the second product that reads them, sum over the
// adapter's rows of job.hidden[row][j] x[row][c] (outer_kernel below has its
// terms), so that x is read from HBM once for both: a wave's 16 x 64 part is
// turned in LDS to the columns-by-rows order of that product (bf16 4096x11008
// rank 32 n8192, dy's 361 MB: 145 us, 2.5 TB/s; its MFMAs 45 and the turning's
// LDS traffic 22 do not lie wholly under the loads).
constexpr int kSliceWaves = 8;
constexpr int kSlice = kSliceWaves * 64;
constexpr int kMaxChunk = 512;
template <class T, int RT, bool SUMS, bool ACC, bool NARROW>
__global__ void __launch_bounds__(kSlice, SUMS && RT > 2 ? 2 : 4) slice_kernel(RowMap rows, Factor fac, Sum job,
                                                                              float *__restrict__ hidden) {
  constexpr int kPitch = 68;  // floats of a turned row: reads by columns fall on different banks
  // part products where f32 MFMAs would bind; f16's two parts do not fit the
  // registers beside the sums of more than 16 ranks.  The same with and without
  // SUMS: what dx comes out as does not depend on dup being asked for.
  constexpr bool SPLIT = std::is_same_v<T, BF16> || (std::is_same_v<T, F16> && RT == 1);
  using raw = typename T::raw;
  __shared__ float red[2][kSliceWaves][16][RT * 16 + 1];  // by tile: one barrier each
  __shared__ float4 turn4[SUMS ? kSliceWaves * 16 * kPitch / 4 : 1];
  __shared__ float hs[SUMS ? 2 : 1][16][RT * 16];
  __shared__ int row_s[kMaxChunk], key_s[kMaxChunk];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo = lane & 15, q = lane >> 4;
  const int width = fac.width, own = blockIdx.x * kSlice + wave * 64, j0 = blockIdx.z * RT * 16;
  const int c0 = NARROW ? own : min(own, width - 64), skip = own - c0;
  const int p0 = blockIdx.y * job.chunk, p1 = min(p0 + job.chunk, rows.n);
  const int ranks = min(RT * 16, fac.rank - j0);
  float *turn = (float *)turn4 + (SUMS ? wave * 16 * kPitch : 0);
  float *to_hidden = hidden + (int64_t)blockIdx.x * rows.n * fac.rank + j0;
  for (int i = threadIdx.x; i < p1 - p0; i += kSlice) {
    row_s[i] = rows.row(p0 + i);
    key_s[i] = rows.adapter(p0 + i);
  }
  __syncthreads();
  for (int i0 = p0; i0 < p1;) {
    const int a = __builtin_amdgcn_readfirstlane(key_s[i0 - p0]);
    int i1 = p1;  // the end of a's run here
    for (int step = i0, hi = p1; step < hi;) {
      const int mid = (step + hi) >> 1;
      if (__builtin_amdgcn_readfirstlane(key_s[mid - p0]) == a) step = mid + 1;
      else i1 = hi = mid;
    }
    const int ra = a < rows.count ? fac.rank_of(a) : 0;
    v4f sums[RT][4] = {};
    if (ra > j0) {
      Quad<T> fv[RT][4];     // f32 factors
      uint4 fp[RT][2][2];    // 16-bit ones: the parts of pieces 2 i and 2 i + 1
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const raw *row = (const raw *)fac.p + ((int64_t)a * fac.rank + min(j0 + 16 * t + lo, ra - 1)) * width;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if constexpr (NARROW) fv[t][m] = Quad<T>::load(row, c0 + 16 * m + 4 * q, width);
          else fv[t][m] = Quad<T>::load(row + c0 + 16 * m + 4 * q);
        }
      }
      if (skip > 0) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int m = 0; m < 4; ++m) fv[t][m].drop(skip - (16 * m + 4 * q));
      }
      if constexpr (SPLIT) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) factor_parts(fv[t][2 * i], fv[t][2 * i + 1], fp[t][i]);
      }
      // what a sum's bits, past kSmallSum's, have to be below: all are looked at
      // beside a factor value not below kLargeFactor
      uint32_t fine = (0x7f800000u - kSmallSum) << 1;
      if constexpr (std::is_same_v<T, BF16>) {  // f16's are below
        u16x2 most = 0;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int m = 0; m < 4; ++m)
            most = __builtin_elementwise_max(
                most, __builtin_elementwise_max(__builtin_bit_cast(u16x2, fv[t][m].v.x & 0x7fff7fff),
                                                __builtin_bit_cast(u16x2, fv[t][m].v.y & 0x7fff7fff)));
        if (__any(max(most.x, most.y) >= kLargeFactor)) fine = 0;
      }
      Quad<F32> xv[2][4];
      constexpr int kHidden = (RT * 256 + kSlice - 1) / kSlice;  // a thread's hidden values of a tile
      float hn[kHidden];
      const int tiles = (i1 - i0 + 15) / 16;
      const auto load = [&](int d, int tile) {
        const int p = i0 + 16 * min(tile, tiles - 1);
        const uint32_t *row = (const uint32_t *)job.x + (int64_t)row_s[min(p + lo, i1 - 1) - p0] * job.xstride;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if constexpr (NARROW) xv[d][m] = Quad<F32>::load(row, c0 + 16 * m + 4 * q, width);
          else xv[d][m] = Quad<F32>::load(row + c0 + 4 * q + 16 * m);
        }
        issued();
      };
      const auto load_hidden = [&](int tile) {
        if constexpr (SUMS) {
#pragma unroll
          for (int n = 0; n < kHidden; ++n) {
            const int e = threadIdx.x + n * kSlice, p = i0 + 16 * tile + e / (RT * 16), j = j0 + e % (RT * 16);
            hn[n] = job.hidden[(int64_t)row_s[min(p, i1 - 1) - p0] * fac.rank + min(j, ra - 1)];
          }
          issued();
        }
      };
      const auto store_hidden = [&](int tile) {
        if constexpr (SUMS) {
#pragma unroll
          for (int n = 0; n < kHidden; ++n) {
            const int e = threadIdx.x + n * kSlice;
            if (e < RT * 256)  // no rows past the run
              (&hs[tile & 1][0][0])[e] = i0 + 16 * tile + e / (RT * 16) < i1 ? hn[n] : 0.0f;
          }
        }
      };
      const auto multiply = [&](int d, int tile) {
        const int p = i0 + 16 * tile;
        if (skip > 0) {
#pragma unroll
          for (int m = 0; m < 4; ++m) xv[d][m].drop(skip - (16 * m + 4 * q));
        }
        v4f acc[RT] = {};
        if constexpr (SUMS) {
#pragma unroll
          for (int m = 0; m < 4; ++m) *(uint4 *)(turn + lo * kPitch + 16 * m + 4 * q) = xv[d][m].v;
          // the run's last tile: no rows past it (the first product has them, as without SUMS)
          if (p + 16 > i1 && p + lo >= i1) {
#pragma unroll
            for (int m = 0; m < 4; ++m) *(uint4 *)(turn + lo * kPitch + 16 * m + 4 * q) = make_uint4(0, 0, 0, 0);
          }
        }
        if constexpr (!SPLIT) {
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int m = 0; m < 4; ++m) fv[t][m].pin();
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
              for (int t = 0; t < RT; ++t) acc[t] = mfma(xv[d][m].get(s), fv[t][m].get(s), acc[t]);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint4 v[2] = {xv[d][2 * i].v, xv[d][2 * i + 1].v};
            const uint4 hi = take_part(v), mid = take_part(v), low = take_part(v);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              acc[t] = mfma16(low, fp[t][i][0], acc[t]);
              if constexpr (kParts<T> == 2) acc[t] = mfma16(mid, fp[t][i][1], acc[t]);
              acc[t] = mfma16(mid, fp[t][i][0], acc[t]);
              if constexpr (kParts<T> == 2) acc[t] = mfma16(hi, fp[t][i][1], acc[t]);
              acc[t] = mfma16(hi, fp[t][i][0], acc[t]);
            }
          }
          // outside [kSmallSum, infinity): below it the difference wraps
          uint32_t far = 0;
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) far = max(far, (f2u(acc[t][r]) << 1) - (kSmallSum << 1));
          bool odd = __any(far >= fine);
          if (__builtin_expect(odd, 0)) {
            bool again = past_parts(xv[d][0].v, xv[d][1].v) || past_parts(xv[d][2].v, xv[d][3].v);
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) again = again || !isfinite(acc[t][r]);
            odd = __any(again);
          }
          if (__builtin_expect(odd, 0)) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              acc[t] = v4f{0, 0, 0, 0};
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                uint4 parts[2] = {fp[t][m / 2][0], fp[t][m / 2][1]};
                pin(parts[0]);  // else converted ahead of the loop, in registers of their own
                pin(parts[1]);
#pragma unroll
                for (int s = 0; s < 4; ++s)
                  acc[t] = mfma(xv[d][m].get(s), from_parts<T>(parts, 4 * (m & 1) + s), acc[t]);
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) red[tile & 1][wave][4 * q + r][16 * t + lo] = acc[t][r];
        if constexpr (SUMS) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 v = *(const float4 *)(turn + (4 * r + q) * kPitch + 4 * lo);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              const float h = hs[tile & 1][4 * r + q][16 * t + lo];
#pragma unroll
              for (int m = 0; m < 4; ++m) sums[t][m] = mfma(h, get4(v, m), sums[t][m]);
            }
          }
        }
        store_hidden(tile + 1);
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * RT * 16; e += kSlice) {
          const int i = e / (RT * 16), j = e % (RT * 16);
          float sum = 0.0f;
#pragma unroll
          for (int w = 0; w < kSliceWaves; ++w) sum += red[tile & 1][w][i][j];
          if (p + i < i1 && j < ranks) to_hidden[(int64_t)row_s[p + i - p0] * fac.rank + j] = j0 + j < ra ? sum : 0.0f;
        }
      };
      load_hidden(0);
      load(0, 0);
      store_hidden(0);
      __syncthreads();
      int tile = 0;
      for (; tile + 1 < tiles; tile += 2) {
        load_hidden(tile + 1);
        load(1, tile + 1);
        multiply(0, tile);
        load_hidden(tile + 2);
        load(0, tile + 2);
        multiply(1, tile + 1);
      }
      if (tile < tiles) multiply(0, tile);
    } else {
      for (int e = threadIdx.x; e < (i1 - i0) * ranks; e += kSlice)
        to_hidden[(int64_t)row_s[i0 - p0 + e / ranks] * fac.rank + e % ranks] = 0.0f;
    }
    if constexpr (SUMS) {
      if (a >= rows.count) break;  // rows without an adapter come last
      const bool began = i0 > p0 || p0 == 0 || rows.adapter(p0 - 1) != a;
      const bool goes_on = i1 == p1 && p1 < rows.n && rows.adapter(p1) == a;
      const Cols<NARROW> cols(c0 + 4 * lo, NARROW ? 0 : max(0, skip - 4 * lo), width);
      store_sums<ACC>(sums, fac, a, ra, j0, q, cols, began, goes_on, job);
    }
    i0 = i1;
  }
}

// --------------------------------------------- rank values over a width
// y[row] = base[row] + s_a sum_j hidden[row][j] factor_a[j].  D[i = row][j =
// column]: lane l holds columns 4 (l % 16) + m of its wave's 64 for the m-th
// of four accumulators, so a row's part is stored as 16-byte words; ranks 4
// (l / 16) + s of each 16 for the s-th MFMA.  Block: four waves, 256 columns,
// 16 rows, all of its loads in flight together.  Short blocks that pass the
// rows in launch order keep HBM busier than longer ones with the next rows'
// loads ahead (8192 x 4096 f32 read and written: 64 rows a block 5.3 TB/s, 128
// rows 4.6), and the factor read again by each comes from L2.  bf16 4096 wide,
// rank 32, 8192 rows with a base: 61 us, 268 MB at 4.4 TB/s, about a copy's rate.
template <class T, int RT, bool NARROW, bool NT>
__global__ void __launch_bounds__(256, RT > 2 ? 3 : 4) up_kernel(RowMap rows, Factor fac,
                                                                const float *__restrict__ hidden, const float *base,
                                                                int64_t bstride, float *y, int64_t ystride) {
  using raw = typename T::raw;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lo = lane & 15, q = lane >> 4;
  const int across = (fac.width + 255) / 256;
  const Cols<NARROW> cols(blockIdx.x % across * 256 + wave * 64 + 4 * lo, fac.width);
  const int p0 = blockIdx.x / across * 16, live = min(16, rows.n - p0);
  const int mine = rows.row(p0 + min(lo, live - 1)), key = rows.adapter(p0 + min(lo, live - 1));
  int to[4];  // the rows this lane's accumulators belong to
#pragma unroll
  for (int r = 0; r < 4; ++r) to[r] = __shfl(mine, 4 * q + r);
  Quad<T> fv[RT][4];
  const auto load_factor = [&](int a, int ra, int g) {
    const raw *f = (const raw *)fac.p + (int64_t)a * fac.rank * fac.width;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        fv[t][s] = cols.template load<T>(f + (int64_t)min(g + 16 * t + 4 * q + s, ra - 1) * fac.width);
  };
  float4 hv[RT], bv[4];
  const float *from = hidden + (int64_t)mine * fac.rank;
  const bool whole = fac.rank % 4 == 0;
  const auto load_hidden = [&](int g) {  // zeros past the rank
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int j = g + 16 * t + 4 * q;
      hv[t] = whole ? load4(from + (j < fac.rank ? j : 0), 0, 4) : load4(from, j, fac.rank);
    }
  };
  int a = __builtin_amdgcn_readfirstlane(key), ra = 0;
  float scale = 0.0f;
  const auto begin = [&] {
    ra = a < rows.count ? fac.rank_of(a) : 0;
    scale = a < rows.count ? fac.scale_of(a) : 0.0f;
    if (ra > 0) load_factor(a, ra, 0);
  };
  begin();
  load_hidden(0);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    bv[r] = make_float4(0, 0, 0, 0);
    if (base) bv[r] = cols.load(base + (int64_t)to[r] * bstride);
  }
  issued();
  for (int i0 = 0;;) {
    const uint64_t same = __ballot(lane < live && key == a);
    const int i1 = i0 + __popcll(same >> i0);
    if (ra > 0) {
      v4f acc[4] = {};
      for (int g = 0; g < ra; g += 16 * RT) {
        if (g > 0) {
          load_factor(a, ra, g);
          load_hidden(g);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if (16 * t >= ra - g) break;
          const int j = g + 16 * t + 4 * q;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            // rank rows past the adapter's are not its: zeros on both sides
            const float h = j + s < ra ? get4(hv[t], s) : 0.0f;
            const float4 f = keep4(j + s < ra, fv[t][s].floats());
#pragma unroll
            for (int m = 0; m < 4; ++m) acc[m] = mfma(h, get4(f, m), acc[m]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * q + r >= i0 && 4 * q + r < i1)
          bv[r] = fma4(scale, make_float4(acc[0][r], acc[1][r], acc[2][r], acc[3][r]), bv[r]);
    }
    if (i1 >= live) break;
    const bool again = ra > 16 * RT;  // hv holds a later group
    i0 = i1;
    a = __builtin_amdgcn_readlane(key, i0);
    begin();
    if (again) load_hidden(0);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * q + r < live && cols.any()) cols.template store<NT>(y + (int64_t)to[r] * ystride, bv[r]);
}

// The same for few rows: a block one row's columns, four a thread, the hidden
// values (added up from their splits) from LDS, rank by rank with eight to
// sixteen factor loads ahead.
template <class T, bool NARROW>
__device__ inline void spread_row(const RowMap &rows, const Factor &fac, const Hidden &h, const float *base,
                                  int64_t bstride, float *y, int64_t ystride, float *hsum, int row, int c0,
                                  float (&hs)[kMaxRank]) {
  const int a = rows.adapter(row);
  const Cols<NARROW> cols(c0, fac.width);
  const int ra = a < rows.count ? fac.rank_of(a) : 0;
  const typename T::raw *f = (const typename T::raw *)fac.p + (int64_t)(ra > 0 ? a : 0) * fac.rank * fac.width;
  float4 sum = make_float4(0, 0, 0, 0);
  Quad<T> v[2][8];
  const auto load = [&](Quad<T> (&to)[8], int j0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j] = cols.template load<T>(f + (int64_t)max(min(j0 + j, ra - 1), 0) * fac.width);
    issued();
  };
  if (base && cols.any()) sum = cols.load(base + (int64_t)row * bstride);
  if (ra > 0) load(v[0], 0);
  if ((int)threadIdx.x < fac.rank) {
    const float at = h.at(row, threadIdx.x);
    hs[threadIdx.x] = at;
    if (hsum) hsum[(int64_t)row * fac.rank + threadIdx.x] = at;
  }
  __syncthreads();
  if (ra > 0) {
    float4 acc = make_float4(0, 0, 0, 0);
    const auto add = [&](const Quad<T> (&from)[8], int j0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j0 + j >= ra) break;
        acc = fma4(hs[j0 + j], from[j].floats(), acc);
      }
    };
    for (int j0 = 0; j0 < ra; j0 += 16) {
      load(v[1], j0 + 8);
      add(v[0], j0);
      load(v[0], j0 + 16);
      add(v[1], j0 + 8);
    }
    sum = fma4(fac.scale_of(a), acc, sum);
  }
  if (cols.any()) cols.store(y + (int64_t)row * ystride, sum);
}
template <class T, bool NARROW>
__global__ void __launch_bounds__(256) up_row_kernel(RowMap rows, Factor fac, Hidden h, const float *base,
                                                     int64_t bstride, float *y, int64_t ystride,
                                                     float *__restrict__ hsum) {
  __shared__ float hs[kMaxRank];
  spread_row<T, NARROW>(rows, fac, h, base, bstride, y, ystride, blockIdx.x == 0 ? hsum : nullptr, blockIdx.y,
                        blockIdx.x * 1024 + 4 * threadIdx.x, hs);
}

// ------------------------------------------------ sums over an adapter's rows
// grad_a[j][c] = s_a sum over a's rows of hidden[row][j] x[row][c].  D[i =
// rank][j = column]: a wave 64 columns (as above), four rows an MFMA, DEPTH
// MFMA steps of loads ahead.  A block takes `chunk` positions of the sorted
// rows, half a block's waves every second four of them: long runs keep twice
// the loads in flight.  It serves ddown, and dup where that is asked for alone:
// beside others dup's sums are slice_kernel's.  x of 8192 x 4096, rank 32: 46
// us, 2.9 TB/s; its MFMAs would take 14, the rest waits for loads at three
// waves a SIMD.
template <bool ACC, int RT, bool NARROW>
__global__ void __launch_bounds__(512, RT > 2 ? 2 : 4) outer_kernel(RowMap rows, Factor fac, Sum job) {
  constexpr int DEPTH = RT >= 4 ? 4 : 8;
  __shared__ float4 half_s[RT][4][256];
  // the rows' offsets: a 64-bit product for each load costs as much as its MFMAs
  __shared__ int64_t x_s[kMaxChunk];
  __shared__ int h_s[kMaxChunk], key_s[kMaxChunk];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3);
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), lo = lane & 15, q = lane >> 4;
  const int j0 = blockIdx.z * RT * 16;
  const int width = job.width, chunk = job.chunk, p0 = (int)blockIdx.y * chunk;
  const Cols<NARROW> cols((int)blockIdx.x * 256 + wave * 64 + 4 * lo, width);
  const int p1 = min(p0 + chunk, rows.n);
  for (int i = threadIdx.x; i < p1 - p0; i += 512) {
    const int row = rows.row(p0 + i);
    x_s[i] = row * job.xstride;
    h_s[i] = row * fac.rank;
    key_s[i] = rows.adapter(p0 + i);
  }
  __syncthreads();
  for (int i0 = p0; i0 < p1;) {
    const int a = __builtin_amdgcn_readfirstlane(key_s[i0 - p0]);
    if (a >= rows.count) break;  // rows without an adapter come last
    int i1 = p1;                 // the end of a's run here
    for (int step = i0, hi = p1; step < hi;) {
      const int mid = (step + hi) >> 1;
      if (__builtin_amdgcn_readfirstlane(key_s[mid - p0]) == a) step = mid + 1;
      else i1 = hi = mid;
    }
    const bool began = i0 > p0 || p0 == 0 || rows.adapter(p0 - 1) != a;
    const bool goes_on = i1 == p1 && p1 < rows.n && rows.adapter(p1) == a;
    const int ra = fac.rank_of(a);
    v4f acc[RT][4] = {};
    if (ra > j0) {
      const int steps = (i1 - i0 + 7) / 8;  // of this half, every second four rows
      const float *hcol[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) hcol[t] = job.hidden + min(j0 + 16 * t + lo, ra - 1);
      float4 xv[DEPTH];
      float hv[DEPTH][RT];
      const auto load = [&](int d, int step) {  // rows past the last repeat it
        const int at = min(i0 + 8 * step + 4 * half + q, i1 - 1) - p0;
        xv[d] = cols.load(job.x + x_s[at]);
        const int h = h_s[at];
#pragma unroll
        for (int t = 0; t < RT; ++t) hv[d][t] = hcol[t][h];
        issued();
      };
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) load(d, d);
      for (int step = 0; step < steps; step += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
          if (step + d < steps) {
            if (i0 + 8 * (step + d) + 8 > i1) {  // the run's end: no rows past it
              const bool on = i0 + 8 * (step + d) + 4 * half + q < i1;
              xv[d] = keep4(on, xv[d]);
#pragma unroll
              for (int t = 0; t < RT; ++t) hv[d][t] = on ? hv[d][t] : 0.0f;
            }
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
              for (int m = 0; m < 4; ++m) acc[t][m] = mfma(hv[d][t], get4(xv[d], m), acc[t][m]);
          }
          load(d, step + d + DEPTH);
        }
      }
    }
    // the second half's sums on top of the first's
    if (half == 1)
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          half_s[t][m][threadIdx.x - 256] = make_float4(acc[t][m][0], acc[t][m][1], acc[t][m][2], acc[t][m][3]);
    __syncthreads();
    if (half == 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float4 v = half_s[t][m][threadIdx.x];
          acc[t][m] += v4f{v.x, v.y, v.z, v.w};
        }
      store_sums<ACC>(acc, fac, a, ra, j0, q, cols, began, goes_on, job);
    }
    __syncthreads();
    i0 = i1;
  }
}

// The adapters that no block wrote whole: their partials added up in order,
// zeros for those no row names.
struct Sums {
  Sum of[2];
  int count;
};
// WORDS: 16-byte words a thread, one where the values are few.
template <bool ACC, int WORDS>
__global__ void __launch_bounds__(256) sum_kernel(RowMap rows, Factor fac, Sums sums) {
  const Sum &job = sums.of[blockIdx.z];
  const float *part = job.part;
  const int a = blockIdx.y, chunk = job.chunk, size = fac.rank * job.width;
  if ((int64_t)blockIdx.x * (WORDS * 1024) >= size) return;
  const int2 at = rows_of(rows.key, rows.n, a);
  float *to = job.grad + (int64_t)a * size;
  const int first = at.x / chunk, last = (at.y - 1) / chunk;
  const bool none = at.x == at.y;
  if (none ? ACC : first == last) return;
  const int edge = fac.rank_of(a) * job.width, e0 = blockIdx.x * (WORDS * 1024) + threadIdx.x * 4;
  const float scale = fac.scale_of(a);
  float4 v[WORDS];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) v[i] = make_float4(0, 0, 0, 0);
  if (!none) {
    constexpr int kAhead = 4 / WORDS;  // blocks whose loads are in flight together
    // its first block's rows went on (slot 1), every later one's began earlier
    const auto block = [&](int b) { return part + ((int64_t)b * 2 + (b == first ? 1 : 0)) * size; };
    int b = first;
    for (; b + kAhead - 1 <= last; b += kAhead) {
      float4 w[kAhead][WORDS];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[k][i] = load4(block(b + k), e0 + i * 1024, size);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int i = 0; i < WORDS; ++i) v[i] = add4(v[i], w[k][i]);
    }
    for (; b <= last; ++b)
#pragma unroll
      for (int i = 0; i < WORDS; ++i) v[i] = add4(v[i], load4(block(b), e0 + i * 1024, size));
  }
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    const int e = e0 + i * 1024;
    if (e >= size) break;
    float4 r = make_float4(e < edge ? v[i].x * scale : 0.0f, e + 1 < edge ? v[i].y * scale : 0.0f,
                           e + 2 < edge ? v[i].z * scale : 0.0f, e + 3 < edge ? v[i].w * scale : 0.0f);
    if constexpr (ACC) r = add4(load4(to, e, size), r);
    store4(to, e, size, r);
  }
}

// ------------------------------------------------------ few rows, backward
// Everything that follows from g of few rows, in one launch: blocks that sum
// one adapter's rows into some columns of a gradient (its rows found by a scan
// of all ids, in their order; the terms as in outer_kernel; zeros where no row
// is the adapter's), then blocks that each spread one row's g over 2048 columns
// of dx.  A wave sums 64 columns of 32 rows; `parts` of a block's eight share
// columns and add up in LDS: two where adapters are many, more for long runs of
// few adapters, whose blocks alone would not fill the CUs (f32 2048x8192 rank 8,
// one adapter's 256 rows: two parts 16.7 us, eight 10.0).
constexpr int kFewRows = 2048;       // rows at most
constexpr int kFewAcross = 1 << 20;  // blocks in the grid's x: 2^32 threads at most
struct FewSum {
  Hidden h;
  const float *x;
  int64_t xstride;
  int width, across, first;  // across: blocks along the width; first: blocks before its own
  float *grad;
};
struct FewSums {
  FewSum of[2];
  int count, parts;
  int blocks, total, groups;  // total: with the rows' blocks; groups: of 16 RT ranks
};
template <class T, int RT, bool ACC, bool NARROW>
__global__ void __launch_bounds__(512, RT > 2 ? 2 : 4) few_kernel(RowMap rows, Factor fac, FewSums sums, Hidden g,
                                                                 const float *base, int64_t bstride, float *dx,
                                                                 int64_t dxstride) {
  constexpr int kPitch = RT * 16;
  // the hidden values of 256 rows, later the sums of half the waves
  __shared__ float4 both_s[RT * 1024];
  float *const hs = (float *)both_s;
  __shared__ int list[kFewRows], found[8];
  __shared__ float spread_s[kMaxRank];
  int block = (int)(blockIdx.y * gridDim.x + blockIdx.x);
  if (block >= sums.total) return;
  if (block >= sums.blocks) {
    block -= sums.blocks;
    const int across = (fac.width + 2047) / 2048;
    spread_row<T, NARROW>(rows, fac, g, base, bstride, dx, dxstride, nullptr, block / across,
                          block % across * 2048 + 4 * threadIdx.x, spread_s);
    return;
  }
  const bool second = sums.count > 1 && block >= sums.of[1].first;
  const FewSum &job = sums.of[second ? 1 : 0];
  block -= job.first;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = 8 / sums.parts, part = wave / waves, lo = lane & 15, q = lane >> 4;
  const int a = block / (job.across * sums.groups), j0 = block / job.across % sums.groups * RT * 16;
  const Cols<NARROW> cols((block % job.across * waves + wave % waves) * 64 + 4 * lo, job.width);
  const int ra = fac.rank_of(a);
  int total = 0;
  for (int r0 = 0; r0 < rows.n; r0 += 512) {
    const int row = r0 + threadIdx.x;
    const bool mine = row < rows.n && rows.adapter(row) == a;
    const uint64_t same = __ballot(mine);
    if (lane == 0) found[wave] = __popcll(same);
    __syncthreads();
    int at = total + __popcll(same & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      at += w < wave ? found[w] : 0;
      total += found[w];
    }
    if (mine) list[at] = row;
    __syncthreads();
  }
  if (ACC && total == 0) return;
  v4f acc[RT][4] = {};
  for (int i0 = 0; i0 < total && ra > j0; i0 += 32 * sums.parts) {
    const int h0 = 32 * part;
    const bool any = i0 + h0 < total;
    float4 xv[8];
    if (any) {
#pragma unroll
      for (int d = 0; d < 8; ++d)
        xv[d] = cols.load(job.x + list[min(i0 + h0 + 4 * d + q, total - 1)] * job.xstride);
      issued();
    }
    for (int e = threadIdx.x; e < min(32 * sums.parts, total - i0 + 3) * RT * 4; e += 512) {
      const int i = e / (RT * 4), j = j0 + e % (RT * 4) * 4;
      float4 h = make_float4(0, 0, 0, 0);
      if (i0 + i < total && j < ra) h = job.h.at4(list[i0 + i], j);
      if (j + 4 > ra) h = make_float4(j < ra ? h.x : 0.0f, j + 1 < ra ? h.y : 0.0f, j + 2 < ra ? h.z : 0.0f, 0.0f);
      *(float4 *)(hs + i * kPitch + j - j0) = h;
    }
    __syncthreads();
    if (any) {
      if (i0 + h0 + 32 > total)
#pragma unroll
        for (int d = 0; d < 8; ++d) xv[d] = keep4(i0 + h0 + 4 * d + q < total, xv[d]);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        if (i0 + h0 + 4 * d >= total) break;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int m = 0; m < 4; ++m)
            acc[t][m] = mfma(hs[(h0 + 4 * d + q) * kPitch + 16 * t + lo], get4(xv[d], m), acc[t][m]);
      }
    }
    __syncthreads();
  }
  for (int upper = sums.parts / 2; upper > 0; upper /= 2) {  // the later parts' sums on top of the earlier ones'
    if (total <= 32 * upper) continue;
    const int at = threadIdx.x & (upper * waves * 64 - 1);
    if (part >= upper && part < 2 * upper)
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          both_s[(4 * t + m) * 256 + at] = make_float4(acc[t][m][0], acc[t][m][1], acc[t][m][2], acc[t][m][3]);
    __syncthreads();
    if (part < upper)
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float4 v = both_s[(4 * t + m) * 256 + at];
          acc[t][m] += v4f{v.x, v.y, v.z, v.w};
        }
    __syncthreads();
  }
  if (part == 0) {
    const Sum to{nullptr, nullptr, 0, job.width, 0, job.grad, nullptr};
    store_sums<ACC>(acc, fac, a, ra, j0, q, cols, true, false, to);
  }
}

// ------------------------------------------------------------------ launches
// Few rows: blocks along k where the rows alone leave CUs idle, at least a step
// of each wave.
int splits_of(int n, int width) {
  return std::max(1, std::min({8, 1024 / std::max(1, n), width / (kDownWaves * kStep)}));
}
int slices_of(int width) { return (width + kSlice - 1) / kSlice; }
// Rows of a block of slice_kernel or outer_kernel: as many as leave two blocks
// to every CU, `across` of them along the width.
int chunk_of(int n, int across) {
  const int64_t rows = ((int64_t)n * across + 512 * 16 - 1) / (512 * 16) * 16;
  return (int)std::max<int64_t>(16, std::min<int64_t>(kMaxChunk, rows));
}
// The forward's slices, without sums: about one block to every CU, for each block
// reads its slice of the factor (whole calls with one and with two: bf16
// 4096x11008 rank 32, 2048 rows 56.6 us / 59.4, 8192 rows 211 / 212; 4096x4096
// rank 16, 4100 rows 47.4 / 50.9).
int forward_chunk_of(int n, int across) {
  const int64_t rows = ((int64_t)n * across + 256 * 8) / (256 * 16) * 16;
  return (int)std::max<int64_t>(16, std::min<int64_t>(kMaxChunk, rows));
}
int rank_groups(int rank) { return rank <= 64 ? 1 : (rank + 63) / 64; }

struct Call {
  int32_t dtype;
  RowMap rows;
  hipStream_t s;
  bool accumulate = false;
};

template <class F>
void by_rank(int rank, F &&f) {
  if (rank <= 16) f(std::integral_constant<int, 1>{});
  else if (rank <= 32) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 4>{});
}
template <class F>
void by_flag(bool flag, F &&f) {
  if (flag) f(std::true_type{});
  else f(std::false_type{});
}

hipError_t launch_down_rows(const Call &c, const Factor &fac, const float *x, int64_t xstride, const Hidden &out) {
  const int split_len = (((fac.width + out.splits - 1) / out.splits) + kStep - 1) / kStep * kStep;
  with_type(c.dtype, [&](auto t) {
    using T = decltype(t);
    const auto launch = [&](auto r) {
      constexpr int R = decltype(r)::value;
      const dim3 grid(c.rows.n, out.splits, (fac.rank + R - 1) / R);
      down_row_kernel<T, R><<<grid, kDownWaves * 64, 0, c.s>>>(c.rows, fac, x, xstride, out, split_len);
    };
    constexpr int kMost = sizeof(typename T::raw) == 4 ? 8 : 16;  // two steps' words in registers
    if (fac.rank <= 4) launch(std::integral_constant<int, 4>{});
    else if (fac.rank <= 8) launch(std::integral_constant<int, 8>{});
    else launch(std::integral_constant<int, kMost>{});
  });
  return hipGetLastError();
}

// hidden's slices added up.
__global__ void __launch_bounds__(256) fold_kernel(const float *__restrict__ from, int slices, int64_t size,
                                                   float *__restrict__ to) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= size) return;
  if (e + 4 <= size) {
    float4 v = load4(from + e, 0, 4);
    int s = 1;
    for (; s + 4 <= slices; s += 4) {
      float4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = load4(from + (int64_t)(s + i) * size + e, 0, 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v = add4(v, w[i]);
    }
    for (; s < slices; ++s) v = add4(v, load4(from + (int64_t)s * size + e, 0, 4));
    store4(to + e, v);
  } else {
    for (int64_t i = e; i < size; ++i) {
      float v = from[i];
      for (int s = 1; s < slices; ++s) v += from[(int64_t)s * size + i];
      to[i] = v;
    }
  }
}

// hidden [n][rank] of many rows, and with `sums` the sums of job.
hipError_t launch_slices(const Call &c, const Factor &fac, const Sum &job, bool sums, bool accumulate, float *slices,
                         float *hidden) {
  const int count = slices_of(fac.width);
  float *to = count > 1 ? slices : hidden;
  by_rank(fac.rank, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    const dim3 grid(count, (c.rows.n + job.chunk - 1) / job.chunk, rank_groups(fac.rank));
    with_type(c.dtype, [&](auto t) {
      by_flag(fac.width < 64, [&](auto narrow) {
        constexpr bool N = decltype(narrow)::value;
        if (!sums) slice_kernel<decltype(t), RT, false, false, N><<<grid, kSlice, 0, c.s>>>(c.rows, fac, job, to);
        else if (accumulate) slice_kernel<decltype(t), RT, true, true, N><<<grid, kSlice, 0, c.s>>>(c.rows, fac, job, to);
        else slice_kernel<decltype(t), RT, true, false, N><<<grid, kSlice, 0, c.s>>>(c.rows, fac, job, to);
      });
    });
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || count == 1) return e;
  const int64_t size = (int64_t)c.rows.n * fac.rank;
  fold_kernel<<<(uint32_t)((size + 1023) / 1024), 256, 0, c.s>>>(slices, count, size, hidden);
  return hipGetLastError();
}

// up_kernel's blocks; a launch takes fewer than 2^32 threads.
int64_t up_blocks(int n, int width) { return (int64_t)((width + 255) / 256) * ((n + 15) / 16); }
bool rows_launchable(int n, int width) { return up_blocks(n, width) * 256 <= UINT32_MAX; }
hipError_t launch_up(const Call &c, const Factor &fac, const Hidden &h, const float *base, int64_t bstride, float *y,
                     int64_t ystride, float *hsum) {
  if (c.rows.order == nullptr) {
    const dim3 grid((fac.width + 1023) / 1024, c.rows.n);
    with_type(c.dtype, [&](auto t) {
      by_flag(fac.width < 4, [&](auto narrow) {
        up_row_kernel<decltype(t), decltype(narrow)::value>
            <<<grid, 256, 0, c.s>>>(c.rows, fac, h, base, bstride, y, ystride, hsum);
      });
    });
    return hipGetLastError();
  }
  by_rank(fac.rank, [&](auto rt) {
    const int64_t grid = up_blocks(c.rows.n, fac.width);
    const bool nt = (int64_t)c.rows.n * fac.width * 4 > kKept;
    with_type(c.dtype, [&](auto t) {
      const auto go = [&](auto narrow, auto past) {
        up_kernel<decltype(t), decltype(rt)::value, decltype(narrow)::value, decltype(past)::value>
            <<<(uint32_t)grid, 256, 0, c.s>>>(c.rows, fac, h.p, base, bstride, y, ystride);
      };
      if (fac.width < 4) go(std::true_type{}, std::false_type{});
      else if (nt) go(std::false_type{}, std::true_type{});
      else go(std::false_type{}, std::false_type{});
    });
  });
  return hipGetLastError();
}

// Fills in the sums' blocks; false where all of them are too many for int
// counters (gradients of 2 TB).
bool plan_few(const RowMap &rows, const Factor &fac, bool dx, FewSums *sums) {
  int64_t grid = 0;
  by_rank(fac.rank, [&](auto rt) { sums->groups = (fac.rank + 16 * decltype(rt)::value - 1) / (16 * decltype(rt)::value); });
  const int share = rows.n / rows.count;  // rows of an adapter
  sums->parts = share >= 128 ? 8 : share >= 64 ? 4 : 2;
  for (int i = 0; i < sums->count; ++i) {
    FewSum &job = sums->of[i];
    job.across = (job.width + 512 / sums->parts - 1) / (512 / sums->parts);
    job.first = (int)grid;
    grid += (int64_t)rows.count * sums->groups * job.across;
    if (grid > INT32_MAX - kFewAcross) return false;
  }
  sums->blocks = (int)grid;
  if (dx) grid += (int64_t)rows.n * ((fac.width + 2047) / 2048);
  sums->total = (int)grid;
  return grid <= INT32_MAX - kFewAcross;
}

hipError_t launch_few(const Call &c, const Factor &fac, const FewSums &sums, const Hidden &g, const float *base,
                      int64_t bstride, float *dx, int64_t dxstride) {
  const int grid = sums.total;
  if (grid == 0) return hipSuccess;
  bool narrow = dx && fac.width < 4;
  for (int i = 0; i < sums.count; ++i) narrow = narrow || sums.of[i].width < 4;
  const dim3 blocks((uint32_t)std::min(grid, kFewAcross), (uint32_t)((grid + kFewAcross - 1) / kFewAcross));
  by_rank(fac.rank, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    with_type(c.dtype, [&](auto t) {
      by_flag(c.accumulate, [&](auto acc) {
        by_flag(narrow, [&](auto nar) {
          few_kernel<decltype(t), RT, decltype(acc)::value, decltype(nar)::value>
              <<<blocks, 512, 0, c.s>>>(c.rows, fac, sums, g, base, bstride, dx, dxstride);
        });
      });
    });
  });
  return hipGetLastError();
}

// `outer`: the one of the sums that slice_kernel has not done, if any.
hipError_t launch_sums(const Call &c, const Factor &fac, const Sums &sums, const Sum *outer) {
  int64_t size = 0;
  for (int i = 0; i < sums.count; ++i) size = std::max(size, (int64_t)fac.rank * sums.of[i].width);
  if (outer) by_rank(fac.rank, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    const dim3 grid((outer->width + 255) / 256, (c.rows.n + outer->chunk - 1) / outer->chunk,
                    (fac.rank + 16 * RT - 1) / (16 * RT));
    by_flag(c.accumulate, [&](auto acc) {
      by_flag(outer->width < 4, [&](auto nar) {
        outer_kernel<decltype(acc)::value, RT, decltype(nar)::value><<<grid, 512, 0, c.s>>>(c.rows, fac, *outer);
      });
    });
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const bool wide = size * c.rows.count * sums.count >= (int64_t)4096 * 1024;  // four blocks a CU at four words
  const int per = wide ? 4096 : 1024;
  const dim3 grid((uint32_t)((size + per - 1) / per), c.rows.count, sums.count);
  by_flag(c.accumulate, [&](auto acc) {
    by_flag(wide, [&](auto w) {
      sum_kernel<decltype(acc)::value, decltype(w)::value ? 4 : 1><<<grid, 256, 0, c.s>>>(c.rows, fac, sums);
    });
  });
  return hipGetLastError();
}

// Whether the rows go one by one.  They then read their factors each for
// itself, from the L2s at some 9 TB/s, in two launches; sorted into tiles they
// share them but take four or more, 12 us and a quarter more per rank at
// least.  Forward, rows one by one against tiles (us): f32 1024x1024 rank 4
// n400 8 / 15; bf16 4096x4096 rank 16 n256 12 / 17, n400 18.6 / 18.4; f16
// 4096x11008 rank 64 n96 23 / 28, n256 42 / 34; bf16 8192x8192 rank 128 n64 24 /
// 34, n192 63 / 44.  Backward, where the tiles' launches are six and their sums
// pass through memory: bf16 4096x4096 rank 16 n512 28 / 48; f16 4096x11008 rank
// 64 n64 26 / 72, n400 79 / 104; bf16 8192x8192 rank 128 n64 37 / 79, n256 117 /
// 118, n400 185 / 132.
bool few_rows(const welvet_hip_adapters &d, int n, bool backward) {
  const int64_t bytes = (int64_t)n * d.rank * ((int64_t)d.in + d.out) * tok::float_size(d.dtype);
  const int64_t limit = (75 << 20) + d.rank * (9 << 18);
  return n <= kFewRows && (backward ? bytes / 3 : bytes) <= limit;
}

// The workspace's parts.
struct Sizes {
  size_t order = 0, hidden = 0, one = 0, part[2] = {0, 0};  // hidden: by split or slice; one: added up
  size_t total() const { return order + hidden + one + part[0] + part[1]; }
};
Sizes sizes_of(const welvet_hip_adapters &d, int n, bool backward) {
  Sizes z;
  if (n == 0) return z;
  const size_t one = (size_t)n * d.rank * sizeof(float);
  const int width = backward ? d.out : d.in;
  if (few_rows(d, n, backward)) {
    z.hidden = pad256(splits_of(n, width) * one);
    return z;
  }
  z.order = order_bytes(n);
  z.one = pad256(one);
  if (slices_of(width) > 1) z.hidden = pad256(slices_of(width) * one);
  if (backward) {
    // each factor's sums in blocks of rows; dup's in those of slice_kernel or
    // outer_kernel, whichever is the more
    const int groups = rank_groups(d.rank);
    const auto bytes = [&](int w, int across) {
      const size_t chunk = chunk_of(n, across * groups);
      return pad256((n + chunk - 1) / chunk * 2 * d.rank * (size_t)w * sizeof(float));
    };
    z.part[0] = bytes(d.in, (d.in + 255) / 256);
    z.part[1] = std::max(bytes(d.out, (d.out + 255) / 256), bytes(d.out, slices_of(d.out)));
  }
  return z;
}

// Enough for any batch up to n: few rows have their splits, and blocks of fewer
// rows can be more.
size_t most_bytes(const welvet_hip_adapters &d, int n, bool backward) {
  const size_t row = d.rank * sizeof(float);
  const int width = backward ? d.out : d.in;
  // splits_of(r, width) r for r <= n: the width's splits, up to 1024 blocks, at least one
  const int64_t few = std::min(n, kFewRows);
  size_t most = pad256(std::max<int64_t>(few, std::min<int64_t>(few * splits_of(1, width), 1024)) * row);
  if (few_rows(d, n, backward)) return most;
  Sizes z = sizes_of(d, n, backward);
  if (backward) {
    const int groups = rank_groups(d.rank);
    const auto bytes = [&](int w, int across) {
      size_t chunks = 0;
      for (int c = 16; c <= kMaxChunk; c += 16) {  // the most rows in blocks of c
        const int64_t rows = c == kMaxChunk ? n : std::min<int64_t>(n, (int64_t)c * 512 / (across * groups));
        chunks = std::max<size_t>(chunks, (rows + c - 1) / c);
      }
      return pad256(chunks * 2 * row * w);
    };
    z.part[0] = bytes(d.in, (d.in + 255) / 256);
    z.part[1] = std::max(bytes(d.out, (d.out + 255) / 256), bytes(d.out, slices_of(d.out)));
  }
  return std::max(most, z.total());
}

bool desc_ok(const welvet_hip_adapters *d, int32_t n) {
  return d && n >= 0 && n <= (1 << 23) && (int64_t)n * d->rank <= INT32_MAX && d->count > 0 && d->count <= 65535 &&
         d->rank > 0 && d->rank <= kMaxRank && d->in > 0 && d->out > 0 &&
         (int64_t)d->rank * std::max(d->in, d->out) <= INT32_MAX / 2;
}

}  // namespace
}  // namespace wh

using namespace wh;
using namespace wh::rt;

namespace {
// The checks both directions share; 0 when the call may go on.
welvet_status check_call(const char *what, const welvet_hip_adapters *d, int32_t n, bool pointers) {
  if (!d) return make_status(kInvalid, "%s: invalid argument", what);
  if (!tok::float_type(d->dtype)) return make_status(kUnsupported, "%s: unsupported dtype %d", what, d->dtype);
  if (!desc_ok(d, n) || !pointers || !d->d_down || !d->d_up) return make_status(kInvalid, "%s: invalid argument", what);
  const int size = tok::float_size(d->dtype);
  if (!tok::aligned(d->d_down, size) || !tok::aligned(d->d_up, size) || !tok::aligned(d->d_ranks, 4) ||
      !tok::aligned(d->d_scales, 4))
    return make_status(kInvalid, "%s: device pointers must be aligned to their elements", what);
  return ok();
}
}  // namespace

extern "C" {

welvet_status welvet_hip_adapters_bytes(const welvet_hip_adapters *desc, int32_t n, size_t *bytes) {
  if (desc && !tok::float_type(desc->dtype))
    return make_status(kUnsupported, "adapters: unsupported dtype %d", desc->dtype);
  if (!desc_ok(desc, n) || !bytes) return make_status(kInvalid, "adapters: invalid argument");
  *bytes = n > 0 ? std::max(most_bytes(*desc, n, false), most_bytes(*desc, n, true)) : 0;
  return ok();
}

welvet_status welvet_hip_adapters_forward(const welvet_hip_adapters *desc, const float *d_x, int64_t x_stride,
                                          const int32_t *d_ids, int32_t n, const float *d_base, int64_t base_stride,
                                          float *d_y, int64_t y_stride, float *d_h, void *d_ws, size_t ws_bytes,
                                          void *stream) {
  welvet_status st = check_call("adapters", desc, n, n == 0 || (d_x && d_ids && d_y));
  if (st.code) return st;
  if (x_stride < desc->in || y_stride < desc->out || (d_base && base_stride < desc->out))
    return make_status(kInvalid, "adapters: row stride below its row");
  for (const void *p : {(const void *)d_x, (const void *)d_ids, (const void *)d_base, (const void *)d_y, (const void *)d_h})
    if (!tok::aligned(p, 4)) return make_status(kInvalid, "adapters: device pointers must be aligned to their elements");
  if (!rows_launchable(n, desc->out)) return make_status(kInvalid, "adapters: more than a launch takes");
  const Sizes z = sizes_of(*desc, n, false);
  if (z.total() > 0 && (!d_ws || ws_bytes < z.total() || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "adapters: %zu bytes of 16-byte aligned workspace are needed", z.total());
  st = require_device();
  if (st.code || n == 0) return st;
  Call c{desc->dtype, {d_ids, nullptr, n, desc->count}, (hipStream_t)stream};
  const Factor down{desc->d_down, desc->d_ranks, desc->d_scales, desc->rank, desc->in};
  const Factor up{desc->d_up, desc->d_ranks, desc->d_scales, desc->rank, desc->out};
  if (few_rows(*desc, n, false)) {
    Hidden h{(float *)d_ws, splits_of(n, desc->in), n, desc->rank};
    if (h.splits == 1 && d_h) h.p = d_h;
    WH_HIP(launch_down_rows(c, down, d_x, x_stride, h));
    WH_HIP(launch_up(c, up, h, d_base, base_stride, d_y, y_stride, h.p == d_h ? nullptr : d_h));
    return ok();
  }
  tok::Order o;
  char *at = (char *)d_ws;
  WH_HIP(tok::launch_order(d_ids, n, desc->count, at, &o, c.s));
  c.rows = {o.skey, o.order, n, desc->count};
  at += z.order;
  float *one = d_h ? d_h : (float *)at, *slices = (float *)(at + z.one);
  const int chunk = forward_chunk_of(n, slices_of(desc->in) * rank_groups(desc->rank));
  const Sum job{nullptr, d_x, x_stride, desc->in, chunk, nullptr, nullptr};
  WH_HIP(launch_slices(c, down, job, false, false, slices, one));
  WH_HIP(launch_up(c, up, Hidden{one, 1, n, desc->rank}, d_base, base_stride, d_y, y_stride, nullptr));
  return ok();
}

welvet_status welvet_hip_adapters_backward(const welvet_hip_adapters *desc, const float *d_x, int64_t x_stride,
                                           const int32_t *d_ids, int32_t n, const float *d_h, const float *d_dy,
                                           int64_t dy_stride, const float *d_dx_base, int64_t dx_base_stride,
                                           float *d_dx, int64_t dx_stride, int32_t accumulate, float *d_ddown,
                                           float *d_dup, void *d_ws, size_t ws_bytes, void *stream) {
  welvet_status st = check_call("adapters backward", desc, n,
                                (d_dx || d_ddown || d_dup) &&
                                    (n == 0 || (d_ids && d_dy && (d_x || !d_ddown) && (d_h || !d_dup))));
  if (st.code) return st;
  if (dy_stride < desc->out || (d_ddown && x_stride < desc->in) || (d_dx && dx_stride < desc->in) ||
      (d_dx && d_dx_base && dx_base_stride < desc->in))
    return make_status(kInvalid, "adapters backward: row stride below its row");
  for (const void *p : {(const void *)d_x, (const void *)d_ids, (const void *)d_h, (const void *)d_dy,
                        (const void *)d_dx_base, (const void *)d_dx, (const void *)d_ddown, (const void *)d_dup})
    if (!tok::aligned(p, 4))
      return make_status(kInvalid, "adapters backward: device pointers must be aligned to their elements");
  const Sizes z = sizes_of(*desc, n, true);
  if (z.total() > 0 && (!d_ws || ws_bytes < z.total() || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "adapters backward: %zu bytes of 16-byte aligned workspace are needed", z.total());
  Call c{desc->dtype, {d_ids, nullptr, n, desc->count}, (hipStream_t)stream, accumulate != 0};
  const Factor down{desc->d_down, desc->d_ranks, desc->d_scales, desc->rank, desc->in};
  const Factor up{desc->d_up, desc->d_ranks, desc->d_scales, desc->rank, desc->out};
  const bool few = few_rows(*desc, n, true);
  const Hidden few_g{(float *)d_ws, few && n > 0 ? splits_of(n, desc->out) : 1, n, desc->rank};
  FewSums few_sums{};
  if (d_ddown) few_sums.of[few_sums.count++] = {few_g, d_x, x_stride, desc->in, 0, 0, d_ddown};
  if (d_dup) few_sums.of[few_sums.count++] = {{const_cast<float *>(d_h), 1, n, desc->rank}, d_dy, dy_stride, desc->out, 0, 0, d_dup};
  if (few ? !plan_few(c.rows, down, d_dx != nullptr, &few_sums) : d_dx && !rows_launchable(n, desc->in))
    return make_status(kInvalid, "adapters backward: more than a launch takes");
  st = require_device();
  if (st.code) return st;
  if (few) {
    if (n > 0 && (d_dx || d_ddown)) WH_HIP(launch_down_rows(c, up, d_dy, dy_stride, few_g));
    WH_HIP(launch_few(c, down, few_sums, few_g, d_dx_base, dx_base_stride, d_dx, dx_stride));
    return ok();
  }
  char *at = (char *)d_ws;
  float *const g = (float *)(at + z.order), *const slices = (float *)(at + z.order + z.one);
  float *const part = (float *)(at + z.order + z.one + z.hidden), *const part2 = (float *)((char *)part + z.part[0]);
  const int groups = rank_groups(desc->rank);
  const bool need_g = d_dx || d_ddown, fused = need_g && d_dup;
  const auto sum_of = [&](const float *hidden, const float *x, int64_t stride, int width, float *grad, float *part, bool slice) {
    const int across = slice ? slices_of(width) : (width + 255) / 256;
    return Sum{hidden, x, stride, width, chunk_of(n, across * groups), grad, part};
  };
  const Sum dup = sum_of(d_h, d_dy, dy_stride, desc->out, d_dup, part2, need_g);
  tok::Order o;
  WH_HIP(tok::launch_order(d_ids, n, desc->count, at, &o, c.s));
  c.rows.key = o.skey;
  c.rows.order = o.order;
  if (need_g) WH_HIP(launch_slices(c, up, dup, fused, c.accumulate, slices, g));
  if (d_dx)
    WH_HIP(launch_up(c, down, Hidden{g, 1, n, desc->rank}, d_dx_base, dx_base_stride, d_dx, dx_stride, nullptr));
  Sums sums{};
  if (d_ddown) sums.of[sums.count++] = sum_of(g, d_x, x_stride, desc->in, d_ddown, part, false);
  if (d_dup) sums.of[sums.count++] = dup;
  // ddown, or dup alone; the slices have done dup beside dx, with no ddown
  const Sum *outer = d_ddown || !fused ? &sums.of[0] : nullptr;
  if (sums.count) WH_HIP(launch_sums(c, down, sums, outer));
  return ok();
}

}  // extern "C"
