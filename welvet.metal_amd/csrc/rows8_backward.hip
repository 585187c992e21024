// rows8_backward.hip — the backward of a layer from activations kept in 8 bits
// (rows8.hpp): with pre = p_t c the pre-activations and x = s_t c the input,
//   dpre = dy act'(pre);  dw = dpre^T x;  dx = dpre W
// Both products run on the f16 matrix cores: codes are exact in f16, and what
// is left of each term, dpre s_t (dw) or dpre v_o (dx, W = v_o w), becomes f16
// parts.  So that f16's range holds them, a channel's (dw) or token's (dx)
// terms are multiplied by the power of two that brings a bound of theirs, max
// |dy| s_t or |dy| v_o times what |act'| can be, to 2^14..2^15: two parts keep
// 22 bits of a term, or 2^-39 of the bound where that is more; the product's
// epilogue divides by it, exactly.  (Three bf16 parts need no bound and half as
// many instructions again.)
//
// Three steps: the codes' images with the sum along their rows, and the
// bounds; dpre and its parts from one pass over dy (dw's transposed); the
// products, which read nothing but whole stages of f16.  bf16 4096 -> 11008 of 8192
// rows: 92 and 232 to 258 us, at 4.4 and 4.5 to 5 TB/s, and 1304 to 1340 and 1203 to 1216
// for dw and dx, 1.1 and 1.2 PFLOP/s of parts, where a library's f16 product reaches 1.5.  f32 2048 ->
// 8192 of 256 rows: 14, 13.5 and 46 in one launch, with 5 to join dx's parts.
#include <hip/hip_runtime.h>

#include <cmath>

#include "rows8.hpp"
#include "int8.hpp"
#include "tiles.hpp"

namespace wh {
namespace {

using namespace r8;
using namespace tiles;

constexpr int kMaxSize = 1 << 20;
__host__ __device__ constexpr int tiles_of(int64_t n, int tile) { return (int)((n + tile - 1) / tile); }
constexpr int kThreads = 512, kRows = 128, kCols = 64;    // of the passes' blocks: 128 x 64 values
constexpr int kBoundCols = 512, kBoundRows = 32;          // of dy a block of the bounds
// ... the rows in whole steps, so that no more than 16 blocks take them, or 128 with
// the columns' together (us of the pass, bf16 5267 rows, 448 channels: 16 of them 34,
// 83 12).
int most_bounds(int64_t out) { return std::max(16, 128 / tiles_of(out, kBoundCols)); }
int bound_rows(int64_t n, int64_t out) { return tiles_of(n, most_bounds(out) * kBoundRows) * kBoundRows; }
int64_t along(int64_t n) { return spread(2 * n) / 2; }    // values between an image's rows

__device__ inline uint16_t half_bits(float v) { return F16::put(v); }
// v as f16 parts, each the rest's nearest; what is not finite is its first part alone.
// One part, 11 bits, is not enough for any type: terms that cancel leave its rounding,
// 2^-12 of the largest, in their sum.
constexpr int kParts = 2;
__device__ inline void split(float v, uint16_t (&part)[kParts]) {
  part[0] = half_bits(v);
  part[1] = fabsf(v) < 65504.0f ? half_bits(v - F16::get(part[0])) : (uint16_t)0;
}

// A block's values, two rows a word, so that columns can be read as rows.  A column's
// sixteen bytes k lie at k ^ 2 (column / 8): a wave's words, eight columns apart, and
// sixteen lanes' reads of a column both touch all of LDS's banks once.
struct Turn {
  static_assert(kRows == 128 && kCols == 64, "sixteen times sixteen bytes a column, eight eights of columns");
  uint32_t word[kCols][kRows / 2];
  __device__ static inline int place(int col, int pair) { return pair ^ (col >> 3) * 8; }
  __device__ inline void put(int col, int pair, uint32_t v) { word[col][place(col, pair)] = v; }
  // Sixteen bytes (eight rows) of a column a thread into the image [cols][pitch]:
  // rows from `row` on (an image's rows hold whole blocks), columns from `col` on.
  __device__ inline void write(uint16_t *image, int64_t pitch, int row, int col, int cols) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = (threadIdx.x >> 4) + kCols / 2 * k, at = (threadIdx.x & 15) * 4;
      if (col + c < cols)
        *(uint4 *)(image + (int64_t)(col + c) * pitch + row + 2 * at) = *(const uint4 *)&word[c][place(c, at)];
    }
  }
};

// Codes [rows][stride] -> f16 [width][pitch], the rows' numbers along it.
struct Image {
  const int8_t *codes;
  int64_t stride, pitch;
  int rows, width, across;
  uint16_t *to;
  int blocks;
  __device__ inline void make(int block, Turn &turn) const {
    const int row = block / across * kRows, col = block % across * kCols;
    const int pair = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;
    uint2 w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = row + 2 * pair + k;
      w[k] = r < rows && col + c < width ? *(const uint2 *)(codes + (int64_t)r * stride + col + c) : make_uint2(0, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      turn.put(c + i, pair, half_bits(value_of(i < 4 ? w[0].x : w[0].y, i & 3)) |
                                ((uint32_t)half_bits(value_of(i < 4 ? w[1].x : w[1].y, i & 3)) << 16));
    __syncthreads();
    turn.write(to, pitch, row, col, width);
  }
};

struct GradArgs {
  const void *dy;
  int64_t dy_stride;
  const int8_t *pre;  // null: Linear
  int64_t pre_stride;
  const float *pre_scales;
  const float *x_scales, *w_scales;  // null: no dw, no dx
  void *dpre;
  int64_t dpre_stride;
  uint16_t *along_n, *along_o;  // dw's parts [kParts][out][n_pitch], dx's [kParts][n][o_pitch]
  int64_t n_pitch, o_pitch;
  uint32_t *col_bound, *row_bound;  // [row blocks][out] of |dy| s_t, [column blocks][n] of |dy| v_o
  float *col_back, *row_back;       // the powers of two that the products are divided by, inverted
  int n, out, act, across;
  int bound_rows, col_parts, row_parts;  // a block's rows, bounds a channel and a token
};
// What |act'| can be, of ReLU2 at a row's pre-activations.
__device__ inline float steepest(const GradArgs &a) { return a.act == kSilu || a.act == kGELU ? 1.25f : 1.0f; }
__device__ inline float steepest(const GradArgs &a, int row) {
  return a.act == kReLU2 ? 256.0f * a.pre_scales[row] : steepest(a);
}
__device__ inline uint32_t finite_bits(float v) { return magnitude(v) < 0x7f800000u ? magnitude(v) : 0; }
// 2^k that brings a bound to 2^14..2^15.
__device__ inline float lift_of(uint32_t bound) {
  const int e = (int)(bound >> 23) - 127;
  return bound == 0 ? 1.0f : u2f((uint32_t)(min(max(14 - e, -126), 126) + 127) << 23);
}

// Bounds of a block's rows and columns; a wave takes four rows of a step, a lane
// eight of the columns.
template <class T, bool EIGHTS>
__device__ inline void bounds(const GradArgs &a, int block, uint32_t *lds) {
  using raw = typename T::raw;
  constexpr int kAhead = kBoundRows / (kThreads / 64);
  const int bm = block / a.row_parts, bn = block % a.row_parts;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = bn * kBoundCols + lane * 8, end = min((bm + 1) * a.bound_rows, a.n);
  // loads without a condition: what there is no scale for reads another's and leaves it
  const bool dw = a.x_scales, dx = a.w_scales, square = a.act == kReLU2;
  const float *xs = dw ? a.x_scales : a.row_back, *ps = square ? a.pre_scales : a.row_back;
  const float *ws = dx ? a.w_scales : a.col_back;
  uint32_t top[8] = {};
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = ws[min(c + i, a.out - 1)];
    v[i] = dx && c + i < a.out ? w : 0.0f;
  }
  for (int r0 = bm * a.bound_rows + wave * kAhead; r0 < end; r0 += kBoundRows) {
    Oct<T> o[kAhead];
    float s[kAhead], steep[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int r = min(r0 + j, end - 1);  // the last row again changes nothing
      const raw *dy = (const raw *)a.dy + (int64_t)r * a.dy_stride;
      // in whole eights a lane past the last column has the last ones again: they change nothing
      if constexpr (EIGHTS) o[j].load(dy + min(c, a.out - 8));
      else o[j].load(dy, min(c, a.out), a.out);
      steep[j] = square ? 256.0f * ps[r] : steepest(a);
      s[j] = dw ? xs[r] * steep[j] : 0.0f;
    }
    uint32_t most[kAhead] = {};
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = o[j].get(i);
        top[i] = max(top[i], finite_bits(d * s[j]));
        most[j] = max(most[j], finite_bits(d * (v[i] * steep[j])));
      }
    if (dx) {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1)
#pragma unroll
        for (int j = 0; j < kAhead; ++j) most[j] = max(most[j], (uint32_t)__shfl_xor((int)most[j], off));
      uint32_t own = most[0];
#pragma unroll
      for (int j = 1; j < kAhead; ++j) own = lane == j ? most[j] : own;
      if (lane < kAhead && r0 + lane < end) a.row_bound[(int64_t)bn * a.n + r0 + lane] = own;
    }
  }
  if (!dw) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) lds[wave * kBoundCols + i * 64 + (lane ^ i * 8)] = top[i];  // a bank a lane, below too
  __syncthreads();
  const int i = threadIdx.x, at = (i & 7) * 64 + (i >> 3 ^ (i & 7) * 8);
  uint32_t most = lds[at];
#pragma unroll
  for (int k = 1; k < kThreads / 64; ++k) most = max(most, lds[k * kBoundCols + at]);
  if (bn * kBoundCols + i < a.out) a.col_bound[(int64_t)bm * a.out + bn * kBoundCols + i] = most;
}
static_assert(kBoundCols == kThreads, "a thread a column at the end");

template <class T>
__global__ void __launch_bounds__(kThreads, 6) prepare_kernel(Image x, Image w, GradArgs a) {
  __shared__ __attribute__((aligned(16))) Turn turn;
  static_assert(sizeof(Turn) >= kThreads / 64 * kBoundCols * 4, "the bounds' place");
  int block = blockIdx.x;
  const int of_dy = a.col_parts * a.row_parts;
  if (block < of_dy) {
    if (a.out % 8 == 0) return bounds<T, true>(a, block, &turn.word[0][0]);
    return bounds<T, false>(a, block, &turn.word[0][0]);
  }
  block -= of_dy;
  if (block < x.blocks) return x.make(block, turn);
  w.make(block - x.blocks, turn);
}

// Many bounds a channel or token into their first.
__global__ void __launch_bounds__(256) fold_kernel(GradArgs a) {
  int i = (int)blockIdx.x * 256 + threadIdx.x;
  const auto fold = [](uint32_t *bound, int parts, int all, int at) {
    uint32_t top = 0;
    for (int p = 0; p < parts; p += 8)
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, bound[(int64_t)min(p + k, parts - 1) * all + at]);
    bound[at] = top;
  };
  if (a.along_n) {
    if (i < a.out) return fold(a.col_bound, a.col_parts, a.out, i);
    i -= a.out;
  }
  if (a.along_o && i < a.n) fold(a.row_bound, a.row_parts, a.n, i);
}

// Powers of two of this block's COUNT rows or columns into `lift`, from `parts`
// bounds each.
template <int COUNT>
__device__ inline void lifts(const uint32_t *bound, int parts, int first, int all, float *back, uint32_t *lds,
                             float *lift) {
  constexpr int kSide = kThreads / COUNT;
  const int i = threadIdx.x % COUNT, part = threadIdx.x / COUNT;
  uint32_t top = 0;
  if (first + i < all)
    for (int p = part; p < parts; p += kSide) top = max(top, bound[(int64_t)p * all + first + i]);
  lds[threadIdx.x] = top;
  __syncthreads();
  if (part == 0) {
#pragma unroll
    for (int k = 1; k < kSide; ++k) top = max(top, lds[k * COUNT + i]);
    const float l = lift_of(top);
    lift[i] = l;
    if (back && first + i < all) back[first + i] = 1.0f / l;
  }
  __syncthreads();
}

// The same of one block of rows without dx, whose columns' bounds lie in the block
// itself: the same products, so that dw has the same bits either way.
template <class T>
__device__ inline void own_lifts(const GradArgs &a, const Oct<T> (&o)[2], int pair, int c, int col, uint32_t *lds,
                                 float *lift) {
  uint32_t top[8] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = 2 * pair + k;
    const float s = r < a.n ? a.x_scales[r] * steepest(a, r) : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top[i] = max(top[i], finite_bits(o[k].get(i) * s));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int off = 8; off < 64; off <<= 1) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], off));
  if ((threadIdx.x & 63) < 8)
#pragma unroll
    for (int i = 0; i < 8; ++i) lds[(threadIdx.x >> 6) * kCols + c - col + i] = top[i];
  __syncthreads();
  if (threadIdx.x < kCols) {
    uint32_t most = lds[threadIdx.x];
#pragma unroll
    for (int k = 1; k < kThreads / 64; ++k) most = max(most, lds[k * kCols + threadIdx.x]);
    const float l = lift_of(most);
    lift[threadIdx.x] = l;
    if (col + (int)threadIdx.x < a.out) a.col_back[col + threadIdx.x] = 1.0f / l;
  }
  __syncthreads();
}

// dpre and its parts.  ONE: a single block of rows without dx; the first blocks
// make the image of the input's codes.
template <class T, bool ONE>
__global__ void __launch_bounds__(kThreads) grad_kernel(Image image, GradArgs a) {
  using raw = typename T::raw;
  __shared__ __attribute__((aligned(16))) Turn turn[kParts];
  __shared__ float lift_n[kRows], lift_o[kCols];
  int block = blockIdx.x;
  if constexpr (ONE) {
    if (block < image.blocks) return image.make(block, turn[0]);
    block -= image.blocks;
  }
  const int row = block / a.across * kRows, col = block % a.across * kCols;
  const int pair = threadIdx.x >> 3, c = col + (threadIdx.x & 7) * 8;
  float v[2][8], s[2] = {0, 0};
  Oct<T> o[2];
  uint2 w[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = row + 2 * pair + k;
    if (a.out % 8 == 0)  // what lies past the last row or column is not used
      o[k].load((const raw *)a.dy + (int64_t)min(r, a.n - 1) * a.dy_stride + min(c, a.out - 8));
    else
      o[k].load((const raw *)a.dy + (int64_t)min(r, a.n - 1) * a.dy_stride, min(c, a.out), a.out);
    if (a.pre) w[k] = *(const uint2 *)(a.pre + (int64_t)min(r, a.n - 1) * a.pre_stride + min(c, (a.out - 1) / 8 * 8));
  }
  uint32_t *lds = &turn[0].word[0][0];
  if constexpr (ONE) own_lifts(a, o, pair, c, col, lds, lift_o);
  if (!ONE && a.along_n)
    lifts<kCols>(a.col_bound, a.col_parts, col, a.out, row == 0 ? a.col_back : nullptr, lds, lift_o);
  if (!ONE && a.along_o)
    lifts<kRows>(a.row_bound, a.row_parts, row, a.n, col == 0 ? a.row_back : nullptr, lds, lift_n);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = row + 2 * pair + k;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[k][i] = o[k].get(i);
    if (r >= a.n || c >= a.out) continue;
    if (a.x_scales) s[k] = a.x_scales[r];
    if (a.pre) {
      const float p = a.pre_scales[r];
      float prime[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) prime[i] = value_of(i < 4 ? w[k].x : w[k].y, i & 3) * p;
      prime8(prime, a.act);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = c + i < a.out ? v[k][i] * prime[i] : 0.0f;
    }
    if (a.dpre) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[k].set(i, v[k][i]);
      o[k].store((raw *)a.dpre + (int64_t)r * a.dpre_stride, c, a.out);
    }
  }
  if (!ONE && a.along_o) {
    float scale[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) scale[i] = c + i < a.out ? a.w_scales[c + i] : 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = row + 2 * pair + k;
      if (r >= a.n) continue;
      const float lift = lift_n[2 * pair + k];
      uint32_t word[kParts][4] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint16_t part[kParts];
        split(c + i < a.out ? v[k][i] * scale[i] * lift : 0.0f, part);
#pragma unroll
        for (int p = 0; p < kParts; ++p) word[p][i >> 1] |= (uint32_t)part[p] << (16 * (i & 1));
      }
#pragma unroll
      for (int p = 0; p < kParts; ++p)
        *(uint4 *)(a.along_o + ((int64_t)p * a.n + r) * a.o_pitch + c) =
            make_uint4(word[p][0], word[p][1], word[p][2], word[p][3]);
    }
  }
  if (a.along_n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint16_t lo[kParts], hi[kParts];
      const float lift = lift_o[c - col + i];
      // rows past the last are nothing, whatever 0 times their values would be
      split(row + 2 * pair < a.n ? v[0][i] * s[0] * lift : 0.0f, lo);
      split(row + 2 * pair + 1 < a.n ? v[1][i] * s[1] * lift : 0.0f, hi);
#pragma unroll
      for (int p = 0; p < kParts; ++p) turn[p].put(c - col + i, pair, lo[p] | ((uint32_t)hi[p] << 16));
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      turn[p].write(a.along_n + (int64_t)p * a.out * a.n_pitch, a.n_pitch, row, col, a.out);
  }
}

// dw over no rows.
__global__ void __launch_bounds__(256) zero_kernel(float *to, int64_t all) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) to[i] = 0.0f;
}

// ---------------------------------------------------------------- products
// Eight results of a row from column c on.
template <class T, bool ADD>
__device__ inline void put8(typename T::raw *to, int c, int cols, const float (&v)[8], float back) {
  Oct<T> o;
  if constexpr (ADD) o.load(to, c, cols);
#pragma unroll
  for (int i = 0; i < 8; ++i) o.set(i, ADD ? o.get(i) + v[i] * back : v[i] * back);
  o.store(to, c, cols);
}
template <class T>
struct Product {  // to[a_rows][b_rows] = back . A . B^T
  Operands g;
  const float *back;
  typename T::raw *to;
  int64_t stride;
  Splits p;
  int tiles_m, tiles_n;
  int blocks() const { return tiles_m * tiles_n * p.splits; }
};
template <class T, bool ADD, class Tile>
__device__ inline void half_tile(const Product<T> &q, int block, bool part, char *lds) {
  const Operands &g = q.g;
  const int tile = part ? block / q.p.splits : block, split = part ? block % q.p.splits : 0;
  const Place at = place(tile, q.tiles_m, q.tiles_n);
  const int m0 = at.m * Tile::kRows, n0 = at.n * Tile::kCols;
  typename Tile::Acc acc[Tile::kTM][Tile::kTN] = {};
  Tile::run(part ? g.part(split * q.p.each, min(q.p.each, g.stages - split * q.p.each)) : g, m0, n0, acc, lds);
  __syncthreads();
  if (part) {
    Tile::template results<4>(m0, n0, acc, lds, [&](int row, int c, const float (&v)[4]) {
      if (row < g.a_rows && c < g.b_rows)
        store4((float *)q.p.parts + split * q.p.parts_values + (int64_t)row * g.b_rows, c, g.b_rows,
               make_float4(v[0], v[1], v[2], v[3]));
    });
    return;
  }
  float *backs = (float *)(lds + Tile::kResults);
  for (int i = threadIdx.x; i < Tile::kRows; i += Tile::kWaves * 64) backs[i] = q.back[min(m0 + i, g.a_rows - 1)];
  __syncthreads();
  if constexpr (std::is_same_v<T, F32>) {
    Tile::template results<4>(m0, n0, acc, lds, [&](int row, int c, const float (&v)[4]) {
      if (row >= g.a_rows || c >= g.b_rows) return;
      float *into = (float *)q.to + row * q.stride;
      float4 sum = mul4(make_float4(v[0], v[1], v[2], v[3]), backs[row - m0]);
      if (ADD) sum = add4(load4(into, c, g.b_rows), sum);
      store4(into, c, g.b_rows, sum);
    });
  } else {
    Tile::template results<8>(m0, n0, acc, lds, [&](int row, int c, const float (&v)[8]) {
      if (row < g.a_rows && c < g.b_rows) put8<T, ADD>(q.to + row * q.stride, c, g.b_rows, v, backs[row - m0]);
    });
  }
}
template <class T, bool ADD, class Tile, bool PART>
__global__ void __launch_bounds__(Tile::kWaves * 64) half_tile_kernel(Product<T> q) {
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  half_tile<T, ADD, Tile>(q, blockIdx.x, PART, lds);
}
// dx's blocks, whose sums are long, then dw's.
template <class T, bool ADD, class Tile>
__global__ void __launch_bounds__(Tile::kWaves * 64) half_pair_kernel(Product<T> x, Product<F32> w, int of_x) {
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  if ((int)blockIdx.x < of_x) return half_tile<T, false, Tile>(x, blockIdx.x, x.p.splits > 1, lds);
  half_tile<F32, ADD, Tile>(w, blockIdx.x - of_x, w.p.splits > 1, lds);
}
// The parts' results in their order; back null: 1.
template <class T, bool ADD>
__global__ void __launch_bounds__(256) half_join_kernel(Splits p, const float *__restrict__ back, typename T::raw *to,
                                                        int64_t stride, int rows, int cols, int per_row) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int row = (int)(i / per_row), c = (int)(i % per_row) * 8;
  if (row >= rows) return;
  const uint32_t *at = (const uint32_t *)p.parts + (int64_t)row * cols;
  float sum[8] = {};
  for (int k = 0; k < p.splits; k += 4) {
    Oct<F32> v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n].load(at + min(k + n, p.splits - 1) * p.parts_values, c, cols);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] = k + n < p.splits ? sum[j] + v[n].get(j) : sum[j];
  }
  put8<T, ADD>(to + row * stride, c, cols, sum, back ? back[row] : 1.0f);
}

// --------------------------------------------------------------- few rows
// Up to kFew rows: dw is as many outer products, bound by its own bytes, dx as
// many rows times the codes as they lie, bound by those; both in f32, from dy
// itself, in one launch.  (The way above makes an image of the codes first, two bytes
// written and read again a weight.  f16 8320 -> 8034, all outputs with the stores, 2
// rows 185 us that way and 68 this, 56 of them dw's and the codes' 334 MB, 6 TB/s; 8
// rows 180 and 76; bf16 2048 -> 2048, 8 rows 42 and 25.5.  Sixteen rows, dx in two
// launches of eight: 42 that way and 56.)
constexpr int kFew = 8;

// dpre, unrounded.
template <class T>
__device__ inline float dpre_of(const GradArgs &a, int t, int o) {
  const float dy = T::get(((const typename T::raw *)a.dy)[(int64_t)t * a.dy_stride + o]);
  return a.pre ? dy * act_prime_f32((float)a.pre[(int64_t)t * a.pre_stride + o] * a.pre_scales[t], a.act) : dy;
}

struct FewArgs {
  const int8_t *x;  // the input's codes
  int64_t x_stride;
  float *dw;
  const int8_t *w;  // the layer's
  int64_t pitch;
  void *dx;
  int64_t dx_stride;
  float *parts;  // of dx, null: whole
  int in, dw_chunks, dx_chunks, dx_blocks, each;
};
constexpr int kDwRows = 32, kDwCols = 1024, kDxCols = 512, kDxRows = 512;
template <int N>
union FewLds {
  float dpre[kDwRows][N];
  struct {
    float terms[kDxRows][N], sums[kThreads / 64][kDxCols];
  } dx;
};

// A block takes 1024 columns of 32 channels, a thread four columns of sixteen, all
// rows; the first columns' block has dpre stored.
template <class T, int N, bool ADD, bool NT>
__device__ inline void dw_few(const GradArgs &a, const FewArgs &f, int block, float (&g)[kDwRows][N]) {
  const int first = block / f.dw_chunks * kDwRows, c = block % f.dw_chunks * kDwCols + (threadIdx.x & 255) * 4;
  const int last = (f.in + kPad - 1) / kPad * kPad - 4;
  float v[N][4];
#pragma unroll
  for (int t = 0; t < N; ++t) {
    const int r = min(t, a.n - 1);
    const uint32_t w = *(const uint32_t *)(f.x + r * f.x_stride + min(c, last));
    const float s = a.x_scales[r];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[t][j] = t < a.n ? value_of(w, j) * s : 0.0f;
  }
  if (threadIdx.x < kDwRows * N) {
    const int o = first + (int)threadIdx.x % kDwRows, t = threadIdx.x / kDwRows;
    const bool there = o < a.out && t < a.n;
    const float d = there ? dpre_of<T>(a, t, o) : 0.0f;
    g[threadIdx.x % kDwRows][t] = d;
    if (a.dpre && there && block % f.dw_chunks == 0)
      ((typename T::raw *)a.dpre)[t * a.dpre_stride + o] = T::put(d);
  }
  __syncthreads();
  if (c >= f.in) return;
#pragma unroll 4
  for (int k = 0; k < kDwRows / 2; ++k) {
    const int r = (threadIdx.x >> 8) * (kDwRows / 2) + k;
    if (first + r >= a.out) break;
    float *to = f.dw + (int64_t)(first + r) * f.in;
    const float4 was = ADD ? load4(to, c, f.in) : make_float4(0, 0, 0, 0);
    float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < N; ++t) sum = fma4(g[r][t], make_float4(v[t][0], v[t][1], v[t][2], v[t][3]), sum);
    if (ADD) sum = add4(was, sum);
    if (NT && c + 4 <= f.in) store4_nt(to + c, sum);
    else store4(to, c, f.in, sum);
  }
}
static_assert(kDwRows * 8 <= kThreads, "a thread a value of dpre");

// A block takes 512 columns and a part of the channels, a lane eight columns, the
// waves every eighth channel; they join in LDS, the parts in half_join_kernel.
template <class T, int N>
__device__ inline void dx_few(const GradArgs &a, const FewArgs &f, int block, float (&terms)[kDxRows][N],
                              float (&sums)[kThreads / 64][kDxCols]) {
  constexpr int kAhead = 8, kWaves = kThreads / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int split = block / f.dx_chunks, first = block % f.dx_chunks * kDxCols;
  const int begin = split * f.each, end = min(begin + f.each, a.out);
  const int8_t *at = f.w + min((int64_t)first + lane * 8, f.pitch - 8);
  float acc[N][8] = {};
  for (int o0 = begin; o0 < end; o0 += kDxRows) {
    const int rows = min(kDxRows, end - o0);
    uint2 next[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      next[k] = *(const uint2 *)(at + (int64_t)min(o0 + wave + k * kWaves, end - 1) * f.pitch);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * N; i += kThreads) {
      const int o = o0 + i / N, t = i % N;
      terms[i / N][t] = t < a.n ? dpre_of<T>(a, t, o) * a.w_scales[o] : 0.0f;
    }
    __syncthreads();
    for (int r = wave; r < rows; r += kAhead * kWaves) {
      uint2 now[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        now[k] = next[k];
        next[k] = *(const uint2 *)(at + (int64_t)min(o0 + r + (kAhead + k) * kWaves, end - 1) * f.pitch);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (r + k * kWaves >= rows) break;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = value_of(j < 4 ? now[k].x : now[k].y, j & 3);
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[t][j] = fmaf(terms[r + k * kWaves][t], v[j], acc[t][j]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < N; ++t) {
    if (t >= a.n) break;
    __syncthreads();
    *(float4 *)&sums[wave][lane * 8] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
    *(float4 *)&sums[wave][lane * 8 + 4] = make_float4(acc[t][4], acc[t][5], acc[t][6], acc[t][7]);
    __syncthreads();
    const int c = first + threadIdx.x;
    float sum = sums[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) sum += sums[k][threadIdx.x];
    if (c >= f.in) continue;
    if (f.parts) f.parts[((int64_t)split * a.n + t) * f.in + c] = sum;
    else ((typename T::raw *)f.dx)[t * f.dx_stride + c] = T::put(sum);
  }
}
static_assert(kDxCols == kThreads, "a thread a column at the end");

// dx's blocks, the longer ones, first.
template <class T, int N, bool ADD, bool NT>
__global__ void __launch_bounds__(kThreads) few_kernel(GradArgs a, FewArgs f) {
  __shared__ __attribute__((aligned(16))) FewLds<N> lds;
  if ((int)blockIdx.x < f.dx_blocks) return dx_few<T, N>(a, f, blockIdx.x, lds.dx.terms, lds.dx.sums);
  dw_few<T, N, ADD, NT>(a, f, blockIdx.x - f.dx_blocks, lds.dpre);
}

template <class T, int N>
hipError_t launch_few(const GradArgs &a, const FewArgs &f, bool add, unsigned blocks, hipStream_t s) {
  const auto go = [&](auto kernel) { kernel<<<blocks, kThreads, 0, s>>>(a, f); };
  if (add) go(few_kernel<T, N, true, false>);
  else if ((int64_t)f.in * a.out * 4 > kKept) go(few_kernel<T, N, false, true>);
  else go(few_kernel<T, N, false, false>);
  return hipGetLastError();
}
template <class T>
hipError_t launch_few(const GradArgs &a, const welvet_hip_rows8 *x, const welvet_hip_int8 *layer, int in, float *dw,
                      bool add, void *dx, int64_t dx_stride, void *parts, hipStream_t s) {
  FewArgs f{};
  f.in = in;
  unsigned blocks = 0;
  int splits = 1;
  const int64_t values = (int64_t)a.n * in;
  if (dw) {
    f.x = x->d_codes;
    f.x_stride = x->stride;
    f.dw = dw;
    f.dw_chunks = tiles_of(in, kDwCols);
    blocks = (unsigned)tiles_of(a.out, kDwRows) * f.dw_chunks;
  }
  if (dx) {
    f.w = layer->codes;
    f.pitch = layer->pitch;
    f.dx = dx;
    f.dx_stride = dx_stride;
    f.dx_chunks = tiles_of(in, kDxCols);
    // two blocks a CU, of 64 channels and more; the parts' workspace holds 2^22 values
    splits = (int)std::max<int64_t>(1, std::min<int64_t>({16, 512 / f.dx_chunks, a.out / 64, ((int64_t)1 << 22) / values}));
    f.each = tiles_of(a.out, splits);
    splits = tiles_of(a.out, f.each);
    f.parts = splits > 1 ? (float *)parts : nullptr;
    f.dx_blocks = f.dx_chunks * splits;
    blocks += f.dx_blocks;
  }
  hipError_t e = a.n == 1   ? launch_few<T, 1>(a, f, add, blocks, s)
                 : a.n == 2 ? launch_few<T, 2>(a, f, add, blocks, s)
                 : a.n <= 4 ? launch_few<T, 4>(a, f, add, blocks, s)
                            : launch_few<T, kFew>(a, f, add, blocks, s);
  if (e != hipSuccess || splits == 1) return e;
  const int per_row = tiles_of(in, 8);
  half_join_kernel<T, false><<<(unsigned)((a.n * per_row + 255) / 256), 256, 0, s>>>(
      Splits(splits, values, parts), nullptr, (typename T::raw *)dx, dx_stride, a.n, in, per_row);
  return hipGetLastError();
}

// 256 x 256, a block a CU, where there is one for each; 128 x 128, two.  (dw and dx
// of bf16 4096 x 4096, 2048 rows, 128 and 256 of the large tiles, with the stores: 324 us
// against 341 without any; of 1024 x 1024, 4096 rows, 64 and 16: 256 with the large, 93
// with the small ones.
// Fewer than four stages are mostly results, which two blocks a CU write beside each
// other's products: dw 9536 x 8512 f32 of 153 rows 101 us, large 125; 8192 x 2048 of
// 256 rows, four stages, 31 and 28.)
using Large = Tile<HalfOp, kParts, 2, 4, 4, 2>;
using Medium = Tile<HalfOp, kParts, 2, 2, 2, 2>;
using Deep = Tile<HalfOp, kParts, 2, 4, 2, 1, 4, 4>;
using Slim = Tile<HalfOp, kParts, 2, 4, 1, 1, 6, 6>;

template <class T, class Tile>
Product<T> product_of(const Operands &g, const float *back, void *to, int64_t stride, void *parts) {
  const int tm = tiles_of(g.a_rows, Tile::kRows), tn = tiles_of(g.b_rows, Tile::kCols);
  return {g, back, (typename T::raw *)to, stride, Splits(tm, tn, g, Tile::kRows, Tile::kParts, parts), tm, tn};
}
template <class T, bool ADD>
hipError_t launch_join(const Product<T> &q, hipStream_t s) {
  if (q.p.splits == 1) return hipGetLastError();
  const int per_row = tiles_of(q.g.b_rows, 8);
  half_join_kernel<T, ADD><<<(unsigned)(((int64_t)q.g.a_rows * per_row + 255) / 256), 256, 0, s>>>(
      q.p, q.back, q.to, q.stride, q.g.a_rows, q.g.b_rows, per_row);
  return hipGetLastError();
}
// Split: the tile of the parts.
template <class T, bool ADD, class Tile, class Split>
hipError_t launch_tiles(const Operands &g, const float *back, void *to, int64_t stride, void *parts, hipStream_t s) {
  const auto q = product_of<T, Tile>(g, back, to, stride, parts);
  const auto go = [&](auto kernel, int waves) { kernel<<<q.blocks(), waves * 64, 0, s>>>(q); };
  if constexpr (Tile::kRows <= kSplitRows) {
    if (q.p.splits > 1) {
      if (Splits::one_a_cu(q.tiles_m * q.tiles_n)) go(half_tile_kernel<T, ADD, Split, true>, Split::kWaves);
      else go(half_tile_kernel<T, ADD, Tile, true>, Tile::kWaves);
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? launch_join<T, ADD>(q, s) : e;
    }
  }
  go(half_tile_kernel<T, ADD, Tile, false>, Tile::kWaves);
  return hipGetLastError();
}
// to[a_rows][b_rows] (+)= back . A . B^T.
template <class T, bool ADD>
hipError_t launch_half(const Operands &g, const float *back, void *to, int64_t stride, void *parts, hipStream_t s) {
  if ((int64_t)tiles_of(g.a_rows, 256) * tiles_of(g.b_rows, 256) >= 256 && g.stages >= 4)
    return launch_tiles<T, ADD, Large, Large>(g, back, to, stride, parts, s);
  if (g.a_rows <= 64) return launch_tiles<T, ADD, Medium, Slim>(g, back, to, stride, parts, s);
  return launch_tiles<T, ADD, Medium, Deep>(g, back, to, stride, parts, s);
}

// dx and dw in one launch of 128 x 128 tiles, two blocks a CU, where dx alone has no
// more tiles than there are CUs (us, both with the stores, in two launches and in one:
// f32 2048 -> 8192 of 256 rows, 32 tiles, 93 and 88.5; bf16 4096 -> 4096 of 64 rows 63
// and 59.5; f32 8512 -> 9536 of 153, 134 tiles, 285 and 258; bf16 2048 -> 11008 of 2000,
// 256 tiles, 529 and 489).
constexpr int kPairTiles = 256;
template <class T, bool ADD>
hipError_t launch_pair(const Product<T> &x, const Product<F32> &w, hipStream_t s) {
  half_pair_kernel<T, ADD, Medium><<<x.blocks() + w.blocks(), Medium::kWaves * 64, 0, s>>>(
      x, w, x.blocks());
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) e = launch_join<T, false>(x, s);
  return e == hipSuccess ? launch_join<F32, ADD>(w, s) : e;
}

// Bounds that the next pass's blocks read in all, each those of its rows and columns,
// past which they are folded first (us of the fold and that pass: bf16 8192 rows,
// 11008 channels, 418304 bounds, 237 to 263 and 296 without; f32 1000 rows, 2048 channels,
// 5120 bounds, 13.4 without, and the fold's launch alone takes 5).
constexpr int64_t kFoldFrom = 1 << 16;

struct Plan {
  size_t grad_w, grad_x, codes_x, codes_w, col_bound, row_bound, col_back, row_back, parts, parts_x;  // offsets
  size_t bytes;
};
Plan plan_of(int64_t n, int64_t in, int64_t out) {
  Plan p{};
  size_t at = 0;
  const auto take = [&](int64_t bytes) {
    const size_t was = at;
    at += pad256((size_t)bytes);
    return was;
  };
  p.grad_w = take(2 * kParts * out * along(n));
  p.codes_x = take(2 * in * along(n));
  p.grad_x = take(2 * kParts * n * along(out));
  p.codes_w = take(2 * in * along(out));
  p.col_bound = take(4 * std::min<int64_t>(most_bounds(out), tiles_of(n, kBoundRows)) * out);  // not fewer than any smaller n needs
  p.row_bound = take(4 * tiles_of(out, kBoundCols) * n);
  p.col_back = take(4 * out);
  p.row_back = take(4 * n);
  p.parts = take(parts_bytes(out, in));
  p.parts_x = take(parts_bytes(n, in));
  p.bytes = at;
  return p;
}

bool sizes_ok(int32_t n, int32_t in, int32_t out) {
  return n >= 0 && n <= kMaxSize && in > 0 && in <= kMaxSize && out > 0 && out <= kMaxSize;
}
// A launch of fewer than 2^32 threads: 512 a 128 x 64 block of the passes.
bool launchable(int64_t n, int64_t in, int64_t out) {
  constexpr int64_t most = (int64_t)1 << 22;
  const int64_t tn = tiles_of(n, kRows), to = tiles_of(out, kRows);
  return tn * tiles_of(out, kCols) < most && tiles_of(in, kCols) * (tn + to) < most;
}

}  // namespace
}  // namespace wh

using namespace wh;
using namespace wh::rt;

extern "C" {

welvet_status welvet_hip_rows8_backward_bytes(int32_t dtype, int32_t n, int32_t in, int32_t out, size_t *bytes) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "rows8 backward: unsupported dtype %d", dtype);
  if (!sizes_ok(n, in, out) || !launchable(n, in, out) || !bytes)
    return make_status(kInvalid, "rows8 backward: invalid argument");
  *bytes = plan_of(n, in, out).bytes;
  return ok();
}

welvet_status welvet_hip_rows8_backward(int32_t act, int32_t dtype, int32_t n, int32_t in, int32_t out,
                                        const void *d_dy, int64_t dy_stride, const welvet_hip_rows8 *pre8,
                                        const welvet_hip_rows8 *x8, const welvet_hip_int8 *layer, void *d_dpre,
                                        int64_t dpre_stride, void *d_dx, int64_t dx_stride, int32_t accumulate,
                                        float *d_dw, void *d_ws, size_t ws_bytes, void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "rows8 backward: unsupported dtype %d", dtype);
  if (!sizes_ok(n, in, out) || !launchable(n, in, out) || (n > 0 && !d_dy) || dy_stride < out ||
      (!d_dpre && !d_dx && !d_dw) || (d_dpre && dpre_stride < out) || (d_dx && dx_stride < in) ||
      (accumulate != 0 && accumulate != 1))
    return make_status(kInvalid, "rows8 backward: invalid argument");
  if (act < kLinear || act > kReLU2) return make_status(kInvalid, "rows8 backward: activation %d", act);
  if (!pre8 && act != kLinear) return make_status(kInvalid, "rows8 backward: the pre-activations are needed");
  if (n > 0 && d_dx && (d_dx == d_dy || d_dx == d_dpre))
    return make_status(kInvalid, "rows8 backward: dx in dy's or dpre's place");
  if (d_dw && !x8) return make_status(kInvalid, "rows8 backward: dw needs the input's rows");
  if (d_dx && (!layer || layer->in != in || layer->out != out))
    return make_status(kInvalid, "rows8 backward: dx needs a layer of %d -> %d", in, out);
  if (const char *why = pre8 && act != kLinear ? r8::rows_fault(pre8, n, out) : nullptr)
    return make_status(kInvalid, "rows8 backward: %s", why);
  if (const char *why = d_dw ? r8::rows_fault(x8, n, in) : nullptr)
    return make_status(kInvalid, "rows8 backward: %s", why);
  if (n > 1 && d_dpre == d_dy && dpre_stride != dy_stride)
    return make_status(kInvalid, "rows8 backward: dpre in the place of dy needs its row stride");
  const int size = tok::float_size(dtype);
  if (!tok::aligned(d_dy, size) || !tok::aligned(d_dpre, size) || !tok::aligned(d_dx, size) || !tok::aligned(d_dw, 4))
    return make_status(kInvalid, "rows8 backward: device pointers must be aligned to their elements");
  const Plan p = plan_of(n, in, out);
  const bool products = d_dw || d_dx;
  if (products && n > 0 && (!d_ws || ws_bytes < p.bytes || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "rows8 backward: %zu bytes of 16-byte aligned workspace are needed", p.bytes);
  welvet_status st = require_device();
  if (st.code) return st;
  hipStream_t s = (hipStream_t)stream;
  if (n == 0) {
    if (d_dw && !accumulate) {
      const int64_t all = (int64_t)out * in;
      zero_kernel<<<(unsigned)std::min<int64_t>((all + 255) / 256, 65536), 256, 0, s>>>(d_dw, all);
      WH_HIP(hipGetLastError());
    }
    return ok();
  }
  char *ws = (char *)d_ws;
  GradArgs a{};
  Image x{}, w{};
  a.dy = d_dy;
  a.dy_stride = dy_stride;
  if (act != kLinear) {
    a.pre = pre8->d_codes;
    a.pre_stride = pre8->stride;
    a.pre_scales = pre8->d_scales;
  }
  a.dpre = d_dpre;
  a.dpre_stride = dpre_stride;
  a.n = n;
  a.out = out;
  a.act = act;
  a.across = tiles_of(out, kCols);
  a.bound_rows = bound_rows(n, out);
  a.col_parts = tiles_of(n, a.bound_rows);
  a.row_parts = tiles_of(out, kBoundCols);
  a.n_pitch = along(n);
  a.o_pitch = along(out);
  a.col_bound = (uint32_t *)(ws + p.col_bound);
  a.row_bound = (uint32_t *)(ws + p.row_bound);
  a.col_back = (float *)(ws + p.col_back);
  a.row_back = (float *)(ws + p.row_back);
  void *parts = ws + p.parts;
  const int in_tiles = tiles_of(in, kCols);
  if (d_dw) {
    a.x_scales = x8->d_scales;
    a.along_n = (uint16_t *)(ws + p.grad_w);
    x = {x8->d_codes, x8->stride, a.n_pitch, n, in, in_tiles, (uint16_t *)(ws + p.codes_x), tiles_of(n, kRows) * in_tiles};
  }
  if (d_dx) {
    a.w_scales = layer->scales;
    a.along_o = (uint16_t *)(ws + p.grad_x);
    w = {layer->codes, layer->pitch, a.o_pitch, out, in, in_tiles, (uint16_t *)(ws + p.codes_w), tiles_of(out, kRows) * in_tiles};
  }
  WH_HIP(tok::with_type(dtype, [&](auto t) -> hipError_t {
    using T = decltype(t);
    hipError_t e = hipSuccess;
    if (n <= kFew) {
      if (products) {
        // dpre in the place of dy, or without dw, comes last, in a launch of its own
        const bool with_dw = d_dw && d_dpre != d_dy;
        a.dpre = with_dw ? d_dpre : nullptr;
        e = launch_few<T>(a, x8, layer, in, d_dw, accumulate, d_dx, dx_stride, ws + p.parts_x, s);
        if (e != hipSuccess || !d_dpre || with_dw) return e;
        a.dpre = d_dpre;
      }
      a.along_n = a.along_o = nullptr;
      grad_kernel<T, false><<<a.across, kThreads, 0, s>>>(x, a);
      return hipGetLastError();
    }
    const bool one = d_dw && !d_dx && n <= kRows;
    if (products && !one) {
      prepare_kernel<T><<<x.blocks + w.blocks + a.col_parts * a.row_parts, kThreads, 0, s>>>(x, w, a);
      if ((e = hipGetLastError()) != hipSuccess) return e;
      if (((d_dw ? a.col_parts : 0) + (d_dx ? a.row_parts : 0)) * (int64_t)tiles_of(n, kRows) * a.across > kFoldFrom) {
        fold_kernel<<<tiles_of((d_dw ? out : 0) + (d_dx ? n : 0), 256), 256, 0, s>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        a.col_parts = a.row_parts = 1;
      }
    }
    // up to 128 rows without dx one launch does both (f16 1001 -> 777, 100 rows: 27 -> 22 us in all)
    if (one) grad_kernel<T, true><<<x.blocks + a.across, kThreads, 0, s>>>(x, a);
    else grad_kernel<T, false><<<(unsigned)tiles_of(n, kRows) * a.across, kThreads, 0, s>>>(x, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    const Operands gw{(const char *)a.along_n, 2 * a.n_pitch, 2 * out * a.n_pitch, out, INT32_MAX,
                      (const char *)x.to, 2 * a.n_pitch, in, tiles_of(2 * (int64_t)n, kStageBytes)};
    const Operands gx{(const char *)a.along_o, 2 * a.o_pitch, 2 * n * a.o_pitch, n, INT32_MAX,
                      (const char *)w.to, 2 * a.o_pitch, in, tiles_of(2 * (int64_t)out, kStageBytes)};
    if (d_dw && d_dx) {
      const auto px = product_of<T, Medium>(gx, a.row_back, d_dx, dx_stride, ws + p.parts_x);
      if (px.tiles_m * px.tiles_n <= kPairTiles) {
        const auto pw = product_of<F32, Medium>(gw, a.col_back, d_dw, in, parts);
        return accumulate ? launch_pair<T, true>(px, pw, s) : launch_pair<T, false>(px, pw, s);
      }
    }
    if (d_dw) {
      e = accumulate ? launch_half<F32, true>(gw, a.col_back, d_dw, in, parts, s)
                     : launch_half<F32, false>(gw, a.col_back, d_dw, in, parts, s);
      if (e != hipSuccess) return e;
    }
    if (d_dx) e = launch_half<T, false>(gx, a.row_back, d_dx, dx_stride, ws + p.parts_x, s);
    return e;
  }));
  return ok();
}

}  // extern "C"
