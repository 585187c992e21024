// int8.hip — a layer whose product runs in 8-bit integers: rows x_t as codes c
// with a scale s_t each (rows8.hpp), weights as codes w with a scale v_o an
// output channel:
//   pre = s_t v_o sum_k c_tk w_ok + bias_o,  post = act(pre)
// The sum is exact in 32 bits (in <= 131072: 127^2 in < 2^31), so how it is
// split changes nothing, and a row has the same results in every batch.
//
// A few rows are bound by the weights' bytes (bf16 4096 -> 11008, one row, 12.1 us;
// 4096 -> 131072, up to 16 rows, 100 us with the store, 5.4 TB/s), many by the matrix
// cores and the operands' way to them: f16 4096 -> 11008 of 8192 rows, 416 to 463 us
// behind a store of 22 to 28, 1.6 to 1.8 POP/s (a library's integer product of these
// sizes alone: 397 us).
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>
#include <vector>

#include "int8.hpp"
#include "rows8.hpp"
#include "tiles.hpp"

namespace wh {
namespace {

using namespace r8;
using namespace tiles;

constexpr int kMaxIn = 131072, kMaxOut = 1 << 24;

struct Out {
  void *pre, *post;
  int64_t pre_stride, post_stride;
  const float *x_scales, *w_scales, *bias;
  int n, out, act;
};
__device__ inline float pre_of(int sum, float scale, float bias) { return fmaf((float)sum, scale, bias); }

// Eight results of a row from channel c on.
template <class T>
__device__ inline void put8(const Out &o, int row, int c, const int (&sum)[8], float s, const float (&scale)[8],
                            const float (&bias)[8]) {
  float v[8];
  Oct<T> out;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = pre_of(sum[i], s * scale[i], bias[i]);
  if (o.pre) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out.set(i, v[i]);
    out.store((typename T::raw *)o.pre + row * o.pre_stride, c, o.out);
  }
  if (o.post) {
    acts<T>(v, o.act);
#pragma unroll
    for (int i = 0; i < 8; ++i) out.set(i, v[i]);
    out.store((typename T::raw *)o.post + row * o.post_stride, c, o.out);
  }
}
// A lane's eight channels: their scales and biases.
__device__ inline void channels(const Out &o, int first, float (&scale)[8], float (&bias)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    scale[i] = o.w_scales[min(first + i, o.out - 1)];
    bias[i] = o.bias[min(first + i, o.out - 1)];
  }
}

// --------------------------------------------------------------- few rows
// Weights are read once and bound the call: a block takes 16 channels, its
// eight waves every eighth 64 bytes of their rows, and joins the waves' sums in
// LDS.  Sixteen rows of x are the matrix instruction's other side, TILES times.
struct Few {
  const int8_t *codes;
  int64_t pitch;
  const int8_t *x;
  int64_t x_stride;
  int last, steps;
};
template <class T, int WAVES, int TILES>
__device__ inline void few_join(const Out &o, int first, const i32x4 (&acc)[TILES], i32x4 *part, const float *x_scales) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int t = 0; t < TILES; ++t) part[(wave * TILES + t) * 64 + lane] = acc[t];
  __syncthreads();
  if (wave >= TILES) return;
  i32x4 sum = part[wave * 64 + lane];
#pragma unroll
  for (int k = 1; k < WAVES; ++k) sum += part[(k * TILES + wave) * 64 + lane];
  const int row = wave * 16 + (lane & 15);
  if (row >= o.n) return;
  const float scale = x_scales[row];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = first + (lane >> 4) * 4 + i;
    if (c >= o.out) break;
    float v[1] = {pre_of(sum[i], scale * o.w_scales[c], o.bias[c])};
    if (o.pre) ((typename T::raw *)o.pre)[row * o.pre_stride + c] = T::put(v[0]);
    if (!o.post) continue;
    acts<T>(v, o.act);
    ((typename T::raw *)o.post)[row * o.post_stride + c] = T::put(v[0]);
  }
}
template <class T, int WAVES, int TILES>
__global__ void __launch_bounds__(WAVES * 64) int8_few_kernel(Few f, Out o) {
  constexpr int kAhead = TILES == 1 ? 8 : 4;
  __shared__ i32x4 part[WAVES * TILES * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int first = blockIdx.x * 16;
  const int8_t *w = f.codes + (int64_t)min(first + r, o.out - 1) * f.pitch + q * 16;
  const int8_t *xs[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) xs[t] = f.x + (int64_t)min(t * 16 + r, o.n - 1) * f.x_stride;
  i32x4 acc[TILES] = {};
  int s = wave;
  for (; s + (kAhead - 1) * WAVES < f.steps; s += kAhead * WAVES) {
    i32x4 a[kAhead], b[kAhead][TILES];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      a[k] = __builtin_nontemporal_load((const i32x4 *)(w + (int64_t)(s + k * WAVES) * 64));
      const int at = min((s + k * WAVES) * 64 + q * 16, f.last);
#pragma unroll
      for (int t = 0; t < TILES; ++t) b[k][t] = *(const i32x4 *)(xs[t] + at);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int t = 0; t < TILES; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][t], acc[t], 0, 0, 0);
  }
  for (; s < f.steps; s += WAVES) {
    const i32x4 a = __builtin_nontemporal_load((const i32x4 *)(w + (int64_t)s * 64));
    const int at = min(s * 64 + q * 16, f.last);
#pragma unroll
    for (int t = 0; t < TILES; ++t)
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *(const i32x4 *)(xs[t] + at), acc[t], 0, 0, 0);
  }
  few_join<T, WAVES, TILES>(o, first, acc, part, o.x_scales);
}

// A few rows straight from x: every block stores them in 8 bits for itself, in
// LDS, while its first weights are under way; one launch instead of two (us, bf16,
// this and the store with int8_few_kernel: 4096 -> 11008 one row 12.1 / 15.4, three
// 16 / 16; 1024 -> 1024 6.1 / 7.2; 8192 -> 1000 one row 9.5 / 12.7).  One row of 4096
// -> 11008 reads its 45 MB at 3.8 TB/s.  The block's waves share the rows.
constexpr int kOwnRows = 4, kOwnCodes = 32768, kOwnWaves = 8;
template <class T>
__global__ void __launch_bounds__(kOwnWaves * 64, 6) int8_own_kernel(Few f, const typename T::raw *x, int64_t x_stride,
                                                                  int in, Out o) {
  constexpr int kAhead = 8, kGroups = sizeof(typename T::raw) == 4 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) uint2 codes[kOwnCodes / 8];
  __shared__ i32x4 part[kOwnWaves * 64];
  __shared__ uint32_t tops[kOwnWaves];
  __shared__ float scales[kOwnRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int first = blockIdx.x * 16, padded_in = f.last + 16;
  const int8_t *w = f.codes + (int64_t)min(first + r, o.out - 1) * f.pitch + q * 16;
  const int waves = o.n == 1 ? kOwnWaves : o.n == 2 ? kOwnWaves / 2 : kOwnWaves / 4;  // of a row
  const int row = min(wave / waves, o.n - 1), own = threadIdx.x % (waves * 64), step = waves * 64;
  const typename T::raw *from = x + row * x_stride;
  const Eights e(in);
  Oct<T> held[kGroups], rest;
  uint32_t top = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
    if (g * step < e.whole) e.load(held[g], from, g * step + own);
  i32x4 a[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)  // past the row's end: its last bytes again, not used
    a[k] = __builtin_nontemporal_load((const i32x4 *)(w + (int64_t)min(wave + k * kOwnWaves, f.steps - 1) * 64));
  issued();
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
    if (g * step < e.whole) raise(top, held[g]);
  if (e.left && own == 0) {
    rest.load(from, e.whole * 8, in);
    raise(top, rest);
  }
  for (int g = kGroups * step; g < e.whole; g += step) {
    Oct<T> h;
    e.load(h, from, g + own);
    raise(top, h);
  }
  top = widened<T>(top);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  for (int k = wave / waves * waves; k < wave / waves * waves + waves; ++k) top = max(top, tops[k]);
  const Scale s8(top);
  int8_t *to = (int8_t *)codes + row * padded_in;
  if (own == 0) {  // waves without a row of theirs have the last one's again
    scales[row] = s8.stored;
    e.finish(to, s8, rest);
  }
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
    if (g * step + own < e.whole) {
      issued();
      *(uint2 *)(to + (g * step + own) * 8) = codes8(s8, [&](int i) { return held[g].get(i); });
    }
  for (int g = kGroups * step + own; g < e.whole; g += step) {
    Oct<T> h;
    e.load(h, from, g);
    *(uint2 *)(to + g * 8) = codes8(s8, [&](int i) { return h.get(i); });
  }
  __syncthreads();
  const char *xs = (const char *)codes + min(r, o.n - 1) * padded_in;
  i32x4 acc[1] = {};
  for (int s = wave; s < f.steps; s += kAhead * kOwnWaves) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (s + k * kOwnWaves < f.steps)
        acc[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
            a[k], *(const i32x4 *)(xs + min((s + k * kOwnWaves) * 64 + q * 16, f.last)), acc[0], 0, 0, 0);
    if (s + kAhead * kOwnWaves < f.steps)
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        a[k] = __builtin_nontemporal_load(
            (const i32x4 *)(w + (int64_t)min(s + (kAhead + k) * kOwnWaves, f.steps - 1) * 64));
  }
  few_join<T, kOwnWaves, 1>(o, first, acc, part, scales);
}

// -------------------------------------------------------------- many rows
template <class T, class Tile, bool PART>
__global__ void __launch_bounds__(Tile::kWaves * 64) int8_tile_kernel(Operands g, Out o, Splits p, int tiles_m,
                                                                      int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  const int tiles = tiles_m * tiles_n, tile = blockIdx.x % tiles, split = blockIdx.x / tiles;  // 0 of the whole
  const Place at = place(tile, tiles_m, tiles_n);
  const int m0 = at.m * Tile::kRows, n0 = at.n * Tile::kCols;
  typename Tile::Acc acc[Tile::kTM][Tile::kTN] = {};
  Tile::run(PART ? g.part(split * p.each, min(p.each, g.stages - split * p.each)) : g, m0, n0, acc, lds);
  __syncthreads();
  if constexpr (PART) {
    Tile::template results<4>(m0, n0, acc, lds, [&](int row, int c, const int (&sum)[4]) {
      if (row >= o.n || c >= o.out) return;
      float *to = (float *)p.parts + split * p.parts_values + (int64_t)row * o.out;
      store4(to, c, o.out, make_float4(__int_as_float(sum[0]), __int_as_float(sum[1]), __int_as_float(sum[2]), __int_as_float(sum[3])));
    });
  } else {
    float *x_scales = (float *)(lds + Tile::kResults);
    for (int i = threadIdx.x; i < Tile::kRows; i += Tile::kWaves * 64) x_scales[i] = o.x_scales[min(m0 + i, o.n - 1)];
    float scale[8], bias[8];  // a lane's channels are the same in all its rows
    channels(o, Tile::first_col(n0), scale, bias);
    __syncthreads();
    Tile::template results<8>(m0, n0, acc, lds, [&](int row, int c, const int (&sum)[8]) {
      if (row < o.n && c < o.out) put8<T>(o, row, c, sum, x_scales[row - m0], scale, bias);
    });
  }
}
template <class T>
__global__ void __launch_bounds__(256) int8_join_kernel(Splits p, Out o, int per_row) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int row = (int)(i / per_row), c = (int)(i % per_row) * 8;
  if (row >= o.n) return;
  const uint32_t *at = (const uint32_t *)p.parts + (int64_t)row * o.out;
  int sum[8] = {};
  for (int k = 0; k < p.splits; k += 4) {
    Oct<F32> v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n].load(at + min(k + n, p.splits - 1) * p.parts_values, c, o.out);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += k + n < p.splits ? (int)v[n].w[j] : 0;
  }
  float scale[8], bias[8];
  channels(o, c, scale, bias);
  put8<T>(o, row, c, sum, o.x_scales[row], scale, bias);
}

using Large = Tile<Int8Op, 1, 2, 4, 4, 2>;   // 256 x 256, eight waves
using Medium = Tile<Int8Op, 1, 2, 2, 2, 2>;  // 128 x 128, four
using Deep = Tile<Int8Op, 1, 2, 4, 2, 1, 4, 4>;  // 128 x 128, eight
using Narrow = Tile<Int8Op, 1, 2, 4, 1, 1, 3, 3>;  // 64 x 128, eight waves, two blocks a CU
using Slim = Tile<Int8Op, 1, 2, 4, 1, 1, 6, 6>;  // 64 x 128, eight: half the copies of x

// Split: the tile of the parts.
template <class T, class Tile, class Split>
hipError_t launch_tiles(const welvet_hip_int8 &l, const int8_t *x, int64_t x_stride, const Out &o, void *parts,
                        hipStream_t s) {
  const int tm = (o.n + Tile::kRows - 1) / Tile::kRows, tn = (o.out + Tile::kCols - 1) / Tile::kCols;
  const Operands g{(const char *)x, x_stride, 0, o.n, (int)padded(l.in) - 16, (const char *)l.codes, l.pitch, l.out,
                   (l.in + kStageBytes - 1) / kStageBytes};
  const Splits p(tm, tn, g, Tile::kRows, 1, parts);
  if constexpr (Tile::kRows <= kSplitRows) {
    if (p.splits > 1) {
      const auto go = [&](auto kernel, int waves) { kernel<<<tm * tn * p.splits, waves * 64, 0, s>>>(g, o, p, tm, tn); };
      if (Splits::one_a_cu(tm * tn)) go(int8_tile_kernel<T, Split, true>, Split::kWaves);
      else go(int8_tile_kernel<T, Tile, true>, Tile::kWaves);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      const int per_row = (o.out + 7) / 8;
      int8_join_kernel<T><<<(unsigned)(((int64_t)o.n * per_row + 255) / 256), 256, 0, s>>>(p, o, per_row);
      return hipGetLastError();
    }
  }
  int8_tile_kernel<T, Tile, false><<<tm * tn, Tile::kWaves * 64, 0, s>>>(g, o, p, tm, tn);
  return hipGetLastError();
}

// Channels for whole 64 x 128 tiles on half the CUs and more (of more than eight rows a
// third), and weights that outweigh a few rows' ways below (us, bf16, with the few-row
// kernels and with tiles: 4096 -> 131072 one row 119 / 97, 16 rows 190 / 102, 5.3 TB/s;
// 1024 -> 32000 one row 28 / 12, 1024 -> 21504 8 rows 11.5 / 14.6; 4096 -> 18432 one row
// 20.9 / 20; 4096 -> 11008 16 rows 20.9 / 18.9, 8 rows 18.2 / 20.1).
bool many_channels(const welvet_hip_int8 &l, int32_t n) {
  return l.out > (n > 8 ? 80 : 128) * Narrow::kCols && (int64_t)l.in * l.out > 30 << 20;
}
hipError_t launch_product(const welvet_hip_int8 &l, int32_t dtype, const int8_t *x, int64_t x_stride, const Out &o,
                          void *parts, hipStream_t s) {
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const Few f{l.codes, l.pitch, x, x_stride, (int)padded(l.in) - 16, (l.in + 63) / 64};
    const unsigned blocks = (unsigned)((l.out + 15) / 16);
    // 16 waves where eight a CU would be all there are (us, up to 16 rows: the tiles'
    // parts take 21 to 23 from 4096 -> 11008, this 17.5 to 21.7; 4096 -> 1024 13 / 10)
    const bool wide = blocks <= 512 && f.steps >= 64;
    if (o.n <= 64 && many_channels(l, o.n)) return launch_tiles<T, Narrow, Narrow>(l, x, x_stride, o, parts, s);
    if (o.n <= 16) {
      if (wide) int8_few_kernel<T, 16, 1><<<blocks, 1024, 0, s>>>(f, o);
      else int8_few_kernel<T, 8, 1><<<blocks, 512, 0, s>>>(f, o);
      return hipGetLastError();
    }
    // small weights: one launch, where the other way's parts take two (us, bf16:
    // 17 to 32 rows 4096 -> 1024 12 to 13 / 14 to 15, 4096 -> 11008 28 / 22; 64 rows
    // 1024 -> 1024 8.9 / 13.6, 6201 -> 640 23 / 16, 4096 -> 11008 38 / 27)
    if ((int64_t)l.in * l.out <= 4 << 20) {
      if (o.n <= 32) {
        if (wide) int8_few_kernel<T, 16, 2><<<blocks, 1024, 0, s>>>(f, o);
        else int8_few_kernel<T, 8, 2><<<blocks, 512, 0, s>>>(f, o);
        return hipGetLastError();
      }
      if (o.n <= 64 && l.in <= 2048) {
        int8_few_kernel<T, 8, 4><<<blocks, 512, 0, s>>>(f, o);
        return hipGetLastError();
      }
    }
    // large tiles, a block a CU, where there is one for each and more than half of it
    // is rows (us, large and small tiles, bf16: 4096 -> 65536 of 128 rows 76 / 58; 4096 -> 11008 of 2048 rows 146 / 142, of 4096 225 / 246; 11008 ->
    // 4096 of 2048 rows, 128 large tiles, 175 / 125)
    if (o.n > 128 && (int64_t)((o.n + 255) / 256) * ((l.out + 255) / 256) >= 256) return launch_tiles<T, Large, Large>(l, x, x_stride, o, parts, s);
    if (o.n <= 64) return launch_tiles<T, Narrow, Slim>(l, x, x_stride, o, parts, s);
    return launch_tiles<T, Medium, Deep>(l, x, x_stride, o, parts, s);
  });
}
// One launch from x, for rows that the caller does not keep; not of short rows where
// blocks come one after the other on a CU.  us, bf16, weights from HBM, a pass among
// others, this and the other way (whose two launches take 11 however small), one row and
// four: out 8192, in 1024 9 / 11 and 9 / 11, 4096 10 / 13 and 12.5 / 13.4; out 9216, in
// 1536 12 / 11 and 12.5 / 11.7, 2560 12.8 / 11.6 and 14.5 / 12.4, 3584 12.8 / 14 and 15.3 /
// 15.3, 4096 12.7 / 15.9 and 15.6 / 16.6, 6144 21.5 / 21.1 and 25 / 22.4, 8192 22 / 26 and
// 26.7 / 27.2; out 14336, in 2560 18 / 14 and 18 / 15, 3584 18.4 / 18.6 and 19.7 / 18.6.
bool own_rows(const welvet_hip_int8 &l, int32_t n) {
  return n <= kOwnRows && n * padded(l.in) <= kOwnCodes && (l.out <= 8192 || l.in > 3200) && !many_channels(l, n);
}
// Whether matrices of n rows share memory.  In one launch a block would read x beside
// others that have written there.
bool meet(const void *a, int64_t a_stride, int32_t a_cols, const void *b, int64_t b_stride, int32_t b_cols, int32_t n,
          int size) {
  const auto end = [&](const void *p, int64_t stride, int32_t cols) {
    return (uintptr_t)p + (uintptr_t)(((n - 1) * stride + cols) * size);
  };
  return a && b && (uintptr_t)a < end(b, b_stride, b_cols) && (uintptr_t)b < end(a, a_stride, a_cols);
}
hipError_t launch_own(const welvet_hip_int8 &l, int32_t dtype, const void *x, int64_t x_stride, const Out &o,
                      hipStream_t s) {
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const Few f{l.codes, l.pitch, nullptr, 0, (int)padded(l.in) - 16, (l.in + 63) / 64};
    int8_own_kernel<T><<<(unsigned)((l.out + 15) / 16), 512, 0, s>>>(f, (const typename T::raw *)x, x_stride, l.in, o);
    return hipGetLastError();
  });
}

// The forward's own rows, then the parts of a split sum.
int64_t row_bytes(int32_t in) { return spread(in); }
size_t parts_at(int32_t in, int64_t n) { return pad256((size_t)n * row_bytes(in)) + pad256((size_t)n * 4); }
size_t forward_bytes(const welvet_hip_int8 &l, int64_t n) { return parts_at(l.in, n) + parts_bytes(n, l.out); }

void free_layer(welvet_hip_int8 *l) {
  if (!l) return;
  (void)hipFree(l->codes);
  (void)hipFree(l->scales);
  (void)hipFree(l->bias);
  delete l;
}

bool shape_ok(int32_t in, int32_t out) { return in <= kMaxIn && out <= kMaxOut && rt::dims_ok(out, in); }

// A layer with zeroed codes and its bias; the caller fills codes and scales.
welvet_status new_layer(int32_t in, int32_t out, int32_t act, const double *bias, size_t bias_len,
                        welvet_hip_int8 **layer) {
  auto *l = new (std::nothrow) welvet_hip_int8{in, out, act, spread(in), nullptr, nullptr,
                                               nullptr};
  if (!l) return rt::make_status(kInternal, "int8: out of memory");
  std::vector<float> b;
  hipError_t e = hipSuccess;
  try {
    b.assign(out, 0.0f);
  } catch (...) {
    e = hipErrorOutOfMemory;
  }
  for (size_t i = 0; e == hipSuccess && bias && i < bias_len && i < (size_t)out; ++i) b[i] = (float)bias[i];
  if (e == hipSuccess) e = rt::dev_malloc(&l->codes, (size_t)out * l->pitch);
  if (e == hipSuccess) e = rt::dev_malloc(&l->scales, (size_t)out * 4);
  if (e == hipSuccess) e = rt::dev_malloc(&l->bias, (size_t)out * 4);
  if (e == hipSuccess) e = hipMemcpy(l->bias, b.data(), (size_t)out * 4, hipMemcpyHostToDevice);
  if (e == hipSuccess) e = hipMemset(l->codes, 0, (size_t)out * l->pitch);
  if (e != hipSuccess) {
    free_layer(l);
    return rt::make_status(kInternal, "int8: %s", hipGetErrorString(e));
  }
  *layer = l;
  return rt::ok();
}
// Device weights [out][in] into a new layer.
welvet_status mount_values(int32_t in, int32_t out, int32_t act, const float *d_W, const double *bias,
                           size_t bias_len, welvet_hip_int8 **layer) {
  welvet_hip_int8 *l = nullptr;
  welvet_status st = new_layer(in, out, act, bias, bias_len, &l);
  if (st.code) return st;
  hipError_t e = launch_store(kFloat32, out, in, d_W, in, l->codes, l->pitch, l->scales, nullptr);
  if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
  if (e != hipSuccess) {
    free_layer(l);
    return rt::make_status(kInternal, "int8: %s", hipGetErrorString(e));
  }
  *layer = l;
  return rt::ok();
}

}  // namespace
}  // namespace wh

using namespace wh;
using namespace wh::rt;

namespace {
welvet_status checked_out(const welvet_hip_int8 *l, int32_t dtype, int32_t n, void *d_pre, int64_t pre_stride,
                          void *d_post, int64_t post_stride) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "int8: unsupported dtype %d", dtype);
  if (!l || n < 0 || n > r8::kMaxRows || (!d_pre && !d_post)) return make_status(kInvalid, "int8: invalid argument");
  if ((d_pre && pre_stride < l->out) || (d_post && post_stride < l->out))
    return make_status(kInvalid, "int8: row stride below out %d", l->out);
  if (n > 0 && d_pre == d_post) return make_status(kInvalid, "int8: pre and post must not be one matrix");
  const int size = tok::float_size(dtype);
  if (!tok::aligned(d_pre, size) || !tok::aligned(d_post, size))
    return make_status(kInvalid, "int8: device pointers must be aligned to their elements");
  // a launch of fewer than 2^32 threads: 256 x 256 results a block of 512
  if (((int64_t)n + 255) / 256 * (((int64_t)l->out + 255) / 256) >= (1 << 22))
    return make_status(kInvalid, "int8: %d rows of %d channels are more than a launch takes", n, l->out);
  return ok();
}
}  // namespace

extern "C" {

welvet_status welvet_hip_int8_mount(int32_t in, int32_t out, int32_t act, const float *W, const double *bias,
                                    size_t bias_len, welvet_hip_int8 **layer) {
  if (!layer) return make_status(kInvalid, "int8: null layer");
  *layer = nullptr;
  if (!shape_ok(in, out) || !W || (bias_len > 0 && !bias)) return make_status(kInvalid, "int8: invalid argument");
  welvet_status st = require_device();
  if (st.code) return st;
  DevBuf w(nullptr, false);
  WH_HIP(w.alloc((size_t)in * out * 4));
  WH_HIP(hipMemcpy(w.p, W, (size_t)in * out * 4, hipMemcpyHostToDevice));
  return mount_values(in, out, act, w.as<float>(), bias, bias_len, layer);
}

welvet_status welvet_hip_int8_mount_device(int32_t in, int32_t out, int32_t act, const float *d_W, const double *bias,
                                           size_t bias_len, welvet_hip_int8 **layer) {
  if (!layer) return make_status(kInvalid, "int8: null layer");
  *layer = nullptr;
  if (!shape_ok(in, out) || !d_W || !tok::aligned(d_W, 16) || (bias_len > 0 && !bias))
    return make_status(kInvalid, "int8: invalid argument");
  welvet_status st = require_device();
  if (st.code) return st;
  return mount_values(in, out, act, d_W, bias, bias_len, layer);
}

welvet_status welvet_hip_int8_mount_codes(int32_t in, int32_t out, int32_t act, const int8_t *codes,
                                          const float *scales, const double *bias, size_t bias_len,
                                          welvet_hip_int8 **layer) {
  if (!layer) return make_status(kInvalid, "int8: null layer");
  *layer = nullptr;
  if (!shape_ok(in, out) || !codes || !scales || (bias_len > 0 && !bias))
    return make_status(kInvalid, "int8: invalid argument");
  for (size_t i = 0; i < (size_t)in * out; ++i)
    if (codes[i] == -128) return make_status(kInvalid, "int8: a code of -128");
  welvet_status st = require_device();
  if (st.code) return st;
  welvet_hip_int8 *l = nullptr;
  st = new_layer(in, out, act, bias, bias_len, &l);
  if (st.code) return st;
  hipError_t e = hipMemcpy2D(l->codes, l->pitch, codes, in, in, out, hipMemcpyHostToDevice);
  if (e == hipSuccess) e = hipMemcpy(l->scales, scales, (size_t)out * 4, hipMemcpyHostToDevice);
  if (e != hipSuccess) {
    free_layer(l);
    return make_status(kInternal, "int8: %s", hipGetErrorString(e));
  }
  *layer = l;
  return ok();
}

welvet_status welvet_hip_int8_mount_dense(welvet_dense_session *s, welvet_hip_int8 **layer) {
  if (!layer) return make_status(kInvalid, "int8: null layer");
  *layer = nullptr;
  if (!s) return make_status(kInvalid, "null session");
  DevBuf w(nullptr);
  std::vector<double> bias;
  int in = 0, out = 0, act = 0;
  welvet_status st = session_values(s, &w, &bias, &in, &out, &act);
  if (st.code) return st;
  return welvet_hip_int8_mount_device(in, out, act, w.as<float>(), bias.data(), bias.size(), layer);
}

welvet_status welvet_hip_int8_weights(welvet_hip_int8 *l, int8_t *codes, float *scales) {
  if (!l) return make_status(kInvalid, "int8: null layer");
  welvet_status st = require_device();
  if (st.code) return st;
  if (codes) WH_HIP(hipMemcpy2D(codes, l->in, l->codes, l->pitch, l->in, l->out, hipMemcpyDeviceToHost));
  if (scales) WH_HIP(hipMemcpy(scales, l->scales, (size_t)l->out * 4, hipMemcpyDeviceToHost));
  return ok();
}

void welvet_hip_int8_release(welvet_hip_int8 *l) { free_layer(l); }

welvet_status welvet_hip_int8_bytes(const welvet_hip_int8 *l, int32_t n, size_t *bytes) {
  if (!l || n < 0 || n > r8::kMaxRows || !bytes) return make_status(kInvalid, "int8: invalid argument");
  *bytes = forward_bytes(*l, n);
  return ok();
}

welvet_status welvet_hip_int8_forward(const welvet_hip_int8 *l, int32_t dtype, int32_t n, const void *d_x,
                                      int64_t x_stride, const welvet_hip_rows8 *rows, void *d_pre, int64_t pre_stride,
                                      void *d_post, int64_t post_stride, void *d_ws, size_t ws_bytes, void *stream) {
  welvet_status st = checked_out(l, dtype, n, d_pre, pre_stride, d_post, post_stride);
  if (st.code) return st;
  if ((n > 0 && !d_x) || x_stride < l->in) return make_status(kInvalid, "int8: invalid argument");
  if (!tok::aligned(d_x, tok::float_size(dtype)))
    return make_status(kInvalid, "int8: device pointers must be aligned to their elements");
  if (const char *why = rows ? r8::rows_fault(rows, n, l->in) : nullptr) return make_status(kInvalid, "int8: %s", why);
  const size_t need = forward_bytes(*l, n);
  if (n > 0 && (!d_ws || ws_bytes < need || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "int8: %zu bytes of 16-byte aligned workspace are needed", need);
  st = require_device();
  if (st.code || n == 0) return st;
  welvet_hip_rows8 r{(int8_t *)d_ws, row_bytes(l->in), (float *)((char *)d_ws + tok::pad256(n * row_bytes(l->in)))};
  if (rows) r = *rows;
  const Out o{d_pre, d_post, pre_stride, post_stride, r.d_scales, l->scales, l->bias, n, l->out, l->act};
  const int size = tok::float_size(dtype);
  if (!rows && own_rows(*l, n) && !meet(d_x, x_stride, l->in, d_pre, pre_stride, l->out, n, size) &&
      !meet(d_x, x_stride, l->in, d_post, post_stride, l->out, n, size)) {
    WH_HIP(launch_own(*l, dtype, d_x, x_stride, o, (hipStream_t)stream));
    return ok();
  }
  WH_HIP(r8::launch_store(dtype, n, l->in, d_x, x_stride, r.d_codes, r.stride, r.d_scales, (hipStream_t)stream));
  WH_HIP(launch_product(*l, dtype, r.d_codes, r.stride, o, (char *)d_ws + parts_at(l->in, n), (hipStream_t)stream));
  return ok();
}

welvet_status welvet_hip_int8_product(const welvet_hip_int8 *l, int32_t dtype, int32_t n, const welvet_hip_rows8 *rows,
                                      void *d_pre, int64_t pre_stride, void *d_post, int64_t post_stride, void *d_ws,
                                      size_t ws_bytes, void *stream) {
  welvet_status st = checked_out(l, dtype, n, d_pre, pre_stride, d_post, post_stride);
  if (st.code) return st;
  if (const char *why = r8::rows_fault(rows, n, l->in)) return make_status(kInvalid, "int8: %s", why);
  const size_t need = forward_bytes(*l, n);
  if (n > 0 && (!d_ws || ws_bytes < need || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "int8: %zu bytes of 16-byte aligned workspace are needed", need);
  st = require_device();
  if (st.code || n == 0) return st;
  const Out o{d_pre, d_post, pre_stride, post_stride, rows->d_scales, l->scales, l->bias, n, l->out, l->act};
  WH_HIP(launch_product(*l, dtype, rows->d_codes, rows->stride, o, (char *)d_ws + parts_at(l->in, n), (hipStream_t)stream));
  return ok();
}

}  // extern "C"
