// adapters.hip — low-rank adapters of many requests beside one shared
// projection: adapter a holds a down factor [rank][in] and an up factor
// [rank][out], and every row of x names its own adapter (or none).
//   forward   h = x . down_a^T             y  = base + s_a h . up_a
//   backward  g = dy . up_a^T              dx = dx_base + s_a g . down_a
//             ddown_a = s_a sum_t g_t x_t  dup_a = s_a sum_t h_t dy_t
// Both factors keep the rank first, so the two directions are the same three
// products: rows by a factor over its width (down_kernel), rank values spread
// over a width (up_kernel), and sums over an adapter's rows (outer_kernel).
// Products and sums are f32 (the f32 MFMA, fma chains in its accumulators):
// activations are f32 and a 16-bit factor is exact in f32.
//
// Rows are taken in the order of their adapters (tokens.hpp), 16 of them a
// tile, so a tile reads each of its adapters once; a tile of several adapters
// computes all 16 rows with each and keeps the adapter's own, so no value of
// another tenant's factor reaches a row, NaN or not.  Few rows (a decode
// step) are tiles of one row in their own order, without the sorting launch.
#include <hip/hip_runtime.h>

#include "tokens.hpp"

namespace wh {
namespace {

using namespace tok;

using v4f = __attribute__((ext_vector_type(4))) float;
__device__ inline v4f mfma(float a, float b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

constexpr int kMaxRank = 256;
constexpr int kFewRows = 128;  // tiles of one row up to here

// The rows of a launch: position p -> row and adapter (count: none).
struct RowMap {
  const int32_t *key;    // adapter by position (sorted), or by row
  const int32_t *order;  // row by position; null: the row itself
  int n, count, tile;    // tile: positions a block takes together (16 or 1)
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
// The products of down_kernel: [splits][n][rank], to be added up.
struct Hidden {
  float *p;
  int splits, n, rank;
  __device__ float at(int row, int j) const {
    const float *q = p + (int64_t)row * rank + j;
    float v = q[0];
    for (int s = 1; s < splits; ++s) v += q[(int64_t)s * n * rank];
    return v;
  }
};

// Four values at row + k of a row of `width`: zeros past its end.
template <bool VEC>
__device__ inline float4 load4(const float *row, int k, int width) {
  if constexpr (VEC) return k < width ? *(const float4 *)(row + k) : make_float4(0, 0, 0, 0);
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = k + i < width ? row[k + i] : 0.0f;
  return make_float4(f[0], f[1], f[2], f[3]);
}
template <class T, bool VEC>
__device__ inline float4 load4t(const typename T::raw *row, int k, int width) {
  if constexpr (VEC && sizeof(typename T::raw) == 4) {
    return k < width ? *(const float4 *)(row + k) : make_float4(0, 0, 0, 0);
  } else if constexpr (VEC) {
    const ushort4 u = k < width ? *(const ushort4 *)(row + k) : make_ushort4(0, 0, 0, 0);
    return make_float4(T::get(u.x), T::get(u.y), T::get(u.z), T::get(u.w));
  } else {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = k + i < width ? T::get(row[k + i]) : 0.0f;
    return make_float4(f[0], f[1], f[2], f[3]);
  }
}
template <bool VEC>
__device__ inline void store4(float *row, int k, int width, float4 v) {
  if constexpr (VEC) {
    if (k < width) *(float4 *)(row + k) = v;
  } else {
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i < width) row[k + i] = f[i];
  }
}
__device__ inline float get4(const float4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// --------------------------------------------------------- rows by a factor
// hidden[split][row][j] = sum over the split's k of x[row][k] factor_a[j][k].
// D[i = row][j = rank] of 16 x 16 x 4 MFMAs: lane l holds row (or rank) l % 16
// and k = 4 (l / 16) + s for the s-th of four MFMAs, so both operands are one
// 4-value load a lane.  A block's waves take 16 k in turn and add up in LDS.
constexpr int kDownWaves = 8;
template <class T, bool VEC, int RT>
__global__ void __launch_bounds__(kDownWaves * 64) down_kernel(RowMap rows, Factor fac, const float *__restrict__ x,
                                                               int64_t xstride, Hidden out, int split_len) {
  __shared__ float red[kDownWaves][16][RT * 16 + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lo = lane & 15, q = lane >> 4;
  const int p0 = blockIdx.x * rows.tile, live = min(rows.tile, rows.n - p0), j0 = blockIdx.z * RT * 16;
  const int kbegin = blockIdx.y * split_len, kend = min(kbegin + split_len, fac.width);
  const int mine = min(lo, live - 1);  // lanes past the tile's rows repeat its last
  const int row = rows.row(p0 + mine), key = rows.adapter(p0 + mine);
  const float *xrow = x + (int64_t)row * xstride;
  float *hidden = out.p + (int64_t)blockIdx.y * out.n * out.rank;
  for (int i0 = 0; i0 < live;) {
    const int a = __builtin_amdgcn_readlane(key, i0);
    // the run of positions [i0, i1) of adapter a
    const uint64_t same = __ballot(lane < live && key == a);
    const int i1 = i0 + __popcll(same >> i0);
    const int ra = a < rows.count ? fac.rank_of(a) : 0;
    v4f acc[RT] = {};
    if (ra > j0) {
      const typename T::raw *f = (const typename T::raw *)fac.p + ((int64_t)a * fac.rank + j0) * fac.width;
      const int most = ra - j0;
      for (int k = kbegin + wave * 16; k < kend; k += kDownWaves * 16) {
        const float4 xv = load4<VEC>(xrow, k + 4 * q, kend);
        float4 fv[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const int j = t * 16 + lo;
          fv[t] = j < most ? load4t<T, VEC>(f + (int64_t)j * fac.width, k + 4 * q, kend) : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t] = mfma(get4(xv, s), get4(fv[t], s), acc[t]);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[wave][4 * q + r][t * 16 + lo] = acc[t][r];
    }
    __syncthreads();
    const int width = min(RT * 16, fac.rank - j0);
    for (int e = threadIdx.x; e < (i1 - i0) * width; e += kDownWaves * 64) {
      const int i = i0 + e / width, j = e % width;
      float sum = 0.0f;
      if (j0 + j < ra)
#pragma unroll
        for (int w = 0; w < kDownWaves; ++w) sum += red[w][i][j];
      hidden[(int64_t)rows.row(p0 + i) * out.rank + j0 + j] = sum;
    }
    __syncthreads();
    i0 = i1;
  }
}

// --------------------------------------------- rank values over a width
// y[row] = base[row] + s_a sum_j hidden[row][j] factor_a[j].  D[i = row][j =
// column]: lane l holds columns 4 (l % 16) + m of its wave's 64 for the m-th
// of four accumulators, so a row's part is stored as 16-byte words; ranks 4
// (l / 16) + s of each 16 for the s-th MFMA.  Block: four waves, 256 columns.
template <class T, bool VEC, int RT>
__global__ void __launch_bounds__(256) up_kernel(RowMap rows, Factor fac, Hidden h, const float *base,
                                                 int64_t bstride, float *y, int64_t ystride,
                                                 float *__restrict__ hsum, int tiles) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lo = lane & 15, q = lane >> 4;
  const int c = blockIdx.x * 256 + wave * 64 + 4 * lo;
  for (int tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
    const int p0 = tile * rows.tile, live = min(rows.tile, rows.n - p0);
    if (hsum && blockIdx.x == 0)
      for (int e = threadIdx.x; e < live * fac.rank; e += 256) {
        const int row = rows.row(p0 + e / fac.rank);
        hsum[(int64_t)row * fac.rank + e % fac.rank] = h.at(row, e % fac.rank);
      }
    const int mine = min(lo, live - 1);
    const int row = rows.row(p0 + mine), key = rows.adapter(p0 + mine);
    int out_row[4], out_key[4];
    float4 sum[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // the rows this lane's accumulators belong to
      out_row[r] = __shfl(row, 4 * q + r);
      out_key[r] = __shfl(key, 4 * q + r);
      sum[r] = make_float4(0, 0, 0, 0);
      if (base && 4 * q + r < live && c < fac.width) sum[r] = load4<VEC>(base + (int64_t)out_row[r] * bstride, c, fac.width);
    }
    for (int i0 = 0; i0 < live;) {
      const int a = __builtin_amdgcn_readlane(key, i0);
      const uint64_t same = __ballot(lane < live && key == a);
      i0 += __popcll(same >> i0);
      if (a >= rows.count) continue;
      const int ra = fac.rank_of(a);
      const float scale = fac.scale_of(a);
      const typename T::raw *f = (const typename T::raw *)fac.p + (int64_t)a * fac.rank * fac.width;
      v4f acc[4] = {};
      for (int g = 0; g < ra; g += 16 * RT) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const int j = g + 16 * t + 4 * q;
          float hv[4];
          float4 fv[4];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            hv[s] = j + s < ra ? h.at(row, j + s) : 0.0f;
            fv[s] = j + s < ra && c < fac.width ? load4t<T, VEC>(f + (int64_t)(j + s) * fac.width, c, fac.width)
                                                : make_float4(0, 0, 0, 0);
          }
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int m = 0; m < 4; ++m) acc[m] = mfma(hv[s], get4(fv[s], m), acc[m]);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (out_key[r] == a)
          sum[r] = make_float4(fmaf(scale, acc[0][r], sum[r].x), fmaf(scale, acc[1][r], sum[r].y),
                               fmaf(scale, acc[2][r], sum[r].z), fmaf(scale, acc[3][r], sum[r].w));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * q + r < live) store4<VEC>(y + (int64_t)out_row[r] * ystride, c, fac.width, sum[r]);
  }
}

// ------------------------------------------------ sums over an adapter's rows
// grad_a[j][c] = s_a sum over a's rows of hidden[row][j] x[row][c].  D[i =
// rank][j = column]: a wave 64 columns (as above), four rows an MFMA.  A block
// takes kSumRows positions of the sorted rows; an adapter whose rows end
// inside them is written from registers, one that reaches into a neighbour's
// leaves a partial (slot 0: began earlier, slot 1: goes on) for sum_kernel.
constexpr int kSumRows = 512;
template <bool VEC, bool ACC, int RT>
__global__ void __launch_bounds__(256) outer_kernel(RowMap rows, Factor fac, Hidden h, const float *__restrict__ x,
                                                    int64_t xstride, float *__restrict__ grad,
                                                    float *__restrict__ part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lo = lane & 15, q = lane >> 4;
  const int c = blockIdx.x * 256 + wave * 64 + 4 * lo, j0 = blockIdx.z * RT * 16;
  const int p0 = blockIdx.y * kSumRows, p1 = min(p0 + kSumRows, rows.n);
  const int64_t size = (int64_t)fac.rank * fac.width;
  for (int i0 = p0; i0 < p1;) {
    const int a = rows.adapter(i0);
    if (a >= rows.count) break;  // rows without an adapter come last
    int i1 = p1;                 // the end of a's run here
    for (int step = i0, hi = p1; step < hi;) {
      const int mid = (step + hi) >> 1;
      if (rows.adapter(mid) == a) step = mid + 1;
      else i1 = hi = mid;
    }
    const bool began = i0 > p0 || p0 == 0 || rows.adapter(p0 - 1) != a;
    const bool goes_on = i1 == p1 && p1 < rows.n && rows.adapter(p1) == a;
    const int ra = fac.rank_of(a);
    v4f acc[RT][4] = {};
    if (ra > j0)
      for (int p = i0; p < i1; p += 4) {
        const bool in = p + q < i1;
        const int row = in ? rows.row(p + q) : 0;
        float4 xv = make_float4(0, 0, 0, 0);
        if (in && c < fac.width) xv = load4<VEC>(x + (int64_t)row * xstride, c, fac.width);
        float hv[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) hv[t] = in && j0 + 16 * t + lo < ra ? h.at(row, j0 + 16 * t + lo) : 0.0f;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[t][m] = mfma(hv[t], get4(xv, m), acc[t][m]);
      }
    const float scale = fac.scale_of(a);
    const bool whole = began && !goes_on;
    float *to = whole ? grad + (int64_t)a * size : part + ((int64_t)blockIdx.y * 2 + (began ? 1 : 0)) * size;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = j0 + 16 * t + 4 * q + r;
        if (j >= fac.rank || c >= fac.width) continue;
        float4 v = j < ra ? make_float4(acc[t][0][r], acc[t][1][r], acc[t][2][r], acc[t][3][r])
                          : make_float4(0, 0, 0, 0);  // 0 times a NaN of x is not 0
        float *at = to + (int64_t)j * fac.width;
        if (whole) {
          v = j < ra ? make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale) : v;
          if constexpr (ACC) {
            const float4 o = load4<VEC>(at, c, fac.width);
            v = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
          }
        }
        store4<VEC>(at, c, fac.width, v);
      }
    i0 = i1;
  }
}

// The adapters outer_kernel did not write: their partials added up in order,
// zeros for those no row names.
template <bool ACC>
__global__ void __launch_bounds__(256) sum_kernel(RowMap rows, Factor fac, const float *__restrict__ part,
                                                  float *__restrict__ grad) {
  const int a = blockIdx.y;
  int bound[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    int lo = 0, hi = rows.n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (rows.key[mid] < a + e) lo = mid + 1;
      else hi = mid;
    }
    bound[e] = lo;
  }
  const int64_t size = (int64_t)fac.rank * fac.width;
  float *to = grad + (int64_t)a * size;
  if (bound[0] == bound[1]) {
    if constexpr (!ACC)
      for (int64_t e = blockIdx.x * 256 + threadIdx.x; e < size; e += (int64_t)gridDim.x * 256) to[e] = 0.0f;
    return;
  }
  const int first = bound[0] / kSumRows, last = (bound[1] - 1) / kSumRows;
  if (first == last) return;
  const int ra = fac.rank_of(a);
  const float scale = fac.scale_of(a);
  for (int64_t e = blockIdx.x * 256 + threadIdx.x; e < size; e += (int64_t)gridDim.x * 256) {
    // its first block's rows went on (slot 1), every later one's began earlier
    float v = part[((int64_t)first * 2 + 1) * size + e];
    for (int b = first + 1; b <= last; ++b) v += part[(int64_t)b * 2 * size + e];
    v = e < (int64_t)ra * fac.width ? v * scale : 0.0f;
    to[e] = ACC ? to[e] + v : v;
  }
}

// ------------------------------------------------------------------ launches
// Blocks along k where the row tiles alone leave CUs idle: at least 512
// values of the width each.
int splits_of(int n, int width) {
  const int tiles = n <= kFewRows ? n : (n + 15) / 16;
  return std::max(1, std::min({16, 512 / std::max(1, tiles), width / 512}));
}

struct Call {
  int32_t dtype;
  RowMap rows;
  hipStream_t s;
};

template <class F>
void by_rank(int rank, F &&f) {
  if (rank <= 16) f(std::integral_constant<int, 1>{});
  else if (rank <= 32) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 4>{});
}
template <class F>
void by_vec(bool vec, F &&f) {
  if (vec) f(std::true_type{});
  else f(std::false_type{});
}

bool vec_ok(const Factor &f, int32_t dtype, std::initializer_list<std::pair<const void *, int64_t>> f32) {
  bool ok = f.width % 4 == 0 && aligned(f.p, 4 * float_size(dtype));
  for (auto &pe : f32) ok = ok && aligned(pe.first, 16) && pe.second % 4 == 0;
  return ok;
}

hipError_t launch_down(const Call &c, const Factor &fac, const float *x, int64_t xstride, const Hidden &out) {
  const int split_len = (((fac.width + out.splits - 1) / out.splits) + 15) / 16 * 16;
  const int tiles = (c.rows.n + c.rows.tile - 1) / c.rows.tile;
  by_rank(fac.rank, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    const dim3 grid(tiles, out.splits, (fac.rank + 16 * RT - 1) / (16 * RT));
    by_vec(vec_ok(fac, c.dtype, {{x, xstride}}), [&](auto vec) {
      with_type(c.dtype, [&](auto t) {
        down_kernel<decltype(t), decltype(vec)::value, RT>
            <<<grid, kDownWaves * 64, 0, c.s>>>(c.rows, fac, x, xstride, out, split_len);
      });
    });
  });
  return hipGetLastError();
}

hipError_t launch_up(const Call &c, const Factor &fac, const Hidden &h, const float *base, int64_t bstride, float *y,
                     int64_t ystride, float *hsum) {
  const int tiles = (c.rows.n + c.rows.tile - 1) / c.rows.tile;
  by_rank(fac.rank, [&](auto rt) {
    const dim3 grid((fac.width + 255) / 256, std::min(tiles, 65535));
    by_vec(vec_ok(fac, c.dtype, {{base, base ? bstride : 0}, {y, ystride}}), [&](auto vec) {
      with_type(c.dtype, [&](auto t) {
        up_kernel<decltype(t), decltype(vec)::value, decltype(rt)::value>
            <<<grid, 256, 0, c.s>>>(c.rows, fac, h, base, bstride, y, ystride, hsum, tiles);
      });
    });
  });
  return hipGetLastError();
}

hipError_t launch_outer(const Call &c, const Factor &fac, const Hidden &h, const float *x, int64_t xstride,
                        bool accumulate, float *grad, float *part) {
  if (c.rows.n > 0) by_rank(fac.rank, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    const dim3 grid((fac.width + 255) / 256, (c.rows.n + kSumRows - 1) / kSumRows, (fac.rank + 16 * RT - 1) / (16 * RT));
    const bool ok = fac.width % 4 == 0 && aligned(x, 16) && xstride % 4 == 0 && aligned(grad, 16);
    by_vec(ok, [&](auto vec) {
      by_vec(accumulate, [&](auto acc) {
        outer_kernel<decltype(vec)::value, decltype(acc)::value, RT>
            <<<grid, 256, 0, c.s>>>(c.rows, fac, h, x, xstride, grad, part);
      });
    });
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t size = (int64_t)fac.rank * fac.width;
  const dim3 grid((uint32_t)std::min<int64_t>((size + 255) / 256, 1024), c.rows.count);
  by_vec(accumulate, [&](auto acc) {
    sum_kernel<decltype(acc)::value><<<grid, 256, 0, c.s>>>(c.rows, fac, part, grad);
  });
  return hipGetLastError();
}

struct Sizes {
  size_t order = 0, hidden = 0, part = 0;
  size_t total() const { return order + hidden + part; }
};
Sizes sizes_of(const welvet_hip_adapters &d, int n, bool backward) {
  Sizes z;
  if (n == 0) return z;
  if (backward || n > kFewRows) z.order = order_bytes(n);
  const int splits = splits_of(n, backward ? d.out : d.in);
  z.hidden = pad256((size_t)splits * n * d.rank * sizeof(float));
  if (backward)
    z.part = pad256(((size_t)n + kSumRows - 1) / kSumRows * 2 * d.rank * (size_t)std::max(d.in, d.out) * sizeof(float));
  return z;
}

bool desc_ok(const welvet_hip_adapters *d, int32_t n) {
  return d && n >= 0 && n <= (1 << 24) && d->count > 0 && d->count <= 65535 && d->rank > 0 && d->rank <= kMaxRank &&
         d->in > 0 && d->out > 0 && d->in <= INT32_MAX - 512 && d->out <= INT32_MAX - 512;
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
  if (!desc_ok(desc, n) || !bytes) return make_status(kInvalid, "adapters: invalid argument");
  *bytes = std::max(sizes_of(*desc, n, false).total(), sizes_of(*desc, n, true).total());
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
  const Sizes z = sizes_of(*desc, n, false);
  if (z.total() > 0 && (!d_ws || ws_bytes < z.total() || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "adapters: %zu bytes of 16-byte aligned workspace are needed", z.total());
  st = require_device();
  if (st.code || n == 0) return st;
  Call c{desc->dtype, {d_ids, nullptr, n, desc->count, 1}, (hipStream_t)stream};
  if (n > kFewRows) {
    tok::Order o;
    WH_HIP(tok::launch_order(d_ids, n, desc->count, d_ws, &o, c.s));
    c.rows = {o.skey, o.order, n, desc->count, 16};
  }
  const Factor down{desc->d_down, desc->d_ranks, desc->d_scales, desc->rank, desc->in};
  const Factor up{desc->d_up, desc->d_ranks, desc->d_scales, desc->rank, desc->out};
  Hidden h{(float *)((char *)d_ws + z.order), splits_of(n, desc->in), n, desc->rank};
  if (h.splits == 1 && d_h) h.p = d_h;
  WH_HIP(launch_down(c, down, d_x, x_stride, h));
  WH_HIP(launch_up(c, up, h, d_base, base_stride, d_y, y_stride, h.p == d_h ? nullptr : d_h));
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
  st = require_device();
  if (st.code) return st;
  Call c{desc->dtype, {nullptr, nullptr, n, desc->count, 16}, (hipStream_t)stream};
  float *part = nullptr;
  Hidden g{nullptr, 1, n, desc->rank};
  const Factor down{desc->d_down, desc->d_ranks, desc->d_scales, desc->rank, desc->in};
  const Factor up{desc->d_up, desc->d_ranks, desc->d_scales, desc->rank, desc->out};
  if (n > 0) {
    tok::Order o;
    WH_HIP(tok::launch_order(d_ids, n, desc->count, d_ws, &o, c.s));
    c.rows.key = o.skey;
    c.rows.order = o.order;
    g.p = (float *)((char *)d_ws + z.order);
    g.splits = splits_of(n, desc->out);
    part = (float *)((char *)d_ws + z.order + z.hidden);
    if (d_dx || d_ddown) WH_HIP(launch_down(c, up, d_dy, dy_stride, g));
    if (d_dx) WH_HIP(launch_up(c, down, g, d_dx_base, dx_base_stride, d_dx, dx_stride, nullptr));
  }
  if (d_ddown) WH_HIP(launch_outer(c, down, g, d_x, x_stride, accumulate != 0, d_ddown, part));
  if (d_dup)
    WH_HIP(launch_outer(c, up, Hidden{const_cast<float *>(d_h), 1, n, desc->rank}, d_dy, dy_stride, accumulate != 0,
                        d_dup, part));
  return ok();
}

}  // extern "C"
