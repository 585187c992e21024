// rows8_backward.hip — the backward of a layer from activations kept in 8 bits
// (rows8.hpp): with pre = p_t c the pre-activations and x = s_t c the input,
//   dpre = dy act'(pre);  dw = dpre^T x;  dx = dpre W
// Both products run on the bf16 matrix cores: codes are exact in bf16, and
// what is left of each term, dpre s_t (dw) or dpre v_o (dx, W = v_o w), is
// split into bf16 parts.  One pass over dy forms dpre and writes those parts
// with the sum along their rows (dw's transposed), a second one the codes'
// images; the products then read nothing but whole stages of bf16.
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
constexpr int kTile = 64;                                     // of the passes: rows and columns a block
int64_t along(int64_t n) { return (n + 31) / 32 * 32; }       // a sum's length in whole stages of bf16

// v as P bf16 parts, each the rest's nearest.  From the largest bf16 on the
// first is infinite and the others nothing.
template <int P>
__device__ inline void split(float v, uint16_t (&part)[P]) {
  part[0] = BF16::put(v);
  const bool whole = fabsf(v) < 0x1.fep127f;
#pragma unroll
  for (int p = 1; p < P; ++p) {
    v -= BF16::get(part[p - 1]);
    part[p] = whole ? BF16::put(v) : (uint16_t)0;
  }
}

// A block's 64 x 64 values, two rows a word, so that columns can be read as rows.
struct Turn {
  uint32_t word[kTile][kTile / 2 + 1];
  __device__ inline void put(int col, int pair, uint32_t v) { word[col][pair] = v; }
  // Sixteen bytes (eight rows) of each column into the image [cols][pitch]:
  // rows from `row` on, up to `pitch`, columns from `col` on, up to `cols`.
  __device__ inline void write(uint16_t *image, int64_t pitch, int row, int col, int cols) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = (threadIdx.x >> 3) + 32 * k, at = (threadIdx.x & 7) * 4;
      if (col + c < cols && row + 2 * at < pitch)
        *(uint4 *)(image + (int64_t)(col + c) * pitch + row + 2 * at) =
            make_uint4(word[c][at], word[c][at + 1], word[c][at + 2], word[c][at + 3]);
    }
  }
};

// Codes [rows][stride] -> bf16 [width][pitch], the rows' numbers along it.
__global__ void __launch_bounds__(256) image_kernel(const int8_t *__restrict__ codes, int64_t stride, int rows,
                                                    int width, int64_t pitch, int across, uint16_t *image) {
  __shared__ Turn turn;
  const int row = (int)(blockIdx.x / across) * kTile, col = (int)(blockIdx.x % across) * kTile;
  const int pair = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;
  uint2 w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = row + 2 * pair + k;
    w[k] = r < rows && col + c < width ? *(const uint2 *)(codes + (int64_t)r * stride + col + c) : make_uint2(0, 0);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float lo = value_of(i < 4 ? w[0].x : w[0].y, i & 3), hi = value_of(i < 4 ? w[1].x : w[1].y, i & 3);
    turn.put(c + i, pair, (f2u(lo) >> 16) | (f2u(hi) & 0xffff0000u));
  }
  __syncthreads();
  turn.write(image, pitch, row, col, width);
}

struct GradArgs {
  const void *dy;
  int64_t dy_stride;
  const int8_t *pre;  // null: Linear
  int64_t pre_stride;
  const float *pre_scales;
  const float *x_scales, *w_scales;
  void *dpre;
  int64_t dpre_stride;
  uint16_t *along_n, *along_o;  // dw's parts [PW][out][n_pitch], dx's [PX][n][o_pitch]
  int64_t n_pitch, o_pitch;
  int n, out, act, across;
};
template <class T, int PW, int PX>
__global__ void __launch_bounds__(256) grad_kernel(GradArgs a) {
  using raw = typename T::raw;
  __shared__ Turn turn[PW];
  const int row = (int)(blockIdx.x / a.across) * kTile, col = (int)(blockIdx.x % a.across) * kTile;
  const int pair = threadIdx.x >> 3, c = col + (threadIdx.x & 7) * 8;
  float v[2][8], s[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = row + 2 * pair + k;
    const bool in = r < a.n && c < a.out;
    Oct<T> o;
    o.load((const raw *)a.dy + (in ? (int64_t)r * a.dy_stride : 0), in ? c : a.out, a.out);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[k][i] = o.get(i);
    if (!in) continue;
    if (a.x_scales) s[k] = a.x_scales[r];
    if (a.pre) {
      const uint2 w = *(const uint2 *)(a.pre + (int64_t)r * a.pre_stride + c);
      const float p = a.pre_scales[r];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[k][i] = c + i < a.out ? v[k][i] * act_prime_f32(value_of(i < 4 ? w.x : w.y, i & 3) * p, a.act) : 0.0f;
    }
    if (a.dpre) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o.set(i, v[k][i]);
      o.store((raw *)a.dpre + (int64_t)r * a.dpre_stride, c, a.out);
    }
  }
  if (a.along_o && c < a.o_pitch) {
    float scale[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) scale[i] = c + i < a.out ? a.w_scales[c + i] : 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = row + 2 * pair + k;
      if (r >= a.n) continue;
      uint32_t w[PX][4] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint16_t part[PX];
        split<PX>(c + i < a.out ? v[k][i] * scale[i] : 0.0f, part);
#pragma unroll
        for (int p = 0; p < PX; ++p) w[p][i >> 1] |= (uint32_t)part[p] << (16 * (i & 1));
      }
#pragma unroll
      for (int p = 0; p < PX; ++p)
        *(uint4 *)(a.along_o + ((int64_t)p * a.n + r) * a.o_pitch + c) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
  }
  if (a.along_n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint16_t lo[PW], hi[PW];
      // rows past the last are nothing, whatever 0 times their values would be
      split<PW>(row + 2 * pair < a.n ? v[0][i] * s[0] : 0.0f, lo);
      split<PW>(row + 2 * pair + 1 < a.n ? v[1][i] * s[1] : 0.0f, hi);
#pragma unroll
      for (int p = 0; p < PW; ++p) turn[p].put(c - col + i, pair, lo[p] | ((uint32_t)hi[p] << 16));
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < PW; ++p)
      turn[p].write(a.along_n + (int64_t)p * a.out * a.n_pitch, a.n_pitch, row, col, a.out);
  }
}

// dw over no rows.
__global__ void __launch_bounds__(256) zero_kernel(float *to, int64_t all) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) to[i] = 0.0f;
}

// ---------------------------------------------------------------- products
template <class T, bool ADD, class Tile>
__global__ void __launch_bounds__(Tile::kWaves * 64) bf16_tile_kernel(Operands g, typename T::raw *to, int64_t stride,
                                                                      int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  const Place at = place(tiles_m, tiles_n);
  const int m0 = at.m * Tile::kRows, n0 = at.n * Tile::kCols;
  typename Tile::Acc acc[Tile::kTM][Tile::kTN] = {};
  Tile::run(g, m0, n0, acc, lds);
  Tile::results(m0, n0, acc, [&](int row, int c, float v) {
    if (row >= g.a_rows || c >= g.b_rows) return;
    typename T::raw *p = to + row * stride + c;
    *p = T::put(ADD ? T::get(*p) + v : v);
  });
}

// 256 x 256 with as many stages in LDS as fit, and 128 x 128.
template <int P>
using Large = Tile<Bf16Op, P, 2, 4, 4, 2, P == 1 ? 4 : P == 2 ? 3 : 2>;
template <int P>
using Medium = Tile<Bf16Op, P, 2, 2, 2, 2, P == 3 ? 3 : 4>;

template <class T, bool ADD, class Tile>
hipError_t launch_tiles(const Operands &g, void *to, int64_t stride, hipStream_t s) {
  const int tm = (g.a_rows + Tile::kRows - 1) / Tile::kRows, tn = (g.b_rows + Tile::kCols - 1) / Tile::kCols;
  bf16_tile_kernel<T, ADD, Tile><<<tm * tn, Tile::kWaves * 64, 0, s>>>(g, (typename T::raw *)to, stride, tm, tn);
  return hipGetLastError();
}
// to[a_rows][b_rows] (+)= A . B^T with A of P parts.
template <class T, bool ADD, int P>
hipError_t launch_bf16(const Operands &g, void *to, int64_t stride, hipStream_t s) {
  if ((int64_t)((g.a_rows + 255) / 256) * ((g.b_rows + 255) / 256) >= 128)
    return launch_tiles<T, ADD, Large<P>>(g, to, stride, s);
  return launch_tiles<T, ADD, Medium<P>>(g, to, stride, s);
}

template <class T>
struct Parts;
template <>
struct Parts<F32> {
  static constexpr int kW = 3, kX = 3;
};
template <>
struct Parts<F16> {
  static constexpr int kW = 2, kX = 2;
};
template <>
struct Parts<BF16> {
  static constexpr int kW = 2, kX = 1;
};

struct Plan {
  size_t grad_w, grad_x, codes_x, codes_w;  // offsets
  size_t bytes;
};
Plan plan_of(int32_t dtype, int64_t n, int64_t in, int64_t out) {
  const int pw = dtype == kFloat32 ? 3 : 2, px = dtype == kFloat32 ? 3 : dtype == kFloat16 ? 2 : 1;
  Plan p{};
  size_t at = 0;
  const auto take = [&](int64_t values) {
    const size_t was = at;
    at += pad256((size_t)values * 2);
    return was;
  };
  p.grad_w = take(pw * out * along(n));
  p.codes_x = take(in * along(n));
  p.grad_x = take(px * n * along(out));
  p.codes_w = take(in * along(out));
  p.bytes = at;
  return p;
}

hipError_t launch_image(const int8_t *codes, int64_t stride, int rows, int width, int64_t pitch, uint16_t *image,
                        hipStream_t s) {
  const int across = (width + kTile - 1) / kTile;
  image_kernel<<<(unsigned)((pitch + kTile - 1) / kTile) * across, 256, 0, s>>>(codes, stride, rows, width, pitch, across, image);
  return hipGetLastError();
}

bool sizes_ok(int32_t n, int32_t in, int32_t out) {
  return n >= 0 && n <= kMaxSize && in > 0 && in <= kMaxSize && out > 0 && out <= kMaxSize;
}
// A launch of fewer than 2^32 threads: 256 a 64 x 64 tile of the passes.
bool launchable(int64_t n, int64_t in, int64_t out) {
  const auto tiles = [](int64_t v) { return (v + kTile - 1) / kTile; };
  constexpr int64_t most = (int64_t)1 << 24;
  return tiles(along(n)) * tiles(along(out)) < most && tiles(along(n)) * tiles(in) < most && tiles(along(out)) * tiles(in) < most;
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
  *bytes = plan_of(dtype, n, in, out).bytes;
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
  const Plan p = plan_of(dtype, n, in, out);
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
  a.across = (int)((along(out) + kTile - 1) / kTile);
  a.n_pitch = along(n);
  a.o_pitch = along(out);
  if (d_dw) {
    a.x_scales = x8->d_scales;
    a.along_n = (uint16_t *)(ws + p.grad_w);
  }
  if (d_dx) {
    a.w_scales = layer->scales;
    a.along_o = (uint16_t *)(ws + p.grad_x);
  }
  uint16_t *codes_x = (uint16_t *)(ws + p.codes_x), *codes_w = (uint16_t *)(ws + p.codes_w);
  const unsigned blocks = (unsigned)((a.n_pitch + kTile - 1) / kTile) * a.across;
  WH_HIP(tok::with_type(dtype, [&](auto t) -> hipError_t {
    using T = decltype(t);
    constexpr int PW = Parts<T>::kW, PX = Parts<T>::kX;
    grad_kernel<T, PW, PX><<<blocks, 256, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && d_dw) {
      e = launch_image(x8->d_codes, x8->stride, n, in, a.n_pitch, codes_x, s);
      if (e != hipSuccess) return e;
      const Operands g{(const char *)a.along_n, 2 * a.n_pitch, 2 * out * a.n_pitch, out, INT32_MAX,
                       (const char *)codes_x, 2 * a.n_pitch, in, (int)(a.n_pitch / 32)};
      e = accumulate ? launch_bf16<F32, true, PW>(g, d_dw, in, s) : launch_bf16<F32, false, PW>(g, d_dw, in, s);
    }
    if (e == hipSuccess && d_dx) {
      e = launch_image(layer->codes, layer->pitch, out, in, a.o_pitch, codes_w, s);
      if (e != hipSuccess) return e;
      const Operands g{(const char *)a.along_o, 2 * a.o_pitch, 2 * n * a.o_pitch, n, INT32_MAX,
                       (const char *)codes_w, 2 * a.o_pitch, in, (int)(a.o_pitch / 32)};
      e = launch_bf16<T, false, PX>(g, d_dx, dx_stride, s);
    }
    return e;
  }));
  return ok();
}

}  // extern "C"
