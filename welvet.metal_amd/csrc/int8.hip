// int8.hip — a layer whose product runs in 8-bit integers: rows x_t as codes c
// with a scale s_t each (rows8.hpp), weights as codes w with a scale v_o an
// output channel:
//   pre = s_t v_o sum_k c_tk w_ok + bias_o,  post = act(pre)
// The sum is exact in 32 bits (in <= 131072: 127^2 in < 2^31), so how it is
// split changes nothing, and a row has the same results in every batch.
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

// ---------------------------------------------------------- up to 64 rows
// Weights are read once and bound the call: a block takes 16 channels, its
// eight waves every eighth 64 bytes of their rows, and joins the waves' sums in
// LDS.  Sixteen rows of x are the matrix instruction's other side, TILES times.
template <class T, int TILES>
__global__ void __launch_bounds__(512) int8_few_kernel(const int8_t *__restrict__ codes, int64_t pitch,
                                                       const int8_t *__restrict__ x, int64_t x_stride, int last,
                                                       int steps, Out o) {
  constexpr int kWaves = 8, kAhead = TILES == 1 ? 8 : 4;
  __shared__ i32x4 part[kWaves][TILES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int first = blockIdx.x * 16;
  const int8_t *w = codes + (int64_t)min(first + r, o.out - 1) * pitch + q * 16;
  const int8_t *xs[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) xs[t] = x + (int64_t)min(t * 16 + r, o.n - 1) * x_stride;
  i32x4 acc[TILES] = {};
  int s = wave;
  for (; s + (kAhead - 1) * kWaves < steps; s += kAhead * kWaves) {
    i32x4 a[kAhead], b[kAhead][TILES];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      a[k] = __builtin_nontemporal_load((const i32x4 *)(w + (int64_t)(s + k * kWaves) * 64));
      const int at = min((s + k * kWaves) * 64 + q * 16, last);
#pragma unroll
      for (int t = 0; t < TILES; ++t) b[k][t] = *(const i32x4 *)(xs[t] + at);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int t = 0; t < TILES; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][t], acc[t], 0, 0, 0);
  }
  for (; s < steps; s += kWaves) {
    const i32x4 a = __builtin_nontemporal_load((const i32x4 *)(w + (int64_t)s * 64));
    const int at = min(s * 64 + q * 16, last);
#pragma unroll
    for (int t = 0; t < TILES; ++t)
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *(const i32x4 *)(xs[t] + at), acc[t], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave >= TILES) return;
  i32x4 sum = part[0][wave][lane];
#pragma unroll
  for (int k = 1; k < kWaves; ++k) sum += part[k][wave][lane];
  const int row = wave * 16 + r;
  if (row >= o.n) return;
  const float scale = o.x_scales[row];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = first + q * 4 + i;
    if (c >= o.out) break;
    const float pre = pre_of(sum[i], scale * o.w_scales[c], o.bias[c]);
    if (o.pre) ((typename T::raw *)o.pre)[row * o.pre_stride + c] = T::put(pre);
    if (o.post) ((typename T::raw *)o.post)[row * o.post_stride + c] = T::put(act_of<T>(pre, o.act));
  }
}

// -------------------------------------------------------------- many rows
template <class T, class Tile>
__global__ void __launch_bounds__(Tile::kWaves * 64) int8_tile_kernel(Operands g, Out o, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  float *x_scales = (float *)(lds + Tile::kResults);
  const Place at = place(tiles_m, tiles_n);
  const int m0 = at.m * Tile::kRows, n0 = at.n * Tile::kCols;
  typename Tile::Acc acc[Tile::kTM][Tile::kTN] = {};
  Tile::run(g, m0, n0, acc, lds);
  __syncthreads();
  for (int i = threadIdx.x; i < Tile::kRows; i += Tile::kWaves * 64) x_scales[i] = o.x_scales[min(m0 + i, o.n - 1)];
  // a lane's channels are the same in all its rows
  const int first = Tile::first_col(n0);
  float scale[8], bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    scale[i] = o.w_scales[min(first + i, o.out - 1)];
    bias[i] = o.bias[min(first + i, o.out - 1)];
  }
  __syncthreads();
  Tile::results(m0, n0, acc, lds, [&](int row, int c, const int (&sum)[8]) {
    if (row >= o.n || c >= o.out) return;
    const float s = x_scales[row - m0];
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
      act8<T>(v, o.act);
#pragma unroll
      for (int i = 0; i < 8; ++i) out.set(i, v[i]);
      out.store((typename T::raw *)o.post + row * o.post_stride, c, o.out);
    }
  });
}

using Large = Tile<Int8Op, 1, 2, 4, 4, 2>;   // 256 x 256, eight waves
using Medium = Tile<Int8Op, 1, 2, 2, 2, 2>;  // 128 x 128, four

template <class T, class Tile>
hipError_t launch_tiles(const welvet_hip_int8 &l, const int8_t *x, int64_t x_stride, const Out &o, hipStream_t s) {
  const int tm = (o.n + Tile::kRows - 1) / Tile::kRows, tn = (o.out + Tile::kCols - 1) / Tile::kCols;
  const Operands g{(const char *)x, x_stride, 0, o.n, (int)padded(l.in) - 16, (const char *)l.codes, l.pitch, l.out,
                   (l.in + kStageBytes - 1) / kStageBytes};
  int8_tile_kernel<T, Tile><<<tm * tn, Tile::kWaves * 64, 0, s>>>(g, o, tm, tn);
  return hipGetLastError();
}

hipError_t launch_product(const welvet_hip_int8 &l, int32_t dtype, const int8_t *x, int64_t x_stride, const Out &o,
                          hipStream_t s) {
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int last = (int)padded(l.in) - 16, steps = (l.in + 63) / 64;
    const unsigned blocks = (unsigned)((l.out + 15) / 16);
    if (o.n <= 16) int8_few_kernel<T, 1><<<blocks, 512, 0, s>>>(l.codes, l.pitch, x, x_stride, last, steps, o);
    else if (o.n <= 32) int8_few_kernel<T, 2><<<blocks, 512, 0, s>>>(l.codes, l.pitch, x, x_stride, last, steps, o);
    else if (o.n <= 64) int8_few_kernel<T, 4><<<blocks, 512, 0, s>>>(l.codes, l.pitch, x, x_stride, last, steps, o);
    else if ((int64_t)((o.n + 255) / 256) * ((l.out + 255) / 256) >= 128)
      return launch_tiles<T, Large>(l, x, x_stride, o, s);
    else return launch_tiles<T, Medium>(l, x, x_stride, o, s);
    return hipGetLastError();
  });
}

// The forward's own rows.
int64_t row_bytes(int32_t in) { return spread(in); }
size_t forward_bytes(int32_t in, int64_t n) { return pad256((size_t)n * row_bytes(in)) + pad256((size_t)n * 4); }

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
  *bytes = forward_bytes(l->in, n);
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
  const size_t need = forward_bytes(l->in, n);
  if (n > 0 && (!d_ws || ws_bytes < need || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "int8: %zu bytes of 16-byte aligned workspace are needed", need);
  st = require_device();
  if (st.code || n == 0) return st;
  welvet_hip_rows8 r{(int8_t *)d_ws, row_bytes(l->in), (float *)((char *)d_ws + tok::pad256(n * row_bytes(l->in)))};
  if (rows) r = *rows;
  const Out o{d_pre, d_post, pre_stride, post_stride, r.d_scales, l->scales, l->bias, n, l->out, l->act};
  WH_HIP(r8::launch_store(dtype, n, l->in, d_x, x_stride, r.d_codes, r.stride, r.d_scales, (hipStream_t)stream));
  WH_HIP(launch_product(*l, dtype, r.d_codes, r.stride, o, (hipStream_t)stream));
  return ok();
}

welvet_status welvet_hip_int8_product(const welvet_hip_int8 *l, int32_t dtype, int32_t n, const welvet_hip_rows8 *rows,
                                      void *d_pre, int64_t pre_stride, void *d_post, int64_t post_stride, void *d_ws,
                                      size_t ws_bytes, void *stream) {
  welvet_status st = checked_out(l, dtype, n, d_pre, pre_stride, d_post, post_stride);
  if (st.code) return st;
  if (const char *why = r8::rows_fault(rows, n, l->in)) return make_status(kInvalid, "int8: %s", why);
  const size_t need = forward_bytes(l->in, n);
  if (n > 0 && (!d_ws || ws_bytes < need || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "int8: %zu bytes of 16-byte aligned workspace are needed", need);
  st = require_device();
  if (st.code || n == 0) return st;
  const Out o{d_pre, d_post, pre_stride, post_stride, rows->d_scales, l->scales, l->bias, n, l->out, l->act};
  WH_HIP(launch_product(*l, dtype, rows->d_codes, rows->stride, o, (hipStream_t)stream));
  return ok();
}

}  // extern "C"
