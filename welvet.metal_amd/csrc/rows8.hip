// rows8.hip — rows of activations in 8 bits: stored, read back, and SwiGLU's
// product between them in both directions.  For a row x:
//   s = max |x| / 127,  c_i = x_i / s to nearest even,  value s c_i
//   h = silu(gate) up;  dgate = dh up silu'(gate),  dup = dh silu(gate)
// Bound by HBM: a row a block, read once into registers, its largest magnitude
// joined across the block, then its codes written.  bf16 8192 x 11008: stored 66 us
// (4.1 TB/s), read back 43, SwiGLU with both kept 147 (4.9 TB/s), its backward 120
// (6); with h in 8 bits beside both 171 to 195, by the values, as its products are formed
// twice.  A few rows
// take 2.5 to 6 us, the launch and one row's loads, join and stores.
#include <hip/hip_runtime.h>

#include "rows8.hpp"

namespace wh {
namespace r8 {
namespace {

// The block's maximum of each value, on every thread.  `lds` alternates
// between a block's rows, so one barrier a row is enough.
template <int WAVES, int N>
__device__ inline void block_max(uint32_t (&top)[N], uint32_t *lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], off));
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) lds[i * WAVES + (threadIdx.x >> 6)] = top[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top[i] = max(top[i], lds[i * WAVES + w]);
  }
}

struct StoreArgs {
  const void *x;
  int64_t x_stride;
  int8_t *codes;
  int64_t codes_stride;
  float *scales;
  int n, width;
};

// GROUPS of eight values a thread stay in registers; a longer row is read again.
template <class T, int WAVES, int GROUPS>
__global__ void __launch_bounds__(WAVES * 64) store_kernel(StoreArgs a) {
  constexpr int kThreads = WAVES * 64;
  __shared__ uint32_t lds[2][WAVES];
  const Eights e(a.width);
  const int tid = threadIdx.x;
  int turn = 0;
  for (int row = blockIdx.x; row < a.n; row += gridDim.x, turn ^= 1) {
    const typename T::raw *x = (const typename T::raw *)a.x + (int64_t)row * a.x_stride;
    int8_t *codes = a.codes + (int64_t)row * a.codes_stride;
    Oct<T> held[GROUPS], rest;
    uint32_t top[1] = {0};
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      if (g * kThreads < e.whole) e.load(held[g], x, g * kThreads + tid);
    if (e.left && tid == 0) {
      rest.load(x, e.whole * 8, a.width);
      raise(top[0], rest);
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      if (g * kThreads < e.whole) raise(top[0], held[g]);
    for (int g = GROUPS * kThreads; g < e.whole; g += kThreads) {
      Oct<T> o;
      e.load(o, x, g + tid);
      raise(top[0], o);
    }
    top[0] = widened<T>(top[0]);
    block_max<WAVES>(top, lds[turn]);
    const Scale q(top[0]);
    if (tid == 0) {
      a.scales[row] = q.stored;
      e.finish(codes, q, rest);
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      if (g * kThreads + tid < e.whole) {
        issued();  // a group at a time: side by side their sums take twice the registers
        *(uint2 *)(codes + (g * kThreads + tid) * 8) = codes8(q, [&](int i) { return held[g].get(i); });
      }
    for (int g = GROUPS * kThreads + tid; g < e.whole; g += kThreads) {
      Oct<T> o;
      e.load(o, x, g);
      *(uint2 *)(codes + g * 8) = codes8(q, [&](int i) { return o.get(i); });
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) load_kernel(StoreArgs a, int per_row) {
  typename T::raw *x = (typename T::raw *)a.x;
  const int64_t all = (int64_t)a.n * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int c = (int)(i - row * per_row) * 8;
    const uint2 w = *(const uint2 *)(a.codes + row * a.codes_stride + c);
    const float s = a.scales[row];
    Oct<T> o;
#pragma unroll
    for (int k = 0; k < 8; ++k) o.set(k, value_of(k < 4 ? w.x : w.y, k & 3) * s);
    o.store(x + row * a.x_stride, c, a.width);
  }
}

struct SwigluArgs {
  const void *gate, *up;
  int64_t gate_stride, up_stride;
  welvet_hip_rows8 gate8, up8, h8;  // d_codes null: not asked for
  void *h;
  int64_t h_stride;
  int n, width;
};
template <class T>
__device__ inline void products(const Oct<T> &gate, const Oct<T> &up, float (&h)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = gate.get(i);
  acts<T, kSilu>(h);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] *= up.get(i);
}

// H8: h's own rows are asked for; its products are formed again for their codes
// (kept, they cost registers for one block a CU instead of two).
template <class T, int WAVES, int GROUPS, bool H8>
__global__ void __launch_bounds__(WAVES * 64) swiglu_kernel(SwigluArgs a) {
  constexpr int kThreads = WAVES * 64;
  using raw = typename T::raw;
  __shared__ uint32_t lds[2][3 * WAVES];
  const Eights e(a.width);
  const int tid = threadIdx.x;
  int turn = 0;
  for (int row = blockIdx.x; row < a.n; row += gridDim.x, turn ^= 1) {
    const raw *gate = (const raw *)a.gate + (int64_t)row * a.gate_stride;
    const raw *up = (const raw *)a.up + (int64_t)row * a.up_stride;
    raw *h = a.h ? (raw *)a.h + (int64_t)row * a.h_stride : nullptr;
    Oct<T> g[GROUPS], u[GROUPS], grest, urest;
    uint32_t top[3] = {0, 0, 0};
    // at: the place of the eight, -1 where another thread has them
    const auto look = [&](const Oct<T> &go, const Oct<T> &uo, int at, int width) {
      raise(top[0], go);
      raise(top[1], uo);
      if (!H8 && !h) return;
      float p[8];
      products(go, uo, p);
      Oct<T> ho;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (H8) top[2] = max(top[2], magnitude(p[i]));
        ho.set(i, p[i]);
      }
      if (h && at >= 0) ho.store(h, at * 8, width);
    };
    const auto place = [&](int at) { return at < e.whole ? at : -1; };
#pragma unroll
    for (int k = 0; k < GROUPS; ++k)
      if (k * kThreads < e.whole) {
        e.load(g[k], gate, k * kThreads + tid);
        e.load(u[k], up, k * kThreads + tid);
      }
    if (e.left && tid == 0) {
      grest.load(gate, e.whole * 8, a.width);
      urest.load(up, e.whole * 8, a.width);
      look(grest, urest, e.whole, a.width);
    }
#pragma unroll
    for (int k = 0; k < GROUPS; ++k)
      if (k * kThreads < e.whole) {
        issued();
        look(g[k], u[k], place(k * kThreads + tid), INT32_MAX);
      }
    for (int k = GROUPS * kThreads; k < e.whole; k += kThreads) {
      Oct<T> go, uo;
      e.load(go, gate, k + tid);
      e.load(uo, up, k + tid);
      look(go, uo, place(k + tid), INT32_MAX);
    }
    top[0] = widened<T>(top[0]);
    top[1] = widened<T>(top[1]);
    block_max<WAVES>(top, lds[turn]);
    const Scale qg(top[0]), qu(top[1]), qh(top[2]);
    int8_t *gc = a.gate8.d_codes ? a.gate8.d_codes + row * a.gate8.stride : nullptr;
    int8_t *uc = a.up8.d_codes ? a.up8.d_codes + row * a.up8.stride : nullptr;
    int8_t *hc = H8 ? a.h8.d_codes + row * a.h8.stride : nullptr;
    if (tid == 0) {
      if (gc) {
        a.gate8.d_scales[row] = qg.stored;
        e.finish(gc, qg, grest);
      }
      if (uc) {
        a.up8.d_scales[row] = qu.stored;
        e.finish(uc, qu, urest);
      }
      if constexpr (H8) {
        a.h8.d_scales[row] = qh.stored;
        Oct<F32> hrest;
        if (e.left) {
          float p[8];
          products(grest, urest, p);
#pragma unroll
          for (int i = 0; i < 8; ++i) hrest.set(i, p[i]);
        }
        e.finish(hc, qh, hrest);
      }
    }
    const auto write = [&](const Oct<T> &go, const Oct<T> &uo, int at) {
      if (gc) *(uint2 *)(gc + at * 8) = codes8(qg, [&](int i) { return go.get(i); });
      if (uc) *(uint2 *)(uc + at * 8) = codes8(qu, [&](int i) { return uo.get(i); });
      if constexpr (H8) {
        float p[8];
        products(go, uo, p);
        *(uint2 *)(hc + at * 8) = codes8(qh, [&](int i) { return p[i]; });
      }
    };
#pragma unroll
    for (int k = 0; k < GROUPS; ++k)
      if (k * kThreads + tid < e.whole) {
        issued();  // a group at a time: side by side their sums take twice the registers
        write(g[k], u[k], k * kThreads + tid);
      }
    for (int k = GROUPS * kThreads + tid; k < e.whole; k += kThreads) {
      Oct<T> go, uo;
      e.load(go, gate, k);
      e.load(uo, up, k);
      write(go, uo, k);
    }
  }
}

struct SwigluBackArgs {
  welvet_hip_rows8 gate8, up8;
  const void *dh;
  int64_t dh_stride;
  void *dgate, *dup;
  int64_t dgate_stride, dup_stride;
  int n, width;
};
template <class T>
__global__ void __launch_bounds__(256) swiglu_backward_kernel(SwigluBackArgs a, int per_row) {
  using raw = typename T::raw;
  const int64_t all = (int64_t)a.n * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int c = (int)(i - row * per_row) * 8;
    const uint2 gw = *(const uint2 *)(a.gate8.d_codes + row * a.gate8.stride + c);
    const uint2 uw = *(const uint2 *)(a.up8.d_codes + row * a.up8.stride + c);
    const float gs = a.gate8.d_scales[row], us = a.up8.d_scales[row];
    Oct<T> d, dg, du;
    d.load((const raw *)a.dh + row * a.dh_stride, c, a.width);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float g = value_of(k < 4 ? gw.x : gw.y, k & 3) * gs, u = value_of(k < 4 ? uw.x : uw.y, k & 3) * us;
      const Sigmoid z(g);
      dg.set(k, d.get(k) * u * fmaf(g * z.z, z.co, z.z));
      du.set(k, d.get(k) * (g * z.z));
    }
    dg.store((raw *)a.dgate + row * a.dgate_stride, c, a.width);
    du.store((raw *)a.dup + row * a.dup_stride, c, a.width);
  }
}

unsigned row_blocks(int n) { return (unsigned)std::min(n, 65536); }
template <class T, bool H8>
hipError_t launch_swiglu(const SwigluArgs &a, hipStream_t s) {
  const unsigned blocks = row_blocks(a.n);
  if (a.width <= 1024) swiglu_kernel<T, 2, 1, H8><<<blocks, 128, 0, s>>>(a);
  else if (a.width <= 4096) swiglu_kernel<T, 4, 2, H8><<<blocks, 256, 0, s>>>(a);
  else if (a.width <= 12288) swiglu_kernel<T, 8, 3, H8><<<blocks, 512, 0, s>>>(a);
  else swiglu_kernel<T, 16, 2, H8><<<blocks, 1024, 0, s>>>(a);
  return hipGetLastError();
}
// Blocks of a kernel that walks `all` items 256 at a time.
unsigned walk_blocks(int64_t all) { return (unsigned)std::min<int64_t>((all + 255) / 256, 65536); }

}  // namespace

hipError_t launch_store(int32_t dtype, int32_t n, int32_t width, const void *x, int64_t x_stride, int8_t *codes,
                        int64_t codes_stride, float *scales, hipStream_t s) {
  const StoreArgs a{x, x_stride, codes, codes_stride, scales, n, width};
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    // the block that holds the row in registers; of few long rows, more waves (bf16
    // 11008, us with four waves and sixteen: 64 rows 8.5 / 4.6, 512 9.6 / 8.1, 1024
    // 12.2 / 14.4; 4096 the same up to 256 rows, 4.7 / 5.5 of 384)
    if (width <= 1024) store_kernel<T, 2, 1><<<row_blocks(n), 128, 0, s>>>(a);
    else if (width <= 4096) store_kernel<T, 4, 2><<<row_blocks(n), 256, 0, s>>>(a);
    else if (width <= 16384 && n <= 512) store_kernel<T, 16, 2><<<row_blocks(n), 1024, 0, s>>>(a);
    else if (width <= 8192) store_kernel<T, 4, 4><<<row_blocks(n), 256, 0, s>>>(a);
    else if (width <= 12288) store_kernel<T, 4, 6><<<row_blocks(n), 256, 0, s>>>(a);
    else store_kernel<T, 16, 4><<<row_blocks(n), 1024, 0, s>>>(a);
    return hipGetLastError();
  });
}

}  // namespace r8
}  // namespace wh

using namespace wh;
using namespace wh::rt;

namespace {
// What the rows' calls share: the type, the size, a float matrix of rows.
bool matrix_ok(const void *p, int64_t stride, int32_t n, int32_t width) { return n == 0 || (p && stride >= width); }
}  // namespace

extern "C" {

welvet_status welvet_hip_rows8_store(int32_t dtype, int32_t n, int32_t width, const void *d_x, int64_t x_stride,
                                     const welvet_hip_rows8 *rows, void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "rows8: unsupported dtype %d", dtype);
  if (!r8::size_ok(n, width) || !matrix_ok(d_x, x_stride, n, width)) return make_status(kInvalid, "rows8: invalid argument");
  if (const char *why = r8::rows_fault(rows, n, width)) return make_status(kInvalid, "rows8: %s", why);
  if (!tok::aligned(d_x, tok::float_size(dtype)))
    return make_status(kInvalid, "rows8: device pointers must be aligned to their elements");
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  WH_HIP(r8::launch_store(dtype, n, width, d_x, x_stride, rows->d_codes, rows->stride, rows->d_scales,
                          (hipStream_t)stream));
  return ok();
}

welvet_status welvet_hip_rows8_load(int32_t dtype, int32_t n, int32_t width, const welvet_hip_rows8 *rows, void *d_x,
                                    int64_t x_stride, void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "rows8: unsupported dtype %d", dtype);
  if (!r8::size_ok(n, width) || !matrix_ok(d_x, x_stride, n, width)) return make_status(kInvalid, "rows8: invalid argument");
  if (const char *why = r8::rows_fault(rows, n, width)) return make_status(kInvalid, "rows8: %s", why);
  if (!tok::aligned(d_x, tok::float_size(dtype)))
    return make_status(kInvalid, "rows8: device pointers must be aligned to their elements");
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  const int per_row = (width + 7) / 8;
  const r8::StoreArgs a{d_x, x_stride, rows->d_codes, rows->stride, rows->d_scales, n, width};
  WH_HIP(tok::with_type(dtype, [&](auto t) {
    r8::load_kernel<decltype(t)><<<r8::walk_blocks((int64_t)n * per_row), 256, 0, (hipStream_t)stream>>>(a, per_row);
    return hipGetLastError();
  }));
  return ok();
}

welvet_status welvet_hip_rows8_swiglu(int32_t dtype, int32_t n, int32_t width, const void *d_gate, int64_t gate_stride,
                                      const void *d_up, int64_t up_stride, const welvet_hip_rows8 *gate8,
                                      const welvet_hip_rows8 *up8, const welvet_hip_rows8 *h8, void *d_h,
                                      int64_t h_stride, void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "rows8 swiglu: unsupported dtype %d", dtype);
  if (!r8::size_ok(n, width) || !matrix_ok(d_gate, gate_stride, n, width) || !matrix_ok(d_up, up_stride, n, width) ||
      (!gate8 && !up8 && !h8 && !d_h) || (d_h && h_stride < width))
    return make_status(kInvalid, "rows8 swiglu: invalid argument");
  for (const welvet_hip_rows8 *r : {gate8, up8, h8})
    if (const char *why = r ? r8::rows_fault(r, n, width) : nullptr)
      return make_status(kInvalid, "rows8 swiglu: %s", why);
  // a row's last values are looked at by more than one thread, and in long rows twice:
  // h in their place only where nothing but h depends on them
  if (n > 0 && d_h && (d_h == d_gate || d_h == d_up)) {
    if (gate8 || up8 || h8) return make_status(kInvalid, "rows8 swiglu: h in an input's place where rows are asked for");
    if (n > 1 && h_stride != (d_h == d_gate ? gate_stride : up_stride))
      return make_status(kInvalid, "rows8 swiglu: h in an input's place needs its row stride");
  }
  const int size = tok::float_size(dtype);
  if (!tok::aligned(d_gate, size) || !tok::aligned(d_up, size) || !tok::aligned(d_h, size))
    return make_status(kInvalid, "rows8 swiglu: device pointers must be aligned to their elements");
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  const welvet_hip_rows8 none{};
  const r8::SwigluArgs a{d_gate, d_up, gate_stride, up_stride, gate8 ? *gate8 : none, up8 ? *up8 : none,
                         h8 ? *h8 : none, d_h, h_stride, n, width};
  WH_HIP(tok::with_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipStream_t s = (hipStream_t)stream;
    return h8 ? r8::launch_swiglu<T, true>(a, s) : r8::launch_swiglu<T, false>(a, s);
  }));
  return ok();
}

welvet_status welvet_hip_rows8_swiglu_backward(int32_t dtype, int32_t n, int32_t width, const welvet_hip_rows8 *gate8,
                                               const welvet_hip_rows8 *up8, const void *d_dh, int64_t dh_stride,
                                               void *d_dgate, int64_t dgate_stride, void *d_dup, int64_t dup_stride,
                                               void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "rows8 swiglu: unsupported dtype %d", dtype);
  if (!r8::size_ok(n, width) || !matrix_ok(d_dh, dh_stride, n, width) || !matrix_ok(d_dgate, dgate_stride, n, width) ||
      !matrix_ok(d_dup, dup_stride, n, width) || (n > 0 && d_dgate == d_dup))
    return make_status(kInvalid, "rows8 swiglu: invalid argument");
  for (const welvet_hip_rows8 *r : {gate8, up8})
    if (const char *why = r8::rows_fault(r, n, width)) return make_status(kInvalid, "rows8 swiglu: %s", why);
  if (n > 1 && ((d_dgate == d_dh && dgate_stride != dh_stride) || (d_dup == d_dh && dup_stride != dh_stride)))
    return make_status(kInvalid, "rows8 swiglu: a gradient in the place of dh needs its row stride");
  const int size = tok::float_size(dtype);
  if (!tok::aligned(d_dh, size) || !tok::aligned(d_dgate, size) || !tok::aligned(d_dup, size))
    return make_status(kInvalid, "rows8 swiglu: device pointers must be aligned to their elements");
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  const int per_row = (width + 7) / 8;
  const r8::SwigluBackArgs a{*gate8, *up8, d_dh, dh_stride, d_dgate, d_dup, dgate_stride, dup_stride, n, width};
  WH_HIP(tok::with_type(dtype, [&](auto t) {
    r8::swiglu_backward_kernel<decltype(t)>
        <<<r8::walk_blocks((int64_t)n * per_row), 256, 0, (hipStream_t)stream>>>(a, per_row);
    return hipGetLastError();
  }));
  return ok();
}

}  // extern "C"
