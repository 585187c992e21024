// tokens.hpp — what the token-side operators (embedding.hip, adapters.hip,
// distill.hip) share: the three float types of their tables, factors and
// logits, 16-byte vectors of them, argument checks, and the order of rows by
// a key (a token, an adapter).  Internal to the library.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.hpp"
#include "runtime.hpp"

namespace wh {
namespace tok {

// ------------------------------------------------------------ element types
// The float types by dtype id (kFloat32, kFloat16, kBFloat16).  Unlike the
// store codecs, which truncate as the reference does, values rounded to 16
// bits here (the logits' gradient) round to nearest even.
struct F32 {
  using raw = uint32_t;
  static constexpr int kPer16 = 4;  // elements of 16 bytes
  __device__ static inline float get(raw v) { return u2f(v); }
  __device__ static inline raw put(float v) { return f2u(v); }
};
struct F16 {
  using raw = uint16_t;
  static constexpr int kPer16 = 8;
  __device__ static inline float get(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  __device__ static inline raw put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};
struct BF16 {
  using raw = uint16_t;
  static constexpr int kPer16 = 8;
  __device__ static inline float get(raw v) { return u2f((uint32_t)v << 16); }
  __device__ static inline raw put(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};

// Elements of one 16-byte word, and back.
template <class T>
__device__ inline void unpack16(const uint4 &v, float (&f)[T::kPer16]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < T::kPer16; ++i) {
    if constexpr (T::kPer16 == 4) f[i] = T::get(w[i]);
    else f[i] = T::get((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
  }
}
template <class T>
__device__ inline uint4 pack16(const float (&f)[T::kPer16]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T::kPer16 == 4) w[i] = T::put(f[i]);
    else w[i] = (uint32_t)T::put(f[2 * i]) | ((uint32_t)T::put(f[2 * i + 1]) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

inline bool float_type(int32_t dtype) {
  return dtype == kFloat32 || dtype == kFloat16 || dtype == kBFloat16;
}
inline int float_size(int32_t dtype) { return dtype == kFloat32 ? 4 : 2; }
inline bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Calls F.template operator()<T>() for the dtype's element type.
template <class F>
inline auto with_type(int32_t dtype, F &&f) {
  return dtype == kFloat32 ? f(F32{}) : dtype == kFloat16 ? f(F16{}) : f(BF16{});
}

// ------------------------------------------------------------- row order
// order[p] = the p-th row by (key, row), skey[p] its key; keys outside
// [0, limit) count as `limit` and come last.  The order of equal keys is the
// rows' own, so sums over a key's rows are the same on every run.
//
// Ranks are counted, not sorted: a row's place among kChunk rows is the number
// of rows before it, one compare and one add per pair.  A block takes 64 rows,
// one a lane, and its 16 waves a sixteenth of the chunk each, whose keys are
// wave-uniform (scalar) operands.  More rows than a chunk: each chunk by
// itself, then every row's places in the other chunks by binary search there.
constexpr int kChunk = 4096;

static __global__ void __launch_bounds__(1024) rank_kernel(const int32_t *__restrict__ key, int n, uint32_t limit,
                                                    int32_t *__restrict__ skey, int32_t *__restrict__ order) {
  __shared__ int count[16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = blockIdx.x * 64 + lane;
  const int begin = blockIdx.x * 64 / kChunk * kChunk, end = min(begin + kChunk, n);
  const uint32_t mine = i < n ? min((uint32_t)key[i], limit) : limit;
  const int per = (((end - begin) + 15) / 16 + 63) & ~63;  // this wave's rows, whole groups of 64
  const int lo = min(begin + wave * per, end), hi = min(lo + per, end);
  const int own = blockIdx.x * 64;
  int less = 0;
  for (int j0 = lo; j0 < hi; j0 += 64) {
    const int stop = min(j0 + 64, hi);
    if (j0 == own) {
      for (int j = j0; j < stop; ++j) {
        const uint32_t u = min((uint32_t)key[j], limit);
        less += (u < mine || (u == mine && j < i)) ? 1 : 0;
      }
    } else {
      const uint32_t bound = mine + (j0 < own ? 1u : 0u);  // equal keys of earlier rows come first
      int j = j0;
      for (; j + 8 <= stop; j += 8) {
#pragma unroll
        for (int k = 0; k < 8; ++k) less += min((uint32_t)key[j + k], limit) < bound ? 1 : 0;
      }
      for (; j < stop; ++j) less += min((uint32_t)key[j], limit) < bound ? 1 : 0;
    }
  }
  count[wave][lane] = less;
  __syncthreads();
  if (wave == 0 && i < n) {
    int at = begin;
#pragma unroll
    for (int w = 0; w < 16; ++w) at += count[w][lane];
    skey[at] = (int32_t)mine;
    order[at] = i;
  }
}

// Joins the sorted chunks: a row's place is its place in its own chunk plus
// the rows before it in each other one (equal keys of earlier chunks first).
constexpr int kMergeStage = 4;  // chunks in LDS at a time
static __global__ void __launch_bounds__(1024) merge_kernel(const int32_t *__restrict__ ckey,
                                                     const int32_t *__restrict__ corder, int n,
                                                     int32_t *__restrict__ skey, int32_t *__restrict__ order) {
  __shared__ int32_t keys[kMergeStage * kChunk];
  const int p = blockIdx.x * 1024 + threadIdx.x;
  const int own = p / kChunk;
  const int32_t mine = p < n ? ckey[p] : 0;
  int at = p - own * kChunk;
  for (int s0 = 0; s0 < n; s0 += kMergeStage * kChunk) {
    const int len = min(kMergeStage * kChunk, n - s0);
    __syncthreads();
    for (int j = threadIdx.x; j < len; j += 1024) keys[j] = ckey[s0 + j];
    __syncthreads();
    if (p >= n) continue;
    for (int c0 = 0; c0 < len; c0 += kChunk) {
      const int c = (s0 + c0) / kChunk;
      if (c == own) continue;
      const int bound = mine + (c < own ? 1 : 0);  // keys are below 2^31: no overflow past limit
      int lo = 0, hi = min(kChunk, len - c0);      // the first place whose key is >= bound
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (keys[c0 + mid] < bound) lo = mid + 1;
        else hi = mid;
      }
      at += lo;
    }
  }
  if (p < n) {
    skey[at] = mine;
    order[at] = corder[p];
  }
}

inline size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }
// Workspace of the order: skey, order and, past one chunk, the chunks'.
inline size_t order_bytes(int64_t n) { return pad256((size_t)n * 4) * (n > kChunk ? 4 : 2); }
struct Order {
  int32_t *skey, *order;
};
inline hipError_t launch_order(const int32_t *key, int n, int32_t limit, void *ws, Order *out, hipStream_t s) {
  const size_t step = pad256((size_t)n * 4);
  char *p = (char *)ws;
  out->skey = (int32_t *)p;
  out->order = (int32_t *)(p + step);
  const bool one = n <= kChunk;
  int32_t *ck = one ? out->skey : (int32_t *)(p + 2 * step), *co = one ? out->order : (int32_t *)(p + 3 * step);
  rank_kernel<<<(n + 63) / 64, 1024, 0, s>>>(key, n, (uint32_t)limit, ck, co);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || one) return e;
  merge_kernel<<<(n + 1023) / 1024, 1024, 0, s>>>(ck, co, n, out->skey, out->order);
  return hipGetLastError();
}

}  // namespace tok
}  // namespace wh
