// tokens.hpp — what the token-side operators (embedding.hip, adapters.hip,
// distill.hip) share: the three float types of their tables, factors and
// logits, 16-byte vectors of them, argument checks, and the order of rows by
// a key (a token, an adapter).  Internal to the library.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

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

// Four values wherever they lie: the hardware loads and stores words at any
// alignment of their elements, so rows of any width and stride take this path.
template <class T>
struct Quad {
  using raw = typename T::raw;
  using bits = std::conditional_t<sizeof(raw) == 4, uint4, uint2>;
  bits v;
  __device__ inline float get(int i) const {
    if constexpr (sizeof(raw) == 4) return T::get(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
    else return T::get((raw)((i < 2 ? v.x : v.y) >> (16 * (i & 1))));
  }
  __device__ inline float4 floats() const { return make_float4(get(0), get(1), get(2), get(3)); }
  __device__ static inline Quad load(const raw *p) {
    Quad q;
    __builtin_memcpy(&q.v, p, sizeof(q.v));
    return q;
  }
  // zeros in the place of the first `skip` values
  __device__ inline void drop(int skip) {
    if constexpr (sizeof(raw) == 4) {
      v.x = skip < 1 ? v.x : 0;
      v.y = skip < 2 ? v.y : 0;
      v.z = skip < 3 ? v.z : 0;
      v.w = skip < 4 ? v.w : 0;
    } else {
      v.x = skip < 1 ? v.x : skip < 2 ? v.x & 0xffff0000u : 0;
      v.y = skip < 3 ? v.y : skip < 4 ? v.y & 0xffff0000u : 0;
    }
  }
  // keeps a 16-bit quad packed through a loop: without it the compiler converts
  // it once ahead of the loop and holds twice the registers
  __device__ inline void pin() {
    if constexpr (sizeof(raw) == 2) asm volatile("" : "+v"(v.x), "+v"(v.y));
  }
  // the values at row + k, zeros from `width` on
  __device__ static inline Quad load(const raw *row, int k, int width) {
    if (k + 4 <= width) return load(row + k);
    raw r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = k + i < width ? row[k + i] : (raw)0;
    return load(r);
  }
};
__device__ inline void store4(float *p, const float4 &v) { __builtin_memcpy(p, &v, sizeof(v)); }
// The same past the caches: results larger than the L2s hold.  Chosen by a
// kernel's template argument: of two such stores on the two sides of a branch
// the compiler makes one, a plain one.
typedef float nt4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ inline void store4_nt(float *p, const float4 &v) {
  __builtin_nontemporal_store(nt4{v.x, v.y, v.z, v.w}, (nt4 *)p);
}
// Bytes of results up to which they may stay there: what the L2s hold.  Past
// them a lookup of 16384 rows x 1024 takes 15.4 us against 20.4, of 16384 x
// 4096 68 / 91, an adapter's 8192 x 4096 rows 89 / 102.  A kernel that does
// nothing but read the result right after pays for it (64 MiB: 0.6 us, 128 MiB:
// 12); a product's loads hide that.
constexpr int64_t kKept = 32 << 20;
__device__ inline void store4(float *row, int k, int width, const float4 &v) {
  if (k + 4 <= width) return store4(row + k, v);
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (k + i < width) row[k + i] = f[i];
}
__device__ inline float4 load4(const float *row, int k, int width) { return Quad<F32>::load((const uint32_t *)row, k, width).floats(); }
// A thread's four columns of a row from c on.  Where those pass the row's end
// it takes the row's last four, `skip` of them another thread's (all, past the
// end), so every load is one word without a condition; only its own are
// stored.  Rows of fewer than four columns (NARROW) go value by value.
template <bool NARROW>
struct Cols {
  int c, skip, width;
  __device__ Cols(int first, int width_) : width(width_) {
    skip = NARROW ? 0 : max(0, first + 4 - width);
    c = first - skip;
  }
  __device__ Cols(int c_, int skip_, int width_) : c(c_), skip(skip_), width(width_) {}
  __device__ bool any() const { return NARROW ? c < width : skip < 4; }
  template <class T>
  __device__ Quad<T> load(const typename T::raw *row) const {
    if constexpr (NARROW) return Quad<T>::load(row, c, width);
    else return Quad<T>::load(row + c);
  }
  __device__ float4 load(const float *row) const { return load<F32>((const uint32_t *)row).floats(); }
  template <bool NT = false>
  __device__ void store(float *row, const float4 &v) const {
    if constexpr (NARROW) return store4(row, c, width, v);
    if (skip == 0) {
      if constexpr (NT) return store4_nt(row + c, v);
      else return store4(row + c, v);
    }
    if (skip < 2) row[c + 1] = v.y;
    if (skip < 3) row[c + 2] = v.z;
    if (skip < 4) row[c + 3] = v.w;
  }
};
__device__ inline float4 add4(const float4 &a, const float4 &b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ inline float4 mul4(const float4 &a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
__device__ inline float4 fma4(float s, const float4 &a, const float4 &b) {
  return make_float4(fmaf(s, a.x, b.x), fmaf(s, a.y, b.y), fmaf(s, a.z, b.z), fmaf(s, a.w, b.w));
}
// A select that keeps no trace of the value left out.
__device__ inline float4 keep4(bool on, const float4 &v) {
  return make_float4(on ? v.x : 0.0f, on ? v.y : 0.0f, on ? v.z : 0.0f, on ? v.w : 0.0f);
}
__device__ inline float get4(const float4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
// Keeps loads in the order they are written in: a wait for the oldest of
// several steps' loads must leave the later ones in flight.
__device__ inline void issued() { __builtin_amdgcn_sched_barrier(0); }

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
// of rows before it, one compare and one add per pair.  A block takes 16 rows;
// four lanes of each of its 16 waves share a row and look at 32 keys each, in
// words of four from LDS.  More rows than a chunk: each chunk by itself, then
// every row's places in the other chunks by binary search there, four threads
// a row, up to kSpan rows.  (2048 rows: 64 rows a block and a lane a row took 8 us on 32 CUs.)
constexpr int kChunk = 2048;
constexpr int kRankRows = 16;

static __global__ void __launch_bounds__(1024) rank_kernel(const int32_t *__restrict__ key, int n, uint32_t limit,
                                                           int32_t *__restrict__ skey, int32_t *__restrict__ order) {
  __shared__ uint4 keys[kChunk / 4];
  __shared__ int count[16][kRankRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lo = lane & 15, q = lane >> 4;
  const int own = blockIdx.x * kRankRows, i = own + lo, begin = own / kChunk * kChunk;
  uint32_t *flat = (uint32_t *)keys;
  for (int j = threadIdx.x; j < kChunk; j += 1024)
    // past the end: after every row, whatever its key
    flat[j] = begin + j < n ? min((uint32_t)key[begin + j], limit) : 0xffffffffu;
  __syncthreads();
  const uint32_t mine = i < n ? flat[i - begin] : limit;
  const int at = own - begin;
  int less = 0;
#pragma unroll
  for (int w = 0; w < kChunk / 256; ++w) {
    const int word = (w * 16 + wave) * 4 + q, j = word * 4;
    const uint4 u = keys[word];
    const uint32_t bound = mine + (j < at ? 1u : 0u);  // equal keys of earlier rows come first
    less += u.x < bound ? 1 : 0;
    less += u.y < bound ? 1 : 0;
    less += u.z < bound ? 1 : 0;
    less += u.w < bound ? 1 : 0;
    if (j >= at && j < at + kRankRows) {  // the block's own rows, counted as later ones above
      less += (u.x == mine && j < at + lo) ? 1 : 0;
      less += (u.y == mine && j + 1 < at + lo) ? 1 : 0;
      less += (u.z == mine && j + 2 < at + lo) ? 1 : 0;
      less += (u.w == mine && j + 3 < at + lo) ? 1 : 0;
    }
  }
  less += __shfl_xor(less, 16);
  less += __shfl_xor(less, 32);
  if (q == 0) count[wave][lo] = less;
  __syncthreads();
  if (threadIdx.x < kRankRows && i < n) {
    int to = begin;
#pragma unroll
    for (int w = 0; w < 16; ++w) to += count[w][lo];
    skey[to] = (int32_t)mine;
    order[to] = i;
  }
}

// Joins the sorted chunks of each `span` rows (whole stages, or all rows): a
// row's place is its place in its own chunk plus the rows before it in each
// other one (equal keys of earlier chunks first).
constexpr int kStage = 8 * kChunk;  // keys in LDS at a time
static __global__ void __launch_bounds__(1024) merge_kernel(const int32_t *__restrict__ ckey,
                                                            const int32_t *__restrict__ corder, int n, int span,
                                                            int32_t *__restrict__ skey, int32_t *__restrict__ order) {
  __shared__ int4 keys4[kStage / 4];
  int32_t *keys = (int32_t *)keys4;
  const int p = blockIdx.x * 256 + (threadIdx.x >> 2), part = threadIdx.x & 3;
  const int own = p / kChunk, begin = (int)blockIdx.x * 256 / span * span, end = min(n, begin + span);
  const int32_t mine = p < n ? ckey[p] : 0;
  int at = 0;
  for (int s0 = begin; s0 < end; s0 += kStage) {
    const int len = min(kStage, end - s0);
    __syncthreads();
    for (int j = threadIdx.x; j < len / 4; j += 1024) keys4[j] = *(const int4 *)(ckey + s0 + 4 * j);
    if ((int)threadIdx.x < (len & 3)) keys[len / 4 * 4 + threadIdx.x] = ckey[s0 + len / 4 * 4 + threadIdx.x];
    __syncthreads();
    for (int c0 = part * kChunk; c0 < len; c0 += 4 * kChunk) {
      const int c = (s0 + c0) / kChunk;
      if (c == own) continue;
      const int32_t bound = mine + (c < own ? 1 : 0);  // keys are below 2^31 - 1
      int lo = 0, hi = min(kChunk, len - c0);          // the first place whose key is >= bound
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (keys[c0 + mid] < bound) lo = mid + 1;
        else hi = mid;
      }
      at += lo;
    }
  }
  at += __shfl_xor(at, 1);
  at += __shfl_xor(at, 2);
  if (p < n && part == 0) {
    at += begin + p - own * kChunk;
    skey[at] = mine;
    order[at] = corder[p];
  }
}

// Joins each eight neighbouring runs of `run` sorted rows, eight threads a row:
// every one searches a run of the row's eight in memory.
static __global__ void __launch_bounds__(256) join_kernel(const int32_t *__restrict__ rkey,
                                                          const int32_t *__restrict__ rorder, int n, int run,
                                                          int32_t *__restrict__ skey, int32_t *__restrict__ order) {
  const int p = (int)blockIdx.x * 32 + (threadIdx.x >> 3), part = threadIdx.x & 7;
  const int own = p / run, first = own / 8 * 8;
  const int32_t mine = p < n ? rkey[p] : 0;
  const int64_t begin = (int64_t)(first + part) * run;
  const int other = first + part;
  int at = 0;
  if (p < n && begin < n && other != own) {
    const int32_t *keys = rkey + begin;
    const int32_t bound = mine + (other < own ? 1 : 0);
    int hi = (int)min((int64_t)run, n - begin);
    while (at < hi) {
      const int mid = (at + hi) >> 1;
      if (keys[mid] < bound) at = mid + 1;
      else hi = mid;
    }
  }
  at += __shfl_xor(at, 1);
  at += __shfl_xor(at, 2);
  at += __shfl_xor(at, 4);
  if (p < n && part == 0) {
    at += first * run + p - own * run;
    skey[at] = mine;
    order[at] = rorder[p];
  }
}

// The first place of the sorted keys whose key is >= v, for each half of a wave
// its own v; the whole wave calls it, each half looking at 32 places a time.
__device__ inline int first_by_half(const int32_t *__restrict__ skey, int n, int32_t v) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  while (__any(lo < hi)) {
    const int step = (hi - lo + 31) / 32, p = lo + lane * step;
    const uint64_t both = __ballot(lo < hi && p < hi && skey[p] < v);
    const int below = __popc((threadIdx.x & 32) ? (uint32_t)(both >> 32) : (uint32_t)both);
    if (below == 0) {
      hi = lo;
    } else if (lo < hi) {
      hi = min(hi, lo + below * step);
      lo = lo + (below - 1) * step + 1;
    }
  }
  return lo;
}
// The sorted rows of key v, from .x up to .y; a whole wave calls it.
__device__ inline int2 rows_of(const int32_t *__restrict__ skey, int n, int32_t v) {
  const int lo = first_by_half(skey, n, v + ((threadIdx.x & 32) ? 1 : 0));
  return {__builtin_amdgcn_readlane(lo, 0), __builtin_amdgcn_readlane(lo, 32)};
}

// The first place of the sorted keys whose key is >= v; a whole wave calls it
// and looks at 64 places a time.
__device__ inline int first_at_least(const int32_t *__restrict__ skey, int n, int32_t v) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64, p = lo + lane * step;
    const int below = __popcll(__ballot(p < hi && skey[p] < v));
    if (below == 0) return lo;
    hi = min(hi, lo + below * step);
    lo = lo + (below - 1) * step + 1;
  }
  return lo;
}

// A launch takes fewer than 2^32 threads, the order's first 1024 for kRankRows rows.
inline bool order_launchable(int64_t n) { return (n + kRankRows - 1) / kRankRows * 1024 <= UINT32_MAX; }
inline size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }
// Workspace of the order: skey, order and, past one chunk, the chunks'.
inline size_t order_bytes(int64_t n) { return pad256((size_t)n * 4) * (n > kChunk ? 4 : 2); }
struct Order {
  int32_t *skey, *order;
};
// Rows up to which one launch joins all chunks; its reads grow with the square
// of the rows.  More are joined in spans of as many, eight neighbours at a time
// (a gradient's whole call, us, by spans and in one launch: 100000 rows 76 / 74,
// 131072 91 / 92, 262144 165 / 226, 2^20 708 / 2247; with spans of 32768 50000
// rows take 52.5 for 49.9).
constexpr int kSpan = 4 * kStage;
inline hipError_t launch_order(const int32_t *key, int n, int32_t limit, void *ws, Order *out, hipStream_t s) {
  const size_t step = pad256((size_t)n * 4);
  int32_t *at[4];
  for (int i = 0; i < 4; ++i) at[i] = (int32_t *)((char *)ws + i * step);
  *out = {at[0], at[1]};
  int passes = n > kChunk ? 1 : 0;  // each from one pair of arrays to the other, the last to the first
  for (int64_t run = kSpan; run < n; run *= 8) ++passes;
  int32_t *from_key = at[passes % 2 * 2], *from = at[passes % 2 * 2 + 1];
  rank_kernel<<<(n + kRankRows - 1) / kRankRows, 1024, 0, s>>>(key, n, (uint32_t)limit, from_key, from);
  hipError_t e = hipGetLastError();
  for (int64_t run = 0; e == hipSuccess && passes > 0; --passes) {
    int32_t *to_key = at[(passes - 1) % 2 * 2], *to = at[(passes - 1) % 2 * 2 + 1];
    if (run == 0) {
      merge_kernel<<<(n + 255) / 256, 1024, 0, s>>>(from_key, from, n, kSpan, to_key, to);
      run = kSpan;
    } else {
      join_kernel<<<(n + 31) / 32, 256, 0, s>>>(from_key, from, n, (int)run, to_key, to);
      run *= 8;
    }
    e = hipGetLastError();
    from_key = to_key;
    from = to;
  }
  return e;
}

}  // namespace tok
}  // namespace wh
