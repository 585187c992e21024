// embedding.hip — rows of a table by token, scaled, and the table's gradient.
//   forward   out[t] = scale * table[token[t]]
//   gradient  dtable[v] = scale * sum of dout[t] over the t with token[t] = v
// A token outside [0, vocab) is padding: its output row is zero and its
// gradient row is left out.  The forward only moves bytes; the gradient adds
// one f32 per value of dout and writes the table's rows, so both are bound by
// HBM and every value is read and written once (16384 tokens: lookups of 1024
// f32 15.4 us, 134 MB; gradient of 4096 into 32000 rows 175 us, 793 MB at 4.5
// TB/s).  Few tokens are bound by the launch (8 tokens of 4096 bf16: 7.7 us).
#include <hip/hip_runtime.h>

#include "codec.hpp"
#include "tokens.hpp"

namespace wh {
namespace {

using namespace tok;

// ---------------------------------------------------------------- forward
// A block takes ROWS tokens and a column tile; a thread four columns of each
// row, all rows' loads in flight before the first store.
template <class T, int ROWS, bool NARROW, bool NT>
__global__ void __launch_bounds__(256) lookup_kernel(const typename T::raw *__restrict__ table, int64_t tstride,
                                                     uint32_t vocab, int dim, const int32_t *__restrict__ tokens,
                                                     int n, float scale, float *__restrict__ out, int64_t ostride,
                                                     int tiles) {
  const int group = blockIdx.x / tiles;
  const Cols<NARROW> cols((blockIdx.x % tiles * blockDim.x + threadIdx.x) * 4, dim);
  if (!cols.any()) return;
  Quad<T> v[ROWS];
  uint32_t id[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) id[r] = (uint32_t)tokens[min(group * ROWS + r, n - 1)];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)  // padding reads row 0
    v[r] = cols.template load<T>(table + (int64_t)(id[r] < vocab ? id[r] : 0) * tstride);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int t = group * ROWS + r;
    if (t >= n) break;
    // padding is +0, also under a negative scale
    cols.template store<NT>(out + (int64_t)t * ostride, keep4(id[r] < vocab, mul4(v[r].floats(), scale)));
  }
}

// The same from a packed store: any of the 34 formats, one element at a time
// (a lookup reads a few rows; what the formats cost is their bit offsets).
template <int DT>
__global__ void __launch_bounds__(256) store_lookup_kernel(const uint8_t *__restrict__ body, float wscale,
                                                           float minv, uint32_t vocab, int dim,
                                                           const int32_t *__restrict__ tokens, float scale,
                                                           float *__restrict__ out, int64_t ostride, int tiles) {
  const int t = blockIdx.x / tiles;
  const uint32_t id = (uint32_t)tokens[t];
  const int c0 = blockIdx.x % tiles * 1024 + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + 256 * i;
    if (c >= dim) break;
    float v = 0.0f;
    if (id < vocab) v = dec_code<DT>(load_code<DT>(body, (int64_t)id * dim + c), wscale, minv) * scale;
    out[(int64_t)t * ostride + c] = v;
  }
}

template <int DT = 0>
hipError_t launch_store_lookup(const DevStore &w, const int32_t *tokens, int n, float scale, float *out,
                               int64_t ostride, hipStream_t s) {
  if constexpr (DT < kNumDTypes) {
    if (w.dtype != DT) return launch_store_lookup<DT + 1>(w, tokens, n, scale, out, ostride, s);
    const int tiles = (w.cols + 1023) / 1024;
    store_lookup_kernel<DT><<<(uint32_t)((int64_t)n * tiles), 256, 0, s>>>(
        w.body, w.scale, w.minv, (uint32_t)w.rows, w.cols, tokens, scale, out, ostride, tiles);
    return hipGetLastError();
  } else {
    return hipErrorInvalidValue;
  }
}

// --------------------------------------------------------------- gradient
// Few tokens: a block takes one of them and a column tile, and where it is
// the first of its token adds up that token's rows.
constexpr int kDirect = 256;
// More: rows in the tokens' order, kRun of them a block and column tile.  A
// token whose rows end inside the block's is written from registers; one that
// reaches into a neighbour's leaves a partial row (slot 0: began earlier,
// slot 1: goes on), and finish_kernel adds those up, in order.
constexpr int kRun = 32;
constexpr int kZeroRows = 4;  // table rows of a zeroing block

template <bool ACC, bool NT, bool NARROW>
__device__ inline void put_row(const Cols<NARROW> &cols, float *row, const float4 &sum, float scale) {
  float4 v = mul4(sum, scale);
  if constexpr (ACC) v = add4(cols.load(row), v);
  cols.template store<NT>(row, v);
}

// A block's zeros into `len` floats, each store a part of one cache line (rows
// of 4099 floats from their own start on: 224 us against 154 for a table of
// 50000).
template <bool NT>
__device__ inline void zero_span(float *p, int len) {
  const float4 zero = make_float4(0, 0, 0, 0);
  const int head = (int)((uintptr_t)p >> 2 & 31);  // floats past a line's start
  for (int c = 4 * (int)threadIdx.x - head; c < len; c += 4 * blockDim.x) {
    if (c >= 0 && c + 4 <= len) {
      if constexpr (NT) store4_nt(p + c, zero);
      else store4(p + c, zero);
    } else {
      for (int i = max(0, -c); i < 4 && c + i < len; ++i) p[c + i] = 0.0f;
    }
  }
}
// Zeros everywhere, ahead of the rows that tokens name: where they are few, a
// table written at the rate of a fill and those rows a second time take less
// than looking each row up among the tokens.  32000 x 4096, fill against lookups
// (us), tokens as many as a 16th of the rows 103 / 113, an 8th 120 / 121, a
// quarter 148 / 132; 68880 x 3340: 177 / 209, 205 / 223, 257 / 247; 2 tokens 135 /
// 171 (skewed tokens; uniform ones a few us further towards the lookups).
// One store a thread in blocks that follow the addresses reaches 6.9 TB/s; four
// a thread 6.0, sixteen 5.3.
__global__ void __launch_bounds__(256) fill_kernel(uint32_t vocab, int dim, float *__restrict__ table, int64_t stride,
                                                   int64_t blocks) {
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const uint32_t at = (uint32_t)(b * 1024 % dim) + 4 * threadIdx.x;
    uint32_t row = (uint32_t)(b * 1024 / dim) + at / (uint32_t)dim, c = at % (uint32_t)dim;
    if (row < vocab && c + 4 <= (uint32_t)dim) {
      store4(table + (int64_t)row * stride + c, make_float4(0, 0, 0, 0));
    } else {
      for (int i = 0; i < 4 && row < vocab; ++i) {
        table[(int64_t)row * stride + c] = 0.0f;
        if (++c == (uint32_t)dim) c = 0, ++row;
      }
    }
  }
}

template <bool ACC, bool NARROW>
__global__ void __launch_bounds__(256) direct_kernel(const int32_t *__restrict__ tokens, int n, uint32_t vocab,
                                                     int dim, const float *__restrict__ dout, int64_t dstride,
                                                     float scale, float *__restrict__ dtable, int64_t tstride,
                                                     int tiles) {
  __shared__ int32_t tok_s[kDirect];
  __shared__ int rows_s[kDirect];
  __shared__ int count_s;
  for (int j = threadIdx.x; j < n; j += blockDim.x) tok_s[j] = tokens[j];
  const int adders = n * tiles;
  if ((int)blockIdx.x >= adders) {  // rows without a token
    __shared__ int named[kZeroRows];
    if (threadIdx.x < kZeroRows) named[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t v0 = ((uint32_t)blockIdx.x - (uint32_t)adders) * kZeroRows;
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
      const uint32_t d = (uint32_t)tok_s[j] - v0;
      if (d < kZeroRows) named[d] = 1;
    }
    __syncthreads();
    for (int r = 0; r < kZeroRows && v0 + r < vocab; ++r)
      if (!named[r]) zero_span<false>(dtable + (int64_t)(v0 + r) * tstride, dim);
    return;
  }
  if (threadIdx.x == 0) count_s = 0;
  __syncthreads();
  const int i = blockIdx.x / tiles;
  const int32_t mine = tok_s[i];
  if ((uint32_t)mine >= vocab) return;
  if (threadIdx.x < 64) {  // this token's rows, in order
    int count = 0;
    bool first = true;
    for (int j0 = 0; j0 < n; j0 += 64) {
      const int j = j0 + threadIdx.x;
      const uint64_t same = __ballot(j < n && tok_s[j] == mine);
      const uint64_t below = threadIdx.x ? ~0ull >> (64 - threadIdx.x) : 0ull;
      if (j < n && tok_s[j] == mine) rows_s[count + __popcll(same & below)] = j;
      if (count == 0 && same) first = j0 + __ffsll((long long)same) - 1 == i;
      count += __popcll(same);
    }
    if (threadIdx.x == 0) count_s = first ? count : 0;
  }
  __syncthreads();
  const int count = count_s;
  const Cols<NARROW> cols((blockIdx.x % tiles * blockDim.x + threadIdx.x) * 4, dim);
  if (count == 0 || !cols.any()) return;
  float4 sum = make_float4(0, 0, 0, 0);
  int r = 0;
  for (; r + 4 <= count; r += 4) {
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = cols.load(dout + (int64_t)rows_s[r + k] * dstride);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum = add4(sum, v[k]);
  }
  for (; r < count; ++r) sum = add4(sum, cols.load(dout + (int64_t)rows_s[r] * dstride));
  put_row<ACC, false>(cols, dtable + (int64_t)mine * tstride, sum, scale);
}

template <bool ACC, bool NARROW, bool NT>
__global__ void __launch_bounds__(256) sums_kernel(const int32_t *__restrict__ skey,
                                                   const int32_t *__restrict__ order, int n, uint32_t vocab, int dim,
                                                   const float *__restrict__ dout, int64_t dstride, float scale,
                                                   float *__restrict__ dtable, int64_t tstride,
                                                   float *__restrict__ part, int tiles) {
  __shared__ int32_t key_s[kRun + 2];  // with the neighbours' nearest
  __shared__ int32_t row_s[kRun];
  const int chunk = blockIdx.x / tiles, p0 = chunk * kRun;
  if (threadIdx.x < kRun + 2) {
    const int p = p0 - 1 + (int)threadIdx.x;
    key_s[threadIdx.x] = p >= 0 && p < n ? skey[p] : -1;
  }
  if (threadIdx.x < kRun) row_s[threadIdx.x] = p0 + (int)threadIdx.x < n ? order[p0 + threadIdx.x] : 0;
  __syncthreads();
  const Cols<NARROW> cols((blockIdx.x % tiles * blockDim.x + threadIdx.x) * 4, dim);
  if (!cols.any()) return;
  const int32_t before = key_s[0], after = key_s[kRun + 1];
  int32_t cur = key_s[1];
  bool began = cur != before;
  float4 sum = make_float4(0, 0, 0, 0);
  const auto done = [&](bool goes_on) {
    if ((uint32_t)cur >= vocab) return;  // padding, or past the last row
    if (!began) cols.store(part + (int64_t)(2 * chunk) * dim, sum);
    else if (goes_on) cols.store(part + (int64_t)(2 * chunk + 1) * dim, sum);
    else put_row<ACC, NT>(cols, dtable + (int64_t)cur * tstride, sum, scale);
  };
#pragma unroll 1
  for (int r0 = 0; r0 < kRun; r0 += 8) {
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = make_float4(0, 0, 0, 0);
      if ((uint32_t)key_s[1 + r0 + k] < vocab) v[k] = cols.load(dout + (int64_t)row_s[r0 + k] * dstride);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int32_t next = key_s[1 + r0 + k];
      if (next != cur) {
        done(false);
        cur = next;
        began = true;
        sum = make_float4(0, 0, 0, 0);
      }
      sum = add4(sum, v[k]);
    }
  }
  done(cur == after);
}

// Tokens whose rows fill more than one block's: the block where one begins
// adds its later blocks' slot 0 to its own slot 1, in order.  The blocks after
// those write the rows without a token, under whose stores the joins' waits
// lie (32000 x 4096, 16384 tokens: 11 us less than a launch of its own).
template <bool ACC, bool NARROW, bool NT>
__global__ void __launch_bounds__(256) finish_kernel(const int32_t *__restrict__ skey, int n, uint32_t vocab, int dim,
                                                   const float *__restrict__ part, float scale,
                                                   float *__restrict__ dtable, int64_t tstride, int tiles, int joins) {
  if ((int)blockIdx.x >= joins) {
    __shared__ int named[kZeroRows];
    const uint32_t v0 = ((uint32_t)blockIdx.x - (uint32_t)joins) * kZeroRows;
    for (uint32_t d = threadIdx.x >> 5; d < kZeroRows; d += blockDim.x >> 5) {  // half a wave a row
      const int at = first_by_half(skey, n, (int32_t)min(v0 + d, vocab));
      if ((threadIdx.x & 31) == 0) named[d] = at < n && (uint32_t)skey[at] == v0 + d;
    }
    __syncthreads();
    for (int r = 0; r < kZeroRows && v0 + r < vocab; ++r)
      if (!named[r]) zero_span<NT>(dtable + (int64_t)(v0 + r) * tstride, dim);
    return;
  }
  const int chunk = blockIdx.x / tiles, p0 = chunk * kRun, p1 = p0 + kRun;
  if (p1 >= n) return;
  const int32_t mine = skey[p1 - 1];
  if ((uint32_t)mine >= vocab || skey[p1] != mine) return;
  if (p0 > 0 && skey[p0 - 1] == mine) return;  // began earlier
  const int last = (first_at_least(skey, n, mine + 1) - 1) / kRun;
  const Cols<NARROW> cols((blockIdx.x % tiles * blockDim.x + threadIdx.x) * 4, dim);
  if (!cols.any()) return;
  float4 sum = cols.load(part + (int64_t)(2 * chunk + 1) * dim);
  int b = chunk + 1;
  for (; b + 8 <= last + 1; b += 8) {
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = cols.load(part + (int64_t)(2 * (b + k)) * dim);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = add4(sum, v[k]);
  }
  for (; b <= last; ++b) sum = add4(sum, cols.load(part + (int64_t)(2 * b) * dim));
  put_row<ACC, NT>(cols, dtable + (int64_t)mine * tstride, sum, scale);
}

size_t gradient_bytes(int dim, int n) {
  if (n <= kDirect) return 0;
  const size_t chunks = ((size_t)n + kRun - 1) / kRun;
  return order_bytes(n) + pad256(chunks * 2 * (size_t)dim * sizeof(float));
}
constexpr int64_t kMostBlocks = 1 << 23;  // of 256 threads; more go round
constexpr int kMostZeros = 1 << 25;       // rows that a launch looks up

// The kernels' int counters, which pass a row's end by a block's step, and a
// lookup's threads (four rows each).
int threads_for(int dim) { return std::min(256, ((dim + 3) / 4 + 63) / 64 * 64); }
int64_t tiles_for(int dim) { return ((int64_t)dim + 4 * threads_for(dim) - 1) / (4 * threads_for(dim)); }
bool sizes_ok(int32_t vocab, int32_t dim, int32_t n) {
  return vocab > 0 && vocab < INT32_MAX && dim > 0 && dim <= INT32_MAX - 4095 && n >= 0 && n <= 1 << 27 &&
         ((int64_t)n + vocab) * (tiles_for(dim) + 1) < INT32_MAX &&
         ((int64_t)n + 3) / 4 * tiles_for(dim) * threads_for(dim) <= UINT32_MAX;
}
// The gradient's: the order's launch, and up to kDirect tokens a block for each
// token and tile.  Those of the zero rows beside them have 2^31 threads at most
// (kMostZeros), the sums' an eighth of a lookup's.
bool gradient_ok(int32_t vocab, int32_t dim, int32_t n) {
  return sizes_ok(vocab, dim, n) && order_launchable(n) &&
         (n > kDirect || n * tiles_for(dim) * threads_for(dim) < (int64_t)1 << 31);
}

template <bool ACC, bool NARROW>
hipError_t launch_gradient(int vocab, int dim, const int32_t *tokens, int n, float scale, const float *dout,
                           int64_t dstride, float *dtable, int64_t tstride, void *ws, hipStream_t s) {
  const int threads = threads_for(dim), tiles = (int)tiles_for(dim);
  const bool nt = (int64_t)vocab * dim * 4 > kKept;  // the table past the caches
  const bool fill = !ACC && (vocab > kMostZeros || (nt && n <= vocab / 8));
  if (fill) {
    const int64_t blocks = ((int64_t)vocab * dim + 1023) / 1024;
    fill_kernel<<<(uint32_t)std::min(blocks, kMostBlocks), 256, 0, s>>>((uint32_t)vocab, dim, dtable, tstride, blocks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int64_t zeros = ACC || fill ? 0 : ((int64_t)vocab + kZeroRows - 1) / kZeroRows;
  if (n <= kDirect) {
    if ((int64_t)n * tiles + zeros == 0) return hipSuccess;
    direct_kernel<ACC, NARROW><<<(uint32_t)((int64_t)n * tiles + zeros), threads, 0, s>>>(
        tokens, n, (uint32_t)vocab, dim, dout, dstride, scale, dtable, tstride, tiles);
    return hipGetLastError();
  }
  Order o;
  hipError_t e = launch_order(tokens, n, vocab, ws, &o, s);
  if (e != hipSuccess) return e;
  float *part = (float *)((char *)ws + order_bytes(n));
  const int64_t chunks = ((int64_t)n + kRun - 1) / kRun, blocks = chunks * tiles;
  const auto go = [&](auto past) {
    constexpr bool NT = decltype(past)::value;
    sums_kernel<ACC, NARROW, NT><<<(uint32_t)blocks, threads, 0, s>>>(
        o.skey, o.order, n, (uint32_t)vocab, dim, dout, dstride, scale, dtable, tstride, part, tiles);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    finish_kernel<ACC, NARROW, NT><<<(uint32_t)(blocks + zeros), threads, 0, s>>>(
        o.skey, n, (uint32_t)vocab, dim, part, scale, dtable, tstride, tiles, (int)blocks);
    return hipGetLastError();
  };
  return nt && !NARROW ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace
}  // namespace wh

using namespace wh;
using namespace wh::rt;

extern "C" {

welvet_status welvet_hip_embedding_forward(int32_t dtype, int32_t vocab, int32_t dim, const void *d_table,
                                           int64_t table_stride, const int32_t *d_tokens, int32_t n, float scale,
                                           float *d_out, int64_t out_stride, void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "embedding: unsupported dtype %d", dtype);
  if (!sizes_ok(vocab, dim, n) || !d_table || (n > 0 && (!d_tokens || !d_out)))
    return make_status(kInvalid, "embedding: invalid argument");
  if (table_stride < dim || out_stride < dim) return make_status(kInvalid, "embedding: row stride below dim %d", dim);
  const int size = tok::float_size(dtype);
  if (!tok::aligned(d_table, size) || !tok::aligned(d_tokens, 4) || !tok::aligned(d_out, 4))
    return make_status(kInvalid, "embedding: device pointers must be aligned to their elements");
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  const int threads = threads_for(dim), tiles = (int)tiles_for(dim);
  // four rows a block where there are blocks enough for every CU several times over
  const int rows = (int64_t)n * tiles >= 8192 ? 4 : 1;
  const uint32_t blocks = (uint32_t)(((int64_t)n + rows - 1) / rows * tiles);
  tok::with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const auto go = [&](auto kernel) {
      kernel<<<blocks, threads, 0, (hipStream_t)stream>>>((const typename T::raw *)d_table, table_stride,
                                                          (uint32_t)vocab, dim, d_tokens, n, scale, d_out, out_stride,
                                                          tiles);
    };
    if (dim < 4) rows == 4 ? go(lookup_kernel<T, 4, true, false>) : go(lookup_kernel<T, 1, true, false>);
    else if (rows == 1) go(lookup_kernel<T, 1, false, false>);
    else if ((int64_t)n * dim * 4 > tok::kKept) go(lookup_kernel<T, 4, false, true>);
    else go(lookup_kernel<T, 4, false, false>);
  });
  WH_HIP(hipGetLastError());
  return ok();
}

welvet_status welvet_hip_embedding_store_forward(welvet_dense_session *s, const int32_t *d_tokens, int32_t n,
                                                 float scale, float *d_out, int64_t out_stride, void *stream) {
  if (!s || n < 0 || (n > 0 && (!d_tokens || !d_out))) return make_status(kInvalid, "embedding: invalid argument");
  std::unique_lock<std::mutex> lock;
  const DevStore w = session_store(s, &lock);
  if ((int64_t)n * ((w.cols + 1023) / 1024) >= 1 << 24) return make_status(kInvalid, "embedding: invalid argument");
  if (out_stride < w.cols) return make_status(kInvalid, "embedding: row stride below dim %d", w.cols);
  if (!tok::aligned(d_tokens, 4) || !tok::aligned(d_out, 4))
    return make_status(kInvalid, "embedding: device pointers must be aligned to their elements");
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  WH_HIP(launch_store_lookup(w, d_tokens, n, scale, d_out, out_stride, (hipStream_t)stream));
  return ok();
}

welvet_status welvet_hip_embedding_backward_bytes(int32_t vocab, int32_t dim, int32_t n, size_t *bytes) {
  if (!gradient_ok(vocab, dim, n) || !bytes) return make_status(kInvalid, "embedding backward: invalid argument");
  *bytes = gradient_bytes(dim, n);
  return ok();
}

welvet_status welvet_hip_embedding_backward(int32_t vocab, int32_t dim, const int32_t *d_tokens, int32_t n,
                                            float scale, const float *d_dout, int64_t dout_stride, int32_t accumulate,
                                            float *d_dtable, int64_t dtable_stride, void *d_ws, size_t ws_bytes,
                                            void *stream) {
  if (!gradient_ok(vocab, dim, n) || !d_dtable || (n > 0 && (!d_tokens || !d_dout)))
    return make_status(kInvalid, "embedding backward: invalid argument");
  if (dout_stride < dim || dtable_stride < dim)
    return make_status(kInvalid, "embedding backward: row stride below dim %d", dim);
  if (!tok::aligned(d_tokens, 4) || !tok::aligned(d_dout, 4) || !tok::aligned(d_dtable, 4))
    return make_status(kInvalid, "embedding backward: device pointers must be aligned to their elements");
  const size_t need = gradient_bytes(dim, n);
  if (need > 0 && (!d_ws || ws_bytes < need || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "embedding backward: %zu bytes of 16-byte aligned workspace are needed", need);
  welvet_status st = require_device();
  if (st.code) return st;
  const auto launch = dim < 4 ? (accumulate ? launch_gradient<true, true> : launch_gradient<false, true>)
                              : (accumulate ? launch_gradient<true, false> : launch_gradient<false, false>);
  WH_HIP(launch(
      vocab, dim, d_tokens, n, scale, d_dout, dout_stride, d_dtable, dtable_stride, d_ws, (hipStream_t)stream));
  return ok();
}

}  // extern "C"
