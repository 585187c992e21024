// distill.hip — the loss of a student's logits against a teacher's top ones,
// and the logits' gradient.  For a row of logits z over the vocabulary and
// the teacher's k entries (index i, logit l_i) at temperature T:
//   q_i = exp(l_i / T - L), L the log-sum of the row's entries, or the
//         teacher's own over its whole vocabulary where that is given
//   p   = softmax(z / T)
//   loss = w T^2 sum_i q_i (log q_i - log p_i)
//   dz_v = w T (p_v sum_i q_i - sum of the q_i of index v)
// An entry with an index outside the vocabulary or a logit of -inf is absent;
// a row without one, or of weight 0, has loss 0 and gradient 0.
//
// A row's maximum and sum of exponentials are one pass over it (each thread a
// running pair, joined across the block), the gradient a second: bound by
// HBM, which reads each logit once where a row's block still holds it and
// writes the gradient once.  Exponentials are taken as 2^(z c - m c) with
// c = log2(e) / T in one fma, whose rounding of m c the sums and g make up
// for.  From |m c| = 2^24 on (a row masked with a large value throughout) that
// rounding is more than a half, in the end more than the exponential's range:
// they are then 2^((z - m) c).
#include <hip/hip_runtime.h>

#include <cmath>

#include "tokens.hpp"

namespace wh {
namespace {

using namespace tok;

constexpr int kMaxEntries = 1024;

struct Args {
  const void *logits;
  int64_t stride;
  int vocab, k;
  const int32_t *index;
  const float *teacher, *teacher_lse, *weight;
  float temperature, c;  // c = log2(e) / T
  float *loss;
  void *grad;
  int64_t gstride;
};

// Maximum of z and sum of 2^((z - m) c).
struct Stat {
  float m, s;
};
// The exponent's offset mc = m c as rounded; huge: of no use (m itself may be +inf).
__device__ inline bool too_large(float mc) { return !(fabsf(mc) < 0x1p24f); }
struct Shift {
  float m, mc;
  bool huge;
  __device__ Shift(float m_, float c) : m(m_), mc(m_ == -INFINITY ? 0.0f : m_ * c) { huge = too_large(mc); }
  // what m c is past the offset taken for it
  __device__ float rest(float c) const { return huge || m == -INFINITY ? 0.0f : fmaf(m, c, -mc); }
};
__device__ inline float term(float z, float c, const Shift &h) {
  return __builtin_amdgcn_exp2f(h.huge ? (z - h.m) * c : fmaf(z, c, -h.mc));
}
// The factor from a sum at maximum `from` to one at `to`; an empty sum's (0) must not be NaN.
__device__ inline float rescale(float from, float to, float c) {
  return from == to ? 1.0f : __builtin_amdgcn_exp2f((from - to) * c);
}
__device__ inline Stat join(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * rescale(a.m, m, c) + b.s * rescale(b.m, m, c)};
}
// A thread's pair as it grows, its sum at the offset of its maximum.
struct Running {
  float m = -INFINITY, s = 0.0f, mc = 0.0f;
  template <int N>
  __device__ inline void take(const float (&z)[N], float c) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    if (top > m) {
      const Shift h(top, c);
      float e = mc - h.mc;
      if (__builtin_expect(h.huge || too_large(mc), 0)) e = (m - top) * c + h.rest(c) - Shift(m, c).rest(c);
      s *= m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(e);
      m = top;
      mc = h.mc;
    }
    float e[N];
    if (__builtin_expect(too_large(mc), 0)) {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = __builtin_amdgcn_exp2f((z[i] - m) * c);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(z[i], c, -mc));
    }
#pragma unroll
    for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
      for (int i = 0; i < n; ++i) e[i] += e[i + n];
    s += e[0];
  }
  __device__ inline Stat stat(float c) const { return {m, s * __builtin_amdgcn_exp2f(-Shift(m, c).rest(c))}; }
};

// The block's pair, on every thread.
template <int WAVES>
__device__ inline Stat block_join(Stat a, float c, Stat *lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a = join(a, {__shfl_xor(a.m, off), __shfl_xor(a.s, off)}, c);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  a = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) a = join(a, lds[w], c);
  return a;
}
template <int WAVES>
__device__ inline float block_sum(float v, float *lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) v += lds[w];
  return v;
}

// n values at p: `head` ones up to a 16-byte boundary, whole 16-byte words,
// `tail` ones.
template <class T>
struct Span {
  const typename T::raw *p;
  int n, head, words, tail;
  __device__ Span(const typename T::raw *p_, int n_) : p(p_), n(n_) {
    const int off = (int)(((uintptr_t)p & 15) / sizeof(typename T::raw));
    head = min(n, off ? T::kPer16 - off : 0);
    words = (n - head) / T::kPer16;
    tail = n - head - words * T::kPer16;
  }
  __device__ const uint4 *word(int i) const { return (const uint4 *)(p + head) + i; }
  // the place of edge value i < head + tail
  __device__ int edge(int i) const { return i < head ? i : n - tail + (i - head); }
};

// The teacher's entries of a row, in LDS.
struct Entries {
  int index[kMaxEntries];
  float q[kMaxEntries];  // log q
  float z[kMaxEntries];  // the student's logit, read before its gradient may take its place
  float top[16], sum[16];  // by wave
};
template <class T>
__device__ inline float logit(const Args &a, int row, int v) {
  return T::get(((const typename T::raw *)a.logits + (int64_t)row * a.stride)[v]);
}
// Three steps, so that a row's own loads can be in flight between them: the
// entries' loads, the distribution q, the student's logits at the entries.
template <class T, int WAVES>
struct Teacher {
  static constexpr int kPer = (kMaxEntries + WAVES * 64 - 1) / (WAVES * 64);
  int index[kPer];
  float l[kPer];
  __device__ inline void load(const Args &a, int row) {
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
      const int i = threadIdx.x + n * WAVES * 64;
      index[n] = -1;
      l[n] = -INFINITY;
      if (i < a.k) {
        index[n] = a.index[(int64_t)row * a.k + i];
        l[n] = a.teacher[(int64_t)row * a.k + i];
      }
    }
  }
  // Fills e.index and e.q (each thread its own entries: a barrier follows before
  // another reads them); *mass = the sum of q; false where the row has no entry.
  __device__ inline bool weigh(const Args &a, int row, Entries &e, float *mass) {
    const double inv = 1.0 / (double)a.temperature;
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
      if (index[n] < 0 || index[n] >= a.vocab || l[n] == -INFINITY) index[n] = -1;
      else top = fmaxf(top, l[n] == l[n] ? l[n] : INFINITY);  // NaN: an entry, and q NaN throughout
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    if ((threadIdx.x & 63) == 0) e.top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = e.top[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, e.top[w]);
    if (top == -INFINITY) return false;
    const double most = a.teacher_lse == nullptr ? (double)top * inv : (double)a.teacher_lse[row];
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
      l[n] = (float)((double)l[n] * inv - most);
      if (index[n] >= 0) sum += expf(l[n]);
    }
    sum = block_sum<WAVES>(sum, e.sum);
    const float log_sum = a.teacher_lse == nullptr ? logf(sum) : 0.0f;
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
      const int i = threadIdx.x + n * WAVES * 64;
      if (i >= a.k) break;
      e.index[i] = index[n];
      e.q[i] = l[n] - log_sum;
    }
    // the entries' own sum leaves 1, or NaN where one of them is NaN or +inf
    *mass = a.teacher_lse == nullptr ? sum / sum : sum;
    return true;
  }
  // e.z, from zs (this row's logits at the entries) or the row itself.
  __device__ inline void gather(const Args &a, int row, const float *zs, Entries &e) {
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
      const int i = threadIdx.x + n * WAVES * 64;
      if (i < a.k && index[n] >= 0) e.z[i] = zs ? zs[i] : logit<T>(a, row, index[n]);
    }
  }
};

// loss of a row from the pair of its logits; every thread calls it.
template <int WAVES>
__device__ inline void write_loss(const Args &a, int row, const Entries &e, Stat st, float weight) {
  const double c = (double)a.c, mc = (double)st.m * c, log2s = log2((double)st.s);
  double loss = 0.0;
  for (int i = threadIdx.x; i < a.k; i += WAVES * 64) {
    if (e.index[i] < 0) continue;
    // no finite logit: p = 0 everywhere
    const double logp = st.s == 0.0f ? -INFINITY : 0.6931471805599453 * ((double)e.z[i] * c - mc - log2s);
    const double q = exp((double)e.q[i]);
    if (q != 0.0) loss += q * ((double)e.q[i] - logp);  // 0 log 0 = 0, also under p = 0
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) loss += __shfl_xor(loss, off);
  __shared__ double lds[WAVES];
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    loss = 0.0;
    for (int w = 0; w < WAVES; ++w) loss += lds[w];
    a.loss[row] = (float)(loss * (double)a.temperature * (double)a.temperature * (double)weight);
  }
}

// The entries' own gradients over the part [begin, begin + n) of the row,
// once every thread's dense values are written: index v's first entry stands
// for all of v's.
template <class T, int WAVES>
__device__ inline void write_entries(const Args &a, int row, const Entries &e, int begin, int n, const Shift &h,
                                     float g, float wt) {
  typename T::raw *out = (typename T::raw *)a.grad + (int64_t)row * a.gstride;
  for (int i = threadIdx.x; i < a.k; i += WAVES * 64) {
    const int v = e.index[i];
    if (v < begin || v >= begin + n) continue;
    float q = 0.0f;
    bool first = true;
    for (int j = 0; j < a.k; ++j) {
      if (e.index[j] != v) continue;
      if (j < i) first = false;
      q += expf(e.q[j]);
    }
    if (first) out[v] = T::put(fmaf(term(e.z[i], a.c, h), g, -q * wt));
  }
}

// Dense values: term * g, for a row whose offset is not too large, or is.
template <bool HUGE>
__device__ inline float dense(float z, float c, const Shift &h, float g) {
  return __builtin_amdgcn_exp2f(HUGE ? (z - h.m) * c : fmaf(z, c, -h.mc)) * g;
}
template <class T, bool HUGE>
__device__ inline uint4 grad_word(const uint4 &word, float c, const Shift &h, float g) {
  float f[T::kPer16];
  unpack16<T>(word, f);
#pragma unroll
  for (int i = 0; i < T::kPer16; ++i) f[i] = dense<HUGE>(f[i], c, h, g);
  return pack16<T>(f);
}
template <class T, int THREADS>
__device__ inline void zero_grad(typename T::raw *out, int n) {
  const Span<T> span(out, n);
  for (int i = threadIdx.x; i < span.words; i += THREADS) *(uint4 *)span.word(i) = make_uint4(0, 0, 0, 0);
  if ((int)threadIdx.x < span.head + span.tail) out[span.edge(threadIdx.x)] = 0;
}

// Words that are not looked at again: past the caches, which then keep those
// of the row's end that are.
typedef uint32_t w4 __attribute__((ext_vector_type(4)));
__device__ inline void put_word(uint4 *p, const uint4 &v) {
  __builtin_nontemporal_store(w4{v.x, v.y, v.z, v.w}, (w4 *)p);
}
__device__ inline uint4 get_word(const uint4 *p) {
  const w4 v = __builtin_nontemporal_load((const w4 *)p);
  return make_uint4(v.x, v.y, v.z, v.w);
}

// A row a block.  Of each thread's 16-byte words of it HOLD stay in registers
// and LDSW in LDS between the two passes, what is left is read again.  The
// teacher's loads go out first, then the row's, and the teacher's arithmetic
// runs while those are under way.  Two blocks a CU, so that one's exponentials
// (about 200 us of the whole) run under the other's loads and stores: 4096 x
// 131072 bf16, 15 % of the rows left out, takes 423 us with 8 waves and 8 + 8
// words held; 8 + 0 took 20 more, 16 waves with the whole row in registers (one
// block a CU) 155.
template <class T, int WAVES, int HOLD, int LDSW, bool GRAD>
__global__ void __launch_bounds__(WAVES * 64, 4) distill_row_kernel(Args a) {
  constexpr int kThreads = WAVES * 64;
  __shared__ Stat lds[WAVES];
  __shared__ Entries e;
  __shared__ uint4 more[LDSW > 0 ? LDSW * kThreads : 1];
  const int row = blockIdx.x, n = a.vocab;
  const float weight = a.weight ? a.weight[row] : 1.0f;
  const Span<T> in((const typename T::raw *)a.logits + (int64_t)row * a.stride, n);
  typename T::raw *out = GRAD ? (typename T::raw *)a.grad + (int64_t)row * a.gstride : nullptr;
  float mass = 0.0f;
  Teacher<T, WAVES> teacher;
  uint4 held[HOLD];
  teacher.load(a, row);
  bool live = weight != 0.0f;
  if (live) {
    issued();
#pragma unroll
    for (int r = 0; r < HOLD; ++r)
      if (r * kThreads < in.words) held[r] = get_word(in.word(min(r * kThreads + (int)threadIdx.x, in.words - 1)));
    issued();
    live = teacher.weigh(a, row, e, &mass);
  }
  if (!live) {
    if (threadIdx.x == 0 && a.loss) a.loss[row] = 0.0f;
    if constexpr (GRAD) zero_grad<T, kThreads>(out, n);
    return;
  }
  teacher.gather(a, row, nullptr, e);
  Running run;
#pragma unroll
  for (int r = 0; r < HOLD; ++r)
    if (r * kThreads + (int)threadIdx.x < in.words) {
      float f[T::kPer16];
      unpack16<T>(held[r], f);
      run.take(f, a.c);
    }
  {
    int i = HOLD * kThreads + threadIdx.x;
    if constexpr (LDSW > 0) {
      for (int r0 = 0; r0 < LDSW && i < in.words; r0 += 4) {
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = get_word(in.word(min(i + k * kThreads, in.words - 1)));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (i < in.words) {
            more[(r0 + k) * kThreads + threadIdx.x] = w[k];
            float f[T::kPer16];
            unpack16<T>(w[k], f);
            run.take(f, a.c);
          }
          i += kThreads;
        }
      }
    }
    for (; i + 3 * kThreads < in.words; i += 4 * kThreads) {
      uint4 w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = *in.word(i + k * kThreads);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[T::kPer16];
        unpack16<T>(w[k], f);
        run.take(f, a.c);
      }
    }
    for (; i < in.words; i += kThreads) {
      float f[T::kPer16];
      unpack16<T>(*in.word(i), f);
      run.take(f, a.c);
    }
  }
  if ((int)threadIdx.x < in.head + in.tail) {
    const float f[1] = {T::get(in.p[in.edge(threadIdx.x)])};
    run.take(f, a.c);
  }
  const Stat st = block_join<WAVES>(run.stat(a.c), a.c, lds);
  if constexpr (!GRAD) write_loss<WAVES>(a, row, e, st, weight);
  if constexpr (GRAD) {
    const Shift h(st.m, a.c);
    const float c = a.c, wt = weight * a.temperature;
    // no finite logit: p = 0
    const float g = st.s == 0.0f ? 0.0f * mass : wt * mass / (st.s * __builtin_amdgcn_exp2f(h.rest(c)));
    const auto write = [&](auto huge) {
      constexpr bool H = decltype(huge)::value;
      if ((((uintptr_t)out ^ (uintptr_t)in.p) & 15) == 0) {
        uint4 *to = (uint4 *)(out + in.head);
#pragma unroll
        for (int r = 0; r < HOLD; ++r) {
          const int i = r * kThreads + threadIdx.x;
          if (i < in.words) put_word(to + i, grad_word<T, H>(held[r], c, h, g));
        }
        int i = HOLD * kThreads + threadIdx.x;
        if constexpr (LDSW > 0) {
          for (int r = 0; r < LDSW && i < in.words; ++r, i += kThreads)
            put_word(to + i, grad_word<T, H>(more[r * kThreads + threadIdx.x], c, h, g));
        }
        for (; i + 3 * kThreads < in.words; i += 4 * kThreads) {
          uint4 w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = *in.word(i + k * kThreads);
#pragma unroll
          for (int k = 0; k < 4; ++k) put_word(to + i + k * kThreads, grad_word<T, H>(w[k], c, h, g));
        }
        for (; i < in.words; i += kThreads) put_word(to + i, grad_word<T, H>(*in.word(i), c, h, g));
        if ((int)threadIdx.x < in.head + in.tail) {
          const int at = in.edge(threadIdx.x);
          out[at] = T::put(dense<H>(T::get(in.p[at]), c, h, g));
        }
      } else {
        for (int i = threadIdx.x; i < n; i += kThreads) out[i] = T::put(dense<H>(T::get(in.p[i]), c, h, g));
      }
    };
    if (h.huge) write(std::true_type{});
    else write(std::false_type{});
    __syncthreads();
    write_entries<T, WAVES>(a, row, e, 0, n, h, g, wt);
    if (a.loss) write_loss<WAVES>(a, row, e, st, weight);
  }
}

// Few rows: `parts` blocks a row.
//   STATS  the part's pair into pairs[row][part], and by part 0 the entries'
//          logits into zs[row][k]
//   else   the part's gradient, and by part 0 the loss
template <class T, int WAVES, bool STATS>
__global__ void __launch_bounds__(WAVES * 64) distill_part_kernel(Args a, int parts, int len, Stat *pairs, float *zs) {
  constexpr int kThreads = WAVES * 64, kHeld = 4;
  __shared__ Stat lds[WAVES];
  const int row = blockIdx.x / parts, part = blockIdx.x % parts, begin = part * len;
  const int n = min(len, a.vocab - begin);
  const float weight = a.weight ? a.weight[row] : 1.0f;
  const Span<T> in((const typename T::raw *)a.logits + (int64_t)row * a.stride + begin, n);
  if constexpr (STATS) {
    Running run;
    if (weight == 0.0f) return;
    if (part == 0)
      for (int i = threadIdx.x; i < a.k; i += kThreads) {
        const int v = a.index[(int64_t)row * a.k + i];
        if (v >= 0 && v < a.vocab) zs[(int64_t)row * a.k + i] = logit<T>(a, row, v);
      }
    int i = threadIdx.x;
    for (; i + 3 * kThreads < in.words; i += 4 * kThreads) {
      uint4 w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = *in.word(i + k * kThreads);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[T::kPer16];
        unpack16<T>(w[k], f);
        run.take(f, a.c);
      }
    }
    for (; i < in.words; i += kThreads) {
      float f[T::kPer16];
      unpack16<T>(*in.word(i), f);
      run.take(f, a.c);
    }
    if ((int)threadIdx.x < in.head + in.tail) {
      const float f[1] = {T::get(in.p[in.edge(threadIdx.x)])};
      run.take(f, a.c);
    }
    const Stat st = block_join<WAVES>(run.stat(a.c), a.c, lds);
    if (threadIdx.x == 0) pairs[(int64_t)row * parts + part] = st;
  } else {
    __shared__ Entries e;
    typename T::raw *out = a.grad ? (typename T::raw *)a.grad + (int64_t)row * a.gstride + begin : nullptr;
    float mass = 0.0f;
    Teacher<T, WAVES> teacher;
    Stat st{-INFINITY, 0.0f};
    uint4 held[kHeld];
    teacher.load(a, row);
    bool live = weight != 0.0f;
    if (live) {  // all the block's first loads, then the teacher's arithmetic
      if ((int)threadIdx.x < parts) st = pairs[(int64_t)row * parts + threadIdx.x];
      if (out) {
#pragma unroll
        for (int r = 0; r < kHeld; ++r)
          if (r * kThreads < in.words) held[r] = *in.word(min(r * kThreads + (int)threadIdx.x, in.words - 1));
      }
      issued();
      live = teacher.weigh(a, row, e, &mass);
    }
    if (!live) {
      if (threadIdx.x == 0 && part == 0 && a.loss) a.loss[row] = 0.0f;
      if (out) zero_grad<T, kThreads>(out, n);
      return;
    }
    teacher.gather(a, row, zs + (int64_t)row * a.k, e);
    for (int i = threadIdx.x + kThreads; i < parts; i += kThreads) st = join(st, pairs[(int64_t)row * parts + i], a.c);
    st = block_join<WAVES>(st, a.c, lds);
    if (!out) {
      if (part == 0) write_loss<WAVES>(a, row, e, st, weight);
      return;
    }
    const Shift h(st.m, a.c);
    const float c = a.c, wt = weight * a.temperature;
    // no finite logit: p = 0
    const float g = st.s == 0.0f ? 0.0f * mass : wt * mass / (st.s * __builtin_amdgcn_exp2f(h.rest(c)));
    const auto write = [&](auto huge) {
      constexpr bool H = decltype(huge)::value;
      if ((((uintptr_t)out ^ (uintptr_t)in.p) & 15) == 0) {
        uint4 *to = (uint4 *)(out + in.head);
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
          const int i = r * kThreads + threadIdx.x;
          if (i < in.words) to[i] = grad_word<T, H>(held[r], c, h, g);
        }
        int i = kHeld * kThreads + threadIdx.x;
        for (; i + 3 * kThreads < in.words; i += 4 * kThreads) {
          uint4 w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = *in.word(i + k * kThreads);
#pragma unroll
          for (int k = 0; k < 4; ++k) to[i + k * kThreads] = grad_word<T, H>(w[k], c, h, g);
        }
        for (; i < in.words; i += kThreads) to[i] = grad_word<T, H>(*in.word(i), c, h, g);
        if ((int)threadIdx.x < in.head + in.tail) {
          const int at = in.edge(threadIdx.x);
          out[at] = T::put(dense<H>(T::get(in.p[at]), c, h, g));
        }
      } else {
        for (int i = threadIdx.x; i < n; i += kThreads) out[i] = T::put(dense<H>(T::get(in.p[i]), c, h, g));
      }
    };
    if (h.huge) write(std::true_type{});
    else write(std::false_type{});
    __syncthreads();
    write_entries<T, WAVES>(a, row, e, begin, n, h, g, wt);
    if (part == 0 && a.loss) write_loss<WAVES>(a, row, e, st, weight);
  }
}

constexpr int kRowBlocks = 256;  // rows from which each has one block
// Parts of a row: one where there are rows for every CU, else as many as give
// each CU two blocks, down to 1024 values (4 rows of 32000 f32 logits, loss and
// gradient, calls one after the other: parts of 4096 and up 10.6 us, of 1024 and
// up 9.7; 64 rows of 32000 bf16 14.8 and 14.0).
int parts_of(int n, int vocab) {
  if (n == 0 || n >= kRowBlocks) return 1;
  return std::max(1, std::min((512 + n - 1) / n, vocab / 1024));
}
int part_len(int64_t vocab, int parts) { return (int)(((vocab + parts - 1) / parts + 63) / 64 * 64); }
size_t pairs_bytes(int n, int vocab) { return pad256((size_t)n * parts_of(n, vocab) * sizeof(Stat)); }
size_t workspace_bytes(int n, int vocab, int k) {
  return parts_of(n, vocab) == 1 ? 0 : pairs_bytes(n, vocab) + pad256((size_t)n * k * sizeof(float));
}

// Enough for any batch up to n: fewer rows can need more, as more parts.
size_t most_workspace_bytes(int n, int vocab, int k) {
  size_t most = 0;
  for (int rows = 1; rows <= std::min(n, kRowBlocks - 1); ++rows) most = std::max(most, workspace_bytes(rows, vocab, k));
  return most;
}

template <class T>
hipError_t launch_distill(const Args &a, int n, void *ws, hipStream_t s) {
  const int most = parts_of(n, a.vocab);
  if (most == 1) {
    const int words = a.vocab / T::kPer16;
    if (a.grad == nullptr) {
      if (words <= 2048) distill_row_kernel<T, 4, 8, 0, false><<<n, 256, 0, s>>>(a);
      else distill_row_kernel<T, 8, 8, 0, false><<<n, 512, 0, s>>>(a);
    } else if (words <= 2048) {
      distill_row_kernel<T, 4, 8, 0, true><<<n, 256, 0, s>>>(a);
    } else if (words <= 4096) {
      distill_row_kernel<T, 8, 8, 0, true><<<n, 512, 0, s>>>(a);
    } else {
      distill_row_kernel<T, 8, 8, 8, true><<<n, 512, 0, s>>>(a);
    }
    return hipGetLastError();
  }
  const int len = part_len(a.vocab, most), parts = (int)(((int64_t)a.vocab + len - 1) / len);
  Stat *pairs = (Stat *)ws;
  float *zs = (float *)((char *)ws + pairs_bytes(n, a.vocab));
  distill_part_kernel<T, 4, true><<<n * parts, 256, 0, s>>>(a, parts, len, pairs, zs);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  distill_part_kernel<T, 4, false><<<n * parts, 256, 0, s>>>(a, parts, len, pairs, zs);
  return hipGetLastError();
}

// vocab: a thread's steps along a row pass its end in int.
bool sizes_ok(int32_t n, int32_t vocab, int32_t k) {
  return n >= 0 && n <= (1 << 22) && vocab > 0 && vocab <= INT32_MAX - 4095 && k > 0 && k <= kMaxEntries;
}

}  // namespace
}  // namespace wh

using namespace wh;
using namespace wh::rt;

extern "C" {

welvet_status welvet_hip_distill_bytes(int32_t dtype, int32_t n, int32_t vocab, int32_t k, size_t *bytes) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "distill: unsupported dtype %d", dtype);
  if (!sizes_ok(n, vocab, k) || !bytes) return make_status(kInvalid, "distill: invalid argument");
  *bytes = most_workspace_bytes(n, vocab, k);
  return ok();
}

welvet_status welvet_hip_distill(int32_t dtype, int32_t n, int32_t vocab, const void *d_logits, int64_t stride,
                                 int32_t k, const int32_t *d_index, const float *d_teacher,
                                 const float *d_teacher_lse, const float *d_weight, float temperature, float *d_loss,
                                 void *d_dlogits, int64_t dstride, void *d_ws, size_t ws_bytes, void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "distill: unsupported dtype %d", dtype);
  if (!sizes_ok(n, vocab, k) || (n > 0 && (!d_logits || !d_index || !d_teacher)) || (!d_loss && !d_dlogits))
    return make_status(kInvalid, "distill: invalid argument");
  const float c = (float)(1.4426950408889634 / (double)temperature);
  if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(c))
    return make_status(kInvalid, "distill: temperature must be positive and finite, as log2(e) / temperature");
  if (stride < vocab || (d_dlogits && dstride < vocab))
    return make_status(kInvalid, "distill: row stride below vocab %d", vocab);
  if (n > 1 && d_dlogits == d_logits && dstride != stride)
    return make_status(kInvalid, "distill: a gradient in the logits' place needs their row stride");
  const int size = tok::float_size(dtype);
  if (!tok::aligned(d_logits, size) || !tok::aligned(d_dlogits, size) || !tok::aligned(d_index, 4) ||
      !tok::aligned(d_teacher, 4) || !tok::aligned(d_teacher_lse, 4) || !tok::aligned(d_weight, 4) ||
      !tok::aligned(d_loss, 4))
    return make_status(kInvalid, "distill: device pointers must be aligned to their elements");
  const size_t need = workspace_bytes(n, vocab, k);
  if (need > 0 && (!d_ws || ws_bytes < need || !tok::aligned(d_ws, 16)))
    return make_status(kInvalid, "distill: %zu bytes of 16-byte aligned workspace are needed", need);
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  const Args a{d_logits, stride, vocab, k, d_index, d_teacher, d_teacher_lse, d_weight, temperature, c,
               d_loss,   d_dlogits, dstride};
  WH_HIP(tok::with_type(dtype, [&](auto t) { return launch_distill<decltype(t)>(a, n, d_ws, (hipStream_t)stream); }));
  return ok();
}

}  // extern "C"
