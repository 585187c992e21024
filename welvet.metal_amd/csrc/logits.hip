// logits.hip — rules that logits pass before an answer is taken from them.  For
// token v of a row, named c times after the prompt:
//   z = z > 0 ? z / r : z r  where the history names v at all
//   z = z - c f - p          where c > 0
//   z = z + the sum of v's biases, in the list's order
//   z = -inf                 where the row's mask shuts v
// A block takes a stretch of a row's vocabulary.  It counts the history's
// tokens of that stretch in LDS (whole numbers: the order does not matter), a
// word a token: how often it was said, whether the prompt names it, which entry
// of the list does.  Then it passes over the stretch once: bound by HBM, as
// nothing of what a mask shuts is read.  In place, only eights with a token that a
// rule names are read, and only the tokens that one names are written.
//   f16 50257, 1000 rows under 40 masks, 1024 said, 100 biases: 49 to 65 us (the
//   second from HBM, 205 MB); bf16 131072, 64 rows, 8192 said, 15.6; f32 32000, 4
//   rows, 4.4, mostly the launch.
#include <hip/hip_runtime.h>

#include <cmath>

#include "rows8.hpp"

namespace wh {
namespace {

using namespace r8;

constexpr int kThreads = 512;
// Tokens a block: with the list 38 KB of LDS, four blocks a CU (blocks of 1024 threads
// with twice the tokens, two a CU: 73 us against 71 for the 50257).
constexpr int kStretch = 8192;
constexpr int kOcts = 2;
static_assert(kOcts * kThreads * 8 >= kStretch && kStretch % 32 == 0, "whole words of a mask, in one go");
constexpr int kMaxHistory = (1 << 20) - 1, kMaxBiases = 1024;
constexpr uint32_t kCount = kMaxHistory, kPrompt = 1u << 31;
constexpr int kEntry = 20;  // bits from here to 30: 1 + the number of a list's entry that names the token
constexpr uint32_t kEntries = 0x7ffu << kEntry;

struct Args {
  welvet_hip_logit_rules r;
  const void *in;
  void *out;
  int64_t in_stride, out_stride;
  int vocab, parts, len;  // parts stretches of len tokens a row
};

struct Row {
  double repetition, frequency, presence;
  __device__ inline double apply(double z, uint32_t word) const {
    const uint32_t c = word & kCount;
    if (c || (word & kPrompt)) z = z > 0.0 ? z / repetition : z * repetition;
    if (c) z = z - (double)c * frequency - presence;
    return z;
  }
};
// Rounded once: through an f32 whose last bit tells that something was cut off.
template <class T>
__device__ inline typename T::raw rounded(double z) {
  float f = (float)z;
  if constexpr (sizeof(typename T::raw) == 2) {
    uint32_t u = f2u(f);
    if ((double)f != z && z == z) {
      if (fabs((double)f) > fabs(z)) --u;
      f = u2f(u | 1u);
    }
  }
  return T::put(f);
}
template <class T>
constexpr typename T::raw kShut = sizeof(typename T::raw) == 4 ? (typename T::raw)0xff800000u
                                  : std::is_same_v<T, F16>     ? (typename T::raw)0xfc00u
                                                               : (typename T::raw)0xff80u;

template <class T, bool INPLACE>
__global__ void __launch_bounds__(kThreads) rules_kernel(Args a) {
  using raw = typename T::raw;
  __shared__ uint4 words[kStretch / 4];
  __shared__ int16_t index[kMaxBiases];  // of the stretch, -1 elsewhere
  __shared__ float biases[kMaxBiases];
  __shared__ int twice;  // a token of this stretch is named by two entries
  uint32_t *count = (uint32_t *)words;
  const int row = blockIdx.x / a.parts, begin = (int)(blockIdx.x % a.parts) * a.len;
  const int len = min(a.len, a.vocab - begin), tid = threadIdx.x;
  const raw *in = (const raw *)a.in + (int64_t)row * a.in_stride + begin;
  raw *out = (raw *)a.out + (int64_t)row * a.out_stride + begin;
  // Loads go out in the order in which they are waited for, each as early as it
  // can: the history's first tokens and the list, the mask, the logits that it leaves.
  constexpr int kFirst = 4, kList = kMaxBiases / kThreads;
  const int32_t *said = a.r.d_history + (int64_t)row * a.r.history_stride;
  int32_t first[kFirst], at[kList];
  float bias[kList];
  if (a.r.history > 0)
#pragma unroll
    for (int k = 0; k < kFirst; ++k)
      if (k * kThreads < a.r.history) first[k] = said[min(k * kThreads + tid, a.r.history - 1)];
  if (a.r.biases > 0)
#pragma unroll
    for (int k = 0; k < kList; ++k)
      if (k * kThreads < a.r.biases) {
        const int64_t i = (int64_t)row * a.r.biases + min(k * kThreads + tid, a.r.biases - 1);
        at[k] = a.r.d_bias_index[i];
        bias[k] = a.r.d_bias[i];
      }
  const uint32_t *mask = nullptr;
  if (a.r.masks > 0) {
    const int id = a.r.d_mask_id ? a.r.d_mask_id[row] : row;
    if (id >= 0 && id < a.r.masks) mask = a.r.d_masks + id * a.r.mask_stride + begin / 32;
  }
  const int history = a.r.history > 0 && a.r.d_history_len ? min(max(a.r.d_history_len[row], 0), a.r.history) : a.r.history;
  const int prompt = a.r.d_prompt_len ? min(max(a.r.d_prompt_len[row], 0), history) : 0;
  const Row rules{a.r.d_repetition ? (double)a.r.d_repetition[row] : 1.0,
                  a.r.d_frequency ? (double)a.r.d_frequency[row] : 0.0,
                  a.r.d_presence ? (double)a.r.d_presence[row] : 0.0};
  const auto open8 = [&](int c) -> uint32_t { return mask ? mask[c >> 5] >> (c & 31) & 0xffu : 0xffu; };
  uint32_t open[kOcts];
  Oct<T> held[kOcts];
#pragma unroll
  for (int k = 0; k < kOcts; ++k) open[k] = open8(min((k * kThreads + tid) * 8, (len - 1) & ~7));
#pragma unroll
  for (int k = 0; k < kOcts; ++k) {
    const int c = (k * kThreads + tid) * 8;
    if (c >= len) open[k] = 0;
    if (!INPLACE && open[k]) held[k].load(in, c, len);
  }
  const bool sparse = history > 0 || a.r.biases > 0;
  if (sparse) {
    if (tid == 0) twice = 0;
    for (int i = tid; i < (len + 3) / 4; i += kThreads) words[i] = make_uint4(0, 0, 0, 0);
    if (a.r.biases > 0)
#pragma unroll
      for (int k = 0; k < kList; ++k) {
        const int i = k * kThreads + tid;
        if (k * kThreads >= a.r.biases) break;
        const int64_t v = (int64_t)at[k] - begin;
        at[k] = i < a.r.biases && v >= 0 && v < len ? (int)v : -1;
        if (i < a.r.biases) {
          index[i] = (int16_t)at[k];
          biases[i] = bias[k];
        }
      }
    __syncthreads();
    const auto count_one = [&](int i, int32_t token) {
      const int64_t v = (int64_t)token - begin;
      if (i >= history || v < 0 || v >= len) return;
      if (i < prompt) atomicOr(&count[v], kPrompt);
      else atomicAdd(&count[v], 1u);
    };
    if (history > 0)
#pragma unroll
      for (int k = 0; k < kFirst; ++k)
        if (k * kThreads < a.r.history) count_one(k * kThreads + tid, first[k]);
    for (int i = kFirst * kThreads + tid; i < history; i += kFirst * kThreads) {
      int32_t more[kFirst];
#pragma unroll
      for (int k = 0; k < kFirst; ++k) more[k] = said[min(i + k * kThreads, history - 1)];
#pragma unroll
      for (int k = 0; k < kFirst; ++k) count_one(i + k * kThreads, more[k]);
    }
    if (a.r.biases > 0)
#pragma unroll
      for (int k = 0; k < kList; ++k) {
        if (k * kThreads >= a.r.biases) break;
        if (at[k] >= 0 && (atomicOr(&count[at[k]], (uint32_t)(k * kThreads + tid + 1) << kEntry) & kEntries)) twice = 1;
      }
    __syncthreads();
  }
  // token v of word w; a token named twice has every token of the list in this stretch
  // look through all of it, as words hold one entry (f32 131072, 64 rows, 1024 biases, 21
  // us; 270 with one named twice in each row, f16 50257, 1000 rows, 100 biases 49 / 64)
  const auto changed = [&](raw was, int v, uint32_t w) {
    double sum = rules.apply((double)T::get(was), w);
    if (w & kEntries) {
      if (!twice) sum += (double)biases[(w >> kEntry & 0x7ffu) - 1];
      else
        for (int j = 0; j < a.r.biases; ++j)
          if (index[j] == v) sum += (double)biases[j];
    }
    return rounded<T>(sum);
  };
  // which of eight tokens a rule names that the mask leaves
  const auto named = [&](int c, uint32_t left) {
    const uint4 w0 = words[c / 4], w1 = words[c / 4 + 1];
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits |= w[i] ? 1u << i : 0u;
    return bits & (c + 8 <= len ? left : left & ((1u << (len - c)) - 1));
  };
  // a token a turn: most lanes have none or one, and a turn is what eight
  // conditions in a row would cost each
  if constexpr (INPLACE) {
    uint32_t here[kOcts];
#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      const int c = (k * kThreads + tid) * 8;
      here[k] = sparse && open[k] ? named(c, open[k]) : 0;
      if (here[k]) held[k].load(in, c, len);
    }
#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      const int c = (k * kThreads + tid) * 8;
      if (c >= len) break;
      if (open[k] == 0) {
        held[k].fill(kShut<T>);
        held[k].store(out, c, len);
        continue;
      }
      if (open[k] != 0xffu)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(open[k] >> i & 1) && c + i < len) out[c + i] = kShut<T>;
      for (; here[k]; here[k] &= here[k] - 1) {
        const int i = __ffs(here[k]) - 1;
        out[c + i] = changed(held[k].at(i), c + i, count[c + i]);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      const int c = (k * kThreads + tid) * 8;
      if (c >= len) break;
      Oct<T> &o = held[k];
      if (open[k] == 0) {
        o.fill(kShut<T>);
      } else {
        if (sparse)
          for (uint32_t here = named(c, open[k]); here; here &= here - 1) {
            const int i = __ffs(here) - 1;
            o.set_at(i, changed(o.at(i), c + i, count[c + i]));
          }
        if (open[k] != 0xffu) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(open[k] >> i & 1)) o.set_raw(i, kShut<T>);
        }
      }
      o.store(out, c, len);
    }
  }
}

// Stretches of a row: as many as give each CU two blocks, of 2048 tokens and
// more, and no longer than the counts' place.
void stretches(int n, int vocab, int *parts, int *len) {
  const int64_t most = (vocab + kStretch - 1) / kStretch;
  const int64_t p = std::max<int64_t>(most, std::min<int64_t>((512 + n - 1) / n, vocab / 2048));
  *len = (int)(((vocab + p - 1) / p + 31) / 32 * 32);
  *parts = (vocab + *len - 1) / *len;
}

}  // namespace
}  // namespace wh

using namespace wh;
using namespace wh::rt;

extern "C" {

welvet_status welvet_hip_logits_rules(int32_t dtype, int32_t n, int32_t vocab, const void *d_logits, int64_t stride,
                                      const welvet_hip_logit_rules *rules, void *d_out, int64_t out_stride,
                                      void *stream) {
  if (!tok::float_type(dtype)) return make_status(kUnsupported, "logits: unsupported dtype %d", dtype);
  if (n < 0 || n > (1 << 20) || vocab <= 0 || vocab > (1 << 30) || !rules || (n > 0 && (!d_logits || !d_out)))
    return make_status(kInvalid, "logits: invalid argument");
  const welvet_hip_logit_rules &r = *rules;
  if (r.history < 0 || r.history > kMaxHistory || r.biases < 0 || r.biases > kMaxBiases || r.masks < 0 ||
      (r.history > 0 && (!r.d_history || r.history_stride < r.history)) ||
      (r.biases > 0 && (!r.d_bias_index || !r.d_bias)) ||
      (r.masks > 0 && (!r.d_masks || r.mask_stride < ((int64_t)vocab + 31) / 32)))
    return make_status(kInvalid, "logits: invalid rules");
  if (stride < vocab || out_stride < vocab) return make_status(kInvalid, "logits: row stride below vocab %d", vocab);
  if (n > 1 && d_out == d_logits && out_stride != stride)
    return make_status(kInvalid, "logits: a result in the logits' place needs their row stride");
  const int size = tok::float_size(dtype);
  if (!tok::aligned(d_logits, size) || !tok::aligned(d_out, size))
    return make_status(kInvalid, "logits: device pointers must be aligned to their elements");
  for (const void *p : {(const void *)r.d_history, (const void *)r.d_history_len, (const void *)r.d_prompt_len,
                        (const void *)r.d_repetition, (const void *)r.d_frequency, (const void *)r.d_presence,
                        (const void *)r.d_bias_index, (const void *)r.d_bias, (const void *)r.d_masks,
                        (const void *)r.d_mask_id})
    if (!tok::aligned(p, 4)) return make_status(kInvalid, "logits: device pointers must be aligned to their elements");
  Args a{r, d_logits, d_out, stride, out_stride, vocab, 1, vocab};
  if (n > 0) stretches(n, vocab, &a.parts, &a.len);
  // a launch of fewer than 2^32 threads
  if ((int64_t)n * a.parts >= (int64_t)1 << 23)
    return make_status(kInvalid, "logits: %d rows of %d are more than a launch takes", n, vocab);
  welvet_status st = require_device();
  if (st.code || n == 0) return st;
  WH_HIP(tok::with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const unsigned blocks = (unsigned)(n * a.parts);
    if (d_out == d_logits) rules_kernel<T, true><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
    else rules_kernel<T, false><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
    return hipGetLastError();
  }));
  return ok();
}

}  // extern "C"
