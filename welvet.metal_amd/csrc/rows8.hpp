// rows8.hpp — rows in 8 bits, shared by rows8.hip (storing them, SwiGLU),
// int8.hip (products of them) and rows8_backward.hip: a row's values as codes
// c in [-127, 127] and one scale s, value = s c.  Internal to the library.
//   s = max |x| / 127, rounded to f32;  c = x / s, to nearest, ties to even
// The code is that of the exact quotient: a product with 1 / s decides unless
// it lies within 2e-5 of a half (it is off by at most 127 2^-23), where the remainder x - k s does, exactly.
// A row of zeros has s = 0; one that holds a NaN or an infinity has s = NaN and
// codes 0, so whatever reads it is NaN.
#pragma once

#include "tokens.hpp"

namespace wh {
namespace r8 {

using namespace tok;

constexpr int kPad = 16;  // a row's codes: whole 16-byte words
inline int64_t padded(int64_t width) { return (width + kPad - 1) / kPad * kPad; }

struct Scale {
  float stored;   // the row's scale
  float s, inv;   // of the lifted values
  float lift;     // 2^64 for rows whose scale is near the smallest float
  bool finite;
  // top: the largest magnitude's bits, above infinity's where a value is NaN
  __device__ explicit Scale(uint32_t top) {
    finite = top < 0x7f800000u;
    stored = finite ? u2f(top) / 127.0f : u2f(0x7fc00000u);
    lift = finite && stored < 0x1p-100f ? 0x1p64f : 1.0f;
    s = stored * lift;
    inv = finite && stored > 0.0f ? 1.0f / s : 0.0f;
  }
  __device__ inline int code(float x) const {
    const float a = fabsf(x) * lift, q = a * inv;
    float t = rintf(q);
    if (fabsf(q - t) > 0.49998f) {
      // within 2e-5 of a half: k + 1/2 against the quotient by the remainder,
      // a multiple of a's or s's last place near s / 2, so the fma does not round
      const float k = floorf(q), d = fmaf(-k, s, a), half = 0.5f * s;
      t = d > half || (d == half && ((int)k & 1)) ? k + 1.0f : k;
    }
    t = fminf(t, 127.0f);  // a scale that was rounded down among the smallest floats
    return (int)copysignf(t, x);
  }
};
__device__ inline uint32_t magnitude(float x) { return f2u(x) & 0x7fffffffu; }

// Eight neighbouring values wherever they lie, as floats; zeros from `width` on.
template <class T>
struct Oct {
  using raw = typename T::raw;
  static constexpr int kWords = sizeof(raw) * 2;
  uint32_t w[kWords];
  __device__ inline void load(const raw *p) { __builtin_memcpy(w, p, sizeof(w)); }
  __device__ inline void load(const raw *row, int64_t c, int64_t width) {
    if (c + 8 <= width) return load(row + c);
    raw r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = c + i < width ? row[c + i] : (raw)0;
    __builtin_memcpy(w, r, sizeof(w));
  }
  __device__ inline raw raw_at(int i) const {
    if constexpr (sizeof(raw) == 4) return w[i];
    else return (raw)(w[i >> 1] >> (16 * (i & 1)));
  }
  __device__ inline float get(int i) const { return T::get(raw_at(i)); }
  __device__ inline void set_raw(int i, raw v) {
    if constexpr (sizeof(raw) == 4) w[i] = v;
    else if (i & 1) w[i >> 1] = (w[i >> 1] & 0xffffu) | ((uint32_t)v << 16);
    else w[i >> 1] = (w[i >> 1] & 0xffff0000u) | v;
  }
  // the same where i is not known to the compiler
  __device__ inline raw at(int i) const {
    constexpr int kPer = 4 / sizeof(raw);
    uint32_t v = 0;  // by masks: of selects the compiler makes an array in memory
#pragma unroll
    for (int k = 0; k < kWords; ++k) v |= w[k] & (0u - (uint32_t)(i / kPer == k));
    return (raw)(v >> (8 * sizeof(raw) * (i % kPer)));
  }
  __device__ inline void set_at(int i, raw v) {
    constexpr int kPer = 4 / sizeof(raw);
    const int by = 8 * sizeof(raw) * (i % kPer);
    const uint32_t mask = (sizeof(raw) == 4 ? 0xffffffffu : 0xffffu) << by;
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] ^= (w[k] ^ (uint32_t)v << by) & mask & (0u - (uint32_t)(i / kPer == k));
  }
  __device__ inline void set(int i, float v) { set_raw(i, T::put(v)); }
  __device__ inline void fill(raw v) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = sizeof(raw) == 4 ? (uint32_t)v : (uint32_t)v * 0x10001u;
  }
  __device__ inline void store(raw *row, int64_t c, int64_t width) const {
    if (c + 8 <= width) {
      __builtin_memcpy(row + c, w, sizeof(w));
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < width) row[c + i] = raw_at(i);
  }
};

// Codes of eight values as two words (0 throughout in a row that is not finite).
// fma(x, inv, 1.5 2^23) is x inv rounded to a whole number, as its last bits.
template <class F>
__device__ inline uint2 codes8(const Scale &q, F &&value) {
  constexpr float kWhole = 0x1.8p23f;
  if (!q.finite) return make_uint2(0, 0);
  uint32_t c[8];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = value(i), r = fmaf(x, q.inv, kWhole);
    c[i] = f2u(r);
    off = fmaxf(off, fabsf(fmaf(x, q.inv, kWhole - r)));
  }
  if (off > 0.49998f || q.lift != 1.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = (uint32_t)q.code(value(i));
  }
  const auto four = [&](int i) {  // the last bytes of four words
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[i + 3], c[i + 2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(c[i + 1], c[i], 0x0c0c0400u), 0x05040100u);
  };
  return make_uint2(four(0), four(4));
}
// A row by eights: `whole` of them in full, loaded without a condition (a branch
// around each load would have it waited for before the next), a thread past
// the last having that again; and what is left, one thread's.
struct Eights {
  int whole, left;
  __device__ explicit Eights(int width) : whole(width / 8), left(width % 8) {}
  template <class T>
  __device__ inline void load(Oct<T> &o, const typename T::raw *row, int at) const {
    o.load(row + (int64_t)min(at, whole - 1) * 8);
  }
  // The row's last codes: those of `o`, where something is left, and zeros up to
  // the row's multiple of 16.
  template <class T>
  __device__ inline void finish(int8_t *codes, const Scale &q, const Oct<T> &o) const {
    int at = whole;
    if (left) *(uint2 *)(codes + 8 * at++) = codes8(q, [&](int i) { return o.get(i); });
    if (at & 1) *(uint2 *)(codes + 8 * at) = make_uint2(0, 0);
  }
};
// The largest magnitude's bits so far, in the type's own width.
template <class T>
__device__ inline void raise(uint32_t &top, const Oct<T> &o) {
  if constexpr (sizeof(typename T::raw) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, o.w[i] & 0x7fffffffu);
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 t = __builtin_bit_cast(u16x2, top);
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, o.w[i] & 0x7fff7fffu));
    top = __builtin_bit_cast(uint32_t, t);
  }
}
// ... as an f32's.
template <class T>
__device__ inline uint32_t widened(uint32_t top) {
  if constexpr (sizeof(typename T::raw) == 4) return top;
  else return magnitude(T::get((typename T::raw)max(top & 0xffffu, top >> 16)));
}
__device__ inline float value_of(uint32_t word, int i) { return (float)(int8_t)(word >> (8 * i)); }

// 2^t below 2^-126 is 0 to the instruction: there it takes 2^(t + 64) (the sum is
// exact) and the result is brought down by this, rounded to what is left of it.
constexpr float kLow = -126.0f, kDown = 0x1p-64f;
// z = 1 / (1 + e^-x) and 1 - z, each within 4 ulp, below 2^-126 within its last place
// more: from e^-|x|, the argument's product with log2 e carried past f32.
struct Sigmoid {
  float z, co;
  __device__ explicit Sigmoid(float x) {
    const float a = fabsf(x), t = -1.44269502f * a;
    const float rest = fmaf(-1.44269502f, a, -t) - 1.92596299e-8f * a;
    float e = __builtin_amdgcn_exp2f(t);
    const auto carry = [&] { e = fmaf(e * rest, 0.693147181f, e); };
    if (__builtin_expect(t <= kLow, 0)) {
      e = __builtin_amdgcn_exp2f(t + 64.0f);
      if (t > -1000.0f) carry();  // else e is 0, and rest may be NaN
      e *= kDown;
    } else {
      carry();
    }
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    z = x < 0.0f ? e * r : r;
    co = x < 0.0f ? r : e * r;
    if (x != x) z = co = x;
  }
};
// The activations and their derivatives in f32, by the formulas of act_value
// and act_prime, but of NaN, a row that is not finite, always NaN: those give
// ReLU's answer and the piecewise derivatives whole values for it.
__device__ inline float gelu_arg(float x) { return 1.59576912f * fmaf(0.044715f * x * x, x, x); }  // 2 u of 0.5 x (1 + tanh u)
__device__ inline float act_f32(float x, int act) {
  switch (act) {
  case kReLU: return x <= 0.0f ? 0.0f : x;
  case kReLU2: return x < 0.0f ? 0.0f : x * x;
  case kLeakyReLU: return x < 0.0f ? (float)((double)x * 0.01) : x;
  case kSilu: return x * Sigmoid(x).z;
  case kSigmoid: return Sigmoid(x).z;
  case kTanh: return tanhf(x);
  case kGELU: return x * Sigmoid(gelu_arg(x)).z;
  }
  return x;
}
// Before a rounding to 16 bits, or SwiGLU's product to 8, from kQuick on: the
// exponential's argument rounded once, which moves z by at most 0.4 2^-24 and x z, for
// x < 0, by |x| 2^-24 of itself.  Below, e^-x or its reciprocal leaves the instructions'
// range.
constexpr float kQuick = -87.0f;
__device__ inline float quick_sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269502f * x));
}
// The activations of N values that become a T, each by itself alone; whether the quick
// sigmoid takes them all is looked at once (a select a value instead: SwiGLU of bf16
// 8192 x 11008 into 8 bits 141 us for 127, f16 int8 4096 -> 11008 of 8192 rows 410 / 402).
template <class T, int ACT, int N>
__device__ inline void acts(float (&v)[N]) {
  if constexpr (sizeof(typename T::raw) == 2 && (ACT == kSilu || ACT == kSigmoid || ACT == kGELU)) {
    float z[N], least = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      z[i] = ACT == kGELU ? gelu_arg(v[i]) : v[i];
      least = fminf(least, z[i]);
    }
    const auto set = [&](int i, float s) { v[i] = ACT == kSigmoid ? s : v[i] * s; };
    if (least >= kQuick) {
#pragma unroll
      for (int i = 0; i < N; ++i) set(i, quick_sigmoid(z[i]));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) set(i, z[i] < kQuick ? Sigmoid(z[i]).z : quick_sigmoid(z[i]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = act_f32(v[i], ACT);
}
template <class T, int N>
__device__ inline void acts(float (&v)[N], int act) {
  const auto each = [&](auto a) { acts<T, decltype(a)::value>(v); };
  switch (act) {
  case kReLU: return each(std::integral_constant<int, kReLU>{});
  case kReLU2: return each(std::integral_constant<int, kReLU2>{});
  case kLeakyReLU: return each(std::integral_constant<int, kLeakyReLU>{});
  case kSilu: return each(std::integral_constant<int, kSilu>{});
  case kSigmoid: return each(std::integral_constant<int, kSigmoid>{});
  case kTanh: return each(std::integral_constant<int, kTanh>{});
  case kGELU: return each(std::integral_constant<int, kGELU>{});
  }
}
__device__ inline float act_prime_f32(float x, int act) {
  switch (act) {
  case kSilu: {
    const Sigmoid s(x);
    return fmaf(x * s.z, s.co, s.z);
  }
  case kSigmoid: {
    const Sigmoid s(x);
    return s.z * s.co;
  }
  case kTanh: {
    const Sigmoid s(2.0f * x);
    return 4.0f * s.z * s.co;
  }
  case kGELU: {
    if (fabsf(x) > 20.0f) return x > 0.0f ? 1.0f : 0.0f;  // where x x x may be infinite
    const Sigmoid s(gelu_arg(x));
    return fmaf(x * s.z * s.co, 1.59576912f * fmaf(0.134145f * x, x, 1.0f), s.z);
  }
  }
  return x != x ? x : act_prime_piecewise(x, act);
}

__device__ inline void prime8(float (&v)[8], int act) {
  const auto each = [&](auto a) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_prime_f32(v[i], decltype(a)::value);
  };
  switch (act) {
  case kReLU: return each(std::integral_constant<int, kReLU>{});
  case kReLU2: return each(std::integral_constant<int, kReLU2>{});
  case kLeakyReLU: return each(std::integral_constant<int, kLeakyReLU>{});
  case kSilu: return each(std::integral_constant<int, kSilu>{});
  case kSigmoid: return each(std::integral_constant<int, kSigmoid>{});
  case kTanh: return each(std::integral_constant<int, kTanh>{});
  case kGELU: return each(std::integral_constant<int, kGELU>{});
  default: return each(std::integral_constant<int, kLinear>{});
  }
}

// What the rows' operators take: widths whose columns an int holds with a
// block's steps past them, rows that a grid walks.
constexpr int32_t kMaxWidth = 1 << 24, kMaxRows = 1 << 24;
inline bool size_ok(int32_t n, int32_t width) { return n >= 0 && n <= kMaxRows && width > 0 && width <= kMaxWidth; }
// A description of n rows: why it cannot be taken, or nullptr.
inline const char *rows_fault(const welvet_hip_rows8 *r, int32_t n, int32_t width) {
  if (!r) return "null rows";
  if (n > 0 && (!r->d_codes || !r->d_scales)) return "null codes or scales";
  if (!aligned(r->d_codes, 16) || r->stride % kPad != 0) return "codes and their stride must be multiples of 16 bytes";
  if (!aligned(r->d_scales, 4)) return "device pointers must be aligned to their elements";
  if (r->stride < padded(width)) return "stride of the codes below the width rounded up to 16";
  return nullptr;
}
// rows8.hip: the store by itself, for the layers' weights and the forward.
hipError_t launch_store(int32_t dtype, int32_t n, int32_t width, const void *x, int64_t x_stride, int8_t *codes,
                        int64_t codes_stride, float *scales, hipStream_t s);

}  // namespace r8
}  // namespace wh
