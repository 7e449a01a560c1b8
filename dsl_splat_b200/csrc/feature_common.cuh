// Device helpers of the feature operators (linear, group norm): element types,
// 16-byte vectors of them and the activations.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "splat_common.cuh"

namespace splat {
namespace feature {

// Codes of the C entry points' dtype and activation arguments.
enum Dtype : int { kF32 = 0, kBf16 = 1, kF16 = 2 };
enum Activation : int { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kSigmoid = 4 };

// Whether dy act' has more digits than dy: a slope of 0 or 1 leaves them.
__host__ __device__ constexpr bool rounds_dz(int activation) { return activation >= kSilu; }

using bf16 = __nv_bfloat16;
using f16 = __half;

SPLAT_DEV float to_float(float v) { return v; }
SPLAT_DEV float to_float(bf16 v) { return __bfloat162float(v); }
SPLAT_DEV float to_float(f16 v) { return __half2float(v); }

// One rounding to nearest even, at the end of each output's fp32 arithmetic.
template <class T>
SPLAT_DEV T from_float(float v);
template <>
SPLAT_DEV float from_float<float>(float v) { return v; }
template <>
SPLAT_DEV bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
SPLAT_DEV f16 from_float<f16>(float v) { return __float2half_rn(v); }

template <class T>
constexpr bool kIsF16 = false;
template <>
inline constexpr bool kIsF16<f16> = true;

// V consecutive values, loaded and stored as one access of V * sizeof(T)
// bytes (at most 16), which the address must be a multiple of.
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// The same for V values at once: 16-bit ones are rounded in pairs.
template <class T, int V>
SPLAT_DEV Vec<T, V> round_values(const float (&v)[V]) {
  Vec<T, V> r;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      if constexpr (kIsF16<T>) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = reinterpret_cast<const uint32_t&>(h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = reinterpret_cast<const uint32_t&>(h);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = from_float<T>(v[j]);
  }
  return r;
}

template <class T, int V>
SPLAT_DEV void widen(const Vec<T, V>& r, float (&v)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      if constexpr (kIsF16<T>) {
        const float2 f = __half22float2(reinterpret_cast<const __half2&>(w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      } else {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_float(r.v[j]);
  }
}

// The first of the two values of T that stand for 16-bit layers' dz, and in v
// what it leaves, which is rounded to T for the second: half a step squared
// relative (2^-16 for bf16, 2^-22 for f16) and half of T's smallest value.  The
// first one is at most T's largest, so that the second brings a v beyond it, an
// infinity or a NaN.
template <class T, int V>
SPLAT_DEV Vec<T, V> take_first(float (&v)[V]) {
  constexpr float kMost = kIsF16<T> ? 65504.0f : 3.38953138925153547590470800371e38f;
  float o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = fminf(fmaxf(v[i], -kMost), kMost);
  const Vec<T, V> first = round_values<T, V>(o);
  widen<T, V>(first, o);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] -= o[i];
  return first;
}

// 2^x and 1/x in one instruction each, within 2 units of 2^-23; results below
// the normal range are 0.
SPLAT_DEV float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
SPLAT_DEV float fast_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 1 / (1 + exp(-z)); exp(-z) overflowing to infinity gives 0.
SPLAT_DEV float logistic(float z) {
  return fast_reciprocal(1.0f + fast_exp2(z * -1.44269504088896341f));
}

// The normal distribution's upper tail at |z| and its density: with
// x = |z| / sqrt 2 and t = 1 / (1 + 0.3275911 x), erfc(x) is
// t (a1 + a2 t + .. + a5 t^4) exp(-x^2) within 1.5e-7 (Abramowitz and Stegun,
// Handbook of Mathematical Functions, 7.1.26).
SPLAT_DEV void normal_tail(float z, float& tail, float& density) {
  const float e = fast_exp2(z * z * -0.72134752044448170f);
  const float t = fast_reciprocal(__fmaf_rn(fabsf(z), 0.23164189f, 1.0f));
  float q = __fmaf_rn(t, 1.061405429f, -1.453152027f);
  q = __fmaf_rn(q, t, 1.421413741f);
  q = __fmaf_rn(q, t, -0.284496736f);
  q = __fmaf_rn(q, t, 0.254829592f);
  tail = 0.5f * q * t * e;
  density = 0.39894228040143268f * e;
}

// NaN passes through every activation.
template <int ACT>
SPLAT_DEV float activate(float z) {
  if constexpr (ACT == kRelu) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == kSilu) return z * logistic(z);
  if constexpr (ACT == kGelu) {
    float tail, density;
    normal_tail(z, tail, density);
    return z * (z < 0.0f ? tail : 1.0f - tail);
  }
  if constexpr (ACT == kSigmoid) return logistic(z);
  return z;
}

// d activate / dz.
template <int ACT>
SPLAT_DEV float slope(float z) {
  if constexpr (ACT == kRelu) return z > 0.0f ? 1.0f : 0.0f;
  if constexpr (ACT == kSilu) {
    const float s = logistic(z);
    return s * (1.0f + z * (1.0f - s));
  }
  if constexpr (ACT == kGelu) {
    float tail, density;
    normal_tail(z, tail, density);
    return (z < 0.0f ? tail : 1.0f - tail) + z * density;
  }
  if constexpr (ACT == kSigmoid) {
    const float s = logistic(z);
    return s * (1.0f - s);
  }
  return 1.0f;
}

// Packed pairs: one instruction for both where there is one.
SPLAT_DEV void logistic2(float& a, float& b) {
  unpack2(mul2(pack2(a, b), pack2(-1.44269504088896341f, -1.44269504088896341f)), a, b);
  unpack2(add2(pack2(fast_exp2(a), fast_exp2(b)), pack2(1.0f, 1.0f)), a, b);
  a = fast_reciprocal(a);
  b = fast_reciprocal(b);
}
// normal_tail of a pair: the distribution function's values and the densities'
// exponentials.
SPLAT_DEV void normal2(f32x2 z, float a, float b, f32x2& cdf, f32x2& e) {
  float u, v;
  unpack2(mul2(mul2(z, z), splat2(-0.72134752044448170f)), u, v);
  e = pack2(fast_exp2(u), fast_exp2(v));
  unpack2(fma2(pack2(fabsf(a), fabsf(b)), splat2(0.23164189f), splat2(1.0f)), u, v);
  const f32x2 t = pack2(fast_reciprocal(u), fast_reciprocal(v));
  f32x2 q = fma2(t, splat2(0.5f * 1.061405429f), splat2(0.5f * -1.453152027f));
  q = fma2(q, t, splat2(0.5f * 1.421413741f));
  q = fma2(q, t, splat2(0.5f * -0.284496736f));
  q = fma2(q, t, splat2(0.5f * 0.254829592f));
  float ta, tb, ua, ub;
  const f32x2 tail = mul2(mul2(q, t), e);
  unpack2(tail, ta, tb);
  unpack2(fma2(tail, splat2(-1.0f), splat2(1.0f)), ua, ub);
  cdf = pack2(a < 0.0f ? ta : ua, b < 0.0f ? tb : ub);
}
template <int ACT>
SPLAT_DEV void activate2(float& a, float& b) {
  if constexpr (ACT == kSilu) {
    float s = a, t = b;
    logistic2(s, t);
    unpack2(mul2(pack2(a, b), pack2(s, t)), a, b);
  } else if constexpr (ACT == kSigmoid) {
    logistic2(a, b);
  } else if constexpr (ACT == kGelu) {
    const f32x2 z = pack2(a, b);
    f32x2 cdf, e;
    normal2(z, a, b, cdf, e);
    unpack2(mul2(z, cdf), a, b);
  } else {
    a = activate<ACT>(a);
    b = activate<ACT>(b);
  }
}

template <int ACT>
SPLAT_DEV void slope2(float& a, float& b) {
  if constexpr (ACT == kSilu || ACT == kSigmoid) {
    float s = a, t = b;
    logistic2(s, t);
    const f32x2 p = pack2(s, t), z = pack2(a, b);
    // s + s z (1 - s), and s (1 - s)
    const f32x2 q = fma2(pack2(-s, -t), ACT == kSilu ? z : p, ACT == kSilu ? z : p);
    unpack2(ACT == kSilu ? fma2(p, q, p) : q, a, b);
  } else if constexpr (ACT == kGelu) {
    const f32x2 z = pack2(a, b);
    f32x2 cdf, e;
    normal2(z, a, b, cdf, e);
    unpack2(fma2(mul2(z, splat2(0.39894228040143268f)), e, cdf), a, b);
  } else {
    a = slope<ACT>(a);
    b = slope<ACT>(b);
  }
}

}  // namespace feature
}  // namespace splat

// Runs `call` with T bound to the element type of `dtype` (validated by the
// caller) and, in the second form, ACT to the activation.
#define SPLAT_FEATURE_TYPE(dtype, ...)                             \
  [&] {                                                            \
    switch (dtype) {                                               \
      case splat::feature::kBf16: {                                \
        using T = splat::feature::bf16;                            \
        return __VA_ARGS__();                                      \
      }                                                            \
      case splat::feature::kF16: {                                 \
        using T = splat::feature::f16;                             \
        return __VA_ARGS__();                                      \
      }                                                            \
      default: {                                                   \
        using T = float;                                           \
        return __VA_ARGS__();                                      \
      }                                                            \
    }                                                              \
  }()

#define SPLAT_FEATURE_ACT(act, ...)                                                      \
  [&] {                                                                                  \
    switch (act) {                                                                       \
      case splat::feature::kRelu: { constexpr int ACT = splat::feature::kRelu; return __VA_ARGS__(); }       \
      case splat::feature::kSilu: { constexpr int ACT = splat::feature::kSilu; return __VA_ARGS__(); }       \
      case splat::feature::kGelu: { constexpr int ACT = splat::feature::kGelu; return __VA_ARGS__(); }       \
      case splat::feature::kSigmoid: { constexpr int ACT = splat::feature::kSigmoid; return __VA_ARGS__(); } \
      default: { constexpr int ACT = splat::feature::kNone; return __VA_ARGS__(); }                          \
    }                                                                                    \
  }()
