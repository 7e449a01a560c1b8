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

// from_float of V values at once: 16-bit ones are rounded in pairs.
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
  Vec<T, V> first;
  uint32_t* w = reinterpret_cast<uint32_t*>(&first);
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    if constexpr (kIsF16<T>)
      asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(v[i + 1]), "f"(v[i]));
    else
      asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(v[i + 1]), "f"(v[i]));
  }
  float o[V];
  widen<T, V>(first, o);
#pragma unroll
  for (int i = 0; i < V; i += 2)
    unpack2(sub2(pack2(v[i], v[i + 1]), pack2(o[i], o[i + 1])), v[i], v[i + 1]);
  return first;
}

// 2^x and 1/x in one instruction each, within 2 units of 2^-23; results below
// the normal range are 0 (of exp2_whole: are not).
SPLAT_DEV float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
SPLAT_DEV float exp2_whole(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
SPLAT_DEV float fast_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The activations work on packed pairs: one instruction for both where there is
// one.  FINE is for fp32, whose results keep their digits however small they
// are; for 16-bit types 2^-14 of a result will do.
//
// 2^(-h C) for C = C_0 + C_1: the rounding of h C_0 alone, 2^-24 of itself, would
// cost the power h C 2^-24.  FINE takes that rounding, C_1 and `rest`, what h
// leaves out of its value (0 for NULL), to first order.  hn is -h.
template <bool FINE>
SPLAT_DEV f32x2 exp2_of(f32x2 hn, float c0, float c1, const f32x2* rest) {
  const f32x2 y = mul2(hn, splat2(c0));
  float a, b;
  unpack2(y, a, b);
  if constexpr (FINE) {
    const f32x2 e = pack2(exp2_whole(a), exp2_whole(b));
    f32x2 less = fma2(hn, splat2(-c1), fma2(hn, splat2(-c0), y));
    if (rest) less = fma2(*rest, splat2(c0), less);
    return fma2(mul2(less, splat2(-0.693147180559945309f)), e, e);
  } else {
    return pack2(fast_exp2(a), fast_exp2(b));
  }
}

// |z|; FINE: at most a value from which every function here is 0 or 1, because
// infinities have no rounding.  NaN stays.
template <bool FINE>
SPLAT_DEV float magnitude(float z, float most) {
  return FINE && fabsf(z) > most ? most : fabsf(z);
}

// e = exp(-|z|) and r = 1 / (1 + e): the logistic function is r or, of negative
// arguments, e r, and the other of them is 1 less it, without cancellation.
template <bool FINE>
SPLAT_DEV void logistic_parts(float a, float b, f32x2& e, f32x2& r) {
  const f32x2 hn = pack2(-magnitude<FINE>(a, 200.0f), -magnitude<FINE>(b, 200.0f));
  e = exp2_of<FINE>(hn, 1.44269504088896341f, 1.925962990e-8f, nullptr);
  float u, v;
  unpack2(add2(e, splat2(1.0f)), u, v);
  r = pack2(fast_reciprocal(u), fast_reciprocal(v));
}
template <bool FINE>
SPLAT_DEV void logistic2(float& a, float& b) {
  if constexpr (FINE) {
    f32x2 e, r;
    logistic_parts<true>(a, b, e, r);
    float u, v, s, t;
    unpack2(mul2(e, r), u, v);
    unpack2(r, s, t);
    a = a < 0.0f ? u : s;
    b = b < 0.0f ? v : t;
  } else {  // exp(-z) overflowing to infinity gives 0
    unpack2(mul2(pack2(a, b), splat2(-1.44269504088896341f)), a, b);
    unpack2(add2(pack2(fast_exp2(a), fast_exp2(b)), splat2(1.0f)), a, b);
    a = fast_reciprocal(a);
    b = fast_reciprocal(b);
  }
}

// The normal distribution function of a pair, and e = exp(-z^2 / 2).  Its tail
// at |z| is e Q(|z|); Q(z) / t with t = 1 / (1 + p z) is a polynomial in t fitted
// to erfc(z / sqrt 2) exp(z^2 / 2) / 2 by least squares whose weights follow the
// relative error (Lawson's iteration): 2.5e-8 relative up to 20 (FINE), 2.9e-5
// up to 13.5.
template <bool FINE>
SPLAT_DEV void normal2(float a, float b, f32x2& cdf, f32x2& e) {
  const float x = magnitude<FINE>(a, 20.0f), y = magnitude<FINE>(b, 20.0f);
  const f32x2 z = pack2(x, y), hn = mul2(z, pack2(-x, -y));
  const f32x2 rest = fma2(z, z, hn);
  e = exp2_of<FINE>(hn, 0.72134752044448170f, 9.62981495e-9f, &rest);
  float u, v;
  unpack2(fma2(z, splat2(FINE ? 0.27f : 0.375f), splat2(1.0f)), u, v);
  const f32x2 t = pack2(fast_reciprocal(u), fast_reciprocal(v));
  f32x2 q;
  if constexpr (FINE) {
    q = fma2(t, splat2(0.0290643238f), splat2(-0.127003357f));
    q = fma2(q, t, splat2(0.170891672f));
    q = fma2(q, t, splat2(-0.0705219954f));
    q = fma2(q, t, splat2(0.108767502f));
    q = fma2(q, t, splat2(0.071631223f));
    q = fma2(q, t, splat2(0.101922527f));
    q = fma2(q, t, splat2(0.107526444f));
    q = fma2(q, t, splat2(0.107721671f));
  } else {
    q = fma2(t, splat2(-0.0909852087f), splat2(0.201043263f));
    q = fma2(q, t, splat2(0.0829740763f));
    q = fma2(q, t, splat2(0.157920063f));
    q = fma2(q, t, splat2(0.149041131f));
  }
  float ta, tb, ua, ub;
  const f32x2 tail = mul2(mul2(q, t), e);
  unpack2(tail, ta, tb);
  unpack2(fma2(tail, splat2(-1.0f), splat2(1.0f)), ua, ub);
  cdf = pack2(a < 0.0f ? ta : ua, b < 0.0f ? tb : ub);
}

// NaN passes through every activation.
template <int ACT, bool FINE>
SPLAT_DEV void activate2(float& a, float& b) {
  if constexpr (ACT == kRelu) {
    a = a < 0.0f ? 0.0f : a;
    b = b < 0.0f ? 0.0f : b;
  } else if constexpr (ACT == kSilu) {
    float s = a, t = b;
    logistic2<FINE>(s, t);
    unpack2(mul2(pack2(a, b), pack2(s, t)), a, b);
  } else if constexpr (ACT == kGelu) {
    f32x2 cdf, e;
    normal2<FINE>(a, b, cdf, e);
    unpack2(mul2(pack2(a, b), cdf), a, b);
  } else if constexpr (ACT == kSigmoid) {
    logistic2<FINE>(a, b);
  }
}

// d activate / dz.
template <int ACT, bool FINE>
SPLAT_DEV void slope2(float& a, float& b) {
  if constexpr (ACT == kRelu) {
    a = a > 0.0f ? 1.0f : 0.0f;
    b = b > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (ACT == kSilu && !FINE) {
    // s + s z (1 - s): where 1 - s cancels, it is small beside the rest
    float s = a, t = b;
    logistic2<false>(s, t);
    const f32x2 p = pack2(s, t), z = pack2(a, b);
    unpack2(fma2(p, fma2(pack2(-s, -t), z, z), p), a, b);
  } else if constexpr (ACT == kSilu || ACT == kSigmoid) {
    f32x2 e, r;
    logistic_parts<FINE>(a, b, e, r);
    const f32x2 other = mul2(e, r), both = mul2(other, r);  // s (1 - s)
    if constexpr (ACT == kSigmoid) {
      unpack2(both, a, b);
    } else {
      float u, v, s, t;
      unpack2(other, u, v);
      unpack2(r, s, t);
      // s + z s (1 - s)
      unpack2(fma2(pack2(a, b), both, pack2(a < 0.0f ? u : s, b < 0.0f ? v : t)), a, b);
    }
  } else if constexpr (ACT == kGelu) {
    f32x2 cdf, e;
    normal2<FINE>(a, b, cdf, e);
    unpack2(fma2(mul2(pack2(a, b), splat2(0.39894228040143268f)), e, cdf), a, b);
  } else {
    a = b = 1.0f;
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
