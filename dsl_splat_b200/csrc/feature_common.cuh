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

// V consecutive values, loaded and stored as one access of V * sizeof(T)
// bytes (at most 16), which the address must be a multiple of.
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// 1 / (1 + exp(-z)): exp2 of a scaled argument and a reciprocal, each within
// a few units of 2^-23; exp(-z) overflowing to infinity gives 0.
SPLAT_DEV float logistic(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// NaN passes through every activation.
template <int ACT>
SPLAT_DEV float activate(float z) {
  if constexpr (ACT == kRelu) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == kSilu) return z * logistic(z);
  if constexpr (ACT == kGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
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
  if constexpr (ACT == kGelu)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
           z * 0.39894228040143268f * __expf(-0.5f * z * z);
  if constexpr (ACT == kSigmoid) {
    const float s = logistic(z);
    return s * (1.0f - s);
  }
  return 1.0f;
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
