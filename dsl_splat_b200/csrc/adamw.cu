// AdamW over many tensors at once:
//
//   m' = b1 m + (1 - b1) g,  v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Bound by memory: 28 bytes a value with fp32 parameters and states, 16 with states
// in 8 bits.  A launch takes up to kMostTensors tensors, whose pieces its blocks find
// in the table that is the launch's parameter.
//
// States in 8 bits.  Runs of 256 values of the flattened tensor share an exponent E,
// the least in [-126, 127] whose largest code reaches the run's largest magnitude.
// A code c of M bits of mantissa stands for 2^E (1 + (c mod 2^M) / 2^M) 2^(c div 2^M - 15),
// or below 2^M for 2^E c 2^(-14 - M): m with a sign and M = 3, the root of v with
// M = 4.  Being a power of two, the run's factor costs no digits, and the root
// halves the range of exponents that v would need.
//
// A moving average's step is smaller than half a step of such a code (v moves by a
// thousandth, the codes are 2^-4 apart), so rounding to the nearest would hold it
// where it is.  Values are rounded down after a dither below one step has been added, a
// hash of the value's place and the step's number: off by less than one step, and
// right on average.  A root that is not zero stays above zero, or m / (0 + eps)
// could follow.  The states' arithmetic is single fp32 operations in a fixed order,
// because a code depends on which side of a border its value lies.
#include <algorithm>
#include <cmath>

#include "feature_common.cuh"
#include "host_runtime.h"
#include "splat200.h"

namespace splat {
namespace adamw {

using feature::bf16;
using feature::f16;
using feature::from_float;
using feature::round_values;
using feature::to_float;
using feature::Vec;
using feature::widen;

constexpr int kThreads = 256;
constexpr int kMostTensors = 96;
constexpr int kRun = 256;           // values that share an exponent
constexpr int kPiece = 4096;        // values of a block
constexpr int kNotFinite = -128;    // exponent of a run with infinities or NaN: all are NaN

struct Tensor {
  void* p;
  const void* g;
  void *m, *v;
  signed char *m_exponents, *v_exponents;
  const long long* device_step;  // or NULL: the host knew the step
  const float* device_lr;        // or NULL: the host knew the learning rate
  double lr, decay, beta1, beta2;
  long long n;
  float shrink, rate, unbias, eps;  // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t step, first_block;
  int vector;  // every base lies on 16 bytes
};
struct Table {
  int count;
  float ascend;  // -1 to maximise
  Tensor t[kMostTensors];
};
static_assert(sizeof(Table) < 32000, "a launch's parameters");

// What the host leaves to the device.
struct Rates {
  float shrink, rate, unbias;
  uint32_t step;
};
SPLAT_DEV Rates rates_of(const Tensor& t) {
  Rates r{t.shrink, t.rate, t.unbias, t.step};
  if (t.device_step || t.device_lr) {
    __shared__ Rates shared;
    if (threadIdx.x == 0) {
      const long long step = t.device_step ? *t.device_step : static_cast<long long>(t.step);
      const double lr = t.device_lr ? static_cast<double>(*t.device_lr) : t.lr;
      r.step = static_cast<uint32_t>(step);
      r.shrink = static_cast<float>(1.0 - lr * t.decay);
      r.rate = static_cast<float>(lr / (1.0 - pow(t.beta1, static_cast<double>(step))));
      r.unbias = static_cast<float>(1.0 / sqrt(1.0 - pow(t.beta2, static_cast<double>(step))));
      shared = r;
    }
    __syncthreads();
    r = shared;
  }
  return r;
}

// The tensor of a block.
SPLAT_DEV int tensor_of(const Table& table) {
  int low = 0, high = table.count;  // first_block[low] <= block < first_block[high]
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (table.t[mid].first_block <= blockIdx.x) low = mid;
    else high = mid;
  }
  return low;
}

struct Betas {
  float b1, c1, b2, c2;
  SPLAT_DEV explicit Betas(const Tensor& t)
      : b1(static_cast<float>(t.beta1)),
        c1(static_cast<float>(1.0 - t.beta1)),
        b2(static_cast<float>(t.beta2)),
        c2(static_cast<float>(1.0 - t.beta2)) {}
};

// One value: m and v become m' and the root of v'; returns p'.
SPLAT_DEV float update(float p, float g, float& m, float& v, float& root, const Betas& b,
                       const Rates& r, float eps) {
  m = __fadd_rn(__fmul_rn(m, b.b1), __fmul_rn(g, b.c1));
  v = __fadd_rn(__fmul_rn(v, b.b2), __fmul_rn(__fmul_rn(g, b.c2), g));
  root = __fsqrt_rn(v);
  return p * r.shrink - m / fmaf(root, r.unbias, eps) * r.rate;
}

// ---- states in 32 bits ---------------------------------------------------------------

template <class T>
__global__ void __launch_bounds__(kThreads) step32_kernel(const __grid_constant__ Table table) {
  const Tensor& t = table.t[tensor_of(table)];
  const Rates r = rates_of(t);
  const Betas betas(t);
  const long long begin = static_cast<long long>(blockIdx.x - t.first_block) * kPiece;
  const long long end = min(begin + kPiece, t.n);
  T* p = static_cast<T*>(t.p);
  const T* g = static_cast<const T*>(t.g);
  float *m = static_cast<float*>(t.m), *v = static_cast<float*>(t.v);
  if (t.vector) {
    constexpr int V = 4;
    const long long whole = begin + (end - begin) / V * V;
    for (long long i = begin + threadIdx.x * V; i < whole; i += kThreads * V) {
      Vec<T, V> pv = *reinterpret_cast<const Vec<T, V>*>(p + i);
      const Vec<T, V> gv = *reinterpret_cast<const Vec<T, V>*>(g + i);
      float4 mv = *reinterpret_cast<const float4*>(m + i);
      float4 vv = *reinterpret_cast<const float4*>(v + i);
      float pf[V], gf[V], root;
      widen<T, V>(pv, pf);
      widen<T, V>(gv, gf);
      float* mf = reinterpret_cast<float*>(&mv);
      float* vf = reinterpret_cast<float*>(&vv);
#pragma unroll
      for (int k = 0; k < V; ++k)
        pf[k] = update(pf[k], gf[k] * table.ascend, mf[k], vf[k], root, betas, r, t.eps);
      *reinterpret_cast<Vec<T, V>*>(p + i) = round_values<T, V>(pf);
      *reinterpret_cast<float4*>(m + i) = mv;
      *reinterpret_cast<float4*>(v + i) = vv;
    }
    // what a last piece has behind its whole vectors
    const long long i = whole + threadIdx.x;
    if (i < end) {
      float root;
      p[i] = from_float<T>(update(to_float(p[i]), to_float(g[i]) * table.ascend, m[i], v[i], root,
                                  betas, r, t.eps));
    }
  } else {
    for (long long i = begin + threadIdx.x; i < end; i += kThreads) {
      float root;
      p[i] = from_float<T>(update(to_float(p[i]), to_float(g[i]) * table.ascend, m[i], v[i], root,
                                  betas, r, t.eps));
    }
  }
}

// ---- states in 8 bits ----------------------------------------------------------------

// 2^e for e in [-127, 127].
SPLAT_DEV float power(int e) {
  return __uint_as_float(e == -127 ? 0x00400000u : static_cast<uint32_t>(e + 127) << 23);
}

// 16 bits for each of the two moments of value i at a step.
SPLAT_DEV uint32_t dither(long long i, uint32_t step) {
  uint32_t h = static_cast<uint32_t>(i) * 0x9e3779b9u + step * 0x6a09e667u +
               static_cast<uint32_t>(i >> 32) * 0xbb67ae85u;
  h = (h ^ (h >> 16)) * 0x3c6ef373u;
  h = (h ^ (h >> 15)) * 0x510e527fu;
  return h ^ (h >> 16);
}

// What a code of M bits of mantissa stands for in a run of the given factor; the
// shifted code is an fp32 number 2^112 below it.
template <int M>
SPLAT_DEV float decode(uint32_t c, float factor) {
  const uint32_t size = M == 3 ? c & 127u : c;
  const float v = __uint_as_float(size << (23 - M)) * 0x1p112f * factor;
  return M == 3 && (c & 128u) ? -v : v;
}
SPLAT_DEV float factor_of(int exponent) {
  return exponent == kNotFinite ? __uint_as_float(0x7fc00000u) : power(exponent);
}

// The run's exponent from its largest magnitude's bits.
template <int M>
SPLAT_DEV int exponent_of(uint32_t most) {
  if (most >= 0x7f800000u) return kNotFinite;
  constexpr uint32_t kTop = (1u << 23) - (1u << (23 - M));  // the largest code's mantissa
  const int e = static_cast<int>(most >> 23) - 127 + ((most & 0x7fffffu) > kTop);
  return min(max(e, -126), 127);
}

// The code of x; noise: 16 bits of a step, the half of which rounds to the nearest.
template <int M>
SPLAT_DEV uint32_t encode(float x, float inverse, uint32_t noise) {
  constexpr int kDrop = 23 - M;
  const float y = fabsf(x) * inverse;
  const uint32_t normal =
      ((__float_as_uint(y) + (noise << (kDrop - 16))) >> kDrop) - (112u << M);
  const uint32_t small = static_cast<uint32_t>(
      floorf(__fadd_rn(y * static_cast<float>(1 << (14 + M)), static_cast<float>(noise) * 0x1p-16f)));
  uint32_t c = y < 0x1p-14f ? small : normal;
  if constexpr (M == 3) {
    return min(c, 127u) | (x < 0.0f ? 128u : 0u);
  } else {
    c = min(c, 255u);
    return c == 0 && x > 0.0f ? 1u : c;
  }
}

// A warp's run: eight values to a lane.
constexpr int kLane = kRun / 32;

template <class S>
SPLAT_DEV void load_lane(const S* from, bool vector, int valid, S (&to)[kLane]) {
  if (vector && valid == kLane) {
    constexpr int B = sizeof(S) * kLane > 16 ? 16 : sizeof(S) * kLane, V = B / sizeof(S);
#pragma unroll
    for (int k = 0; k < kLane; k += V)
      reinterpret_cast<Vec<S, V>&>(to[k]) = *reinterpret_cast<const Vec<S, V>*>(from + k);
  } else {
#pragma unroll
    for (int k = 0; k < kLane; ++k) to[k] = k < valid ? from[k] : S(0.0f);
  }
}
template <class S>
SPLAT_DEV void store_lane(S* to, bool vector, int valid, const S (&from)[kLane]) {
  if (vector && valid == kLane) {
    constexpr int B = sizeof(S) * kLane > 16 ? 16 : sizeof(S) * kLane, V = B / sizeof(S);
#pragma unroll
    for (int k = 0; k < kLane; k += V)
      *reinterpret_cast<Vec<S, V>*>(to + k) = reinterpret_cast<const Vec<S, V>&>(from[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kLane; ++k)
      if (k < valid) to[k] = from[k];
  }
}

// The codes of a run and its exponent.
template <int M>
SPLAT_DEV void store_run(const float (&x)[kLane], const uint32_t (&noise)[kLane], bool vector,
                         int valid, unsigned char* codes, signed char* exponent) {
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < kLane; ++k)
    if (k < valid) most = max(most, __float_as_uint(x[k]) & 0x7fffffffu);
  most = __reduce_max_sync(0xffffffffu, most);
  const int e = exponent_of<M>(most);
  const float inverse = power(e == kNotFinite ? 0 : -e);
  alignas(16) unsigned char c[kLane];
#pragma unroll
  for (int k = 0; k < kLane; ++k)
    c[k] = static_cast<unsigned char>(encode<M>(x[k], inverse, noise[k]));
  store_lane(codes, vector, valid, c);
  if ((threadIdx.x & 31) == 0) *exponent = static_cast<signed char>(e);
}

template <class T>
__global__ void __launch_bounds__(kThreads) step8_kernel(const __grid_constant__ Table table) {
  const Tensor& t = table.t[tensor_of(table)];
  const Rates r = rates_of(t);
  const Betas betas(t);
  const long long block = blockIdx.x - t.first_block;
  const int lane = threadIdx.x & 31;
  for (int k = threadIdx.x >> 5; k < kPiece / kRun; k += kThreads / 32) {
    const long long run = block * (kPiece / kRun) + k;
    if (run * kRun >= t.n) break;
    const long long i = run * kRun + lane * kLane;
    const int valid = static_cast<int>(max(0LL, min(t.n - i, static_cast<long long>(kLane))));
    alignas(16) T p[kLane], g[kLane];
    alignas(16) unsigned char mc[kLane], vc[kLane];
    load_lane(static_cast<const T*>(t.p) + i, t.vector, valid, p);
    load_lane(static_cast<const T*>(t.g) + i, t.vector, valid, g);
    load_lane(static_cast<const unsigned char*>(t.m) + i, t.vector, valid, mc);
    load_lane(static_cast<const unsigned char*>(t.v) + i, t.vector, valid, vc);
    const float mf = factor_of(t.m_exponents[run]), vf = factor_of(t.v_exponents[run]);
    float m[kLane], root[kLane];
    uint32_t low[kLane], high[kLane];
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      m[j] = decode<3>(mc[j], mf);
      const float before = decode<4>(vc[j], vf);
      float v = __fmul_rn(before, before);
      p[j] = from_float<T>(update(to_float(p[j]), to_float(g[j]) * table.ascend, m[j], v, root[j],
                                  betas, r, t.eps));
      const uint32_t h = dither(i + j, r.step);
      low[j] = h & 0xffffu;
      high[j] = h >> 16;
    }
    store_lane(static_cast<T*>(t.p) + i, t.vector, valid, p);
    store_run<3>(m, low, t.vector, valid, static_cast<unsigned char*>(t.m) + i,
                 t.m_exponents + run);
    store_run<4>(root, high, t.vector, valid, static_cast<unsigned char*>(t.v) + i,
                 t.v_exponents + run);
  }
}

// Codes -> the values that they stand for (squared: of v), and back, to the nearest.
template <bool SQUARED>
__global__ void __launch_bounds__(kThreads)
    decode_kernel(long long n, const unsigned char* codes, const signed char* exponents,
                  bool vector, float* values) {
  const int lane = threadIdx.x & 31;
  const long long runs = (n + kRun - 1) / kRun, step = gridDim.x * (kThreads / 32LL);
  for (long long run = blockIdx.x * (kThreads / 32LL) + (threadIdx.x >> 5); run < runs;
       run += step) {
    const long long i = run * kRun + lane * kLane;
    const int valid = static_cast<int>(max(0LL, min(n - i, static_cast<long long>(kLane))));
    alignas(16) unsigned char c[kLane];
    alignas(16) float v[kLane];
    load_lane(codes + i, vector, valid, c);
    const float factor = factor_of(exponents[run]);
#pragma unroll
    for (int k = 0; k < kLane; ++k) {
      v[k] = decode<SQUARED ? 4 : 3>(c[k], factor);
      if (SQUARED) v[k] = __fmul_rn(v[k], v[k]);
    }
    store_lane(values + i, vector, valid, v);
  }
}
template <bool SQUARED>
__global__ void __launch_bounds__(kThreads)
    encode_kernel(long long n, const float* values, bool vector, unsigned char* codes,
                  signed char* exponents) {
  const int lane = threadIdx.x & 31;
  const long long runs = (n + kRun - 1) / kRun, step = gridDim.x * (kThreads / 32LL);
  for (long long run = blockIdx.x * (kThreads / 32LL) + (threadIdx.x >> 5); run < runs;
       run += step) {
    const long long i = run * kRun + lane * kLane;
    const int valid = static_cast<int>(max(0LL, min(n - i, static_cast<long long>(kLane))));
    alignas(16) float v[kLane];
    uint32_t half[kLane];
    load_lane(values + i, vector, valid, v);
#pragma unroll
    for (int k = 0; k < kLane; ++k) {
      if (SQUARED) v[k] = __fsqrt_rn(v[k]);
      half[k] = 0x8000u;
    }
    store_run<SQUARED ? 4 : 3>(v, half, vector, valid, codes + i, exponents + run);
  }
}

int check_moment(long long n, const void* codes, const void* exponents, const void* values) {
  if (n < 1) return host::fail(kInvalidArgument, "adamw_moment: sizes");
  if (!codes || !exponents || !values)
    return host::fail(kInvalidArgument, "adamw_moment: null pointer");
  return kOk;
}
unsigned moment_grid(long long n) {
  return static_cast<unsigned>(std::min<long long>((n + kPiece / 2 - 1) / (kPiece / 2),
                                                   32LL * host::sm_count()));
}
bool aligned16(std::initializer_list<const void*> all) {
  return std::all_of(all.begin(), all.end(), [](const void* p) { return host::aligned(p, 16); });
}

template <class T>
int launch_step(const Table& table, unsigned blocks, int bits, cudaStream_t s) {
  if (bits == 8) step8_kernel<T><<<blocks, kThreads, 0, host::counted(s)>>>(table);
  else step32_kernel<T><<<blocks, kThreads, 0, host::counted(s)>>>(table);
  return host::check_launch("adamw");
}

}  // namespace adamw
}  // namespace splat

using namespace splat;
using namespace splat::adamw;

extern "C" {

int splat_adamw(int dtype, int bits, int count, const SplatAdamwTensor* tensors, int maximize,
                void* stream) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "adamw: dtype");
  if (bits != 8 && bits != 32) return host::fail(kInvalidArgument, "adamw: bits");
  if (count < 0 || (count && !tensors)) return host::fail(kInvalidArgument, "adamw: tensors");
  for (int i = 0; i < count; ++i) {
    const SplatAdamwTensor& from = tensors[i];
    if (from.n < 0) return host::fail(kInvalidArgument, "adamw: sizes");
    if (from.n > 1LL << 40) return host::fail(kTooLarge, "adamw: too many values");
    if (from.n && (!from.p || !from.g || !from.m || !from.v ||
                   (bits == 8 && (!from.m_exponents || !from.v_exponents))))
      return host::fail(kInvalidArgument, "adamw: null pointer");
    if (!from.device_step && from.step < 1) return host::fail(kInvalidArgument, "adamw: step");
  }
  auto s = static_cast<cudaStream_t>(stream);
  for (int next = 0; next < count;) {
    Table table;
    table.count = 0;
    table.ascend = maximize ? -1.0f : 1.0f;
    long long blocks = 0;
    for (; next < count && table.count < kMostTensors; ++next) {
      const SplatAdamwTensor& from = tensors[next];
      if (!from.n) continue;
      const long long more = (from.n + kPiece - 1) / kPiece;
      if (blocks && blocks + more >= 1LL << 31) break;
      Tensor& t = table.t[table.count++];
      t.p = from.p, t.g = from.g, t.m = from.m, t.v = from.v;
      t.m_exponents = static_cast<signed char*>(from.m_exponents);
      t.v_exponents = static_cast<signed char*>(from.v_exponents);
      t.device_step = from.device_step, t.device_lr = from.device_lr;
      t.lr = from.lr, t.decay = from.weight_decay, t.beta1 = from.beta1, t.beta2 = from.beta2;
      t.n = from.n, t.eps = static_cast<float>(from.eps);
      t.step = static_cast<uint32_t>(from.step);
      t.shrink = static_cast<float>(1.0 - t.lr * t.decay);
      t.rate = t.unbias = 0.0f;
      if (!from.device_step) {
        const double step = static_cast<double>(from.step);
        t.rate = static_cast<float>(t.lr / (1.0 - std::pow(t.beta1, step)));
        t.unbias = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(t.beta2, step)));
      }
      t.vector = aligned16({t.p, t.g, t.m, t.v});
      t.first_block = static_cast<uint32_t>(blocks);
      blocks += more;
    }
    if (!table.count) break;
    const int status = SPLAT_FEATURE_TYPE(dtype, [&] {
      return launch_step<T>(table, static_cast<unsigned>(blocks), bits, s);
    });
    if (status != kOk) return status;
  }
  return kOk;
}

int splat_adamw_decode(long long n, const void* codes, const void* exponents, int squared,
                       float* values, void* stream) {
  const int bad = check_moment(n, codes, exponents, values);
  if (bad != kOk) return bad;
  auto s = host::counted(static_cast<cudaStream_t>(stream));
  const auto* c = static_cast<const unsigned char*>(codes);
  const auto* e = static_cast<const signed char*>(exponents);
  const bool vector = aligned16({codes, values});
  if (squared) decode_kernel<true><<<moment_grid(n), kThreads, 0, s>>>(n, c, e, vector, values);
  else decode_kernel<false><<<moment_grid(n), kThreads, 0, s>>>(n, c, e, vector, values);
  return host::check_launch("adamw_decode");
}

int splat_adamw_encode(long long n, const float* values, int squared, void* codes,
                       void* exponents, void* stream) {
  const int bad = check_moment(n, codes, exponents, values);
  if (bad != kOk) return bad;
  auto s = host::counted(static_cast<cudaStream_t>(stream));
  auto* c = static_cast<unsigned char*>(codes);
  auto* e = static_cast<signed char*>(exponents);
  const bool vector = aligned16({codes, values});
  if (squared) encode_kernel<true><<<moment_grid(n), kThreads, 0, s>>>(n, values, vector, c, e);
  else encode_kernel<false><<<moment_grid(n), kThreads, 0, s>>>(n, values, vector, c, e);
  return host::check_launch("adamw_encode");
}

}  // extern "C"
