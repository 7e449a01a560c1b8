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
//
// 59 million fp32 values: 246 us with states in 32 bits (6.7 TB/s); 256 in 8 (3.7 TB/s), of
// which the codes' arithmetic takes its part (ALU pipe 56 %, DRAM 41 % of its cycles), while the
// states take 118 MB instead of 472.  Reading both moments back takes 135.  Steps and rates on
// the device cost each block two powers in 64 bits: 2 us and 12.
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
constexpr int kPiece8 = 16384;      // with states in 8 bits, whose blocks load ahead
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
  float b1, c1, b2, c2;             // the betas and 1 - them
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

// One value: m and v become m' and v', root that of v'; returns p'.  FAST: the quotient
// is off by two units of 2^-23 instead of a half (the root is at least 2^-75 or 0).
template <bool FAST>
SPLAT_DEV float update(float p, float g, float& m, float& v, float& root, const Tensor& t,
                       const Rates& r) {
  m = __fadd_rn(__fmul_rn(m, t.b1), __fmul_rn(g, t.c1));
  v = __fadd_rn(__fmul_rn(v, t.b2), __fmul_rn(__fmul_rn(g, t.c2), g));
  root = __fsqrt_rn(v);
  const float below = fmaf(root, r.unbias, t.eps);
  return fmaf(p, r.shrink, -(FAST ? __fdividef(m, below) : m / below) * r.rate);
}

// ---- states in 32 bits ---------------------------------------------------------------

template <class T>
__global__ void __launch_bounds__(kThreads) step32_kernel(const __grid_constant__ Table table) {
  const Tensor& t = table.t[tensor_of(table)];
  const Rates r = rates_of(t);
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
        pf[k] = update<false>(pf[k], gf[k] * table.ascend, mf[k], vf[k], root, t, r);
      *reinterpret_cast<Vec<T, V>*>(p + i) = round_values<T, V>(pf);
      *reinterpret_cast<float4*>(m + i) = mv;
      *reinterpret_cast<float4*>(v + i) = vv;
    }
    // what a last piece has behind its whole vectors
    const long long i = whole + threadIdx.x;
    if (i < end) {
      float root;
      p[i] = from_float<T>(update<false>(to_float(p[i]), to_float(g[i]) * table.ascend, m[i], v[i],
                                         root, t, r));
    }
  } else {
    for (long long i = begin + threadIdx.x; i < end; i += kThreads) {
      float root;
      p[i] = from_float<T>(update<false>(to_float(p[i]), to_float(g[i]) * table.ascend, m[i], v[i],
                                         root, t, r));
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

// What a code of M bits of mantissa stands for in a run of the given factor: the shifted
// code is an fp32 number 2^112 below it.  Both powers of two are exact, but for results
// below fp32's normal range, which are rounded once.
struct Factor {
  float near, far;  // 2^(112 + E), of which far is what fp32 cannot hold
};
SPLAT_DEV Factor factor_of(int exponent) {
  if (exponent == kNotFinite) return {__uint_as_float(0x7fc00000u), 1.0f};
  const int near = min(exponent, 15);
  return {power(112 + near), power(exponent - near)};
}
// The four codes of a word.
template <int M>
SPLAT_DEV void decode4(uint32_t word, const Factor& factor, float* v) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t top = word << (24 - 8 * k);  // the code in the highest byte
    const uint32_t bits = M == 3 ? static_cast<uint32_t>(static_cast<int>(top) >> 4) & 0x87f00000u
                                 : (top >> 5) & 0x07f80000u;
    v[k] = __uint_as_float(bits) * factor.near;
  }
  if (factor.far != 1.0f) {  // of a whole run
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= factor.far;
  }
}

// The run's exponent from its largest magnitude's bits.
template <int M>
SPLAT_DEV int exponent_of(uint32_t most) {
  if (most >= 0x7f800000u) return kNotFinite;
  constexpr uint32_t kTop = (1u << 23) - (1u << (23 - M));  // the largest code's mantissa
  const int e = static_cast<int>(most >> 23) - 127 + ((most & 0x7fffffu) > kTop);
  return min(max(e, -126), 127);
}

// The code of |x| 2^-E = y; noise: 16 bits of a step, the half of which rounds to the
// nearest.  That of y below the normal codes is taken apart because it is rare.
template <int M>
SPLAT_DEV uint32_t encode_normal(float y, uint32_t noise) {
  constexpr int kDrop = 23 - M;
  return min((__float_as_uint(y) + (noise << (kDrop - 16)) - (112u << 23)) >> kDrop,
             M == 3 ? 127u : 255u);
}
template <int M>
SPLAT_DEV uint32_t encode_small(float y, uint32_t noise) {
  const uint32_t c = static_cast<uint32_t>(floorf(__fadd_rn(
      y * static_cast<float>(1 << (14 + M)), static_cast<float>(noise) * 0x1p-16f)));
  return M == 4 && c == 0 && y > 0.0f ? 1u : c;
}
constexpr float kLeastNormal = 0x1p-14f;

// A warp's run: eight values to a lane, four of each half, so that every access of the
// warp is contiguous.
constexpr int kLane = kRun / 32;
SPLAT_DEV int place_of(int k) { return (k >> 2) * 128 + (threadIdx.x & 31) * 4 + (k & 3); }

// left: values of the run.
template <class S>
SPLAT_DEV void load_lane(const S* run, bool vector, int left, S (&to)[kLane]) {
#pragma unroll
  for (int k = 0; k < kLane; k += 4) {
    const int at = place_of(k);
    if (vector && at + 4 <= left) {
      reinterpret_cast<Vec<S, 4>&>(to[k]) = *reinterpret_cast<const Vec<S, 4>*>(run + at);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) to[k + j] = at + j < left ? run[at + j] : S(0.0f);
    }
  }
}
template <class S>
SPLAT_DEV void store_lane(S* run, bool vector, int left, const S (&from)[kLane]) {
#pragma unroll
  for (int k = 0; k < kLane; k += 4) {
    const int at = place_of(k);
    if (vector && at + 4 <= left) {
      *reinterpret_cast<Vec<S, 4>*>(run + at) = reinterpret_cast<const Vec<S, 4>&>(from[k]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at + j < left) run[at + j] = from[k + j];
    }
  }
}
SPLAT_DEV int left_of(long long n, long long run) {
  return static_cast<int>(max(0LL, min(n - run * kRun, static_cast<long long>(kRun))));
}

// A lane's codes, four to a word.
SPLAT_DEV void load_codes(const unsigned char* run, bool vector, int left, uint32_t (&w)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = place_of(4 * h);
    w[h] = 0;
    if (vector && at + 4 <= left) {
      w[h] = *reinterpret_cast<const uint32_t*>(run + at);
    } else {
      for (int j = 0; j < 4; ++j)
        if (at + j < left) w[h] |= static_cast<uint32_t>(run[at + j]) << (8 * j);
    }
  }
}
SPLAT_DEV void store_codes(unsigned char* run, bool vector, int left, const uint32_t (&w)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = place_of(4 * h);
    if (vector && at + 4 <= left) {
      *reinterpret_cast<uint32_t*>(run + at) = w[h];
    } else {
      for (int j = 0; j < 4; ++j)
        if (at + j < left) run[at + j] = static_cast<unsigned char>(w[h] >> (8 * j));
    }
  }
}

// The codes of a run and its exponent; SHIFT: of 16 bits of noise in each word.  Values
// behind the run's last are zeros.
template <int M, int SHIFT>
SPLAT_DEV void store_run(const float (&x)[kLane], const uint32_t (&noise)[kLane], bool vector,
                         int left, unsigned char* codes, signed char* exponent) {
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < kLane; ++k) most = max(most, __float_as_uint(x[k]) & 0x7fffffffu);
  most = __reduce_max_sync(0xffffffffu, most);
  const int e = exponent_of<M>(most);
  const float inverse = power(e == kNotFinite ? 0 : -e);
  uint32_t w[2];
  float least = INFINITY;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = 4 * h + j;
      const float y = fabsf(x[k]) * inverse;
      least = fminf(least, y);
      c[j] = encode_normal<M>(y, noise[k] >> SHIFT & 0xffffu);
      if (M == 3) c[j] |= __float_as_uint(x[k]) >> 24 & 128u;
    }
    w[h] = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
  }
  if (__any_sync(0xffffffffu, least < kLeastNormal)) {
#pragma unroll
    for (int k = 0; k < kLane; ++k) {
      const float y = fabsf(x[k]) * inverse;
      const uint32_t c = encode_small<M>(y, noise[k] >> SHIFT & 0xffffu) |
                         (M == 3 && x[k] < 0.0f ? 128u : 0u);
      const int at = 8 * (k & 3);
      if (y < kLeastNormal) w[k >> 2] = (w[k >> 2] & ~(255u << at)) | c << at;
    }
  }
  store_codes(codes, vector, left, w);
  if ((threadIdx.x & 31) == 0) *exponent = static_cast<signed char>(e);
}

// What a warp reads of a run.
template <class T>
struct Run {
  alignas(16) T p[kLane];
  alignas(16) T g[kLane];
  uint32_t m[2], v[2];
  int m_exponent, v_exponent;
  SPLAT_DEV void load(const Tensor& t, long long run) {
    const int left = left_of(t.n, run);
    const long long i = run * kRun;
    load_lane(static_cast<const T*>(t.p) + i, t.vector, left, p);
    load_lane(static_cast<const T*>(t.g) + i, t.vector, left, g);
    load_codes(static_cast<const unsigned char*>(t.m) + i, t.vector, left, m);
    load_codes(static_cast<const unsigned char*>(t.v) + i, t.vector, left, v);
    m_exponent = left ? t.m_exponents[run] : 0;
    v_exponent = left ? t.v_exponents[run] : 0;
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads, 3) step8_kernel(const __grid_constant__ Table table) {
  const Tensor& t = table.t[tensor_of(table)];
  const Rates r = rates_of(t);
  constexpr int kWarps = kThreads / 32;
  long long run = static_cast<long long>(blockIdx.x - t.first_block) * (kPiece8 / kRun) +
                  (threadIdx.x >> 5);
  Run<T> next;
  next.load(t, run);
  for (int k = 0; k < kPiece8 / kRun; k += kWarps, run += kWarps) {
    if (run * kRun >= t.n) break;
    Run<T> now = next;
    if (k + kWarps < kPiece8 / kRun) next.load(t, run + kWarps);
    const long long i = run * kRun;
    const int left = left_of(t.n, run);
    const Factor mf = factor_of(now.m_exponent), vf = factor_of(now.v_exponent);
    float m[kLane], root[kLane];
    uint32_t noise[kLane];
    decode4<3>(now.m[0], mf, m);
    decode4<3>(now.m[1], mf, m + 4);
    decode4<4>(now.v[0], vf, root);
    decode4<4>(now.v[1], vf, root + 4);
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      float v = __fmul_rn(root[j], root[j]);
      now.p[j] = from_float<T>(update<true>(to_float(now.p[j]), to_float(now.g[j]) * table.ascend,
                                            m[j], v, root[j], t, r));
      noise[j] = dither(i + place_of(j), r.step);
    }
    store_lane(static_cast<T*>(t.p) + i, t.vector, left, now.p);
    store_run<3, 0>(m, noise, t.vector, left, static_cast<unsigned char*>(t.m) + i,
                    t.m_exponents + run);
    store_run<4, 16>(root, noise, t.vector, left, static_cast<unsigned char*>(t.v) + i,
                     t.v_exponents + run);
  }
}

// Codes -> the values that they stand for (squared: of v), and back, to the nearest.
template <bool SQUARED>
__global__ void __launch_bounds__(kThreads)
    decode_kernel(long long n, const unsigned char* codes, const signed char* exponents,
                  bool vector, float* values) {
  constexpr int U = 2;  // runs in flight
  const long long runs = (n + kRun - 1) / kRun, step = gridDim.x * (kThreads / 32LL);
  for (long long run0 = blockIdx.x * (kThreads / 32LL) + (threadIdx.x >> 5); run0 < runs;
       run0 += U * step) {
    uint32_t c[U][2];
    int e[U], left[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long run = run0 + u * step;
      left[u] = left_of(n, run);
      load_codes(codes + run * kRun, vector, left[u], c[u]);
      e[u] = run < runs ? exponents[run] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Factor factor = factor_of(e[u]);
      alignas(16) float v[kLane];
      decode4<SQUARED ? 4 : 3>(c[u][0], factor, v);
      decode4<SQUARED ? 4 : 3>(c[u][1], factor, v + 4);
      if (SQUARED)
#pragma unroll
        for (int k = 0; k < kLane; ++k) v[k] = __fmul_rn(v[k], v[k]);
      store_lane(values + (run0 + u * step) * kRun, vector, left[u], v);
    }
  }
}
template <bool SQUARED>
__global__ void __launch_bounds__(kThreads)
    encode_kernel(long long n, const float* values, bool vector, unsigned char* codes,
                  signed char* exponents) {
  const long long runs = (n + kRun - 1) / kRun, step = gridDim.x * (kThreads / 32LL);
  for (long long run = blockIdx.x * (kThreads / 32LL) + (threadIdx.x >> 5); run < runs;
       run += step) {
    const int left = left_of(n, run);
    alignas(16) float v[kLane];
    uint32_t half[kLane];
    load_lane(values + run * kRun, vector, left, v);
#pragma unroll
    for (int k = 0; k < kLane; ++k) {
      if (SQUARED) v[k] = __fsqrt_rn(v[k]);
      half[k] = 0x8000u;
    }
    store_run<SQUARED ? 4 : 3, 0>(v, half, vector, left, codes + run * kRun, exponents + run);
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
      const int piece = bits == 8 ? kPiece8 : kPiece;
      const long long more = (from.n + piece - 1) / piece;
      if (blocks && blocks + more >= 1LL << 31) break;
      Tensor& t = table.t[table.count++];
      t.p = from.p, t.g = from.g, t.m = from.m, t.v = from.v;
      t.m_exponents = static_cast<signed char*>(from.m_exponents);
      t.v_exponents = static_cast<signed char*>(from.v_exponents);
      t.device_step = from.device_step, t.device_lr = from.device_lr;
      t.lr = from.lr, t.decay = from.weight_decay, t.beta1 = from.beta1, t.beta2 = from.beta2;
      t.b1 = static_cast<float>(t.beta1), t.c1 = static_cast<float>(1.0 - t.beta1);
      t.b2 = static_cast<float>(t.beta2), t.c2 = static_cast<float>(1.0 - t.beta2);
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
