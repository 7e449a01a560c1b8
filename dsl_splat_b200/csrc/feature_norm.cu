// Group norm with an activation over channel-last tensors, forward and
// backward.
//
//   y = act(u),  u = xhat w_c + b_c,  xhat = (x - mean_bg) rstd_bg
//
// x is (samples B, positions S, channels C); the mean and the biased variance
// of sample b and group g run over its S positions and C/G channels.  With
// du = dy act'(u) and n = S C/G the gradients are
//
//   db_c = sum_bs du            dw_c = sum_bs du xhat
//   dx   = rstd (w_c du - m1 - xhat m2),  m1 = sum_g w_c du / n,
//                                         m2 = sum_g w_c du xhat / n
//
// Both directions are a reduction of two sums per channel over the rows of a
// sample, a small kernel that joins the blocks' sums, and a pass that writes
// the result.  Sums over channels of a group are taken after the sums over
// rows, so one layout serves any C and G: see Layout.
#include <algorithm>
#include <numeric>

#include "feature_common.cuh"
#include "host_runtime.h"
#include "splat200.h"

namespace splat {
namespace feature {

// How a sample's S*C values are dealt to threads.  They are read as vectors
// of V values in memory order; the channels of vector i repeat with a period
// of C / gcd(C, V) vectors.  A block of a whole number of periods steps by
// its own width, so that a thread meets the same V channels at every step and
// keeps their sums and parameters in registers, and a block's loads are
// contiguous whatever C is.  Where one period is wider than a block, `columns`
// blocks share it.
struct Layout {
  long long span;   // values of a sample, S * C
  int channels;
  int period;       // vectors
  int threads;      // of a block
  int columns;      // blocks that share a period (1 unless period > kMaxThreads)
  int step;         // vectors between a thread's steps
  int steps;        // of a sample
  int blocks;       // of a sample along its rows; a block takes per_block steps
  int per_block;
};

constexpr int kMaxThreads = 256;

struct NormParams {
  Layout l;
  int samples, groups, group_channels;
  const void* x;
  const void* dy;
  const void* weight;  // (C) or NULL: 1
  const void* bias;    // (C) or NULL: 0
  void* out;           // y or dx
  float* mean;         // (B, G)
  float* rstd;
  float2* partial;     // (B, blocks * columns, C)
  float2* moments;     // (B, G): m1, m2
  double2* channel;    // (B, C): sums of du and du xhat
  float eps;
};

// V fp32 values as packed pairs (one plain value when V is 1): what a thread
// keeps of its channels, and the arithmetic on them.
template <int V>
struct Pairs {
  static constexpr int N = (V + 1) / 2;
  f32x2 v[N];
  SPLAT_DEV void set(const float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = pack2(x[2 * i], V == 1 ? 0.0f : x[2 * i + 1 < V ? 2 * i + 1 : 0]);
  }
  SPLAT_DEV void get(float (&x)[V]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float a, b;
      unpack2(v[i], a, b);
      x[2 * i] = a;
      if (2 * i + 1 < V) x[2 * i + 1] = b;
    }
  }
};
template <int V>
SPLAT_DEV Pairs<V> operator+(Pairs<V> a, const Pairs<V>& b) {
#pragma unroll
  for (int i = 0; i < Pairs<V>::N; ++i) a.v[i] = add2(a.v[i], b.v[i]);
  return a;
}
template <int V>
SPLAT_DEV Pairs<V> operator*(Pairs<V> a, const Pairs<V>& b) {
#pragma unroll
  for (int i = 0; i < Pairs<V>::N; ++i) a.v[i] = mul2(a.v[i], b.v[i]);
  return a;
}
template <int V>
SPLAT_DEV Pairs<V> fma(Pairs<V> a, const Pairs<V>& b, const Pairs<V>& c) {
#pragma unroll
  for (int i = 0; i < Pairs<V>::N; ++i) a.v[i] = fma2(a.v[i], b.v[i], c.v[i]);
  return a;
}
template <int ACT, int V>
SPLAT_DEV Pairs<V> activate(Pairs<V> x) {
#pragma unroll
  for (int i = 0; i < Pairs<V>::N; ++i) {
    float a, b;
    unpack2(x.v[i], a, b);
    if constexpr (V == 1) a = activate<ACT>(a);
    else activate2<ACT>(a, b);
    x.v[i] = pack2(a, b);
  }
  return x;
}
template <int ACT, int V>
SPLAT_DEV Pairs<V> slope(Pairs<V> x) {
#pragma unroll
  for (int i = 0; i < Pairs<V>::N; ++i) {
    float a, b;
    unpack2(x.v[i], a, b);
    if constexpr (V == 1) a = slope<ACT>(a);
    else slope2<ACT>(a, b);
    x.v[i] = pack2(a, b);
  }
  return x;
}

template <class T, int V>
SPLAT_DEV Pairs<V> widen_pairs(const Vec<T, V>& r) {
  float f[V];
  widen<T, V>(r, f);
  Pairs<V> p;
  p.set(f);
  return p;
}
// Values read for the last time, and results, which need not stay in the L2.
template <class V>
SPLAT_DEV V load_last(const V* p) {
  if constexpr (sizeof(V) == 16) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    return reinterpret_cast<const V&>(u);
  } else {
    return *p;
  }
}
template <class V>
SPLAT_DEV void store_streaming(V* p, const V& v) {
  if constexpr (sizeof(V) == 16)
    __stcs(reinterpret_cast<uint4*>(p), reinterpret_cast<const uint4&>(v));
  else
    *p = v;
}
template <class T, int V>
SPLAT_DEV Vec<T, V> round_pairs(const Pairs<V>& p) {
  float f[V];
  p.get(f);
  return round_values<T, V>(f);
}
// The vector that a lone sample may end inside: its `left` values.
template <class T, int V>
SPLAT_DEV Vec<T, V> load_part(const T* p, int left) {
  Vec<T, V> r;
#pragma unroll
  for (int j = 0; j < V; ++j) r.v[j] = j < left ? p[j] : from_float<T>(0.0f);
  return r;
}
template <class T, int V>
SPLAT_DEV void store_part(T* p, const Vec<T, V>& r, int left) {
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (j < left) p[j] = r.v[j];
}

// What a thread of any of the passes works on: `count` whole vectors, the
// first at `first` (values from the sample's start) and `stride` values apart,
// and the part of a last one (`left` values, usually none) behind them.
struct Place {
  int sample, part, column;  // part: the block along the sample's rows
  int vector;                // of the period(s) at a step
  int count, left;
  long long first, stride;
};

template <int V>
SPLAT_DEV Place place(const Layout& l) {
  Place p;
  unsigned b = blockIdx.x;
  p.column = 0;
  if (l.columns > 1) {
    p.column = b % l.columns;
    b /= l.columns;
  }
  p.sample = b / l.blocks;
  p.part = b - p.sample * l.blocks;
  p.vector = p.column * l.threads + threadIdx.x;
  const int begin = p.part * l.per_block, end = min(begin + l.per_block, l.steps);
  p.first = (static_cast<long long>(begin) * l.step + p.vector) * V;
  p.stride = static_cast<long long>(l.step) * V;
  p.count = p.left = 0;
  if (p.vector < l.step) {
    // every step but the sample's last is whole
    p.count = end - begin;
    if (end == l.steps) {
      const long long o = p.first + (p.count - 1) * p.stride;
      if (o + V > l.span) {
        --p.count;
        p.left = static_cast<int>(max(l.span - o, 0LL));
      }
    }
  }
  return p;
}

// Sums the block's per-thread sums over the threads that share a channel and
// writes one pair per channel, in a fixed order.
template <int V>
SPLAT_DEV void write_partial(const NormParams& p, const Place& at, const float (&s1)[V],
                             const float (&s2)[V]) {
  __shared__ float2 sums[kMaxThreads * V];
  const Layout& l = p.l;
#pragma unroll
  for (int j = 0; j < V; ++j) sums[threadIdx.x * V + j] = make_float2(s1[j], s2[j]);
  __syncthreads();
  const int first = at.column * l.threads * V;  // flat position of sums[0] in a step
  const int count = min(l.threads, l.step - at.column * l.threads) * V;
  float2* out = p.partial +
                ((static_cast<long long>(at.sample) * l.blocks + at.part) * l.columns + at.column) *
                    l.channels;
  for (int c = threadIdx.x; c < l.channels; c += l.threads) {
    int i = c - first % l.channels;
    if (i < 0) i += l.channels;
    float a = 0.0f, b = 0.0f;
    for (; i < count; i += l.channels) {
      a += sums[i].x;
      b += sums[i].y;
    }
    out[c] = make_float2(a, b);
  }
}

// Sums of x - pivot and its square per channel; the pivot is the sample's
// first row, so that a large common offset does not cancel.
template <class T, int V>
__global__ void __launch_bounds__(kMaxThreads, 4) norm_sums_kernel(const NormParams p) {
  using Values = Vec<T, V>;
  const Layout& l = p.l;
  const Place at = place<V>(l);
  const T* x = static_cast<const T*>(p.x) + at.sample * l.span;
  float zero[V] = {}, pivot[V];
  Pairs<V> minus, s1, s2;
  s1.set(zero);
  s2.set(zero);
  const bool active = at.count || at.left;
#pragma unroll
  for (int j = 0; j < V; ++j)
    pivot[j] =
        active ? -to_float(x[(static_cast<long long>(at.vector) * V + j) % l.channels]) : 0.0f;
  minus.set(pivot);
  const T* from = x + at.first;
  constexpr int U = 4;
  int i = 0;
  for (; i + U <= at.count; i += U) {
    Values v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = *reinterpret_cast<const Values*>(from + u * at.stride);
    from += U * at.stride;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Pairs<V> d = widen_pairs<T, V>(v[u]) + minus;
      s1 = s1 + d;
      s2 = fma(d, d, s2);
    }
  }
  for (; i < at.count; ++i, from += at.stride) {
    const Pairs<V> d = widen_pairs<T, V>(*reinterpret_cast<const Values*>(from)) + minus;
    s1 = s1 + d;
    s2 = fma(d, d, s2);
  }
  float a[V], b[V];
  s1.get(a);
  s2.get(b);
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (j < at.left) {
      const float d = to_float(from[j]) + pivot[j];
      a[j] += d;
      b[j] += d * d;
    }
  write_partial<V>(p, at, a, b);
}

SPLAT_DEV double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The blocks' sums of up to kJoinChannels channels from c0 on, joined in
// shared memory: neighbouring threads read neighbouring channels of a block's
// row, and the threads of a channel are added up in a fixed order.
constexpr int kJoinThreads = 256, kJoinChannels = 32;

SPLAT_DEV void channel_sums(const NormParams& p, int sample, int c0, int count,
                            double2 (&joined)[kJoinChannels]) {
  __shared__ double2 sums[kJoinThreads];
  const int parts = p.l.blocks * p.l.columns;
  const float2* in =
      p.partial + static_cast<long long>(sample) * parts * p.l.channels + c0;
  const int lanes = kJoinThreads / count, c = threadIdx.x % count, lane = threadIdx.x / count;
  double a = 0.0, b = 0.0;
  if (lane < lanes) {
#pragma unroll 8
    for (int i = lane; i < parts; i += lanes) {
      const float2 v = in[static_cast<long long>(i) * p.l.channels + c];
      a += v.x;
      b += v.y;
    }
  }
  __syncthreads();
  sums[threadIdx.x] = make_double2(a, b);
  __syncthreads();
  // a warp to a channel: its lanes' sums, then those of the warp
  for (int k = threadIdx.x >> 5; k < count; k += kJoinThreads / 32) {
    a = b = 0.0;
    for (int i = threadIdx.x & 31; i < lanes; i += 32) {
      a += sums[i * count + k].x;
      b += sums[i * count + k].y;
    }
    a = warp_sum(a);
    b = warp_sum(b);
    if ((threadIdx.x & 31) == 0) joined[k] = make_double2(a, b);
  }
  __syncthreads();
}

// Mean and reciprocal deviation of one group: the channels' (count, mean, sum
// of squared deviations) joined one after another, in doubles:
//   M = M_a + M_b + (mean_b - mean_a)^2 n_a n_b / (n_a + n_b).
template <class T>
__global__ void __launch_bounds__(kJoinThreads) norm_join_kernel(const NormParams p) {
  __shared__ double2 joined[kJoinChannels];
  const int sample = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
  const double rows = static_cast<double>(p.l.span / p.l.channels);
  const T* x = static_cast<const T*>(p.x) + sample * p.l.span;
  double n = 0.0, mean = 0.0, m2 = 0.0;
  for (int k0 = 0; k0 < p.group_channels; k0 += kJoinChannels) {
    const int c0 = g * p.group_channels + k0, count = min(kJoinChannels, p.group_channels - k0);
    channel_sums(p, sample, c0, count, joined);
    if (threadIdx.x == 0) {
      for (int k = 0; k < count; ++k) {
        const double2 s = joined[k];
        const double channel_mean = s.x / rows + static_cast<double>(to_float(x[c0 + k]));
        const double channel_m2 = s.y - s.x * s.x / rows;
        const double d = channel_mean - mean, total = n + rows;
        m2 += channel_m2 + d * d * n * rows / total;
        mean += d * rows / total;
        n = total;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    // rounding can leave a constant group a hair below zero; NaN stays
    const double var = m2 < 0.0 ? 0.0 : m2 / n;
    p.mean[blockIdx.x] = static_cast<float>(mean);
    p.rstd[blockIdx.x] = static_cast<float>(1.0 / sqrt(var + static_cast<double>(p.eps)));
  }
}

// The parameters of a thread's V channels: -mean, rstd w, b, and for the
// backward -rstd m1 and -rstd^2 m2, so that with d = x - mean
//   u = d (rstd w) + b,  dx = du (rstd w) - d rstd^2 m2 - rstd m1.
template <class T, int V, bool BACKWARD>
struct Channels {
  Pairs<V> minus, scale, bias, k1, k2;
  SPLAT_DEV void load(const NormParams& p, const Place& at) {
    float m[V], s[V], b[V], x1[V], x2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = static_cast<int>((static_cast<long long>(at.vector) * V + j) % p.l.channels);
      const int g = at.sample * p.groups + c / p.group_channels;
      const float rstd = p.rstd[g];
      m[j] = -p.mean[g];
      s[j] = rstd * (p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0f);
      b[j] = p.bias ? to_float(static_cast<const T*>(p.bias)[c]) : 0.0f;
      if constexpr (BACKWARD) {
        const float2 sums = p.moments[g];
        x1[j] = -rstd * sums.x;
        x2[j] = -rstd * rstd * sums.y;
      }
    }
    minus.set(m);
    scale.set(s);
    bias.set(b);
    if constexpr (BACKWARD) {
      k1.set(x1);
      k2.set(x2);
    }
  }
};

// The passes that write go through a block's steps backwards: what the pass
// before read last is still in the L2.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads, 4) norm_apply_kernel(const NormParams p) {
  using Values = Vec<T, V>;
  const Layout& l = p.l;
  const Place at = place<V>(l);
  if (!at.count && !at.left) return;
  const long long end = at.sample * l.span + at.first + at.count * at.stride;
  const T* from = static_cast<const T*>(p.x) + end;
  T* to = static_cast<T*>(p.out) + end;
  Channels<T, V, false> ch;
  ch.load(p, at);
  const auto result = [&](const Values& v) {
    return round_pairs<T, V>(
        activate<ACT, V>(fma(widen_pairs<T, V>(v) + ch.minus, ch.scale, ch.bias)));
  };
  if (at.left) store_part<T, V>(to, result(load_part<T, V>(from, at.left)), at.left);
  constexpr int U = 4;
  int i = at.count;
  for (; i >= U; i -= U) {
    Values v[U];
    from -= U * at.stride;
    to -= U * at.stride;
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = load_last(reinterpret_cast<const Values*>(from + u * at.stride));
#pragma unroll
    for (int u = 0; u < U; ++u)
      store_streaming(reinterpret_cast<Values*>(to + u * at.stride), result(v[u]));
  }
  for (; i > 0; --i) {
    from -= at.stride;
    to -= at.stride;
    store_streaming(reinterpret_cast<Values*>(to),
                    result(load_last(reinterpret_cast<const Values*>(from))));
  }
}

// Sums of du and du (x - mean) per channel.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads, 3) norm_backward_sums_kernel(const NormParams p) {
  using Values = Vec<T, V>;
  const Layout& l = p.l;
  const Place at = place<V>(l);
  float a[V] = {}, b[V] = {};
  Pairs<V> s1, s2;
  s1.set(a);
  s2.set(a);
  if (at.count || at.left) {
    const T* from = static_cast<const T*>(p.x) + at.sample * l.span + at.first;
    const T* grad = static_cast<const T*>(p.dy) + at.sample * l.span + at.first;
    Channels<T, V, false> ch;
    ch.load(p, at);
    const auto add = [&](const Values& v, const Values& g) {
      const Pairs<V> d = widen_pairs<T, V>(v) + ch.minus;
      const Pairs<V> du = slope<ACT, V>(fma(d, ch.scale, ch.bias)) * widen_pairs<T, V>(g);
      s1 = s1 + du;
      s2 = fma(du, d, s2);
    };
    constexpr int U = 2;
    int i = 0;
    for (; i + U <= at.count; i += U, from += U * at.stride, grad += U * at.stride) {
      Values v[U], g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u] = *reinterpret_cast<const Values*>(from + u * at.stride);
        g[u] = *reinterpret_cast<const Values*>(grad + u * at.stride);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) add(v[u], g[u]);
    }
    for (; i < at.count; ++i, from += at.stride, grad += at.stride)
      add(*reinterpret_cast<const Values*>(from), *reinterpret_cast<const Values*>(grad));
    // an upstream of 0 behind the end adds nothing unless x - mean is not
    // finite, which the sums of the values before it are not then either
    if (at.left) add(load_part<T, V>(from, at.left), load_part<T, V>(grad, at.left));
  }
  s1.get(a);
  s2.get(b);
  write_partial<V>(p, at, a, b);
}

template <class T>
__global__ void __launch_bounds__(kJoinThreads) norm_backward_join_kernel(const NormParams p) {
  __shared__ double2 joined[kJoinChannels];
  const int sample = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
  const double rstd = p.rstd[blockIdx.x];
  double m1 = 0.0, m2 = 0.0;
  for (int k0 = 0; k0 < p.group_channels; k0 += kJoinChannels) {
    const int c0 = g * p.group_channels + k0, count = min(kJoinChannels, p.group_channels - k0);
    channel_sums(p, sample, c0, count, joined);
    if (threadIdx.x < count) {
      joined[threadIdx.x].y *= rstd;  // of du (x - mean) to du xhat
      p.channel[static_cast<long long>(sample) * p.l.channels + c0 + threadIdx.x] =
          joined[threadIdx.x];
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int k = 0; k < count; ++k) {
        const double w = p.weight ? to_float(static_cast<const T*>(p.weight)[c0 + k]) : 1.0;
        m1 += w * joined[k].x;
        m2 += w * joined[k].y;
      }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double n = static_cast<double>(p.l.span / p.l.channels) * p.group_channels;
    p.moments[blockIdx.x] = make_float2(static_cast<float>(m1 / n), static_cast<float>(m2 / n));
  }
}

// dw and db: the samples' channel sums added in order.
template <class T>
__global__ void norm_parameters_kernel(const NormParams p, T* dweight, T* dbias) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= p.l.channels) return;
  double a = 0.0, b = 0.0;
  for (int s = 0; s < p.samples; ++s) {
    const double2 v = p.channel[static_cast<long long>(s) * p.l.channels + c];
    a += v.x;
    b += v.y;
  }
  if (dbias) dbias[c] = from_float<T>(static_cast<float>(a));
  if (dweight) dweight[c] = from_float<T>(static_cast<float>(b));
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads, 3) norm_backward_apply_kernel(const NormParams p) {
  using Values = Vec<T, V>;
  const Layout& l = p.l;
  const Place at = place<V>(l);
  if (!at.count && !at.left) return;
  const long long end = at.sample * l.span + at.first + at.count * at.stride;
  const T* from = static_cast<const T*>(p.x) + end;
  const T* grad = static_cast<const T*>(p.dy) + end;
  T* to = static_cast<T*>(p.out) + end;
  Channels<T, V, true> ch;
  ch.load(p, at);
  const auto result = [&](const Values& v, const Values& g) {
    const Pairs<V> d = widen_pairs<T, V>(v) + ch.minus;
    const Pairs<V> du = slope<ACT, V>(fma(d, ch.scale, ch.bias)) * widen_pairs<T, V>(g);
    return round_pairs<T, V>(fma(du, ch.scale, fma(d, ch.k2, ch.k1)));
  };
  if (at.left)
    store_part<T, V>(to, result(load_part<T, V>(from, at.left), load_part<T, V>(grad, at.left)),
                     at.left);
  constexpr int U = 2;
  int i = at.count;
  for (; i >= U; i -= U) {
    Values v[U], g[U];
    from -= U * at.stride;
    grad -= U * at.stride;
    to -= U * at.stride;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = load_last(reinterpret_cast<const Values*>(from + u * at.stride));
      g[u] = load_last(reinterpret_cast<const Values*>(grad + u * at.stride));
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      store_streaming(reinterpret_cast<Values*>(to + u * at.stride), result(v[u], g[u]));
  }
  for (; i > 0; --i) {
    from -= at.stride;
    grad -= at.stride;
    to -= at.stride;
    store_streaming(reinterpret_cast<Values*>(to),
                    result(load_last(reinterpret_cast<const Values*>(from)),
                           load_last(reinterpret_cast<const Values*>(grad))));
  }
}

// ---- host ------------------------------------------------------------------

// Values per vector: 16 bytes' worth, halved until every sample starts on a
// vector (the tensors' bases are 16-byte aligned; one sample alone may end
// inside its last vector).
int vector_width(int value_bytes, int samples, long long span) {
  int v = 16 / value_bytes;
  while (v > 1 && samples > 1 && span % v) v /= 2;
  return v;
}

Layout make_layout(int samples, long long positions, int channels, int v, int per_sm) {
  Layout l;
  l.span = positions * channels;
  l.channels = channels;
  l.period = channels / std::gcd(channels, v);
  if (l.period <= kMaxThreads) {
    l.threads = l.period * std::max(1, kMaxThreads / l.period);
    l.columns = 1;
    l.step = l.threads;
  } else {
    l.threads = kMaxThreads;
    l.columns = (l.period + kMaxThreads - 1) / kMaxThreads;
    l.step = l.period;
  }
  const long long vectors = (l.span + v - 1) / v;
  l.steps = static_cast<int>((vectors + l.step - 1) / l.step);
  const long long wanted =
      std::max(1LL, static_cast<long long>(host::sm_count()) * per_sm /
                        (static_cast<long long>(samples) * l.columns));
  // at least four steps to a block, so that its loads overlap
  const long long most = std::max(1, (l.steps + 3) / 4);
  l.per_block = static_cast<int>((l.steps + std::min(wanted, most) - 1) / std::min(wanted, most));
  l.blocks = (l.steps + l.per_block - 1) / l.per_block;
  return l;
}

// As many as the kernels' registers let share an SM.
constexpr int kForwardBlocksPerSm = 4, kBackwardBlocksPerSm = 3;

template <int V, class F>
int with_width(int v, F f) {
  if constexpr (V > 1) {
    if (v < V) return with_width<V / 2>(v, f);
  }
  return f(std::integral_constant<int, V>{});
}

size_t round_up(size_t n) { return (n + 15) / 16 * 16; }

size_t partial_bytes(int samples, const Layout& l) {
  return round_up(static_cast<size_t>(samples) * l.blocks * l.columns * l.channels *
                  sizeof(float2));
}

int check_norm(int dtype, int samples, long long positions, int channels, int groups,
               int activation) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "feature_norm: dtype");
  if (activation < 0 || activation > 4)
    return host::fail(kInvalidArgument, "feature_norm: activation");
  if (samples < 1 || positions < 1 || channels < 1)
    return host::fail(kInvalidArgument, "feature_norm: sizes");
  if (groups < 1 || channels % groups)
    return host::fail(kInvalidArgument, "feature_norm: groups must divide channels");
  // a thread's step count and the grid are 32-bit
  if (positions > (1LL << 31) - 1 || positions * channels > (1LL << 40) ||
      static_cast<long long>(samples) * channels > (1LL << 30))
    return host::fail(kTooLarge, "feature_norm: too many positions or samples");
  return kOk;
}

int bytes_of(int dtype) { return dtype == kF32 ? 4 : 2; }

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

size_t splat_feature_norm_workspace_bytes(int dtype, int samples, long long positions,
                                          int channels, int groups, int backward) {
  if (check_norm(dtype, samples, positions, channels, groups, 0) != kOk) return 0;
  const int v = vector_width(bytes_of(dtype), samples, positions * channels);
  const Layout l = make_layout(samples, positions, channels, v, backward ? kBackwardBlocksPerSm : kForwardBlocksPerSm);
  size_t bytes = partial_bytes(samples, l);
  if (backward)
    bytes += round_up(static_cast<size_t>(samples) * groups * sizeof(float2)) +
             static_cast<size_t>(samples) * channels * sizeof(double2);
  return bytes;
}

int splat_feature_norm(int dtype, int samples, long long positions, int channels, int groups,
                       const void* x, const void* weight, const void* bias, float eps,
                       int activation, void* y, float* mean, float* rstd, void* workspace,
                       size_t workspace_bytes, void* stream) {
  const int bad = check_norm(dtype, samples, positions, channels, groups, activation);
  if (bad != kOk) return bad;
  if (!x || !y || !mean || !rstd || !workspace)
    return host::fail(kInvalidArgument, "feature_norm: null pointer");
  if (!host::aligned(x, 16) || !host::aligned(y, 16) || !host::aligned(workspace, 16))
    return host::fail(kInvalidArgument, "feature_norm: x, y and workspace must be 16-byte aligned");
  if (workspace_bytes <
      splat_feature_norm_workspace_bytes(dtype, samples, positions, channels, groups, 0))
    return host::fail(kWorkspaceTooSmall, "feature_norm: workspace");
  const int v = vector_width(bytes_of(dtype), samples, positions * channels);
  NormParams p{};
  p.l = make_layout(samples, positions, channels, v, kForwardBlocksPerSm);
  p.samples = samples;
  p.groups = groups;
  p.group_channels = channels / groups;
  p.x = x;
  p.weight = weight;
  p.bias = bias;
  p.out = y;
  p.mean = mean;
  p.rstd = rstd;
  p.partial = static_cast<float2*>(workspace);
  p.eps = eps;
  auto s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(samples) * p.l.blocks * p.l.columns;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return with_width<16 / sizeof(T)>(v, [&](auto width) {
      constexpr int V = decltype(width)::value;
      norm_sums_kernel<T, V><<<grid, p.l.threads, 0, host::counted(s)>>>(p);
      norm_join_kernel<T><<<samples * groups, kJoinThreads, 0, host::counted(s)>>>(p);
      return SPLAT_FEATURE_ACT(activation, [&] {
        norm_apply_kernel<T, V, ACT><<<grid, p.l.threads, 0, host::counted(s)>>>(p);
        return host::check_launch("feature_norm");
      });
    });
  });
}

int splat_feature_norm_backward(int dtype, int samples, long long positions, int channels,
                                int groups, const void* x, const void* weight, const void* bias,
                                const float* mean, const float* rstd, int activation,
                                const void* dy, void* dx, void* dweight, void* dbias,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_norm(dtype, samples, positions, channels, groups, activation);
  if (bad != kOk) return bad;
  if (!x || !dy || !mean || !rstd || !workspace)
    return host::fail(kInvalidArgument, "feature_norm_backward: null pointer");
  if (!host::aligned(x, 16) || !host::aligned(dy, 16) || !host::aligned(dx, 16) ||
      !host::aligned(workspace, 16))
    return host::fail(kInvalidArgument,
                      "feature_norm_backward: tensors and workspace must be 16-byte aligned");
  if (workspace_bytes <
      splat_feature_norm_workspace_bytes(dtype, samples, positions, channels, groups, 1))
    return host::fail(kWorkspaceTooSmall, "feature_norm_backward: workspace");
  const int v = vector_width(bytes_of(dtype), samples, positions * channels);
  NormParams p{};
  p.l = make_layout(samples, positions, channels, v, kBackwardBlocksPerSm);
  p.samples = samples;
  p.groups = groups;
  p.group_channels = channels / groups;
  p.x = x;
  p.dy = dy;
  p.weight = weight;
  p.bias = bias;
  p.out = dx;
  p.mean = const_cast<float*>(mean);
  p.rstd = const_cast<float*>(rstd);
  char* at = static_cast<char*>(workspace);
  p.partial = reinterpret_cast<float2*>(at);
  at += partial_bytes(samples, p.l);
  p.moments = reinterpret_cast<float2*>(at);
  at += round_up(static_cast<size_t>(samples) * groups * sizeof(float2));
  p.channel = reinterpret_cast<double2*>(at);
  auto s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(samples) * p.l.blocks * p.l.columns;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return with_width<16 / sizeof(T)>(v, [&](auto width) {
      constexpr int V = decltype(width)::value;
      return SPLAT_FEATURE_ACT(activation, [&] {
        norm_backward_sums_kernel<T, V, ACT><<<grid, p.l.threads, 0, host::counted(s)>>>(p);
        norm_backward_join_kernel<T>
            <<<samples * groups, kJoinThreads, 0, host::counted(s)>>>(p);
        if (dweight || dbias)
          norm_parameters_kernel<T>
              <<<host::blocks_for(channels, 128), 128, 0, host::counted(s)>>>(
                  p, static_cast<T*>(dweight), static_cast<T*>(dbias));
        if (dx)
          norm_backward_apply_kernel<T, V, ACT><<<grid, p.l.threads, 0, host::counted(s)>>>(p);
        return host::check_launch("feature_norm_backward");
      });
    });
  });
}

}  // extern "C"
