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

template <class T, int V>
SPLAT_DEV void load_values(const T* base, long long at, long long span, float (&v)[V], float fill) {
  if (at + V <= span) {
    const Vec<T, V> r = *reinterpret_cast<const Vec<T, V>*>(base + at);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_float(r.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = at + j < span ? to_float(base[at + j]) : fill;
  }
}

template <class T, int V>
SPLAT_DEV void store_values(T* base, long long at, long long span, const float (&v)[V]) {
  if (at + V <= span) {
    Vec<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = from_float<T>(v[j]);
    *reinterpret_cast<Vec<T, V>*>(base + at) = r;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (at + j < span) base[at + j] = from_float<T>(v[j]);
  }
}

// What a thread of any of the passes works on.
struct Place {
  int sample, part, column;  // part: the block along the sample's rows
  int vector;                // of the period(s) at a step
  bool active;
};

SPLAT_DEV Place place(const Layout& l) {
  Place p;
  long long b = blockIdx.x;
  p.column = static_cast<int>(b % l.columns);
  b /= l.columns;
  p.part = static_cast<int>(b % l.blocks);
  p.sample = static_cast<int>(b / l.blocks);
  p.vector = p.column * l.threads + threadIdx.x;
  p.active = p.vector < l.step;
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
__global__ void __launch_bounds__(kMaxThreads) norm_sums_kernel(const NormParams p) {
  const Layout& l = p.l;
  const Place at = place(l);
  const T* x = static_cast<const T*>(p.x) + at.sample * l.span;
  float s1[V] = {}, s2[V] = {};
  if (at.active) {
    float pivot[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      pivot[j] = to_float(x[(static_cast<long long>(at.vector) * V + j) % l.channels]);
    const int begin = at.part * l.per_block, end = min(begin + l.per_block, l.steps);
#pragma unroll 4
    for (int i = begin; i < end; ++i) {
      const long long o = (static_cast<long long>(i) * l.step + at.vector) * V;
      if (o + V <= l.span) {
        float v[V];
        load_values<T, V>(x, o, l.span, v, 0.0f);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = v[j] - pivot[j];
          s1[j] += d;
          s2[j] += d * d;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (o + j < l.span) {
            const float d = to_float(x[o + j]) - pivot[j];
            s1[j] += d;
            s2[j] += d * d;
          }
      }
    }
  }
  write_partial<V>(p, at, s1, s2);
}

SPLAT_DEV double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Joins the blocks' sums of one channel (a warp per call).
SPLAT_DEV double2 channel_sums(const NormParams& p, int sample, int c) {
  const int parts = p.l.blocks * p.l.columns;
  const float2* in = p.partial + static_cast<long long>(sample) * parts * p.l.channels + c;
  double a = 0.0, b = 0.0;
  for (int i = threadIdx.x & 31; i < parts; i += 32) {
    const float2 v = in[static_cast<long long>(i) * p.l.channels];
    a += v.x;
    b += v.y;
  }
  return make_double2(warp_sum(a), warp_sum(b));
}

constexpr int kJoinWarps = 8;

// Mean and reciprocal deviation of one group: each channel's (count, mean,
// sum of squared deviations) joined pairwise, in doubles:
//   M = M_a + M_b + (mean_b - mean_a)^2 n_a n_b / (n_a + n_b).
template <class T>
__global__ void __launch_bounds__(kJoinWarps * 32) norm_join_kernel(const NormParams p) {
  const int sample = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
  const int warp = threadIdx.x >> 5;
  const double rows = static_cast<double>(p.l.span / p.l.channels);
  const T* x = static_cast<const T*>(p.x) + sample * p.l.span;
  double n = 0.0, mean = 0.0, m2 = 0.0;
  for (int k = warp; k < p.group_channels; k += kJoinWarps) {
    const int c = g * p.group_channels + k;
    const double2 s = channel_sums(p, sample, c);
    const double channel_mean = s.x / rows + static_cast<double>(to_float(x[c]));
    const double channel_m2 = s.y - s.x * s.x / rows;
    const double d = channel_mean - mean, total = n + rows;
    m2 += channel_m2 + d * d * n * rows / total;
    mean += d * rows / total;
    n = total;
  }
  __shared__ double joined[kJoinWarps][3];
  if ((threadIdx.x & 31) == 0) {
    joined[warp][0] = n;
    joined[warp][1] = mean;
    joined[warp][2] = m2;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    n = joined[0][0], mean = joined[0][1], m2 = joined[0][2];
    for (int w = 1; w < kJoinWarps; ++w) {
      const double nb = joined[w][0];
      if (nb == 0.0) continue;
      const double d = joined[w][1] - mean, total = n + nb;
      m2 += joined[w][2] + d * d * n * nb / total;
      mean += d * nb / total;
      n = total;
    }
    // rounding can leave a constant group a hair below zero; NaN stays
    const double var = m2 < 0.0 ? 0.0 : m2 / n;
    p.mean[blockIdx.x] = static_cast<float>(mean);
    p.rstd[blockIdx.x] = static_cast<float>(1.0 / sqrt(var + static_cast<double>(p.eps)));
  }
}

// The parameters of a thread's V channels.
template <class T, int V>
struct Channels {
  float mean[V], rstd[V], weight[V], bias[V];
  SPLAT_DEV void load(const NormParams& p, const Place& at) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = static_cast<int>((static_cast<long long>(at.vector) * V + j) % p.l.channels);
      const int g = at.sample * p.groups + c / p.group_channels;
      mean[j] = p.mean[g];
      rstd[j] = p.rstd[g];
      weight[j] = p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0f;
      bias[j] = p.bias ? to_float(static_cast<const T*>(p.bias)[c]) : 0.0f;
    }
  }
};

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads) norm_apply_kernel(const NormParams p) {
  const Layout& l = p.l;
  const Place at = place(l);
  if (!at.active) return;
  const T* x = static_cast<const T*>(p.x) + at.sample * l.span;
  T* y = static_cast<T*>(p.out) + at.sample * l.span;
  Channels<T, V> ch;
  ch.load(p, at);
  const int begin = at.part * l.per_block, end = min(begin + l.per_block, l.steps);
#pragma unroll 4
  for (int i = begin; i < end; ++i) {
    const long long o = (static_cast<long long>(i) * l.step + at.vector) * V;
    if (o >= l.span) break;
    float v[V];
    load_values<T, V>(x, o, l.span, v, 0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j)
      v[j] = activate<ACT>((v[j] - ch.mean[j]) * ch.rstd[j] * ch.weight[j] + ch.bias[j]);
    store_values<T, V>(y, o, l.span, v);
  }
}

// Sums of du and du xhat per channel.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads) norm_backward_sums_kernel(const NormParams p) {
  const Layout& l = p.l;
  const Place at = place(l);
  float s1[V] = {}, s2[V] = {};
  if (at.active) {
    const T* x = static_cast<const T*>(p.x) + at.sample * l.span;
    const T* dy = static_cast<const T*>(p.dy) + at.sample * l.span;
    Channels<T, V> ch;
    ch.load(p, at);
    const int begin = at.part * l.per_block, end = min(begin + l.per_block, l.steps);
#pragma unroll 2
    for (int i = begin; i < end; ++i) {
      const long long o = (static_cast<long long>(i) * l.step + at.vector) * V;
      if (o >= l.span) break;
      float v[V], d[V];
      load_values<T, V>(x, o, l.span, v, 0.0f);
      load_values<T, V>(dy, o, l.span, d, 0.0f);  // 0 past the end: adds nothing
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float hat = (v[j] - ch.mean[j]) * ch.rstd[j];
        const float du = d[j] * slope<ACT>(hat * ch.weight[j] + ch.bias[j]);
        s1[j] += o + j < l.span ? du : 0.0f;
        s2[j] += o + j < l.span ? du * hat : 0.0f;
      }
    }
  }
  write_partial<V>(p, at, s1, s2);
}

template <class T>
__global__ void __launch_bounds__(kJoinWarps * 32) norm_backward_join_kernel(const NormParams p) {
  const int sample = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
  const int warp = threadIdx.x >> 5;
  double m1 = 0.0, m2 = 0.0;
  for (int k = warp; k < p.group_channels; k += kJoinWarps) {
    const int c = g * p.group_channels + k;
    const double2 s = channel_sums(p, sample, c);
    const double w = p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0;
    m1 += w * s.x;
    m2 += w * s.y;
    if ((threadIdx.x & 31) == 0)
      p.channel[static_cast<long long>(sample) * p.l.channels + c] = s;
  }
  __shared__ double joined[kJoinWarps][2];
  if ((threadIdx.x & 31) == 0) {
    joined[warp][0] = m1;
    joined[warp][1] = m2;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    m1 = m2 = 0.0;
    for (int w = 0; w < kJoinWarps; ++w) {
      m1 += joined[w][0];
      m2 += joined[w][1];
    }
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
__global__ void __launch_bounds__(kMaxThreads) norm_backward_apply_kernel(const NormParams p) {
  const Layout& l = p.l;
  const Place at = place(l);
  if (!at.active) return;
  const T* x = static_cast<const T*>(p.x) + at.sample * l.span;
  const T* dy = static_cast<const T*>(p.dy) + at.sample * l.span;
  T* dx = static_cast<T*>(p.out) + at.sample * l.span;
  Channels<T, V> ch;
  ch.load(p, at);
  float m1[V], m2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = static_cast<int>((static_cast<long long>(at.vector) * V + j) % l.channels);
    const float2 m = p.moments[at.sample * p.groups + c / p.group_channels];
    m1[j] = m.x;
    m2[j] = m.y;
  }
  const int begin = at.part * l.per_block, end = min(begin + l.per_block, l.steps);
#pragma unroll 2
  for (int i = begin; i < end; ++i) {
    const long long o = (static_cast<long long>(i) * l.step + at.vector) * V;
    if (o >= l.span) break;
    float v[V], d[V];
    load_values<T, V>(x, o, l.span, v, 0.0f);
    load_values<T, V>(dy, o, l.span, d, 0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float hat = (v[j] - ch.mean[j]) * ch.rstd[j];
      const float du = d[j] * slope<ACT>(hat * ch.weight[j] + ch.bias[j]);
      v[j] = ch.rstd[j] * (ch.weight[j] * du - m1[j] - hat * m2[j]);
    }
    store_values<T, V>(dx, o, l.span, v);
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

constexpr int kBlocksPerSm = 6;

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
  const Layout l = make_layout(samples, positions, channels, v, kBlocksPerSm);
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
  p.l = make_layout(samples, positions, channels, v, kBlocksPerSm);
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
      norm_join_kernel<T><<<samples * groups, kJoinWarps * 32, 0, host::counted(s)>>>(p);
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
  p.l = make_layout(samples, positions, channels, v, kBlocksPerSm);
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
            <<<samples * groups, kJoinWarps * 32, 0, host::counted(s)>>>(p);
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
