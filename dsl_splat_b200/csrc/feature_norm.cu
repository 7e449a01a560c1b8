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
// the result; small samples take one launch for all of it.  Sums over channels of a group are taken after the sums over
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

constexpr int kMaxThreads = 512;

struct NormParams {
  Layout l;
  int samples, groups, group_channels;
  int keep;  // small samples: the values stay in shared memory, or are read again
  const void* x;
  const void* dy;
  const void* weight;  // (C) or NULL: 1
  const void* bias;    // (C) or NULL: 0
  void* out;           // y or dx
  float* mean;         // (B, G)
  float* rstd;
  // (B, blocks * columns, C): double2 of the forward, float2 of the backward
  void* partial;
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
template <int ACT, bool FINE, int V>
SPLAT_DEV Pairs<V> activate(Pairs<V> x) {
#pragma unroll
  for (int i = 0; i < Pairs<V>::N; ++i) {
    float a, b;
    unpack2(x.v[i], a, b);
    if constexpr (V == 1) b = a;
    activate2<ACT, FINE>(a, b);
    x.v[i] = pack2(a, b);
  }
  return x;
}
template <int ACT, bool FINE, int V>
SPLAT_DEV Pairs<V> slope(Pairs<V> x) {
#pragma unroll
  for (int i = 0; i < Pairs<V>::N; ++i) {
    float a, b;
    unpack2(x.v[i], a, b);
    if constexpr (V == 1) b = a;
    slope2<ACT, FINE>(a, b);
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
  // a cluster's last blocks may have no steps
  const int begin = min(p.part * l.per_block, l.steps);
  const int end = min(begin + l.per_block, l.steps);
  p.first = (static_cast<long long>(begin) * l.step + p.vector) * V;
  p.stride = static_cast<long long>(l.step) * V;
  p.count = p.left = 0;
  if (p.vector < l.step && begin < end) {
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
  float2* out = static_cast<float2*>(p.partial) +
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

// A thread's sums of x - pivot and its square per channel.  The pivot is the
// thread's first value and moves to the mean of those so far after every
// fourfold of the first few, so that the sums of squares never exceed a few
// times the squared deviations that they hold, whichever values come first.  (A
// pivot for the whole sample cancels where it is unlike the rest: the sample's
// first row, 300 deviations away, cost the variance of 1600 x 1200 positions
// 1e-3 of itself.)
template <class T, int V>
struct Deviations {
  Pairs<V> minus, s1, s2;  // minus: -pivot
  SPLAT_DEV void start(const T* first, int valid) {
    float zero[V] = {}, pivot[V];
#pragma unroll
    for (int j = 0; j < V; ++j) pivot[j] = j < valid ? -to_float(first[j]) : 0.0f;
    minus.set(pivot);
    s1.set(zero);
    s2.set(zero);
  }
  SPLAT_DEV void add(const Vec<T, V>& v) {
    const Pairs<V> d = widen_pairs<T, V>(v) + minus;
    s1 = s1 + d;
    s2 = fma(d, d, s2);
  }
  // Sums of squares that have overflowed stay infinite.
  static SPLAT_DEV float less(float a, float b) {
    return a == __int_as_float(0x7f800000) ? a : a - b;
  }
  SPLAT_DEV void move(int count) {
    float m[V], a[V], b[V];
    minus.get(m);
    s1.get(a);
    s2.get(b);
    const float n = static_cast<float>(count), inverse = 1.0f / n;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float to = m[j] - a[j] * inverse, by = m[j] - to, rest = a[j] - n * by;
      b[j] = less(b[j], by * (a[j] + rest));
      a[j] = rest;
      m[j] = to;
    }
    minus.set(m);
    s1.set(a);
    s2.set(b);
  }
  // (mean - x0, sum of squared deviations) of count values and, in the channels
  // below `left`, of a last one; x0(j): the sample's first row.
  template <class F>
  SPLAT_DEV void finish(int count, const T* last, int left, F x0, float2 (&r)[V]) const {
    float m[V], a[V], b[V];
    minus.get(m);
    s1.get(a);
    s2.get(b);
    const float more = 1.0f / static_cast<float>(count + 1);
    const float inverse = count ? 1.0f / static_cast<float>(count) : 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (j < left) {
        const float d = to_float(last[j]) + m[j];
        a[j] += d;
        b[j] += d * d;
      } else if (count == 0) {
        r[j] = make_float2(0.0f, 0.0f);
        continue;
      }
      const float mean = a[j] * (j < left ? more : inverse), rest = less(b[j], a[j] * mean);
      r[j] = make_float2((-m[j] - x0(j)) + mean, rest < 0.0f ? 0.0f : rest);
    }
  }
};

// Joins the block's threads: for every channel their (mean - x0, sum of squared
// deviations) in `slots`, of `count` flat positions of a step from `first` on, to
// the sums of x - x0 and its square.  The squared deviations are the threads' and
// those of their means from the block's, so nothing cancels in fp32.  Whole warps
// work, up to 32 threads to a channel, in a fixed order.
template <int V, class F>
SPLAT_DEV void join_threads(const Layout& l, int part, int first, int count, const float2* slots,
                            F write) {
  const int begin = min(part * l.per_block, l.steps), end = min(begin + l.per_block, l.steps);
  const int steps = end - begin, whole = l.threads & ~31;
  // positions from `cut` on are one value short: the sample ends before them
  const long long cut =
      steps && end == l.steps ? l.span - (l.steps - 1LL) * l.step * V - first : count;
  int lanes = 32;
  while (lanes > 1 && l.channels * lanes > whole) lanes /= 2;
  const int lane = threadIdx.x & (lanes - 1), groups = whole / lanes;
  if (static_cast<int>(threadIdx.x) >= whole) return;
  const auto sum = [&](auto v) {
    for (int o = lanes / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  for (int c0 = 0; c0 < l.channels; c0 += groups) {
    const int c = c0 + static_cast<int>(threadIdx.x) / lanes;
    int from = c - first % l.channels;
    if (from < 0) from += l.channels;
    from = c < l.channels ? from + lane * l.channels : count;
    const int by = lanes * l.channels;
    int n = 0;
    float a = 0.0f;
    for (int i = from; i < count; i += by) {
      const int ni = steps - (i >= cut ? 1 : 0);
      n += ni;
      a += static_cast<float>(ni) * slots[i].x;
    }
    n = sum(n);
    a = sum(a);
    const float mean = n ? a / static_cast<float>(n) : 0.0f;
    float b = 0.0f;
    for (int i = from; i < count; i += by) {
      const float apart = slots[i].x - mean;
      b += slots[i].y + static_cast<float>(steps - (i >= cut ? 1 : 0)) * (apart * apart);
    }
    b = sum(b);
    if (lane == 0 && c < l.channels) {
      const double m = mean;
      write(c, n * m, b + n * m * m);
    }
  }
}

template <class T, int V>
__global__ void __launch_bounds__(kMaxThreads, 2) norm_sums_kernel(const NormParams p) {
  using Values = Vec<T, V>;
  __shared__ float2 slots[kMaxThreads * V];
  const Layout& l = p.l;
  const Place at = place<V>(l);
  const T* x = static_cast<const T*>(p.x) + at.sample * l.span;
  const T* from = x + at.first;
  Deviations<T, V> sums;
  sums.start(from, at.count ? V : at.left);
  constexpr int U = 4;
  int i = 0, move = U;
  for (; i + U <= at.count; i += U) {
    Values v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = *reinterpret_cast<const Values*>(from + u * at.stride);
    from += U * at.stride;
#pragma unroll
    for (int u = 0; u < U; ++u) sums.add(v[u]);
    if (i + U == move) {
      sums.move(move);
      move = move < 1 << 28 ? move * 4 : 0;
    }
  }
  for (; i < at.count; ++i, from += at.stride)
    sums.add(*reinterpret_cast<const Values*>(from));
  float2 r[V];
  sums.finish(at.count, from, at.left, [&](int j) {
    return to_float(x[(static_cast<long long>(at.vector) * V + j) % l.channels]);
  }, r);
#pragma unroll
  for (int j = 0; j < V; ++j) slots[threadIdx.x * V + j] = r[j];
  __syncthreads();
  const int first = at.column * l.threads * V;  // flat position of slots[0] in a step
  const long long block = (static_cast<long long>(at.sample) * l.blocks + at.part) * l.columns;
  double2* out = static_cast<double2*>(p.partial) + (block + at.column) * l.channels;
  join_threads<V>(l, at.part, first, min(l.threads, l.step - at.column * l.threads) * V, slots,
                  [&](int c, double a, double b) { out[c] = make_double2(a, b); });
}

SPLAT_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
SPLAT_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// A value in the shared memory of another block of the cluster, at the address
// that it has in this one.
SPLAT_DEV double load_cluster(const double* own, uint32_t rank) {
  const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  uint32_t there;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(there) : "memory");
  return v;
}
SPLAT_DEV double2 load_cluster(const double2* own, uint32_t rank) {
  return make_double2(load_cluster(&own->x, rank), load_cluster(&own->y, rank));
}
SPLAT_DEV float2 load_cluster(const float2* own, uint32_t rank) {
  const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  uint32_t there;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(there)
               : "memory");
  return v;
}

SPLAT_DEV double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The blocks' sums of up to kJoinChannels channels from c0 on, joined in
// shared memory: neighbouring threads read neighbouring channels of a block's
// row, and the threads of a channel are added up in a fixed order.
constexpr int kJoinThreads = 1024, kJoinChannels = 32, kMaxCluster = 8;

template <class Pair>  // double2 or float2
SPLAT_DEV void channel_sums(const NormParams& p, int sample, int c0, int count,
                            double2 (&joined)[kJoinChannels]) {
  __shared__ double2 sums[kJoinThreads];
  const int parts = p.l.blocks * p.l.columns;
  const Pair* in = static_cast<const Pair*>(p.partial) +
                   static_cast<long long>(sample) * parts * p.l.channels + c0;
  const int lanes = kJoinThreads / count, c = threadIdx.x % count, lane = threadIdx.x / count;
  double a = 0.0, b = 0.0;
  if (lane < lanes) {
    constexpr int U = 8;  // reads in flight
    for (int i0 = lane; i0 < parts; i0 += U * lanes) {
      Pair v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * lanes;
        v[u] = i < parts ? in[static_cast<long long>(i) * p.l.channels + c] : Pair{};
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a += v[u].x;
        b += v[u].y;
      }
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

// A group's moments from its channels' sums of x - x0 (x0: the sample's first
// row), in doubles, where an x0 far from the rest costs nothing: (count, mean, sum of
// squared deviations) of up to 32 channels at a time, a lane to a channel, and
// such blocks joined by
//   M = M_a + M_b + (mean_b - mean_a)^2 n_a n_b / (n_a + n_b).
struct Moments {
  double n, mean, m2;
  // Called by a whole warp; the pivot (x0) and sums of lanes from `count` on are ignored.
  SPLAT_DEV void join(double rows, int count, double2 sums, double pivot) {
    const bool in = (threadIdx.x & 31) < count;
    const double inverse = 1.0 / rows;
    const double channel_mean = in ? sums.x * inverse + pivot : 0.0;
    const double block_mean = warp_sum(channel_mean) / count, d = channel_mean - block_mean;
    const double block_m2 =
        warp_sum(in ? sums.y - sums.x * sums.x * inverse + rows * d * d : 0.0);
    add(rows * count, block_mean, block_m2);
  }
  SPLAT_DEV void add(double nb, double mean_b, double m2_b) {
    if (nb == 0.0) return;
    const double total = n + nb, apart = mean_b - mean;
    m2 += m2_b + apart * apart * (n * nb / total);
    mean += apart * (nb / total);
    n = total;
  }
  SPLAT_DEV void finish(float eps, float* mean_to, float* rstd_to) const {
    // rounding can leave a constant group a hair below zero; NaN stays
    const double var = m2 < 0.0 ? 0.0 : m2 / n;
    *mean_to = static_cast<float>(mean);
    *rstd_to = static_cast<float>(1.0 / sqrt(var + static_cast<double>(eps)));
  }
};

// A cluster to a group, its blocks take 32 channels at a time in turn.
template <class T>
__global__ void __launch_bounds__(kJoinThreads) norm_join_kernel(const NormParams p, int blocks) {
  __shared__ double2 joined[kJoinChannels];
  __shared__ double mine[3];
  const int group = blockIdx.x / blocks, rank = blockIdx.x - group * blocks;
  const int sample = group / p.groups, g = group - sample * p.groups;
  const double rows = static_cast<double>(p.l.span / p.l.channels);
  const T* x = static_cast<const T*>(p.x) + sample * p.l.span;
  Moments m{};
  for (int k0 = rank * kJoinChannels; k0 < p.group_channels; k0 += blocks * kJoinChannels) {
    const int c0 = g * p.group_channels + k0, count = min(kJoinChannels, p.group_channels - k0);
    channel_sums<double2>(p, sample, c0, count, joined);
    if (threadIdx.x < 32) {
      const int k = min(static_cast<int>(threadIdx.x), count - 1);
      m.join(rows, count, joined[k], to_float(x[c0 + k]));
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) mine[0] = m.n, mine[1] = m.mean, mine[2] = m.m2;
  cluster_sync();
  if (rank == 0 && threadIdx.x == 0) {
    for (int r = 1; r < blocks; ++r) m.add(load_cluster(mine, r), load_cluster(mine + 1, r),
                                           load_cluster(mine + 2, r));
    m.finish(p.eps, p.mean + group, p.rstd + group);
  }
  cluster_sync();  // no block leaves while its sums are read
}

// The parameters of a thread's V channels: -mean, rstd w, b, and for the
// backward -rstd m1 and -rstd^2 m2, so that with d = x - mean
//   u = d (rstd w) + b,  dx = du (rstd w) - d rstd^2 m2 - rstd m1.
template <class T, int V, bool BACKWARD>
struct Channels {
  Pairs<V> minus, scale, bias, k1, k2;
  // moments: the sample's (mean, rstd) per group where they are not in p's
  // arrays yet; sums: its (m1, m2) likewise
  SPLAT_DEV void load(const NormParams& p, const Place& at, const float2* moments = nullptr,
                      const float2* sums = nullptr) {
    float m[V], s[V], b[V], x1[V], x2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = static_cast<int>((static_cast<long long>(at.vector) * V + j) % p.l.channels);
      const int own = c / p.group_channels, g = at.sample * p.groups + own;
      const float rstd = moments ? moments[own].y : p.rstd[g];
      m[j] = -(moments ? moments[own].x : p.mean[g]);
      s[j] = rstd * (p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0f);
      b[j] = p.bias ? to_float(static_cast<const T*>(p.bias)[c]) : 0.0f;
      if constexpr (BACKWARD) {
        const float2 s12 = sums ? sums[own] : p.moments[g];
        x1[j] = -rstd * s12.x;
        x2[j] = -rstd * rstd * s12.y;
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
__global__ void __launch_bounds__(kMaxThreads, 2) norm_apply_kernel(const NormParams p) {
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
        activate<ACT, sizeof(T) == 4, V>(fma(widen_pairs<T, V>(v) + ch.minus, ch.scale, ch.bias)));
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
__global__ void __launch_bounds__(kMaxThreads, 1) norm_backward_sums_kernel(const NormParams p) {
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
      const Pairs<V> du =
          slope<ACT, sizeof(T) == 4, V>(fma(d, ch.scale, ch.bias)) * widen_pairs<T, V>(g);
      s1 = s1 + du;
      s2 = fma(du, d, s2);
    };
    constexpr int U = 4;
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
__global__ void __launch_bounds__(kJoinThreads)
    norm_backward_join_kernel(const NormParams p, int blocks, T* dweight, T* dbias) {
  __shared__ double2 joined[kJoinChannels];
  __shared__ double mine[2];
  const int group = blockIdx.x / blocks, rank = blockIdx.x - group * blocks;
  const int sample = group / p.groups, g = group - sample * p.groups;
  const double rstd = p.rstd[group];
  double m1 = 0.0, m2 = 0.0;
  for (int k0 = rank * kJoinChannels; k0 < p.group_channels; k0 += blocks * kJoinChannels) {
    const int c0 = g * p.group_channels + k0, count = min(kJoinChannels, p.group_channels - k0);
    channel_sums<float2>(p, sample, c0, count, joined);
    if (threadIdx.x < 32) {
      const int k = threadIdx.x;
      double2 v = joined[min(k, count - 1)];
      v.y *= rstd;  // of du (x - mean) to du xhat
      if (k < count) {
        if (p.samples > 1) p.channel[static_cast<long long>(sample) * p.l.channels + c0 + k] = v;
        if (dbias) dbias[c0 + k] = from_float<T>(static_cast<float>(v.x));
        if (dweight) dweight[c0 + k] = from_float<T>(static_cast<float>(v.y));
      }
      const double w =
          k < count && p.weight ? to_float(static_cast<const T*>(p.weight)[c0 + k]) : 1.0;
      m1 += warp_sum(k < count ? w * v.x : 0.0);
      m2 += warp_sum(k < count ? w * v.y : 0.0);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) mine[0] = m1, mine[1] = m2;
  cluster_sync();
  if (rank == 0 && threadIdx.x == 0) {
    for (int r = 1; r < blocks; ++r) {
      m1 += load_cluster(mine, r);
      m2 += load_cluster(mine + 1, r);
    }
    const double n = static_cast<double>(p.l.span / p.l.channels) * p.group_channels;
    p.moments[group] = make_float2(static_cast<float>(m1 / n), static_cast<float>(m2 / n));
  }
  cluster_sync();  // no block leaves while its sums are read
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
__global__ void __launch_bounds__(kMaxThreads, 1) norm_backward_apply_kernel(const NormParams p) {
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
    const Pairs<V> du =
        slope<ACT, sizeof(T) == 4, V>(fma(d, ch.scale, ch.bias)) * widen_pairs<T, V>(g);
    return round_pairs<T, V>(fma(du, ch.scale, fma(d, ch.k2, ch.k1)));
  };
  if (at.left)
    store_part<T, V>(to, result(load_part<T, V>(from, at.left), load_part<T, V>(grad, at.left)),
                     at.left);
  constexpr int U = 4;
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

// ---- small samples: one launch ---------------------------------------------------
//
// One cluster of up to 8 blocks takes a sample.  Where its values fit in their
// shared memory they are read once, every thread keeping its own; larger ones
// are read again, out of the L2.  The blocks exchange
// their channel sums through distributed shared memory, and each forms the
// group's moments for itself.  One launch and no workspace: a call on
// 37x53x35 fp32 takes 15 us against 22 in passes, on 80x80x32 fp32 (819 KB) 17
// against 22.

constexpr int kSmallThreads = 512;
constexpr size_t kMostShared = 226 * 1024;
constexpr int kSmallForward = 450000, kSmallBackward = 600000;  // values of a sample
constexpr int kFewSamples = 8;
constexpr long long kManyBytes = 1792 * 1024;
constexpr int kSmallChannels = 1024;

// The cluster's sums per channel of its blocks' in `own`; all blocks end with
// them in `channel`.
template <class Pair>  // double2 or float2
SPLAT_DEV void join_cluster(const Layout& l, const Pair* own, double2* channel) {
  cluster_sync();
  for (int c = threadIdx.x; c < l.channels; c += l.threads) {
    double a = 0.0, b = 0.0;
    for (int r = 0; r < l.blocks; ++r) {
      const Pair v = load_cluster(own + c, r);
      a += v.x;
      b += v.y;
    }
    channel[c] = make_double2(a, b);
  }
  cluster_sync();  // no block leaves while its sums are read
}

// Sums the threads' sums over the block and then over the cluster.
template <int V>
SPLAT_DEV void cluster_sums(const Layout& l, const float (&s1)[V], const float (&s2)[V],
                            float2* per_thread, float2* own, double2* channel) {
#pragma unroll
  for (int j = 0; j < V; ++j) per_thread[threadIdx.x * V + j] = make_float2(s1[j], s2[j]);
  __syncthreads();
  const int count = l.threads * V;
  for (int c = threadIdx.x; c < l.channels; c += l.threads) {
    float a = 0.0f, b = 0.0f;
    for (int i = c; i < count; i += l.channels) {
      a += per_thread[i].x;
      b += per_thread[i].y;
    }
    own[c] = make_float2(a, b);
  }
  join_cluster(l, own, channel);
}

// Shared memory of the small kernels: the values, then the sums.
__host__ __device__ inline size_t kept_bytes(const Layout& l, int vector_bytes, int arrays) {
  return (static_cast<size_t>(arrays) * l.per_block * l.threads * vector_bytes + 15) / 16 * 16;
}
template <class T, int V, class Own>  // Own: double2 (forward) or float2
struct SmallShared {
  float2* per_thread;
  Own* own;
  double2* channel;
  float2* group;  // per group: mean and rstd, or m1 and m2
  SPLAT_DEV SmallShared(unsigned char* base, const Layout& l, int arrays) {
    base += kept_bytes(l, sizeof(Vec<T, V>), arrays);  // arrays: 0 when nothing is kept
    channel = reinterpret_cast<double2*>(base);
    own = reinterpret_cast<Own*>(channel + l.channels);
    per_thread = reinterpret_cast<float2*>(own + l.channels);
    group = per_thread + l.threads * V;
  }
};
size_t small_bytes(const Layout& l, int v, int value_bytes, int groups, int arrays,
                   bool backward) {
  return kept_bytes(l, v * value_bytes, arrays) +
         static_cast<size_t>(l.channels) *
             (sizeof(double2) + (backward ? sizeof(float2) : sizeof(double2))) +
         static_cast<size_t>(l.threads) * v * sizeof(float2) +
         static_cast<size_t>(groups) * sizeof(float2);
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kSmallThreads) norm_small_kernel(const NormParams p) {
  using Values = Vec<T, V>;
  extern __shared__ __align__(16) unsigned char shared[];
  const Layout& l = p.l;
  const Place at = place<V>(l);
  const SmallShared<T, V, double2> mem(shared, l, p.keep ? 1 : 0);
  Values* kept = reinterpret_cast<Values*>(shared) + threadIdx.x;
  const T* x = static_cast<const T*>(p.x) + at.sample * l.span;
  const T* from = x + at.first;
  const bool active = at.count || at.left;
  Deviations<T, V> sums;
  sums.start(from, at.count ? V : at.left);
  float x0[V];
#pragma unroll
  for (int j = 0; j < V; ++j)
    x0[j] = active ? to_float(x[(at.vector * V + j) % l.channels]) : 0.0f;
  constexpr int U = 8;  // reads in flight
  for (int i0 = 0, move = U; i0 < at.count; i0 += U) {
    Values v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < at.count)
        v[u] = *reinterpret_cast<const Values*>(from + (i0 + u) * at.stride);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < at.count) {
        if (p.keep) kept[(i0 + u) * l.threads] = v[u];
        sums.add(v[u]);
      }
    if (i0 + U == move && move <= at.count) {
      sums.move(move);
      move *= 4;
    }
  }
  if (at.left && p.keep)
    kept[at.count * l.threads] = load_part<T, V>(from + at.count * at.stride, at.left);
  float2 r[V];
  sums.finish(at.count, from + at.count * at.stride, at.left, [&](int j) { return x0[j]; }, r);
#pragma unroll
  for (int j = 0; j < V; ++j) mem.per_thread[threadIdx.x * V + j] = r[j];
  __syncthreads();
  join_threads<V>(l, at.part, 0, l.threads * V, mem.per_thread,
                  [&](int c, double s1, double s2) { mem.own[c] = make_double2(s1, s2); });
  join_cluster(l, mem.own, mem.channel);
  __syncthreads();
  const double rows = static_cast<double>(l.span / l.channels);
  // whole warps only (there is one: a block has more than 128 threads)
  const int whole = l.threads / 32, lane = threadIdx.x & 31;
  if (static_cast<int>(threadIdx.x >> 5) < whole) {
    for (int g = threadIdx.x >> 5; g < p.groups; g += whole) {
      Moments m{};
      for (int k0 = 0; k0 < p.group_channels; k0 += 32) {
        const int count = min(32, p.group_channels - k0);
        const int c = g * p.group_channels + k0 + min(lane, count - 1);
        m.join(rows, count, mem.channel[c], to_float(x[c]));
      }
      if (lane == 0) {
        float2 r;
        m.finish(p.eps, &r.x, &r.y);
        mem.group[g] = r;
        if (p.mean && cluster_rank() == 0) {
          p.mean[at.sample * p.groups + g] = r.x;
          p.rstd[at.sample * p.groups + g] = r.y;
        }
      }
    }
  }
  __syncthreads();
  if (!active) return;
  Channels<T, V, false> ch;
  ch.load(p, at, mem.group, nullptr);
  T* to = static_cast<T*>(p.out) + at.sample * l.span + at.first;
  const auto result = [&](const Values& v) {
    return round_pairs<T, V>(
        activate<ACT, sizeof(T) == 4, V>(fma(widen_pairs<T, V>(v) + ch.minus, ch.scale, ch.bias)));
  };
  for (int i0 = 0; i0 < at.count; i0 += U) {
    Values v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < at.count)
        v[u] = p.keep ? kept[(i0 + u) * l.threads]
                      : *reinterpret_cast<const Values*>(from + (i0 + u) * at.stride);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < at.count)
        *reinterpret_cast<Values*>(to + (i0 + u) * at.stride) = result(v[u]);
  }
  if (at.left)
    store_part<T, V>(to + at.count * at.stride,
                     result(p.keep ? kept[at.count * l.threads]
                                   : load_part<T, V>(from + at.count * at.stride, at.left)),
                     at.left);
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kSmallThreads)
    norm_backward_small_kernel(const NormParams p, T* dweight, T* dbias) {
  using Values = Vec<T, V>;
  extern __shared__ __align__(16) unsigned char shared[];
  const Layout& l = p.l;
  const Place at = place<V>(l);
  const SmallShared<T, V, float2> mem(shared, l, p.keep ? 2 : 0);
  Values* kept_x = reinterpret_cast<Values*>(shared) + threadIdx.x;
  Values* kept_g = kept_x + l.per_block * l.threads;
  const long long offset = at.sample * l.span + at.first;
  const T* from = static_cast<const T*>(p.x) + offset;
  const T* grad = static_cast<const T*>(p.dy) + offset;
  float a[V] = {}, b[V] = {};
  Pairs<V> s1, s2;
  s1.set(a);
  s2.set(a);
  const bool active = at.count || at.left;
  Channels<T, V, false> ch;
  if (active) {
    ch.load(p, at, nullptr, nullptr);
    const auto add = [&](const Values& v, const Values& g) {
      const Pairs<V> d = widen_pairs<T, V>(v) + ch.minus;
      const Pairs<V> du =
          slope<ACT, sizeof(T) == 4, V>(fma(d, ch.scale, ch.bias)) * widen_pairs<T, V>(g);
      s1 = s1 + du;
      s2 = fma(du, d, s2);
    };
    constexpr int U = 4;  // pairs of reads in flight
    for (int i0 = 0; i0 < at.count; i0 += U) {
      Values v[U], g[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < at.count) {
          v[u] = *reinterpret_cast<const Values*>(from + (i0 + u) * at.stride);
          g[u] = *reinterpret_cast<const Values*>(grad + (i0 + u) * at.stride);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < at.count) {
          if (p.keep) {
            kept_x[(i0 + u) * l.threads] = v[u];
            kept_g[(i0 + u) * l.threads] = g[u];
          }
          add(v[u], g[u]);
        }
    }
    if (at.left) {
      const Values v = load_part<T, V>(from + at.count * at.stride, at.left);
      const Values g = load_part<T, V>(grad + at.count * at.stride, at.left);
      if (p.keep) {
        kept_x[at.count * l.threads] = v;
        kept_g[at.count * l.threads] = g;
      }
      add(v, g);
    }
  }
  s1.get(a);
  s2.get(b);
  cluster_sums<V>(l, a, b, mem.per_thread, mem.own, mem.channel);
  __syncthreads();
  const bool first = cluster_rank() == 0;
  const double n = static_cast<double>(l.span / l.channels) * p.group_channels;
  for (int c = threadIdx.x; c < l.channels; c += l.threads) {
    double2 s = mem.channel[c];
    s.y *= p.rstd[at.sample * p.groups + c / p.group_channels];
    mem.channel[c] = s;
    if (first) {
      if (p.samples > 1) p.channel[static_cast<long long>(at.sample) * l.channels + c] = s;
      if (dbias) dbias[c] = from_float<T>(static_cast<float>(s.x));
      if (dweight) dweight[c] = from_float<T>(static_cast<float>(s.y));
    }
  }
  if (!p.out) return;
  __syncthreads();
  for (int g = threadIdx.x; g < p.groups; g += l.threads) {
    double m1 = 0.0, m2 = 0.0;
    for (int k = 0; k < p.group_channels; ++k) {
      const int c = g * p.group_channels + k;
      const double w = p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0;
      m1 += w * mem.channel[c].x;
      m2 += w * mem.channel[c].y;
    }
    mem.group[g] = make_float2(static_cast<float>(m1 / n), static_cast<float>(m2 / n));
  }
  __syncthreads();
  if (!active) return;
  Channels<T, V, true> k;
  k.load(p, at, nullptr, mem.group);
  T* to = static_cast<T*>(p.out) + offset;
  const auto result = [&](const Values& v, const Values& g) {
    const Pairs<V> d = widen_pairs<T, V>(v) + k.minus;
    const Pairs<V> du =
        slope<ACT, sizeof(T) == 4, V>(fma(d, k.scale, k.bias)) * widen_pairs<T, V>(g);
    return round_pairs<T, V>(fma(du, k.scale, fma(d, k.k2, k.k1)));
  };
  constexpr int U = 4;
  for (int i0 = 0; i0 < at.count; i0 += U) {
    Values v[U], g[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < at.count) {
        v[u] = p.keep ? kept_x[(i0 + u) * l.threads]
                      : *reinterpret_cast<const Values*>(from + (i0 + u) * at.stride);
        g[u] = p.keep ? kept_g[(i0 + u) * l.threads]
                      : *reinterpret_cast<const Values*>(grad + (i0 + u) * at.stride);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < at.count)
        *reinterpret_cast<Values*>(to + (i0 + u) * at.stride) = result(v[u], g[u]);
  }
  if (at.left) {
    const long long o = at.count * at.stride;
    store_part<T, V>(to + o,
                     result(p.keep ? kept_x[at.count * l.threads]
                                   : load_part<T, V>(from + o, at.left),
                            p.keep ? kept_g[at.count * l.threads]
                                   : load_part<T, V>(grad + o, at.left)),
                     at.left);
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

Layout make_layout(int samples, long long positions, int channels, int v, int per_sm,
                   int threads) {
  Layout l;
  l.span = positions * channels;
  l.channels = channels;
  l.period = channels / std::gcd(channels, v);
  if (l.period <= threads) {
    l.threads = l.period * std::max(1, threads / l.period);
    l.columns = 1;
    l.step = l.threads;
  } else {
    l.threads = threads;
    l.columns = (l.period + threads - 1) / threads;
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
constexpr int kForwardBlocksPerSm = 2, kBackwardBlocksPerSm = 1;

// How a call is run: in clusters of l.blocks (small), or in passes.
struct Plan {
  Layout l;
  int vector;
  bool small, keep;
  size_t shared_bytes;
};

Plan make_plan(int value_bytes, int samples, long long positions, int channels, int groups,
               bool backward) {
  Plan plan;
  plan.vector = vector_width(value_bytes, samples, positions * channels);
  const int per_sm = backward ? kBackwardBlocksPerSm : kForwardBlocksPerSm;
  const long long bytes = positions * channels * value_bytes * (backward ? 2 : 1);
  plan.l = make_layout(samples, positions, channels, plan.vector, per_sm, kSmallThreads);
  // few samples, whose clusters run at once, or many that are quick: a cluster is
  // slower than the passes' many blocks (forward, 1 and 4 of 100x100x32 fp32 in 19
  // us each against 22 and 25 in passes, one of 130x130x32 25 against 22; 16 and 64
  // of 20x20x32 21 and 49 against 23 and 35, of 10x10x32 15 and 15 against 22 and
  // 33).  The backward, which waits for the host in a training step, takes more for
  // its fewer launches (2 of 67x101x48 fp32 trained 125 us against 134, where the
  // kernels alone take 25 and 22; one of 170x170x32 bf16 39 against 25)
  plan.small = plan.l.columns == 1 && channels <= kSmallChannels &&
               positions * channels <= (backward ? kSmallBackward : kSmallForward) &&
               (samples <= kFewSamples || samples * bytes <= kManyBytes);
  plan.shared_bytes = 0;
  if (!plan.small) {
    plan.l = make_layout(samples, positions, channels, plan.vector, per_sm, kMaxThreads);
  } else {
    // 8 KB to a block at least, where the sample has them
    int blocks = 1;
    while (blocks < kMaxCluster && blocks * 8192LL < bytes && blocks < plan.l.steps) blocks *= 2;
    plan.l.blocks = blocks;
    plan.l.per_block = (plan.l.steps + blocks - 1) / blocks;
    const auto need = [&](int arrays) {
      return small_bytes(plan.l, plan.vector, value_bytes, groups, arrays, backward);
    };
    plan.keep = need(backward ? 2 : 1) <= kMostShared;
    plan.shared_bytes = need(!plan.keep ? 0 : backward ? 2 : 1);
  }
  return plan;
}

template <class... A, class... B>
int launch_cluster(void (*kernel)(A...), unsigned grid, int threads, int blocks,
                   size_t shared_bytes, cudaStream_t s, B... args) {
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = blocks;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared_bytes;
  config.stream = host::counted(s);
  config.attrs = &cluster;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, kernel, args...) != cudaSuccess)
    return host::check_launch("feature_norm");
  return kOk;
}

// A small sample's kernel, as clusters of the layout's blocks.
template <auto* kernel, class... A>
int launch_small(const Plan& plan, int samples, cudaStream_t s, A... args) {
  if (!host::allow_shared<kernel>()) return host::check_launch("feature_norm: shared memory");
  return launch_cluster(kernel, static_cast<unsigned>(samples) * plan.l.blocks, plan.l.threads,
                        plan.l.blocks, plan.shared_bytes, s, args...);
}

// Blocks that join a group's channels.
int join_blocks(int group_channels) {
  return std::min(kMaxCluster, (group_channels + kJoinChannels - 1) / kJoinChannels);
}

template <int V, class F>
int with_width(int v, F f) {
  if constexpr (V > 1) {
    if (v < V) return with_width<V / 2>(v, f);
  }
  return f(std::integral_constant<int, V>{});
}

size_t round_up(size_t n) { return (n + 15) / 16 * 16; }

size_t partial_bytes(int samples, const Layout& l, bool backward) {
  return round_up(static_cast<size_t>(samples) * l.blocks * l.columns * l.channels *
                  (backward ? sizeof(float2) : sizeof(double2)));
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
  const Plan plan =
      make_plan(bytes_of(dtype), samples, positions, channels, groups, backward != 0);
  const size_t moments = round_up(static_cast<size_t>(samples) * groups * sizeof(float2));
  if (!backward) return plan.small ? 16 : partial_bytes(samples, plan.l, false) + moments;
  return (plan.small ? 0 : partial_bytes(samples, plan.l, true)) + moments +
         static_cast<size_t>(samples) * channels * sizeof(double2);
}

int splat_feature_norm(int dtype, int samples, long long positions, int channels, int groups,
                       const void* x, const void* weight, const void* bias, float eps,
                       int activation, void* y, float* mean, float* rstd, void* workspace,
                       size_t workspace_bytes, void* stream) {
  const int bad = check_norm(dtype, samples, positions, channels, groups, activation);
  if (bad != kOk) return bad;
  if (!x || !y || !mean != !rstd)
    return host::fail(kInvalidArgument, "feature_norm: null pointer");
  if (!host::aligned(x, 16) || !host::aligned(y, 16) || !host::aligned(workspace, 16))
    return host::fail(kInvalidArgument, "feature_norm: x, y and workspace must be 16-byte aligned");
  const Plan plan = make_plan(bytes_of(dtype), samples, positions, channels, groups, false);
  const size_t partial = plan.small ? 0 : partial_bytes(samples, plan.l, false);
  const size_t moments = round_up(static_cast<size_t>(samples) * groups * sizeof(float2));
  if (!plan.small && (!workspace || workspace_bytes < partial + moments))
    return host::fail(kWorkspaceTooSmall, "feature_norm: workspace");
  NormParams p{};
  p.l = plan.l;
  p.keep = plan.small && plan.keep;
  p.samples = samples;
  p.groups = groups;
  p.group_channels = channels / groups;
  p.x = x;
  p.weight = weight;
  p.bias = bias;
  p.out = y;
  p.mean = mean;
  p.rstd = rstd;
  p.partial = workspace;
  if (!mean && !plan.small) {  // the passes hand them on all the same
    p.mean = reinterpret_cast<float*>(static_cast<char*>(workspace) + partial);
    p.rstd = p.mean + static_cast<size_t>(samples) * groups;
  }
  p.eps = eps;
  auto s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(samples) * p.l.blocks * p.l.columns;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return with_width<16 / sizeof(T)>(plan.vector, [&](auto width) {
      constexpr int V = decltype(width)::value;
      if (plan.small)
        return SPLAT_FEATURE_ACT(activation, [&] {
          return launch_small<norm_small_kernel<T, V, ACT>>(plan, samples, s, p);
        });
      norm_sums_kernel<T, V><<<grid, p.l.threads, 0, host::counted(s)>>>(p);
      const int joins = join_blocks(p.group_channels);
      const int status = launch_cluster(norm_join_kernel<T>,
                                        static_cast<unsigned>(samples) * groups * joins,
                                        kJoinThreads, joins, 0, s, p, joins);
      if (status != kOk) return status;
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
  const Plan plan = make_plan(bytes_of(dtype), samples, positions, channels, groups, true);
  if (workspace_bytes < (plan.small ? 0 : partial_bytes(samples, plan.l, true)) +
                            round_up(static_cast<size_t>(samples) * groups * sizeof(float2)) +
                            static_cast<size_t>(samples) * channels * sizeof(double2))
    return host::fail(kWorkspaceTooSmall, "feature_norm_backward: workspace");
  NormParams p{};
  p.l = plan.l;
  p.keep = plan.small && plan.keep;
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
  p.partial = at;
  at += plan.small ? 0 : partial_bytes(samples, p.l, true);
  p.moments = reinterpret_cast<float2*>(at);
  at += round_up(static_cast<size_t>(samples) * groups * sizeof(float2));
  p.channel = reinterpret_cast<double2*>(at);
  auto s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(samples) * p.l.blocks * p.l.columns;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return with_width<16 / sizeof(T)>(plan.vector, [&](auto width) {
      constexpr int V = decltype(width)::value;
      T *dw = static_cast<T*>(dweight), *db = static_cast<T*>(dbias);
      return SPLAT_FEATURE_ACT(activation, [&] {
        // a lone sample's sums are the parameters' gradients
        const bool one = samples == 1;
        T *dw1 = one ? dw : nullptr, *db1 = one ? db : nullptr;
        if (plan.small) {
          const int status = launch_small<norm_backward_small_kernel<T, V, ACT>>(
              plan, samples, s, p, dw1, db1);
          if (status != kOk) return status;
        } else {
          norm_backward_sums_kernel<T, V, ACT><<<grid, p.l.threads, 0, host::counted(s)>>>(p);
          const int joins = join_blocks(p.group_channels);
          const int status = launch_cluster(norm_backward_join_kernel<T>,
                                            static_cast<unsigned>(samples) * groups * joins,
                                            kJoinThreads, joins, 0, s, p, joins, dw1, db1);
          if (status != kOk) return status;
        }
        if (!one && (dw || db))
          norm_parameters_kernel<T>
              <<<host::blocks_for(channels, 128), 128, 0, host::counted(s)>>>(p, dw, db);
        if (dx && !plan.small)
          norm_backward_apply_kernel<T, V, ACT><<<grid, p.l.threads, 0, host::counted(s)>>>(p);
        return host::check_launch("feature_norm_backward");
      });
    });
  });
}

}  // extern "C"
