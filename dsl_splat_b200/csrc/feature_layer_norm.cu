// Layer norm over the last dimension of channel-last rows, with an activation:
//
//   h = (x - mean) rstd,  u = h w + b,  y = act(u)
//   du = dy act'(u),  d = du w
//   dx = rstd (d - mean(d) - h mean(d h)),  dw = sum du h,  db = sum du over rows
//
// A row's values stay in the registers of a group of lanes (up to 1024 of them) or
// of a block (up to 8192), so that x and dy are read once.  The mean is taken twice:
// the second time of the deviations from the first, whose squares give the
// variance without a subtraction of like numbers.  The backward takes both again
// from x, which it has to read: two floats kept per row would cost a row of 32
// 16-bit channels an eighth of its bytes each way.  A thread meets the same channels
// in all of its rows and adds their du and du h in registers; blocks' sums are
// joined in a fixed order.
#include <algorithm>

#include "feature_common.cuh"
#include "feature_join.cuh"
#include "host_runtime.h"
#include "splat200.h"

namespace splat {
namespace feature {

constexpr int kNormThreads = 256;
constexpr int kMostLaneValues = 32;                              // of a row, in a thread
constexpr int kMostGroupChannels = 32 * kMostLaneValues;         // of a row, in a warp
constexpr int kMostBlockChannels = kNormThreads * kMostLaneValues;
constexpr int kMostChannels = 65535;

struct LayerNormParams {
  long long rows;
  int channels, lanes;  // lanes of a row: a power of two, up to 32
  const void *x, *weight, *bias, *dy;
  void *y, *dx;    // y: the forward's; dx: NULL if not wanted
  float* partial;  // (blocks, 2, channels) sums of du h and du, or NULL
  float* moments;  // (3, rows) of rows longer than a block's registers
  float eps;
  int activation;
};

// Sums over the lanes of a row, all lanes get them.
template <bool BLOCK, int K>
SPLAT_DEV void sum_lanes(float (&v)[K], int lanes) {
  for (int o = (BLOCK ? 32 : lanes) / 2; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (BLOCK) {
    __shared__ float sums[K][kNormThreads / 32];
    __syncthreads();  // the sums before have been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) sums[k][threadIdx.x >> 5] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < kNormThreads / 32; ++i) v[k] += sums[k][i];
    }
  }
}

// x of a row -> its deviations from the mean; returns rstd.
template <bool BLOCK, int N>
SPLAT_DEV float centre(float (&v)[N], const bool (&in)[N], int lanes, float inverse, float eps) {
  float sum[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < N; ++i) sum[0] += v[i];
  sum_lanes<BLOCK>(sum, lanes);
  const float mean = sum[0] * inverse;
  float rest[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = in[i] ? v[i] - mean : 0.0f;
    rest[0] += v[i];
    rest[1] += v[i] * v[i];
  }
  sum_lanes<BLOCK>(rest, lanes);
  const float more = rest[0] * inverse;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] -= more;
  return rsqrtf(fmaxf(rest[1] * inverse - more * more, 0.0f) + eps);
}

template <int N, bool FINE>
SPLAT_DEV void activate_all(int activation, float (&u)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    switch (activation) {
      case kRelu: activate2<kRelu, FINE>(u[i], u[i + 1]); break;
      case kSilu: activate2<kSilu, FINE>(u[i], u[i + 1]); break;
      case kGelu: activate2<kGelu, FINE>(u[i], u[i + 1]); break;
      case kSigmoid: activate2<kSigmoid, FINE>(u[i], u[i + 1]); break;
      default: break;
    }
  }
}
template <int N, bool FINE>
SPLAT_DEV void slope_all(int activation, float (&u)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    switch (activation) {
      case kRelu: slope2<kRelu, FINE>(u[i], u[i + 1]); break;
      case kSilu: slope2<kSilu, FINE>(u[i], u[i + 1]); break;
      case kGelu: slope2<kGelu, FINE>(u[i], u[i + 1]); break;
      case kSigmoid: slope2<kSigmoid, FINE>(u[i], u[i + 1]); break;
      default: u[i] = u[i + 1] = 1.0f;
    }
  }
}

// V values a load, J loads a row and thread.
template <class T, int V, int J, bool BLOCK, bool BACKWARD>
__global__ void __launch_bounds__(kNormThreads) layer_norm_kernel(const LayerNormParams p) {
  constexpr int N = V * J;
  constexpr bool kFine = sizeof(T) == 4;
  using Piece = Vec<T, V>;
  const int lanes = BLOCK ? kNormThreads : p.lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int C = p.channels;
  const float inverse = 1.0f / static_cast<float>(C);
  bool in[N];
  float w[N], b[N];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (j * lanes + lane) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      in[j * V + i] = c < C;  // C is a multiple of V
      w[j * V + i] = c < C && p.weight ? to_float(static_cast<const T*>(p.weight)[c + i]) : 1.0f;
      b[j * V + i] = c < C && p.bias ? to_float(static_cast<const T*>(p.bias)[c + i]) : 0.0f;
    }
  }
  float dw[BACKWARD ? N : 1] = {}, db[BACKWARD ? N : 1] = {};
  // a warp's groups step together
  const int groups = BLOCK ? 1 : 32 / lanes;
  const int group = BLOCK ? 0 : (threadIdx.x & 31) / lanes;
  const long long first =
      BLOCK ? blockIdx.x : (blockIdx.x * (kNormThreads / 32LL) + (threadIdx.x >> 5)) * groups;
  const long long step = BLOCK ? gridDim.x : gridDim.x * (kNormThreads / 32LL) * groups;
  for (long long row0 = first; row0 < p.rows; row0 += step) {
    const long long row = row0 + group, at = row * C;
    const bool here = row < p.rows;
    Piece raw[J], up[BACKWARD ? J : 1];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      raw[j] = Piece{};
      if (here && in[j * V])
        raw[j] = *reinterpret_cast<const Piece*>(static_cast<const T*>(p.x) + at +
                                                 (j * lanes + lane) * V);
    }
    if constexpr (BACKWARD) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        up[j] = Piece{};
        if (here && in[j * V])
          up[j] = *reinterpret_cast<const Piece*>(static_cast<const T*>(p.dy) + at +
                                                  (j * lanes + lane) * V);
      }
    }
    float h[N], u[N];
#pragma unroll
    for (int j = 0; j < J; ++j) widen<T, V>(raw[j], reinterpret_cast<float(&)[V]>(h[j * V]));
    const float rstd = centre<BLOCK>(h, in, lanes, inverse, p.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      h[i] *= rstd;
      u[i] = fmaf(h[i], w[i], b[i]);
    }
    if constexpr (!BACKWARD) {
      activate_all<N, kFine>(p.activation, u);
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (here && in[j * V])
          *reinterpret_cast<Piece*>(static_cast<T*>(p.y) + at + (j * lanes + lane) * V) =
              round_values<T, V>(reinterpret_cast<const float(&)[V]>(u[j * V]));
    } else {
      float g[N], sums[2] = {0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < J; ++j) widen<T, V>(up[j], reinterpret_cast<float(&)[V]>(g[j * V]));
      slope_all<N, kFine>(p.activation, u);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        g[i] *= u[i];
        db[i] += g[i];
        dw[i] = fmaf(g[i], h[i], dw[i]);
        g[i] *= w[i];
        sums[0] += g[i];
        sums[1] = fmaf(g[i], h[i], sums[1]);
      }
      if (p.dx) {
        sum_lanes<BLOCK>(sums, lanes);
        const float less = sums[0] * inverse, along = sums[1] * inverse;
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = rstd * (g[i] - fmaf(h[i], along, less));
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (here && in[j * V])
            *reinterpret_cast<Piece*>(static_cast<T*>(p.dx) + at + (j * lanes + lane) * V) =
                round_values<T, V>(reinterpret_cast<const float(&)[V]>(g[j * V]));
      }
    }
  }
  if constexpr (BACKWARD) {
    if (!p.partial) return;
    float* to = p.partial + 2LL * blockIdx.x * C;
    if constexpr (BLOCK) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!in[i]) continue;
        const int c = (i / V * lanes + lane) * V + i % V;
        to[c] = dw[i];
        to[C + c] = db[i];
      }
    } else {
      // the groups of a warp, then the warps one after another
      __shared__ float sums[2 * kMostGroupChannels];
      for (int o = lanes; o < 32; o *= 2)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
          db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
        }
      for (int k = 0; k < kNormThreads / 32; ++k) {
        if (static_cast<int>(threadIdx.x >> 5) == k && group == 0) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (!in[i]) continue;
            const int c = (i / V * lanes + lane) * V + i % V;
            sums[c] = (k ? sums[c] : 0.0f) + dw[i];
            sums[C + c] = (k ? sums[C + c] : 0.0f) + db[i];
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < 2 * C; c += kNormThreads) to[c] = sums[c];
    }
  }
}

// ---- rows longer than a block's registers -----------------------------------------

// A block to a row, which it reads again from the caches for each sum.
template <class T, bool BACKWARD>
__global__ void __launch_bounds__(kNormThreads) long_rows_kernel(const LayerNormParams p) {
  constexpr bool kFine = sizeof(T) == 4;
  const int C = p.channels;
  const float inverse = 1.0f / static_cast<float>(C);
  const T *w = static_cast<const T*>(p.weight), *b = static_cast<const T*>(p.bias);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * C;
    const T* dy = static_cast<const T*>(p.dy) + row * C;
    float sum[1] = {0.0f}, rest[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < C; c += kNormThreads) sum[0] += to_float(x[c]);
    sum_lanes<true>(sum, kNormThreads);
    const float mean = sum[0] * inverse;
    for (int c = threadIdx.x; c < C; c += kNormThreads) {
      const float d = to_float(x[c]) - mean;
      rest[0] += d;
      rest[1] += d * d;
    }
    sum_lanes<true>(rest, kNormThreads);
    const float more = rest[0] * inverse;
    const float rstd = rsqrtf(fmaxf(rest[1] * inverse - more * more, 0.0f) + p.eps);
    if (BACKWARD && threadIdx.x == 0) {
      p.moments[row] = mean;
      p.moments[p.rows + row] = more;
      p.moments[2 * p.rows + row] = rstd;
    }
    if (BACKWARD && !p.dx) continue;
    float less = 0.0f, along = 0.0f;
    // the backward's first pass adds up, its second one writes
    for (int pass = BACKWARD ? 0 : 1; pass < 2; ++pass) {
      float sums[2] = {0.0f, 0.0f};
      for (int c = threadIdx.x; c < C; c += kNormThreads) {
        const float h = (to_float(x[c]) - mean - more) * rstd, scale = w ? to_float(w[c]) : 1.0f;
        float u[2] = {fmaf(h, scale, b ? to_float(b[c]) : 0.0f), 0.0f};
        if constexpr (!BACKWARD) {
          activate_all<2, kFine>(p.activation, u);
          static_cast<T*>(p.y)[row * C + c] = from_float<T>(u[0]);
        } else {
          slope_all<2, kFine>(p.activation, u);
          const float g = to_float(dy[c]) * u[0] * scale;
          if (pass == 0) {
            sums[0] += g;
            sums[1] = fmaf(g, h, sums[1]);
          } else {
            static_cast<T*>(p.dx)[row * C + c] =
                from_float<T>(rstd * (g - fmaf(h, along, less)));
          }
        }
      }
      if (BACKWARD && pass == 0) {
        sum_lanes<true>(sums, kNormThreads);
        less = sums[0] * inverse;
        along = sums[1] * inverse;
      }
    }
  }
}

// Their sums over rows: a thread to a channel, a block to a range of rows.
template <class T>
__global__ void __launch_bounds__(kNormThreads)
    long_columns_kernel(const LayerNormParams p, long long range) {
  constexpr bool kFine = sizeof(T) == 4;
  const int C = p.channels, c = blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= C) return;
  const float w = p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0f;
  const float b = p.bias ? to_float(static_cast<const T*>(p.bias)[c]) : 0.0f;
  const long long begin = blockIdx.y * range, end = min(begin + range, p.rows);
  float dw = 0.0f, db = 0.0f;
#pragma unroll 4
  for (long long row = begin; row < end; ++row) {
    const float h = (to_float(static_cast<const T*>(p.x)[row * C + c]) - p.moments[row] -
                     p.moments[p.rows + row]) *
                    p.moments[2 * p.rows + row];
    float u[2] = {fmaf(h, w, b), 0.0f};
    slope_all<2, kFine>(p.activation, u);
    const float g = to_float(static_cast<const T*>(p.dy)[row * C + c]) * u[0];
    db += g;
    dw = fmaf(g, h, dw);
  }
  float* to = p.partial + 2LL * blockIdx.y * C;
  to[c] = dw;
  to[C + c] = db;
}

// ---- launching -------------------------------------------------------------------

struct LayerNormPlan {
  int blocks, lanes;  // lanes: 0: a block to a row
  bool longer;        // than a block's registers
  long long range;    // of rows, of their columns' sums
};

template <class T>
LayerNormPlan plan_norm(long long rows, int channels, bool backward) {
  constexpr int V = 16 / sizeof(T);
  LayerNormPlan plan{};
  const int sms = host::sm_count();
  plan.longer = channels > kMostBlockChannels;
  if (plan.longer) {
    plan.blocks = static_cast<int>(std::min<long long>(rows, 4LL * sms));
    const long long most = std::max(1LL, 4LL * sms / host::blocks_for(channels, kNormThreads));
    plan.range = (rows + most - 1) / most;
    return plan;
  }
  long long rows_at_once = 1;
  if (channels <= kMostGroupChannels) {
    // eight values a lane, where rows are whole 16-byte pieces and where not
    const int width = channels % V == 0 ? std::max(V, 8) : 8;
    plan.lanes = 1;
    while (plan.lanes < 32 && plan.lanes * width < channels) plan.lanes *= 2;
    rows_at_once = kNormThreads / plan.lanes;
  }
  plan.blocks = static_cast<int>(std::min<long long>((rows + rows_at_once - 1) / rows_at_once,
                                                     (backward ? 4LL : 8LL) * sms));
  return plan;
}

template <class T, bool BACKWARD>
void launch_norm(const LayerNormPlan& plan, LayerNormParams& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  p.lanes = plan.lanes;
  const auto run = [&](auto* kernel) {
    kernel<<<plan.blocks, kNormThreads, 0, host::counted(s)>>>(p);
  };
  if (plan.longer) return run(long_rows_kernel<T, BACKWARD>);
  const int lanes = plan.lanes ? plan.lanes : kNormThreads;
  const int each = (p.channels + lanes - 1) / lanes;  // values a lane
  const bool vector = p.channels % V == 0 && host::aligned(p.x, 16) && host::aligned(p.y, 16) &&
                      host::aligned(p.dy, 16) && host::aligned(p.dx, 16);
  if (!plan.lanes) {
    if (vector) run(layer_norm_kernel<T, V, 32 / V, true, BACKWARD>);
    else run(layer_norm_kernel<T, 1, 32, true, BACKWARD>);
  } else if (each <= 8) {
    if (vector) run(layer_norm_kernel<T, V, 8 / V, false, BACKWARD>);
    else run(layer_norm_kernel<T, 1, 8, false, BACKWARD>);
  } else if (each <= 16) {
    if (vector) run(layer_norm_kernel<T, V, 16 / V, false, BACKWARD>);
    else run(layer_norm_kernel<T, 1, 16, false, BACKWARD>);
  } else {
    if (vector) run(layer_norm_kernel<T, V, 32 / V, false, BACKWARD>);
    else run(layer_norm_kernel<T, 1, 32, false, BACKWARD>);
  }
}

int check_layer_norm(int dtype, long long rows, int channels, int activation) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "feature_layer_norm: dtype");
  if (activation < 0 || activation > 4)
    return host::fail(kInvalidArgument, "feature_layer_norm: activation");
  if (rows < 1 || channels < 1) return host::fail(kInvalidArgument, "feature_layer_norm: sizes");
  if (channels > kMostChannels || rows > (1LL << 40))
    return host::fail(kTooLarge, "feature_layer_norm: too many rows or channels");
  return kOk;
}

// Bytes of the long rows' moments, before the partial sums.
size_t moments_bytes(const LayerNormPlan& plan, long long rows) {
  return plan.longer ? static_cast<size_t>((3 * rows * 4 + 15) / 16 * 16) : 0;
}
int sums(const LayerNormPlan& plan, long long rows) {
  return plan.longer ? static_cast<int>((rows + plan.range - 1) / plan.range) : plan.blocks;
}

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

int splat_feature_layer_norm(int dtype, long long rows, int channels, const void* x,
                             const void* weight, const void* bias, float eps, int activation,
                             void* y, void* stream) {
  const int bad = check_layer_norm(dtype, rows, channels, activation);
  if (bad != kOk) return bad;
  if (!x || !y) return host::fail(kInvalidArgument, "feature_layer_norm: null pointer");
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    LayerNormParams p{};
    p.rows = rows, p.channels = channels;
    p.x = x, p.weight = weight, p.bias = bias, p.y = y;
    p.eps = eps, p.activation = activation;
    launch_norm<T, false>(plan_norm<T>(rows, channels, false), p,
                          static_cast<cudaStream_t>(stream));
    return host::check_launch("feature_layer_norm");
  });
}

size_t splat_feature_layer_norm_backward_workspace_bytes(int dtype, long long rows, int channels) {
  if (check_layer_norm(dtype, rows, channels, 0) != kOk) return 0;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    const LayerNormPlan plan = plan_norm<T>(rows, channels, true);
    return moments_bytes(plan, rows) + static_cast<size_t>(sums(plan, rows)) * 2 * channels * 4;
  });
}

int splat_feature_layer_norm_backward(int dtype, long long rows, int channels, const void* x,
                                      const void* weight, const void* bias, float eps,
                                      int activation, const void* dy, void* dx, void* dweight,
                                      void* dbias, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const int bad = check_layer_norm(dtype, rows, channels, activation);
  if (bad != kOk) return bad;
  if (!x || !dy || !workspace)
    return host::fail(kInvalidArgument, "feature_layer_norm_backward: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument,
                      "feature_layer_norm_backward: workspace not 16-byte aligned");
  if (workspace_bytes < splat_feature_layer_norm_backward_workspace_bytes(dtype, rows, channels))
    return host::fail(kWorkspaceTooSmall, "feature_layer_norm_backward: workspace");
  auto s = static_cast<cudaStream_t>(stream);
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    const LayerNormPlan plan = plan_norm<T>(rows, channels, true);
    LayerNormParams p{};
    p.rows = rows, p.channels = channels;
    p.x = x, p.weight = weight, p.bias = bias, p.dy = dy, p.dx = dx;
    p.eps = eps, p.activation = activation;
    p.moments = static_cast<float*>(workspace);
    if (dweight || dbias)
      p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                           moments_bytes(plan, rows));
    launch_norm<T, true>(plan, p, s);
    if (p.partial) {
      const int count = sums(plan, rows);
      if (plan.longer)
        long_columns_kernel<T>
            <<<dim3(host::blocks_for(channels, kNormThreads), count), kNormThreads, 0,
               host::counted(s)>>>(p, plan.range);
      join_splits<T>(p.partial, 2LL * channels, count, channels, channels, dweight, dbias, s);
    }
    return host::check_launch("feature_layer_norm_backward");
  });
}

}  // extern "C"
