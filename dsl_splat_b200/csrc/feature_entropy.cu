// Softmax cross entropy of a linear head over a vocabulary:
//
//   z = x W^T + b,  lse_i = log sum_j exp z_ij,  l_i = lse_i - z_i,t_i
//   dz_ij = u_i (exp(z_ij - lse_i) - [j = t_i]),  dx = dz W,  dW = dz^T x,  db = sum_i dz_i
//
// The logits are never kept: they are formed for a piece of the rows at a time, and
// formed again in the backward.  u_i is the upstream gradient of row i's loss (divided by
// the number of rows that count for their mean) and 0 for the others.
//
// dz is held in T for the products.  It is taken relative to the power of two E that
// is not below any |u_i|, times 2^15 of float16, whose smallest value would otherwise
// swallow the tail of a large vocabulary; the products' fp32 results are multiplied by the
// inverse before their rounding.
#include <algorithm>

#include "feature_join.cuh"
#include "feature_launch.cuh"
#include "splat200.h"

namespace splat {
namespace feature {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLog2E = 1.44269504088896341f;

enum Reduction : int { kEach = 0, kSum = 1, kMean = 2 };

// What the rows' kernels read.
struct Rows {
  long long rows;
  int vocabulary, id_bytes, reduction;
  long long ignored;
  const void* target;
  int* error;
};

// A row's label, or -1 where it does not count.
SPLAT_DEV int label_of(const Rows& p, long long row) {
  const long long t = p.id_bytes == 8 ? static_cast<const long long*>(p.target)[row]
                                      : static_cast<const int*>(p.target)[row];
  if (t == p.ignored) return -1;
  if (t >= 0 && t < p.vocabulary) return static_cast<int>(t);
  atomicCAS(p.error, 0, kInconsistentInput);
  return -1;
}

// ---- softmax statistics ------------------------------------------------------------

// Largest exponent so far and the sum relative to it.  A row that holds nothing but
// minus infinities (or nothing at all) has the sum 0.
struct Partial {
  float top, sum;
};
SPLAT_DEV Partial join(Partial a, Partial b) {
  const float top = fmaxf(a.top, b.top);  // NaN lies in the sums
  if (top == -INFINITY) return {top, a.sum + b.sum};
  return {top, a.sum * exp2f((a.top - top) * kLog2E) + b.sum * exp2f((b.top - top) * kLog2E)};
}
SPLAT_DEV void take(Partial& s, float z) {
  if (z > s.top) {
    s.sum = s.sum * exp2f((s.top - z) * kLog2E) + 1.0f;
    s.top = z;
  } else {
    // -inf - -inf: nothing yet; NaN compares false and comes in here
    s.sum += z == -INFINITY ? 0.0f : exp2f((z - s.top) * kLog2E);
  }
}

// Rows of logits (fp32, ld apart) -> lse and losses; a warp or a block to a row.
template <class T, bool BLOCK>
__global__ void __launch_bounds__(kThreads)
    row_loss_kernel(const Rows p, long long first, int rows, const float* z, int ld,
                    const T* bias, float* lse, float* loss) {
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31, lanes = BLOCK ? kThreads : 32;
  const int r = BLOCK ? blockIdx.x : blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const float* from = z + static_cast<long long>(r) * ld;
  Partial s{-INFINITY, 0.0f};
  for (int j = lane; j < p.vocabulary; j += lanes)
    take(s, from[j] + (bias ? to_float(bias[j]) : 0.0f));
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const Partial other{__shfl_xor_sync(0xffffffffu, s.top, o),
                        __shfl_xor_sync(0xffffffffu, s.sum, o)};
    s = join(s, other);
  }
  if constexpr (BLOCK) {
    __shared__ Partial all[kWarps];
    if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = s;
    __syncthreads();
    s = all[0];
    for (int w = 1; w < kWarps; ++w) s = join(s, all[w]);
  }
  if (lane != 0) return;
  const float value = s.top + logf(s.sum);
  lse[first + r] = value;
  const int t = label_of(p, first + r);
  loss[first + r] = t < 0 ? 0.0f : value - (from[t] + (bias ? to_float(bias[t]) : 0.0f));
}

// The losses' sum or mean and the number of rows that count, in doubles and in a fixed
// order: blocks over ranges of rows, then one over the blocks.
constexpr int kLossBlocks = 128;
struct LossSum {
  double sum;
  long long count;
};
SPLAT_DEV LossSum block_sum(LossSum s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s.sum += __shfl_xor_sync(0xffffffffu, s.sum, o);
    s.count += __shfl_xor_sync(0xffffffffu, s.count, o);
  }
  __shared__ LossSum all[kWarps];
  if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = s;
  __syncthreads();
  s = all[0];
  for (int w = 1; w < kWarps; ++w) s.sum += all[w].sum, s.count += all[w].count;
  return s;
}
__global__ void __launch_bounds__(kThreads)
    loss_sums_kernel(const Rows p, const float* loss, LossSum* sums) {
  LossSum s{0.0, 0};
  for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < p.rows;
       i += static_cast<long long>(kThreads) * gridDim.x) {
    if (label_of(p, i) < 0) continue;
    s.sum += loss[i];
    ++s.count;
  }
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}
__global__ void __launch_bounds__(kThreads)
    loss_total_kernel(int reduction, const LossSum* sums, int count, float* loss, float* counted) {
  LossSum s{0.0, 0};
  if (threadIdx.x < count) s = sums[threadIdx.x];
  s = block_sum(s);
  if (threadIdx.x) return;
  const double number = static_cast<double>(s.count > 0 ? s.count : 1);
  *loss = static_cast<float>(reduction == kMean ? s.sum / number : s.sum);
  if (counted) *counted = static_cast<float>(number);
}

// ---- gradients -----------------------------------------------------------------------

// Factors of the backward: of u_i on the way into dz, and of the products' results.
struct Factors {
  float in, out;
};

// The power of two that is not below any finite |u|.
__global__ void __launch_bounds__(1024)
    factors_kernel(long long rows, int reduction, const float* upstream, const float* counted,
                   float within, Factors* factors) {
  uint32_t most = 0;
  const long long n = reduction == kEach ? rows : 1;
  for (long long i = threadIdx.x; i < n; i += 1024) {
    float u = upstream[i];
    if (reduction == kMean) u /= *counted;
    const uint32_t bits = __float_as_uint(u) & 0x7fffffffu;
    if (bits < 0x7f800000u) most = max(most, bits);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  __shared__ uint32_t all[32];
  if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 32; ++w) most = max(most, all[w]);
  // 2^e with e in [-100, 126], whose inverse times `within` is finite; 0 of nothing
  int e = static_cast<int>(most >> 23) - 127 + ((most & 0x7fffffu) != 0);
  e = min(max(e, -100), 126);
  factors->in = most ? __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * within : 0.0f;
  factors->out = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) / within;
}

SPLAT_DEV float upstream_of(const Rows& p, long long row, const float* upstream,
                            const float* counted) {
  const float u = upstream[p.reduction == kEach ? row : 0];
  return p.reduction == kMean ? u / *counted : u;
}

// Logits -> dz of TO, rows ld_out apart; a warp or a block to a row.  May be in place.
template <class T, class TO, bool BLOCK>
__global__ void __launch_bounds__(kThreads)
    row_slope_kernel(const Rows p, long long first, int rows, const float* z, int ld,
                     const T* bias, const float* lse, const float* upstream,
                     const float* counted, const Factors* factors, TO* dz, int ld_out) {
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31, lanes = BLOCK ? kThreads : 32;
  const int r = BLOCK ? blockIdx.x : blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const float* from = z + static_cast<long long>(r) * ld;
  TO* to = dz + static_cast<long long>(r) * ld_out;
  const int t = label_of(p, first + r);
  const float u = t < 0 ? 0.0f : upstream_of(p, first + r, upstream, counted) * factors->in;
  const float less = lse[first + r];
  for (int j = lane; j < ld_out; j += lanes) {
    float v = 0.0f;
    if (t >= 0 && j < p.vocabulary) {
      v = expf(from[j] + (bias ? to_float(bias[j]) : 0.0f) - less);
      v = (j == t ? v - 1.0f : v) * u;
    }
    to[j] = from_float<TO>(v);
  }
}

// Column sums of dz's values before their rounding, over ranges of 256 rows.
constexpr int kSumRows = 256;
template <class T>
__global__ void __launch_bounds__(kThreads)
    column_slopes_kernel(const Rows p, long long first, int rows, const float* z, int ld,
                         const T* bias, const float* lse, const float* upstream,
                         const float* counted, const Factors* factors, float* sums) {
  const int j = blockIdx.x * kThreads + threadIdx.x;
  if (j >= p.vocabulary) return;
  const int begin = blockIdx.y * kSumRows, end = min(begin + kSumRows, rows);
  const float b = to_float(bias[j]);
  float sum = 0.0f;
  for (int r = begin; r < end; ++r) {
    const int t = label_of(p, first + r);
    if (t < 0) continue;
    float v = expf(z[static_cast<long long>(r) * ld + j] + b - lse[first + r]);
    v = j == t ? v - 1.0f : v;
    sum = fmaf(v, upstream_of(p, first + r, upstream, counted) * factors->in, sum);
  }
  sums[static_cast<long long>(blockIdx.y) * p.vocabulary + j] = sum;
}
// Adds a piece's ranges to the sums of the pieces before.
__global__ void __launch_bounds__(kThreads)
    add_columns_kernel(int vocabulary, int ranges, const float* sums, bool begin, float* total) {
  const int j = blockIdx.x * kThreads + threadIdx.x;
  if (j >= vocabulary) return;
  float sum = begin ? 0.0f : total[j];
#pragma unroll 8
  for (int r = 0; r < ranges; ++r) sum += sums[static_cast<long long>(r) * vocabulary + j];
  total[j] = sum;
}

// fp32 sums (of several splits, `stride` values apart) times the factor, rounded.
template <class T>
__global__ void __launch_bounds__(kThreads)
    finish_kernel(long long count, int splits, long long stride, const float* from,
                  const Factors* factors, T* to) {
  const float factor = factors->out;
  for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < count;
       i += static_cast<long long>(kThreads) * gridDim.x) {
    float sum = 0.0f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) sum += from[s * stride + i];
    to[i] = from_float<T>(sum * factor);
  }
}
template <class T>
void finish(long long count, int splits, long long stride, const float* from,
            const Factors* factors, void* to, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(
      std::min<long long>((count + kThreads - 1) / kThreads, 16LL * host::sm_count()));
  finish_kernel<T><<<grid, kThreads, 0, host::counted(s)>>>(count, splits, stride, from, factors,
                                                            static_cast<T*>(to));
}

// ---- launching -----------------------------------------------------------------------

constexpr int kMostVocabulary = 1 << 20;
constexpr long long kPieceBytes = 256LL << 20;

// The rows of a piece, and where its parts lie in the workspace.
struct EntropyPlan {
  int piece, splits;
  long long split_rows;
  size_t logits, dz, x_planes, w_planes, dz_planes, weight_sums, column_sums, column_total, dx,
      losses, lse, loss_sums, factors, bytes;
};

template <class T>
EntropyPlan plan_entropy(long long rows, int k, int vocabulary, bool backward) {
  EntropyPlan plan{};
  long long piece = std::max(1LL, kPieceBytes / 4 / vocabulary / kTileRows) * kTileRows;
  piece = std::min({piece, rows, 1LL << 23});  // 65535 ranges of 256 rows, and below
  plan.piece = static_cast<int>(piece);
  const auto take = [&](size_t n) {
    const size_t at = plan.bytes;
    plan.bytes += (n + 255) / 256 * 256;
    return at;
  };
  plan.factors = take(sizeof(Factors));
  plan.loss_sums = take(sizeof(LossSum) * kLossBlocks);
  plan.logits = take(4ull * piece * vocabulary);
  plan.x_planes = take(plane_bytes<T>(piece, k));
  plan.w_planes = take(plane_bytes<T>(vocabulary, k));
  if (!backward) {
    plan.lse = take(4ull * rows);
    plan.losses = take(4ull * rows);
    return plan;
  }
  if (sizeof(T) == 2) plan.dz = take(2ull * piece * round_to(vocabulary, 8));
  else plan.dz_planes = take(plane_bytes<T>(piece, vocabulary));
  plan.dx = take(4ull * piece * k);
  const long long tiles = ((vocabulary + 127LL) / 128) * ((k + 127) / 128);
  const long long wanted = std::max(1LL, 2LL * host::sm_count() / tiles);
  const long long most = std::min(wanted, (piece + 511) / 512);
  plan.split_rows = round_to((piece + most - 1) / most, kChunk);
  plan.splits = static_cast<int>((piece + plan.split_rows - 1) / plan.split_rows);
  plan.weight_sums = take(4ull * plan.splits * vocabulary * k);
  plan.column_sums = take(4ull * ((piece + kSumRows - 1) / kSumRows) * vocabulary);
  plan.column_total = take(4ull * vocabulary);
  return plan;
}

// The logits of rows [first, first + rows).
template <class T>
int launch_logits(int rows, int k, int vocabulary, const Planes& x, const Planes& w, float* z,
                  cudaStream_t s) {
  constexpr int P = kOperandParts<T>;
  ProductParams p{};
  p.m = rows, p.k = k, p.n = vocabulary;
  use_planes(p, x, w);
  p.k_per_split = k, p.splits = 1;
  p.out = z;
  return launch_product<T, P, false, T, P, false, float, float, kPlain>(p, s);
}

template <class F>
void by_row(int rows, int vocabulary, F launch) {
  if (vocabulary <= 2048) launch(std::false_type{}, (rows + kWarps - 1) / kWarps);
  else launch(std::true_type{}, rows);
}

int check_entropy(int dtype, long long rows, int k, int vocabulary, int id_bytes, int reduction) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "feature_entropy: dtype");
  if (rows < 1 || k < 1 || vocabulary < 1)
    return host::fail(kInvalidArgument, "feature_entropy: sizes");
  if (id_bytes != 4 && id_bytes != 8)
    return host::fail(kInvalidArgument, "feature_entropy: targets are of 4 or 8 bytes");
  if (reduction < kEach || reduction > kMean)
    return host::fail(kInvalidArgument, "feature_entropy: reduction");
  if (k > 65535 || vocabulary > kMostVocabulary || rows > 1LL << 31)
    return host::fail(kTooLarge, "feature_entropy: too many rows, inputs or words");
  return kOk;
}

template <class T>
int launch_forward(const Rows& r, int k, const void* x, const void* weight, const void* bias,
                   float* loss, float* lse, float* counted, char* ws, cudaStream_t s) {
  const int vocabulary = r.vocabulary;
  const EntropyPlan plan = plan_entropy<T>(r.rows, k, vocabulary, false);
  float* z = reinterpret_cast<float*>(ws + plan.logits);
  if (!lse) lse = reinterpret_cast<float*>(ws + plan.lse);
  float* each = r.reduction == kEach ? loss : reinterpret_cast<float*>(ws + plan.losses);
  const Planes w = split<T>(weight, vocabulary, k, ws + plan.w_planes, s);
  for (long long first = 0; first < r.rows; first += plan.piece) {
    const int rows = static_cast<int>(std::min<long long>(plan.piece, r.rows - first));
    const Planes xs = split<T>(static_cast<const T*>(x) + first * k, rows, k,
                               ws + plan.x_planes, s);
    const int status = launch_logits<T>(rows, k, vocabulary, xs, w, z, s);
    if (status != kOk) return status;
    by_row(rows, vocabulary, [&](auto block, int grid) {
      row_loss_kernel<T, decltype(block)::value><<<grid, kThreads, 0, host::counted(s)>>>(
          r, first, rows, z, vocabulary, static_cast<const T*>(bias), lse, each);
    });
  }
  if (r.reduction != kEach) {
    auto* sums = reinterpret_cast<LossSum*>(ws + plan.loss_sums);
    const int blocks = static_cast<int>(std::min<long long>((r.rows + kThreads - 1) / kThreads,
                                                            kLossBlocks));
    loss_sums_kernel<<<blocks, kThreads, 0, host::counted(s)>>>(r, each, sums);
    loss_total_kernel<<<1, kThreads, 0, host::counted(s)>>>(r.reduction, sums, blocks, loss,
                                                            counted);
  }
  return host::check_launch("feature_entropy");
}

template <class T>
int launch_backward(const Rows& r, int k, const void* x, const void* weight, const void* bias,
                    const float* lse, const float* counted, const float* upstream, void* dx,
                    void* dweight, void* dbias, char* ws, cudaStream_t s) {
  constexpr int P = kOperandParts<T>;
  const int vocabulary = r.vocabulary;
  const EntropyPlan plan = plan_entropy<T>(r.rows, k, vocabulary, true);
  float* z = reinterpret_cast<float*>(ws + plan.logits);
  auto* factors = reinterpret_cast<Factors*>(ws + plan.factors);
  float* weight_sums = reinterpret_cast<float*>(ws + plan.weight_sums);
  float* dx_sums = reinterpret_cast<float*>(ws + plan.dx);
  float* column_sums = reinterpret_cast<float*>(ws + plan.column_sums);
  float* column_total = reinterpret_cast<float*>(ws + plan.column_total);
  factors_kernel<<<1, 1024, 0, host::counted(s)>>>(
      r.rows, r.reduction, upstream, counted, kIsF16<T> ? 32768.0f : 1.0f, factors);
  const Planes w = split<T>(weight, vocabulary, k, ws + plan.w_planes, s);
  const T* b = static_cast<const T*>(bias);
  int splits = 0;  // that have sums
  for (long long first = 0; first < r.rows; first += plan.piece) {
    const int rows = static_cast<int>(std::min<long long>(plan.piece, r.rows - first));
    const Planes xs = split<T>(static_cast<const T*>(x) + first * k, rows, k,
                               ws + plan.x_planes, s);
    int status = launch_logits<T>(rows, k, vocabulary, xs, w, z, s);
    if (status != kOk) return status;
    if (dbias) {
      const int ranges = (rows + kSumRows - 1) / kSumRows;
      column_slopes_kernel<T>
          <<<dim3(host::blocks_for(vocabulary, kThreads), ranges), kThreads, 0,
             host::counted(s)>>>(r, first, rows, z, vocabulary, b, lse, upstream, counted,
                                 factors, column_sums);
      add_columns_kernel<<<host::blocks_for(vocabulary, kThreads), kThreads, 0,
                           host::counted(s)>>>(vocabulary, ranges, column_sums, first == 0,
                                               column_total);
    }
    if (!dx && !dweight) continue;
    Planes dz;
    by_row(rows, vocabulary, [&](auto block, int grid) {
      constexpr bool kBlock = decltype(block)::value;
      if constexpr (sizeof(T) == 2) {
        dz.ld = static_cast<int>(round_to(vocabulary, 8));
        dz.data = ws + plan.dz;
        dz.rows = dz.plane_rows = rows;
        row_slope_kernel<T, T, kBlock><<<grid, kThreads, 0, host::counted(s)>>>(
            r, first, rows, z, vocabulary, b, lse, upstream, counted, factors,
            static_cast<T*>(dz.data), dz.ld);
      } else {
        row_slope_kernel<T, float, kBlock><<<grid, kThreads, 0, host::counted(s)>>>(
            r, first, rows, z, vocabulary, b, lse, upstream, counted, factors, z, vocabulary);
      }
    });
    if constexpr (sizeof(T) == 4) dz = split<T>(z, rows, vocabulary, ws + plan.dz_planes, s);
    if (dx) {
      ProductParams p{};
      p.m = rows, p.k = vocabulary, p.n = k;
      use_planes(p, dz, w);
      p.k_per_split = vocabulary, p.splits = 1;
      p.out = dx_sums;
      status = launch_product<T, P, false, T, P, true, float, float, kPlain>(p, s);
      if (status != kOk) return status;
      finish<T>(static_cast<long long>(rows) * k, 1, 0, dx_sums, factors,
                static_cast<T*>(dx) + first * k, s);
    }
    if (dweight) {
      ProductParams p{};
      p.m = vocabulary, p.k = rows, p.n = k;
      use_planes(p, dz, xs);
      // a last, shorter piece has fewer splits
      p.k_per_split = plan.split_rows;
      p.splits = static_cast<int>((rows + plan.split_rows - 1) / plan.split_rows);
      p.accumulate = first != 0;
      p.out = weight_sums;
      status = launch_product<T, P, true, T, P, true, float, float, kPlain>(p, s);
      if (status != kOk) return status;
      splits = std::max(splits, p.splits);
    }
  }
  const long long weights = static_cast<long long>(vocabulary) * k;
  if (dweight) finish<T>(weights, splits, weights, weight_sums, factors, dweight, s);
  if (dbias) finish<T>(vocabulary, 1, 0, column_total, factors, dbias, s);
  return host::check_launch("feature_entropy_backward");
}

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

size_t splat_feature_entropy_workspace_bytes(int dtype, long long rows, int k, int vocabulary,
                                             int backward) {
  if (check_entropy(dtype, rows, k, vocabulary, 8, 0) != kOk) return 0;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return plan_entropy<T>(rows, k, vocabulary, backward != 0).bytes;
  });
}

int splat_feature_entropy(int dtype, long long rows, int k, int vocabulary, const void* x,
                          const void* weight, const void* bias, int id_bytes, const void* target,
                          long long ignored, int reduction, float* loss, float* lse,
                          float* counted, void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_entropy(dtype, rows, k, vocabulary, id_bytes, reduction);
  if (bad != kOk) return bad;
  if (!x || !weight || !target || !loss || !workspace)
    return host::fail(kInvalidArgument, "feature_entropy: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument, "feature_entropy: workspace not 16-byte aligned");
  if (workspace_bytes < splat_feature_entropy_workspace_bytes(dtype, rows, k, vocabulary, 0))
    return host::fail(kWorkspaceTooSmall, "feature_entropy: workspace");
  Rows r{rows, vocabulary, id_bytes, reduction, ignored, target, host::device_error_word()};
  if (!r.error) return kCudaError;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return launch_forward<T>(r, k, x, weight, bias, loss, lse, counted,
                             static_cast<char*>(workspace), static_cast<cudaStream_t>(stream));
  });
}

int splat_feature_entropy_backward(int dtype, long long rows, int k, int vocabulary,
                                   const void* x, const void* weight, const void* bias,
                                   int id_bytes, const void* target, long long ignored,
                                   int reduction, const float* lse, const float* counted,
                                   const float* upstream, void* dx, void* dweight, void* dbias,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_entropy(dtype, rows, k, vocabulary, id_bytes, reduction);
  if (bad != kOk) return bad;
  if (!x || !weight || !target || !lse || !upstream || !workspace ||
      (reduction == kMean && !counted) || (dbias && !bias))
    return host::fail(kInvalidArgument, "feature_entropy_backward: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument,
                      "feature_entropy_backward: workspace not 16-byte aligned");
  if (workspace_bytes < splat_feature_entropy_workspace_bytes(dtype, rows, k, vocabulary, 1))
    return host::fail(kWorkspaceTooSmall, "feature_entropy_backward: workspace");
  Rows r{rows, vocabulary, id_bytes, reduction, ignored, target, host::device_error_word()};
  if (!r.error) return kCudaError;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return launch_backward<T>(r, k, x, weight, bias, lse, counted, upstream, dx, dweight, dbias,
                              static_cast<char*>(workspace), static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
