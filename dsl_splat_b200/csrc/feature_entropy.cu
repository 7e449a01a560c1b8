// Softmax cross entropy of a linear head over a vocabulary:
//
//   z = x W^T + b,  l_i = log sum_j exp z_ij - z_i,t_i
//   dz_ij = u_i (exp(z_ij) / sum_k exp z_ik - [j = t_i])
//   dx = dz W,  dW = dz^T x,  db = sum_i dz_i
//
// The logits are never kept.  They never leave the chip (feature_vocabulary.cuh) but those of
// rows so long that they take several accumulators, which are formed for a piece of the
// rows at a time.  The backward forms them again, and dz for a piece of the rows.  u_i is
// the upstream gradient of row i's loss (divided by the number of rows that count for their
// mean) and 0 for the others.
//
// dz is held in T for the products.  A u that all rows share is multiplied to the products'
// fp32 results before their rounding; of u_i of their own dz is taken relative to the power of two
// that is not below any |u_i|, and the results are multiplied by that.  float16, whose
// smallest value would otherwise swallow the tail of a large vocabulary, has 2^15 times dz.
//
// What dz's rounding costs, as relative 2-norms of dx's error over those of its own rounding
// (bf16 1.66e-3, fp16 2.07e-4; 2048 rows x 64 over 512 words, logits of deviation 4; dW is
// alike):
//
//                                  labels: random   drawn from the softmax   the largest logit
//   one value, u shared                     1.12            1.34                   1.45
//   one value, u of the rows' own           1.40            1.45                   1.45
//   two values                              1.00            1.00                   1.00
//
// A shared u takes one: p - 1 of a head that has learnt nothing is nearly -1, whose rounding is
// small, and that of one that has costs as much as dx's own.  Two would take 3550 us instead of
// 2390 (307200 x 64 over 4096 words, bf16, training) and 11900 instead of 7700 (65536 x
// 512 over 32768).  u of the rows' own takes two, because every label's dz has the full
// rounding there.  Layers beyond on_chip() keep the one.
#include <algorithm>

#include "feature_join.cuh"
#include "feature_launch.cuh"
#include "feature_vocabulary.cuh"
#include "splat200.h"

namespace splat {
namespace feature {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// ---- softmax statistics ------------------------------------------------------------

// Partial results of fp32 logits, whose top is the logit itself: its rounding to units of
// log 2 would cost digits of the exponentials.
SPLAT_DEV void take(Partial& s, float z) {
  if (z > s.top) {
    s.sum = s.sum * expf(s.top - z) + 1.0f;
    s.top = z;
  } else {  // NaN compares false and comes in here
    s.sum += expf(z - s.top);
  }
}
SPLAT_DEV Partial join_logits(Partial a, Partial b) {
  const float top = fmaxf(a.top, b.top);  // NaN lies in the sums
  return {top, a.sum * expf(a.top - top) + b.sum * expf(b.top - top)};
}

// Rows of logits (fp32, ld apart) -> moments and losses; a warp or a block to a row.
template <class T, bool BLOCK>
__global__ void __launch_bounds__(kThreads)
    row_loss_kernel(const Rows p, long long first, int rows, const float* z, int ld,
                    const T* bias, Partial* moments, float* loss) {
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31, lanes = BLOCK ? kThreads : 32;
  const int r = BLOCK ? blockIdx.x : blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const float* from = z + static_cast<long long>(r) * ld;
  Partial s{kLowest, 0.0f};
  for (int j = lane; j < p.vocabulary; j += lanes)
    take(s, from[j] + (bias ? to_float(bias[j]) : 0.0f));
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const Partial other{__shfl_xor_sync(0xffffffffu, s.top, o),
                        __shfl_xor_sync(0xffffffffu, s.sum, o)};
    s = join_logits(s, other);
  }
  if constexpr (BLOCK) {
    __shared__ Partial all[kWarps];
    if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = s;
    __syncthreads();
    s = all[0];
    for (int w = 1; w < kWarps; ++w) s = join_logits(s, all[w]);
  }
  if (lane != 0) return;
  moments[first + r] = s;
  // the logits' difference first: of a label that is the largest it is 0
  const int t = label_of(p, first + r);
  loss[first + r] =
      t < 0 ? 0.0f : s.top - (from[t] + (bias ? to_float(bias[t]) : 0.0f)) + logf(s.sum);
}

// The partial results of vocabulary_kernel -> moments and losses.
__global__ void __launch_bounds__(kThreads)
    join_partials_kernel(const Rows p, int partials, const Partial* from,
                         const float* label_logits, Partial* moments, float* loss) {
  const long long row = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x;
  if (row >= p.rows) return;
  Partial s = from[row];
#pragma unroll 4
  for (int i = 1; i < partials; ++i) s = join(s, from[i * p.rows + row]);
  moments[row] = s;
  // the logits' difference first, as the exponentials took it
  loss[row] = label_of(p, row) < 0 ? 0.0f
                                   : 0.693147180559945309f *
                                         (log2f(s.sum) - fmaf(label_logits[row], kLog2E, -s.top));
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

// The factors: of rows' own u the power of two that is not below any finite one's
// magnitude, which one block looks for (19 us of 307200 rows, 203 of 4 million).
__global__ void __launch_bounds__(1024)
    factors_kernel(long long rows, int reduction, const float* upstream, const float* counted,
                   float within, Factors* factors) {
  if (reduction != kEach) {
    if (threadIdx.x) return;
    factors->in = within;
    factors->out = (reduction == kMean ? *upstream / *counted : *upstream) / within;
    return;
  }
  uint32_t most = 0;
  for (long long i = threadIdx.x; i < rows; i += 1024) {
    const uint32_t bits = __float_as_uint(upstream[i]) & 0x7fffffffu;
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

// Logits -> dz of TO, rows ld_out apart; a warp or a block to a row.  May be in place.
template <class T, class TO, bool BLOCK>
__global__ void __launch_bounds__(kThreads)
    row_slope_kernel(const Rows p, long long first, int rows, const float* z, int ld,
                     const T* bias, const Partial* moments, const float* upstream,
                     const Factors* factors, TO* dz, int ld_out) {
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31, lanes = BLOCK ? kThreads : 32;
  const int r = BLOCK ? blockIdx.x : blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const float* from = z + static_cast<long long>(r) * ld;
  TO* to = dz + static_cast<long long>(r) * ld_out;
  const int t = label_of(p, first + r);
  const float u = t < 0 ? 0.0f : upstream_of(p, first + r, upstream, factors);
  const Partial s = moments[first + r];
  const float factor = u / s.sum;
  for (int j = lane; j < ld_out; j += lanes) {
    float v = 0.0f;
    if (t >= 0 && j < p.vocabulary) {
      v = expf(from[j] + (bias ? to_float(bias[j]) : 0.0f) - s.top) * factor;
      if (j == t) v -= u;
    }
    to[j] = from_float<TO>(v);
  }
}

// Column sums of dz's values before their rounding, over ranges of 256 rows.
constexpr int kSumRows = 256;
template <class T>
__global__ void __launch_bounds__(kThreads)
    column_slopes_kernel(const Rows p, long long first, int rows, const float* z, int ld,
                         const T* bias, const Partial* moments, const float* upstream,
                         const Factors* factors, float* sums) {
  const int j = blockIdx.x * kThreads + threadIdx.x;
  if (j >= p.vocabulary) return;
  const int begin = blockIdx.y * kSumRows, end = min(begin + kSumRows, rows);
  const float b = to_float(bias[j]);
  float sum = 0.0f;
  for (int r = begin; r < end; ++r) {
    const int t = label_of(p, first + r);
    if (t < 0) continue;
    const Partial s = moments[first + r];
    const float u = upstream_of(p, first + r, upstream, factors);
    const float v = expf(z[static_cast<long long>(r) * ld + j] + b - s.top) * (u / s.sum);
    sum += j == t ? v - u : v;
  }
  sums[static_cast<long long>(blockIdx.y) * p.vocabulary + j] = sum;
}
// Adds a piece's ranges to the sums of the pieces before: 32 threads to a column.
constexpr int kAddThreads = 32;
__global__ void __launch_bounds__(32 * kAddThreads)
    add_columns_kernel(int vocabulary, int ranges, const float* sums, bool begin, float* total) {
  const int j = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.0f;
  if (j < vocabulary) {
#pragma unroll 8
    for (int r = threadIdx.y; r < ranges; r += kAddThreads)
      sum += sums[static_cast<long long>(r) * vocabulary + j];
  }
  __shared__ float all[kAddThreads][32];
  all[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y || j >= vocabulary) return;
  sum = begin ? 0.0f : total[j];
#pragma unroll
  for (int w = 0; w < kAddThreads; ++w) sum += all[w][threadIdx.x];
  total[j] = sum;
}
void add_columns(int vocabulary, int ranges, const float* sums, bool begin, float* total,
                 cudaStream_t s) {
  add_columns_kernel<<<host::blocks_for(vocabulary, 32), dim3(32, kAddThreads), 0,
                       host::counted(s)>>>(vocabulary, ranges, sums, begin, total);
}

// What dW is formed of: x without the rows that do not count, which may hold infinities and
// NaN (0 times them would reach every word; 20 us of 2410 for 307200 x 64 bf16).  `from`:
// rows of 16-byte pieces, which are copied; or NULL: planes of parts, in place.
__global__ void __launch_bounds__(kThreads)
    keep_counted_kernel(const Rows p, long long first, int rows, int pieces, const uint4* from,
                        int parts, long long plane_pieces, uint4* to) {
  // a piece's values are below 2^30 (plan_entropy)
  const uint32_t i = blockIdx.x * static_cast<uint32_t>(kThreads) + threadIdx.x;
  const int row = static_cast<int>(i / static_cast<uint32_t>(pieces));
  if (row >= rows) return;
  const bool counts = label_of(p, first + row) >= 0;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if (from) to[i] = counts ? from[i] : zero;
  else if (!counts)
    for (int part = 0; part < parts; ++part) to[part * plane_pieces + i] = zero;
}

// fp32 sums (of several splits, `stride` values apart) times the factor, rounded; V of
// them to an access.  columns: of dx's rows, of which those that do not count get zeros whatever
// W and the factor are; 0 for sums over rows, of which those of nothing are 0 for any factor.
template <class T, int V>
__global__ void __launch_bounds__(kThreads)
    finish_kernel(long long count, int splits, long long stride, const float* from,
                  const Factors* factors, const Rows p, long long first, int columns, T* to) {
  const float factor = factors->out;
  const long long step = static_cast<long long>(kThreads) * gridDim.x * V;
  for (long long i = (blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x) * V; i < count;
       i += step) {
    float sum[V] = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const Vec<float, V> v = *reinterpret_cast<const Vec<float, V>*>(from + s * stride + i);
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] += v.v[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float plain = sum[k];
      sum[k] *= factor;
      // rows that do not count have sums of 0, or of 0 times what W has
      if (!isfinite(sum[k]) &&
          (columns ? label_of(p, first + (i + k) / columns) < 0 : plain == 0.0f))
        sum[k] = 0.0f;
    }
    *reinterpret_cast<Vec<T, V>*>(to + i) = round_values<T, V>(sum);
  }
}
template <class T>
void finish(long long count, int splits, long long stride, const float* from,
            const Factors* factors, void* to, cudaStream_t s, const Rows& rows = {},
            long long first = 0, int columns = 0) {
  const bool vector = count % 4 == 0 && stride % 4 == 0 && host::aligned(to, 4 * sizeof(T));
  const int per_block = kThreads * (vector ? 4 : 1);
  const unsigned grid = static_cast<unsigned>(
      std::min<long long>((count + per_block - 1) / per_block, 1LL << 30));
  auto* kernel = vector ? finish_kernel<T, 4> : finish_kernel<T, 1>;
  kernel<<<grid, kThreads, 0, host::counted(s)>>>(count, splits, stride, from, factors, rows,
                                                  first, columns, static_cast<T*>(to));
}

// ---- launching -----------------------------------------------------------------------

constexpr int kMostVocabulary = 1 << 20;
constexpr long long kMostRows = 1 << 29;  // three planes of them have 2^31 rows at most
constexpr long long kPieceBytes = 1LL << 30;

// Whether the logits stay on the chip: their sums take one accumulator.
template <class T>
bool on_chip(int k) {
  return k <= (sizeof(T) == 2 ? kMostAdditions * 16 : kExactSum);
}

// The rows of a piece, and where its parts lie in the workspace.
struct EntropyPlan {
  bool on_chip;
  int piece;
  PairSplits dx_splits, dw_splits;
  // of vocabulary_kernel
  int tile_n, tiles, ranges, tiles_per_range;
  size_t logits, dz, x_planes, w_planes, weight_sums, column_sums, column_total, dx, losses,
      moments, loss_sums, factors, partials, label_logits, bytes;
};

// Ranges of words that make the busiest pair of blocks take the fewest tiles, a third of a
// tile for each range's start among them.
int word_ranges(int row_blocks, int tiles) {
  const int pairs = std::max(1, host::sm_count() / 2);
  int best = 1;
  double least = 1e30;
  for (int n = 1; n <= std::min(tiles, 64); ++n) {
    const int per = (tiles + n - 1) / n;
    const long long rounds = (static_cast<long long>(row_blocks) * n + pairs - 1) / pairs;
    const double cost = rounds * (per + 0.3);
    if (cost < least * 0.99) least = cost, best = n;
  }
  return best;
}

// What a workspace is for.
enum Purpose : int { kForwardLoss = 0, kSharedUpstream = 1, kOwnUpstreams = 2 };
int purpose_of(int reduction) { return reduction == kEach ? kOwnUpstreams : kSharedUpstream; }
// Parts of dz.
template <class T>
constexpr int dz_parts(bool each) {
  return sizeof(T) == 4 ? 3 : each ? 2 : 1;
}

template <class T>
EntropyPlan plan_entropy(long long rows, int k, int vocabulary, int purpose) {
  constexpr int P = kOperandParts<T>;
  const bool backward = purpose != kForwardLoss, each = purpose == kOwnUpstreams;
  EntropyPlan plan{};
  plan.on_chip = on_chip<T>(k);
  const int unit = plan.on_chip ? kPairRows : kTileRows;
  long long piece;
  if (plan.on_chip && !backward) {
    piece = rows;
  } else {
    // bytes of a row's logits, or of its dz, and of its dx before the rounding
    const long long slopes = plan.on_chip ? 2LL * dz_parts<T>(each) : 4LL;
    const long long row = std::max(vocabulary * slopes, 4LL * k);
    piece = std::max(1LL, kPieceBytes / row / unit) * unit;
    piece = std::min({piece, rows, 1LL << 23});  // 65535 ranges of 256 rows, and below
  }
  plan.piece = static_cast<int>(piece);
  plan.tile_n = pair_tile_n<P>(vocabulary);
  plan.tiles = (vocabulary + plan.tile_n - 1) / plan.tile_n;
  plan.ranges = word_ranges(static_cast<int>((piece + kPairRows - 1) / kPairRows), plan.tiles);
  plan.tiles_per_range = (plan.tiles + plan.ranges - 1) / plan.ranges;
  plan.ranges = (plan.tiles + plan.tiles_per_range - 1) / plan.tiles_per_range;
  const auto take = [&](size_t n) {
    const size_t at = plan.bytes;
    plan.bytes += (n + 255) / 256 * 256;
    return at;
  };
  plan.factors = take(sizeof(Factors));
  plan.loss_sums = take(sizeof(LossSum) * kLossBlocks);
  if (!plan.on_chip) plan.logits = take(4ull * piece * vocabulary);
  // 16-bit rows that lie well need no planes, which their address decides; those of x have a
  // copy for dW
  plan.x_planes = take(sizeof(T) == 2 && k % 8 == 0 && !backward ? 0 : plane_bytes<T>(piece, k));
  plan.w_planes = take(sizeof(T) == 2 && k % 8 == 0 ? 0 : plane_bytes<T>(vocabulary, k));
  if (!backward) {
    plan.moments = take(sizeof(Partial) * rows);
    plan.losses = take(4ull * rows);
    if (plan.on_chip) {
      plan.partials = take(kVocabularyParts * static_cast<size_t>(plan.ranges) * rows *
                           sizeof(Partial));
      plan.label_logits = take(4ull * rows);
    }
    return plan;
  }
  plan.dz = take(2ull * dz_parts<T>(each) * round_to(piece, 64) * round_to(vocabulary, 8));
  // ranges of words for dx and of rows for dW, whose sums are joined
  if (plan.on_chip) {
    const long long dx_tiles = pair_tiles<P>(piece, k), dw_tiles = pair_tiles<P>(vocabulary, k);
    const auto split = [&](auto parts) {
      constexpr int DZ = decltype(parts)::value;
      plan.dx_splits = pair_splits<DZ, P>(dx_tiles, vocabulary);
      plan.dw_splits = pair_splits<DZ, P>(dw_tiles, piece);
    };
    if (each) split(std::integral_constant<int, dz_parts<T>(true)>{});
    else split(std::integral_constant<int, dz_parts<T>(false)>{});
  } else {
    const long long tiles = ((vocabulary + 127LL) / 128) * ((k + 127) / 128);
    const long long wanted = std::max(1LL, 2LL * host::sm_count() / tiles);
    const long long most = std::min(wanted, (piece + 511) / 512);
    plan.dx_splits = {1, vocabulary};
    plan.dw_splits.k = round_to((piece + most - 1) / most, kChunk);
    plan.dw_splits.count = static_cast<int>((piece + plan.dw_splits.k - 1) / plan.dw_splits.k);
  }
  plan.dx = take(4ull * plan.dx_splits.count * piece * k);
  plan.weight_sums = take(4ull * plan.dw_splits.count * vocabulary * k);
  plan.column_sums = take(plan.on_chip
                              ? 4ull * round_to(piece, kPairRows) / 32 * vocabulary
                              : 4ull * ((piece + kSumRows - 1) / kSumRows) * vocabulary);
  plan.column_total = take(4ull * vocabulary);
  return plan;
}

// What both launches of vocabulary_kernel share.
template <class T, int DZ>
int launch_vocabulary(VocabularyParams& p, const EntropyPlan& plan, const Rows& r, long long first,
                      int count, int k, const Planes& x, const Planes& w, const void* bias,
                      cudaStream_t s) {
  p.rows = r, p.first = first, p.count = count, p.k = k, p.bias = bias;
  p.tile_n = plan.tile_n, p.tiles = plan.tiles;
  p.row_blocks = static_cast<int>((count + static_cast<long long>(kPairRows) - 1) / kPairRows);
  p.splits = plan.ranges, p.tiles_per_split = plan.tiles_per_range;
  constexpr int P = kOperandParts<T>;
  p.x_plane_rows = x.plane_rows, p.w_plane_rows = w.plane_rows;
  if (!make_operand_map<T, P, false>(p.x_map, x, count, k, 128) ||
      !make_operand_map<T, P, false>(p.w_map, w, r.vocabulary, k, plan.tile_n / 2))
    return host::fail(kInvalidArgument, "feature_entropy: operand maps");
  const int fixed = 1024 + (DZ ? kVocabularyWarps * 4096 : 0);
  const int stage = P * (kAPlane + plan.tile_n / 2 * 128);
  p.stages = std::min(kPairStages, (kOneBlockBytes - fixed) / stage);
  constexpr auto* kernel = vocabulary_kernel<T, P, DZ>;
  if (!host::allow_shared<kernel>())
    return host::check_launch("feature_entropy: shared memory");
  const long long items = static_cast<long long>(p.row_blocks) * p.splits;
  if (items >= 1LL << 31) return host::fail(kTooLarge, "feature_entropy: too many tiles");
  const int pairs = static_cast<int>(std::min<long long>(items, host::sm_count() / 2));
  kernel<<<2 * pairs, kVocabularyThreads, fixed + p.stages * stage, host::counted(s)>>>(p);
  return host::check_launch("feature_entropy");
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

// keep_counted_kernel of a piece's x, whose planes lie in the workspace or are x itself.
template <class T>
Planes keep_counted(const Rows& r, long long first, int rows, const Planes& xs, void* to,
                    cudaStream_t s) {
  const bool copies = xs.data != to;
  const int pieces = xs.ld / 8;
  keep_counted_kernel<<<host::blocks_for(static_cast<long long>(rows) * pieces, kThreads),
                        kThreads, 0, host::counted(s)>>>(
      r, first, rows, pieces, copies ? static_cast<const uint4*>(xs.data) : nullptr,
      kOperandParts<T>, static_cast<long long>(xs.plane_rows) * pieces, static_cast<uint4*>(to));
  Planes kept = xs;
  kept.data = to;
  return kept;
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
  if (k > 65535 || vocabulary > kMostVocabulary || rows > kMostRows)
    return host::fail(kTooLarge, "feature_entropy: too many rows, inputs or words");
  return kOk;
}

// Whether 16-bit rows that need no planes lie as the workspace's size takes them to, and
// the bias as it is read.
bool lies_well(int dtype, int k, const void* x, const void* weight, const void* bias) {
  return host::aligned(bias, 16) &&
         (dtype == kF32 || k % 8 || (host::aligned(x, 16) && host::aligned(weight, 16)));
}

template <class T>
int launch_forward(const Rows& r, int k, const void* x, const void* weight, const void* bias,
                   float* loss, Partial* moments, float* counted, char* ws, cudaStream_t s) {
  const int vocabulary = r.vocabulary;
  const EntropyPlan plan = plan_entropy<T>(r.rows, k, vocabulary, kForwardLoss);
  float* z = reinterpret_cast<float*>(ws + plan.logits);
  if (!moments) moments = reinterpret_cast<Partial*>(ws + plan.moments);
  float* each = r.reduction == kEach ? loss : reinterpret_cast<float*>(ws + plan.losses);
  const Planes w = split<T>(weight, vocabulary, k, ws + plan.w_planes, s);
  for (long long first = 0; first < r.rows; first += plan.piece) {
    const int rows = static_cast<int>(std::min<long long>(plan.piece, r.rows - first));
    const Planes xs = split<T>(static_cast<const T*>(x) + first * k, rows, k,
                               ws + plan.x_planes, s);
    if (plan.on_chip) {  // all rows at once
      VocabularyParams p{};
      p.partials = reinterpret_cast<Partial*>(ws + plan.partials);
      p.label_logits = reinterpret_cast<float*>(ws + plan.label_logits);
      const int status = launch_vocabulary<T, 0>(p, plan, r, first, rows, k, xs, w, bias, s);
      if (status != kOk) return status;
      join_partials_kernel<<<host::blocks_for(rows, kThreads), kThreads, 0, host::counted(s)>>>(
          r, kVocabularyParts * plan.ranges, p.partials, p.label_logits, moments, each);
      continue;
    }
    const int status = launch_logits<T>(rows, k, vocabulary, xs, w, z, s);
    if (status != kOk) return status;
    by_row(rows, vocabulary, [&](auto block, int grid) {
      row_loss_kernel<T, decltype(block)::value><<<grid, kThreads, 0, host::counted(s)>>>(
          r, first, rows, z, vocabulary, static_cast<const T*>(bias), moments, each);
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
                    const Partial* moments, const float* counted, const float* upstream, void* dx,
                    void* dweight, void* dbias, char* ws, cudaStream_t s) {
  constexpr int P = kOperandParts<T>;
  const int vocabulary = r.vocabulary;
  const EntropyPlan plan = plan_entropy<T>(r.rows, k, vocabulary, purpose_of(r.reduction));
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
    Planes dz;
    dz.ld = static_cast<int>(round_to(vocabulary, 8));
    dz.data = ws + plan.dz;
    dz.rows = rows;
    const bool each = plan.on_chip && r.reduction == kEach;
    const int parts = dz_parts<T>(each);
    dz.plane_rows = static_cast<int>(parts == 1 ? rows : round_to(rows, 64));
    int status = kOk;
    if (plan.on_chip) {
      VocabularyParams p{};
      p.moments = moments, p.upstream = upstream, p.factors = factors;
      p.dz_plane_rows = dz.plane_rows;
      if (dbias) p.column_sums = column_sums;
      const long long dz_rows = static_cast<long long>(dz.plane_rows) * parts;
      if (!make_map<PairOperand<T>>(p.dz_map, dz.data, dz_rows, vocabulary, dz.ld, 32, 32))
        return host::fail(kInvalidArgument, "feature_entropy_backward: map");
      status = each ? launch_vocabulary<T, dz_parts<T>(true)>(p, plan, r, first, rows, k, xs, w,
                                                              bias, s)
                    : launch_vocabulary<T, dz_parts<T>(false)>(p, plan, r, first, rows, k, xs, w,
                                                               bias, s);
      if (status != kOk) return status;
      if (dbias)
        add_columns(vocabulary, (rows + 31) / 32, column_sums, first == 0, column_total, s);
    }
    if (!plan.on_chip) status = launch_logits<T>(rows, k, vocabulary, xs, w, z, s);
    if (status != kOk) return status;
    if (dbias && !plan.on_chip) {
      const int ranges = (rows + kSumRows - 1) / kSumRows;
      column_slopes_kernel<T>
          <<<dim3(host::blocks_for(vocabulary, kThreads), ranges), kThreads, 0,
             host::counted(s)>>>(r, first, rows, z, vocabulary, b, moments, upstream, factors,
                                 column_sums);
      add_columns(vocabulary, ranges, column_sums, first == 0, column_total, s);
    }
    if (!dx && !dweight) continue;
    if (!plan.on_chip) by_row(rows, vocabulary, [&](auto block, int grid) {
      constexpr bool kBlock = decltype(block)::value;
      if constexpr (sizeof(T) == 2) {
        row_slope_kernel<T, T, kBlock><<<grid, kThreads, 0, host::counted(s)>>>(
            r, first, rows, z, vocabulary, b, moments, upstream, factors,
            static_cast<T*>(dz.data), dz.ld);
      } else {
        row_slope_kernel<T, float, kBlock><<<grid, kThreads, 0, host::counted(s)>>>(
            r, first, rows, z, vocabulary, b, moments, upstream, factors, z, vocabulary);
      }
    });
    if constexpr (sizeof(T) == 4) {
      if (!plan.on_chip) dz = split<T>(z, rows, vocabulary, ws + plan.dz, s);
    }
    if (dx) {
      if (plan.on_chip) {
        status = each ? launch_pairs<T, dz_parts<T>(true), false, true>(
                            rows, k, vocabulary, dz, w, plan.dx_splits, dx_sums, false, s)
                      : launch_pairs<T, dz_parts<T>(false), false, true>(
                            rows, k, vocabulary, dz, w, plan.dx_splits, dx_sums, false, s);
      } else {
        ProductParams p{};
        p.m = rows, p.k = vocabulary, p.n = k;
        use_planes(p, dz, w);
        p.k_per_split = vocabulary, p.splits = 1;
        p.out = dx_sums;
        status = launch_product<T, P, false, T, P, true, float, float, kPlain>(p, s);
      }
      if (status != kOk) return status;
      const long long values = static_cast<long long>(rows) * k;
      finish<T>(values, plan.dx_splits.count, values, dx_sums, factors,
                static_cast<T*>(dx) + first * k, s, r, first, k);
    }
    if (dweight) {
      // a last, shorter piece has fewer splits
      PairSplits dw = plan.dw_splits;
      dw.count = static_cast<int>((rows + dw.k - 1) / dw.k);
      const Planes counted_xs = keep_counted<T>(r, first, rows, xs, ws + plan.x_planes, s);
      if (plan.on_chip) {
        status = each ? launch_pairs<T, dz_parts<T>(true), true, true>(
                            vocabulary, k, rows, dz, counted_xs, dw, weight_sums, first != 0, s)
                      : launch_pairs<T, dz_parts<T>(false), true, true>(
                            vocabulary, k, rows, dz, counted_xs, dw, weight_sums, first != 0, s);
      } else {
        ProductParams p{};
        p.m = vocabulary, p.k = rows, p.n = k;
        use_planes(p, dz, counted_xs);
        p.k_per_split = dw.k, p.splits = dw.count;
        p.accumulate = first != 0;
        p.out = weight_sums;
        status = launch_product<T, P, true, T, P, true, float, float, kPlain>(p, s);
      }
      if (status != kOk) return status;
      splits = std::max(splits, dw.count);
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
  if (backward < kForwardLoss || backward > kOwnUpstreams ||
      check_entropy(dtype, rows, k, vocabulary, 8, 0) != kOk)
    return 0;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return plan_entropy<T>(rows, k, vocabulary, backward).bytes;
  });
}

int splat_feature_entropy(int dtype, long long rows, int k, int vocabulary, const void* x,
                          const void* weight, const void* bias, int id_bytes, const void* target,
                          long long ignored, int reduction, float* loss, float* moments,
                          float* counted, void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_entropy(dtype, rows, k, vocabulary, id_bytes, reduction);
  if (bad != kOk) return bad;
  if (!x || !weight || !target || !loss || !workspace)
    return host::fail(kInvalidArgument, "feature_entropy: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument, "feature_entropy: workspace not 16-byte aligned");
  if (workspace_bytes < splat_feature_entropy_workspace_bytes(dtype, rows, k, vocabulary, 0))
    return host::fail(kWorkspaceTooSmall, "feature_entropy: workspace");
  if (!lies_well(dtype, k, x, weight, bias))
    return host::fail(kInvalidArgument,
                      "feature_entropy: x, weight and bias must be 16-byte aligned");
  Rows r{rows, vocabulary, id_bytes, reduction, ignored, target, host::device_error_word()};
  if (!r.error) return kCudaError;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return launch_forward<T>(r, k, x, weight, bias, loss, reinterpret_cast<Partial*>(moments),
                             counted, static_cast<char*>(workspace),
                             static_cast<cudaStream_t>(stream));
  });
}

int splat_feature_entropy_backward(int dtype, long long rows, int k, int vocabulary,
                                   const void* x, const void* weight, const void* bias,
                                   int id_bytes, const void* target, long long ignored,
                                   int reduction, const float* moments, const float* counted,
                                   const float* upstream, void* dx, void* dweight, void* dbias,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_entropy(dtype, rows, k, vocabulary, id_bytes, reduction);
  if (bad != kOk) return bad;
  if (!x || !weight || !target || !moments || !upstream || !workspace ||
      (reduction == kMean && !counted) || (dbias && !bias))
    return host::fail(kInvalidArgument, "feature_entropy_backward: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument,
                      "feature_entropy_backward: workspace not 16-byte aligned");
  if (workspace_bytes < splat_feature_entropy_workspace_bytes(dtype, rows, k, vocabulary,
                                                              purpose_of(reduction)))
    return host::fail(kWorkspaceTooSmall, "feature_entropy_backward: workspace");
  if (!lies_well(dtype, k, x, weight, bias))
    return host::fail(kInvalidArgument,
                      "feature_entropy_backward: x, weight and bias must be 16-byte aligned");
  Rows r{rows, vocabulary, id_bytes, reduction, ignored, target, host::device_error_word()};
  if (!r.error) return kCudaError;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return launch_backward<T>(r, k, x, weight, bias, reinterpret_cast<const Partial*>(moments),
                              counted, upstream, dx, dweight, dbias,
                              static_cast<char*>(workspace), static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
