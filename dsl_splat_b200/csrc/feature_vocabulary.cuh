// Tiles of z = x W^T that never reach memory, for 16-bit x and W: what is left of them are the
// rows' softmax statistics, or dz.
//
//   statistics:  top_i = max_j z_ij, sum_i = sum_j exp(z_ij - top_i), z_i,t_i
//   slopes:      dz_ij = u_i (exp(z_ij - lse_i) - [j = t_i]), and its column sums
//
// A pair of blocks (tensor_core.cuh) takes 256 rows x 256 words: per SM, a chunk of 64 k
// is 16 KB of x and 16 KB of W, half of what two blocks on their own would read from the
// L2.  In each block one thread starts the tensor copies, and sixteen epilogue warps read
// the finished accumulators (two of 256 columns, all of the tensor memory), 64 words of 32
// rows each, and give them back before they work on them; the leading block's product warp
// issues.  A pair stays with 256 rows over a range of words, so that a row's running maximum
// and sum stay in a thread's registers; ranges and quarters of the columns leave a
// partial result each, joined in a fixed order.  Exponentials take the
// special-function pipe 2048 cycles a tile, the products 8 a k: the pipe binds below 256
// features, the tensor core above.
#pragma once
#include "feature_pairs.cuh"

namespace splat {
namespace feature {

constexpr int kVocabularyWarps = 16;  // of the epilogue
constexpr int kVocabularyThreads = 32 * kVocabularyWarps + 64;
constexpr float kLog2E = 1.44269504088896341f;

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

enum Reduction : int { kEach = 0, kSum = 1, kMean = 2 };

// Factors of the backward: of u_i on the way into dz, and of the products' results.
struct Factors {
  float in, out;
};
SPLAT_DEV float upstream_of(const Rows& p, long long row, const float* upstream,
                            const float* counted) {
  const float u = upstream[p.reduction == kEach ? row : 0];
  return p.reduction == kMean ? u / *counted : u;
}

// A row's largest logit in units of log 2 so far, and the sum of powers of two relative
// to it.  top is finite (but for rows with infinities), so that logits of minus infinity
// add nothing.
struct Partial {
  float top, sum;
};
constexpr float kLowest = -3.402823466e38f;
SPLAT_DEV Partial join(Partial a, Partial b) {
  const float top = fmaxf(a.top, b.top);  // NaN lies in the sums
  return {top, a.sum * exp2f(a.top - top) + b.sum * exp2f(b.top - top)};
}
SPLAT_DEV float log_sum(Partial s) { return 0.693147180559945309f * (s.top + log2f(s.sum)); }

struct VocabularyParams {
  CUtensorMap x_map, w_map, dz_map;
  Rows rows;           // of all pieces
  long long first;     // row of the piece
  int count;           // its rows
  int k, tile_n;       // 64, 128 or 256 words
  int tiles, row_blocks, splits, tiles_per_split;
  int stages;
  const void* bias;
  // statistics: (splits, tile_n / 64, count), and the labels' logits (count)
  Partial* partials;
  float* label_logits;
  // slopes
  const float *lse, *upstream, *counted;
  const Factors* factors;
  float* column_sums;  // (count / 32 rounded up to whole tiles, vocabulary) or NULL
};

template <class T, bool SLOPES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kVocabularyThreads, 1)
    vocabulary_kernel(const __grid_constant__ VocabularyParams p) {
  extern __shared__ unsigned char dynamic[];
  __shared__ PairBarriers barriers;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const int warp = tc::uniform(threadIdx.x >> 5);
  const uint32_t rank = tc::cluster_rank();
  const int half_n = p.tile_n / 2, groups = p.tile_n / 64;
  const uint32_t stage_bytes = kAPlane + half_n * 128;
  // patches of the epilogue warps, their words' biases, the ring
  const uint32_t bias_at = base + (SLOPES ? kVocabularyWarps * 4096 : 0);
  const uint32_t ring_at = bias_at + kVocabularyWarps * 256;
  const uint32_t tmem = pair_begin(barriers, p.stages, 8 * groups);
  const int items = p.row_blocks * p.splits;
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  bool ok = true;

  if (warp == kVocabularyWarps) {
    if ((threadIdx.x & 31) == 0) {
      PairRing ring(barriers, ring_at, stage_bytes, p.stages, rank);
      for (int item = pair; item < items && ok; item += pairs) {
        const int block = item % p.row_blocks, split = item / p.row_blocks;
        const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
        const int row = block * kPairRows + rank * 128;
        for (int t = split * p.tiles_per_split; t < t1 && ok; ++t)
          for (int k = 0; k < p.k && ok; k += kChunk)
            ok = ring.fill([&](uint32_t at, uint32_t bar) {
              tc::copy_in_pair(at, &p.x_map, k, row, bar);
              tc::copy_in_pair(at + kAPlane, &p.w_map, k, t * p.tile_n + rank * half_n, bar);
            });
      }
      ok = ring.drain() && ok;
    }
  } else if (warp == kVocabularyWarps + 1) {
    if (rank == 0) {
      PairIssue issue(barriers, ring_at, stage_bytes, p.stages, tmem,
                      tc::instruction_pair(!kIsF16<T>, false, false, p.tile_n));
      for (int item = pair; item < items && ok; item += pairs) {
        const int split = item / p.row_blocks;
        const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
        for (int t = split * p.tiles_per_split; t < t1 && ok; ++t)
          ok = issue.template tile<false, false>(p.k);
      }
      ok = issue.drain() && ok;
    }
  } else if (warp < 4 * groups) {
    // a thread to a row, a warp to 64 of the tile's words
    const int lane = threadIdx.x & 31, lane_block = warp & 3, group = warp >> 2;
    const T* bias = static_cast<const T*>(p.bias);
    const int V = p.rows.vocabulary;
    float* own_bias = reinterpret_cast<float*>(
        dynamic + (bias_at - tc::shared_address(dynamic)) + warp * 256);
    const uint32_t patch = base + warp * 4096;
    uint32_t read = 0;  // accumulators
    for (int item = pair; item < items && ok; item += pairs) {
      const int block = item % p.row_blocks, split = item / p.row_blocks;
      const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
      const int row0 = block * kPairRows + static_cast<int>(rank) * 128 + lane_block * 32;
      const int row = row0 + lane;
      const bool here = row < p.count;
      const int label = here ? label_of(p.rows, p.first + row) : -1;
      Partial s{kLowest, 0.0f};
      float less = 0.0f, u = 0.0f;
      if (SLOPES && label >= 0) {
        less = p.lse[p.first + row] * kLog2E;
        u = upstream_of(p.rows, p.first + row, p.upstream, p.counted) * p.factors->in;
      }
      for (int t = split * p.tiles_per_split; t < t1; ++t, ++read) {
        const uint32_t acc = read & 1;
        const int col0 = t * p.tile_n + group * 64;  // of this warp
        const bool with_bias = bias || col0 + 64 > V;
        if (with_bias) {
          // in units of log 2; words behind the last have minus infinity
          __syncwarp();  // the tile before has been read
#pragma unroll
          for (int j = lane; j < 64; j += 32)
            own_bias[j] = col0 + j >= V ? -INFINITY
                          : bias        ? to_float(bias[col0 + j]) * kLog2E
                                        : 0.0f;
          __syncwarp();
        }
        if (!(ok = tc::barrier_wait(tc::shared_address(&barriers.acc_full[acc]), (read >> 1) & 1)))
          break;
        tc::fence_after_sync();
        float v[64];
        tc::tmem_load64(tmem + (lane_block << 21) + acc * 256 + group * 64, v);
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0)
          tc::barrier_arrive_remote(
              tc::address_in(tc::shared_address(&barriers.acc_empty[acc]), 0));
        if (with_bias) {
#pragma unroll
          for (int j = 0; j < 64; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(own_bias + j);
            v[j] = fmaf(v[j], kLog2E, b.x);
            v[j + 1] = fmaf(v[j + 1], kLog2E, b.y);
            v[j + 2] = fmaf(v[j + 2], kLog2E, b.z);
            v[j + 3] = fmaf(v[j + 3], kLog2E, b.w);
          }
        }
        const int at = label - col0;  // of the label among these words
        const bool hit = at >= 0 && at < 64;
        if constexpr (!SLOPES) {
          if (__any_sync(0xffffffffu, hit)) {
            float z = 0.0f;
#pragma unroll
            for (int j = 0; j < 64; ++j) z = j == at ? v[j] : z;
            if (hit) p.label_logits[row] = with_bias ? z * 0.693147180559945309f : z;
          }
          float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int j = 4; j < 64; ++j) most[j & 3] = fmaxf(most[j & 3], v[j]);
          most[0] = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
          if (!with_bias) most[0] *= kLog2E;
          if (most[0] > s.top) {
            s.sum *= exp2f(s.top - most[0]);
            s.top = most[0];
          }
          float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          if (with_bias) {
#pragma unroll
            for (int j = 0; j < 64; ++j) sum[j & 3] += fast_exp2(v[j] - s.top);
          } else {
#pragma unroll
            for (int j = 0; j < 64; ++j) sum[j & 3] += fast_exp2(fmaf(v[j], kLog2E, -s.top));
          }
          s.sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        } else {
          if (with_bias) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = fast_exp2(v[j] - less);
          } else {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = fast_exp2(fmaf(v[j], kLog2E, -less));
          }
          if (__any_sync(0xffffffffu, hit)) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = j == at ? v[j] - 1.0f : v[j];
          }
          // rows that do not count have no gradient, whatever their logits are
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = label < 0 ? 0.0f : v[j] * u;
          if (p.column_sums) {  // before dz is rounded
            float* sums = p.column_sums + static_cast<long long>(row0 / 32) * V + col0 + lane;
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
              const float sum = sum_rows<32>(reinterpret_cast<const float(&)[32]>(v[c]));
              if (row0 < p.count && col0 + c + lane < V) sums[c] = sum;
            }
          }
          // a patch of 32 rows and 64 words for a tensor copy
          if (lane == 0) tc::copies_out_read();
          __syncwarp();
#pragma unroll
          for (int piece = 0; piece < 8; ++piece) {
            const Vec<T, 8> r =
                round_values<T, 8>(reinterpret_cast<const float(&)[8]>(v[piece * 8]));
            store_shared(patch + lane * 128 + ((piece ^ (lane & 7)) << 4),
                         reinterpret_cast<const uint4&>(r));
          }
          tc::fence_async_proxy();
          __syncwarp();
          if (lane == 0 && row0 < p.count && col0 < V)
            tc::copy_out(&p.dz_map, col0, row0, patch);
        }
      }
      if (!SLOPES && here)
        p.partials[static_cast<long long>(split * groups + group) * p.count + row] = s;
    }
    if (SLOPES && lane == 0) tc::copies_out_read();
  }
  pair_end(tmem, ok, p.rows.error);
}

}  // namespace feature
}  // namespace splat
