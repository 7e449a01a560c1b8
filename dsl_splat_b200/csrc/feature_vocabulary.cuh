// Tiles of z = x W^T that never reach memory: what is left of them are the rows' softmax
// statistics, or dz.
//
//   statistics:  top_i = max_j z_ij, sum_i = sum_j exp(z_ij - top_i), z_i,t_i
//   slopes:      dz_ij = u_i (exp(z_ij - top_i) / sum_i - [j = t_i]), and its column sums
//
// A pair of blocks (tensor_core.cuh) takes 256 rows x 256 words of 16-bit x and W, or 256 x
// 128 of fp32 ones in three parts: per SM, a chunk of 64 k is 16 KB of x and 16 KB of W,
// half of what two blocks on their own would read from the L2.  In each block one thread
// starts the tensor copies, and sixteen epilogue warps read the finished
// accumulators, 32 words of 32 rows at a time, and give them back before they work on the
// last of them; the leading block's product warp issues.  One half of the epilogue takes
// the even tiles and the other the odd ones, so that the one's exponentials run under the
// other's waits and maxima (slopes of 65536 rows and 8192 words 258 to 314 us with 64 to
// 256 bf16 features; 290 to 347 with all warps on each tile; as long at 512).  A pair stays
// with 256 rows over a range of words, so that a row's running maximum and sum stay in a
// thread's registers; ranges and groups of warps leave a partial result each, joined in a
// fixed order.  Exponentials take the special-function pipe 2048 cycles a tile of 256 words,
// the products 8 a k: the pipe binds below 256 features, the tensor core above.
//
// 65536 x 512 bf16 features and 32768 words: statistics 1.41 ms (1560 TFLOP/s, tensor pipe 85 %
// of a piece's cycles), slopes 1.96 (1125, 59 %: 4.3 GB of dz go out beside the
// exponentials).  307200 x 64 and 4096: 540 us (special-function pipe 56 %) and 840 (36 %),
// without a bias 450 and 620: its addition and db's sums take issue slots.  Direct stores of dz
// instead of patches took longer; so did chunks of 64 words, whose registers spill, and
// biases loaded before the logits.
//
// top and sum are kept apart for the slopes: rounded into one logarithm, they would cost
// each probability 2^-24 of that logarithm.
#pragma once
#include "feature_pairs.cuh"

namespace splat {
namespace feature {

// Epilogue warps.  Half of them take a tile: four the rows, two the halves of its words.
constexpr int kVocabularyWarps = 16, kVocabularyThreads = 32 * kVocabularyWarps + 64;
constexpr int kVocabularyParts = 4;  // partial results of a row in a range of words
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

// Factors of the backward: of u_i on the way into dz, and of the products' results.  Where
// all rows have the same u it is left to the results: rounded to 16 bits with each label's
// dz, which is nearly -u before a head has learnt, it would cost all of dx and dW the same error.
struct Factors {
  float in, out;
};
SPLAT_DEV float upstream_of(const Rows& p, long long row, const float* upstream,
                            const Factors* factors) {
  return p.reduction == kEach ? upstream[row] * factors->in : factors->in;
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

struct VocabularyParams {
  CUtensorMap x_map, w_map, dz_map;
  int x_plane_rows, w_plane_rows, dz_plane_rows;  // of operands in parts
  Rows rows;           // of all pieces
  long long first;     // row of the piece
  int count;           // its rows
  int k, tile_n;       // 64, 128 or 256 words
  int tiles, row_blocks, splits, tiles_per_split;
  int stages;
  const void* bias;
  // statistics: (splits, kVocabularyParts, count), and the labels' logits (count)
  Partial* partials;
  float* label_logits;
  // slopes
  const Partial* moments;  // (rows)
  const float* upstream;
  const Factors* factors;
  float* column_sums;  // (count / 32 rounded up to whole tiles, vocabulary) or NULL
};

// 32 logits of a row: those of parts are the sums of two accumulators.
template <int P>
SPLAT_DEV void load_logits(uint32_t from, float (&v)[32]) {
  tc::tmem_load32(from, v);
  if constexpr (P > 1) {
    float low[32];
    tc::tmem_load32(from + 128, low);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] += low[j];
  }
}

// v -> exp(v) 2^-top, in pairs.
SPLAT_DEV void exponentials(float (&v)[32], float top) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    unpack2(fma2(pack2(v[j], v[j + 1]), splat2(kLog2E), splat2(-top)), v[j], v[j + 1]);
    v[j] = fast_exp2(v[j]);
    v[j + 1] = fast_exp2(v[j + 1]);
  }
}

// Adds the biases of 32 words, of which so many exist: the others get minus infinity.
template <class T>
SPLAT_DEV void add_bias(float (&v)[32], const T* bias, int words) {
  if (words >= 32) {
    if (!bias) return;
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 32; j += N) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(bias + j));
      float b[N];
      widen<T, N>(reinterpret_cast<const Vec<T, N>&>(raw), b);
#pragma unroll
      for (int i = 0; i < N; i += 2)
        unpack2(add2(pack2(v[j + i], v[j + i + 1]), pack2(b[i], b[i + 1])), v[j + i],
                v[j + i + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      v[j] = j >= words ? -INFINITY : bias ? v[j] + to_float(bias[j]) : v[j];
  }
}

// The sums over a warp's rows of 32 columns: lane j gets column j's.  Every step halves the
// columns of a lane.  Through shared memory, whose wavefronts they then were most of, the
// slopes of 307200 rows and 4096 words took 955 us instead of 840.
template <int N>
SPLAT_DEV float column_sum(const float (&v)[N]) {
  if constexpr (N == 1) {
    return v[0];
  } else {
    const bool upper = threadIdx.x & (N / 2);
    float half[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float sent = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + N / 2], N / 2);
      half[i] = (upper ? v[i + N / 2] : v[i]) + sent;
    }
    return column_sum(half);
  }
}

// P: parts of x and W; DZ: parts of dz, 0 for the statistics.
template <class T, int P, int DZ>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kVocabularyThreads, 1)
    vocabulary_kernel(const __grid_constant__ VocabularyParams p) {
  constexpr int kEpilogue = kVocabularyWarps;
  constexpr bool SLOPES = DZ > 0;
  extern __shared__ unsigned char dynamic[];
  __shared__ PairBarriers barriers;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const int warp = tc::uniform(threadIdx.x >> 5);
  const uint32_t rank = tc::cluster_rank();
  const int half_n = p.tile_n / 2;
  const uint32_t b_plane = half_n * 128;
  // patches of the epilogue warps, the ring
  const uint32_t ring_at = base + (SLOPES ? kEpilogue * 4096 : 0);
  const uint32_t tmem = pair_begin(barriers, p.stages, kEpilogue);
  const int items = p.row_blocks * p.splits;
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  bool ok = true;

  if (warp == kEpilogue) {
    if ((threadIdx.x & 31) == 0) {
      PairRing ring(barriers, ring_at, P * (kAPlane + b_plane), p.stages, rank);
      for (int item = pair; item < items && ok; item += pairs) {
        const int block = item % p.row_blocks, split = item / p.row_blocks;
        const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
        const int row = block * kPairRows + rank * 128;
        for (int t = split * p.tiles_per_split; t < t1 && ok; ++t)
          for (int k = 0; k < p.k && ok; k += kChunk)
            ok = ring.fill([&](uint32_t at, uint32_t bar) {
              const int word = t * p.tile_n + rank * half_n;
#pragma unroll
              for (int i = 0; i < P; ++i, at += kAPlane)
                tc::copy_in_pair(at, &p.x_map, k, row + i * p.x_plane_rows, bar);
#pragma unroll
              for (int i = 0; i < P; ++i, at += b_plane)
                tc::copy_in_pair(at, &p.w_map, k, word + i * p.w_plane_rows, bar);
            });
      }
      ok = ring.drain() && ok;
    }
  } else if (warp == kEpilogue + 1) {
    if (rank == 0) {
      PairIssue<P, P> issue(barriers, ring_at, b_plane, p.stages, tmem,
                         tc::instruction_pair(!kIsF16<T>, false, false, p.tile_n));
      for (int item = pair; item < items && ok; item += pairs) {
        const int split = item / p.row_blocks;
        const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
        for (int t = split * p.tiles_per_split; t < t1 && ok; ++t)
          ok = issue.template sum<false, false>(p.k);
      }
      ok = issue.drain() && ok;
    }
  } else {
    // a thread to a row; the first eight warps take the even tiles, the others the odd ones
    const int lane = threadIdx.x & 31, lane_block = warp & 3, part = warp >> 2;
    const uint32_t own = part >> 1;
    const int first = (part & 1) * half_n, end = first + half_n;
    const T* bias = static_cast<const T*>(p.bias);
    const int V = p.rows.vocabulary;
    const uint32_t patch_at = base + warp * 4096;
    uint32_t read = 0, patches = 0;  // accumulators; copied out
    for (int item = pair; item < items && ok; item += pairs) {
      const int block = item % p.row_blocks, split = item / p.row_blocks;
      const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
      const int row0 = block * kPairRows + static_cast<int>(rank) * 128 + lane_block * 32;
      const int row = row0 + lane;
      const bool here = row < p.count;
      const int label = here ? label_of(p.rows, p.first + row) : -1;
      Partial s{kLowest, 0.0f};
      float u = 0.0f, factor = 0.0f;
      bool cleared = false;  // some rows' dz is not what 0 times their exponentials gives
      if constexpr (SLOPES) {
        if (here) {
          s = p.moments[p.first + row];
          if (label >= 0) {
            u = upstream_of(p.rows, p.first + row, p.upstream, p.factors);
            factor = u / s.sum;
          }
        }
        // a row that does not count has no gradient, whatever its logits are
        cleared = __any_sync(0xffffffffu, label < 0 && !(here && isfinite(s.top + s.sum)));
      }
      for (int t = split * p.tiles_per_split; t < t1; ++t, ++read) {
        if ((read & 1) != own) continue;
        const uint32_t acc = read & 1;
        if (!(ok = tc::barrier_wait(tc::shared_address(&barriers.acc_full[acc]), (read >> 1) & 1)))
          break;
        tc::fence_after_sync();
        for (int c = first; c < end; c += 32) {
          const int col0 = t * p.tile_n + c;
          float v[32];
          load_logits<P>(tmem + (lane_block << 21) + acc * 256 + c, v);
          if (c + 32 == end) pair_release(barriers, acc);
          if (bias || col0 + 32 > V) add_bias<T>(v, bias ? bias + col0 : nullptr, V - col0);
          const int at = label - col0;  // of the label among these words
          const bool hit = at >= 0 && at < 32;
          if constexpr (!SLOPES) {
            if (__any_sync(0xffffffffu, hit)) {
              float z = 0.0f;
#pragma unroll
              for (int j = 0; j < 32; ++j) z = j == at ? v[j] : z;
              if (hit) p.label_logits[row] = z;
            }
            float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int j = 4; j < 32; ++j) most[j & 3] = fmaxf(most[j & 3], v[j]);
            most[0] = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * kLog2E;
            if (most[0] > s.top) {
              s.sum *= exp2f(s.top - most[0]);
              s.top = most[0];
            }
            exponentials(v, s.top);
            f32x2 sum[4] = {pack2(s.sum, 0.0f), 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 32; j += 2)
              sum[j / 2 & 3] = add2(sum[j / 2 & 3], pack2(v[j], v[j + 1]));
            float a, b;
            unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), a, b);
            s.sum = a + b;
          } else {
            exponentials(v, s.top);
#pragma unroll
            for (int j = 0; j < 32; j += 2)
              unpack2(mul2(pack2(v[j], v[j + 1]), splat2(factor)), v[j], v[j + 1]);
            if (__any_sync(0xffffffffu, hit)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = j == at ? v[j] - u : v[j];
            }
            if (cleared) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = label < 0 ? 0.0f : v[j];
            }
            if (p.column_sums) {  // before dz is rounded
              const float sum = column_sum(v);
              if (row0 < p.count && col0 + lane < V)
                p.column_sums[static_cast<long long>(row0 / 32) * V + col0 + lane] = sum;
            }
            // patches of 32 rows and 32 words for tensor copies, two in turn; planes of
            // parts have zeros in the rows behind the last
#pragma unroll
            for (int i = 0; i < DZ; ++i, ++patches) {
              const Patch<PairOperand<T>> patch{patch_at + (patches & 1) * 2048};
              constexpr bool kLasts[3] = {DZ == 1, DZ == 2, true};
              if (lane == 0) tc::copies_out_read_but<1>();
              __syncwarp();
#pragma unroll
              for (int piece = 0; piece < 4; ++piece) {
                float* o = v + piece * 8;
                uint4 r;
                if constexpr (P == 1) {
                  const Vec<T, 8> rounded =
                      kLasts[i] ? round_values<T, 8>(reinterpret_cast<float(&)[8]>(*o))
                                : take_first<T, 8>(reinterpret_cast<float(&)[8]>(*o));
                  r = reinterpret_cast<const uint4&>(rounded);
                } else {
                  r = kLasts[i] ? make_uint4(take_part<true>(o[0], o[1]),
                                             take_part<true>(o[2], o[3]),
                                             take_part<true>(o[4], o[5]),
                                             take_part<true>(o[6], o[7]))
                                : make_uint4(take_part<false>(o[0], o[1]),
                                             take_part<false>(o[2], o[3]),
                                             take_part<false>(o[4], o[5]),
                                             take_part<false>(o[6], o[7]));
                }
                store_shared(patch.at(lane, piece), r);
              }
              tc::fence_async_proxy();
              __syncwarp();
              if (lane == 0) {
                if (row0 < (DZ == 1 ? p.count : p.dz_plane_rows) && col0 < V)
                  tc::copy_out(&p.dz_map, col0, row0 + i * p.dz_plane_rows, patch.base);
                else
                  tc::copy_out_none();  // counts too
              }
            }
          }
        }
      }
      if (!SLOPES && here)
        p.partials[static_cast<long long>(split * kVocabularyParts + part) * p.count + row] = s;
    }
    if (SLOPES && lane == 0) tc::copies_out_read();
  }
  pair_end(tmem, ok, p.rows.error);
}

}  // namespace feature
}  // namespace splat
