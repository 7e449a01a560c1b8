// Tiles of z = x W^T that never reach memory, for 16-bit x and W: what is left of them are the
// rows' softmax statistics, or dz.
//
//   statistics:  top_i = max_j z_ij, sum_i = sum_j exp(z_ij - top_i), z_i,t_i
//   slopes:      dz_ij = u_i (exp(z_ij - lse_i) - [j = t_i]), and its column sums
//
// A pair of blocks (tensor_core.cuh) takes 256 rows x 256 words: per SM, a chunk of 64 k
// is 16 KB of x and 16 KB of W, half of what two blocks on their own would read from the
// L2.  In each block one thread starts the tensor copies, and eight epilogue warps read
// the finished accumulators (two of 256 columns, all of the tensor memory); the leading
// block's product warp issues.  A pair stays with 256 rows over a range of words, so that
// a row's running maximum and sum stay in a thread's registers; ranges and column halves
// leave a partial result each, joined in a fixed order.  Exponentials take the
// special-function pipe 2048 cycles a tile, the products 8 a k: the pipe binds below 256
// features, the tensor core above.
#pragma once
#include "feature_product.cuh"

namespace splat {
namespace feature {

constexpr int kPairRows = 256, kPairThreads = 320;  // eight epilogue warps, copies, products
constexpr int kPairStages = 8;
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
  int k, tile_n;       // 128 or 256 words
  int tiles, row_blocks, splits, tiles_per_split;
  int stages;
  const void* bias;
  // statistics: (splits, 2, count), and the labels' logits (count)
  Partial* partials;
  float* label_logits;
  // slopes
  const float *lse, *upstream, *counted;
  const Factors* factors;
  float* column_sums;  // (count / 32 rounded up to whole tiles, vocabulary) or NULL
};

template <class T, bool SLOPES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    vocabulary_kernel(const __grid_constant__ VocabularyParams p) {
  extern __shared__ unsigned char dynamic[];
  __shared__ alignas(8) unsigned long long full[kPairStages], empty[kPairStages], acc_full[2],
      acc_empty[2], drained;
  __shared__ uint32_t tmem_base;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const int warp = tc::uniform(threadIdx.x >> 5);
  const uint32_t rank = tc::cluster_rank();
  const int half_n = p.tile_n / 2;
  const uint32_t stage_bytes = 128 * 128 + half_n * 128;
  // patches of the epilogue warps, their words' biases, the ring
  const uint32_t bias_at = base + (SLOPES ? 8 * 8192 : 0), ring = bias_at + 4096;
  const int chunks = (p.k + 63) / 64;
  constexpr uint32_t kColumns = 512;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      tc::barrier_init(tc::shared_address(&full[i]), 1);
      tc::barrier_init(tc::shared_address(&empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::barrier_init(tc::shared_address(&acc_full[i]), 1);
      tc::barrier_init(tc::shared_address(&acc_empty[i]), 16);  // epilogue warps of the pair
    }
    tc::barrier_init(tc::shared_address(&drained), 1);
    tc::barrier_init_fence();
  }
  if (warp == 0) tc::tmem_alloc_pair(tc::shared_address(&tmem_base), kColumns);
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = tc::uniform(tmem_base);
  const int items = p.row_blocks * p.splits;
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  bool ok = true;

  if (warp == 8) {
    // ---- copies
    if ((threadIdx.x & 31) == 0) {
      int stage = 0, started = 0;
      uint32_t parity = 1;  // a fresh barrier's previous phase counts as complete
      for (int item = pair; item < items && ok; item += pairs) {
        const int block = item % p.row_blocks, split = item / p.row_blocks;
        const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
        const int row = block * kPairRows + rank * 128;
        for (int t = split * p.tiles_per_split; t < t1 && ok; ++t)
          for (int c = 0; c < chunks; ++c) {
            if (!(ok = tc::barrier_wait(tc::shared_address(&empty[stage]), parity))) break;
            const uint32_t at = ring + stage * stage_bytes;
            // both blocks' copies are told to the leading one's barrier
            const uint32_t own = tc::shared_address(&full[stage]);
            if (rank == 0) tc::barrier_expect(own, 2 * stage_bytes);
            const uint32_t bar = tc::address_in(own, 0);
            tc::copy_in_pair(at, &p.x_map, c * 64, row, bar);
            tc::copy_in_pair(at + 128 * 128, &p.w_map, c * 64, t * p.tile_n + rank * half_n, bar);
            started = max(started, stage + 1);
            if (++stage == p.stages) stage = 0, parity ^= 1;
          }
      }
      // no copy of either block is in flight past the pair's last barrier, also after a
      // wait that ran out: parity ^ 1 is the phase of the ring's current round, parity the
      // last one's
      if (rank == 0)
        for (int i = 0; i < started; ++i)
          ok = tc::barrier_wait_pair(tc::shared_address(&full[i]),
                                     i < stage ? parity ^ 1 : parity) && ok;
    }
  } else if (warp == 9) {
    // ---- products
    if (rank == 0) {
      const uint32_t lead = tc::elected();
      const uint32_t instruction = tc::instruction_pair(!kIsF16<T>, false, false, p.tile_n);
      int stage = 0;
      uint32_t parity = 0, n = 0;  // accumulators filled
      for (int item = pair; item < items && ok; item += pairs) {
        const int split = item / p.row_blocks;
        const int t1 = min((split + 1) * p.tiles_per_split, p.tiles);
        for (int t = split * p.tiles_per_split; t < t1 && ok; ++t, ++n) {
          const uint32_t acc = n & 1;
          if (!(ok = tc::barrier_wait_pair(tc::shared_address(&acc_empty[acc]),
                                           ((n >> 1) & 1) ^ 1)))
            break;
          tc::fence_after_sync();
          const uint32_t d = tmem + acc * 256;
          for (int c = 0; c < chunks; ++c) {
            if (!(ok = tc::barrier_wait_pair(tc::shared_address(&full[stage]), parity))) break;
            tc::fence_after_sync();
            const uint32_t at = ring + stage * stage_bytes;
            uint64_t a = tc::descriptor_k_major(at), b = tc::descriptor_k_major(at + 128 * 128);
            const int steps = (min(p.k - c * 64, 64) + 15) / 16;
#pragma unroll 4
            for (int s = 0; s < steps; ++s) {
              tc::mma_pair(lead, d, a, b, instruction, c > 0 || s > 0);
              a += tc::kStepK >> 4;
              b += tc::kStepK >> 4;
            }
            tc::commit_pair(lead, tc::shared_address(&empty[stage]));
            if (++stage == p.stages) stage = 0, parity ^= 1;
          }
          tc::commit_pair(lead, tc::shared_address(&acc_full[acc]));
        }
      }
      // whichever way the loop ended, no product is in flight past this point
      tc::commit_pair(lead, tc::shared_address(&drained));
      ok = tc::barrier_wait(tc::shared_address(&drained), 0) && ok;
    }
  } else {
    // ---- epilogue: a thread to a row, four warps to half of the columns
    const int lane = threadIdx.x & 31, lane_block = warp & 3, half = warp >> 2;
    const T* bias = static_cast<const T*>(p.bias);
    const int V = p.rows.vocabulary;
    float* own_bias = reinterpret_cast<float*>(
        dynamic + (bias_at - tc::shared_address(dynamic)) + warp * 512);
    uint32_t n = 0;       // accumulators read
    uint32_t patches = 0;  // written
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
      for (int t = split * p.tiles_per_split; t < t1; ++t, ++n) {
        const uint32_t acc = n & 1;
        const int col0 = t * p.tile_n + half * half_n;  // of this warp
        const bool with_bias = bias || col0 + half_n > V;
        if (with_bias) {
          // in units of log 2; words behind the last have minus infinity
          __syncwarp();  // the tile before has been read
          for (int j = lane; j < half_n; j += 32)
            own_bias[j] = col0 + j >= V ? -INFINITY
                          : bias        ? to_float(bias[col0 + j]) * kLog2E
                                        : 0.0f;
          __syncwarp();
        }
        if (!(ok = tc::barrier_wait(tc::shared_address(&acc_full[acc]), (n >> 1) & 1))) break;
        tc::fence_after_sync();
        for (int c = 0; c < half_n; c += 32) {
          float v[32];
          tc::tmem_load32(tmem + (lane_block << 21) + acc * 256 + half * half_n + c, v);
          if (with_bias) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 b = *reinterpret_cast<const float4*>(own_bias + c + j);
              v[j] = fmaf(v[j], kLog2E, b.x);
              v[j + 1] = fmaf(v[j + 1], kLog2E, b.y);
              v[j + 2] = fmaf(v[j + 2], kLog2E, b.z);
              v[j + 3] = fmaf(v[j + 3], kLog2E, b.w);
            }
          }
          const int at = label - (col0 + c);  // of the label among these words
          const bool hit = at >= 0 && at < 32;
          if constexpr (!SLOPES) {
            if (__any_sync(0xffffffffu, hit)) {
              float z = 0.0f;
#pragma unroll
              for (int j = 0; j < 32; ++j) z = j == at ? v[j] : z;
              if (hit) p.label_logits[row] = with_bias ? z * 0.693147180559945309f : z;
            }
            float most = v[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) most = fmaxf(most, v[j]);
            if (!with_bias) most *= kLog2E;
            if (most > s.top) {
              s.sum *= exp2f(s.top - most);
              s.top = most;
            }
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (with_bias) {
#pragma unroll
              for (int j = 0; j < 32; ++j) sum[j & 3] += fast_exp2(v[j] - s.top);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) sum[j & 3] += fast_exp2(fmaf(v[j], kLog2E, -s.top));
            }
            s.sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          } else {
            if (with_bias) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = fast_exp2(v[j] - less);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = fast_exp2(fmaf(v[j], kLog2E, -less));
            }
            if (__any_sync(0xffffffffu, hit)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = j == at ? v[j] - 1.0f : v[j];
            }
            // rows that do not count have no gradient, whatever their logits are
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = label < 0 ? 0.0f : v[j] * u;
            // a patch of 32 rows and 64 words for a tensor copy, in two steps
            const uint32_t patch = base + warp * 8192 + (patches & 1) * 4096;
            if (!(c & 32)) {
              if (lane == 0) tc::copies_out_read_but<1>();
              __syncwarp();
            }
#pragma unroll
            for (int piece = 0; piece < 4; ++piece) {
              const Vec<T, 8> r = round_values<T, 8>(reinterpret_cast<const float(&)[8]>(v[piece * 8]));
              const uint32_t to = patch + lane * 128 +
                                  ((((c & 32) >> 3) + piece) ^ (lane & 7)) * 16;
              const uint4& w = reinterpret_cast<const uint4&>(r);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w.x),
                           "r"(w.y), "r"(w.z), "r"(w.w)
                           : "memory");
            }
            if (c & 32) {
              tc::fence_async_proxy();
              __syncwarp();
              if (lane == 0) {
                // patches without a copy count too, see copies_out_read_but
                if (row0 < p.count && col0 + c - 32 < V)
                  tc::copy_out(&p.dz_map, col0 + c - 32, row0, patch);
                else
                  tc::copy_out_none();
              }
              ++patches;
            }
            if (p.column_sums) {  // before dz is rounded
              const float sum = sum_rows<32>(v);
              if (row0 < p.count && col0 + c + lane < V)
                p.column_sums[static_cast<long long>(row0 / 32) * V + col0 + c + lane] = sum;
            }
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0)
          tc::barrier_arrive_remote(tc::address_in(tc::shared_address(&acc_empty[acc]), 0));
      }
      if (!SLOPES && here)
        p.partials[static_cast<long long>(split * 2 + half) * p.count + row] = s;
    }
    if (SLOPES && lane == 0) tc::copies_out_read();
  }
  if (!ok) atomicCAS(p.rows.error, 0, kDeviceTimeout);
  tc::fence_before_sync();
  __syncthreads();
  __syncwarp();
  tc::cluster_sync();
  if (warp == 0) tc::tmem_free_pair(tmem, kColumns);
}

}  // namespace feature
}  // namespace splat
