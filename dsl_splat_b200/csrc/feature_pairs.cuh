// C(m, n) = sum_k A(m, k) B(n, k) of 16-bit operands on pairs of blocks (tensor_core.cuh),
// fp32 sums over ranges of k: the long products of a vocabulary's gradients.
//
// A pair takes 256 x tile_n tiles; each of its blocks copies its 128 rows of A and its half
// of B's in chunks of 64 k, half of what a block on its own would read for the same work.
// No accumulator takes more than kMostAdditions (feature_product.cuh).
#pragma once
#include <algorithm>

#include "feature_launch.cuh"

namespace splat {
namespace feature {

constexpr int kPairRows = 256, kPairStages = 8;
constexpr int kPairThreads = 320;  // eight epilogue warps, copies, products

struct PairParams {
  CUtensorMap a_map, b_map;
  int m, n, tile_n, stages;
  long long k, k_per_split;  // k_per_split: a multiple of 64
  int tiles_m, tiles_n, splits;
  float* out;      // (splits, m, n)
  int accumulate;  // onto what is there
  int* error;
};

// The barriers of a pair's ring and accumulators.
struct PairBarriers {
  alignas(8) unsigned long long full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2],
      drained;
  uint32_t tmem;
};
// All threads of both blocks; readers: epilogue warps of both.  Returns the tensor memory.
SPLAT_DEV uint32_t pair_begin(PairBarriers& b, int stages, int readers) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      tc::barrier_init(tc::shared_address(&b.full[i]), 1);
      tc::barrier_init(tc::shared_address(&b.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::barrier_init(tc::shared_address(&b.acc_full[i]), 1);
      tc::barrier_init(tc::shared_address(&b.acc_empty[i]), readers);
    }
    tc::barrier_init(tc::shared_address(&b.drained), 1);
    tc::barrier_init_fence();
  }
  if (threadIdx.x < 32) tc::tmem_alloc_pair(tc::shared_address(&b.tmem), 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();
  tc::fence_after_sync();
  return tc::uniform(b.tmem);
}
SPLAT_DEV void pair_end(uint32_t tmem, bool ok, int* error) {
  if (!ok) atomicCAS(error, 0, kDeviceTimeout);
  tc::fence_before_sync();
  __syncthreads();
  __syncwarp();
  tc::cluster_sync();
  if (threadIdx.x < 32) tc::tmem_free_pair(tmem, 512);
}

// One thread of each block: its half of the stages' copies, which are told to the leading
// block's barriers.
struct PairRing {
  PairBarriers& b;
  uint32_t base, stage_bytes;
  int stages;
  uint32_t rank;
  int stage = 0, started = 0;
  uint32_t parity = 1;  // a fresh barrier's previous phase counts as complete

  SPLAT_DEV PairRing(PairBarriers& b, uint32_t base, uint32_t stage_bytes, int stages,
                     uint32_t rank)
      : b(b), base(base), stage_bytes(stage_bytes), stages(stages), rank(rank) {}

  // start(address of the stage, barrier) starts copies of stage_bytes in all
  template <class F>
  SPLAT_DEV bool fill(F start) {
    if (!tc::barrier_wait(tc::shared_address(&b.empty[stage]), parity)) return false;
    const uint32_t own = tc::shared_address(&b.full[stage]);
    if (rank == 0) tc::barrier_expect(own, 2 * stage_bytes);
    start(base + stage * stage_bytes, tc::address_in(own, 0));
    started = max(started, stage + 1);
    if (++stage == stages) stage = 0, parity ^= 1;
    return true;
  }
  // no copy of either block is in flight past the pair's last barrier, also after a wait that
  // ran out: parity ^ 1 is the phase of the ring's current round, parity the last one's
  SPLAT_DEV bool drain() {
    bool ok = true;
    if (rank == 0)
      for (int i = 0; i < started; ++i)
        ok = tc::barrier_wait_pair(tc::shared_address(&b.full[i]),
                                   i < stage ? parity ^ 1 : parity) && ok;
    return ok;
  }
};

// The leading block's product warp.
struct PairIssue {
  PairBarriers& b;
  uint32_t base, stage_bytes, tmem, lead, instruction;
  int stages, stage = 0;
  uint32_t parity = 0, filled = 0;  // accumulators

  SPLAT_DEV PairIssue(PairBarriers& b, uint32_t base, uint32_t stage_bytes, int stages,
                      uint32_t tmem, uint32_t instruction)
      : b(b), base(base), stage_bytes(stage_bytes), tmem(tmem), lead(tc::elected()),
        instruction(instruction), stages(stages) {}

  // A tile over `length` k.
  template <bool AMN, bool BMN>
  SPLAT_DEV bool tile(long long length) {
    const uint32_t acc = filled & 1;
    if (!tc::barrier_wait_pair(tc::shared_address(&b.acc_empty[acc]), ((filled >> 1) & 1) ^ 1))
      return false;
    tc::fence_after_sync();
    const uint32_t d = tmem + acc * 256;
    for (long long k = 0; k < length; k += kChunk) {
      if (!tc::barrier_wait_pair(tc::shared_address(&b.full[stage]), parity)) return false;
      tc::fence_after_sync();
      const uint32_t at = base + stage * stage_bytes;
      uint64_t a = AMN ? tc::descriptor_mn_major(at, kChunk * 128) : tc::descriptor_k_major(at);
      uint64_t v = BMN ? tc::descriptor_mn_major(at + kAPlane, kChunk * 128)
                       : tc::descriptor_k_major(at + kAPlane);
      const int steps = static_cast<int>((min(length - k, static_cast<long long>(kChunk)) + 15) / 16);
#pragma unroll 4
      for (int s = 0; s < steps; ++s) {
        tc::mma_pair(lead, d, a, v, instruction, k > 0 || s > 0);
        a += (AMN ? tc::kStepMn : tc::kStepK) >> 4;
        v += (BMN ? tc::kStepMn : tc::kStepK) >> 4;
      }
      tc::commit_pair(lead, tc::shared_address(&b.empty[stage]));
      if (++stage == stages) stage = 0, parity ^= 1;
    }
    tc::commit_pair(lead, tc::shared_address(&b.acc_full[acc]));
    ++filled;
    return true;
  }
  // Whichever way the loop ended, no product is in flight past this point.
  SPLAT_DEV bool drain() {
    tc::commit_pair(lead, tc::shared_address(&b.drained));
    return tc::barrier_wait(tc::shared_address(&b.drained), 0);
  }
};

template <class T, bool AMN, bool BMN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_product_kernel(const __grid_constant__ PairParams p) {
  extern __shared__ unsigned char dynamic[];
  __shared__ PairBarriers barriers;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const int warp = tc::uniform(threadIdx.x >> 5);
  const uint32_t rank = tc::cluster_rank();
  const int half_n = p.tile_n / 2;
  const uint32_t stage_bytes = kAPlane + b_plane_bytes<BMN>(half_n);
  const uint32_t tmem = pair_begin(barriers, p.stages, 16);
  const int tiles_mn = p.tiles_m * p.tiles_n, tiles = tiles_mn * p.splits;
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  bool ok = true;

  if (warp == 8) {
    if ((threadIdx.x & 31) == 0) {
      PairRing ring(barriers, base, stage_bytes, p.stages, rank);
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int split = t / tiles_mn, rest = t % tiles_mn;
        const int m0 = rest / p.tiles_n * kPairRows + rank * 128;
        const int n0 = rest % p.tiles_n * p.tile_n + rank * half_n;
        const long long k1 = min((split + 1) * p.k_per_split, p.k);
        for (long long k = split * p.k_per_split; k < k1 && ok; k += kChunk)
          ok = ring.fill([&](uint32_t at, uint32_t bar) {
            const int k0 = static_cast<int>(k);
            if constexpr (AMN) {
              tc::copy_in_pair(at, &p.a_map, m0, k0, bar);
              tc::copy_in_pair(at + kChunk * 128, &p.a_map, m0 + 64, k0, bar);
            } else {
              tc::copy_in_pair(at, &p.a_map, k0, m0, bar);
            }
            if constexpr (BMN) {
              for (int i = 0; i * 64 < half_n; ++i)
                tc::copy_in_pair(at + kAPlane + i * (kChunk * 128), &p.b_map, n0 + i * 64, k0, bar);
            } else {
              tc::copy_in_pair(at + kAPlane, &p.b_map, k0, n0, bar);
            }
          });
      }
      ok = ring.drain() && ok;
    }
  } else if (warp == 9) {
    if (rank == 0) {
      PairIssue issue(barriers, base, stage_bytes, p.stages, tmem,
                      tc::instruction_pair(!kIsF16<T>, AMN, BMN, p.tile_n));
      for (int t = pair; t < tiles && ok; t += pairs) {
        const long long k0 = t / tiles_mn * p.k_per_split;
        ok = issue.template tile<AMN, BMN>(min(p.k_per_split, p.k - k0));
      }
      ok = issue.drain() && ok;
    }
  } else {
    // a thread to a row; the sums are few beside what they were taken from
    const int lane = threadIdx.x & 31, lane_block = warp & 3, half = warp >> 2;
    const bool vector = p.n % 4 == 0;
    uint32_t read = 0;
    for (int t = pair; t < tiles && ok; t += pairs, ++read) {
      const int split = t / tiles_mn, rest = t % tiles_mn;
      const int row = rest / p.tiles_n * kPairRows + static_cast<int>(rank) * 128 +
                      lane_block * 32 + lane;
      const int col0 = rest % p.tiles_n * p.tile_n + half * half_n;
      const uint32_t acc = read & 1;
      if (!(ok = tc::barrier_wait(tc::shared_address(&barriers.acc_full[acc]), (read >> 1) & 1)))
        break;
      tc::fence_after_sync();
      float* out = p.out + (static_cast<long long>(split) * p.m + row) * p.n + col0;
      for (int c = 0; c < half_n; c += 32) {
        float v[32];
        tc::tmem_load32(tmem + (lane_block << 21) + acc * 256 + half * half_n + c, v);
        if (row >= p.m) continue;
        if (vector) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            if (col0 + c + j >= p.n) break;
            float4 sum = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            float4* to = reinterpret_cast<float4*>(out + c + j);
            if (p.accumulate) {
              const float4 o = *to;
              sum.x += o.x, sum.y += o.y, sum.z += o.z, sum.w += o.w;
            }
            *to = sum;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (col0 + c + j >= p.n) break;
            out[c + j] = p.accumulate ? out[c + j] + v[j] : v[j];
          }
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0)
        tc::barrier_arrive_remote(tc::address_in(tc::shared_address(&barriers.acc_empty[acc]), 0));
    }
  }
  pair_end(tmem, ok, p.error);
}

// How a pair product of so many tiles and chunks of 64 k is split: such that the busiest
// pair takes the fewest chunks, twelve for a tile's start and end among them, and no
// accumulator more than its additions.
struct PairSplits {
  int count;
  long long k;  // of a split
};
inline PairSplits pair_splits(long long tiles, long long k) {
  const int pairs = std::max(1, host::sm_count() / 2);
  const long long chunks = (k + kChunk - 1) / kChunk;
  const long long most = kMostAdditions * 16 / kChunk;
  const long long fewest = (chunks + most - 1) / most;
  PairSplits best{};
  double least = 1e30;
  for (long long n = fewest; n <= std::min(chunks, fewest + 31); ++n) {
    const long long per = (chunks + n - 1) / n;
    const double cost = static_cast<double>((tiles * n + pairs - 1) / pairs) * (per + 12);
    if (cost < least * 0.98) {
      least = cost;
      best.k = per * kChunk;
      best.count = static_cast<int>((chunks + per - 1) / per);
    }
  }
  return best;
}

inline int pair_tile_n(int n) { return n <= 64 ? 64 : n <= 128 ? 128 : 256; }
inline long long pair_tiles(long long m, int n) {
  const int tile_n = pair_tile_n(n);
  return (m + kPairRows - 1) / kPairRows * ((n + tile_n - 1) / tile_n);
}

// a: (m, k) rows or, AMN, (k, m); b: (n, k) or, BMN, (k, n); out (splits, m, n).
template <class T, bool AMN, bool BMN>
int launch_pairs(int m, int n, long long k, const void* a, long long a_ld, const void* b,
                 long long b_ld, const PairSplits& splits, float* out, bool accumulate,
                 cudaStream_t s) {
  PairParams p{};
  p.m = m, p.n = n, p.k = k, p.k_per_split = splits.k, p.splits = splits.count;
  p.tile_n = pair_tile_n(n);
  p.tiles_m = (m + kPairRows - 1) / kPairRows;
  p.tiles_n = (n + p.tile_n - 1) / p.tile_n;
  p.out = out, p.accumulate = accumulate;
  if (!make_map<T>(p.a_map, a, AMN ? k : m, AMN ? m : k, a_ld, 64, AMN ? kChunk : 128) ||
      !make_map<T>(p.b_map, b, BMN ? k : n, BMN ? n : k, b_ld, 64, BMN ? kChunk : p.tile_n / 2))
    return host::fail(kInvalidArgument, "feature products: operand maps");
  p.error = host::device_error_word();
  if (!p.error) return kCudaError;
  const int stage = kAPlane + b_plane_bytes<BMN>(p.tile_n / 2);
  p.stages = std::min(kPairStages, (kOneBlockBytes - 1024) / stage);
  constexpr auto* kernel = pair_product_kernel<T, AMN, BMN>;
  if (!host::allow_shared<kernel>())
    return host::check_launch("feature products: shared memory");
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n * p.splits;
  if (tiles >= 1LL << 31) return host::fail(kTooLarge, "feature products: too many tiles");
  const int pairs = static_cast<int>(std::min<long long>(tiles, host::sm_count() / 2));
  kernel<<<2 * pairs, kPairThreads, 1024 + p.stages * stage, host::counted(s)>>>(p);
  return host::check_launch("feature products");
}

}  // namespace feature
}  // namespace splat
