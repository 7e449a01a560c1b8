// C(m, n) = sum_k A(m, k) B(n, k) on pairs of blocks (tensor_core.cuh): the long products of
// a vocabulary's gradients.  Operands are 16-bit, A in one plane or in two whose sum it is,
// or fp32 as planes of three bf16 parts (feature_product.cuh); results are fp32 sums over
// ranges of k.
//
// A pair takes 256 x tile_n tiles; each of its blocks copies its 128 rows of A and its half
// of B's in chunks of 64 k, half of what a block on its own would read for the same work.
// No accumulator takes more than kMostAdditions of 16-bit products; those of parts take
// kExactSum k in two accumulators, which the epilogue adds up in registers.
//
// 65536 x 512 bf16 features and 32768 words: dx 1.46 ms (1510 TFLOP/s), dW 1.6 (1370) at the
// 1.5 to 1.6 GHz that the power allows; a piece of it on its own has the tensor pipe 92 and 84 %
// busy.  307200 x 64 and
// 4096: 450 and 400 us, of which reading dz (2.5 GB) is the most: DRAM 73 and 77 %.
#pragma once
#include <algorithm>

#include "feature_launch.cuh"

namespace splat {
namespace feature {

constexpr int kPairRows = 256, kPairStages = 8;
constexpr int kPairThreads = 320;  // eight epilogue warps, copies, products
constexpr int kPairPatches = 8 * 4096;

struct PairParams {
  CUtensorMap a_map, b_map, out_map;
  int a_plane_rows, b_plane_rows;  // of operands in parts
  int m, n, tile_n, stages;
  long long k, k_per_split;  // k_per_split: a multiple of 64
  int tiles_m, tiles_n, splits;
  float* out;      // (splits, m, n)
  int accumulate;  // onto what is there
  int copy_out;    // by tensor copies
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

// The leading block's product warp.  PA, PB: parts of the operands.
template <int PA, int PB>
struct PairIssue {
  PairBarriers& b;
  uint32_t base, stage_bytes, b_plane, tmem, lead, instruction;
  int stages, stage = 0;
  uint32_t parity = 0, filled = 0;  // accumulators

  SPLAT_DEV PairIssue(PairBarriers& b, uint32_t base, uint32_t b_plane, int stages,
                      uint32_t tmem, uint32_t instruction)
      : b(b), base(base), stage_bytes(PA * kAPlane + PB * b_plane), b_plane(b_plane), tmem(tmem),
        lead(tc::elected()), instruction(instruction), stages(stages) {}

  // One accumulator of a tile, over `length` k; that of the lower products of parts lies
  // 128 columns on.
  template <bool AMN, bool BMN>
  SPLAT_DEV bool sum(long long length) {
    const uint32_t acc = filled & 1;
    if (!tc::barrier_wait_pair(tc::shared_address(&b.acc_empty[acc]), ((filled >> 1) & 1) ^ 1))
      return false;
    tc::fence_after_sync();
    const uint32_t d = tmem + acc * 256;
    for (long long k = 0; k < length; k += kChunk) {
      if (!tc::barrier_wait_pair(tc::shared_address(&b.full[stage]), parity)) return false;
      tc::fence_after_sync();
      const uint32_t a_at = base + stage * stage_bytes, b_at = a_at + PA * kAPlane;
      const long long here = min(length - k, static_cast<long long>(kChunk));
      const int steps = static_cast<int>((here + 15) / 16);
      // products of parts i and j with i + j < PA, the smallest first
#pragma unroll
      for (int part = PA - 1; part >= 0; --part)
#pragma unroll
        for (int i = 0; i <= part; ++i) {
          if (part - i >= PB) continue;
          const uint32_t ao = a_at + i * kAPlane, bo = b_at + (part - i) * b_plane;
          uint64_t a = AMN ? tc::descriptor_mn_major(ao, kChunk * 128) : tc::descriptor_k_major(ao);
          uint64_t v = BMN ? tc::descriptor_mn_major(bo, kChunk * 128) : tc::descriptor_k_major(bo);
          const uint32_t to = d + (PB > 1 && part > 0 ? 128 : 0);
          // the first product into an accumulator overwrites it
          const bool first = k == 0 && (PB > 1 ? i == 0 && (part == 0 || part == PA - 1)
                                               : part == PA - 1);
#pragma unroll 4
          for (int s = 0; s < steps; ++s) {
            tc::mma_pair(lead, to, a, v, instruction, !first || s > 0);
            a += (AMN ? tc::kStepMn : tc::kStepK) >> 4;
            v += (BMN ? tc::kStepMn : tc::kStepK) >> 4;
          }
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

// An epilogue warp gives an accumulator back to the leading block.
SPLAT_DEV void pair_release(PairBarriers& b, uint32_t acc) {
  tc::fence_before_sync();
  __syncwarp();
  if ((threadIdx.x & 31) == 0)
    tc::barrier_arrive_remote(tc::address_in(tc::shared_address(&b.acc_empty[acc]), 0));
}

// The kernels' operands as they are copied.
template <class T>
using PairOperand = std::conditional_t<kIsF16<T>, f16, bf16>;

// k of an accumulator.
template <int PA, int PB>
constexpr long long kPairSum = PB > 1 ? kExactSum : kMostAdditions * 16 / PA;

template <class T, int PA, int PB, bool AMN, bool BMN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_product_kernel(const __grid_constant__ PairParams p) {
  extern __shared__ unsigned char dynamic[];
  __shared__ PairBarriers barriers;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const uint32_t ring_at = base + kPairPatches;
  const int warp = tc::uniform(threadIdx.x >> 5);
  const uint32_t rank = tc::cluster_rank();
  const int half_n = p.tile_n / 2;
  const uint32_t b_plane = b_plane_bytes<BMN>(half_n);
  constexpr long long kSum = kPairSum<PA, PB>;
  const uint32_t tmem = pair_begin(barriers, p.stages, 16);
  const int tiles_mn = p.tiles_m * p.tiles_n, tiles = tiles_mn * p.splits;
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  bool ok = true;

  if (warp == 8) {
    if ((threadIdx.x & 31) == 0) {
      PairRing ring(barriers, ring_at, PA * kAPlane + PB * b_plane, p.stages, rank);
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int split = t / tiles_mn, rest = t % tiles_mn;
        const int m0 = rest / p.tiles_n * kPairRows + rank * 128;
        const int n0 = rest % p.tiles_n * p.tile_n + rank * half_n;
        const long long k1 = min((split + 1) * p.k_per_split, p.k);
        for (long long k = split * p.k_per_split; k < k1 && ok; k += kChunk)
          ok = ring.fill([&](uint32_t at, uint32_t bar) {
            const int k0 = static_cast<int>(k);
#pragma unroll
            for (int i = 0; i < PA; ++i, at += kAPlane) {
              if constexpr (AMN) {
                tc::copy_in_pair(at, &p.a_map, m0, k0 + i * p.a_plane_rows, bar);
                tc::copy_in_pair(at + kChunk * 128, &p.a_map, m0 + 64, k0 + i * p.a_plane_rows,
                                 bar);
              } else {
                tc::copy_in_pair(at, &p.a_map, k0, m0 + i * p.a_plane_rows, bar);
              }
            }
#pragma unroll
            for (int i = 0; i < PB; ++i, at += b_plane) {
              if constexpr (BMN) {
                for (int j = 0; j * 64 < half_n; ++j)
                  tc::copy_in_pair(at + j * (kChunk * 128), &p.b_map, n0 + j * 64,
                                   k0 + i * p.b_plane_rows, bar);
              } else {
                tc::copy_in_pair(at, &p.b_map, k0, n0 + i * p.b_plane_rows, bar);
              }
            }
          });
      }
      ok = ring.drain() && ok;
    }
  } else if (warp == 9) {
    if (rank == 0) {
      PairIssue<PA, PB> issue(barriers, ring_at, b_plane, p.stages, tmem,
                         tc::instruction_pair(!kIsF16<T>, AMN, BMN, p.tile_n));
      for (int t = pair; t < tiles && ok; t += pairs) {
        const long long k0 = t / tiles_mn * p.k_per_split, k1 = min(k0 + p.k_per_split, p.k);
        for (long long k = k0; k < k1 && ok; k += kSum)
          ok = issue.template sum<AMN, BMN>(min(kSum, k1 - k));
      }
      ok = issue.drain() && ok;
    }
  } else {
    // a thread to a row, four warps to half of the columns
    const int lane = threadIdx.x & 31, lane_block = warp & 3, half = warp >> 2;
    const Patch<float> patch{base + warp * 4096};
    const uint32_t lanes = lane_block << 21;
    const bool vector = p.n % 4 == 0;
    uint32_t read = 0;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int split = t / tiles_mn, rest = t % tiles_mn;
      const int row0 = rest / p.tiles_n * kPairRows + static_cast<int>(rank) * 128 +
                       lane_block * 32;
      const int col0 = rest % p.tiles_n * p.tile_n + half * half_n, rows = min(p.m - row0, 32);
      const long long out_row = static_cast<long long>(split) * p.m + row0;
      // 32 columns of the tile, from c on
      const auto put = [&](int c, const float (&v)[32]) {
        const int cols = min(p.n - col0 - c, 32);
        if (rows <= 0 || cols <= 0) return;
        // the rows behind a split's last are the next one's
        const bool copies = p.copy_out && rows == 32;
        if (lane == 0) tc::copies_out_read();
        __syncwarp();  // the patch before has been read
#pragma unroll
        for (int j = 0; j < 8; ++j)
          store_shared(patch.at(lane, j),
                       make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                  __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3])));
        if (copies) {
          tc::fence_async_proxy();
          __syncwarp();
          if (lane == 0) {
            const int at = static_cast<int>(out_row);
            if (p.accumulate) tc::add_out(&p.out_map, col0 + c, at, patch.base);
            else tc::copy_out(&p.out_map, col0 + c, at, patch.base);
          }
        } else {
          __syncwarp();
          patch.store(p.out + out_row * p.n + col0 + c, p.n, rows, cols, vector, p.accumulate);
        }
      };
      if constexpr (PB == 1) {  // a split is one sum
        const uint32_t acc = read & 1;
        if (!(ok = tc::barrier_wait(tc::shared_address(&barriers.acc_full[acc]), (read >> 1) & 1)))
          break;
        ++read;
        tc::fence_after_sync();
        for (int c = 0; c < half_n; c += 32) {
          float v[32];
          tc::tmem_load32(tmem + lanes + acc * 256 + half * half_n + c, v);
          put(c, v);
        }
        pair_release(barriers, acc);
      } else {
        // tiles of 64 or 128 columns: 64 of a warp at most
        float held[2][32] = {};
        const long long k0 = split * p.k_per_split, k1 = min(k0 + p.k_per_split, p.k);
        for (long long k = k0; k < k1; k += kSum, ++read) {
          const uint32_t acc = read & 1;
          if (!(ok = tc::barrier_wait(tc::shared_address(&barriers.acc_full[acc]),
                                      (read >> 1) & 1)))
            break;
          tc::fence_after_sync();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (c * 32 >= half_n) break;
            float v[32], low[32];
            const uint32_t from = tmem + lanes + acc * 256 + half * half_n + c * 32;
            tc::tmem_load32(from, v);
            tc::tmem_load32(from + 128, low);
#pragma unroll
            for (int j = 0; j < 32; ++j) held[c][j] += v[j] + low[j];
          }
          pair_release(barriers, acc);
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (c * 32 < half_n) put(c * 32, held[c]);
      }
    }
    if (lane == 0) tc::copies_out_read();
  }
  pair_end(tmem, ok, p.error);
}

// How a pair product of so many tiles and chunks of 64 k is split: such that the busiest
// pair takes the fewest chunks, three for a tile's start among them, and no accumulator
// of 16-bit products more than its additions.
struct PairSplits {
  int count;
  long long k;  // of a split
};
template <int PA, int PB>
PairSplits pair_splits(long long tiles, long long k) {
  const int pairs = std::max(1, host::sm_count() / 2);
  const long long chunks = (k + kChunk - 1) / kChunk;
  const long long most = kPairSum<PA, PB> / kChunk;
  const long long fewest = PB == 1 ? (chunks + most - 1) / most : 1;
  PairSplits best{};
  double least = 1e30;
  for (long long n = fewest; n <= std::min(chunks, fewest + 31); ++n) {
    const long long per = (chunks + n - 1) / n;
    const double cost = static_cast<double>((tiles * n + pairs - 1) / pairs) * (per + 3);
    if (cost < least * 0.98) {
      least = cost;
      best.k = per * kChunk;
      best.count = static_cast<int>((chunks + per - 1) / per);
    }
  }
  return best;
}

// Columns of a tile; parts have two accumulators of half the width.
template <int P>
int pair_tile_n(int n) {
  return n <= 64 ? 64 : n <= 128 || P > 1 ? 128 : 256;
}
template <int P>
long long pair_tiles(long long m, int n) {
  const int tile_n = pair_tile_n<P>(n);
  return (m + kPairRows - 1) / kPairRows * ((n + tile_n - 1) / tile_n);
}

// The map of an operand: planes of its parts (one alone has as many rows as there are),
// whose rows are k or, MN, m or n.
template <class T, int P, bool MN>
bool make_operand_map(CUtensorMap& map, const Planes& x, int mn, long long k, int box_rows) {
  const long long rows = P == 1 ? (MN ? k : mn) : static_cast<long long>(x.plane_rows) * P;
  return make_map<PairOperand<T>>(map, x.data, rows, MN ? mn : k, x.ld, 64, MN ? kChunk : box_rows);
}

// a: (m, k) rows or, AMN, (k, m), of PA parts; b: (n, k) or, BMN, (k, n); out (splits, m, n).
template <class T, int PA, bool AMN, bool BMN>
int launch_pairs(int m, int n, long long k, const Planes& a, const Planes& b,
                 const PairSplits& splits, float* out, bool accumulate, cudaStream_t s) {
  constexpr int PB = kOperandParts<T>;
  PairParams p{};
  p.m = m, p.n = n, p.k = k, p.k_per_split = splits.k, p.splits = splits.count;
  p.tile_n = pair_tile_n<PB>(n);
  p.tiles_m = (m + kPairRows - 1) / kPairRows;
  p.tiles_n = (n + p.tile_n - 1) / p.tile_n;
  p.out = out, p.accumulate = accumulate;
  p.a_plane_rows = a.plane_rows, p.b_plane_rows = b.plane_rows;
  if (!make_operand_map<T, PA, AMN>(p.a_map, a, m, k, 128) ||
      !make_operand_map<T, PB, BMN>(p.b_map, b, n, k, p.tile_n / 2))
    return host::fail(kInvalidArgument, "feature products: operand maps");
  p.copy_out = make_map<float>(p.out_map, out, static_cast<long long>(splits.count) * m, n, n, 32,
                               32);
  p.error = host::device_error_word();
  if (!p.error) return kCudaError;
  const int stage = PA * kAPlane + PB * b_plane_bytes<BMN>(p.tile_n / 2);
  p.stages = std::min(kPairStages, (kOneBlockBytes - 1024 - kPairPatches) / stage);
  constexpr auto* kernel = pair_product_kernel<T, PA, PB, AMN, BMN>;
  if (!host::allow_shared<kernel>())
    return host::check_launch("feature products: shared memory");
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n * p.splits;
  if (tiles >= 1LL << 31) return host::fail(kTooLarge, "feature products: too many tiles");
  const int pairs = static_cast<int>(std::min<long long>(tiles, host::sm_count() / 2));
  kernel<<<2 * pairs, kPairThreads, 1024 + kPairPatches + p.stages * stage, host::counted(s)>>>(p);
  return host::check_launch("feature products");
}

}  // namespace feature
}  // namespace splat
