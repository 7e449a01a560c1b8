// Looking rows up in a table, with a factor, and the table's gradient:
//
//   y_i = s T[id_i]          dT[v] = s sum of dy_i over id_i = v
//
// Bound by memory.  The gradient sorts the rows by id (a stable counting
// sort of up to 10 bits of the id a pass), walks them in that order and adds up
// each entry's run in fp32: a group of lanes to a few rows, the runs that cross
// groups joined in shared memory and those that cross blocks by a second kernel,
// all in the order of the rows, so that no result depends on the order of blocks.
// A few rows are found by comparing their ids with each entry instead.
//
// 1000000 rows of 8192 x 64 bf16: the lookup 26 us (4.9 TB/s), the gradient 90, of which the
// sort takes 45 in two passes and the sums 40 (3.2 TB/s: rows of 128 bytes in the ids' order).
#include <algorithm>

#include "feature_common.cuh"
#include "host_runtime.h"
#include "splat200.h"

namespace splat {
namespace feature {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// An id, or -1 where it lies outside the table.
template <class I>
SPLAT_DEV int id_at(const void* ids, long long i, int entries) {
  const I id = static_cast<const I*>(ids)[i];
  return id >= 0 && id < static_cast<I>(entries) ? static_cast<int>(id) : -1;
}

// ---- forward -----------------------------------------------------------------------

// Rows of `units` pieces of V values, `lanes` threads to a row; a warp takes 32 rows, whose
// ids its lanes read at once.
template <class T, class I, int V>
__global__ void __launch_bounds__(kThreads, 5)
    lookup_kernel(long long count, int entries, int channels, int units, int lanes,
                  const void* ids, const T* table, float scale, T* y, int* error) {
  constexpr int U = 4;  // rows in flight
  using Piece = Vec<T, V>;
  const int lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) / lanes;
  const int groups = 32 / lanes;
  const long long step = gridDim.x * static_cast<long long>(kThreads);
  for (long long row0 = blockIdx.x * static_cast<long long>(kThreads) + (threadIdx.x & ~31u);
       row0 < count; row0 += step) {
    const long long own = row0 + (threadIdx.x & 31);
    int id = -1;
    if (own < count) {
      id = id_at<I>(ids, own, entries);
      if (id < 0) atomicCAS(error, 0, kInconsistentInput);
    }
    const int rows = static_cast<int>(min(count - row0, 32LL));
    for (int r0 = group; r0 < 32; r0 += U * groups) {
      int at[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        at[u] = __shfl_sync(0xffffffffu, id, (r0 + u * groups) & 31);
      for (int q = lane; q < units; q += lanes) {
        Piece v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          v[u] = Piece{};
          if (r0 + u * groups < rows && at[u] >= 0)
            v[u] = *reinterpret_cast<const Piece*>(
                table + static_cast<long long>(at[u]) * channels + q * V);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (scale != 1.0f) {
            float f[V];
            widen<T, V>(v[u], f);
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] *= scale;
            v[u] = round_values<T, V>(f);
          }
          if (r0 + u * groups < rows)
            *reinterpret_cast<Piece*>(y + (row0 + r0 + u * groups) * channels + q * V) = v[u];
        }
      }
    }
  }
}

// ---- sorting indices by id ---------------------------------------------------------

// Bits of a pass.  A million rows of 13 bits in one pass, whose 8192 counters for each
// warp leave an SM one block, took 50 us, in two passes of 7 and 6 bits 45.
constexpr int kMostBits = 10;

// A row and its id.
struct Sorted {
  int row, id;
};

struct SortPass {
  const void* ids;
  const Sorted* order;    // of the pass before; NULL: as they lie
  const int* valid;       // how many of them (with `order`)
  long long count;
  int entries, shift, bins;
  int* counts;            // (bins, blocks)
  int* totals;            // (bins)
  Sorted* out;
  int* out_valid;
};

// id: -1 outside the table, and from `end` on.
template <class I>
SPLAT_DEV Sorted sort_item(const SortPass& p, long long i, long long end) {
  if (i >= end) return {0, -1};
  if (p.order) return p.order[i];
  return {static_cast<int>(i), id_at<I>(p.ids, i, p.entries)};
}
constexpr int kAhead = 8;  // items that a thread reads at once

// Rows of a block: whole warps' worth to each warp.
SPLAT_DEV long long rows_per_warp(long long count) {
  const long long warps = static_cast<long long>(gridDim.x) * kWarps;
  return (count + warps * 32 - 1) / (warps * 32) * 32;
}

template <class I>
__global__ void __launch_bounds__(kThreads) count_digits_kernel(const SortPass p) {
  extern __shared__ __align__(16) int bins[];
  const long long count = p.order ? *p.valid : p.count;
  for (int d = threadIdx.x; d < p.bins; d += kThreads) bins[d] = 0;
  __syncthreads();
  const long long per = rows_per_warp(count) * kWarps;
  const long long begin = blockIdx.x * per, end = min(begin + per, count);
  for (long long i0 = begin + threadIdx.x; i0 < end; i0 += kAhead * kThreads) {
    Sorted v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = sort_item<I>(p, i0 + u * kThreads, end);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v[u].id >= 0) atomicAdd(&bins[(v[u].id >> p.shift) & (p.bins - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.bins; d += kThreads)
    p.counts[static_cast<long long>(d) * gridDim.x + blockIdx.x] = bins[d];
}

// Of each digit, what the blocks before have: a warp to a digit.
__global__ void __launch_bounds__(kThreads) digit_prefix_kernel(const SortPass p, int blocks) {
  const int d = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (d >= p.bins) return;
  int* counts = p.counts + static_cast<long long>(d) * blocks;
  int carry = 0;
  for (int b0 = 0; b0 < blocks; b0 += 32 * kAhead) {
    int v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int b = b0 + u * 32 + lane;
      v[u] = b < blocks ? counts[b] : 0;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      int upto = v[u];
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int before = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += before;
      }
      const int b = b0 + u * 32 + lane;
      if (b < blocks) counts[b] = carry + upto - v[u];
      carry += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  if (lane == 0) p.totals[d] = carry;
}

// Places a block's indices: each warp takes consecutive rows in their order, so
// that equal digits keep it.
template <class I>
__global__ void __launch_bounds__(kThreads) place_kernel(const SortPass p) {
  extern __shared__ __align__(16) int bins[];  // first places
  // (warps, bins)
  unsigned short* own = reinterpret_cast<unsigned short*>(bins + (p.bins + 3) / 4 * 4);
  __shared__ int warp_sums[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long count = p.order ? *p.valid : p.count;
  const long long per = rows_per_warp(count);
  const long long begin = (static_cast<long long>(blockIdx.x) * kWarps + warp) * per;
  const long long end = min(begin + per, count);
  // the digits' first places: an exclusive sum of the totals, of which each warp takes a part
  const int part = (p.bins + 32 * kWarps - 1) / (32 * kWarps) * 32;
  const int part_begin = min(warp * part, p.bins), part_end = min(part_begin + part, p.bins);
  int carry = 0;
  for (int d0 = part_begin; d0 < part_end; d0 += 32 * kAhead) {
    int v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int d = d0 + u * 32 + lane;
      v[u] = d < part_end ? p.totals[d] : 0;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      int upto = v[u];
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int before = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += before;
      }
      const int d = d0 + u * 32 + lane;
      if (d < part_end) bins[d] = carry + upto - v[u];
      carry += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  if (lane == 0) warp_sums[warp] = carry;
  uint4* zeros = reinterpret_cast<uint4*>(own);
  for (int i = threadIdx.x; i < kWarps * p.bins / 8; i += kThreads)
    zeros[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    int all = 0;
    for (int w = 0; w < kWarps; ++w) all += warp_sums[w];
    *p.out_valid = all;
  }
  for (int d = threadIdx.x; d < p.bins; d += kThreads) {
    int place = bins[d] + p.counts[static_cast<long long>(d) * gridDim.x + blockIdx.x];
    for (int w = 0; w < d / part; ++w) place += warp_sums[w];
    bins[d] = place;
  }
  // the warps' counts, two to a word (a block has less than 2^16 rows, see plan_embedding)
  int* words = reinterpret_cast<int*>(own + static_cast<long long>(warp) * p.bins);
  for (long long i0 = begin + lane; i0 < end; i0 += kAhead * 32) {
    Sorted v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = sort_item<I>(p, i0 + u * 32, end);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (v[u].id < 0) continue;
      const int d = (v[u].id >> p.shift) & (p.bins - 1);
      atomicAdd(&words[d >> 1], 1 << ((d & 1) * 16));
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.bins; d += kThreads) {
    int before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int n = own[w * p.bins + d];
      own[w * p.bins + d] = static_cast<unsigned short>(before);
      before += n;
    }
  }
  __syncthreads();
  unsigned short* next = own + static_cast<long long>(warp) * p.bins;
  for (long long i0 = begin; i0 < end; i0 += kAhead * 32) {
    Sorted v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = sort_item<I>(p, i0 + u * 32 + lane, end);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int d = v[u].id >= 0 ? (v[u].id >> p.shift) & (p.bins - 1) : -1;
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      const int rank = __popc(peers & lanemask_lt());
      int first = 0;
      if (d >= 0) first = next[d];
      __syncwarp();
      if (d >= 0 && rank == 0) next[d] = static_cast<unsigned short>(first + __popc(peers));
      __syncwarp();
      if (d >= 0) p.out[bins[d] + first + rank] = v[u];
    }
  }
}

// ---- sums of sorted rows -------------------------------------------------------------

// Bits of a block's flags: its first rows continue the entry of the block before;
// all of its rows do, and the entry goes on behind it; its last rows begin an entry
// that goes on behind it.
constexpr int kHead = 1, kThrough = 2, kTail = 4;
constexpr int kMostBlockRows = 2048;

struct RunParams {
  const Sorted* order;
  const int* valid;
  int channels, lanes, rows;  // rows of a group
  const void* dy;
  float scale;
  void* dtable;
  float *heads, *tails;  // (blocks, channels)
  int* flags;            // (blocks)
};

template <class T, int V>
__global__ void __launch_bounds__(kThreads, 4) sum_runs_kernel(const RunParams p) {
  using Piece = Vec<T, V>;
  __shared__ int index[kMostBlockRows], key_at[kMostBlockRows + 2];
  __shared__ float head[kThreads * V], tail[kThreads * V];
  __shared__ unsigned char flags[kThreads];
  const int lanes = p.lanes, groups = kThreads / lanes, R = p.rows;
  const int count = *p.valid;
  const int begin = blockIdx.x * groups * R;
  if (begin >= count) {
    if (blockIdx.y == 0 && threadIdx.x == 0) p.flags[blockIdx.x] = 0;
    return;
  }
  const int rows = min(groups * R, count - begin);
  // key_at[i + 1] is row i's id; of the rows before and behind the block too
  for (int i = threadIdx.x; i < rows + 2; i += kThreads) {
    const int at = begin + i - 1;
    int key = -1;
    if (at >= 0 && at < count) {
      const Sorted v = p.order[at];
      key = v.id;
      if (i > 0 && i <= rows) index[i - 1] = v.row;
    }
    key_at[i] = key;
  }
  __syncthreads();
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes;
  const int c = (blockIdx.y * lanes + lane) * V;
  const bool in = c < p.channels;
  const int a = group * R, b = min(a + R, rows);
  const auto write = [&](int key, const float (&sum)[V]) {
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = sum[k] * p.scale;
    if (in)
      *reinterpret_cast<Piece*>(static_cast<T*>(p.dtable) +
                                static_cast<long long>(key) * p.channels + c) =
          round_values<T, V>(f);
  };
  if (a < b) {
    const T* dy = static_cast<const T*>(p.dy) + c;
    float sum[V] = {};
    int start = a, found = 0;
    constexpr int U = 8;  // rows in flight
    for (int i0 = a; i0 < b; i0 += U) {
      Piece v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u] = Piece{};
        if (i0 + u < b && in)
          v[u] = *reinterpret_cast<const Piece*>(
              dy + static_cast<long long>(index[i0 + u]) * p.channels);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u;
        if (i >= b) break;
        float f[V];
        widen<T, V>(v[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += f[k];
        const int key = key_at[i + 1];
        if (i + 1 < b && key_at[i + 2] == key) continue;
        // a run ends here
        const bool before = start == a && key_at[a] == key;
        const bool behind = i + 1 == b && key_at[b + 1] == key;
        if (!before && !behind) {
          write(key, sum);
        } else {
          float* to = (before ? head : tail) + threadIdx.x * V;
#pragma unroll
          for (int k = 0; k < V; ++k) to[k] = sum[k];
          found |= before ? (behind ? kHead | kThrough : kHead) : kTail;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] = 0.0f;
        start = i + 1;
      }
    }
    if (lane == 0) flags[group] = static_cast<unsigned char>(found);
  }
  __syncthreads();
  if (a >= b) return;
  // the runs across groups: from where each begins
  const int last = (rows + R - 1) / R;
  // adds the heads of groups g, g + 1, ...; true if the run goes on behind the block
  const auto chain = [&](float (&sum)[V], int g) {
    for (; g < last; ++g) {
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] += head[(g * lanes + lane) * V + k];
      if (!(flags[g] & kThrough)) return false;
    }
    return true;
  };
  const long long slot = static_cast<long long>(blockIdx.x) * p.channels + c;
  int found = 0;
  if (group == 0 && (flags[0] & kHead)) {
    float sum[V] = {};
    found = chain(sum, 0) ? kHead | kThrough : kHead;
    if (in)
#pragma unroll
      for (int k = 0; k < V; ++k) p.heads[slot + k] = sum[k];
  }
  if (flags[group] & kTail) {
    float sum[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] = tail[threadIdx.x * V + k];
    if (!chain(sum, group + 1)) {
      write(key_at[b], sum);
    } else {  // of one group at most
      found |= kTail;
      if (in)
#pragma unroll
        for (int k = 0; k < V; ++k) p.tails[slot + k] = sum[k];
    }
  }
  if (blockIdx.y == 0 && lane == 0 && found) atomicOr(&p.flags[blockIdx.x], found);
}

// The runs across blocks.
template <class T>
__global__ void __launch_bounds__(kThreads) join_runs_kernel(const RunParams p, int block_rows) {
  if (!(p.flags[blockIdx.x] & kTail)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the last block that the run reaches
  int end = blockIdx.x + 1;
  while (true) {
    const bool through = end + lane < static_cast<int>(gridDim.x) &&
                         (p.flags[end + lane] & kThrough);
    const uint32_t all = __ballot_sync(0xffffffffu, through);
    if (all != 0xffffffffu) {
      end += __ffs(~all) - 1;
      break;
    }
    end += 32;
  }
  const int key = p.order[static_cast<long long>(blockIdx.x + 1) * block_rows - 1].id;
  __shared__ float sums[kWarps][32];
  for (int c0 = blockIdx.y * 32; c0 < p.channels; c0 += gridDim.y * 32) {
    const int c = c0 + lane;
    float sum = 0.0f;
    if (c < p.channels) {
      if (warp == 0) sum = p.tails[static_cast<long long>(blockIdx.x) * p.channels + c];
#pragma unroll 4
      for (int b = blockIdx.x + 1 + warp; b <= end; b += kWarps)
        sum += p.heads[static_cast<long long>(b) * p.channels + c];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.channels) {
      sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += sums[w][lane];
      static_cast<T*>(p.dtable)[static_cast<long long>(key) * p.channels + c] =
          from_float<T>(sum * p.scale);
    }
    __syncthreads();
  }
}

// ---- few rows: each entry looks for its own --------------------------------------------

constexpr int kMostScanned = 1024;

// A warp to an entry and every gridDim.y-th 32 of its channels.
template <class T, class I>
__global__ void __launch_bounds__(kThreads)
    scan_ids_kernel(int count, int entries, int channels, const void* ids, const T* dy,
                    float scale, T* dtable) {
  __shared__ int id[kMostScanned];
  for (int i = threadIdx.x; i < count; i += kThreads) id[i] = id_at<I>(ids, i, entries);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int v = blockIdx.x * kWarps + (threadIdx.x >> 5); v < entries; v += gridDim.x * kWarps)
    for (int c0 = blockIdx.y * 32; c0 < channels; c0 += gridDim.y * 32) {
      const int c = c0 + lane;
      float sum = 0.0f;
      for (int i0 = 0; i0 < count; i0 += 32) {
        uint32_t hits = __ballot_sync(0xffffffffu, i0 + lane < count && id[i0 + lane] == v);
        if (!hits || c >= channels) continue;
        const T* rows = dy + static_cast<long long>(i0) * channels + c;
        if (__popc(hits) > 4) {  // a common entry's loads are in flight together
          constexpr int U = 16;
          for (int r0 = 0; r0 < 32; r0 += U) {
            T raw[U];
#pragma unroll
            for (int r = 0; r < U; ++r) {
              raw[r] = from_float<T>(0.0f);
              if (hits >> (r0 + r) & 1) raw[r] = rows[static_cast<long long>(r0 + r) * channels];
            }
#pragma unroll
            for (int r = 0; r < U; ++r) sum += to_float(raw[r]);
          }
        } else {
          for (; hits; hits &= hits - 1)
            sum += to_float(rows[static_cast<long long>(__ffs(hits) - 1) * channels]);
        }
      }
      if (c < channels)
        dtable[static_cast<long long>(v) * channels + c] = from_float<T>(sum * scale);
    }
}

// ---- launching -----------------------------------------------------------------------

int check_embedding(int dtype, int id_bytes, long long count, int entries, int channels) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "feature_embedding: dtype");
  if (id_bytes != 4 && id_bytes != 8)
    return host::fail(kInvalidArgument, "feature_embedding: ids are of 4 or 8 bytes");
  if (count < 1 || entries < 1 || channels < 1)
    return host::fail(kInvalidArgument, "feature_embedding: sizes");
  if (count > 1LL << 30 || channels > 65535 || entries > 1 << 30)
    return host::fail(kTooLarge, "feature_embedding: too many ids, entries or channels");
  return kOk;
}

// Whether each entry looks for its rows.  What bounds it is either all warps' steps together
// (64 rows of 8192 entries x 512, 2^18 steps, take 15 us where sorting takes 29; 256 rows,
// 2^20, 32 where it takes 29) or the warp of the commonest entry, which the sizes do not tell: rows
// that are all alike take 10 us for 256 of them and 37 for 1024, unlike ones of 300 entries x
// 512 take 8, and sorting 1024 takes 22 to 25 (47 where its launches are not captured).
bool scans(long long count, int entries, int channels) {
  return count <= kMostScanned &&
         (count + 31) / 32 * entries * ((channels + 31) / 32) <= 1LL << 19;
}

struct EmbeddingPlan {
  int passes, bits[3], sort_blocks;
  int lanes, columns, rows;    // of sum_runs_kernel: lanes of a row, column tiles, rows a group
  int block_rows, run_blocks;
  size_t order, order2, counts, totals, valid, heads, tails, flags, bytes;  // offsets
};

EmbeddingPlan plan_embedding(long long count, int entries, int channels, int values) {
  EmbeddingPlan plan{};
  int bits = 1;
  while (bits < 31 && (1LL << bits) < entries) ++bits;
  plan.passes = (bits + kMostBits - 1) / kMostBits;
  for (int i = 0; i < plan.passes; ++i)
    plan.bits[i] = bits / plan.passes + (i < bits % plan.passes);
  // 2^15 rows to a block at most: its warps count in 16 bits
  plan.sort_blocks = static_cast<int>(std::max<long long>(
      std::min<long long>((count + 2047) / 2048, 8LL * host::sm_count()), (count + 32767) / 32768));
  const int units = (channels + values - 1) / values;
  plan.lanes = 1;
  while (plan.lanes < 32 && plan.lanes < units) plan.lanes *= 2;
  plan.columns = (units + plan.lanes - 1) / plan.lanes;
  const int groups = kThreads / plan.lanes;
  plan.rows = std::min(32, kMostBlockRows / groups);
  plan.block_rows = groups * plan.rows;
  plan.run_blocks = static_cast<int>((count + plan.block_rows - 1) / plan.block_rows);
  const auto take = [&](size_t n) {
    const size_t at = plan.bytes;
    plan.bytes += (n + 255) / 256 * 256;
    return at;
  };
  plan.flags = take(4ull * plan.run_blocks);
  plan.order = take(sizeof(Sorted) * count);
  plan.order2 = plan.passes > 1 ? take(sizeof(Sorted) * count) : plan.order;
  plan.counts = take(4ull * plan.sort_blocks << kMostBits);
  plan.totals = take(4ull << kMostBits);
  plan.valid = take(16);
  plan.heads = take(4ull * plan.run_blocks * channels);
  plan.tails = take(4ull * plan.run_blocks * channels);
  return plan;
}

// Values of a piece that rows and bases allow.
template <class T>
int piece_values(int channels, const void* a, const void* b) {
  int v = 16 / static_cast<int>(sizeof(T));
  while (v > 1 && (channels % v || !host::aligned(a, v * sizeof(T)) ||
                   !host::aligned(b, v * sizeof(T))))
    v /= 2;
  return v;
}

template <class T, class I>
int launch_lookup(long long count, int entries, int channels, const void* ids, const void* table,
                  float scale, void* y, cudaStream_t s) {
  int* error = host::device_error_word();
  if (!error) return kCudaError;
  const int v = piece_values<T>(channels, table, y);
  const int units = channels / v;
  int lanes = 1;
  while (lanes < 32 && lanes < units) lanes *= 2;
  const unsigned grid = static_cast<unsigned>(
      std::min<long long>((count + kThreads - 1) / kThreads, 1LL << 30));
  const auto run = [&](auto* kernel) {
    kernel<<<grid, kThreads, 0, host::counted(s)>>>(count, entries, channels, units, lanes, ids,
                                                    static_cast<const T*>(table), scale,
                                                    static_cast<T*>(y), error);
  };
  if constexpr (sizeof(T) == 2) {
    if (v == 8) run(lookup_kernel<T, I, 8>);
  }
  if (v == 4) run(lookup_kernel<T, I, 4>);
  else if (v == 2) run(lookup_kernel<T, I, 2>);
  else if (v == 1) run(lookup_kernel<T, I, 1>);
  return host::check_launch("feature_embedding");
}

template <class T, class I>
int launch_gradient(long long count, int entries, int channels, const void* ids, const void* dy,
                    float scale, void* dtable, char* ws, cudaStream_t s) {
  if (scans(count, entries, channels)) {
    // the channels of few entries are spread over blocks
    const int wanted = 8 * host::sm_count(), columns = (channels + 31) / 32;
    const int blocks = std::min((entries + kWarps - 1) / kWarps, wanted);
    const dim3 grid(blocks, std::min(columns, std::max(1, wanted / blocks)));
    scan_ids_kernel<T, I><<<grid, kThreads, 0, host::counted(s)>>>(
        static_cast<int>(count), entries, channels, ids, static_cast<const T*>(dy), scale,
        static_cast<T*>(dtable));
    return host::check_launch("feature_embedding_backward");
  }
  constexpr int V = 16 / sizeof(T);
  const int v = piece_values<T>(channels, dy, dtable) == V ? V : 1;
  const EmbeddingPlan plan = plan_embedding(count, entries, channels, v);
  if (cudaMemsetAsync(dtable, 0, sizeof(T) * entries * static_cast<size_t>(channels), s) !=
          cudaSuccess ||
      cudaMemsetAsync(ws + plan.flags, 0, 4ull * plan.run_blocks, s) != cudaSuccess)
    return host::check_launch("feature_embedding_backward: zeros");
  int shift = 0;
  const Sorted* order = nullptr;
  int* valid = reinterpret_cast<int*>(ws + plan.valid);
  for (int i = 0; i < plan.passes; ++i) {
    SortPass p{};
    p.ids = ids, p.order = order, p.count = count, p.entries = entries;
    p.valid = valid + (i + 1) % 2, p.out_valid = valid + i % 2;
    p.shift = shift, p.bins = 1 << plan.bits[i];
    p.counts = reinterpret_cast<int*>(ws + plan.counts);
    p.totals = reinterpret_cast<int*>(ws + plan.totals);
    p.out = reinterpret_cast<Sorted*>(ws + (i % 2 ? plan.order2 : plan.order));
    count_digits_kernel<I><<<plan.sort_blocks, kThreads, 4 * p.bins, host::counted(s)>>>(p);
    digit_prefix_kernel<<<host::blocks_for(p.bins, kWarps), kThreads, 0, host::counted(s)>>>(
        p, plan.sort_blocks);
    place_kernel<I><<<plan.sort_blocks, kThreads, 4 * ((p.bins + 3) / 4 * 4) + 2 * kWarps * p.bins,
                      host::counted(s)>>>(p);
    order = p.out;
    shift += plan.bits[i];
  }
  RunParams r{};
  r.order = order, r.valid = valid + (plan.passes - 1) % 2;
  r.channels = channels, r.lanes = plan.lanes, r.rows = plan.rows;
  r.dy = dy, r.scale = scale, r.dtable = dtable;
  r.heads = reinterpret_cast<float*>(ws + plan.heads);
  r.tails = reinterpret_cast<float*>(ws + plan.tails);
  r.flags = reinterpret_cast<int*>(ws + plan.flags);
  const dim3 grid(plan.run_blocks, plan.columns);
  if (v == V) sum_runs_kernel<T, V><<<grid, kThreads, 0, host::counted(s)>>>(r);
  else sum_runs_kernel<T, 1><<<grid, kThreads, 0, host::counted(s)>>>(r);
  const dim3 join_grid(plan.run_blocks, std::min((channels + 31) / 32, 64));
  join_runs_kernel<T><<<join_grid, kThreads, 0, host::counted(s)>>>(r, plan.block_rows);
  return host::check_launch("feature_embedding_backward");
}

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

int splat_feature_embedding(int dtype, int id_bytes, long long count, int entries, int channels,
                            const void* ids, const void* table, float scale, void* y,
                            void* stream) {
  const int bad = check_embedding(dtype, id_bytes, count, entries, channels);
  if (bad != kOk) return bad;
  if (!ids || !table || !y)
    return host::fail(kInvalidArgument, "feature_embedding: null pointer");
  auto s = static_cast<cudaStream_t>(stream);
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return id_bytes == 8
               ? launch_lookup<T, long long>(count, entries, channels, ids, table, scale, y, s)
               : launch_lookup<T, int>(count, entries, channels, ids, table, scale, y, s);
  });
}

size_t splat_feature_embedding_backward_workspace_bytes(int dtype, long long count, int entries,
                                                        int channels) {
  if (check_embedding(dtype, 8, count, entries, channels) != kOk) return 0;
  if (scans(count, entries, channels)) return 16;
  // of either width of pieces
  const int v = dtype == kF32 ? 4 : 8;
  return std::max(plan_embedding(count, entries, channels, v).bytes,
                  plan_embedding(count, entries, channels, 1).bytes);
}

int splat_feature_embedding_backward(int dtype, int id_bytes, long long count, int entries,
                                     int channels, const void* ids, const void* dy, float scale,
                                     void* dtable, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  const int bad = check_embedding(dtype, id_bytes, count, entries, channels);
  if (bad != kOk) return bad;
  if (!ids || !dy || !dtable || (!workspace && !scans(count, entries, channels)))
    return host::fail(kInvalidArgument, "feature_embedding_backward: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument,
                      "feature_embedding_backward: workspace not 16-byte aligned");
  if (workspace_bytes <
      splat_feature_embedding_backward_workspace_bytes(dtype, count, entries, channels))
    return host::fail(kWorkspaceTooSmall, "feature_embedding_backward: workspace");
  auto s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return id_bytes == 8
               ? launch_gradient<T, long long>(count, entries, channels, ids, dy, scale, dtable,
                                               ws, s)
               : launch_gradient<T, int>(count, entries, channels, ids, dy, scale, dtable, ws, s);
  });
}

}  // extern "C"
