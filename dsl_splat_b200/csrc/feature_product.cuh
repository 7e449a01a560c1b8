// C(m, n) = sum_k A(m, k) B(n, k) on the tensor cores, with the epilogues of a
// linear layer and its backward.
//
// Numbers.  Operands are 16-bit for tcgen05.mma.  What has more digits is
// split into 2 or 3 bf16 parts, v = v0 + v1 + v2 with v_i rounded from what
// v_0 .. v_{i-1} leave (8 digits each), and the products of parts i and j with
// i + j < parts are summed: three parts reproduce an fp32 product to 2^-24, two
// a 16-bit value exactly.  Accumulators are fp32 in tensor memory.
//
// Work.  A persistent block takes 128 x NT tiles.  Four producer warps move
// 64-wide chunks of k from global memory into a ring of stages (converting and
// zero-filling on the way: any row length, any row count), one thread issues
// the products, and eight epilogue warps take the finished accumulator, of which
// there are two, so that loads, products and epilogues of neighbouring tiles
// overlap.  Where the whole of B fits beside the ring it is loaded once per
// block.
#pragma once
#include "feature_common.cuh"
#include "tensor_core.cuh"

namespace splat {
namespace feature {

constexpr int kTileRows = 128;
constexpr int kChunk = 64;             // k of a stage: 128 bytes of 16-bit values
constexpr int kEpilogueWarps = 8;                  // epilogue warps
constexpr int kMaxStages = 8;
constexpr int kStagingBytes = 4096;    // of an epilogue warp: 32 x 32 fp32
constexpr int kAPlane = kTileRows * 128;

// Producer threads.  One-part operands are copied as they are and the copies
// wait in the ring; those that are split pass through registers, so there it
// is threads that keep loads in flight.
__host__ __device__ constexpr int producers(int pa, int pb) { return pa == 1 && pb == 1 ? 128 : 256; }
// fp32 operands keep the products of lower parts in an accumulator of their
// own: the tensor core truncates its sums, so each addition at full magnitude
// costs up to 2^-24, and the lower products must not add to their number.
// 16-bit results do not show it.
__host__ __device__ constexpr int accumulators(int pa, int pb) { return pa == 3 || pb == 3 ? 2 : 1; }
// k that such an accumulator sums before it is added up in fp32 (32 additions).
constexpr int kExactSum = 512;

// act(C + bias) + residual; dy act'(C + bias); C.
enum Epilogue : int { kForward = 0, kSlope = 1, kPlain = 2 };

struct ProductParams {
  long long m, k;  // k of all splits
  int n;
  // row-major sources: A is (m, k) rows or, transposed, (k, m); B likewise
  const void* a;
  const void* b;
  long long a_ld, b_ld;
  int a_vector, b_vector;  // bytes that every row start and chunk is aligned to
  long long k_per_split;   // a multiple of kChunk unless there is one split
  long long k_per_sum;     // of one accumulator; the tile's sums are added in `out` (fp32)
  int splits, tile_n, tiles_n;
  long long tiles_m, tiles;
  int stages, resident, activation;
  int lag;                 // stages whose copies may be in flight; 0: through registers
  uint32_t tmem_columns;
  const void* bias;   // (n) or NULL
  const void* extra;  // residual or dy (m, n), or NULL
  void* out;          // (splits, m, n)
  int out_vector;     // rows of extra and out start on whole vectors
  int* error;
};

// ---- global memory -> operand planes -----------------------------------------

// 8 values in memory order, read with loads of VB bytes; values from `valid`
// on are zero.
template <class S, int VB>
SPLAT_DEV Vec<S, 8> load8(const S* p, int valid) {
  Vec<S, 8> r;
  constexpr int E = VB / static_cast<int>(sizeof(S));  // values per load
#pragma unroll
  for (int j = 0; j < 8 / E; ++j) {
    Vec<S, E> part;
    if (j * E < valid) {
      if constexpr (VB == 16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + j);
        part = reinterpret_cast<const Vec<S, E>&>(u);
      } else if constexpr (VB == 8) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p) + j);
        part = reinterpret_cast<const Vec<S, E>&>(u);
      } else if constexpr (VB == 4) {
        const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(p) + j);
        part = reinterpret_cast<const Vec<S, E>&>(u);
      } else {
        const uint16_t u = __ldg(reinterpret_cast<const uint16_t*>(p) + j);
        part = reinterpret_cast<const Vec<S, E>&>(u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) part.v[e] = from_float<S>(0.0f);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) r.v[j * E + e] = part.v[e];
  }
  return r;
}

// Part of two values as a packed pair, and what it leaves of them.
SPLAT_DEV uint32_t take_part(float& a, float& b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const uint32_t u = reinterpret_cast<const uint32_t&>(h);
  a -= __uint_as_float(u << 16);
  b -= __uint_as_float(u & 0xffff0000u);
  return u;
}

template <class S, int P>
SPLAT_DEV void to_parts(const Vec<S, 8>& v, uint4 (&out)[P]) {
  if constexpr (P == 1 && sizeof(S) == 2) {
    out[0] = reinterpret_cast<const uint4&>(v);
  } else {
    uint32_t w[P][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = to_float(v.v[2 * j]), b = to_float(v.v[2 * j + 1]);
#pragma unroll
      for (int p = 0; p < P; ++p) w[p][j] = take_part(a, b);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) out[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
  }
}

SPLAT_DEV void store_shared(uint32_t address, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}
SPLAT_DEV float4 load_shared(uint32_t address) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(address)
               : "memory");
  return v;
}

// Fills `rows` rows of a block (and of its parts' planes, `plane` bytes apart)
// with `pieces` 16-byte pieces each from src (already at the block's corner):
// rows from rows_valid and columns from cols_valid on are zero.
template <class S, int P, int VB>
SPLAT_DEV void fill_block(uint32_t dst, uint32_t plane, int rows, int pieces, const S* src,
                          long long ld, long long rows_valid, long long cols_valid, int thread,
                          int threads) {
  constexpr int U = P == 1 && VB == 16 ? 8 : 4;  // pieces in flight per thread
  const int shift = pieces <= 1 ? 0 : pieces <= 2 ? 1 : pieces <= 4 ? 2 : 3;
  const int total = rows << shift;
  for (int i0 = thread; i0 < total; i0 += U * threads) {
    Vec<S, 8> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * threads, row = i >> shift, piece = i & ((1 << shift) - 1);
      const long long left = cols_valid - piece * 8;
      const int valid = i < total && row < rows_valid && piece < pieces && left > 0
                            ? static_cast<int>(left < 8 ? left : 8)
                            : 0;
      v[u] = load8<S, VB>(src + row * ld + piece * 8, valid);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * threads, row = i >> shift, piece = i & ((1 << shift) - 1);
      if (i < total && piece < pieces) {
        uint4 parts[P];
        to_parts<S, P>(v[u], parts);
        const uint32_t at = dst + row * 128 + ((piece ^ (row & 7)) << 4);
#pragma unroll
        for (int p = 0; p < P; ++p) store_shared(at + p * plane, parts[p]);
      }
    }
  }
}

template <class S, int P>
SPLAT_DEV void fill(int vector, uint32_t dst, uint32_t plane, int rows, int pieces, const S* src,
                    long long ld, long long rows_valid, long long cols_valid, int thread,
                    int threads) {
  if (vector >= 16)
    fill_block<S, P, 16>(dst, plane, rows, pieces, src, ld, rows_valid, cols_valid, thread,
                         threads);
  else if (vector >= 8)
    fill_block<S, P, 8>(dst, plane, rows, pieces, src, ld, rows_valid, cols_valid, thread,
                        threads);
  else if (vector >= 4 || sizeof(S) == 4)
    fill_block<S, P, 4>(dst, plane, rows, pieces, src, ld, rows_valid, cols_valid, thread,
                        threads);
  else
    fill_block<S, P, sizeof(S)>(dst, plane, rows, pieces, src, ld, rows_valid, cols_valid, thread,
                                threads);
}

// The same for one-part operands whose rows are 16-byte aligned, by copies that
// the thread does not wait for.
template <class S>
SPLAT_DEV void fill_async(uint32_t dst, int rows, int pieces, const S* src, long long ld,
                          long long rows_valid, long long cols_valid, int thread, int threads) {
  const int shift = pieces <= 1 ? 0 : pieces <= 2 ? 1 : pieces <= 4 ? 2 : 3;
  const int total = rows << shift;
  const int piece = thread & ((1 << shift) - 1);  // threads is a multiple of 8
  if (piece >= pieces) return;
  const long long left = cols_valid - piece * 8;
  const int bytes = left <= 0 ? 0 : static_cast<int>(left < 8 ? left : 8) * 2;
  src += piece * 8;
#pragma unroll 4
  for (int i = thread; i < total; i += threads) {
    const int row = i >> shift;
    const bool in = row < rows_valid && bytes;
    // a copy of no bytes fills with zeros; its address stays inside the source
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     dst + row * 128 + ((piece ^ (row & 7)) << 4)),
                 "l"(in ? src + row * ld : src - piece * 8), "r"(in ? bytes : 0)
                 : "memory");
  }
}

// Waits until at most `lag` groups of the thread's copies are in flight.
SPLAT_DEV void wait_copies(int lag) {
  switch (lag) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    case 6: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 7;" ::: "memory"); break;
  }
}

// One operand's chunk: `width` m or n from mn0 and kChunk k from k0 (k_valid of
// them real).  K-major operands are one block of `width` rows; MN-major ones
// are blocks of 64 m or n, each of kChunk rows.
template <class S, int P, bool MN>
SPLAT_DEV void fill_chunk(bool async, int vector, uint32_t dst, uint32_t plane, int width,
                          const S* src, long long ld, long long mn0, long long mn_valid,
                          long long k0, int k_valid, int thread, int threads) {
  const int rows = MN ? min((k_valid + 15) / 16 * 16, kChunk) : width;
  const int pieces = MN ? 8 : min((k_valid + 15) / 16 * 2, 8);
  for (int b = 0; b == 0 || (MN && b * 64 < width && b * 64 < mn_valid); ++b) {
    const S* corner = MN ? src + k0 * ld + mn0 + b * 64 : src + mn0 * ld + k0;
    const long long rows_valid = MN ? k_valid : mn_valid;
    const long long cols_valid = MN ? mn_valid - b * 64 : k_valid;
    const uint32_t at = dst + b * (kChunk * 128);
    if constexpr (P == 1) {
      if (async) {
        fill_async<S>(at, rows, pieces, corner, ld, rows_valid, cols_valid, thread, threads);
        continue;
      }
    }
    fill<S, P>(vector, at, plane, rows, pieces, corner, ld, rows_valid, cols_valid, thread,
               threads);
  }
}

// ---- epilogue ------------------------------------------------------------------

template <int EPI, int ACT>
SPLAT_DEV float finish(float z, float extra) {
  if constexpr (EPI == kForward) return activate<ACT>(z) + extra;
  if constexpr (EPI == kSlope) return extra * slope<ACT>(z);
  return z;
}

// A 32 x 32 patch of the accumulator: staged through the warp's shared memory
// so that global accesses run along rows.
SPLAT_DEV void stage_patch(uint32_t staging, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    store_shared(staging + lane * 128 + ((j ^ (lane & 7)) << 4),
                 make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                            __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3])));
  __syncwarp();
}

template <int EPI, int ACT, class TE, class TO>
SPLAT_DEV void write_patch(const ProductParams& p, uint32_t staging, long long row0, int col0,
                           TO* out, bool add) {
  const int lane = threadIdx.x & 31;
  const TE* extra = static_cast<const TE*>(p.extra);
  const TE* bias = static_cast<const TE*>(p.bias);
  if (p.out_vector) {
    constexpr int V = sizeof(TE) == 2 ? 8 : 4;  // columns of a lane
    constexpr int kLanes = 32 / V, kRows = 32 / kLanes;
    const int c = lane % kLanes, col = col0 + c * V;
    if (col < p.n) {
      float b[V] = {};
      if (bias) {
        const Vec<TE, V> raw = *reinterpret_cast<const Vec<TE, V>*>(bias + col);
#pragma unroll
        for (int j = 0; j < V; ++j) b[j] = to_float(raw.v[j]);
      }
#pragma unroll 4
      for (int i = 0; i < 32 / kRows; ++i) {
        const int r = i * kRows + lane / kLanes;
        const long long row = row0 + r;
        if (row >= p.m) break;
        Vec<TE, V> e;
        if (extra) e = *reinterpret_cast<const Vec<TE, V>*>(extra + row * p.n + col);
        float z[V];
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
          const float4 q = load_shared(staging + r * 128 + (((c * (V / 4) + j) ^ (r & 7)) << 4));
          z[4 * j] = q.x, z[4 * j + 1] = q.y, z[4 * j + 2] = q.z, z[4 * j + 3] = q.w;
        }
        constexpr int W = 16 / sizeof(TO);  // values of one store
#pragma unroll
        for (int h = 0; h < V; h += W < V ? W : V) {
          Vec<TO, (W < V ? W : V)> o;
#pragma unroll
          for (int j = 0; j < (W < V ? W : V); ++j)
            o.v[j] = from_float<TO>(finish<EPI, ACT>(z[h + j] + b[h + j],
                                                extra ? to_float(e.v[h + j]) : 0.0f));
          auto* at = reinterpret_cast<Vec<TO, (W < V ? W : V)>*>(out + row * p.n + col + h);
          if constexpr (EPI == kPlain && sizeof(TO) == 4) {
            if (add) {
              const Vec<TO, (W < V ? W : V)> sum = *at;
#pragma unroll
              for (int j = 0; j < (W < V ? W : V); ++j) o.v[j] += sum.v[j];
            }
          }
          *at = o;
        }
      }
    }
  } else {
    const int col = col0 + lane;
    if (col < p.n) {
      const float b = bias ? to_float(bias[col]) : 0.0f;
#pragma unroll 8
      for (int r = 0; r < 32; ++r) {
        const long long row = row0 + r;
        if (row >= p.m) break;
        const float e = extra ? to_float(extra[row * p.n + col]) : 0.0f;
        float z;
        asm volatile("ld.shared.f32 %0, [%1];"
                     : "=f"(z)
                     : "r"(staging + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4)
                     : "memory");
        float value = finish<EPI, ACT>(z + b, e);
        if constexpr (EPI == kPlain && sizeof(TO) == 4) {
          if (add) value += out[row * p.n + col];
        }
        out[row * p.n + col] = from_float<TO>(value);
      }
    }
  }
}

template <int EPI, class TE, class TO>
SPLAT_DEV void store_patch(const ProductParams& p, uint32_t staging, const float (&v)[32],
                           long long row0, int col0, TO* out, bool add) {
  stage_patch(staging, v);
  if constexpr (EPI == kPlain) {
    write_patch<EPI, kNone, TE, TO>(p, staging, row0, col0, out, add);
  } else {
    switch (p.activation) {
      case kRelu: write_patch<EPI, kRelu, TE, TO>(p, staging, row0, col0, out, false); break;
      case kSilu: write_patch<EPI, kSilu, TE, TO>(p, staging, row0, col0, out, false); break;
      case kGelu: write_patch<EPI, kGelu, TE, TO>(p, staging, row0, col0, out, false); break;
      case kSigmoid: write_patch<EPI, kSigmoid, TE, TO>(p, staging, row0, col0, out, false); break;
      default: write_patch<EPI, kNone, TE, TO>(p, staging, row0, col0, out, false);
    }
  }
}

// ---- the kernel ------------------------------------------------------------------

template <class S>
constexpr bool kIsF16 = false;
template <>
inline constexpr bool kIsF16<f16> = true;

// Bytes of a plane of B's chunk.
template <bool MN>
__host__ __device__ constexpr int b_plane_bytes(int tile_n) {
  return MN ? (tile_n + 63) / 64 * (kChunk * 128) : tile_n * 128;
}

struct ProductTile {
  long long m0, k0, k1;
  int n0, split;
  SPLAT_DEV ProductTile(const ProductParams& p, long long t) {
    n0 = static_cast<int>(t % p.tiles_n) * p.tile_n;
    t /= p.tiles_n;
    m0 = (t % p.tiles_m) * kTileRows;
    split = static_cast<int>(t / p.tiles_m);
    k0 = split * p.k_per_split;
    k1 = min(k0 + p.k_per_split, p.k);
  }
};

template <class SA, int PA, bool AMN, class SB, int PB, bool BMN, class TE, class TO, int EPI>
__global__ void __launch_bounds__(kEpilogueWarps * 32 + producers(PA, PB) + 32,
                                  producers(PA, PB) == 128 ? 2 : 1)
    product_kernel(const __grid_constant__ ProductParams p) {
  constexpr int kProducers = producers(PA, PB), kAcc = accumulators(PA, PB);
  extern __shared__ unsigned char dynamic[];
  __shared__ alignas(8) unsigned long long full[kMaxStages], empty[kMaxStages], acc_full[2],
      acc_empty[2], resident_full, drained;
  __shared__ uint32_t tmem_base;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const uint32_t b_plane = b_plane_bytes<BMN>(p.tile_n);
  const uint32_t a_bytes = PA * kAPlane, b_bytes = PB * b_plane;
  const uint32_t staging = base;
  const uint32_t resident = staging + kEpilogueWarps * kStagingBytes;
  const int chunks_all = static_cast<int>((p.k + kChunk - 1) / kChunk);
  const uint32_t ring = resident + (p.resident ? chunks_all * b_bytes : 0);
  const uint32_t stage_bytes = a_bytes + (p.resident ? 0 : b_bytes);
  const int warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      tc::barrier_init(tc::shared_address(&full[i]), kProducers);
      tc::barrier_init(tc::shared_address(&empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::barrier_init(tc::shared_address(&acc_full[i]), 1);
      tc::barrier_init(tc::shared_address(&acc_empty[i]), kEpilogueWarps * 32);
    }
    tc::barrier_init(tc::shared_address(&resident_full), kProducers);
    tc::barrier_init(tc::shared_address(&drained), 1);
    tc::barrier_init_fence();
  }
  if (warp == 0) tc::tmem_alloc(tc::shared_address(&tmem_base), p.tmem_columns);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  bool ok = true;

  if (warp >= kEpilogueWarps && warp < kEpilogueWarps + kProducers / 32) {
    // ---- producers
    const int thread = threadIdx.x - kEpilogueWarps * 32;
    const SA* a = static_cast<const SA*>(p.a);
    const SB* b = static_cast<const SB*>(p.b);
    if (p.resident) {
      for (int c = 0; c < chunks_all; ++c)
        fill_chunk<SB, PB, BMN>(false, p.b_vector, resident + c * b_bytes, b_plane, p.tile_n, b, p.b_ld,
                                0, p.n, static_cast<long long>(c) * kChunk,
                                static_cast<int>(min(p.k - static_cast<long long>(c) * kChunk,
                                                     static_cast<long long>(kChunk))),
                                thread, kProducers);
      tc::fence_async_proxy();
      tc::barrier_arrive(tc::shared_address(&resident_full));
    }
    int stage = 0, in_flight = 0, landed = 0;
    uint32_t parity = 1;  // a fresh barrier's previous phase counts as complete
    for (long long t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
      const ProductTile tile(p, t);
      for (long long k = tile.k0; k < tile.k1; k += kChunk) {
        if (!(ok = tc::barrier_wait(tc::shared_address(&empty[stage]), parity))) break;
        const uint32_t at = ring + stage * stage_bytes;
        const int k_valid = static_cast<int>(min(tile.k1 - k, static_cast<long long>(kChunk)));
        fill_chunk<SA, PA, AMN>(p.lag, p.a_vector, at, kAPlane, kTileRows, a, p.a_ld, tile.m0,
                                p.m - tile.m0, k, k_valid, thread, kProducers);
        if (!p.resident)
          fill_chunk<SB, PB, BMN>(p.lag, p.b_vector, at + a_bytes, b_plane, p.tile_n, b, p.b_ld,
                                  tile.n0, p.n - tile.n0, k, k_valid, thread, kProducers);
        if (p.lag) {
          asm volatile("cp.async.commit_group;" ::: "memory");
          if (++in_flight > p.lag) {
            wait_copies(p.lag);
            tc::fence_async_proxy();
            tc::barrier_arrive(tc::shared_address(&full[landed]));
            if (++landed == p.stages) landed = 0;
            --in_flight;
          }
        } else {
          tc::fence_async_proxy();
          tc::barrier_arrive(tc::shared_address(&full[stage]));
        }
        if (++stage == p.stages) stage = 0, parity ^= 1;
      }
    }
    if (p.lag) {
      wait_copies(0);
      tc::fence_async_proxy();
      for (; in_flight; --in_flight) {
        tc::barrier_arrive(tc::shared_address(&full[landed]));
        if (++landed == p.stages) landed = 0;
      }
    }
  } else if (warp == kEpilogueWarps + kProducers / 32) {
    // ---- one thread issues the products
    if ((threadIdx.x & 31) == 0) {
      constexpr bool kBf16 = !(PA == 1 && PB == 1 && kIsF16<SA>);
      constexpr int kParts = PA > PB ? PA : PB;
      // the part of A in the first product of the smallest kind
      constexpr int first_part = kParts - 1 < PB ? 0 : kParts - PB;
      const uint32_t instruction = tc::instruction(kBf16, AMN, BMN, p.tile_n);
      // 128 m in one block of 64: the second half repeats the first, and its
      // rows of the result are not stored
      const uint32_t a_block = p.m > 64 ? kChunk * 128 : 0;
      if (p.resident) ok = tc::barrier_wait(tc::shared_address(&resident_full), 0);
      int stage = 0;
      uint32_t parity = 0, acc = 0, acc_parity = 1;
      for (long long t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
        const ProductTile tile(p, t);
        int c = 0;
        for (long long sum_k = tile.k0; sum_k < tile.k1 && ok; sum_k += p.k_per_sum) {
          if (!(ok = tc::barrier_wait(tc::shared_address(&acc_empty[acc]), acc_parity))) break;
          tc::fence_after_sync();
          const uint32_t d = tmem + acc * kAcc * p.tile_n;
          const long long sum_end = min(sum_k + p.k_per_sum, tile.k1);
          for (long long k = sum_k; k < sum_end; k += kChunk, ++c) {
            if (!(ok = tc::barrier_wait(tc::shared_address(&full[stage]), parity))) break;
            tc::fence_after_sync();
            const uint32_t at = ring + stage * stage_bytes;
            const uint32_t b_at = p.resident ? resident + c * b_bytes : at + a_bytes;
            const int steps = static_cast<int>(
                (min(sum_end - k, static_cast<long long>(kChunk)) + 15) / 16);
#pragma unroll
            for (int sum = kParts - 1; sum >= 0; --sum)
#pragma unroll
              for (int i = 0; i < PA; ++i) {
                const int j = sum - i;
                if (j < 0 || j >= PB) continue;
                // the first product into an accumulator overwrites it
                const bool own = sum == 0 && kAcc == 2;
                const bool first = k == sum_k && (own || (sum == kParts - 1 && i == first_part));
                for (int s = 0; s < steps; ++s) {
                  const uint32_t ao = at + i * kAPlane + s * (AMN ? tc::kStepMn : tc::kStepK);
                  const uint32_t bo = b_at + j * b_plane + s * (BMN ? tc::kStepMn : tc::kStepK);
                  tc::mma(d + (own ? 0 : (kAcc - 1) * p.tile_n),
                          AMN ? tc::descriptor_mn_major(ao, a_block) : tc::descriptor_k_major(ao),
                          BMN ? tc::descriptor_mn_major(bo, kChunk * 128)
                              : tc::descriptor_k_major(bo),
                          instruction, !(first && s == 0));
                }
              }
            tc::commit(tc::shared_address(&empty[stage]));
            if (++stage == p.stages) stage = 0, parity ^= 1;
          }
          tc::commit(tc::shared_address(&acc_full[acc]));
          acc ^= 1;
          if (acc == 0) acc_parity ^= 1;
        }
      }
      // whichever way the loop ended, no product is in flight past this point
      tc::commit(tc::shared_address(&drained));
      ok = tc::barrier_wait(tc::shared_address(&drained), 0) && ok;
    }
  } else if (warp < kEpilogueWarps) {
    // ---- epilogue
    const int lane_block = warp & 3, half = warp >> 2;
    uint32_t acc = 0, parity = 0;
    for (long long t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
      const ProductTile tile(p, t);
      const long long row0 = tile.m0 + lane_block * 32;
      TO* out = static_cast<TO*>(p.out) + static_cast<long long>(tile.split) * p.m * p.n;
      for (long long sum_k = tile.k0; sum_k < tile.k1; sum_k += p.k_per_sum) {
        if (!(ok = tc::barrier_wait(tc::shared_address(&acc_full[acc]), parity))) break;
        tc::fence_after_sync();
        for (int c = half; c * 32 < p.tile_n; c += kEpilogueWarps / 4) {
          const int col0 = tile.n0 + c * 32;
          if (col0 >= p.n || row0 >= p.m) break;
          const uint32_t from = tmem + (lane_block << 21) + acc * kAcc * p.tile_n + c * 32;
          float v[32];
          tc::tmem_load32(from, v);
          if constexpr (kAcc == 2) {
            float low[32];
            tc::tmem_load32(from + p.tile_n, low);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += low[i];
          }
          store_patch<EPI, TE, TO>(p, staging + warp * kStagingBytes, v, row0, col0, out,
                                   sum_k != tile.k0);
        }
        tc::fence_before_sync();
        tc::barrier_arrive(tc::shared_address(&acc_empty[acc]));
        acc ^= 1;
        if (acc == 0) parity ^= 1;
      }
    }
  }
  if (!ok) atomicCAS(p.error, 0, kDeviceTimeout);
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_free(tmem, p.tmem_columns);
}

}  // namespace feature
}  // namespace splat
