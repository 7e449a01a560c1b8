// C(m, n) = sum_k A(m, k) B(n, k) on the tensor cores, with the epilogues of a
// linear layer and its backward.
//
// Numbers.  Operands are 16-bit for tcgen05.mma.  fp32 ones are split into three
// bf16 parts, v = v0 + v1 + v2 with v_i rounded from what v_0 .. v_{i-1} leave (8
// digits each), and the products of parts i and j with i + j < 3 are summed,
// which reproduces an fp32 product to 2^-24.  The dz of 16-bit layers is two
// values of their type (take_first).  Accumulators are fp32 in tensor memory.
//
// Work.  A persistent block takes 128 x NT tiles.  64-wide chunks of k go from
// global memory into a ring of stages: 16-bit operands with 16-byte rows by
// tensor copies that one thread starts, all others through four or eight
// producer warps (converting and zero-filling on the way: any row length, any
// row count).  These take the tiles of a short-rowed A, which are contiguous,
// from bulk copies that run two tiles ahead.  What would be converted again and
// again (fp32 operands of several tiles, long unaligned rows) is laid out as
// planes of parts by a pass before, and copied as well.  One warp issues
// the products, and eight epilogue warps take the finished accumulators, of
// which there are two or four, so that loads, products and epilogues of
// neighbouring tiles overlap.  Where the whole of B fits beside the ring it is
// loaded once per block.
//
// Bound by memory and the epilogue's arithmetic where k and n are small (64 -> 64
// bf16 silu with residual over 1600x1200 rows 132 us, 112 us of copying; 32 -> 64
// silu 96 us, 56 us of copying and 55 of two special-function instructions a
// value).  Wide fp32 layers (300 -> 300 over 200000 rows 401 us for 216 GFLOP of
// parts, the tensor pipe busy 34 %) have a ring of one stage: three parts of 64 k
// of both operands are 96 KB, beside which the epilogue's patches leave no room
// for another, so that a stage's copies wait for its products.
#pragma once
#include <type_traits>

#include "feature_common.cuh"
#include "tensor_core.cuh"

namespace splat {
namespace feature {

constexpr int kTileRows = 128;
constexpr int kChunk = 64;             // k of a stage: 128 bytes of 16-bit values
constexpr int kEpilogueWarps = 8;                  // epilogue warps
constexpr int kMaxStages = 8, kMaxAccumulators = 4;
constexpr int kAPlane = kTileRows * 128;

// Producer threads: operands that are split always pass through registers, so
// there it is threads that keep loads in flight.  Two-part ones always lie in
// memory as two planes and are copied.
__host__ __device__ constexpr int producers(int pa, int pb) {
  return pa <= 2 && pb <= 2 ? 128 : 256;
}
// fp32 operands keep the products of lower parts in an accumulator of their
// own: the tensor core truncates its sums, so each addition at full magnitude
// costs up to 2^-24, and the lower products must not add to their number.
// 16-bit results do not show it.
__host__ __device__ constexpr int accumulators(int pa, int pb) { return pa == 3 || pb == 3 ? 2 : 1; }
// k that such an accumulator sums before it is added up in fp32 (32 additions).
constexpr int kExactSum = 512;
// Additions into an accumulator of a 16-bit layer: each costs it up to 2^-23, so
// that they stay below a quarter of half a step of f16.
constexpr int kMostAdditions = 1024;

// act(C + bias) + residual; dy act'(C + bias); C.
enum Epilogue : int { kForward = 0, kSlope = 1, kPlain = 2 };

struct ProductParams {
  CUtensorMap a_map, b_map, extra_map, out_map;
  CUtensorMap a_second_map, out_second_map;  // of the second of two parts
  int copy_operands, copy_extra, copy_out;  // by tensor copies
  // the operands' parts lie in memory as 16-bit planes of so many rows (0: they
  // are made on the way)
  int a_plane_rows, b_plane_rows;
  int raw_bytes;   // of a tile of A as it is in memory, copied ahead; 0: none
  int staging;     // bytes of an epilogue warp
  long long m, k;  // k of all splits
  int n;
  // row-major sources: A is (m, k) rows or, transposed, (k, m); B likewise
  const void* a;
  const void* b;
  const void* a_second;  // A in two parts: the second's plane, like a's
  long long a_ld, b_ld;
  int a_vector, b_vector;  // bytes that every row start and chunk is aligned to
  long long k_per_split;   // a multiple of kChunk unless there is one split
  long long k_per_sum;     // of one accumulator; the tile's sums are added in `out` (fp32)
  int held;                // or, of 16-bit results, in shared memory
  int splits, tile_n;
  int accumulate;          // fp32 results of a plain product are added to what `out` holds
  uint32_t tiles_n, tiles_m, tiles;  // tiles = splits * tiles_m * tiles_n, below 2^31
  int stages, resident, activation;
  // accumulators of a block: 2, whose columns the two groups of four epilogue
  // warps share; or 4 (alternate), each finished by one group, for tiles of 32
  // columns, which leave a second group nothing to do
  int accumulators, alternate;
  uint32_t tmem_columns;
  const void* bias;   // (n) or NULL
  const void* extra;  // residual or dy (m, n), or NULL
  void* out;          // (splits, m, n), rows out_ld values apart
  void* out_second;   // kSlope: dz in two parts, the second's plane; or NULL
  long long out_ld;
  float* column_sums; // kSlope: (4 tiles_m, n) sums of dz over 32 rows each, or NULL
  int extra_vector, out_vector;  // their rows are whole 16-byte pieces
  int bias_shared;    // values of the bias kept in shared memory (0: too many)
  int* error;
};

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

// Part of two values as a packed pair, and what it leaves of them.  A part that
// others follow is at most bf16's largest value, so that the last one brings an
// infinity, which then meets the other operand's leading part alone.
template <bool LAST>
SPLAT_DEV uint32_t take_part(float& a, float& b) {
  uint32_t u;
  if constexpr (LAST)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
  else
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(b), "f"(a));
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
      for (int p = 0; p < P; ++p)
        w[p][j] = p == P - 1 ? take_part<true>(a, b) : take_part<false>(a, b);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) out[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
  }
}

// The same from shared memory.
template <class S, int VB>
SPLAT_DEV Vec<S, 8> load8_shared(uint32_t p, int valid) {
  Vec<S, 8> r;
  constexpr int E = VB / static_cast<int>(sizeof(S));  // values per load
#pragma unroll
  for (int j = 0; j < 8 / E; ++j) {
    Vec<S, E> part;
    if (j * E < valid) {
      if constexpr (VB == 16) {
        const float4 u = load_shared(p + j * 16);
        part = reinterpret_cast<const Vec<S, E>&>(u);
      } else if constexpr (VB == 8) {
        float2 u;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                     : "=f"(u.x), "=f"(u.y)
                     : "r"(p + j * 8)
                     : "memory");
        part = reinterpret_cast<const Vec<S, E>&>(u);
      } else if constexpr (VB == 4) {
        float u;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(u) : "r"(p + j * 4) : "memory");
        part = reinterpret_cast<const Vec<S, E>&>(u);
      } else {
        unsigned short u;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(p + j * 2) : "memory");
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

// Fills `rows` rows of a block (and of its parts' planes, `plane` bytes apart)
// with `pieces` (2, 4, 6 or 8) 16-byte pieces each; load(row, piece, valid)
// gives a piece's values.  Rows from rows_valid and columns from cols_valid on
// are zero.
template <class S, int P, int U, class L>
SPLAT_DEV void fill_pieces(uint32_t dst, uint32_t plane, int rows, int pieces,
                           long long rows_valid, long long cols_valid, int thread, int threads,
                           L load) {
  // i / pieces as a product and a shift, exact for i < 2^15
  const int factor = pieces == 6 ? 10923 : 65536 / pieces;
  const int total = rows * pieces;
  for (int i0 = thread; i0 < total; i0 += U * threads) {
    Vec<S, 8> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * threads, row = (i * factor) >> 16, piece = i - row * pieces;
      const int left = static_cast<int>(min(cols_valid, 1LL << 20)) - piece * 8;
      const int valid = i < total && row < rows_valid && left > 0 ? min(left, 8) : 0;
      v[u] = load(row, piece, valid);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * threads, row = (i * factor) >> 16, piece = i - row * pieces;
      if (i < total) {
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
  const auto run = [&](auto bytes) {
    constexpr int VB = decltype(bytes)::value;
    // pieces in flight per thread
    fill_pieces<S, P, P == 1 && VB == 16 ? 8 : 4>(
        dst, plane, rows, pieces, rows_valid, cols_valid, thread, threads,
        [&](int row, int piece, int valid) {
          return load8<S, VB>(src + row * ld + piece * 8, valid);
        });
  };
  if (vector >= 16) run(std::integral_constant<int, 16>{});
  else if (vector >= 8) run(std::integral_constant<int, 8>{});
  else if (vector >= 4 || sizeof(S) == 4) run(std::integral_constant<int, 4>{});
  else run(std::integral_constant<int, static_cast<int>(sizeof(S))>{});
}

// From rows of row_bytes in shared memory.
template <class S, int P>
SPLAT_DEV void fill_shared(int vector, uint32_t dst, uint32_t plane, int rows, int pieces,
                           uint32_t src, int row_bytes, int rows_valid, int cols_valid,
                           int thread, int threads) {
  const auto run = [&](auto bytes) {
    constexpr int VB = decltype(bytes)::value;
    fill_pieces<S, P, 2>(dst, plane, rows, pieces, rows_valid, cols_valid, thread, threads,
                         [&](int row, int piece, int valid) {
                           return load8_shared<S, VB>(
                               src + row * row_bytes + piece * 8 * static_cast<int>(sizeof(S)),
                               valid);
                         });
  };
  if (vector >= 16) run(std::integral_constant<int, 16>{});
  else if (vector >= 8) run(std::integral_constant<int, 8>{});
  else if (vector >= 4 || sizeof(S) == 4) run(std::integral_constant<int, 4>{});
  else run(std::integral_constant<int, static_cast<int>(sizeof(S))>{});
}

// A contiguous run of values (its start 16-byte aligned) into shared memory by
// one bulk copy; the values behind its last whole 16 bytes are stored by the
// calling thread.  The barrier takes this thread's arrival.
template <class S>
SPLAT_DEV void copy_run(uint32_t dst, const S* src, int values, uint32_t bar) {
  const int bytes = values * static_cast<int>(sizeof(S)), whole = bytes & ~15;
  for (int i = whole / static_cast<int>(sizeof(S)); i < values; ++i) {
    const uint32_t to = dst + i * static_cast<int>(sizeof(S));
    if constexpr (sizeof(S) == 4)
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(src[i]) : "memory");
    else
      asm volatile("st.shared.u16 [%0], %1;" ::"r"(to),
                   "h"(reinterpret_cast<const unsigned short&>(src[i]))
                   : "memory");
  }
  if (whole) {
    tc::barrier_expect(bar, whole);
    tc::bulk_in(dst, src, whole, bar);
  } else {
    tc::barrier_arrive(bar);
  }
}

// One operand's chunk: `width` m or n from mn0 and kChunk k from k0 (k_valid of
// them real).  K-major operands are one block of `width` rows; MN-major ones
// are blocks of 64 m or n, each of kChunk rows.
template <class S, int P, bool MN>
SPLAT_DEV void fill_chunk(int vector, uint32_t dst, uint32_t plane, int width,
                          const S* src, long long ld, long long mn0, long long mn_valid,
                          long long k0, int k_valid, int thread, int threads) {
  const int rows = MN ? min((k_valid + 15) / 16 * 16, kChunk) : width;
  const int pieces = MN ? 8 : min((k_valid + 15) / 16 * 2, 8);
  for (int b = 0; b == 0 || (MN && b * 64 < width && b * 64 < mn_valid); ++b) {
    const S* corner = MN ? src + k0 * ld + mn0 + b * 64 : src + mn0 * ld + k0;
    const long long rows_valid = MN ? k_valid : mn_valid;
    const long long cols_valid = MN ? mn_valid - b * 64 : k_valid;
    const uint32_t at = dst + b * (kChunk * 128);
    fill<S, P>(vector, at, plane, rows, pieces, corner, ld, rows_valid, cols_valid, thread,
               threads);
  }
}

// The same by tensor copies of boxes of 64 columns (MN-major: of 64 k rows);
// returns the bytes that will arrive.
template <bool MN>
SPLAT_DEV uint32_t chunk_bytes(int width, long long mn_valid) {
  return MN ? static_cast<uint32_t>(min((mn_valid + 63) / 64, (width + 63LL) / 64)) * (kChunk * 128)
            : width * 128;
}
template <int P, bool MN>
SPLAT_DEV void copy_chunk(const CUtensorMap* map, const CUtensorMap* second_map, uint32_t dst,
                          uint32_t plane, int plane_rows, int width, long long mn0,
                          long long mn_valid, long long k0, uint32_t bar) {
#pragma unroll
  for (int i = 0; i < P; ++i, dst += plane) {
    if (P == 2 && i == 1) map = second_map, plane_rows = 0;
    if constexpr (MN) {
      for (int b = 0; b * 64 < width && b * 64 < mn_valid; ++b)
        tc::copy_in(dst + b * (kChunk * 128), map, static_cast<int>(mn0) + b * 64,
                    static_cast<int>(k0) + i * plane_rows, bar);
    } else {
      tc::copy_in(dst, map, static_cast<int>(k0), static_cast<int>(mn0) + i * plane_rows, bar);
    }
  }
}

// ---- epilogue ------------------------------------------------------------------

// A patch of 32 rows x W values of T in a warp's staging memory: 16-byte
// pieces, permuted so that both a lane's own row and 16 bytes per lane along
// rows are accessed without bank conflicts.
template <class T, int W = 32>
struct Patch {
  static constexpr int kPieces = W * sizeof(T) / 16;  // of a row
  static constexpr int V = 16 / sizeof(T);            // values of a piece
  uint32_t base;
  SPLAT_DEV uint32_t at(int row, int piece) const {
    const int turn = kPieces == 2 ? (row >> 2) & 1 : kPieces == 4 ? (row >> 1) & 3 : row & 7;
    return base + row * (W * sizeof(T)) + ((piece ^ turn) << 4);
  }

  // Rows of ld values in shared memory -> staging.
  SPLAT_DEV void load_shared_rows(uint32_t src, int ld, int rows, int cols, bool vector) const {
    const int lane = threadIdx.x & 31;
    constexpr int kSize = sizeof(T);
    if (vector) {
      constexpr int kRows = 32 / kPieces;
      const int piece = lane % kPieces, r0 = lane / kPieces;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int r = i * kRows + r0;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < rows && piece * V < cols) v = load_shared(src + (r * ld + piece * V) * kSize);
        store_shared(at(r, piece), reinterpret_cast<const uint4&>(v));
      }
    } else {
      constexpr int kRows = 32 / W;
      const int col = lane % W;
#pragma unroll 8
      for (int i = 0; i < W; ++i) {
        const int r = i * kRows + lane / W;
        const uint32_t from = src + (r * ld + col) * kSize;
        const uint32_t to = at(r, col / V) + col % V * kSize;
        const bool in = r < rows && col < cols;
        if constexpr (kSize == 4) {
          float v = 0.0f;
          if (in) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(from) : "memory");
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
        } else {
          unsigned short v = 0;
          if (in) asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(v) : "memory");
        }
      }
    }
  }

  // Global memory (its corner, rows of ld values) -> staging.  vector: rows
  // start on 16 bytes and cols is a whole number of pieces.
  SPLAT_DEV void load(const T* src, long long ld, int rows, int cols, bool vector) const {
    const int lane = threadIdx.x & 31;
    if (vector) {
      constexpr int kRows = 32 / kPieces;
      const int piece = lane % kPieces, r0 = lane / kPieces;
      uint4 v[kPieces];
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int r = i * kRows + r0;
        v[i] = make_uint4(0, 0, 0, 0);
        if (r < rows && piece * V < cols)
          v[i] = __ldg(reinterpret_cast<const uint4*>(src + r * ld + piece * V));
      }
#pragma unroll
      for (int i = 0; i < kPieces; ++i) store_shared(at(i * kRows + r0, piece), v[i]);
    } else {
      constexpr int kRows = 32 / W;
      const int col = lane % W;
      src += lane / W * ld + col;
#pragma unroll 8
      for (int i = 0; i < W; ++i) {
        const int r = i * kRows + lane / W;
        const T v = r < rows && col < cols ? src[i * kRows * ld] : from_float<T>(0.0f);
        const uint32_t to = at(r, col / V) + col % V * sizeof(T);
        if constexpr (sizeof(T) == 4)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
        else
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(to),
                       "h"(reinterpret_cast<const unsigned short&>(v))
                       : "memory");
      }
    }
  }

  // Adds what this warp stored in global memory (fp32 only) onto the staging.
  SPLAT_DEV void add(const T* src, long long ld, int rows, int cols, bool vector) const {
    static_assert(sizeof(T) == 4);
    const int lane = threadIdx.x & 31;
    if (vector) {
      constexpr int kRows = 32 / kPieces;
      const int piece = lane % kPieces, r0 = lane / kPieces;
      if (piece * V >= cols) return;
      src += r0 * ld + piece * V;
#pragma unroll
      for (int i = 0; i < kPieces; ++i, src += kRows * ld) {
        if (i * kRows + r0 >= rows) break;
        const uint32_t to = at(i * kRows + r0, piece);
        float4 v = load_shared(to);
        const float4 o = *reinterpret_cast<const float4*>(src);
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        store_shared(to, reinterpret_cast<const uint4&>(v));
      }
    } else {
      constexpr int kRows = 32 / W;
      const int col = lane % W;
      if (col >= cols) return;
      src += lane / W * ld + col;
      for (int r = lane / W; r < rows; r += kRows, src += kRows * ld) {
        const uint32_t to = at(r, col / V) + col % V * sizeof(T);
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(to) : "memory");
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(v + *src) : "memory");
      }
    }
  }

  // Staging -> global memory; add (fp32 only): onto what is there.
  SPLAT_DEV void store(T* dst, long long ld, int rows, int cols, bool vector, bool add) const {
    const int lane = threadIdx.x & 31;
    if (vector) {
      constexpr int kRows = 32 / kPieces;
      const int piece = lane % kPieces, r0 = lane / kPieces;
      if (piece * V >= cols) return;
      dst += r0 * ld + piece * V;
#pragma unroll
      for (int i = 0; i < kPieces; ++i, dst += kRows * ld) {
        if (i * kRows + r0 >= rows) break;
        float4 v = load_shared(at(i * kRows + r0, piece));
        if constexpr (sizeof(T) == 4) {
          if (add) {
            const float4 o = *reinterpret_cast<const float4*>(dst);
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
          }
        }
        *reinterpret_cast<float4*>(dst) = v;
      }
    } else {
      constexpr int kRows = 32 / W;
      const int col = lane % W;
      if (col >= cols) return;
      dst += lane / W * ld + col;
#pragma unroll 4
      for (int r = lane / W; r < rows; r += kRows, dst += kRows * ld) {
        const uint32_t from = at(r, col / V) + col % V * sizeof(T);
        if constexpr (sizeof(T) == 4) {
          float v;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(from) : "memory");
          *dst = add ? v + *dst : v;
        } else {
          unsigned short v;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
          *dst = reinterpret_cast<const T&>(v);
        }
      }
    }
  }
};

// The epilogue's arithmetic on a lane's row: v becomes act(v) + e, or
// e act'(v); the extra values e lie in the patch.
template <int EPI, int ACT, class TE, int W>
SPLAT_DEV void finish_row(const Patch<TE, W>& extra, bool with_extra, float (&v)[W]) {
  const int lane = threadIdx.x & 31;
  constexpr int V = Patch<TE, W>::V;
#pragma unroll
  for (int piece = 0; piece < Patch<TE, W>::kPieces; ++piece) {
    float* z = v + piece * V;
    if constexpr (EPI == kForward) {
#pragma unroll
      for (int j = 0; j < V; j += 2) activate2<ACT, sizeof(TE) == 4>(z[j], z[j + 1]);
    }
    if (EPI == kSlope || with_extra) {
      const float4 raw = load_shared(extra.at(lane, piece));
      float e[V];
      widen<TE, V>(reinterpret_cast<const Vec<TE, V>&>(raw), e);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        if constexpr (EPI == kForward)
          unpack2(add2(pack2(z[j], z[j + 1]), pack2(e[j], e[j + 1])), z[j], z[j + 1]);
        else {
          slope2<ACT, sizeof(TE) == 4>(z[j], z[j + 1]);
          unpack2(mul2(pack2(z[j], z[j + 1]), pack2(e[j], e[j + 1])), z[j], z[j + 1]);
        }
      }
    }
  }
}

// The sums over a warp's rows of W columns, a lane's row each: halving steps,
// after which lane l has column l of 32 (of 16: column l / 2, in two lanes).
template <int HALF, int BIT, int W>
SPLAT_DEV void fold_rows(float (&v)[W]) {
  if constexpr (HALF > 0) {
    const bool upper = threadIdx.x & BIT;
#pragma unroll
    for (int j = 0; j < HALF; ++j) {
      const float mine = upper ? v[j + HALF] : v[j], theirs = upper ? v[j] : v[j + HALF];
      v[j] = mine + __shfl_xor_sync(0xffffffffu, theirs, BIT);
    }
    fold_rows<HALF / 2, BIT / 2>(v);
  }
}
template <int W>
SPLAT_DEV float sum_rows(const float (&row)[W]) {
  float v[W];
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] = row[j];
  fold_rows<W / 2, 16>(v);
  return W == 16 ? v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1) : v[0];
}

// ---- operands as planes ----------------------------------------------------------

// src (rows, cols) as `P` planes of plane_rows x ld 16-bit parts; rows behind
// the last are zero, columns behind the last are not written (nor read).
template <class S, int P, int VB>
__global__ void __launch_bounds__(256)
    split_kernel(const S* src, long long rows, int cols, int pieces, long long plane_rows, int ld,
                 uint16_t* dst) {
  const long long total = plane_rows * pieces;
  constexpr int U = 4;
  for (long long i0 = blockIdx.x * 256LL + threadIdx.x; i0 < total; i0 += U * 256LL * gridDim.x) {
    Vec<S, 8> v[U];
    long long row[U];
    int piece[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * 256LL * gridDim.x;
      row[u] = i >= total ? plane_rows
               : total <= 0xffffffffLL
                   ? static_cast<uint32_t>(i) / static_cast<uint32_t>(pieces)
                   : i / pieces;
      piece[u] = static_cast<int>(i - row[u] * pieces);
      v[u] = load8<S, VB>(src + row[u] * cols + piece[u] * 8,
                          row[u] < rows ? min(cols - piece[u] * 8, 8) : 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] < plane_rows) {
        uint4 parts[P];
        to_parts<S, P>(v[u], parts);
#pragma unroll
        for (int p = 0; p < P; ++p)
          *reinterpret_cast<uint4*>(dst + (p * plane_rows + row[u]) * ld + piece[u] * 8) = parts[p];
      }
  }
}

// ---- the kernel ------------------------------------------------------------------

// Bytes of a plane of B's chunk.
template <bool MN>
__host__ __device__ constexpr int b_plane_bytes(int tile_n) {
  return MN ? (tile_n + 63) / 64 * (kChunk * 128) : tile_n * 128;
}

struct ProductTile {
  long long m0, k0, k1;
  int n0, split;
  // divisions only where there is something to divide: every warp passes here
  // for every tile
  SPLAT_DEV ProductTile(const ProductParams& p, uint32_t t) {
    uint32_t rest = t;
    n0 = split = 0;
    if (p.tiles_n > 1) {
      rest = t / p.tiles_n;
      n0 = (t - rest * p.tiles_n) * p.tile_n;
    }
    if (p.splits > 1) {
      split = rest / p.tiles_m;
      rest -= split * p.tiles_m;
    }
    m0 = static_cast<long long>(rest) * kTileRows;
    k0 = split * p.k_per_split;
    k1 = min(k0 + p.k_per_split, p.k);
  }
};

template <class SA, int PA, bool AMN, class SB, int PB, bool BMN, class TE, class TO, int EPI>
__global__ void __launch_bounds__(producers(PA, PB) == 128 ? 512 : 544,
                                  producers(PA, PB) == 128 ? 2 : 1)  // 64 and 120 registers
    product_kernel(const __grid_constant__ ProductParams p) {
  constexpr int kProducers = producers(PA, PB), kAcc = accumulators(PA, PB);
  extern __shared__ unsigned char dynamic[];
  __shared__ alignas(8) unsigned long long full[kMaxStages], empty[kMaxStages],
      acc_full[kMaxAccumulators], acc_empty[kMaxAccumulators], resident_full, drained, extra_full[kEpilogueWarps], raw_full[2],
      raw_read[2];
  __shared__ uint32_t tmem_base;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const uint32_t b_plane = b_plane_bytes<BMN>(p.tile_n);
  const uint32_t a_bytes = PA * kAPlane, b_bytes = PB * b_plane;
  const uint32_t bias_at = base + kEpilogueWarps * p.staging;
  const uint32_t resident = bias_at + (p.bias_shared * 4 + 1023) / 1024 * 1024;
  const int chunks_all = static_cast<int>((p.k + kChunk - 1) / kChunk);
  const uint32_t ring = resident + (p.resident ? chunks_all * b_bytes : 0);
  const uint32_t stage_bytes = a_bytes + (p.resident ? 0 : b_bytes);
  const int warp = tc::uniform(threadIdx.x >> 5);
  // copies need no more than one producer warp
  const int product_warp = kEpilogueWarps + (p.copy_operands ? 1 : kProducers / 32);

  if (threadIdx.x == 0) {
    const int arrivals = p.copy_operands ? 1 : p.raw_bytes ? kProducers / 2 : kProducers;
    for (int i = 0; i < kEpilogueWarps; ++i)
      tc::barrier_init(tc::shared_address(&extra_full[i]), 1);
    for (int i = 0; i < p.stages; ++i) {
      tc::barrier_init(tc::shared_address(&full[i]), arrivals);
      tc::barrier_init(tc::shared_address(&empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::barrier_init(tc::shared_address(&raw_full[i]), 1);
      tc::barrier_init(tc::shared_address(&raw_read[i]), kProducers / 2);
    }
    for (int i = 0; i < p.accumulators; ++i) {
      tc::barrier_init(tc::shared_address(&acc_full[i]), 1);
      tc::barrier_init(tc::shared_address(&acc_empty[i]),
                       kEpilogueWarps * (p.alternate ? 16 : 32));
    }
    tc::barrier_init(tc::shared_address(&resident_full), p.copy_operands ? 1 : kProducers);
    tc::barrier_init(tc::shared_address(&drained), 1);
    tc::barrier_init_fence();
  }
  if (p.bias) {
    for (int i = threadIdx.x; i < p.bias_shared; i += blockDim.x)
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(bias_at + i * 4),
                   "f"(i < p.n ? to_float(static_cast<const TE*>(p.bias)[i]) : 0.0f)
                   : "memory");
  }
  if (warp == 0) tc::tmem_alloc(tc::shared_address(&tmem_base), p.tmem_columns);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tc::uniform(tmem_base);
  bool ok = true;

  if (warp >= kEpilogueWarps && warp < product_warp) {
    // ---- producers
    const int thread = threadIdx.x - kEpilogueWarps * 32;
    int stage = 0;
    uint32_t parity = 1;  // a fresh barrier's previous phase counts as complete
    if (p.copy_operands) {
      if (thread == 0) {
        if (p.resident) {
          const uint32_t bar = tc::shared_address(&resident_full);
          tc::barrier_expect(bar, chunks_all * PB * chunk_bytes<BMN>(p.tile_n, p.n));
          for (int c = 0; c < chunks_all; ++c)
            copy_chunk<PB, BMN>(&p.b_map, nullptr, resident + c * b_bytes, b_plane,
                                p.b_plane_rows, p.tile_n, 0, p.n,
                                static_cast<long long>(c) * kChunk, bar);
        }
        int started = 0;  // stages that have been filled at least once
        for (uint32_t t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
          const ProductTile tile(p, t);
          for (long long k = tile.k0; k < tile.k1; k += kChunk) {
            if (!(ok = tc::barrier_wait(tc::shared_address(&empty[stage]), parity))) break;
            const uint32_t at = ring + stage * stage_bytes, bar = tc::shared_address(&full[stage]);
            tc::barrier_expect(bar,
                               PA * chunk_bytes<AMN>(kTileRows, p.m - tile.m0) +
                                   (p.resident ? 0
                                               : PB * chunk_bytes<BMN>(p.tile_n, p.n - tile.n0)));
            copy_chunk<PA, AMN>(&p.a_map, &p.a_second_map, at, kAPlane, p.a_plane_rows,
                                kTileRows, tile.m0, p.m - tile.m0, k, bar);
            if (!p.resident)
              copy_chunk<PB, BMN>(&p.b_map, nullptr, at + a_bytes, b_plane, p.b_plane_rows,
                                  p.tile_n, tile.n0, p.n - tile.n0, k, bar);
            started = max(started, stage + 1);
            if (++stage == p.stages) stage = 0, parity ^= 1;
          }
        }
        // no copy is in flight past this point, also after a wait that ran out:
        // parity ^ 1 is the phase of the ring's current round, parity the last one's
        if (p.resident) ok = tc::barrier_wait(tc::shared_address(&resident_full), 0) && ok;
        for (int i = 0; i < started; ++i)
          ok = tc::barrier_wait(tc::shared_address(&full[i]), i < stage ? parity ^ 1 : parity) && ok;
      }
    } else if constexpr (PA != 2) {
      const SA* a = static_cast<const SA*>(p.a);
      const SB* b = static_cast<const SB*>(p.b);
      if (p.resident) {
        for (int c = 0; c < chunks_all; ++c)
          fill_chunk<SB, PB, BMN>(p.b_vector, resident + c * b_bytes, b_plane, p.tile_n, b, p.b_ld,
                                  0, p.n, static_cast<long long>(c) * kChunk,
                                  static_cast<int>(min(p.k - static_cast<long long>(c) * kChunk,
                                                       static_cast<long long>(kChunk))),
                                  thread, kProducers);
        tc::fence_async_proxy();
        tc::barrier_arrive(tc::shared_address(&resident_full));
      }
      if (!AMN && p.raw_bytes) {
        // two groups of producers take turns at the tiles, whose fixed costs
        // (waits, the proxy fence) then overlap; each has a buffer of its own,
        // which bulk copies fill while the other group converts
        constexpr int kGroup = kProducers / 2;
        const int group = thread / kGroup, own = thread % kGroup;
        const uint32_t raw_at = ring + p.stages * stage_bytes + group * p.raw_bytes;
        const uint32_t raw_bar = tc::shared_address(&raw_full[group]);
        const uint32_t read_bar = tc::shared_address(&raw_read[group]);
        const int row_bytes = static_cast<int>(p.k) * static_cast<int>(sizeof(SA));
        uint32_t copied = 0;  // tiles, by the group's first thread
        const auto copy_tile = [&](uint32_t t) {
          const long long m0 = ProductTile(p, t).m0;
          copy_run<SA>(raw_at, a + m0 * p.k,
                       static_cast<int>(min(p.m - m0, static_cast<long long>(kTileRows)) * p.k),
                       raw_bar);
          ++copied;
        };
        // and stages of its own, so that its waits on a stage follow one another
        const int first_stage = group ? (p.stages + 1) / 2 : 0;
        const int end_stage = group ? p.stages : (p.stages + 1) / 2;
        stage = first_stage;
        const uint32_t step = 2 * gridDim.x, first = blockIdx.x + group * gridDim.x;
        if (own == 0 && first < p.tiles) copy_tile(first);
        uint32_t round = 0;
        for (uint32_t t = first; t < p.tiles && ok; t += step, round ^= 1) {
          const ProductTile tile(p, t);
          const int rows =
              static_cast<int>(min(p.m - tile.m0, static_cast<long long>(kTileRows)));
          if (!(ok = tc::barrier_wait(raw_bar, round))) break;
          for (int c = 0; c < chunks_all; ++c) {
            if (!(ok = tc::barrier_wait(tc::shared_address(&empty[stage]), parity))) break;
            const uint32_t at = ring + stage * stage_bytes;
            const int k_valid = min(static_cast<int>(p.k) - c * kChunk, kChunk);
            fill_shared<SA, PA>(p.a_vector, at, kAPlane, kTileRows,
                                min((k_valid + 15) / 16 * 2, 8),
                                raw_at + c * kChunk * static_cast<int>(sizeof(SA)), row_bytes,
                                rows, k_valid, own, kGroup);
            if (!p.resident)
              fill_chunk<SB, PB, BMN>(p.b_vector, at + a_bytes, b_plane, p.tile_n, b, p.b_ld,
                                      tile.n0, p.n - tile.n0, c * kChunk, k_valid, own, kGroup);
            tc::fence_async_proxy();
            tc::barrier_arrive(tc::shared_address(&full[stage]));
            if (++stage == end_stage) stage = first_stage, parity ^= 1;
          }
          if (!ok) break;
          tc::barrier_arrive(read_bar);
          if (own == 0 && p.tiles - t > step) {
            if (!(ok = tc::barrier_wait(read_bar, round))) break;
            copy_tile(t + step);
          }
        }
        // no copy is in flight past this point, also after a wait that ran out
        if (copied) ok = tc::barrier_wait(raw_bar, (copied - 1) & 1) && ok;
      } else {
        for (uint32_t t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
          const ProductTile tile(p, t);
          for (long long k = tile.k0; k < tile.k1; k += kChunk) {
            if (!(ok = tc::barrier_wait(tc::shared_address(&empty[stage]), parity))) break;
            const uint32_t at = ring + stage * stage_bytes;
            const int k_valid = static_cast<int>(min(tile.k1 - k, static_cast<long long>(kChunk)));
            fill_chunk<SA, PA, AMN>(p.a_vector, at, kAPlane, kTileRows, a, p.a_ld, tile.m0,
                                    p.m - tile.m0, k, k_valid, thread, kProducers);
            if (!p.resident)
              fill_chunk<SB, PB, BMN>(p.b_vector, at + a_bytes, b_plane, p.tile_n, b, p.b_ld,
                                      tile.n0, p.n - tile.n0, k, k_valid, thread, kProducers);
            tc::fence_async_proxy();
            tc::barrier_arrive(tc::shared_address(&full[stage]));
            if (++stage == p.stages) stage = 0, parity ^= 1;
          }
        }
      }
    }
  } else if (warp == product_warp) {
    // ---- one warp issues the products
    {
      const uint32_t lead = tc::elected();
      constexpr bool kBf16 = !kIsF16<SA>;
      constexpr int kParts = PA > PB ? PA : PB;
      // the part of A in the first product of the smallest kind
      constexpr int first_part = kParts - 1 < PB ? 0 : kParts - PB;
      const uint32_t instruction = tc::instruction(kBf16, AMN, BMN, p.tile_n);
      // 128 m in one block of 64: the second half repeats the first, and its
      // rows of the result are not stored
      const uint32_t a_block = p.m > 64 ? kChunk * 128 : 0;
      if (p.resident) ok = tc::barrier_wait(tc::shared_address(&resident_full), 0);
      // the stages of the one ring, or of the two groups of producers in turn
      const int half_stages = p.raw_bytes ? (p.stages + 1) / 2 : p.stages;
      int stage = 0, other_stage = half_stages;
      uint32_t parity = 0, other_parity = 0, i_acc = 0;  // accumulators filled
      int end_stage = half_stages, other_end = p.stages;
      for (uint32_t t = blockIdx.x; t < p.tiles && ok; t += gridDim.x) {
        const ProductTile tile(p, t);
        int c = 0;
        for (long long sum_k = tile.k0; sum_k < tile.k1 && ok; sum_k += p.k_per_sum) {
          const uint32_t acc = i_acc & (p.accumulators - 1);
          const uint32_t round = p.alternate ? i_acc >> 2 : i_acc >> 1;
          if (!(ok = tc::barrier_wait(tc::shared_address(&acc_empty[acc]), (round & 1) ^ 1))) break;
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
                const uint32_t ao = at + i * kAPlane, bo = b_at + j * b_plane;
                tc::mma_steps(lead, d + (own ? 0 : (kAcc - 1) * p.tile_n),
                              AMN ? tc::descriptor_mn_major(ao, a_block)
                                  : tc::descriptor_k_major(ao),
                              BMN ? tc::descriptor_mn_major(bo, kChunk * 128)
                                  : tc::descriptor_k_major(bo),
                              AMN ? tc::kStepMn : tc::kStepK, BMN ? tc::kStepMn : tc::kStepK,
                              steps, instruction, !first);
              }
            tc::commit(lead, tc::shared_address(&empty[stage]));
            if (++stage == end_stage) {
              stage = p.raw_bytes && end_stage == p.stages ? half_stages : 0;
              parity ^= 1;
            }
          }
          tc::commit(lead, tc::shared_address(&acc_full[acc]));
          ++i_acc;
        }
        if (p.raw_bytes) {  // the other group's tile is next
          const int s = stage, e = end_stage;
          const uint32_t q = parity;
          stage = other_stage, end_stage = other_end, parity = other_parity;
          other_stage = s, other_end = e, other_parity = q;
        }
      }
      // whichever way the loop ended, no product is in flight past this point
      tc::commit(lead, tc::shared_address(&drained));
      ok = tc::barrier_wait(tc::shared_address(&drained), 0) && ok;
    }
  } else if (warp < kEpilogueWarps) {
    // ---- epilogue
    const int lane_block = warp & 3, half = warp >> 2;
    constexpr bool kExtra = EPI != kPlain;
    const Patch<TE> extra_patch{base + warp * p.staging + 1024 * static_cast<int>(sizeof(TO))};
    const Patch<TO> out_patch{base + warp * p.staging};
    const bool leader = (threadIdx.x & 31) == 0;
    const uint32_t extra_bar = tc::shared_address(&extra_full[warp]);
    // the accumulators and tiles of this warp, and its first chunk of columns
    const uint32_t i_step = p.alternate ? 2 : 1, t_step = gridDim.x * i_step;
    const uint32_t t_first = blockIdx.x + (p.alternate ? half * gridDim.x : 0);
    const int c_first = p.alternate ? 0 : half;
    uint32_t i_acc = p.alternate ? half : 0, extra_parity = 0;
    bool extra_coming = false;
    // starts the copy of the extra values of a tile's patch
    const auto fetch_extra = [&](const ProductTile& tile, int c) {
      const long long row0 = tile.m0 + lane_block * 32;
      if (c * 32 >= p.tile_n || tile.n0 + c * 32 >= p.n || row0 >= p.m) return;
      if (leader) {
        tc::barrier_expect(extra_bar, 1024 * sizeof(TE));
        tc::copy_in(extra_patch.base, &p.extra_map, tile.n0 + c * 32, static_cast<int>(row0),
                    extra_bar);
      }
      extra_coming = true;
    };
    if (kExtra && p.copy_extra && t_first < p.tiles)
      fetch_extra(ProductTile(p, t_first), c_first);
    for (uint32_t t = t_first; t < p.tiles && ok; t += t_step) {
      const ProductTile tile(p, t);
      const long long row0 = tile.m0 + lane_block * 32;
      const int rows = static_cast<int>(min(p.m - row0, 32LL));
      const long long out_at = (tile.split * p.m + row0) * p.out_ld;
      for (long long sum_k = tile.k0; sum_k < tile.k1; sum_k += p.k_per_sum) {
        bool waited = false;
        const uint32_t acc = i_acc & (p.accumulators - 1);
        const uint32_t parity = (p.alternate ? i_acc >> 2 : i_acc >> 1) & 1;
        for (int c = c_first; c * 32 < p.tile_n; c += kEpilogueWarps / 4) {
          const int col0 = tile.n0 + c * 32, cols = min(p.n - col0, 32);
          if (cols <= 0 || rows <= 0) break;
          if (kExtra && p.extra && !p.copy_extra && sum_k + p.k_per_sum >= tile.k1) {
            __syncwarp();  // the patch before has been read
            extra_patch.load(static_cast<const TE*>(p.extra) + row0 * p.n + col0, p.n, rows, cols,
                             p.extra_vector);
            __syncwarp();
          }
          if (!waited) {
            if (!(ok = tc::barrier_wait(tc::shared_address(&acc_full[acc]), parity))) break;
            tc::fence_after_sync();
            waited = true;
          }
          const uint32_t from = tmem + (lane_block << 21) + acc * kAcc * p.tile_n + c * 32;
          float v[32];
          tc::tmem_load32(from, v);
          if constexpr (kAcc == 2) {
            float low[32];
            tc::tmem_load32(from + p.tile_n, low);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += low[i];
          }
          // 16-bit results of several sums: a lane holds its row's in shared memory
          if constexpr (sizeof(TO) == 2) {
            if (p.held) {
              const Patch<float> held{out_patch.base + 1024 * static_cast<int>(sizeof(TO)) +
                                      (p.extra ? 1024 * static_cast<int>(sizeof(TE)) : 0)};
              const bool last = sum_k + p.k_per_sum >= tile.k1;
              const int lane = threadIdx.x & 31;
#pragma unroll
              for (int j = 0; j < Patch<float>::kPieces; ++j) {
                const uint32_t place = held.at(lane, j);
                if (sum_k != tile.k0) {
                  const float4 s = load_shared(place);
                  v[4 * j] += s.x, v[4 * j + 1] += s.y, v[4 * j + 2] += s.z, v[4 * j + 3] += s.w;
                }
                if (!last)
                  store_shared(place,
                               make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                          __float_as_uint(v[4 * j + 2]),
                                          __float_as_uint(v[4 * j + 3])));
              }
              if (!last) continue;
            }
          }
          // fp32 ones: the sums before the last are stored, each onto the ones
          // before, and the last takes them from there
          if constexpr (kExtra && kAcc == 2) {
            if (p.k_per_sum < p.k) {
              TO* to = static_cast<TO*>(p.out) + out_at + col0;
              const bool last = sum_k + p.k_per_sum >= tile.k1;
              const int lane = threadIdx.x & 31;
              __syncwarp();  // the results before have left the patch
#pragma unroll
              for (int j = 0; j < Patch<TO>::kPieces; ++j)
                store_shared(out_patch.at(lane, j),
                             make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                        __float_as_uint(v[4 * j + 2]),
                                        __float_as_uint(v[4 * j + 3])));
              __syncwarp();
              if (!last) {
                out_patch.store(to, p.out_ld, rows, cols, p.out_vector, sum_k != tile.k0);
                continue;
              }
              out_patch.add(to, p.out_ld, rows, cols, p.out_vector);
              __syncwarp();
#pragma unroll
              for (int j = 0; j < Patch<TO>::kPieces; ++j) {
                const float4 s = load_shared(out_patch.at(lane, j));
                v[4 * j] = s.x, v[4 * j + 1] = s.y, v[4 * j + 2] = s.z, v[4 * j + 3] = s.w;
              }
            }
          }
          if constexpr (kExtra) {
            if (p.bias) {
              if (p.bias_shared) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 b = load_shared(bias_at + (col0 + j * 4) * 4);
                  unpack2(add2(pack2(v[4 * j], v[4 * j + 1]), pack2(b.x, b.y)), v[4 * j],
                          v[4 * j + 1]);
                  unpack2(add2(pack2(v[4 * j + 2], v[4 * j + 3]), pack2(b.z, b.w)), v[4 * j + 2],
                          v[4 * j + 3]);
                }
              } else {
                const TE* bias = static_cast<const TE*>(p.bias) + col0;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (j < cols) v[j] += to_float(bias[j]);
              }
            }
            if (p.copy_extra) {
              if (!(ok = tc::barrier_wait(extra_bar, extra_parity))) break;
              extra_parity ^= 1;
              extra_coming = false;
            }
            const bool e = p.extra;
            switch (p.activation) {
              case kRelu: finish_row<EPI, kRelu, TE>(extra_patch, e, v); break;
              case kSilu: finish_row<EPI, kSilu, TE>(extra_patch, e, v); break;
              case kGelu: finish_row<EPI, kGelu, TE>(extra_patch, e, v); break;
              case kSigmoid: finish_row<EPI, kSigmoid, TE>(extra_patch, e, v); break;
              default: finish_row<EPI, kNone, TE>(extra_patch, e, v);
            }
            if constexpr (EPI == kSlope) {
              if (p.column_sums) {  // before dz is rounded
                if (static_cast<int>(threadIdx.x & 31) >= rows) {
#pragma unroll
                  for (int j = 0; j < 32; ++j) v[j] = 0.0f;
                }
                __syncwarp();
                const float sum = sum_rows<32>(v);
                const int lane = threadIdx.x & 31;
                if (lane < cols)
                  p.column_sums[(tile.m0 / 32 + lane_block) * p.n + col0 + lane] = sum;
              }
            }
            if (p.copy_extra) {  // the next patch's, once this one has been read
              __syncwarp();
              const int next = c + kEpilogueWarps / 4;
              if (next * 32 < p.tile_n && tile.n0 + next * 32 < p.n)
                fetch_extra(tile, next);
              else if (p.tiles - t > t_step)
                fetch_extra(ProductTile(p, t + t_step), c_first);
            }
          }
          // first: round to what leaves a second value, which v becomes
          const auto put = [&](auto first, const CUtensorMap* map, void* out) {
            if (leader && p.copy_out) tc::copies_out_read();
            __syncwarp();  // the results before have left the patch
#pragma unroll
            for (int j = 0; j < Patch<TO>::kPieces; ++j) {
              constexpr int V = Patch<TO>::V;
              float o[V];
#pragma unroll
              for (int i = 0; i < V; ++i) o[i] = v[j * V + i];
              Vec<TO, V> r;
              if constexpr (decltype(first)::value) {
                r = take_first<TO, V>(o);
#pragma unroll
                for (int i = 0; i < V; ++i) v[j * V + i] = o[i];
              } else {
                r = round_values<TO, V>(o);
              }
              store_shared(out_patch.at(threadIdx.x & 31, j), reinterpret_cast<const uint4&>(r));
            }
            if (p.copy_out) {
              tc::fence_async_proxy();
              __syncwarp();
              if (leader) tc::copy_out(map, col0, static_cast<int>(row0), out_patch.base);
            } else {
              __syncwarp();
              out_patch.store(static_cast<TO*>(out) + out_at + col0, p.out_ld, rows, cols,
                              p.out_vector,
                              !kExtra && sizeof(TO) == 4 &&
                                  (sum_k != tile.k0 || p.accumulate));
            }
          };
          if constexpr (EPI == kSlope && sizeof(TO) == 2) {
            if (p.out_second) {
              put(std::true_type{}, &p.out_map, p.out);
              put(std::false_type{}, &p.out_second_map, p.out_second);
              continue;
            }
          }
          put(std::false_type{}, &p.out_map, p.out);
        }
        if (!ok) break;
        if (!waited) {  // a warp without a patch still takes part
          if (!(ok = tc::barrier_wait(tc::shared_address(&acc_full[acc]), parity))) break;
          if (kExtra && p.copy_extra && !extra_coming && p.tiles - t > t_step)
            fetch_extra(ProductTile(p, t + t_step), c_first);
        }
        tc::fence_before_sync();
        tc::barrier_arrive(tc::shared_address(&acc_empty[acc]));
        i_acc += i_step;
      }
    }
    if (extra_coming) ok = tc::barrier_wait(extra_bar, extra_parity) && ok;
    if (leader && p.copy_out) tc::copies_out_read();
  }
  if (!ok) atomicCAS(p.error, 0, kDeviceTimeout);
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_free(tmem, p.tmem_columns);
}

}  // namespace feature
}  // namespace splat
