// Host side of the linear layer's products: tiling and launch.
#pragma once
#include <algorithm>
#include <type_traits>

#include "feature_product.cuh"
#include "host_runtime.h"

namespace splat {
namespace feature {

// ---- launching a product -------------------------------------------------------

// The widest of 16, 8, 4 and 2 bytes that rows of ld values start on.
template <class S>
int row_vector(const void* base, long long ld) {
  int v = 16;
  while (v > static_cast<int>(sizeof(S)) &&
         ((ld * static_cast<long long>(sizeof(S))) % v || !host::aligned(base, v)))
    v /= 2;
  return v;
}

// The map of a row-major matrix (rows x columns, ld values between rows) for
// tensor copies of boxes of box_columns x box_rows, swizzled over their row
// length (64 or 128 bytes) as the kernels' shared layouts are.  False where
// the matrix cannot be copied so.
template <class T>
bool make_map(CUtensorMap& map, const void* base, long long rows, long long columns, long long ld,
              int box_columns, int box_rows) {
  if (!base || rows >= 1LL << 31 || !host::aligned(base, 16) || ld * sizeof(T) % 16) return false;
  return host::encode_map(&map,
                          sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                          : kIsF16<T>    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          base, rows, columns, ld * sizeof(T), box_columns, box_rows,
                          box_columns * sizeof(T) == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                                         : CU_TENSOR_MAP_SWIZZLE_64B);
}

// Shared memory of a block when one, two or three share an SM (228 KB, of which
// each block costs 1 KB besides its own), less the barriers and the rounding
// of the base to 1 KB.
constexpr int kOneBlockBytes = 225 * 1024, kTwoBlocksBytes = 110 * 1024,
              kThreeBlocksBytes = 73 * 1024;
constexpr int kMaxSharedBias = 4096;  // values
constexpr long long kFewRows = 16384;
constexpr int kMaxResidentBytes = 128 * 1024;

// Fills in the tiling of p (its sources, sizes and epilogue set) and launches.
template <class SA, int PA, bool AMN, class SB, int PB, bool BMN, class TE, class TO, int EPI>
int launch_product(ProductParams p, cudaStream_t s) {
  // a plain product's tiles are as wide as they can be; behind one with
  // arithmetic two blocks' epilogues share an SM (512 -> 512 fp16 gelu over
  // 131072 rows 111 us against 119 in 256-wide tiles, 256 -> 256 bf16 silu 43
  // against 48)
  constexpr long long kMostSum = kMostAdditions * 16 / PA;  // of a 16-bit layer's accumulator
  // 16-bit results of more are added up in shared memory, a patch to a warp
  p.held = sizeof(TO) == 2 && p.k > kMostSum;
  const int widest = p.held ? 64 : PA <= 2 && PB == 1 && EPI == kPlain ? 256 : 128;
  p.tiles_n = (p.n + widest - 1) / widest;
  p.tile_n = ((p.n + p.tiles_n - 1) / p.tiles_n + 31) / 32 * 32;
  const long long tiles_m = (p.m + kTileRows - 1) / kTileRows;
  if (tiles_m * p.tiles_n * p.splits >= 1LL << 31)
    return host::fail(kTooLarge, "feature_linear: too many tiles");
  p.tiles_m = static_cast<uint32_t>(tiles_m);
  p.tiles = p.tiles_m * p.tiles_n * p.splits;
  p.a_vector = row_vector<SA>(p.a, p.a_ld);
  p.b_vector = row_vector<SB>(p.b, p.b_ld);
  p.extra_vector =
      p.n * static_cast<long long>(sizeof(TE)) % 16 == 0 && host::aligned(p.extra, 16);
  if (!p.out_ld) p.out_ld = p.n;
  p.out_vector = p.n * static_cast<long long>(sizeof(TO)) % 16 == 0 &&
                 p.out_ld * static_cast<long long>(sizeof(TO)) % 16 == 0 &&
                 host::aligned(p.out, 16);
  const int columns = static_cast<int>(p.tiles_n) * p.tile_n;
  p.bias_shared = p.bias && columns <= kMaxSharedBias ? columns : 0;
  p.tmem_columns = 32;
  constexpr int kAcc = accumulators(PA, PB);
  // sums of several accumulators are joined in fp32 outputs
  p.k_per_sum = kAcc == 2 ? kExactSum : kMostSum;
  // (35 -> 32 fp32 gelu over 10^6 rows 114 us against 187 without, 32 -> 3 bf16
  // over 1.9 10^6 66 against 85, 64 -> 32 bf16 69 against 69)
  p.alternate = p.tile_n == 32 && p.k_per_sum >= p.k_per_split;
  p.accumulators = p.alternate ? 4 : 2;
  while (p.tmem_columns < static_cast<uint32_t>(p.accumulators * kAcc * p.tile_n))
    p.tmem_columns *= 2;
  const int b_bytes = PB * b_plane_bytes<BMN>(p.tile_n), a_bytes = PA * kAPlane;
  const long long chunks = (p.k + kChunk - 1) / kChunk;
  const long long whole_b = chunks * b_bytes;
  // a patch of results, and one of the extra values
  p.staging =
      1024 * static_cast<int>(sizeof(TO) + (p.extra ? sizeof(TE) : 0) + (p.held ? 4 : 0));
  int fixed = kEpilogueWarps * p.staging + (p.bias_shared * 4 + 1023) / 1024 * 1024;
  // B stays where two stages of A fit beside it
  p.resident = p.splits == 1 && p.tiles_n == 1 && whole_b <= kMaxResidentBytes &&
               fixed + whole_b + 2 * a_bytes <= kOneBlockBytes;
  if (p.resident) fixed += static_cast<int>(whole_b);
  const int stage = a_bytes + (p.resident ? 0 : b_bytes);
  int blocks = 2, budget = kTwoBlocksBytes;
  if (producers(PA, PB) > 128 || p.tmem_columns > 256 || fixed + 2 * stage > budget)
    blocks = 1, budget = kOneBlockBytes;
  if constexpr (PA == 2) {
    const long long a_rows = AMN ? p.k : p.m, a_columns = AMN ? p.m : p.k;
    const int a_box = AMN ? kChunk : kTileRows;
    p.copy_operands =
        make_map<SA>(p.a_map, p.a, a_rows, a_columns, p.a_ld, kChunk, a_box) &&
        make_map<SA>(p.a_second_map, p.a_second, a_rows, a_columns, p.a_ld, kChunk, a_box) &&
        make_map<SB>(p.b_map, p.b, BMN ? p.k : p.n, BMN ? p.n : p.k, p.b_ld, kChunk,
                     BMN ? kChunk : p.tile_n);
    if (!p.copy_operands) return host::fail(kInvalidArgument, "feature_linear: operand planes");
  } else if (p.a_plane_rows) {
    // both operands are planes; f16 ones hold f16, all others bf16 parts
    using H = std::conditional_t<kIsF16<SA>, f16, bf16>;
    p.copy_operands =
        make_map<H>(p.a_map, p.a, static_cast<long long>(p.a_plane_rows) * PA, AMN ? p.m : p.k,
                    p.a_ld, kChunk, AMN ? kChunk : kTileRows) &&
        make_map<H>(p.b_map, p.b, static_cast<long long>(p.b_plane_rows) * PB, BMN ? p.n : p.k,
                    p.b_ld, kChunk, BMN ? kChunk : p.tile_n);
    if (!p.copy_operands) return host::fail(kInvalidArgument, "feature_linear: operand planes");
  } else if constexpr (PA == 1 && PB == 1) {
    p.copy_operands =
        make_map<SA>(p.a_map, p.a, AMN ? p.k : p.m, AMN ? p.m : p.k, p.a_ld, kChunk,
                     AMN ? kChunk : kTileRows) &&
        make_map<SB>(p.b_map, p.b, BMN ? p.k : p.n, BMN ? p.n : p.k, p.b_ld, kChunk,
                     BMN ? kChunk : p.tile_n);
  }
  // two tiles of A as they are in memory, where two stages fit beside them
  // (35 -> 32 fp32 gelu over 10^6 rows 112 us against 152 read as needed,
  // 35 -> 64 bf16 73 against 79)
  if (PA != 2 && !p.copy_operands && !AMN && p.tiles_n == 1 && p.a_ld == p.k &&
      host::aligned(p.a, 16)) {
    const long long raw = (kTileRows * p.k * static_cast<long long>(sizeof(SA)) + 127) / 128 * 128;
    if (fixed + 2 * stage + 2 * raw > budget && blocks == 2) blocks = 1, budget = kOneBlockBytes;
    if (fixed + 2 * stage + 2 * raw <= budget) p.raw_bytes = static_cast<int>(raw);
  }
  // blocks without register-filling producers are small enough for three
  // (64 -> 64 bf16 with residual over 1.9 10^6 rows 129 us against 139 with two)
  if (p.copy_operands && blocks == 2 && 3 * p.tmem_columns <= 512 &&
      fixed + 2 * stage <= kThreeBlocksBytes)
    blocks = 3, budget = kThreeBlocksBytes;
  p.stages = std::min(kMaxStages, (budget - fixed - 2 * p.raw_bytes) / stage);
  if (p.stages < 1) return host::fail(kTooLarge, "feature_linear: no room for a stage");
  if (EPI != kPlain) p.copy_extra = make_map<TE>(p.extra_map, p.extra, p.m, p.n, p.n, 32, 32);
  // partial sums are added to or lie one split behind the other
  if (p.splits == 1 && (p.k_per_sum >= p.k || p.held))
    p.copy_out = make_map<TO>(p.out_map, p.out, p.m, p.n, p.out_ld, 32, 32) &&
                 (!p.out_second ||
                  make_map<TO>(p.out_second_map, p.out_second, p.m, p.n, p.out_ld, 32, 32));
  p.error = host::device_error_word();
  if (!p.error) return kCudaError;
  const int bytes = fixed + p.stages * stage + 2 * p.raw_bytes + 1024;
  constexpr auto* kernel = product_kernel<SA, PA, AMN, SB, PB, BMN, TE, TO, EPI>;
  if (!host::allow_shared<kernel>())
    return host::check_launch("feature_linear: shared memory");
  const long long grid =
      std::min<long long>(p.tiles, static_cast<long long>(host::sm_count()) * blocks);
  const int threads = kEpilogueWarps * 32 + (p.copy_operands ? 32 : producers(PA, PB)) + 32;
  kernel<<<static_cast<unsigned>(grid), threads, bytes, host::counted(s)>>>(p);
  return host::check_launch("feature_linear");
}

// Parts of an operand of the linear layer's products, but for the dz of 16-bit
// types, which has two where its activation's slope adds digits to dy's: one would
// add half a step to each dz, which dx and dW show as much as their own rounding
// (2.4e-3 relative instead of 1.7e-3 for bf16).
template <class T>
constexpr int kOperandParts = sizeof(T) == 4 ? 3 : 1;

// A matrix (rows, cols) of T as planes of its parts.
struct Planes {
  void* data = nullptr;
  long long rows = 0;
  int plane_rows = 0, ld = 0;
};
inline long long round_to(long long n, long long m) { return (n + m - 1) / m * m; }
template <class T>
size_t plane_bytes(long long rows, int cols) {
  return static_cast<size_t>(kOperandParts<T>) * round_to(rows, 64) * round_to(cols, 8) * 2;
}
template <class T>
Planes split(const void* src, long long rows, int cols, void* to, cudaStream_t s) {
  Planes p;
  if (sizeof(T) == 2 && row_vector<T>(src, cols) == 16) {  // it is one as it lies
    p.data = const_cast<void*>(src);
    p.rows = rows, p.plane_rows = static_cast<int>(rows), p.ld = cols;
    return p;
  }
  p.data = to;
  p.rows = rows;
  p.plane_rows = static_cast<int>(round_to(rows, 64));
  p.ld = static_cast<int>(round_to(cols, 8));
  const int pieces = p.ld / 8;
  const long long total = static_cast<long long>(p.plane_rows) * pieces;
  const unsigned grid = static_cast<unsigned>(
      std::min<long long>((total + 1023) / 1024, 8LL * host::sm_count()));
  const auto run = [&](auto bytes) {
    split_kernel<T, kOperandParts<T>, decltype(bytes)::value><<<grid, 256, 0, host::counted(s)>>>(
        static_cast<const T*>(src), rows, cols, pieces, p.plane_rows, p.ld,
        static_cast<uint16_t*>(to));
  };
  const int vector = row_vector<T>(src, cols);
  if (vector == 16) run(std::integral_constant<int, 16>{});
  else if (vector >= 4) run(std::integral_constant<int, 4>{});
  else run(std::integral_constant<int, static_cast<int>(sizeof(T))>{});
  return p;
}

// Whether the wide layers' products take planes: fp32 operands, and rows that
// are not whole 16-byte pieces.  The pass that makes them pays from about
// kFewRows on: 300 -> 300 fp32 over 4000, 16384 and 100000 rows 29, 55 and
// 251 us with planes, 25, 57 and 289 without; 301 -> 200 bf16 over 4000 and
// 100000 rows 23 and 73 with, 21 and 108 without (ReLU training: 275 against 717).
template <class T>
bool wants_planes(long long rows, int k, int n) {
  const int whole = 16 / static_cast<int>(sizeof(T));
  return rows >= kFewRows && kOperandParts<T> * round_to(rows, 64) < 1LL << 31 &&
         (sizeof(T) == 4 || k % whole || n % whole);
}

template <class T>
ProductParams forward_params(long long rows, int k, int n, const void* x, const void* weight,
                             const void* bias, const void* extra, int activation, void* out) {
  ProductParams p{};
  p.m = rows, p.k = k, p.n = n;
  p.a = x, p.a_ld = k;
  p.b = weight, p.b_ld = k;
  p.k_per_split = k, p.splits = 1;
  p.bias = bias, p.extra = extra, p.activation = activation, p.out = out;
  return p;
}

inline void use_planes(ProductParams& p, const Planes& a, const Planes& b) {
  p.a = a.data, p.a_ld = a.ld, p.a_plane_rows = a.plane_rows;
  p.b = b.data, p.b_ld = b.ld, p.b_plane_rows = b.plane_rows;
}

int check_linear(int dtype, long long rows, int k, int n, int activation);

}  // namespace feature
}  // namespace splat
