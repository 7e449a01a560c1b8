// A linear layer over feature rows with bias, activation and residual in its
// epilogue, forward and backward.
//
//   y  = act(z) + r,  z = x W^T + b        x (M, K), W (N, K), b (N), r, y (M, N)
//   dz = dy act'(z)
//   dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dr = dy
//
// The backward recomputes z from x and W (x is read for dW anyway), so the
// forward keeps nothing besides its inputs.
#include <algorithm>

#include "feature_common.cuh"
#include "feature_product.cuh"
#include "host_runtime.h"
#include "splat200.h"

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

// Shared memory of a block when one or two share an SM (228 KB, of which each
// block costs 1 KB besides its own), less the barriers and the rounding of the
// base to 1 KB.
constexpr int kOneBlockBytes = 225 * 1024, kTwoBlocksBytes = 110 * 1024;
constexpr int kMaxSharedBias = 4096;  // values
constexpr int kMaxResidentBytes = 128 * 1024;

// Fills in the tiling of p (its sources, sizes and epilogue set) and launches.
template <class SA, int PA, bool AMN, class SB, int PB, bool BMN, class TE, class TO, int EPI>
int launch_product(ProductParams p, cudaStream_t s) {
  const int widest = PA == 1 && PB == 1 ? 256 : 128;
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
  p.out_vector = p.n * static_cast<long long>(sizeof(TO)) % 16 == 0 && host::aligned(p.out, 16);
  const int columns = static_cast<int>(p.tiles_n) * p.tile_n;
  p.bias_shared = p.bias && columns <= kMaxSharedBias ? columns : 0;
  p.tmem_columns = 32;
  constexpr int kAcc = accumulators(PA, PB);
  while (p.tmem_columns < 2u * kAcc * p.tile_n) p.tmem_columns *= 2;
  // sums of several accumulators are joined in fp32 outputs; an operand row of
  // more values than kExactSum is summed in one
  p.k_per_sum = kAcc == 2 && EPI == kPlain && sizeof(TO) == 4 ? kExactSum : p.k_per_split;
  const int b_bytes = PB * b_plane_bytes<BMN>(p.tile_n), a_bytes = PA * kAPlane;
  const long long chunks = (p.k + kChunk - 1) / kChunk;
  const long long whole_b = chunks * b_bytes;
  p.resident = p.splits == 1 && p.tiles_n == 1 && whole_b <= kMaxResidentBytes;
  const int fixed = kEpilogueWarps * kStagingBytes + (p.bias_shared * 4 + 1023) / 1024 * 1024 + (p.resident ? static_cast<int>(whole_b) : 0);
  const int stage = a_bytes + (p.resident ? 0 : b_bytes);
  int blocks = 2, budget = kTwoBlocksBytes;
  if (producers(PA, PB) > 128 || p.tmem_columns > 256 || fixed + 2 * stage > budget)
    blocks = 1, budget = kOneBlockBytes;
  p.stages = std::min(kMaxStages, (budget - fixed) / stage);
  if (p.stages < 1) return host::fail(kTooLarge, "feature_linear: no room for a stage");
  const bool copied = PA == 1 && PB == 1 && p.a_vector == 16 &&
                      (p.resident || p.b_vector == 16) && sizeof(SA) == 2;
  p.lag = copied ? p.stages - 1 : 0;
  p.error = host::device_error_word();
  if (!p.error) return kCudaError;
  const int bytes = fixed + p.stages * stage + 1024;
  auto* kernel = product_kernel<SA, PA, AMN, SB, PB, BMN, TE, TO, EPI>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
      cudaSuccess)
    return host::check_launch("feature_linear: shared memory");
  const long long grid = std::min<long long>(p.tiles, static_cast<long long>(host::sm_count()) * blocks);
  kernel<<<static_cast<unsigned>(grid), kEpilogueWarps * 32 + producers(PA, PB) + 32, bytes, host::counted(s)>>>(p);
  return host::check_launch("feature_linear");
}

// Parts of an operand that is T in memory (beside a one-part operand f16 goes
// as it is), and of the fp32 dz: a 16-bit gradient's products take dz in two
// parts (2^-16), so that it is rounded once, at the end.
template <class T>
constexpr int kSourceParts = sizeof(T) == 4 ? 3 : kIsF16<T> ? 2 : 1;
template <class T>
constexpr int kNativeParts = sizeof(T) == 4 ? 3 : 1;
template <class T>
constexpr int kGradientParts = sizeof(T) == 4 ? 3 : 2;

// ---- sums over splits and rows ---------------------------------------------------

// Adds the splits' partial sums in a fixed order: 8 threads to a value.
template <class T>
__global__ void __launch_bounds__(256)
    join_splits_kernel(const float* partial, long long count, int splits, T* out) {
  const long long i = blockIdx.x * 32LL + threadIdx.x;
  float s = 0.0f;
  if (i < count)
    for (int k = threadIdx.y; k < splits; k += 8) s += partial[k * count + i];
  __shared__ float sums[8][32];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && i < count) {
    for (int k = 1; k < 8; ++k) s += sums[k][threadIdx.x];
    out[i] = from_float<T>(s);
  }
}

template <class T>
void join_splits(const float* partial, long long count, int splits, void* out, cudaStream_t s) {
  join_splits_kernel<T><<<host::blocks_for(count, 32), dim3(32, 8), 0, host::counted(s)>>>(
      partial, count, splits, static_cast<T*>(out));
}

// Column sums of dz (m, n) over ranges of rows.
template <class S>
__global__ void __launch_bounds__(256) column_sums_kernel(const S* dz, long long m, int n,
                                                          long long rows, float* partial) {
  const int c = blockIdx.x * 32 + threadIdx.x;
  const long long begin = blockIdx.y * rows, end = min(begin + rows, m);
  float s = 0.0f;
  if (c < n) {
#pragma unroll 8
    for (long long r = begin + threadIdx.y; r < end; r += 8) s += to_float(dz[r * n + c]);
  }
  __shared__ float sums[8][32];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < n) {
    for (int i = 1; i < 8; ++i) s += sums[i][threadIdx.x];
    partial[static_cast<long long>(blockIdx.y) * n + c] = s;
  }
}

int check_linear(int dtype, long long rows, int k, int n, int activation) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "feature_linear: dtype");
  if (activation < 0 || activation > 4)
    return host::fail(kInvalidArgument, "feature_linear: activation");
  if (rows < 1 || k < 1 || n < 1) return host::fail(kInvalidArgument, "feature_linear: sizes");
  if (k > 65535 || n > 65535 || rows > (1LL << 36))
    return host::fail(kTooLarge, "feature_linear: too many rows, inputs or outputs");
  return kOk;
}

// Ranges of rows whose sums of dz^T x (and of dz) are joined afterwards:
// enough tiles for two blocks on every SM, 512 rows to a range at least.
struct Splits {
  int count;
  long long rows;
};
Splits weight_splits(long long rows, int k, int n) {
  const long long tiles = ((n + 127LL) / 128) * ((k + 127) / 128);
  const long long wanted = std::max(1LL, 2LL * host::sm_count() / tiles);
  const long long most = (rows + 511) / 512;
  const long long per = (rows + std::min(wanted, most) - 1) / std::min(wanted, most);
  Splits s;
  s.rows = (per + kChunk - 1) / kChunk * kChunk;
  s.count = static_cast<int>((rows + s.rows - 1) / s.rows);
  return s;
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

size_t dz_bytes(long long rows, int n, int activation) {
  return activation == kNone ? 0 : round16(static_cast<size_t>(rows) * n * 4);
}

// The two products of the backward, from dz as S.
template <class T, class S, int PZ, int PT>
int launch_gradients(long long rows, int k, int n, const S* dz, const void* x,
                     const void* weight, void* dx, void* dweight, void* dbias, float* partial,
                     cudaStream_t s) {
  if (dx) {
    ProductParams p{};
    p.m = rows, p.k = n, p.n = k;
    p.a = dz, p.a_ld = n;
    p.b = weight, p.b_ld = k;
    p.k_per_split = n, p.splits = 1;
    p.out = dx;
    const int status = launch_product<S, PZ, false, T, PT, true, T, T, kPlain>(p, s);
    if (status != kOk) return status;
  }
  const Splits splits = weight_splits(rows, k, n);
  if (dweight) {
    ProductParams p{};
    p.m = n, p.k = rows, p.n = k;
    p.a = dz, p.a_ld = n;
    p.b = x, p.b_ld = k;
    p.k_per_split = splits.rows, p.splits = splits.count;
    p.out = partial;
    const int status = launch_product<S, PZ, true, T, PT, true, float, float, kPlain>(p, s);
    if (status != kOk) return status;
    join_splits<T>(partial, static_cast<long long>(n) * k, splits.count, dweight, s);
  }
  if (dbias) {
    float* sums = partial + static_cast<long long>(splits.count) * n * k;
    column_sums_kernel<S><<<dim3(host::blocks_for(n, 32), splits.count), dim3(32, 8), 0,
                            host::counted(s)>>>(dz, rows, n, splits.rows, sums);
    join_splits<T>(sums, n, splits.count, dbias, s);
  }
  return host::check_launch("feature_linear_backward");
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

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

int splat_feature_linear(int dtype, long long rows, int k, int n, const void* x,
                         const void* weight, const void* bias, const void* residual,
                         int activation, void* y, void* stream) {
  const int bad = check_linear(dtype, rows, k, n, activation);
  if (bad != kOk) return bad;
  if (!x || !weight || !y) return host::fail(kInvalidArgument, "feature_linear: null pointer");
  auto s = static_cast<cudaStream_t>(stream);
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    constexpr int P = kNativeParts<T>;
    return launch_product<T, P, false, T, P, false, T, T, kForward>(
        forward_params<T>(rows, k, n, x, weight, bias, residual, activation, y), s);
  });
}

size_t splat_feature_linear_backward_workspace_bytes(int dtype, long long rows, int k, int n,
                                                     int activation) {
  if (check_linear(dtype, rows, k, n, activation) != kOk) return 0;
  const Splits splits = weight_splits(rows, k, n);
  return dz_bytes(rows, n, activation) +
         static_cast<size_t>(splits.count) * n * (static_cast<size_t>(k) + 1) * 4;
}

int splat_feature_linear_backward(int dtype, long long rows, int k, int n, const void* x,
                                  const void* weight, const void* bias, int activation,
                                  const void* dy, void* dx, void* dweight, void* dbias,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_linear(dtype, rows, k, n, activation);
  if (bad != kOk) return bad;
  if (!x || !weight || !dy || !workspace)
    return host::fail(kInvalidArgument, "feature_linear_backward: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument, "feature_linear_backward: workspace not 16-byte aligned");
  if (workspace_bytes <
      splat_feature_linear_backward_workspace_bytes(dtype, rows, k, n, activation))
    return host::fail(kWorkspaceTooSmall, "feature_linear_backward: workspace");
  auto s = static_cast<cudaStream_t>(stream);
  float* dz = static_cast<float*>(workspace);
  float* partial = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                            dz_bytes(rows, n, activation));
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    constexpr int P = kNativeParts<T>;
    if (activation == kNone)  // dz is dy
      return launch_gradients<T, T, P, P>(rows, k, n, static_cast<const T*>(dy), x, weight, dx,
                                          dweight, dbias, partial, s);
    const int status = launch_product<T, P, false, T, P, false, T, float, kSlope>(
        forward_params<T>(rows, k, n, x, weight, bias, dy, activation, dz), s);
    if (status != kOk) return status;
    return launch_gradients<T, float, kGradientParts<T>, kSourceParts<T>>(
        rows, k, n, dz, x, weight, dx, dweight, dbias, partial, s);
  });
}

}  // extern "C"
