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
#include "host_runtime.h"
#include "splat200.h"

namespace splat {
namespace feature {

constexpr int kTileM = 64, kTileN = 64, kTileK = 16;

// C(i, j) = sum_k A(i, k) B(j, k) with element strides, in 64x64 tiles of
// fp32 sums; blockIdx.z takes a range of k and then writes fp32 partial sums.
struct ProductParams {
  long long m, k;
  int n;
  const void* a;
  long long a_row, a_k;
  const void* b;
  long long b_row, b_k;
  long long k_per_split;
  // epilogue
  const void* bias;      // (n), added to C
  const void* residual;  // (m, n), added after the activation
  const void* dy;        // (m, n): C becomes dy * act'(C)
  void* out;             // (m, n); (splits, m, n) fp32 with several splits
};

enum Epilogue : int { kForward = 0, kSlope = 1, kPlain = 2 };

template <class TA, class TB, class TO, int EPI, int ACT>
__global__ void __launch_bounds__(256) product_kernel(const ProductParams p) {
  __shared__ float as[kTileK][kTileM + 1], bs[kTileK][kTileN + 1];
  const TA* a = static_cast<const TA*>(p.a);
  const TB* b = static_cast<const TB*>(p.b);
  const long long row0 = static_cast<long long>(blockIdx.x) * kTileM;
  const int col0 = blockIdx.y * kTileN;
  const long long k_begin = blockIdx.z * p.k_per_split;
  const long long k_end = min(k_begin + p.k_per_split, p.k);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (long long k0 = k_begin; k0 < k_end; k0 += kTileK) {
    for (int i = threadIdx.x; i < kTileM * kTileK; i += 256) {
      // neighbouring threads take neighbouring addresses of either layout
      const int r = p.a_k == 1 ? i / kTileK : i % kTileM;
      const int k = p.a_k == 1 ? i % kTileK : i / kTileM;
      const bool in = row0 + r < p.m && k0 + k < k_end;
      as[k][r] = in ? to_float(a[(row0 + r) * p.a_row + (k0 + k) * p.a_k]) : 0.0f;
    }
    for (int i = threadIdx.x; i < kTileN * kTileK; i += 256) {
      const int r = p.b_k == 1 ? i / kTileK : i % kTileN;
      const int k = p.b_k == 1 ? i % kTileK : i / kTileN;
      const bool in = col0 + r < p.n && k0 + k < k_end;
      bs[k][r] = in ? to_float(b[(col0 + r) * p.b_row + (k0 + k) * p.b_k]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += as[k][ty * 4 + i] * bs[k][tx * 4 + j];
    __syncthreads();
  }
  TO* out = static_cast<TO*>(p.out) + blockIdx.z * p.m * p.n;
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + ty * 4 + i;
    if (row >= p.m) break;
    for (int j = 0; j < 4; ++j) {
      const int col = col0 + tx * 4 + j;
      if (col >= p.n) break;
      float z = acc[i][j];
      if (p.bias) z += to_float(static_cast<const TB*>(p.bias)[col]);
      if constexpr (EPI == kForward) {
        z = activate<ACT>(z);
        if (p.residual) z += to_float(static_cast<const TA*>(p.residual)[row * p.n + col]);
      }
      if constexpr (EPI == kSlope)
        z = to_float(static_cast<const TA*>(p.dy)[row * p.n + col]) * slope<ACT>(z);
      out[row * p.n + col] = from_float<TO>(z);
    }
  }
}

// Adds the splits' partial sums in order.
template <class T>
__global__ void join_splits_kernel(const float* partial, long long count, int splits, T* out) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= count) return;
  float s = 0.0f;
  for (int k = 0; k < splits; ++k) s += partial[k * count + i];
  out[i] = from_float<T>(s);
}

// Column sums of dz (m, n) over ranges of rows.
__global__ void column_sums_kernel(const float* dz, long long m, int n, long long rows,
                                   float* partial) {
  const int c = blockIdx.x * 32 + threadIdx.x;
  const long long begin = blockIdx.y * rows, end = min(begin + rows, m);
  float s = 0.0f;
  if (c < n)
    for (long long r = begin + threadIdx.y; r < end; r += 8) s += dz[r * n + c];
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

constexpr int kMaxSplits = 256;

int dweight_splits(long long rows) {
  return static_cast<int>(std::min<long long>(kMaxSplits, (rows + 4095) / 4096));
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

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
  ProductParams p{};
  p.m = rows, p.k = k, p.n = n;
  p.a = x, p.a_row = k, p.a_k = 1;
  p.b = weight, p.b_row = k, p.b_k = 1;
  p.k_per_split = k;
  p.bias = bias, p.residual = residual, p.out = y;
  const dim3 grid(host::blocks_for(rows, kTileM), host::blocks_for(n, kTileN));
  auto s = static_cast<cudaStream_t>(stream);
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return SPLAT_FEATURE_ACT(activation, [&] {
      product_kernel<T, T, T, kForward, ACT><<<grid, 256, 0, host::counted(s)>>>(p);
      return host::check_launch("feature_linear");
    });
  });
}

size_t splat_feature_linear_backward_workspace_bytes(int dtype, long long rows, int k, int n,
                                                     int activation) {
  if (check_linear(dtype, rows, k, n, activation) != kOk) return 0;
  const size_t splits = dweight_splits(rows);
  return round16(static_cast<size_t>(rows) * n * 4) + splits * n * (static_cast<size_t>(k) + 1) * 4;
}

int splat_feature_linear_backward(int dtype, long long rows, int k, int n, const void* x,
                                  const void* weight, const void* bias, int activation,
                                  const void* dy, void* dx, void* dweight, void* dbias,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_linear(dtype, rows, k, n, activation);
  if (bad != kOk) return bad;
  if (!x || !weight || !dy || !workspace)
    return host::fail(kInvalidArgument, "feature_linear_backward: null pointer");
  if (workspace_bytes <
      splat_feature_linear_backward_workspace_bytes(dtype, rows, k, n, activation))
    return host::fail(kWorkspaceTooSmall, "feature_linear_backward: workspace");
  auto s = static_cast<cudaStream_t>(stream);
  float* dz = static_cast<float*>(workspace);
  float* partial =
      reinterpret_cast<float*>(static_cast<char*>(workspace) + round16(rows * n * 4));
  const int splits = dweight_splits(rows);
  const long long rows_per_split = (rows + splits - 1) / splits;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    ProductParams p{};
    p.m = rows, p.k = k, p.n = n;
    p.a = x, p.a_row = k, p.a_k = 1;
    p.b = weight, p.b_row = k, p.b_k = 1;
    p.k_per_split = k;
    p.bias = bias, p.dy = dy, p.out = dz;
    SPLAT_FEATURE_ACT(activation, [&] {
      const dim3 grid(host::blocks_for(rows, kTileM), host::blocks_for(n, kTileN));
      product_kernel<T, T, float, kSlope, ACT><<<grid, 256, 0, host::counted(s)>>>(p);
    });
    if (dx) {
      ProductParams q{};
      q.m = rows, q.k = n, q.n = k;
      q.a = dz, q.a_row = n, q.a_k = 1;
      q.b = weight, q.b_row = 1, q.b_k = k;
      q.k_per_split = n;
      q.out = dx;
      const dim3 grid(host::blocks_for(rows, kTileM), host::blocks_for(k, kTileN));
      product_kernel<float, T, T, kPlain, kNone><<<grid, 256, 0, host::counted(s)>>>(q);
    }
    if (dweight) {
      ProductParams q{};
      q.m = n, q.k = rows, q.n = k;
      q.a = dz, q.a_row = 1, q.a_k = n;
      q.b = x, q.b_row = 1, q.b_k = k;
      q.k_per_split = rows_per_split;
      q.out = partial;
      const dim3 grid(host::blocks_for(n, kTileM), host::blocks_for(k, kTileN), splits);
      product_kernel<float, T, float, kPlain, kNone><<<grid, 256, 0, host::counted(s)>>>(q);
      const long long count = static_cast<long long>(n) * k;
      join_splits_kernel<T><<<host::blocks_for(count, 256), 256, 0, host::counted(s)>>>(
          partial, count, splits, static_cast<T*>(dweight));
    }
    if (dbias) {
      float* sums = partial + static_cast<long long>(splits) * n * k;
      column_sums_kernel<<<dim3(host::blocks_for(n, 32), splits), dim3(32, 8), 0,
                           host::counted(s)>>>(dz, rows, n, rows_per_split, sums);
      join_splits_kernel<T><<<host::blocks_for(n, 256), 256, 0, host::counted(s)>>>(
          sums, n, splits, static_cast<T*>(dbias));
    }
    return host::check_launch("feature_linear_backward");
  });
}

}  // extern "C"
