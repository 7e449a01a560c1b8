// The backward of a linear layer (feature_linear.cu):
//
//   z = x W^T + b,  dz = dy act'(z)
//   dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dr = dy
//
// Narrow layers take one pass over the rows (feature_fused.cuh).  Wider ones
// form dz (in fp32, or in two values of a 16-bit type) and take a product each for
// dx and dW, the latter over ranges of rows whose sums are joined in a fixed order.
#include <algorithm>

#include "feature_fused.cuh"
#include "feature_join.cuh"
#include "feature_launch.cuh"
#include "feature_narrow.cuh"
#include "splat200.h"

namespace splat {
namespace feature {

// ---- sums over splits and rows ---------------------------------------------------

// Column sums of dz (m, n) over ranges of rows: a thread adds V neighbouring
// columns (V is 1 where rows are not whole 16-byte pieces), the block's eight
// rows of threads are joined in a fixed order.
template <class S, int V>
__global__ void __launch_bounds__(256) column_sums_kernel(const S* dz, long long m, int n,
                                                          long long rows, float* partial) {
  const int c = (blockIdx.x * 32 + threadIdx.x) * V;
  const long long begin = blockIdx.y * rows, end = min(begin + rows, m);
  float s[V] = {};
  if (c < n) {
    constexpr int U = 4;  // rows in flight
    const S* from = dz + (begin + threadIdx.y) * n + c;
    const long long stride = 8LL * n;
    for (long long r = begin + threadIdx.y; r < end; r += 8 * U, from += U * stride) {
      Vec<S, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + 8 * u < end) v[u] = *reinterpret_cast<const Vec<S, V>*>(from + u * stride);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + 8 * u < end) {
          float f[V];
          widen<S, V>(v[u], f);
#pragma unroll
          for (int j = 0; j < V; ++j) s[j] += f[j];
        }
    }
  }
  __shared__ float sums[8][32 * V];
#pragma unroll
  for (int j = 0; j < V; ++j) sums[threadIdx.y][threadIdx.x * V + j] = s[j];
  __syncthreads();
  const int t = threadIdx.y * 32 + threadIdx.x, col = blockIdx.x * 32 * V + t;
  if (t < 32 * V && col < n) {
    float a = 0.0f;
    for (int i = 0; i < 8; ++i) a += sums[i][t];
    partial[static_cast<long long>(blockIdx.y) * n + col] = a;
  }
}

constexpr int kMaxColumnSplits = 256;

// Their ranges of rows: eight blocks to an SM, 256 rows to a range at least.
template <class T>
int sum_columns(const T* dz, long long rows, int n, float* partial, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vector = n % V == 0 && host::aligned(dz, 16);
  const int blocks = host::blocks_for(n, vector ? 32 * V : 32);
  const long long wanted = std::max(1LL, 8LL * host::sm_count() / blocks);
  const long long count =
      std::min({wanted, (rows + 255) / 256, static_cast<long long>(kMaxColumnSplits)});
  const long long per = (rows + count - 1) / count;
  const int splits = static_cast<int>((rows + per - 1) / per);
  const dim3 grid(blocks, splits), block(32, 8);
  if (vector)
    column_sums_kernel<T, V><<<grid, block, 0, host::counted(s)>>>(dz, rows, n, per, partial);
  else
    column_sums_kernel<T, 1><<<grid, block, 0, host::counted(s)>>>(dz, rows, n, per, partial);
  return splits;
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

// dz: (rows, n); of 16-bit types in two parts, planes whose rows start on 16
// bytes.
bool two_parts(int dtype, int activation) { return dtype != kF32 && rounds_dz(activation); }
size_t dz_plane_bytes(long long rows, int n) {
  return static_cast<size_t>(rows) * round_to(n, 8) * 2;
}
size_t dz_bytes(int dtype, long long rows, int n, int activation) {
  if (two_parts(dtype, activation)) return 2 * dz_plane_bytes(rows, n);
  return activation == kNone ? 0 : round16(static_cast<size_t>(rows) * n * (dtype == kF32 ? 4 : 2));
}
// Whether x, W and a dz of one plane are laid out as planes before the products.
// With a dz of two the products copy all their operands.
template <class T>
bool backward_planes(int dtype, long long rows, int k, int n, int activation) {
  return two_parts(dtype, activation) ? k % 8 != 0 : wants_planes<T>(rows, k, n);
}

// Sums of dz over 32 rows each, of whole tiles.
size_t column_sums_bytes(long long rows, int n, int activation) {
  return activation == kNone
             ? 0
             : round16(static_cast<size_t>((rows + kTileRows - 1) / kTileRows) * 4 * n * 4);
}

// What the wide layers' products read: the tensors, or planes of them.
struct Sources {
  const void *x, *weight, *dz, *dz_second;    // dz_second: NULL: one part
  Planes x_planes, weight_planes, dz_planes;  // data: NULL without planes
  const float* column_sums;                   // NULL: dz is dy
};

// The two products of the backward; P: parts of dz.
template <class T, int P>
int launch_gradients(long long rows, int k, int n, const Sources& from, void* dx, void* dweight,
                     void* dbias, float* partial, cudaStream_t s) {
  constexpr int PB = kOperandParts<T>;
  const bool planes = from.dz_planes.data != nullptr;
  // a dz of two parts, by the matrix of whole 16-byte rows beside it
  const auto use_parts = [&](ProductParams& p, const Planes& b, const void* as_it_is) {
    p.a = from.dz, p.a_second = from.dz_second, p.a_ld = round_to(n, 8);
    p.b = b.data ? b.data : as_it_is, p.b_ld = b.data ? b.ld : k;
  };
  if (dx) {
    ProductParams p{};
    p.m = rows, p.k = n, p.n = k;
    p.a = from.dz, p.a_ld = n;
    p.b = from.weight, p.b_ld = k;
    p.k_per_split = n, p.splits = 1;
    p.out = dx;
    if constexpr (P == 2) use_parts(p, from.weight_planes, from.weight);
    else if (planes) use_planes(p, from.dz_planes, from.weight_planes);
    const int status = launch_product<T, P, false, T, PB, true, T, T, kPlain>(p, s);
    if (status != kOk) return status;
  }
  const Splits splits = weight_splits(rows, k, n);
  if (dweight) {
    ProductParams p{};
    p.m = n, p.k = rows, p.n = k;
    p.a = from.dz, p.a_ld = n;
    p.b = from.x, p.b_ld = k;
    p.k_per_split = splits.rows, p.splits = splits.count;
    p.out = partial;
    if constexpr (P == 2) use_parts(p, from.x_planes, from.x);
    else if (planes) use_planes(p, from.dz_planes, from.x_planes);
    const int status = launch_product<T, P, true, T, PB, true, float, float, kPlain>(p, s);
    if (status != kOk) return status;
    const long long count = static_cast<long long>(n) * k;
    join_splits<T>(partial, count, splits.count, count, 0, dweight, nullptr, s);
  }
  if (dbias) {
    float* sums = partial + static_cast<long long>(splits.count) * n * k;
    // of dy, or of the sums that the pass over z left of dz before its rounding
    const int count =
        from.column_sums
            ? sum_columns<float>(from.column_sums, (rows + 31) / 32, n, sums, s)
            : sum_columns<T>(static_cast<const T*>(from.dz), rows, n, sums, s);
    join_splits<T>(sums, n, count, n, 0, dbias, nullptr, s);
  }
  return host::check_launch("feature_linear_backward");
}

// ---- narrow layers: one pass -----------------------------------------------------

// How a narrow layer's pass is launched; blocks == 0: the layer is too wide.
struct FusedPlan {
  int blocks;
  bool copies;  // by tensor copies
  bool raw;     // or by bulk copies
  size_t bytes;
  uint32_t tmem_columns;
};

int round32(int n) { return (n + 31) / 32 * 32; }

template <class T>
FusedPlan plan_fused(long long rows, int k, int n, int activation) {
  using F = Fused<T>;
  FusedPlan plan{};
  if (k > kFusedWidth || n > kFusedWidth) return plan;
  const int k32 = round32(k), n32 = round32(n);
  plan.tmem_columns = 32;
  while (plan.tmem_columns < static_cast<uint32_t>(std::max(k32, n32) + F::kAcc * k32))
    plan.tmem_columns *= 2;
  const int row_align = 16 / static_cast<int>(sizeof(T));
  plan.copies = sizeof(T) == 2 && k % row_align == 0 && n % row_align == 0 && rows < 1LL << 31;
  int per_sm = 1;
  if (plan.copies) {
    plan.bytes = narrow_bytes(k, n, n32, rounds_dz(activation));
    plan.tmem_columns = 32;
    while (plan.tmem_columns < static_cast<uint32_t>(n32 + 2 * k32)) plan.tmem_columns *= 2;
    if (k <= 64 && n <= 64) per_sm = 2;
  } else {
    plan.bytes = F::shared_bytes(k, n, n32, false);
    if (plan.tmem_columns > 512 || plan.bytes > kOneBlockBytes) return plan;
    if (sizeof(T) == 2 && plan.tmem_columns <= 256 && plan.bytes <= kTwoBlocksBytes) per_sm = 2;
    const size_t raw = F::shared_bytes(k, n, n32, true);
    plan.raw = raw <= static_cast<size_t>(per_sm == 2 ? kTwoBlocksBytes : kOneBlockBytes);
    if (plan.raw) plan.bytes = raw;
  }
  // as many as are resident; of 16-bit types so many times more that no dW takes
  // more than kMostAdditions in tensor memory
  const long long tiles = (rows + kTileRows - 1) / kTileRows;
  long long blocks = static_cast<long long>(host::sm_count()) * per_sm;
  if (sizeof(T) == 2) {
    const bool two = rounds_dz(activation) && !(plan.copies && n <= 64);  // products a tile
    const long long most = kMostAdditions * 16 / kTileRows / (two ? 2 : 1);
    blocks *= std::max(1LL, (tiles + blocks * most - 1) / (blocks * most));
  }
  plan.blocks = static_cast<int>(std::min(tiles, blocks));
  return plan;
}

template <class T>
int launch_narrow(const FusedPlan& plan, long long rows, int k, int n, const void* x,
                  const void* weight, const void* bias, int activation, const void* dy, void* dx,
                  float* partial, cudaStream_t s) {
  NarrowParams p{};
  p.rows = rows, p.k = k, p.n = n, p.k32 = round32(k), p.n32 = round32(n);
  p.bias = bias, p.with_dx = dx != nullptr, p.partial = partial, p.activation = activation;
  p.tiles = static_cast<uint32_t>((rows + kTileRows - 1) / kTileRows);
  p.tmem_columns = plan.tmem_columns;
  p.error = host::device_error_word();
  if (!p.error) return kCudaError;
  if (!make_map<T>(p.x_map, x, rows, k, k, 64, kTileRows) ||
      !make_map<T>(p.dy_map, dy, rows, n, n, 64, kTileRows) ||
      !make_map<T>(p.w_map, weight, n, k, k, 64, p.n32) ||
      (dx && !make_map<T>(p.dx_map, dx, rows, k, k, 32, 32)))
    return host::fail(kInvalidArgument,
                      "feature_linear_backward: tensors must be 16-byte aligned");
  const bool wide = k > 64 || n > 64;
  if (!(wide ? host::allow_shared<narrow_backward_kernel<T, true>>()
             : host::allow_shared<narrow_backward_kernel<T, false>>()))
    return host::check_launch("feature_linear_backward: shared memory");
  auto* kernel = wide ? narrow_backward_kernel<T, true> : narrow_backward_kernel<T, false>;
  kernel<<<plan.blocks, kNarrowThreads, plan.bytes, host::counted(s)>>>(p);
  return host::check_launch("feature_linear_backward");
}

template <class T>
int launch_fused(const FusedPlan& plan, long long rows, int k, int n, const void* x,
                 const void* weight, const void* bias, int activation, const void* dy, void* dx,
                 void* dweight, void* dbias, float* partial, cudaStream_t s) {
  if (!dweight && !dbias) partial = nullptr;
  if constexpr (sizeof(T) == 2) {
    if (plan.copies) {
      const int status =
          launch_narrow<T>(plan, rows, k, n, x, weight, bias, activation, dy, dx, partial, s);
      if (status != kOk) return status;
    }
  }
  if (!plan.copies) {
    FusedParams p{};
    p.rows = rows, p.k = k, p.n = n, p.k32 = round32(k), p.n32 = round32(n);
    p.x = x, p.weight = weight, p.bias = bias, p.dy = dy, p.dx = dx;
    p.partial = partial;
    p.activation = activation;
    p.raw = plan.raw;
    if (p.raw && !(host::aligned(x, 16) && host::aligned(dy, 16)))
      return host::fail(kInvalidArgument,
                        "feature_linear_backward: x and dy must be 16-byte aligned");
    p.x_vector = row_vector<T>(x, k);
    p.w_vector = row_vector<T>(weight, k);
    p.dy_vector = n * sizeof(T) % 16 == 0 && host::aligned(dy, 16);
    p.dx_vector = k * sizeof(T) % 16 == 0 && host::aligned(dx, 16);
    p.tiles = static_cast<uint32_t>((rows + kTileRows - 1) / kTileRows);
    p.tmem_columns = plan.tmem_columns;
    p.error = host::device_error_word();
    if (!p.error) return kCudaError;
    if (!host::allow_shared<fused_backward_kernel<T>>())
      return host::check_launch("feature_linear_backward: shared memory");
    fused_backward_kernel<T><<<plan.blocks, kFusedThreads, plan.bytes, host::counted(s)>>>(p);
  }
  if (partial) {
    const long long count = static_cast<long long>(n) * k;
    join_splits<T>(partial, count + n, plan.blocks, count, n, dweight, dbias, s);
  }
  return host::check_launch("feature_linear_backward");
}

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

size_t splat_feature_linear_backward_workspace_bytes(int dtype, long long rows, int k, int n,
                                                     int activation) {
  if (check_linear(dtype, rows, k, n, activation) != kOk) return 0;
  const FusedPlan plan = SPLAT_FEATURE_TYPE(dtype, [&] {
    return plan_fused<T>(rows, k, n, activation);
  });
  const size_t sums = static_cast<size_t>(n) * (static_cast<size_t>(k) + 1) * 4;
  if (plan.blocks) return plan.blocks * sums;
  return dz_bytes(dtype, rows, n, activation) +
         round16(static_cast<size_t>(weight_splits(rows, k, n).count) * n * k * 4) +
         round16(static_cast<size_t>(kMaxColumnSplits) * n * 4) +
         column_sums_bytes(rows, n, activation) +
         SPLAT_FEATURE_TYPE(dtype, [&] {
           return backward_planes<T>(dtype, rows, k, n, activation)
                      ? plane_bytes<T>(rows, k) + plane_bytes<T>(n, k) +
                            (two_parts(dtype, activation) ? 0 : plane_bytes<T>(rows, n))
                      : static_cast<size_t>(0);
         });
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
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    const FusedPlan plan = plan_fused<T>(rows, k, n, activation);
    if (plan.blocks)
      return launch_fused<T>(plan, rows, k, n, x, weight, bias, activation, dy, dx, dweight,
                             dbias, static_cast<float*>(workspace), s);
    constexpr int P = kOperandParts<T>;
    char* at = static_cast<char*>(workspace);
    void* dz = at;
    at += dz_bytes(dtype, rows, n, activation);
    float* partial = reinterpret_cast<float*>(at);
    at += round16(static_cast<size_t>(weight_splits(rows, k, n).count) * n * k * 4) +
          round16(static_cast<size_t>(kMaxColumnSplits) * n * 4);
    float* column_sums = reinterpret_cast<float*>(at);
    at += column_sums_bytes(rows, n, activation);
    Sources from{x, weight, activation == kNone ? dy : dz, nullptr, {}, {}, {}, nullptr};
    const bool planes = backward_planes<T>(dtype, rows, k, n, activation);
    if (two_parts(dtype, activation)) {
      if (rows >= 1LL << 31)
        return host::fail(kTooLarge, "feature_linear_backward: too many rows of a wide layer");
      if (!planes && !(host::aligned(x, 16) && host::aligned(weight, 16)))
        return host::fail(kInvalidArgument,
                          "feature_linear_backward: tensors must be 16-byte aligned");
      from.dz_second = static_cast<char*>(dz) + dz_plane_bytes(rows, n);
    }
    if (planes) {
      if (dweight || activation != kNone) from.x_planes = split<T>(x, rows, k, at, s);
      at += plane_bytes<T>(rows, k);
      if (dx || activation != kNone) from.weight_planes = split<T>(weight, n, k, at, s);
      at += plane_bytes<T>(n, k);
    }
    if (activation != kNone) {
      ProductParams p = forward_params<T>(rows, k, n, x, weight, bias, dy, activation, dz);
      if (planes) use_planes(p, from.x_planes, from.weight_planes);
      if (from.dz_second) {
        p.out_second = const_cast<void*>(from.dz_second);
        p.out_ld = round_to(n, 8);
      }
      if (dbias) from.column_sums = p.column_sums = column_sums;
      const int status = launch_product<T, P, false, T, P, false, T, T, kSlope>(p, s);
      if (status != kOk) return status;
    }
    if constexpr (sizeof(T) == 2) {
      if (from.dz_second)
        return launch_gradients<T, 2>(rows, k, n, from, dx, dweight, dbias, partial, s);
    }
    if (planes && (dx || dweight)) from.dz_planes = split<T>(from.dz, rows, n, at, s);
    return launch_gradients<T, P>(rows, k, n, from, dx, dweight, dbias, partial, s);
  });
}

}  // extern "C"
