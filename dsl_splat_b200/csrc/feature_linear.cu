// A linear layer over feature rows with bias, activation and residual in its
// epilogue:
//
//   y = act(x W^T + b) + r      x (M, K), W (N, K), b (N), r, y (M, N)
//
// Its backward (feature_linear_backward.cu) recomputes x W^T + b, so nothing
// besides the inputs is kept.
#include "feature_launch.cuh"
#include "splat200.h"

namespace splat {
namespace feature {

int check_linear(int dtype, long long rows, int k, int n, int activation) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "feature_linear: dtype");
  if (activation < 0 || activation > 4)
    return host::fail(kInvalidArgument, "feature_linear: activation");
  if (rows < 1 || k < 1 || n < 1) return host::fail(kInvalidArgument, "feature_linear: sizes");
  if (k > 65535 || n > 65535 || rows > (1LL << 36))
    return host::fail(kTooLarge, "feature_linear: too many rows, inputs or outputs");
  return kOk;
}

// The forward takes planes where its x would be converted for several tiles
// (n above 128) or its rows are long.  Over 200000 rows: 128 -> 128 fp32 69 us
// without against 106 with, 101 -> 128 bf16 46 against 56, 255 -> 128 bf16 106
// against 96.
template <class T>
bool forward_planes(long long rows, int k, int n) {
  if (sizeof(T) == 2 && k % 8 == 0) return false;  // copied as it is
  const int longest = sizeof(T) == 4 ? 128 : 192;
  return wants_planes<T>(rows, k, n) && (n > 128 || k > longest);
}

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

size_t splat_feature_linear_workspace_bytes(int dtype, long long rows, int k, int n) {
  if (check_linear(dtype, rows, k, n, 0) != kOk) return 0;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    return forward_planes<T>(rows, k, n) ? plane_bytes<T>(rows, k) + plane_bytes<T>(n, k)
                                         : static_cast<size_t>(16);
  });
}

int splat_feature_linear(int dtype, long long rows, int k, int n, const void* x,
                         const void* weight, const void* bias, const void* residual,
                         int activation, void* y, void* workspace, size_t workspace_bytes,
                         void* stream) {
  const int bad = check_linear(dtype, rows, k, n, activation);
  if (bad != kOk) return bad;
  if (!x || !weight || !y) return host::fail(kInvalidArgument, "feature_linear: null pointer");
  auto s = static_cast<cudaStream_t>(stream);
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    constexpr int P = kOperandParts<T>;
    ProductParams p =
        forward_params<T>(rows, k, n, x, weight, bias, residual, activation, y);
    if (forward_planes<T>(rows, k, n)) {
      const size_t x_bytes = plane_bytes<T>(rows, k);
      if (!workspace || workspace_bytes < x_bytes + plane_bytes<T>(n, k))
        return host::fail(kWorkspaceTooSmall, "feature_linear: workspace");
      if (!host::aligned(workspace, 16))
        return host::fail(kInvalidArgument, "feature_linear: workspace not 16-byte aligned");
      char* at = static_cast<char*>(workspace);
      use_planes(p, split<T>(x, rows, k, at, s), split<T>(weight, n, k, at + x_bytes, s));
    }
    return launch_product<T, P, false, T, P, false, T, T, kForward>(p, s);
  });
}

}  // extern "C"
