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
    constexpr int P = kOperandParts<T>;
    return launch_product<T, P, false, T, P, false, T, T, kForward>(
        forward_params<T>(rows, k, n, x, weight, bias, residual, activation, y), s);
  });
}

}  // extern "C"
