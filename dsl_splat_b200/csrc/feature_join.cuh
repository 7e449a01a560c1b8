// Joining the partial sums of blocks or splits in a fixed order.
#pragma once
#include "feature_common.cuh"
#include "host_runtime.h"

namespace splat {
namespace feature {

// Adds the splits' partial sums, `stride` values apart, in a fixed order and in
// doubles (there may be a million): 32 threads to a value.  The first count_a
// values go to a, the rest to b.
constexpr int kJoinLanes = 32;
template <class T>
__global__ void __launch_bounds__(32 * kJoinLanes)
    join_splits_kernel(const float* partial, long long stride, int splits, long long count_a,
                       long long count_b, T* a, T* b) {
  const long long i = blockIdx.x * 32LL + threadIdx.x, count = count_a + count_b;
  double s = 0.0;
  if (i < count) {
    constexpr int U = 8;  // reads in flight
    for (int k0 = threadIdx.y; k0 < splits; k0 += U * kJoinLanes) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = k0 + u * kJoinLanes < splits ? partial[(k0 + u * kJoinLanes) * stride + i] : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) s += v[u];
    }
  }
  __shared__ double sums[kJoinLanes][33];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  // a warp to a value, its lanes' sums in a fixed tree
  s = sums[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const long long j = blockIdx.x * 32LL + threadIdx.y;
  if (threadIdx.x == 0 && j < count) {
    T* to = j < count_a ? a : b;
    if (to) to[j < count_a ? j : j - count_a] = from_float<T>(static_cast<float>(s));
  }
}

// The same with four neighbouring values to a thread, for few splits and one
// destination.
template <class T>
__global__ void __launch_bounds__(256)
    join_quads_kernel(const float4* partial, long long stride, int splits, long long count, T* a) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= count) return;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int k = 0; k < splits; ++k) {
    const float4 v = partial[k * stride + i];
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const float f[4] = {s.x, s.y, s.z, s.w};
  reinterpret_cast<Vec<T, 4>*>(a)[i] = round_values<T, 4>(f);
}

template <class T>
void join_splits(const float* partial, long long stride, int splits, long long count_a,
                 long long count_b, void* a, void* b, cudaStream_t s) {
  // enough quads to fill the device without several threads to a value
  if (!b && count_b == 0 && count_a % 4 == 0 && stride % 4 == 0 && count_a >= 1 << 16 &&
      host::aligned(a, 16) && host::aligned(partial, 16)) {
    join_quads_kernel<T><<<host::blocks_for(count_a / 4, 256), 256, 0, host::counted(s)>>>(
        reinterpret_cast<const float4*>(partial), stride / 4, splits, count_a / 4,
        static_cast<T*>(a));
    return;
  }
  join_splits_kernel<T>
      <<<host::blocks_for(count_a + count_b, 32), dim3(32, kJoinLanes), 0, host::counted(s)>>>(
          partial, stride, splits, count_a, count_b, static_cast<T*>(a), static_cast<T*>(b));
}

}  // namespace feature
}  // namespace splat
