// Host-side helpers shared by the translation units of libsplat200: status
// reporting (splat_last_error), the launch counter (splat_launch_count) and
// argument checks.  Defined in splat200.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace splat {
namespace host {

// Records `what` as the calling thread's last error and returns `status`.
int fail(int status, const char* what);
// kOk, or kCudaError (recording the CUDA error) when a launch failed.
int check_launch(const char* what);
// Counts one kernel launch and returns its stream; every launch passes its
// stream through here.
cudaStream_t counted(cudaStream_t s);
// The current device's error word (splat_device_error), or NULL with the CUDA
// error recorded.
int* device_error_word();
// A tensor map of a row-major matrix for boxes of box_columns x box_rows;
// false when the driver does not make one.
bool encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows,
                long long columns, long long row_bytes, int box_columns, int box_rows,
                CUtensorMapSwizzle swizzle);
// Streaming multiprocessors of the current device (148 on B200).
int sm_count();

// Lets a kernel (of less than 1 KB of static shared memory) take as much
// dynamic shared memory as a block can have, once per device.
template <auto* kernel>
bool allow_shared() {
  static unsigned long long done[2] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  unsigned long long* word = &done[(dev >> 6) & 1];
  const unsigned long long bit = 1ULL << (dev & 63);
  if (__atomic_load_n(word, __ATOMIC_ACQUIRE) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           226 * 1024) != cudaSuccess)
    return false;
  __atomic_fetch_or(word, bit, __ATOMIC_RELEASE);
  return true;
}

inline unsigned blocks_for(long long n, int block) {
  return static_cast<unsigned>((n + block - 1) / block);
}

// float2/float4 rows and 16-byte async copies need 8/16-byte aligned
// addresses (NULL passes; it means "absent").
inline bool aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

}  // namespace host
}  // namespace splat
