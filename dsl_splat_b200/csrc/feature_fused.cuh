// The backward of a linear layer in one pass over its rows:
//
//   z = x W^T + b, dz = dy act'(z), dx = dz W, dW += dz^T x, db += dz^T 1
//
// for layers whose W and one 128-row tile of x and dz fit in shared memory.
// x and dy are read once and dx is written once; the three products of a tile
// take the same copies of x, dz and W, as K-major operands in one and MN-major
// ones in the other.  dW stays in tensor memory (16-bit types; a block has no more
// tiles than kMostAdditions allow) or is added up in registers after every tile
// (fp32).  db is folded from the
// lanes' rows of dz before dz is rounded or split.
//
// A block of 16 warps does each tile's steps together: load, product,
// activation slope, products, store, while bulk copies bring the next tile's x
// and dy (contiguous whatever their row lengths) to shared memory; where those
// do not fit beside the operands, the steps read global memory.
// 16-bit types with 16-byte rows take the pass of feature_narrow.cuh instead.
// Bound by the steps' latencies one after another: 35 -> 32 fp32 gelu over 10^6
// rows 365 us where 408 MB take 62 us to copy.
#pragma once
#include "feature_product.cuh"

namespace splat {
namespace feature {

struct FusedParams {
  long long rows;
  int k, n, k32, n32;  // widths rounded up to 32
  const void *x, *weight, *bias, *dy;
  void* dx;        // (rows, k) or NULL
  float* partial;  // per block: (n, k) of dW, then (n) of db; NULL: neither
  int activation, x_vector, w_vector, dy_vector, dx_vector;
  // x and dy are copied ahead (training of 35 -> 64 bf16 over 10^6 rows 254 us
  // against 286 read as needed, 35 -> 32 fp32 468 against 534)
  int raw;
  uint32_t tiles, tmem_columns;
  int* error;
};

constexpr int kFusedThreads = 512, kFusedWarps = kFusedThreads / 32;
// Widest k and n: what fits in shared memory there is faster in one pass
// (silu training over 500000 rows against the products: 64 -> 64 bf16 118 us
// against 192, 128 -> 128 bf16 202 against 337, 64 -> 64 fp32 297 against 462,
// 128 -> 64 fp32 636 against 648).
constexpr int kFusedWidth = 128;
constexpr int kJoinBytes = 4 * kFusedWidth * 4;  // db of the four blocks of rows

template <class T>
struct Fused {
  static constexpr int P = sizeof(T) == 4 ? 3 : 1;   // parts of x and W
  static constexpr int PZ = sizeof(T) == 4 ? 3 : 2;  // of dz (take_first)
  static constexpr int kAcc = sizeof(T) == 4 ? 2 : 1;  // accumulators of dW
  __host__ __device__ static int blocks64(int n) { return (n + 63) / 64; }
  // a patch of 32 x 16 values for each warp
  __host__ __device__ static int staging_bytes() { return kFusedWarps * 512 * sizeof(T); }
  // a tile of rows of n values as it is in memory
  __host__ __device__ static int raw_bytes(int n) {
    return (kTileRows * n * static_cast<int>(sizeof(T)) + 127) / 128 * 128;
  }
  __host__ __device__ static int x_plane(int k) { return blocks64(k) * kAPlane; }
  __host__ __device__ static int w_plane(int k, int n32) { return blocks64(k) * n32 * 128; }
  static size_t shared_bytes(int k, int n, int n32, bool raw) {
    return static_cast<size_t>(staging_bytes()) + P * x_plane(k) + PZ * x_plane(n) +
           P * w_plane(k, n32) + kJoinBytes + 1024 + kFusedWidth * 4 +
           (raw ? raw_bytes(k) + raw_bytes(n) : 0);
  }
};

template <class T>
__global__ void __launch_bounds__(kFusedThreads, sizeof(T) == 4 ? 1 : 2)
    fused_backward_kernel(const __grid_constant__ FusedParams p) {
  using F = Fused<T>;
  constexpr int kAcc = F::kAcc;
  constexpr int P = F::P, PZ = F::PZ;
  extern __shared__ unsigned char dynamic[];
  __shared__ alignas(8) unsigned long long z_done, dx_done, dw_done, drained, x_raw, dy_raw;
  __shared__ uint32_t tmem_base;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const uint32_t x_plane = F::x_plane(p.k), z_plane = F::x_plane(p.n);
  const uint32_t w_plane = F::w_plane(p.k, p.n32);
  const uint32_t x_at = base + F::staging_bytes();
  const uint32_t z_at = x_at + P * x_plane;
  const uint32_t w_at = z_at + PZ * z_plane;
  const uint32_t join_at = w_at + P * w_plane;
  const uint32_t bias_at = join_at + kJoinBytes;
  const int warp = tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // a warp's patches: 16 columns from 16 group on, and from 64 + 16 group on
  const int lane_block = warp & 3, group = warp >> 2;
  const Patch<T, 16> patch{base + warp * static_cast<uint32_t>(512 * sizeof(T))};
  const uint32_t x_raw_at = bias_at + kFusedWidth * 4;
  const uint32_t dy_raw_at = x_raw_at + F::raw_bytes(p.k);
  const T* x = static_cast<const T*>(p.x);
  // one thread: copies of a tile
  const auto copy_rows = [&](const void* from, int width, uint32_t tile, uint32_t to,
                             unsigned long long& bar) {
    const long long m0 = static_cast<long long>(tile) * kTileRows;
    copy_run<T>(to, static_cast<const T*>(from) + m0 * width,
                static_cast<int>(min(p.rows - m0, static_cast<long long>(kTileRows))) * width,
                tc::shared_address(&bar));
  };
  const bool with_z = p.activation != kNone;
  // parts of dz: its 16-bit values have one where dz has dy's digits
  const int z_parts = sizeof(T) == 4 ? PZ : rounds_dz(p.activation) ? 2 : 1;

  if (threadIdx.x == 0) {
    tc::barrier_init(tc::shared_address(&z_done), 1);
    tc::barrier_init(tc::shared_address(&dx_done), 1);
    tc::barrier_init(tc::shared_address(&dw_done), 1);
    tc::barrier_init(tc::shared_address(&drained), 1);
    tc::barrier_init(tc::shared_address(&x_raw), 1);
    tc::barrier_init(tc::shared_address(&dy_raw), 1);
    tc::barrier_init_fence();
    if (p.raw) {
      copy_rows(p.x, p.k, blockIdx.x, x_raw_at, x_raw);
      copy_rows(p.dy, p.n, blockIdx.x, dy_raw_at, dy_raw);
    }
  }
  if (warp == 0) tc::tmem_alloc(tc::shared_address(&tmem_base), p.tmem_columns);
  // W and the bias stay for all tiles
  for (int c = 0; c * 64 < p.k; ++c)
    fill<T, P>(p.w_vector, w_at + c * p.n32 * 128, w_plane, p.n32, 8,
                static_cast<const T*>(p.weight) + c * 64, p.k, p.n, p.k - c * 64, threadIdx.x,
                kFusedThreads);
  for (int i = threadIdx.x; i < p.n32; i += kFusedThreads)
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(bias_at + i * 4),
                 "f"(p.bias && i < p.n ? to_float(static_cast<const T*>(p.bias)[i]) : 0.0f)
                 : "memory");

  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tc::uniform(tmem_base);
  const uint32_t acc_w = tmem + max(p.k32, p.n32);

  float sum_w[kAcc == 2 ? 2 : 1][16] = {};  // fp32: this thread's part of dW
  // db of this lane's columns, from dz before its rounding
  float sum_b[2] = {0.0f, 0.0f};
  uint32_t parity = 0;
  bool ok = true, fresh = true;
  for (uint32_t t = blockIdx.x; t < p.tiles; t += gridDim.x, parity ^= 1) {
    const long long row0 = static_cast<long long>(t) * kTileRows + lane_block * 32;
    const int rows = static_cast<int>(max(min(p.rows - row0, 32LL), 0LL));
    const long long m0 = static_cast<long long>(t) * kTileRows;
    const bool next = p.tiles - t > gridDim.x;
    if (p.raw) ok = tc::barrier_wait(tc::shared_address(&x_raw), parity) && ok;
    for (int c = 0; c * 64 < p.k; ++c) {
      const int valid = p.k - c * 64, pieces = min((valid + 15) / 16 * 2, 8);
      if (p.raw)
        fill_shared<T, P>(p.x_vector, x_at + c * kAPlane, x_plane, kTileRows, pieces,
                          x_raw_at + c * 64 * static_cast<int>(sizeof(T)),
                          p.k * static_cast<int>(sizeof(T)),
                          static_cast<int>(min(p.rows - m0, static_cast<long long>(kTileRows))),
                          valid, threadIdx.x, kFusedThreads);
      else
        fill<T, P>(p.x_vector, x_at + c * kAPlane, x_plane, kTileRows, pieces, x + m0 * p.k + c * 64,
                   p.k, p.rows - m0, valid, threadIdx.x, kFusedThreads);
    }
    tc::fence_async_proxy();
    tc::fence_before_sync();
    // x is there, and the previous tile's accumulators have been read
    if (__syncthreads_or(!ok)) break;
    if (threadIdx.x == 32 && p.raw && next)
      copy_rows(p.x, p.k, t + gridDim.x, x_raw_at, x_raw);
    if (warp == 0 && with_z) {
      const uint32_t lead = tc::elected();
      tc::fence_after_sync();
      const uint32_t instruction = tc::instruction(!kIsF16<T>, false, false, p.n32);
      bool first = true;
#pragma unroll
      for (int sum = P - 1; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i <= sum; ++i)
          for (int c = 0; c * 64 < p.k; ++c) {
            tc::mma_steps(lead, tmem, tc::descriptor_k_major(x_at + i * x_plane + c * kAPlane),
                          tc::descriptor_k_major(w_at + (sum - i) * w_plane + c * p.n32 * 128),
                          tc::kStepK, tc::kStepK, min((p.k - c * 64 + 15) / 16, 4), instruction,
                          !first);
            first = false;
          }
      tc::commit(lead, tc::shared_address(&z_done));
    }
    // dz: a lane's row of each patch
    bool waited = !with_z;
    if (p.raw) ok = tc::barrier_wait(tc::shared_address(&dy_raw), parity) && ok;
    for (int c = group * 16; c < p.n32; c += 64) {
      const int cols = min(p.n - c, 16);
      __syncwarp();
      if (p.raw)
        patch.load_shared_rows(
            dy_raw_at + ((lane_block * 32) * p.n + c) * static_cast<int>(sizeof(T)), p.n, rows, cols,
            p.dy_vector);
      else
        patch.load(static_cast<const T*>(p.dy) + row0 * p.n + c, p.n, rows, cols, p.dy_vector);
      __syncwarp();
      float v[16];
      if (!waited) {
        ok = tc::barrier_wait(tc::shared_address(&z_done), parity) && ok;
        tc::fence_after_sync();
        waited = true;
      }
      if (with_z) {
        tc::tmem_load16(tmem + (lane_block << 21) + c, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 b = load_shared(bias_at + (c + j * 4) * 4);
          unpack2(add2(pack2(v[4 * j], v[4 * j + 1]), pack2(b.x, b.y)), v[4 * j], v[4 * j + 1]);
          unpack2(add2(pack2(v[4 * j + 2], v[4 * j + 3]), pack2(b.z, b.w)), v[4 * j + 2],
                  v[4 * j + 3]);
        }
      }
      switch (p.activation) {
        case kRelu: finish_row<kSlope, kRelu, T>(patch, true, v); break;
        case kSilu: finish_row<kSlope, kSilu, T>(patch, true, v); break;
        case kGelu: finish_row<kSlope, kGelu, T>(patch, true, v); break;
        case kSigmoid: finish_row<kSlope, kSigmoid, T>(patch, true, v); break;
        default: finish_row<kSlope, kNone, T>(patch, true, v);
      }
      if (lane >= rows) {  // rows past the end add nothing to dW
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.0f;
      }
      __syncwarp();
      const float columns = sum_rows<16>(v);
      if (c < 64) sum_b[0] += columns;
      else sum_b[1] += columns;
      const int row = lane_block * 32 + lane;
      const uint32_t at = z_at + (c >> 6) * kAPlane + row * 128;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4 parts[PZ];
        if constexpr (sizeof(T) == 2) {
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = v[j * 8 + i];
          const Vec<T, 8> r = z_parts == 1 ? round_values<T, 8>(o) : take_first<T, 8>(o);
          parts[0] = reinterpret_cast<const uint4&>(r);
          const Vec<T, 8> second = round_values<T, 8>(o);
          parts[1] = reinterpret_cast<const uint4&>(second);
        } else {
          Vec<float, 8> o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o.v[i] = v[j * 8 + i];
          to_parts<float, PZ>(o, parts);
        }
#pragma unroll
        for (int q = 0; q < PZ; ++q)
          store_shared(at + q * z_plane + ((((c & 63) / 8 + j) ^ (row & 7)) << 4), parts[q]);
      }
    }
    tc::fence_async_proxy();
    tc::fence_before_sync();
    __syncthreads();  // dz is there, z has been read
    if (threadIdx.x == 32 && p.raw && next)
      copy_rows(p.dy, p.n, t + gridDim.x, dy_raw_at, dy_raw);
    if (warp == 0) {
      const uint32_t lead = tc::elected();
      tc::fence_after_sync();
      if (p.dx) {
        const uint32_t instruction = tc::instruction(!kIsF16<T>, false, true, p.k32);
        bool first = true;
#pragma unroll
        for (int sum = PZ - 1; sum >= 0; --sum)
#pragma unroll
          for (int i = 0; i < PZ; ++i) {
            const int j = sum - i;
            if (j < 0 || j >= P || i >= z_parts) continue;
            for (int c = 0; c * 64 < p.n; ++c) {
              tc::mma_steps(lead, tmem, tc::descriptor_k_major(z_at + i * z_plane + c * kAPlane),
                            tc::descriptor_mn_major(w_at + j * w_plane + c * 4 * tc::kStepMn,
                                                    p.n32 * 128),
                            tc::kStepK, tc::kStepMn, min((p.n - c * 64 + 15) / 16, 4),
                            instruction, !first);
              first = false;
            }
          }
      }
      tc::commit(lead, tc::shared_address(&dx_done));
      if (p.partial) {
        // n of up to 64 take one block of dz twice; the upper lanes are not read
        const uint32_t z_block = p.n > 64 ? kAPlane : 0;
        const uint32_t wide = tc::instruction(!kIsF16<T>, true, true, p.k32);
        // the first product into an accumulator overwrites it
        bool start = kAcc == 2 || fresh;
#pragma unroll
        for (int sum = PZ - 1; sum >= 0; --sum)
#pragma unroll
          for (int i = 0; i < PZ; ++i) {
            const int j = sum - i;
            if (j < 0 || j >= P || i >= z_parts) continue;
            const bool own = sum == 0 && kAcc == 2;
            const bool first = start || own;
            if (!own) start = false;
            tc::mma_steps(lead, acc_w + (own ? 0 : (kAcc - 1) * p.k32),
                          tc::descriptor_mn_major(z_at + i * z_plane, z_block),
                          tc::descriptor_mn_major(x_at + j * x_plane, kAPlane), tc::kStepMn,
                          tc::kStepMn, kTileRows / 16, wide, !first);
          }
      }
      tc::commit(lead, tc::shared_address(&dw_done));
    }
    fresh = false;
    if (p.dx) {
      ok = tc::barrier_wait(tc::shared_address(&dx_done), parity) && ok;
      tc::fence_after_sync();
      for (int c = group * 16; c < p.k; c += 64) {
        float v[16];
        tc::tmem_load16(tmem + (lane_block << 21) + c, v);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < Patch<T, 16>::kPieces; ++j) {
          constexpr int V = Patch<T, 16>::V;
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] = v[j * V + i];
          const Vec<T, V> r = round_values<T, V>(o);
          store_shared(patch.at(lane, j), reinterpret_cast<const uint4&>(r));
        }
        __syncwarp();
        patch.store(static_cast<T*>(p.dx) + row0 * p.k + c, p.k, rows, min(p.k - c, 16),
                    p.dx_vector, false);
      }
    }
    // the tile's operands are free once its last products are done
    ok = tc::barrier_wait(tc::shared_address(&dw_done), parity) && ok;
    tc::fence_after_sync();
    if constexpr (kAcc == 2) {
      if (p.partial && lane_block * 32 < p.n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = group * 16 + 64 * i;
          if (c < p.k) {
            float v[16];
            tc::tmem_load16(acc_w + (lane_block << 21) + c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) sum_w[i][j] += v[j];
            tc::tmem_load16(acc_w + (lane_block << 21) + p.k32 + c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) sum_w[i][j] += v[j];
          }
        }
      }
    }
  }

  // this block's sums
  if (p.partial && !fresh) {
    float* out = p.partial + static_cast<size_t>(blockIdx.x) * p.n * (p.k + 1);
    const int row = lane_block * 32 + lane;
    if (lane_block * 32 < p.n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = group * 16 + 64 * i;
        if (c < p.k) {
          float v[16];
          if constexpr (kAcc == 2) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = sum_w[i][j];
          } else {
            tc::tmem_load16(acc_w + (lane_block << 21) + c, v);
          }
          if (row < p.n) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (c + j < p.k) out[row * p.k + c + j] = v[j];
          }
        }
      }
    }
    // both lanes of a column have its sum
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = group * 16 + 64 * i + lane / 2;
      if (lane % 2 == 0 && c < p.n)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(join_at + (lane_block * kFusedWidth + c) * 4),
                     "f"(sum_b[i])
                     : "memory");
    }
  }
  if (threadIdx.x == 0) {  // nothing is in flight past this, also after a wait that ran out
    if (p.raw && !ok) {
      tc::barrier_wait(tc::shared_address(&x_raw), parity);
      tc::barrier_wait(tc::shared_address(&dy_raw), parity);
      tc::barrier_wait(tc::shared_address(&x_raw), parity ^ 1);
      tc::barrier_wait(tc::shared_address(&dy_raw), parity ^ 1);
    }
  }
  if (warp == 0) {
    tc::commit(tc::elected(), tc::shared_address(&drained));
    ok = tc::barrier_wait(tc::shared_address(&drained), 0) && ok;
  }
  if (!ok) atomicCAS(p.error, 0, kDeviceTimeout);
  tc::fence_before_sync();
  __syncthreads();
  if (p.partial && !fresh && threadIdx.x < p.n) {
    float s = 0.0f;
    for (int q = 0; q < 4; ++q) {
      float v;
      asm volatile("ld.shared.f32 %0, [%1];"
                   : "=f"(v)
                   : "r"(join_at + (q * kFusedWidth + threadIdx.x) * 4)
                   : "memory");
      s += v;
    }
    p.partial[static_cast<size_t>(blockIdx.x) * p.n * (p.k + 1) + p.n * p.k + threadIdx.x] = s;
  }
  if (warp == 0) tc::tmem_free(tmem, p.tmem_columns);
}

}  // namespace feature
}  // namespace splat
