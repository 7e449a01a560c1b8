// The backward of a narrow linear layer in one pass (feature_fused.cuh has the
// formulas) for 16-bit types whose rows are whole 16-byte pieces, so that
// tensor copies bring x and dy to shared memory and take dx from it.
//
// Two tiles are in flight.  dy arrives in the layout of a tensor-core operand
// and dz overwrites it in place: its first value (take_first).  The second
// values have one plane, which is written once the products of the tile before
// have read it; without an activation and for ReLU dz has dy's digits and there
// are none.  While the eight compute warps turn dy into dz for tile t, the products of tile t - 1
// finish; they then store its dx while the tensor core forms z of tile t + 1, dW
// and dx of tile t.  db is summed in registers from dz before its rounding.
//
// Bound by memory and by the latency of 16 compute warps to an SM: 64 -> 64 bf16
// over 1600x1200 rows moves 737 MB in 140 us without an activation and in 193 with
// SiLU (112 us at the copy rate).  There dW's second values take the tensor core's
// idle lanes: as a product of their own 206 us.
#pragma once
#include "feature_product.cuh"

namespace splat {
namespace feature {

struct NarrowParams {
  CUtensorMap x_map, dy_map, w_map, dx_map;
  long long rows;
  int k, n, k32, n32;
  const void* bias;
  int with_dx;
  float* partial;  // per block: (n, k) of dW, then (n) of db; NULL: neither
  int activation;
  uint32_t tiles, tmem_columns;
  int* error;
};

constexpr int kNarrowThreads = 320;  // eight compute warps, one for products, one for copies
constexpr int kNarrowWidth = 128;

__host__ __device__ inline int blocks64(int n) { return (n + 63) / 64; }

// x and dy of two tiles, dz's second values, W, a patch per warp, the bias and
// db's joins.
inline size_t narrow_bytes(int k, int n, int n32, bool second) {
  return (2 * (blocks64(k) + blocks64(n)) + (second ? blocks64(n) : 0)) *
             static_cast<size_t>(kAPlane) +
         static_cast<size_t>(blocks64(k)) * n32 * 128 + 8 * 2048 + 5 * kNarrowWidth * 4 + 1024;
}

// WIDE: k or n above 64; such a block has an SM to itself.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kNarrowThreads, WIDE ? 1 : 2)
    narrow_backward_kernel(const __grid_constant__ NarrowParams p) {
  constexpr int C = WIDE ? 2 : 1;  // 32-wide chunks of a warp
  extern __shared__ unsigned char dynamic[];
  __shared__ alignas(8) unsigned long long full[2], spent[2], dz_ready[2], w_full, z_done, dx_done,
      dx_read, all_done;
  __shared__ uint32_t tmem_base;
  const uint32_t base = (tc::shared_address(dynamic) + 1023u) & ~1023u;
  const uint32_t x_bytes = blocks64(p.k) * kAPlane, z_bytes = blocks64(p.n) * kAPlane;
  const bool with_z = p.activation != kNone, with_second = rounds_dz(p.activation);
  const uint32_t x_at = base, z_at = x_at + 2 * x_bytes, second_at = z_at + 2 * z_bytes;
  const uint32_t w_at = second_at + (with_second ? z_bytes : 0);
  const uint32_t w_block = p.n32 * 128;
  const uint32_t patch_at = w_at + blocks64(p.k) * w_block;
  const uint32_t bias_at = patch_at + 8 * 2048, join_at = bias_at + kNarrowWidth * 4;
  const int warp = tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const auto bar = [](const unsigned long long& b) { return tc::shared_address(&b); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::barrier_init(bar(full[i]), 1);
      tc::barrier_init(bar(spent[i]), 1);
      tc::barrier_init(bar(dz_ready[i]), 256);
    }
    tc::barrier_init(bar(w_full), 1);
    tc::barrier_init(bar(z_done), 1);
    tc::barrier_init(bar(dx_done), 1);
    tc::barrier_init(bar(dx_read), 256);
    tc::barrier_init(bar(all_done), 1);
    tc::barrier_init_fence();
  }
  if (warp == 0) tc::tmem_alloc(tc::shared_address(&tmem_base), p.tmem_columns);
  for (int i = threadIdx.x; i < p.n32; i += kNarrowThreads)
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(bias_at + i * 4),
                 "f"(p.bias && i < p.n ? to_float(static_cast<const T*>(p.bias)[i]) : 0.0f)
                 : "memory");
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tc::uniform(tmem_base);
  const uint32_t z_tmem = tmem, dx_tmem = z_tmem + p.n32, w_tmem = dx_tmem + p.k32;
  const uint32_t count = (p.tiles - blockIdx.x + gridDim.x - 1) / gridDim.x;  // of this block
  bool ok = true;

  if (warp == 9) {
    // ---- copies
    if (lane == 0) {
      tc::barrier_expect(bar(w_full), blocks64(p.k) * w_block);
      for (int c = 0; c * 64 < p.k; ++c)
        tc::copy_in(w_at + c * w_block, &p.w_map, c * 64, 0, bar(w_full));
      uint32_t i = 0;
      for (; i < count; ++i) {
        const uint32_t b = i & 1;
        if (i >= 2 && !(ok = tc::barrier_wait(bar(spent[b]), ((i >> 1) - 1) & 1))) break;
        const int row = static_cast<int>((blockIdx.x + i * gridDim.x) * kTileRows);
        tc::barrier_expect(bar(full[b]), x_bytes + z_bytes);
        for (int c = 0; c * 64 < p.k; ++c)
          tc::copy_in(x_at + b * x_bytes + c * kAPlane, &p.x_map, c * 64, row, bar(full[b]));
        for (int c = 0; c * 64 < p.n; ++c)
          tc::copy_in(z_at + b * z_bytes + c * kAPlane, &p.dy_map, c * 64, row, bar(full[b]));
      }
      // no copy is in flight past this point, also after a wait that ran out
      ok = tc::barrier_wait(bar(w_full), 0) && ok;
      for (uint32_t j = i < 2 ? 0 : i - 2; j < i; ++j)
        ok = tc::barrier_wait(bar(full[j & 1]), (j >> 1) & 1) && ok;
    }
  } else if (warp == 8) {
    // ---- products
    {
      const uint32_t lead = tc::elected();
      const uint32_t z_instruction = tc::instruction(!kIsF16<T>, false, false, p.n32);
      const uint32_t dx_instruction = tc::instruction(!kIsF16<T>, false, true, p.k32);
      const uint32_t w_instruction = tc::instruction(!kIsF16<T>, true, true, p.k32);
      // n of up to 64 leave lanes 64 and up to the second values (or, without them,
      // to the first ones again, which are not read)
      const uint32_t beside = p.n <= 64 && with_second;
      const auto form_z = [&](uint32_t i) {
        const uint32_t b = i & 1;
        if (!(ok = tc::barrier_wait(bar(full[b]), (i >> 1) & 1) && ok)) return;
        tc::fence_after_sync();
        if (!with_z) return;
        for (int c = 0; c * 64 < p.k; ++c)
          tc::mma_steps(lead, z_tmem, tc::descriptor_k_major(x_at + b * x_bytes + c * kAPlane),
                        tc::descriptor_k_major(w_at + c * w_block), tc::kStepK, tc::kStepK,
                        min((p.k - c * 64 + 15) / 16, 4), z_instruction, c > 0);
        tc::commit(lead, bar(z_done));
      };
      ok = tc::barrier_wait(bar(w_full), 0);
      if (ok) form_z(0);
      for (uint32_t i = 0; i < count && ok; ++i) {
        const uint32_t b = i & 1;
        if (!(ok = tc::barrier_wait(bar(dz_ready[b]), (i >> 1) & 1))) break;
        tc::fence_after_sync();
        if (i + 1 < count) form_z(i + 1);
        const uint32_t x_now = x_at + b * x_bytes, z_now = z_at + b * z_bytes;
        if (p.partial) {
          const uint32_t z_block = p.n > 64 ? kAPlane : beside ? second_at - z_now : 0;
          tc::mma_steps(lead, w_tmem, tc::descriptor_mn_major(z_now, z_block),
                        tc::descriptor_mn_major(x_now, kAPlane), tc::kStepMn, tc::kStepMn,
                        kTileRows / 16, w_instruction, i > 0);
          if (with_second && !beside)
            tc::mma_steps(lead, w_tmem, tc::descriptor_mn_major(second_at, kAPlane),
                          tc::descriptor_mn_major(x_now, kAPlane), tc::kStepMn, tc::kStepMn,
                          kTileRows / 16, w_instruction, true);
        }
        if (p.with_dx) {
          if (i > 0 && !(ok = tc::barrier_wait(bar(dx_read), (i - 1) & 1) && ok)) break;
          tc::fence_after_sync();
          for (int part = 0; part <= (with_second ? 1 : 0); ++part)
            for (int c = 0; c * 64 < p.n; ++c)
              tc::mma_steps(lead, dx_tmem,
                            tc::descriptor_k_major((part ? second_at : z_now) + c * kAPlane),
                            tc::descriptor_mn_major(w_at + c * 4 * tc::kStepMn, w_block),
                            tc::kStepK, tc::kStepMn, min((p.n - c * 64 + 15) / 16, 4),
                            dx_instruction, part > 0 || c > 0);
        }
        tc::commit(lead, bar(dx_done));
        tc::commit(lead, bar(spent[b]));
      }
      // whichever way the loop ended, no product is in flight past this point
      tc::commit(lead, bar(all_done));
      ok = tc::barrier_wait(bar(all_done), 0) && ok;
    }
  } else {
    // ---- dz and dx
    const int lane_block = warp & 3, half = warp >> 2;
    const int row = lane_block * 32 + lane;
    const uint32_t turn = row & 7;
    const bool leader = lane == 0;
    const Patch<T> patch{patch_at + warp * 2048};
    f32x2 sum_b[C][16];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum_b[c][j] = pack2(0.0f, 0.0f);

    const auto form_dz = [&](auto act, uint32_t z_row, uint32_t i_tile) {
      constexpr int ACT = decltype(act)::value;
#pragma unroll
      for (int cc = 0; cc < C; ++cc) {
        const int c = half + 2 * cc;
        if (c * 32 >= p.n32) break;
        float v[32];
        if constexpr (ACT != kNone) {
          tc::tmem_load32(z_tmem + (lane_block << 21) + c * 32, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 b = load_shared(bias_at + (c * 32 + j * 4) * 4);
            unpack2(add2(pack2(v[4 * j], v[4 * j + 1]), pack2(b.x, b.y)), v[4 * j], v[4 * j + 1]);
            unpack2(add2(pack2(v[4 * j + 2], v[4 * j + 3]), pack2(b.z, b.w)), v[4 * j + 2],
                    v[4 * j + 3]);
          }
        }
        const uint32_t at = z_row + (c >> 1) * kAPlane;
        const uint32_t to_second = second_at - (z_at + (i_tile & 1) * z_bytes);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t piece = at + ((((c & 1) * 4 + j) ^ turn) << 4);
          const float4 raw = load_shared(piece);
          float e[8];
          widen<T, 8>(reinterpret_cast<const Vec<T, 8>&>(raw), e);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            f32x2 dz = pack2(e[i], e[i + 1]);
            if constexpr (ACT != kNone) {
              slope2<ACT, false>(v[j * 8 + i], v[j * 8 + i + 1]);
              dz = mul2(dz, pack2(v[j * 8 + i], v[j * 8 + i + 1]));
            }
            f32x2& sum = sum_b[cc][j * 4 + i / 2];
            sum = add2(sum, dz);
            if constexpr (ACT != kNone) unpack2(dz, v[j * 8 + i], v[j * 8 + i + 1]);
          }
        }
        if constexpr (ACT == kRelu) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = v[j * 8 + i];
            const Vec<T, 8> r = round_values<T, 8>(e);
            store_shared(at + ((((c & 1) * 4 + j) ^ turn) << 4), reinterpret_cast<const uint4&>(r));
          }
        }
        if constexpr (rounds_dz(ACT)) {
          // the products of the tile before have read its second values
          if (cc == 0 && i_tile > 0 &&
              !(ok = tc::barrier_wait(bar(dx_done), (i_tile - 1) & 1)))
            return;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t piece = at + ((((c & 1) * 4 + j) ^ turn) << 4);
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = v[j * 8 + i];
            const Vec<T, 8> first = take_first<T, 8>(e);
            store_shared(piece, reinterpret_cast<const uint4&>(first));
            const Vec<T, 8> second = round_values<T, 8>(e);
            store_shared(piece + to_second, reinterpret_cast<const uint4&>(second));
          }
        }
      }
    };
    const auto store_dx = [&](uint32_t i) {
      if (!(ok = tc::barrier_wait(bar(dx_done), i & 1))) return;
      tc::fence_after_sync();
      const long long row0 =
          static_cast<long long>(blockIdx.x + i * gridDim.x) * kTileRows + lane_block * 32;
      for (int c = half; c < 2 * C; c += 2) {
        const bool in = c * 32 < p.k32, last = c + 2 >= 2 * C;
        float v[32];
        if (in) tc::tmem_load32(dx_tmem + (lane_block << 21) + c * 32, v);
        if (last) {
          tc::fence_before_sync();
          tc::barrier_arrive(bar(dx_read));
        }
        if (!in || c * 32 >= p.k || row0 >= p.rows) continue;
        if (leader) tc::copies_out_read();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float o[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) o[q] = v[j * 8 + q];
          const Vec<T, 8> r = round_values<T, 8>(o);
          store_shared(patch.at(lane, j), reinterpret_cast<const uint4&>(r));
        }
        tc::fence_async_proxy();
        __syncwarp();
        if (leader) tc::copy_out(&p.dx_map, c * 32, static_cast<int>(row0), patch.base);
      }
    };

    for (uint32_t i = 0; i < count && ok; ++i) {
      const uint32_t b = i & 1;
      if (!(ok = tc::barrier_wait(bar(full[b]), (i >> 1) & 1))) break;
      if (with_z && !(ok = tc::barrier_wait(bar(z_done), i & 1))) break;
      tc::fence_after_sync();
      const uint32_t z_row = z_at + b * z_bytes + row * 128;
      switch (p.activation) {
        case kRelu: form_dz(std::integral_constant<int, kRelu>{}, z_row, i); break;
        case kSilu: form_dz(std::integral_constant<int, kSilu>{}, z_row, i); break;
        case kGelu: form_dz(std::integral_constant<int, kGelu>{}, z_row, i); break;
        case kSigmoid: form_dz(std::integral_constant<int, kSigmoid>{}, z_row, i); break;
        default: form_dz(std::integral_constant<int, kNone>{}, z_row, i);
      }
      if (!ok) break;
      tc::fence_async_proxy();
      tc::fence_before_sync();
      tc::barrier_arrive(bar(dz_ready[b]));
      if (p.with_dx && i > 0) store_dx(i - 1);
    }
    if (ok && p.with_dx) store_dx(count - 1);
    if (leader) tc::copies_out_read();

    // this block's sums
    if (p.partial) {
      ok = tc::barrier_wait(bar(all_done), 0) && ok;
      tc::fence_after_sync();
      float* out = p.partial + static_cast<size_t>(blockIdx.x) * p.n * (p.k + 1);
      // dW of the second values in lanes 64 and up goes by way of x's buffers
      const bool beside = with_second && p.n <= 64;
      const uint32_t half_at = x_at + (row & 63) * 4;
      const auto each_chunk = [&](auto use) {
#pragma unroll
        for (int cc = 0; cc < C; ++cc) {
          const int c = half + 2 * cc;
          if (c * 32 >= p.k32) break;
          float v[32];
          tc::tmem_load32(w_tmem + (lane_block << 21) + c * 32, v);
          use(c, v);
        }
      };
      const bool upper = beside && lane_block >= 2;
      if (upper)
        each_chunk([&](int c, const float (&v)[32]) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(half_at + (c * 32 + j) * 256), "f"(v[j])
                         : "memory");
        });
      if (beside) asm volatile("bar.sync 1, 256;" ::: "memory");
      if (!upper && lane_block * 32 < p.n)
        each_chunk([&](int c, float (&v)[32]) {
          if (beside) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              float second;
              asm volatile("ld.shared.f32 %0, [%1];"
                           : "=f"(second)
                           : "r"(half_at + (c * 32 + j) * 256)
                           : "memory");
              v[j] += second;
            }
          }
          if (row < p.n) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c * 32 + j < p.k) out[row * p.k + c * 32 + j] = v[j];
          }
        });
#pragma unroll
      for (int cc = 0; cc < C; ++cc) {
        const int c = half + 2 * cc;
        if (c * 32 >= p.n32) break;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float s[2];
          unpack2(sum_b[cc][j], s[0], s[1]);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int o = 16; o; o >>= 1) s[q] += __shfl_xor_sync(0xffffffffu, s[q], o);
            if (leader)
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(
                               join_at + (lane_block * kNarrowWidth + c * 32 + j * 2 + q) * 4),
                           "f"(s[q])
                           : "memory");
          }
        }
      }
    }
  }
  if (!ok) atomicCAS(p.error, 0, kDeviceTimeout);
  tc::fence_before_sync();
  __syncthreads();
  if (p.partial && threadIdx.x < p.n) {
    float s = 0.0f;
    for (int q = 0; q < 4; ++q) {
      float v;
      asm volatile("ld.shared.f32 %0, [%1];"
                   : "=f"(v)
                   : "r"(join_at + (q * kNarrowWidth + threadIdx.x) * 4)
                   : "memory");
      s += v;
    }
    p.partial[static_cast<size_t>(blockIdx.x) * p.n * (p.k + 1) + p.n * p.k + threadIdx.x] = s;
  }
  if (warp == 0) tc::tmem_free(tmem, p.tmem_columns);
}

}  // namespace feature
}  // namespace splat
