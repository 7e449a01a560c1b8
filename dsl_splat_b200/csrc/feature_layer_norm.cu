// Layer norm over the last dimension of channel-last rows, with an activation:
//
//   h = (x - mean) rstd,  u = h w + b,  y = act(u)
//   du = dy act'(u),  d = du w
//   dx = rstd (d - mean(d) - h mean(d h)),  dw = sum du h,  db = sum du over rows
//
// Rows of up to 1024 channels are staged: bulk copies bring tiles of whole rows into each
// warp's ring in shared memory, a group of lanes holds a row in registers and puts the
// results in its place, and bulk copies take them out.  So any channel count moves in
// contiguous 16-byte pieces, and enough of them are in flight however few registers are left.
// Longer rows stay in a block's registers (up to 8192) or are read again from the caches.  The
// mean is taken twice: the second time of the deviations from the first, whose squares give the
// variance without a subtraction of like numbers.  The backward takes both again from x,
// which it has to read: two floats kept per row would cost a row of 32 16-bit channels an
// eighth of its bytes each way.  A thread meets the same channels in all of its rows and adds
// their du and du h in registers; blocks' sums are joined in a fixed order.
//
// Bound by memory, and where rows have an activation by the issue of the arithmetic: 1920000 x
// 64 bf16 SiLU 118 us (4.2 TB/s), 1000000 x 35 fp32 GELU 84 us (3.3 TB/s), its backward 117
// (3.6 TB/s), 30000 x 2000 bf16 82 us and 169.  With rows loaded into registers without the
// ring, whose loads in flight fall with the registers that are left, they took 144, 151 and 247.
#include <algorithm>
#include <type_traits>

#include "feature_common.cuh"
#include "feature_join.cuh"
#include "host_runtime.h"
#include "splat200.h"
#include "tensor_core.cuh"

namespace splat {
namespace feature {

constexpr int kNormThreads = 256;
constexpr int kMostLaneValues = 32;                              // of a row, in a thread
constexpr int kMostGroupChannels = 32 * kMostLaneValues;         // of a row, in a warp
constexpr int kMostBlockChannels = kNormThreads * kMostLaneValues;
constexpr int kMostChannels = 65535;
constexpr int kMostNormStages = 3;

struct LayerNormParams {
  long long rows;
  int channels, lanes;  // lanes of a row: a power of two, up to 32
  const void *x, *weight, *bias, *dy;
  void *y, *dx;    // y: the forward's; dx: NULL if not wanted
  float* partial;  // (blocks, 2, channels) sums of du h and du, or NULL
  float* moments;  // (3, rows) of rows longer than a block's registers
  float eps;
  int activation;
  int* error;
};

// Sums over the lanes of a row, all lanes get them.
template <bool BLOCK, int K>
SPLAT_DEV void sum_lanes(float (&v)[K], int lanes) {
  for (int o = (BLOCK ? 32 : lanes) / 2; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (BLOCK) {
    __shared__ float sums[K][kNormThreads / 32];
    __syncthreads();  // the sums before have been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) sums[k][threadIdx.x >> 5] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < kNormThreads / 32; ++i) v[k] += sums[k][i];
    }
  }
}

SPLAT_DEV float add_halves(f32x2 v) {
  float a, b;
  unpack2(v, a, b);
  return a + b;
}
// Pairs of values where there are channels, zeros elsewhere.
template <int M>
SPLAT_DEV f32x2 masked(f32x2 v, const bool (&in)[2 * M], int i) {
  float a, b;
  unpack2(v, a, b);
  return pack2(in[2 * i] ? a : 0.0f, in[2 * i + 1] ? b : 0.0f);
}

// x of a row, in pairs -> its normal form (x - mean) rstd; returns rstd.  FULL: every value
// is a channel's.
template <bool BLOCK, bool FULL, int M>
SPLAT_DEV float normalise(f32x2 (&v)[M], const bool (&in)[2 * M], int lanes, float inverse,
                          float eps) {
  f32x2 total = v[0];
#pragma unroll
  for (int i = 1; i < M; ++i) total = add2(total, v[i]);
  float sum[1] = {add_halves(total)};
  sum_lanes<BLOCK>(sum, lanes);
  const f32x2 mean = splat2(-sum[0] * inverse);
  f32x2 rests = 0, squares = 0;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    v[i] = add2(v[i], mean);
    if constexpr (!FULL) v[i] = masked<M>(v[i], in, i);
    rests = add2(rests, v[i]);
    squares = fma2(v[i], v[i], squares);
  }
  float rest[2] = {add_halves(rests), add_halves(squares)};
  sum_lanes<BLOCK>(rest, lanes);
  const float more = rest[0] * inverse;
  const float rstd = rsqrtf(fmaxf(rest[1] * inverse - more * more, 0.0f) + eps);
#pragma unroll
  for (int i = 0; i < M; ++i) v[i] = fma2(v[i], splat2(rstd), splat2(-more * rstd));
  return rstd;
}

template <int ACT, int M, bool FINE, bool SLOPE>
SPLAT_DEV void each_pair(f32x2 (&u)[M]) {
#pragma unroll
  for (int i = 0; i < M; ++i) {
    float a, b;
    unpack2(u[i], a, b);
    if constexpr (SLOPE) slope2<ACT, FINE>(a, b);
    else activate2<ACT, FINE>(a, b);
    u[i] = pack2(a, b);
  }
}
// u -> act(u), or act'(u).
template <bool FINE, bool SLOPE, int M>
SPLAT_DEV void all_pairs(int activation, f32x2 (&u)[M]) {
  switch (activation) {
    case kRelu: each_pair<kRelu, M, FINE, SLOPE>(u); break;
    case kSilu: each_pair<kSilu, M, FINE, SLOPE>(u); break;
    case kGelu: each_pair<kGelu, M, FINE, SLOPE>(u); break;
    case kSigmoid: each_pair<kSigmoid, M, FINE, SLOPE>(u); break;
    default: each_pair<kNone, M, FINE, SLOPE>(u);
  }
}

template <bool FINE, bool SLOPE>
SPLAT_DEV float one_value(int activation, float u) {
  f32x2 pair[1] = {pack2(u, 0.0f)};
  all_pairs<FINE, SLOPE>(activation, pair);
  float a, b;
  unpack2(pair[0], a, b);
  return a;
}

// A pair of channels' weights and biases, in shared memory, where they cost fewer registers
// and the lanes of all rows read the same; those of a row's lanes lie side by side.
SPLAT_DEV float4 load_float4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at));
  return v;
}
struct Affine {
  f32x2 w, b;
};
SPLAT_DEV Affine affine(uint32_t at, int i, int lanes) {
  const float4 v = load_float4(at + i * lanes * 16);
  return {pack2(v.x, v.y), pack2(v.z, v.w)};
}

// A row's x -> y, in place.
template <class T, bool BLOCK, bool FULL, int M>
SPLAT_DEV void norm_row(const LayerNormParams& p, f32x2 (&h)[M], const bool (&in)[2 * M],
                        uint32_t affine_at, int lanes, float inverse) {
  normalise<BLOCK, FULL>(h, in, lanes, inverse, p.eps);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const Affine a = affine(affine_at, i, lanes);
    h[i] = fma2(h[i], a.w, a.b);
  }
  all_pairs<sizeof(T) == 4, false>(p.activation, h);
}

// A row's x and dy -> dx in dy's place; its du h and du are added to dw and db.
template <class T, bool BLOCK, bool FULL, int M>
SPLAT_DEV void norm_row_backward(const LayerNormParams& p, f32x2 (&h)[M], f32x2 (&g)[M],
                                 const bool (&in)[2 * M], uint32_t affine_at, int lanes,
                                 float inverse, f32x2 (&dw)[M], f32x2 (&db)[M]) {
  const float rstd = normalise<BLOCK, FULL>(h, in, lanes, inverse, p.eps);
  if (p.activation != kNone) {
    f32x2 u[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const Affine a = affine(affine_at, i, lanes);
      u[i] = fma2(h[i], a.w, a.b);
    }
    all_pairs<sizeof(T) == 4, true>(p.activation, u);
#pragma unroll
    for (int i = 0; i < M; ++i) g[i] = mul2(g[i], u[i]);
  }
  f32x2 less2 = 0, along2 = 0;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    db[i] = add2(db[i], g[i]);
    dw[i] = fma2(g[i], h[i], dw[i]);
    g[i] = mul2(g[i], affine(affine_at, i, lanes).w);
    less2 = add2(less2, g[i]);
    along2 = fma2(g[i], h[i], along2);
  }
  if (!p.dx) return;
  float sums[2] = {add_halves(less2), add_halves(along2)};
  sum_lanes<BLOCK>(sums, lanes);
  // rstd (d - mean(d) - h mean(d h))
  const f32x2 less = splat2(-sums[0] * inverse * rstd), along = splat2(-sums[1] * inverse * rstd);
#pragma unroll
  for (int i = 0; i < M; ++i) g[i] = fma2(g[i], splat2(rstd), fma2(h[i], along, less));
}

// The channels of a thread: V neighbouring ones of each of N / V pieces.
template <int V, int N>
SPLAT_DEV int channel_of(int i, int lane, int lanes) {
  return (i / V * lanes + lane) * V + i % V;
}
// TIGHT: N is the least of its kind for the row (plan_norm), so that all but the last
// values are channels'.
template <int V, int N, bool TIGHT>
SPLAT_DEV void own_channels(int channels, int lane, int lanes, bool (&in)[N]) {
  constexpr int kSure = !TIGHT || N <= 8 ? 0 : N - (V > 1 ? 8 : N > 16 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < N; ++i)
    in[i] = i < kSure || channel_of<V, N>(i, lane, lanes) < channels;
}
// Lays out the block's weights and biases for affine(), which a thread calls with the place
// of the first plus lane * 16.
template <class T, int V, int N>
SPLAT_DEV void lay_out_affine(const LayerNormParams& p, int lanes, float* to) {
  for (int k = threadIdx.x; k < lanes * N; k += blockDim.x) {
    const int lane = k / N, i = k % N, c = channel_of<V, N>(i, lane, lanes);
    const bool in = c < p.channels;
    float* pair = to + (i / 2 * lanes + lane) * 4 + i % 2;
    pair[0] = in && p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0f;
    pair[2] = in && p.bias ? to_float(static_cast<const T*>(p.bias)[c]) : 0.0f;
  }
}

// A thread's values of a row, in pairs: zeros where there are none.
template <class T, int V, int N>
SPLAT_DEV void load_row(const T* row, int lane, int lanes, bool here, const bool (&in)[N],
                        f32x2 (&v)[N / 2]) {
  float f[N];
#pragma unroll
  for (int j = 0; j < N; j += V) {
    Vec<T, V> raw{};
    if (here && in[j]) raw = *reinterpret_cast<const Vec<T, V>*>(row + (j / V * lanes + lane) * V);
    widen<T, V>(raw, reinterpret_cast<float(&)[V]>(f[j]));
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) v[i] = pack2(f[2 * i], f[2 * i + 1]);
}
template <class T, int V, int N>
SPLAT_DEV void store_row(T* row, int lane, int lanes, bool here, const bool (&in)[N],
                         const f32x2 (&v)[N / 2]) {
  float f[N];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) unpack2(v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int j = 0; j < N; j += V)
    if (here && in[j])
      *reinterpret_cast<Vec<T, V>*>(row + (j / V * lanes + lane) * V) =
          round_values<T, V>(reinterpret_cast<const float(&)[V]>(f[j]));
}

// ---- rows of up to 1024 channels ----------------------------------------------------

// Each warp's ring of stages of shared memory: a tile of x (and of dy), whose results go
// out of it.  Warps do not wait for one another.
struct Staging {
  int rows, stages;  // of a tile; of a ring
  int bytes;         // of a tile, a multiple of 16
  long long tiles;
};

// What the last whole 16 bytes of a run of bytes leave -> shared memory.
SPLAT_DEV void copy_rest(uint32_t to, const void* from, int bytes) {
  for (int i = bytes & ~15; i < bytes; i += 2)
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + i),
                 "h"(*reinterpret_cast<const unsigned short*>(static_cast<const char*>(from) + i))
                 : "memory");
}

// Blocks of 256 threads that an SM holds at once.
constexpr int resident_blocks(int values, bool backward) {
  return values > 16 ? (backward ? 1 : 2) : backward ? 2 : 3;
}

template <class T, int V, int N, bool FULL, bool BACKWARD>
__global__ void __launch_bounds__(kNormThreads, resident_blocks(N, BACKWARD))
    staged_norm_kernel(const LayerNormParams p, const Staging ring) {
  extern __shared__ unsigned char dynamic[];
  __shared__ alignas(8) unsigned long long barriers[kNormThreads / 32][kMostNormStages];
  constexpr int M = N / 2;
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool leader = (threadIdx.x & 31) == 0;
  const uint32_t base = (tc::shared_address(dynamic) + 15u) & ~15u;
  const int stage_bytes = (BACKWARD ? 2 : 1) * ring.bytes;
  const uint32_t own_at = base + warp * ring.stages * stage_bytes;
  const uint32_t rings_end = base + warps * ring.stages * stage_bytes;
  unsigned char* own = dynamic + (own_at - tc::shared_address(dynamic));
  const uint32_t full = tc::shared_address(barriers[warp]);
  const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1), groups = 32 / lanes;
  const int group = (threadIdx.x & 31) / lanes, C = p.channels;
  const float inverse = 1.0f / static_cast<float>(C);
  bool in[N], ok = true;
  f32x2 dw[BACKWARD ? M : 1] = {}, db[BACKWARD ? M : 1] = {};
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* out = static_cast<T*>(BACKWARD ? p.dx : p.y);
  const long long first = static_cast<long long>(blockIdx.x) * warps + warp;
  const long long step = static_cast<long long>(gridDim.x) * warps;
  const auto rows_of = [&](long long tile) {
    return static_cast<int>(min(p.rows - tile * ring.rows, static_cast<long long>(ring.rows)));
  };
  int started = 0;  // by the leader
  const auto fetch = [&](long long tile, int stage) {
    const uint32_t bar = full + stage * 8, to = own_at + stage * stage_bytes;
    const int bytes = rows_of(tile) * C * static_cast<int>(sizeof(T)), whole = bytes & ~15;
    const long long at = tile * ring.rows * C;
    copy_rest(to, x + at, bytes);
    if constexpr (BACKWARD) copy_rest(to + ring.bytes, dy + at, bytes);
    tc::barrier_expect(bar, (BACKWARD ? 2 : 1) * whole);
    if (whole) {
      tc::bulk_in(to, x + at, whole, bar);
      if constexpr (BACKWARD) tc::bulk_in(to + ring.bytes, dy + at, whole, bar);
    }
    ++started;
  };
  if (leader) {
    for (int i = 0; i < ring.stages; ++i) tc::barrier_init(full + i * 8, 1);
    tc::barrier_init_fence();
    long long tile = first;
    for (int i = 0; i < ring.stages - 1 && tile < ring.tiles; ++i, tile += step) fetch(tile, i);
  }
  own_channels<V, N, true>(C, lane, lanes, in);
  lay_out_affine<T, V, N>(p, lanes, reinterpret_cast<float*>(
                                        dynamic + (rings_end - tc::shared_address(dynamic))));
  const uint32_t affine_at = rings_end + lane * 16;
  __syncthreads();
  int stage = 0, waited = 0;
  uint32_t parity = 0;
  for (long long tile = first; tile < ring.tiles; tile += step) {
    if (!(ok = tc::barrier_wait(full + stage * 8, parity))) break;
    ++waited;
    const int rows = rows_of(tile);
    unsigned char* at = own + stage * stage_bytes;
    for (int r0 = 0; r0 < rows; r0 += groups) {
      const int r = r0 + group;
      const bool here = r < rows;
      T* row = reinterpret_cast<T*>(at) + r * C;
      f32x2 h[M];
      load_row<T, V>(row, lane, lanes, here, in, h);
      if constexpr (BACKWARD) {
        f32x2 g[M];
        load_row<T, V>(reinterpret_cast<const T*>(at + ring.bytes) + r * C, lane, lanes, here, in,
                       g);
        norm_row_backward<T, false, FULL>(p, h, g, in, affine_at, lanes, inverse, dw, db);
        if (out) store_row<T, V>(row, lane, lanes, here, in, g);
      } else {
        norm_row<T, false, FULL>(p, h, in, affine_at, lanes, inverse);
        store_row<T, V>(row, lane, lanes, here, in, h);
      }
    }
    tc::fence_async_proxy();
    __syncwarp();
    if (leader) {
      if (out) {
        const int bytes = rows * C * static_cast<int>(sizeof(T)), whole = bytes & ~15;
        char* to = reinterpret_cast<char*>(out + tile * ring.rows * C);
        if (whole) tc::bulk_out(to, own_at + stage * stage_bytes, whole);
        for (int i = whole; i < bytes; i += 2)
          *reinterpret_cast<unsigned short*>(to + i) =
              *reinterpret_cast<const unsigned short*>(at + i);
      }
      // the stage before this one is free once its results have been read
      const long long next = tile + (ring.stages - 1) * step;
      if (next < ring.tiles) {
        if (out) tc::copies_out_read_but<1>();
        fetch(next, stage ? stage - 1 : ring.stages - 1);
      }
    }
    if (++stage == ring.stages) stage = 0, parity ^= 1;
  }
  if (leader) {
    // no copy is in flight past this point, also after a wait that ran out
    for (int i = waited; i < started; ++i) {
      ok = tc::barrier_wait(full + stage * 8, parity) && ok;
      if (++stage == ring.stages) stage = 0, parity ^= 1;
    }
    if (out) tc::copies_out_read();
  }
  if (!ok) atomicCAS(p.error, 0, kDeviceTimeout);
  if constexpr (BACKWARD) {
    if (!p.partial) return;
    __syncthreads();
    // the groups of a warp, then the warps one after another
    float* sums = reinterpret_cast<float*>(dynamic + (base - tc::shared_address(dynamic)));
    for (int o = lanes; o < 32; o *= 2)
#pragma unroll
      for (int i = 0; i < M; ++i) {
        dw[i] = add2(dw[i], __shfl_xor_sync(0xffffffffu, dw[i], o));
        db[i] = add2(db[i], __shfl_xor_sync(0xffffffffu, db[i], o));
      }
    for (int k = 0; k < warps; ++k) {
      if (warp == k && group == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (!in[i]) continue;
          const int c = channel_of<V, N>(i, lane, lanes);
          float a[2], d[2];
          unpack2(dw[i / 2], a[0], a[1]);
          unpack2(db[i / 2], d[0], d[1]);
          sums[c] = (k ? sums[c] : 0.0f) + a[i % 2];
          sums[C + c] = (k ? sums[C + c] : 0.0f) + d[i % 2];
        }
      }
      __syncthreads();
    }
    float* to = p.partial + 2LL * blockIdx.x * C;
    for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) to[c] = sums[c];
  }
}

// ---- rows of up to 8192 channels: a block each ----------------------------------------

// Of them, that an SM holds at once: a block's sums wait for all of its warps.
constexpr int resident_rows(int values, bool backward) {
  return (values <= 8 ? 6 : values <= 16 ? 4 : 2) / (backward ? 2 : 1);
}

template <class T, int V, int N, bool BACKWARD>
__global__ void __launch_bounds__(kNormThreads, resident_rows(N, BACKWARD))
    block_norm_kernel(const LayerNormParams p) {
  constexpr int M = N / 2;
  const int lane = threadIdx.x, lanes = kNormThreads, C = p.channels;
  const float inverse = 1.0f / static_cast<float>(C);
  bool in[N];
  f32x2 dw[BACKWARD ? M : 1] = {}, db[BACKWARD ? M : 1] = {};
  extern __shared__ float4 weights[];
  own_channels<V, N, false>(C, lane, lanes, in);
  lay_out_affine<T, V, N>(p, lanes, reinterpret_cast<float*>(weights));
  const uint32_t affine_at = tc::shared_address(weights) + lane * 16;
  __syncthreads();
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const long long at = row * C;
    f32x2 h[M];
    load_row<T, V>(static_cast<const T*>(p.x) + at, lane, lanes, true, in, h);
    if constexpr (BACKWARD) {
      f32x2 g[M];
      load_row<T, V>(static_cast<const T*>(p.dy) + at, lane, lanes, true, in, g);
      norm_row_backward<T, true, false>(p, h, g, in, affine_at, lanes, inverse, dw, db);
      if (p.dx) store_row<T, V>(static_cast<T*>(p.dx) + at, lane, lanes, true, in, g);
    } else {
      norm_row<T, true, false>(p, h, in, affine_at, lanes, inverse);
      store_row<T, V>(static_cast<T*>(p.y) + at, lane, lanes, true, in, h);
    }
  }
  if constexpr (BACKWARD) {
    if (!p.partial) return;
    float* to = p.partial + 2LL * blockIdx.x * C;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!in[i]) continue;
      const int c = channel_of<V, N>(i, lane, lanes);
      float a[2], d[2];
      unpack2(dw[i / 2], a[0], a[1]);
      unpack2(db[i / 2], d[0], d[1]);
      to[c] = a[i % 2];
      to[C + c] = d[i % 2];
    }
  }
}

// ---- rows longer than a block's registers -----------------------------------------

// A block to a row, which it reads again from the caches for each sum.
template <class T, bool BACKWARD>
__global__ void __launch_bounds__(kNormThreads) long_rows_kernel(const LayerNormParams p) {
  constexpr bool kFine = sizeof(T) == 4;
  const int C = p.channels;
  const float inverse = 1.0f / static_cast<float>(C);
  const T *w = static_cast<const T*>(p.weight), *b = static_cast<const T*>(p.bias);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * C;
    const T* dy = static_cast<const T*>(p.dy) + row * C;
    float sum[1] = {0.0f}, rest[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < C; c += kNormThreads) sum[0] += to_float(x[c]);
    sum_lanes<true>(sum, kNormThreads);
    const float mean = sum[0] * inverse;
    for (int c = threadIdx.x; c < C; c += kNormThreads) {
      const float d = to_float(x[c]) - mean;
      rest[0] += d;
      rest[1] += d * d;
    }
    sum_lanes<true>(rest, kNormThreads);
    const float more = rest[0] * inverse;
    const float rstd = rsqrtf(fmaxf(rest[1] * inverse - more * more, 0.0f) + p.eps);
    if (BACKWARD && threadIdx.x == 0) {
      p.moments[row] = mean;
      p.moments[p.rows + row] = more;
      p.moments[2 * p.rows + row] = rstd;
    }
    if (BACKWARD && !p.dx) continue;
    float less = 0.0f, along = 0.0f;
    // the backward's first pass adds up, its second one writes
    for (int pass = BACKWARD ? 0 : 1; pass < 2; ++pass) {
      float sums[2] = {0.0f, 0.0f};
      for (int c = threadIdx.x; c < C; c += kNormThreads) {
        const float h = (to_float(x[c]) - mean - more) * rstd, scale = w ? to_float(w[c]) : 1.0f;
        const float u = fmaf(h, scale, b ? to_float(b[c]) : 0.0f);
        if constexpr (!BACKWARD) {
          static_cast<T*>(p.y)[row * C + c] =
              from_float<T>(one_value<kFine, false>(p.activation, u));
        } else {
          const float g =
              to_float(dy[c]) * one_value<kFine, true>(p.activation, u) * scale;
          if (pass == 0) {
            sums[0] += g;
            sums[1] = fmaf(g, h, sums[1]);
          } else {
            static_cast<T*>(p.dx)[row * C + c] =
                from_float<T>(rstd * (g - fmaf(h, along, less)));
          }
        }
      }
      if (BACKWARD && pass == 0) {
        sum_lanes<true>(sums, kNormThreads);
        less = sums[0] * inverse;
        along = sums[1] * inverse;
      }
    }
  }
}

// Their sums over rows: a thread to a channel, a block to a range of rows.
template <class T>
__global__ void __launch_bounds__(kNormThreads)
    long_columns_kernel(const LayerNormParams p, long long range) {
  constexpr bool kFine = sizeof(T) == 4;
  const int C = p.channels, c = blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= C) return;
  const float w = p.weight ? to_float(static_cast<const T*>(p.weight)[c]) : 1.0f;
  const float b = p.bias ? to_float(static_cast<const T*>(p.bias)[c]) : 0.0f;
  const long long begin = blockIdx.y * range, end = min(begin + range, p.rows);
  float dw = 0.0f, db = 0.0f;
#pragma unroll 4
  for (long long row = begin; row < end; ++row) {
    const float h = (to_float(static_cast<const T*>(p.x)[row * C + c]) - p.moments[row] -
                     p.moments[p.rows + row]) *
                    p.moments[2 * p.rows + row];
    const float g = to_float(static_cast<const T*>(p.dy)[row * C + c]) *
                    one_value<kFine, true>(p.activation, fmaf(h, w, b));
    db += g;
    dw = fmaf(g, h, dw);
  }
  float* to = p.partial + 2LL * blockIdx.y * C;
  to[c] = dw;
  to[C + c] = db;
}

// ---- launching -------------------------------------------------------------------

struct LayerNormPlan {
  int blocks, lanes;  // lanes: 0: a block to a row
  bool vector;        // rows are whole 16-byte pieces
  int values;         // of a lane
  int warps;          // of a block
  Staging ring;
  size_t shared;
  bool longer;        // than a block's registers
  long long range;    // of rows, of their columns' sums
};

// Bytes of a warp's tile, that three stages for all of an SM's warps fit.
constexpr int kTileBytes = 2900, kBackwardTileBytes = 2250;

template <class T>
LayerNormPlan plan_norm(long long rows, int channels, bool backward) {
  constexpr int V = 16 / sizeof(T);
  LayerNormPlan plan{};
  const int sms = host::sm_count();
  plan.vector = channels % V == 0;
  plan.longer = channels > kMostBlockChannels;
  if (plan.longer) {
    plan.blocks = static_cast<int>(std::min<long long>(rows, 4LL * sms));
    const long long most = std::max(1LL, 4LL * sms / host::blocks_for(channels, kNormThreads));
    plan.range = (rows + most - 1) / most;
    return plan;
  }
  if (channels > kMostGroupChannels) {
    const int each = (channels + kNormThreads - 1) / kNormThreads;
    plan.values = each <= 8 ? 8 : each <= 16 ? 16 : 32;
    plan.blocks = static_cast<int>(
        std::min(rows, static_cast<long long>(resident_rows(plan.values, backward)) * sms));
    return plan;
  }
  // up to 16 values a lane, of which the last piece may be idle; more in whole warps
  plan.lanes = 1;
  while (plan.lanes < 32 && plan.lanes * 16 < channels) plan.lanes *= 2;
  const int each = (channels + plan.lanes - 1) / plan.lanes;
  plan.values = plan.vector ? (each <= 8 ? 8 : each <= 16 ? 16 : each <= 24 ? 24 : 32)
                : each <= 8 ? 8 : each <= 16 ? (each + 1) / 2 * 2 : (each + 3) / 4 * 4;
  // tiles of whole passes that start on 16 bytes: four or eight rows off them, which from some
  // 380 channels on leave room for few warps (backward of 40 million fp32 values: 1023 channels
  // 191 us, 1024 96)
  const int at_once = 32 / plan.lanes, row_bytes = channels * static_cast<int>(sizeof(T));
  int unit = at_once;
  while (unit * row_bytes % 16) unit *= 2;
  const int most =
      std::max(1, (backward ? kBackwardTileBytes : kTileBytes) / (unit * row_bytes));
  // no longer than what there is for a warp
  const long long wanted = (rows + 16LL * sms * unit - 1) / (16LL * sms * unit);
  plan.ring.rows = unit * static_cast<int>(std::min<long long>(most, wanted));
  plan.ring.bytes = (plan.ring.rows * row_bytes + 15) / 16 * 16;
  plan.ring.tiles = (rows + plan.ring.rows - 1) / plan.ring.rows;
  // three stages a warp, in half of an SM's shared memory at most
  const int stage = (backward ? 2 : 1) * plan.ring.bytes;
  plan.ring.stages = kMostNormStages;
  plan.warps = kNormThreads / 32;
  while (plan.warps > 1 && plan.warps * plan.ring.stages * stage > 100 * 1024) plan.warps /= 2;
  plan.shared = 16 + static_cast<size_t>(std::max(plan.warps * plan.ring.stages * stage,
                                                  8 * channels)) +
                8 * plan.lanes * plan.values;
  const int fit = static_cast<int>(220 * 1024 / (plan.shared + 1024));
  // no more blocks than run at once: each takes its share of the tiles
  const int resident = std::max(
      1, std::min(fit, resident_blocks(plan.values, backward) * kNormThreads / 32 / plan.warps));
  plan.blocks = static_cast<int>(std::min<long long>(
      (plan.ring.tiles + plan.warps - 1) / plan.warps, static_cast<long long>(resident) * sms));
  return plan;
}

template <class T, bool BACKWARD>
int launch_norm(const LayerNormPlan& plan, LayerNormParams& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  p.lanes = plan.lanes;
  if (plan.longer) {
    long_rows_kernel<T, BACKWARD><<<plan.blocks, kNormThreads, 0, host::counted(s)>>>(p);
    return kOk;
  }
  const bool aligned = host::aligned(p.x, 16) && host::aligned(p.y, 16) &&
                       host::aligned(p.dy, 16) && host::aligned(p.dx, 16);
  if (!plan.lanes) {
    const auto run = [&](auto values) {
      constexpr int kValues = decltype(values)::value;
      constexpr auto* wide = block_norm_kernel<T, V, kValues, BACKWARD>;
      constexpr auto* narrow = block_norm_kernel<T, 1, kValues, BACKWARD>;
      if (!host::allow_shared<wide>() || !host::allow_shared<narrow>())
        return host::check_launch("feature_layer_norm: shared memory");
      (plan.vector && aligned ? wide : narrow)<<<plan.blocks, kNormThreads,
                                                 8 * kNormThreads * kValues, host::counted(s)>>>(p);
      return static_cast<int>(kOk);
    };
    if (plan.values == 8) return run(std::integral_constant<int, 8>{});
    if (plan.values == 16) return run(std::integral_constant<int, 16>{});
    return run(std::integral_constant<int, 32>{});
  }
  if (!aligned)
    return host::fail(kInvalidArgument, "feature_layer_norm: tensors must be 16-byte aligned");
  p.error = host::device_error_word();
  if (!p.error) return kCudaError;
  const auto run = [&](auto width, auto values) {
    constexpr int kWidth = decltype(width)::value, kValues = decltype(values)::value;
    const auto launch = [&](auto full) {
      constexpr auto* kernel =
          staged_norm_kernel<T, kWidth, kValues, decltype(full)::value, BACKWARD>;
      if (!host::allow_shared<kernel>())
        return host::check_launch("feature_layer_norm: shared memory");
      kernel<<<plan.blocks, 32 * plan.warps, plan.shared, host::counted(s)>>>(p, plan.ring);
      return static_cast<int>(kOk);
    };
    if constexpr (kWidth > 1) {
      if (plan.lanes * kValues == p.channels) return launch(std::true_type{});
    }
    return launch(std::false_type{});
  };
#define SPLAT_NORM_VALUES(width, n) \
  case n: return run(std::integral_constant<int, width>{}, std::integral_constant<int, n>{})
  if (plan.vector) {
    switch (plan.values) {
      SPLAT_NORM_VALUES(V, 8);
      SPLAT_NORM_VALUES(V, 16);
      SPLAT_NORM_VALUES(V, 24);
      default: return run(std::integral_constant<int, V>{}, std::integral_constant<int, 32>{});
    }
  }
  switch (plan.values) {
    SPLAT_NORM_VALUES(1, 8);
    SPLAT_NORM_VALUES(1, 10);
    SPLAT_NORM_VALUES(1, 12);
    SPLAT_NORM_VALUES(1, 14);
    SPLAT_NORM_VALUES(1, 16);
    SPLAT_NORM_VALUES(1, 20);
    SPLAT_NORM_VALUES(1, 24);
    SPLAT_NORM_VALUES(1, 28);
    default: return run(std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
  }
#undef SPLAT_NORM_VALUES
}

int check_layer_norm(int dtype, long long rows, int channels, int activation) {
  if (dtype < 0 || dtype > 2) return host::fail(kInvalidArgument, "feature_layer_norm: dtype");
  if (activation < 0 || activation > 4)
    return host::fail(kInvalidArgument, "feature_layer_norm: activation");
  if (rows < 1 || channels < 1) return host::fail(kInvalidArgument, "feature_layer_norm: sizes");
  if (channels > kMostChannels || rows > (1LL << 40))
    return host::fail(kTooLarge, "feature_layer_norm: too many rows or channels");
  return kOk;
}

// Bytes of the long rows' moments, before the partial sums.
size_t moments_bytes(const LayerNormPlan& plan, long long rows) {
  return plan.longer ? static_cast<size_t>((3 * rows * 4 + 15) / 16 * 16) : 0;
}
int sums(const LayerNormPlan& plan, long long rows) {
  return plan.longer ? static_cast<int>((rows + plan.range - 1) / plan.range) : plan.blocks;
}

}  // namespace feature
}  // namespace splat

using namespace splat;
using namespace splat::feature;

extern "C" {

int splat_feature_layer_norm(int dtype, long long rows, int channels, const void* x,
                             const void* weight, const void* bias, float eps, int activation,
                             void* y, void* stream) {
  const int bad = check_layer_norm(dtype, rows, channels, activation);
  if (bad != kOk) return bad;
  if (!x || !y) return host::fail(kInvalidArgument, "feature_layer_norm: null pointer");
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    LayerNormParams p{};
    p.rows = rows, p.channels = channels;
    p.x = x, p.weight = weight, p.bias = bias, p.y = y;
    p.eps = eps, p.activation = activation;
    const int status = launch_norm<T, false>(plan_norm<T>(rows, channels, false), p,
                                             static_cast<cudaStream_t>(stream));
    return status != kOk ? status : host::check_launch("feature_layer_norm");
  });
}

size_t splat_feature_layer_norm_backward_workspace_bytes(int dtype, long long rows, int channels) {
  if (check_layer_norm(dtype, rows, channels, 0) != kOk) return 0;
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    const LayerNormPlan plan = plan_norm<T>(rows, channels, true);
    return moments_bytes(plan, rows) + static_cast<size_t>(sums(plan, rows)) * 2 * channels * 4;
  });
}

int splat_feature_layer_norm_backward(int dtype, long long rows, int channels, const void* x,
                                      const void* weight, const void* bias, float eps,
                                      int activation, const void* dy, void* dx, void* dweight,
                                      void* dbias, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const int bad = check_layer_norm(dtype, rows, channels, activation);
  if (bad != kOk) return bad;
  if (!x || !dy || !workspace)
    return host::fail(kInvalidArgument, "feature_layer_norm_backward: null pointer");
  if (!host::aligned(workspace, 16))
    return host::fail(kInvalidArgument,
                      "feature_layer_norm_backward: workspace not 16-byte aligned");
  if (workspace_bytes < splat_feature_layer_norm_backward_workspace_bytes(dtype, rows, channels))
    return host::fail(kWorkspaceTooSmall, "feature_layer_norm_backward: workspace");
  auto s = static_cast<cudaStream_t>(stream);
  return SPLAT_FEATURE_TYPE(dtype, [&] {
    const LayerNormPlan plan = plan_norm<T>(rows, channels, true);
    LayerNormParams p{};
    p.rows = rows, p.channels = channels;
    p.x = x, p.weight = weight, p.bias = bias, p.dy = dy, p.dx = dx;
    p.eps = eps, p.activation = activation;
    p.moments = static_cast<float*>(workspace);
    if (dweight || dbias)
      p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                           moments_bytes(plan, rows));
    const int status = launch_norm<T, true>(plan, p, s);
    if (status != kOk) return status;
    if (p.partial) {
      const int count = sums(plan, rows);
      if (plan.longer)
        long_columns_kernel<T>
            <<<dim3(host::blocks_for(channels, kNormThreads), count), kNormThreads, 0,
               host::counted(s)>>>(p, plan.range);
      join_splits<T>(p.partial, 2LL * channels, count, channels, channels, dweight, dbias, s);
    }
    return host::check_launch("feature_layer_norm_backward");
  });
}

}  // extern "C"
