// Thin wrappers of the sm_100a instructions that the feature operators use:
// mbarriers with bounded waits, tensor memory, and tcgen05.mma on operands in
// 128-byte-swizzled shared memory.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "splat_common.cuh"

namespace splat {
namespace tc {

SPLAT_DEV uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ---- mbarriers -------------------------------------------------------------

SPLAT_DEV void barrier_init(uint32_t bar, uint32_t arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
SPLAT_DEV void barrier_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
SPLAT_DEV void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Nanoseconds after which a wait gives up, and the time that one poll may
// sleep in hardware.
constexpr unsigned long long kWaitLimit = 2000000000ull;
constexpr uint32_t kPollSleep = 100000;

SPLAT_DEV bool barrier_poll(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(kPollSleep)
      : "memory");
  return done;
}
SPLAT_DEV unsigned long long nanoseconds() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// Waits for the phase of the given parity to complete.  False when the limit
// runs out: the caller records an error and leaves.
SPLAT_DEV bool barrier_wait(uint32_t bar, uint32_t parity) {
  if (barrier_poll(bar, parity)) return true;
  const unsigned long long start = nanoseconds();
  while (!barrier_poll(bar, parity))
    if (nanoseconds() - start > kWaitLimit) return false;
  return true;
}

// One arrival, and bytes that copies will bring before the phase completes.
SPLAT_DEV void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// ---- tensor copies -----------------------------------------------------------

// A box of a row-major matrix at (column, row) of global memory, whose
// out-of-range values read as zeros, into shared memory; the barrier is told.
SPLAT_DEV void copy_in(uint32_t dst, const CUtensorMap* map, int column, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(column), "r"(row), "r"(bar)
      : "memory");
}
// The reverse; out-of-range values are not written.
SPLAT_DEV void copy_out(const CUtensorMap* map, int column, int row, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   map),
               "r"(column), "r"(row), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// fp32 values onto those of global memory.
SPLAT_DEV void add_out(const CUtensorMap* map, int column, int row, uint32_t src) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::
          "l"(map),
      "r"(column), "r"(row), "r"(src)
      : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Contiguous bytes (a multiple of 16, both addresses 16-byte aligned).
SPLAT_DEV void bulk_in(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
// Contiguous bytes, as bulk_in.
SPLAT_DEV void bulk_out(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src),
               "r"(bytes)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
SPLAT_DEV void copy_out_none() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// Until the sources of this thread's copy_outs, but for the last N of them and of
// copy_out_nones, may be written again.
template <int N>
SPLAT_DEV void copies_out_read_but() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
// Until the sources of this thread's copy_outs may be written again.
SPLAT_DEV void copies_out_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// Orders this thread's shared-memory accesses before later accesses of the
// async proxy (the tensor core's operand reads) that it hands on to.
SPLAT_DEV void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory -----------------------------------------------------------

// One whole warp; columns a power of two, at least 32.  The address lands in
// shared memory.
SPLAT_DEV void tmem_alloc(uint32_t where, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
SPLAT_DEV void tmem_free(uint32_t address, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address),
               "r"(columns));
}

SPLAT_DEV void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
SPLAT_DEV void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the calling warp's 32 lanes: thread t gets lane t's row.
SPLAT_DEV void tmem_load32(uint32_t address, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(address)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 16 columns of the same.
SPLAT_DEV void tmem_load16(uint32_t address, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(address)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// ---- matrix products ---------------------------------------------------------

// Operands lie in shared memory as blocks of rows of 128 bytes (64 16-bit
// values), the 16-byte pieces of row r permuted by piece ^ (r & 7), every
// block on a 1024-byte boundary.
//
// K-major: a row holds 64 consecutive k of one m (or n); rows follow m.
// MN-major: a row holds 64 consecutive m (or n) of one k; rows follow k, and
// the next 64 m are `block` bytes on.
SPLAT_DEV uint64_t descriptor_k_major(uint32_t address) {
  return static_cast<uint64_t>((address & 0x3FFFF) >> 4) | (1ull << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
SPLAT_DEV uint64_t descriptor_mn_major(uint32_t address, uint32_t block) {
  return static_cast<uint64_t>((address & 0x3FFFF) >> 4) |
         (static_cast<uint64_t>(block >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Bytes from one step of 16 k to the next.
constexpr uint32_t kStepK = 32, kStepMn = 2048;

// kind::f16 with fp32 accumulators, both operands bf16 or both f16, M = 128.
__host__ __device__ constexpr uint32_t instruction(bool is_bf16, bool a_mn, bool b_mn, int n) {
  return (1u << 4) | ((is_bf16 ? 1u : 0u) << 7) | ((is_bf16 ? 1u : 0u) << 10) |
         ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

// One lane of a warp, chosen by the hardware: 1 there, 0 in the others.  What
// issues products runs in the whole warp, its instructions guarded by this
// value: the operands then live in uniform registers, while in one lane's
// branch each of them is moved there for every instruction (about 100 cycles a
// product).
SPLAT_DEV uint32_t elected() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}
// A value that all lanes of the warp have, as the compiler does not know.
SPLAT_DEV uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// D (tensor memory) = A B^T, or += with accumulate; issued by the elected lane.
SPLAT_DEV void mma(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t instruction,
                   bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(accumulate)), "r"(elected)
      : "memory");
}
// A run of products over `steps` steps of 16 k: descriptors advance by da and
// db (bytes) a step.
SPLAT_DEV void mma_steps(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t da,
                         uint32_t db, int steps, uint32_t instruction, bool accumulate) {
#pragma unroll 4
  for (int s = 0; s < steps; ++s) {
    mma(elected, d, a, b, instruction, accumulate || s > 0);
    a += da >> 4;
    b += db >> 4;
  }
}
// The barrier gets one arrival when all earlier mma of this lane are done.
SPLAT_DEV void commit(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          bar),
      "r"(elected)
      : "memory");
}

// ---- pairs of blocks -----------------------------------------------------------

// A cluster of two blocks works on one product: 256 rows of A, of which each holds 128, and n
// rows of B, of which each holds half.  The block of rank 0 issues; each finds the results
// of its own rows in its tensor memory.
SPLAT_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address that this block's shared memory has in the block of the given rank.
SPLAT_DEV uint32_t address_in(uint32_t address, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
  return r;
}
// All threads of both blocks.
SPLAT_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
SPLAT_DEV void barrier_arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}
SPLAT_DEV bool barrier_poll_pair(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(kPollSleep)
      : "memory");
  return done;
}
// barrier_wait for a barrier of this block that the other one arrives at too.
SPLAT_DEV bool barrier_wait_pair(uint32_t bar, uint32_t parity) {
  if (barrier_poll_pair(bar, parity)) return true;
  const unsigned long long start = nanoseconds();
  while (!barrier_poll_pair(bar, parity))
    if (nanoseconds() - start > kWaitLimit) return false;
  return true;
}
// copy_in whose barrier may lie in the other block.
SPLAT_DEV void copy_in_pair(uint32_t dst, const CUtensorMap* map, int column, int row,
                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(column), "r"(row), "r"(bar)
      : "memory");
}
SPLAT_DEV void tmem_alloc_pair(uint32_t where, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
SPLAT_DEV void tmem_free_pair(uint32_t address, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address),
               "r"(columns));
}
__host__ __device__ constexpr uint32_t instruction_pair(bool is_bf16, bool a_mn, bool b_mn,
                                                        int n) {
  return (instruction(is_bf16, a_mn, b_mn, n) & ~(0x1fu << 24)) | ((256u >> 4) << 24);
}
SPLAT_DEV void mma_pair(uint32_t elected, uint32_t d, uint64_t a, uint64_t b,
                        uint32_t instruction, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(accumulate)), "r"(elected)
      : "memory");
}
// The barriers at this address in both blocks get an arrival when all earlier products of
// this lane are done.
SPLAT_DEV void commit_pair(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %2;\n\t}" ::"r"(bar),
      "r"(elected), "h"(static_cast<unsigned short>(3))
      : "memory");
}

}  // namespace tc
}  // namespace splat
