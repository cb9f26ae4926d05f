// Inline-PTX wrappers for the Blackwell (sm_100a) units the Flash-MVPA kernels use:
// mbarrier, TMA (cp.async.bulk.tensor, no cluster multicast anywhere), tcgen05 MMA with
// TMEM accumulators, tcgen05.ld/st, and the shared-memory / instruction descriptors.
//
// Every wait is bounded in time: once a deadline on the %globaltimer clock has passed it records a
// code in a status word and returns false, so a protocol bug surfaces as an error status instead
// of a hung GPU.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

namespace mvpa {
namespace ptx {

constexpr uint64_t kDefaultWaitNs = 2000000000ull;  // a wait gives up after two seconds
constexpr uint32_t kPollsPerClockRead = 32;         // try_wait polls between two looks at the clock
// Per translation unit: a non-zero value (microseconds) replaces the default deadline.  Only the wait
// self-test sets it (to make a wait run out quickly); product kernels run with the default.
static __device__ unsigned int g_wait_limit_us = 0;

__device__ __forceinline__ uint64_t global_timer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ uint64_t wait_limit_ns() {
  const unsigned int us = *(volatile unsigned int*)&g_wait_limit_us;
  return us != 0 ? (uint64_t)us * 1000ull : kDefaultWaitNs;
}
__device__ __forceinline__ void record_giveup(int* status, int code) {
  if (status != nullptr) {
    atomicCAS(status, 0, code);
    status[(code % 100) & 63] = code;  // every wait that gave up, for diagnosis (the first word keeps the first)
  }
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ------------------------------- mbarrier -----------------------------------
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_fence_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait.  On time-out stores `code` to *status (first writer wins) and returns false.
// A phase that has already completed is caught by the non-suspending test first; the clock is
// only consulted once a first batch of polls has failed, so a short wait never reads it.
// (The polls are loops, not unrolled: a kernel has some thirty waits, and unrolled they were a third to a half of its
// instructions - tc_fwd_kernel<128, 128> 139 KB against 100, tc_bwd_kv_kernel<128, 128> 105 against 59 - which the caches
// in front of the scheduler do not hold.)
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  if (mbar_test_wait(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < kPollsPerClockRead; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
  }
  const uint64_t t0 = global_timer_ns(), limit = wait_limit_ns();
  do {
#pragma unroll 1
    for (uint32_t i = 0; i < kPollsPerClockRead; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
    }
  } while (global_timer_ns() - t0 < limit);
  record_giveup(status, code);
  return false;
}

// Variants on a shared-space address (the MMA-issuing warp keeps barrier addresses as integers
// so that no generic-to-shared conversion sits in its instruction stream).
__device__ __forceinline__ bool mbar_test_wait_a(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_try_wait_a(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_a(uint32_t bar, uint32_t parity, int* status, int code) {
  if (mbar_test_wait_a(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < kPollsPerClockRead; ++i) {
    if (mbar_try_wait_a(bar, parity)) return true;
  }
  const uint64_t t0 = global_timer_ns(), limit = wait_limit_ns();
  do {
#pragma unroll 1
    for (uint32_t i = 0; i < kPollsPerClockRead; ++i) {
      if (mbar_try_wait_a(bar, parity)) return true;
    }
  } while (global_timer_ns() - t0 < limit);
  record_giveup(status, code);
  return false;
}
// --------------------------------- TMA --------------------------------------
__device__ __forceinline__ void prefetch_tensormap(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}
// 2-D and 3-D tiled loads (x = innermost).  x must keep the 16-byte rule: x * sizeof(elem) % 16 == 0.
__device__ __forceinline__ void tma_load_2d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x,
                                            int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x,
                                            int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x,
                                            int y, int z, int w, int v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5, %6, %7}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* m, uint32_t smem_src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(m)),
               "r"(smem_src), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, const void* smem_src, int x, int y,
                                             int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
// 5-D tiled store; elements outside the tensor are not written.  Coordinates must not be negative.
__device__ __forceinline__ void tma_store_5d(const CUtensorMap* m, const void* smem_src, int x, int y,
                                             int z, int w, int v) {
  asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {  // all but the last N groups have been read from shared memory
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tma_store_wait_all() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// Generic-proxy writes to shared memory -> visible to the async proxy (TMA store, tcgen05.mma).
__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ------------------------------- tcgen05 ------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* smem_result, uint32_t ncols) {  // one full warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)),
               "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {  // one full warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// TMEM -> registers: each thread of a warp reads its own lane (row), N consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, "
      "%34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, "
      "%54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld1(uint32_t taddr, uint32_t& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st1(uint32_t taddr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ------------------------------ descriptors ---------------------------------
// Shared-memory matrix descriptor, 128-byte swizzle, sm_100 version field = 1.
//   bits [0,14)  start address >> 4      bits [16,30) leading byte offset >> 4
//   bits [32,46) stride byte offset >> 4 bits [46,48) version = 1     bits [61,64) layout = 2 (SW128)
// K-major operand  (rows of 64 bf16 = 128 B, 8-row groups of 1024 B): SBO = 1024, LBO unused (1).
// MN-major operand (MN contiguous, 64 per 128-B row; one row per K index): SBO = 1024 between
//   groups of 8 K-rows, LBO = byte distance between 64-wide MN chunks.
__device__ __forceinline__ uint64_t make_desc_sw128(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFF);
  d |= (uint64_t)((lbo_bytes >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((sbo_bytes >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// The same descriptor split into 32-bit halves: the low word carries the start address (and LBO),
// so stepping through a tile is one 32-bit add per MMA instead of rebuilding 64 bits.
struct DescHalves {
  uint32_t lo, hi;
};
__device__ __forceinline__ DescHalves make_desc_halves_sw128(uint32_t smem_addr, uint32_t lbo_bytes,
                                                             uint32_t sbo_bytes) {
  DescHalves d;
  d.lo = ((smem_addr >> 4) & 0x3FFF) | (((lbo_bytes >> 4) & 0x3FFF) << 16);
  d.hi = ((sbo_bytes >> 4) & 0x3FFF) | (1u << 14) | (2u << 29);
  return d;
}
// ---------------------- warp-convergent issue (elected lane) ----------------------
// The tcgen05 instructions take their descriptors and addresses from warp-uniform registers.  Issued
// from a branch only one lane enters, each MMA costs that lane 80-160 cycles (more when the other warps
// of the SM are busy); issued by the whole warp in convergent code, with only the instruction itself
// guarded by the elected lane's predicate, the same stream runs at the tensor pipe's own rate (64 cycles
// for M128 N128 K16).  These variants take that predicate (`el`, 1 on the elected lane, 0 elsewhere);
// every lane of the warp must call them together with identical arguments.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred;
}
__device__ __forceinline__ void mma_commit_w(uint32_t el, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred pe;\n\tsetp.ne.b32 pe, %1, 0;\n\t"
      "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(el)
      : "memory");
}
__device__ __forceinline__ void mma_ss_w(uint32_t el, uint32_t d_tmem, DescHalves a, uint32_t a_off_bytes,
                                         DescHalves b, uint32_t b_off_bytes, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, pe;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 pe, %7, 0;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem),
      "r"(a.lo + (a_off_bytes >> 4)), "r"(a.hi), "r"(b.lo + (b_off_bytes >> 4)), "r"(b.hi), "r"(idesc),
      "r"(accumulate), "r"(el)
      : "memory");
}
// Four consecutive K-steps of 32 bytes, D[tmem] = A[smem] * B[smem] for 8-bit operands, K-major in 128-byte rows; the first
// step overwrites D.
__device__ __forceinline__ void mma_f8_ss_x4_w(uint32_t el, uint32_t d_tmem, DescHalves a, DescHalves b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p0, p1, pe;\n\t.reg .b64 da, db;\n\t.reg .b32 la, lb;\n\t"
      "setp.ne.b32 p0, 0, 0;\n\t"
      "setp.eq.b32 p1, 0, 0;\n\t"
      "setp.ne.b32 pe, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t mov.b64 db, {%3, %4};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p0;\n\t"
      "add.u32 la, %1, 2;\n\t add.u32 lb, %3, 2;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p1;\n\t"
      "add.u32 la, %1, 4;\n\t add.u32 lb, %3, 4;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p1;\n\t"
      "add.u32 la, %1, 6;\n\t add.u32 lb, %3, 6;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p1;\n\t}" ::"r"(d_tmem),
      "r"(a.lo), "r"(a.hi), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"(el)
      : "memory");
}
// ---- pairs: one product over two CTAs of a cluster (cta_group::2: ranks 2 i and 2 i + 1), issued by the first ----
// M = 256: each CTA stages its 128 rows of A and its half of B's rows, and holds its 128 rows of D in its own TMEM.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_map(uint32_t smem_addr, uint32_t rank) {  // the same place in another CTA
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// (`bar` from cluster_map.  Release at the scope of the CTA, as in mbar_arrive: what such an arrival orders is TMEM, by
// tc_fence_before, or shared memory that the tensor cores of this very CTA read next, by fence_proxy_async_smem.  At the scope of
// the cluster it is a fence that waits for every load and store of the thread: the 8-bit product, whose warps arrive once a block
// with the next blocks' scales still on their way, took 1.6 times as long.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_result, uint32_t ncols) {  // one full warp of each CTA
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// A load into this CTA's shared memory that counts at a barrier of either CTA of the pair (`bar` from cluster_map), issued by the
// elected lane of a convergent warp.
__device__ __forceinline__ void tma_load_2d_pair_w(uint32_t el, uint32_t smem_dst, const CUtensorMap* m, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n\t.reg .pred pe;\n\tsetp.ne.b32 pe, %5, 0;\n\t"
      "@pe cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(
          smem_dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(el)
      : "memory");
}
// The barrier of this place in each CTA of the cluster whose bit is set.
__device__ __forceinline__ void mma_commit_pair_w(uint32_t el, uint16_t ctas, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred pe;\n\tsetp.ne.b32 pe, %1, 0;\n\t"
      "@pe tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(bar),
      "r"(el), "h"(ctas)
      : "memory");
}
__device__ __forceinline__ void mma_f8_ss_x4_pair_w(uint32_t el, uint32_t d_tmem, DescHalves a, DescHalves b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p0, p1, pe;\n\t.reg .b64 da, db;\n\t.reg .b32 la, lb;\n\t"
      "setp.ne.b32 p0, 0, 0;\n\t"
      "setp.eq.b32 p1, 0, 0;\n\t"
      "setp.ne.b32 pe, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t mov.b64 db, {%3, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p0;\n\t"
      "add.u32 la, %1, 2;\n\t add.u32 lb, %3, 2;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p1;\n\t"
      "add.u32 la, %1, 4;\n\t add.u32 lb, %3, 4;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p1;\n\t"
      "add.u32 la, %1, 6;\n\t add.u32 lb, %3, 6;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p1;\n\t}" ::"r"(d_tmem),
      "r"(a.lo), "r"(a.hi), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"(el)
      : "memory");
}
// ---- the same with a scale (e8m0) for each row's 32 neighbours along K, read from TMEM (kind::mxf8f6f4) ----
// A matrix of up to 128 rows has its scales in four columns of TMEM: row r in lane r % 32 of column r / 32, in the byte of the
// word that the instruction descriptor names (A's in bits [29,31), B's in [4,6)), in each quarter of the lanes.  Shared memory
// holds them as 32 lines of four words; the copy below spreads them over the quarters, in both CTAs from their own shared memory.
__device__ __forceinline__ void tmem_copy_scales_pair_w(uint32_t el, uint32_t d_tmem, uint32_t smem_addr) {
  const uint32_t lo = ((smem_addr >> 4) & 0x3FFF) | (1u << 16), hi = (128u >> 4) | (1u << 14);  // 8 lines 128 bytes apart, no swizzle
  asm volatile(
      "{\n\t.reg .pred pe;\n\t.reg .b64 d;\n\tsetp.ne.b32 pe, %3, 0;\n\tmov.b64 d, {%1, %2};\n\t"
      "@pe tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(d_tmem),
      "r"(lo), "r"(hi), "r"(el)
      : "memory");
}
// Four consecutive K-steps; the first one overwrites D if `accumulate` is 0.
__device__ __forceinline__ void mma_mxf8_ss_x4_pair_w(uint32_t el, uint32_t d_tmem, DescHalves a, DescHalves b, uint32_t idesc,
                                                      uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p0, p1, pe;\n\t.reg .b64 da, db;\n\t.reg .b32 la, lb;\n\t"
      "setp.ne.b32 p0, %9, 0;\n\t"
      "setp.eq.b32 p1, 0, 0;\n\t"
      "setp.ne.b32 pe, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t mov.b64 db, {%3, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %5, [%7], [%8], p0;\n\t"
      "add.u32 la, %1, 2;\n\t add.u32 lb, %3, 2;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %5, [%7], [%8], p1;\n\t"
      "add.u32 la, %1, 4;\n\t add.u32 lb, %3, 4;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %5, [%7], [%8], p1;\n\t"
      "add.u32 la, %1, 6;\n\t add.u32 lb, %3, 6;\n\t mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t"
      "@pe tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %5, [%7], [%8], p1;\n\t}" ::"r"(d_tmem),
      "r"(a.lo), "r"(a.hi), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"(el), "r"(scale_a), "r"(scale_b), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts_w(uint32_t el, uint32_t d_tmem, uint32_t a_tmem, DescHalves b,
                                         uint32_t b_off_bytes, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, pe;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.ne.b32 pe, %6, 0;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b.lo + (b_off_bytes >> 4)), "r"(b.hi), "r"(idesc), "r"(accumulate), "r"(el)
      : "memory");
}
// Four consecutive K-steps of  D[tmem] (+)= A[tmem] * B[smem]  (A: 16 keys = 8 packed columns per
// step; B: MN-major, `b_step16` 16-byte descriptor units per step from low word `b_lo`).
__device__ __forceinline__ void mma_ts_x4_w(uint32_t el, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo,
                                            uint32_t b_hi, uint32_t b_step16, uint32_t idesc,
                                            uint32_t accumulate_first) {
  asm volatile(
      "{\n\t.reg .pred p0, p1, pe;\n\t.reg .b64 db;\n\t.reg .b32 lo;\n\t"
      "setp.ne.b32 p0, %6, 0;\n\t"
      "setp.ne.b32 pe, %7, 0;\n\t"
      "setp.eq.b32 p1, 0, 0;\n\t"
      "mov.b32 lo, %2;\n\t"
      "mov.b64 db, {lo, %3};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %5, p0;\n\t"
      "add.u32 lo, lo, %4;\n\t mov.b64 db, {lo, %3};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1 + 8], db, %5, p1;\n\t"
      "add.u32 lo, lo, %4;\n\t mov.b64 db, {lo, %3};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1 + 16], db, %5, p1;\n\t"
      "add.u32 lo, lo, %4;\n\t mov.b64 db, {lo, %3};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1 + 24], db, %5, p1;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(b_step16), "r"(idesc), "r"(accumulate_first), "r"(el)
      : "memory");
}

// Instruction descriptor for kind::f16 with bf16 A/B and fp32 accumulation.
//   [4,6) D fmt = 1 (f32)  [7,10) A fmt = 1 (bf16)  [10,13) B fmt = 1 (bf16)
//   [15] A major (0 = K)   [16] B major (0 = K, 1 = MN)   [17,23) N >> 3   [24,29) M >> 4
__host__ __device__ constexpr uint32_t make_idesc_bf16(int M, int N, int b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// Instruction descriptor for kind::f8f6f4 with e4m3 A/B (format 0), K-major, and fp32 accumulation.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Instruction descriptor for kind::mxf8f6f4: e4m3 A/B, K-major, e8m0 scales (bit 23), M >> 7 in [27,29); accumulation is always fp32.
__host__ __device__ constexpr uint32_t make_idesc_e4m3_scaled(int M, int N) {
  return ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27);
}

// make_idesc_bf16 with both operand majors selectable (bit 15: A is MN-major, bit 16: B is MN-major).
__host__ __device__ constexpr uint32_t make_idesc_bf16_ab(int M, int N, int a_mn_major, int b_mn_major) {
  return make_idesc_bf16(M, N, b_mn_major) | ((uint32_t)a_mn_major << 15);
}

// Byte offset of element (row, col) of a [rows x 64] bf16 tile stored with the 128-byte swizzle
// TMA and tcgen05 agree on: 16-byte chunk index XOR (row mod 8).  Tile base must be 1024-aligned.
__device__ __forceinline__ uint32_t sw128_offset(int row, int col) {
  const int chunk = (col >> 3) ^ (row & 7);
  return (uint32_t)(row * 128 + chunk * 16 + (col & 7) * 2);
}

// Programmatic dependent launch: let the next kernel's CTAs start / wait until the previous grid has completed and
// its writes are visible (returns at once in a kernel launched without the attribute).
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// packed fp32 arithmetic: two elements per instruction, each rounded like the scalar operation
__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

}  // namespace ptx
}  // namespace mvpa
