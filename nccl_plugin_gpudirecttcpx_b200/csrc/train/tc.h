// The sm_100a instructions that the attention kernels are built from: barriers in shared memory
// with bounded waits, tiled TMA loads, matrix instructions with accumulators in tensor memory.
#pragma once
#include <cuda.h>

#include "common.h"

namespace tcpxb_train {

constexpr int kStatusTimeout = 3;  // TCPXB_ST_TIMEOUT

__device__ __forceinline__ uint32_t smemAddr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// A value that is the same in all lanes, told to the compiler: descriptors and addresses of matrix
// instructions are then kept where those take them from.
template <class T> __device__ __forceinline__ T uniform(T x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ bool electOne() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// ---- barriers
__device__ __forceinline__ void barInit(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barArrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barExpect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barTry(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ uint64_t nowNs() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for the phase of `parity` to end, two seconds at most.  After that `*dead` makes every wait
// of the block return at once: its loops run to their end on whatever memory they own, and the
// block reports a timeout.  Until `dead[1]` tells that the block has its tensor memory the two seconds
// do not begin: another kernel may hold that for any time, and the products do not start before.
__device__ __forceinline__ void barWaitLong(uint32_t bar, uint32_t parity, volatile int* dead) {
#pragma unroll 1
  for (int i = 0; i < 64; i++)
    if (barTry(bar, parity)) return;
  uint64_t began = nowNs();
#pragma unroll 1
  while (!barTry(bar, parity)) {
    if (*dead) return;
    if (!dead[1]) began = nowNs();
    if (nowNs() - began > 2000000000ull) {
      *dead = 1;
      return;
    }
  }
}
__device__ __forceinline__ void barWait(uint32_t bar, uint32_t parity, volatile int* dead) {
  if (barTry(bar, parity) || barTry(bar, parity)) return;
  barWaitLong(bar, parity, dead);
}

// ---- TMA: a box of 64 elements by 64 or 128 rows of [head size, tokens, heads, batch], 128-byte swizzle
__device__ __forceinline__ void tmaLoad(uint32_t dst, const CUtensorMap* map, uint32_t bar, int col, int row, int head, int batch) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(col), "r"(row), "r"(head), "r"(batch)
      : "memory");
}
// Moves registers between the block's warpgroups: out of the shares of those that load and issue.
template <int N> __device__ __forceinline__ void moreRegisters() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewerRegisters() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void fenceAsyncShared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fenceBarInit() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }

// ---- tensor memory
__device__ __forceinline__ void tmemAlloc(uint32_t dst, int cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmemFree(uint32_t at, int cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory");
}
__device__ __forceinline__ void tcBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmemWaitLoad() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmemWaitStore() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: thread i holds lane i's.
__device__ __forceinline__ void tmemLoad32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tmemStore32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmemStore16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmemLoad16(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
template <int N> __device__ __forceinline__ void tmemLoad(uint32_t at, uint32_t* r) {
  static_assert(N % 32 == 0, "columns");
#pragma unroll
  for (int k = 0; k < N; k += 32) tmemLoad32(at + k, r + k);
}
template <int N> __device__ __forceinline__ void tmemStore(uint32_t at, const uint32_t* r) {
  static_assert(N == 16 || N == 32, "columns");
  if constexpr (N == 32) tmemStore32(at, r);
  else tmemStore16(at, r);
}

// The other arrangement: 16 lanes by 8 columns, of which thread i holds columns 2 (i % 4) and the
// next, of lanes i / 4 and i / 4 + 8: r[4b .. 4b + 3] are those four of column block b.  `at` names
// the first of the 16 lanes.  N registers, 2 N columns.
template <int N> __device__ __forceinline__ void tmemLoadBlocks(uint32_t at, uint32_t* r) {
  static_assert(N == 16 || N == 32, "registers");
  if constexpr (N == 16)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
// Back in 16 bits: 16 lanes by 4 columns of two elements each; r[2b] and r[2b + 1] are thread i's
// pair of block b in lanes i / 4 and i / 4 + 8.
template <int N> __device__ __forceinline__ void tmemStoreBlocks(uint32_t at, const uint32_t* r) {
  static_assert(N == 8 || N == 16, "registers");
  if constexpr (N == 8)
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  else
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

// ---- matrix instructions: D[128 x n] (+)= A[128 x 16] B[n x 16], 32-bit sums
template <class T> struct MmaType;
template <> struct MmaType<__half> { static constexpr uint32_t code = 0; };
template <> struct MmaType<__nv_bfloat16> { static constexpr uint32_t code = 1; };

// `bRows`: B lies as [16][n] (n contiguous) instead of [n][16].
template <class T> __device__ __forceinline__ constexpr uint32_t mmaShape(int n, bool bRows) {
  return 1u << 4 | MmaType<T>::code << 7 | MmaType<T>::code << 10 | (bRows ? 1u << 16 : 0u) | uint32_t(n / 8) << 17 | 8u << 24;
}
// Operand tiles are panels of 64 elements x 128 rows (a panel of score columns has 64 rows with heads up to 64):
// a row of 128 bytes, groups of eight rows 1024 bytes apart.
constexpr uint32_t kPanelBytes = 128 * 128;
__device__ __forceinline__ uint64_t operandDesc(uint32_t addr, uint32_t panelStride) {
  return uint64_t((addr & 0x3ffff) >> 4) | uint64_t(panelStride >> 4) << 16 | uint64_t(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(shape), "r"(uint32_t(add))
      : "memory");
}
__device__ __forceinline__ void mmaFromTmem(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(shape), "r"(uint32_t(add))
      : "memory");
}
// One tile product is a run of instructions whose operands lie constants apart: only the first
// descriptors are computed, so that the issuing thread keeps ahead of the matrix units (with
// descriptors built for each instruction it needed 90 cycles for what they do in 32 to 64).
// d = A B^T over `steps` x 16 head elements, both tiles in shared memory.
template <int P> __device__ __forceinline__ void mmaTiles(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, int steps) {
  const uint64_t da = operandDesc(a, 16), db = operandDesc(b, 16);
#pragma unroll
  for (int k = 0; k < P * 4; k++) {
    const uint64_t off = (k / 4 * kPanelBytes + k % 4 * 32) >> 4;
    if (k < steps) mma(d, da + off, db + off, shape, k > 0);
  }
}
// d (+)= A B over the K rows of B, the summed index: A lies in tensor memory, two elements a
// column, in two runs of K / 4 columns that begin kHalf columns apart.
template <int K, int kHalf> __device__ __forceinline__ void mmaTmemTile(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, bool add) {
  const uint64_t db = operandDesc(b, K * 128);
#pragma unroll
  for (int k = 0; k < K / 16; k++) mmaFromTmem(d, a + k / (K / 32) * kHalf + k % (K / 32) * 8, db + k * (2048 >> 4), shape, add || k > 0);
}
// The barrier gets one arrival when all matrix instructions that this thread has issued are done.
__device__ __forceinline__ void mmaCommit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// ---- arithmetic
__device__ __forceinline__ float exp2Fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
}  // namespace tcpxb_train
