// Building blocks of the matrix kernels: tensor maps, tiled TMA loads, tcgen05 matrix
// products with their accumulators in tensor memory, and waits that always end.
//
// Tiles lie in shared memory as TMA writes them with the 128-byte swizzle: lines of 128
// bytes (64 elements of 16 bits), eight lines to a 1024-byte block.  An operand whose lines
// run along the summed index k (K-major) has a line per row; one whose lines run along its
// own index (MN-major) a line per k, and 64 of its rows in each such panel.
#pragma once
#include <cuda.h>

#include "layers.cuh"
#include "pipeline.cuh"

namespace hipress {

// ------------------------------------------------------------------ bounded waits
// A wait that ran out marks the CTA: all its other waits return at once, so that every role
// leaves its loop.  The host learns of it from the status word.
struct Guard {
  volatile uint32_t gave_up;
  uint32_t* status;
};
constexpr uint64_t kWaitNs = 2000000000ull;  // nothing remote is behind these waits

__device__ __forceinline__ bool guard_wait(uint64_t* bar, uint32_t parity, Guard& g, uint32_t code, uint64_t limit = kWaitNs) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  for (uint32_t polls = 1;; ++polls) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((polls & 63u) == 0) {
      if (g.gave_up) return false;
      const uint64_t now = global_timer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > limit) {
        g.gave_up = 1;
        record_status(g.status, HP_STATUS_TIMEOUT | code);
        return false;
      }
    }
  }
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// address of this CTA's `p` in the CTA of the given rank of the cluster
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// Arrival at a barrier of another CTA.  It orders nothing but the reads of tensor memory that a
// tcgen05 fence put in front of it; a release for the cluster made each one wait for the warp's
// stores, 1 us.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_async_shared() {   // plain stores, then TMA or the tensor cores
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(p));
  return p;
}
// a value that is the same in all threads of the warp, so that the compiler knows
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
// a whole warp waits
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Guard& g, uint32_t code) {
  return __all_sync(0xffffffffu, guard_wait(bar, parity, g, code));
}

// A warpgroup's registers a thread from here on.  The sum over the CTA's warpgroups is at most
// what the CTA was launched with.
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// ----------------------------------------------------------------------- TMA
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* m, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// the same in a pair of CTAs whose barrier is the first one's
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, const void* src, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(m), "r"(x),
               "r"(y), "r"(z), "r"(w), "r"(smem_u32(src))
               : "memory");
}
// shared -> global; outside the tensor nothing is written
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* m, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(m), "r"(x),
               "r"(y), "r"(z), "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>   // all but the last N groups have read what they store
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------- tensor memory
// By one whole warp.  The right to allocate is given up at once: while a CTA holds it, no other
// one is started on the SM.
//
// An allocation waits until there is room, and that wait has no bound.  What ends it: a CTA lets
// the kernel behind it start (dependents_may_start()) only once its own allocation is made, behind
// a barrier of the CTA.  So a CTA that holds tensor memory while it waits for the kernel in front
// waits for CTAs that all have theirs, whatever fits an SM beside one another.
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t cols) {
  if (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {   // the same warp
  if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: thread t gets lane t's
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 columns of this warp's lanes, written
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// ------------------------------------------------------------ matrix products
// 64-bit descriptor of an operand's tile at shared address `a` (128-byte swizzle).  lead and
// stride in bytes: MN-major, the distance of panels of 64 rows and of blocks of eight k;
// K-major, (unused) and the distance of blocks of eight rows.  A tile that starts n bytes further
// on has the descriptor plus n / 16.
constexpr uint32_t kNegateA = 1u << 13;   // of an instruction descriptor
__device__ __forceinline__ uint64_t mma_desc(uint32_t a, uint32_t lead, uint32_t stride) {
  return (uint64_t)((a & 0x3FFFF) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 |
         2ull << 61;
}
// The same for a tile without swizzle, K-major: blocks of 8 rows by 16 bytes; `lead` is the distance
// of blocks along k, `stride` along the rows.
__device__ __forceinline__ uint64_t mma_desc_plain(uint32_t a, uint32_t lead, uint32_t stride) {
  return (uint64_t)((a & 0x3FFFF) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46;
}
// instruction descriptor: fp32 accumulators, both operands of `type`
__host__ __device__ constexpr uint32_t mma_idesc(int m, int n, bool bf16, bool a_kmajor, bool b_kmajor) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_kmajor ? 0u : 1u << 15) | (b_kmajor ? 0u : 1u << 16) |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// Matrix products are issued by one thread of a warp, but all its threads go through the code, and
// `leader` (elect_one()) says which of them does it: in a branch of one thread the compiler cannot
// keep descriptors in uniform registers, and moving them there took 90 cycles for each product.
__host__ __device__ constexpr uint32_t mma_idesc_tf32(int m, int n) {
  return 1u << 4 | 2u << 7 | 2u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// eight k of 32-bit operands, of which the upper 19 bits count
__device__ __forceinline__ void mma_tf32(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if (CG == 1)
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
        : "memory");
}
// the same with the left operand in tensor memory, two 16-bit values to a column
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
// arrives at `bar` once the products issued so far are done (CG 2: at both CTAs' barriers)
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t leader, uint64_t* bar) {
  if (CG == 1)
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar)),
        "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.b32 q, %2, 0;\n"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3), "r"(leader)
        : "memory");
}

// ------------------------------------------------------------------- host side
// A tensor of `rank` axes (the first one dense) in boxes of 128 bytes by rows, swizzled;
// loads read zeros outside it.  False where the driver refuses it.
bool tensor_map(CUtensorMap* m, const void* base, int type, int rank, const uint64_t* sizes, const uint64_t* strides_bytes,
                const uint32_t* box);

// The word that kernels report expired waits in (one for each device, host memory that the
// device sees), or NULL; HP_ERR_TIMEOUT in *rc where an earlier kernel has.
uint32_t* layer_status(int* rc);
int layer_sms();   // of the current device

}  // namespace hipress
