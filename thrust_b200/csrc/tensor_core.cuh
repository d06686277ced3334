// The fifth-generation tensor cores: descriptors of operands in shared memory, matrix instructions into tensor memory, and the way back to registers.
#pragma once
#include "thrust_b200/bulk_copy.cuh"

namespace tb200_tc {

// One lane of a whole warp, the same one each time.  What it issues has its operands in registers that the whole warp shares, and the compiler sees that they are: a
// warp whose loop is one lane's alone (`if (lane == 0)`) took 130 cycles for each box it asked for and 120 for each matrix instruction.
__device__ __forceinline__ bool elected() {
  unsigned p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// ---------------------------------------------------------------- tensor memory, by whole warps; PAIR: by one of each of two CTAs, for both
template <bool PAIR> __device__ __forceinline__ void tmem_alloc(unsigned* where, unsigned columns) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tb200::smem_addr(where)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tb200::smem_addr(where)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <bool PAIR> __device__ __forceinline__ void tmem_free(unsigned at, unsigned columns) {
  if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}

// 32 columns of the 32 lanes that warp % 4 may read: lane l of the warp gets columns at, at + 1, ... of lane l
__device__ __forceinline__ void tmem_load(float (&v)[32], unsigned at) {
  unsigned r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// and back
__device__ __forceinline__ void tmem_store(const float (&v)[32], unsigned at) {
  unsigned r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
      "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ---------------------------------------------------------------- operands
// Operands lie in shared memory as the copy engine leaves boxes of 128-byte rows with the 128-byte swizzle: 8 rows are an atom of 1024 bytes, on a
// boundary of as much.  K-major: a row has 64 neighbouring k of one m (or n), atoms follow one another along m.  MN-major: a row has 64
// neighbouring m of one k, atoms follow one another along k, and the next 64 m are `chunk` bytes on.
constexpr unsigned long long DESCRIPTOR = 1ull << 46 | 2ull << 61;      // version, 128-byte swizzle
__device__ __forceinline__ unsigned long long operand(unsigned smem, bool mn_major, unsigned chunk) {
  return DESCRIPTOR | (unsigned long long)(1024 >> 4) << 32 | (unsigned long long)(mn_major ? chunk >> 4 : 1) << 16 | (smem & 0x3ffff) >> 4;
}
// D (F32, m x n in tensor memory) = or += A (m x 16) B (n x 16) of 16-bit elements: m = 128, n a multiple of 16 up to 256.  PAIR: m = 256, n a multiple of 32; each of
// the two CTAs has half of A's m, half of B's n and the whole of n for its half of D's m.
template <bool PAIR> __device__ __forceinline__ unsigned instruction(bool bf16, bool a_mn_major, bool b_mn_major, unsigned n) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_mn_major ? 1u << 15 : 0u) | (b_mn_major ? 1u << 16 : 0u) | (n >> 3) << 17 | ((PAIR ? 256u : 128u) >> 4) << 24;
}
template <bool PAIR> __device__ __forceinline__ void multiply(unsigned d, unsigned long long a, unsigned long long b, unsigned what, bool add) {
  if (PAIR)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(what), "r"((unsigned)add) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(what), "r"((unsigned)add) : "memory");
}
// an arrival on `bar`, PAIR: on that of both CTAs, once this thread's matrix instructions so far are done
template <bool PAIR> __device__ __forceinline__ void commit(unsigned long long* bar) {
  if (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(tb200::smem_addr(bar)), "h"((unsigned short)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tb200::smem_addr(bar)) : "memory");
}

// the same on this CTA's alone
template <bool PAIR> __device__ __forceinline__ void commit_here(unsigned long long* bar) {
  if (PAIR) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tb200::smem_addr(bar)) : "memory");
  else commit<false>(bar);
}

// ---------------------------------------------------------------- two CTAs
__device__ __forceinline__ unsigned rank_in_pair() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned first_ones(const void* p) {      // the first CTA's counterpart of something in shared memory
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tb200::smem_addr(p)));
  return r;
}
__device__ __forceinline__ void arrive_there(unsigned bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool try_wait_pair(unsigned long long* bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(tb200::smem_addr(bar)), "r"(parity), "r"(1000u) : "memory");
  return ok != 0;
}
__device__ __forceinline__ void meet_pair() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---------------------------------------------------------------- boxes by the copy engine
// into this CTA's shared memory; PAIR: counted by a barrier in that of either CTA
struct box_at { int x, y, z, w, v; };
template <bool PAIR> __device__ __forceinline__ void load_box(unsigned dst, const void* map, box_at c, unsigned bar) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(map), "r"(c.x),
                 "r"(c.y), "r"(c.z), "r"(c.w), "r"(c.v), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(map), "r"(c.x), "r"(c.y), "r"(c.z),
                 "r"(c.w), "r"(c.v), "r"(bar)
                 : "memory");
}

}  // namespace tb200_tc
