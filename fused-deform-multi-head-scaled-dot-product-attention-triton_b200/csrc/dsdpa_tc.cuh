// Fifth-generation tensor cores (tcgen05) and tiled TMA loads: thin wrappers over the PTX instructions,
// and the operand layouts that the attention kernels use.
//
// A tile of R rows with up to 128 16-bit elements lies in shared memory as panels of 64 elements: panel n
// holds elements 64n .. 64n+63 of all R rows, 128 bytes a row, 16-byte chunks XORed with the row's low
// three bits (the 128-byte swizzle of TMA and of the matrix descriptors).  The same tile serves as an
// operand whose contraction runs along the elements (K-major: q k^T, dout v^T) and as one whose
// contraction runs along the rows (MN-major: p v, ds k), so that nothing is transposed in memory.
#pragma once

#include <cuda.h>

#include "dsdpa_common.cuh"

namespace dsdpa {

constexpr int kPanel = 64;              // elements of a panel row: 128 bytes

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
// Box at element x of row y of (head z, batch w); x is a multiple of 64 elements, rows and elements
// outside the tensor read as zero.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(map) : "memory");
}

// ---- tensor memory -----------------------------------------------------------------------------
// 128 lanes x 512 columns of 32 bits a SM; an address has the lane in its upper half, the column below.
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, unsigned columns) {   // one whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, unsigned columns) {          // the same warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: thread l gets lane l's values.  (The values are valid after tmem_wait_ld.)
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]),
          "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]),
          "=r"(u[30]), "=r"(u[31])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* u) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        :: "r"(addr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
           "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]),
           "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]),
           "r"(u[30]), "r"(u[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* u) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        :: "r"(addr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
           "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]) : "memory");
}

// ---- matrix instructions -------------------------------------------------------------------------
// D (fp32, tensor memory) [+]= A B, A: 128 rows, B: N columns, 16 of the contraction an instruction; both
// operands of the one 16-bit type.
template <typename T>
__host__ __device__ constexpr uint32_t mma_desc(int n, bool b_rows_contracted, bool negate_a = false) {
    const uint32_t fmt = DtypeOf<T>::value == DSDPA_BF16 ? 1u : 0u;
    return 1u << 4 | fmt << 7 | fmt << 10 | (negate_a ? 1u << 13 : 0u) | (b_rows_contracted ? 1u << 16 : 0u) |
           (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
// Shared-memory operand, 128-byte swizzle.  `lead`: bytes between panels (used by the MN-major form); groups
// of eight rows are 1024 bytes apart in both forms.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// The barrier gets one arrival when all matrix instructions issued so far by this thread are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}

// d[128 x N] = a[128 x HD] b[N x HD]^T: both tiles K-major, HD elements a row (panels of a: 128 rows, of b: N rows).
template <int HD>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, int n, uint32_t idesc) {
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) {
        const uint32_t in = (s % 4) * 32, pan = s / 4;
        mma_ss(d, smem_desc(a + pan * 128 * 128 + in, 16), smem_desc(b + pan * n * 128 + in, 16), idesc, s > 0);
    }
}
// d[128 x HD] (+)= p[128 x R] b[R x HD]: p in tensor memory (two 16-bit elements a column), b's rows contracted.
template <int R>
__device__ __forceinline__ void mma_weights(uint32_t d, uint32_t p, uint32_t b, uint32_t idesc, bool add) {
#pragma unroll
    for (int s = 0; s < R / 16; ++s)
        mma_ts(d, p + s * 8, smem_desc(b + s * 2048, R * 128), idesc, add || s > 0);
}

// Registers a thread, for all warps of a warpgroup: given back, or taken from what the block was launched with.
template <int N> __device__ __forceinline__ void regs_release() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N> __device__ __forceinline__ void regs_claim() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }

// Two fp32 values rounded to the storage type and packed, the first in the lower half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

}  // namespace dsdpa
