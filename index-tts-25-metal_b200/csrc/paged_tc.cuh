// mbarriers, TMA loads of cache blocks and tcgen05 operations of the paged
// attention tile kernels.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "paged_attn.cuh"

namespace itts {
namespace paged {

__device__ __forceinline__ void mbar_init(unsigned long long* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect(unsigned long long* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(unsigned long long* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// Limit of a wait that lasts as long as the work on an item: 2^30 keys take a CTA
// up to a minute.  The roles that do the work wait for each unit with the limit
// above and raise the abort flag, which ends this wait, too.
constexpr unsigned long long kItemLimitNs = 120 * 1000000000ull;

// Waits for a phase of `bar`.  Gives up when the time limit passes (and raises
// the CTA's abort flag) or, if `abort` is given, when another role has raised it.
__device__ __forceinline__ bool mbar_wait(unsigned long long* bar, uint32_t parity, int* abort,
                                          unsigned long long limit = kWaitLimitNs) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    for (uint32_t i = 0;; ++i) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 15u) == 15u) {
            if (abort && *reinterpret_cast<volatile int*>(abort)) return false;
            if (globaltimer_ns() - t0 > limit) {
                if (abort) *reinterpret_cast<volatile int*>(abort) = 1;
                return false;
            }
        }
    }
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// The same value in every lane, and known to be: the products' operands then
// stay in uniform registers.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}

// Rows of one block and head from token on, 128 bytes of each (x: first element).
__device__ __forceinline__ void tma_block(uint32_t dst, const CUtensorMap* map, int x, int token, int head, int block,
                                          unsigned long long* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(token), "r"(head), "r"(block), "r"(smem_u32(bar))
        : "memory");
}

// A box of query rows (tokens x heads), 128 bytes of each.
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int token,
                                         unsigned long long* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tc_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// ... that also ties the registers that the loads fill to the wait: no use of them moves above it.
template <int N>
__device__ __forceinline__ void tc_wait_ld(uint32_t (&v)[N]) {
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors, 128-byte swizzle (rows of 128 bytes, groups of
// eight rows 1024 bytes apart), descriptor version 1.  K-major operand: rows
// are the M or N index.  MN-major: rows are the K index, `lead` bytes between
// the blocks of 64 M or N elements.  The high word is the same for all; the low
// word holds address / 16 and lead / 16, so stepping through an operand adds
// to it.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lead) {
    return ((addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16);
}

#define ITTS_R32(v, o)                                                                                             \
    "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]),     \
        "=r"(v[o + 7]), "=r"(v[o + 8]), "=r"(v[o + 9]), "=r"(v[o + 10]), "=r"(v[o + 11]), "=r"(v[o + 12]),          \
        "=r"(v[o + 13]), "=r"(v[o + 14]), "=r"(v[o + 15]), "=r"(v[o + 16]), "=r"(v[o + 17]), "=r"(v[o + 18]),       \
        "=r"(v[o + 19]), "=r"(v[o + 20]), "=r"(v[o + 21]), "=r"(v[o + 22]), "=r"(v[o + 23]), "=r"(v[o + 24]),       \
        "=r"(v[o + 25]), "=r"(v[o + 26]), "=r"(v[o + 27]), "=r"(v[o + 28]), "=r"(v[o + 29]), "=r"(v[o + 30]),       \
        "=r"(v[o + 31])

// 32 columns of this warp's 32 lanes of tensor memory: lane = row.
template <int N>
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[N], int o = 0) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : ITTS_R32(v, o)
        : "r"(addr));
}
template <int N>
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&v)[N]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(addr)
                 : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[N]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
        : "memory");
}
#undef ITTS_R32

// Tensor map of a paged cache tensor: [blocks][heads][block_size][head_dim]
// at its strides, read as boxes of up to `tokens` tokens of one block and head x
// 128 bytes, 128-byte swizzled.  Blocks outside the cache read as zeros.
cudaError_t make_block_map(CUtensorMap* map, const itts_paged_cache& c, bool v, int tokens);

}  // namespace paged
}  // namespace itts
