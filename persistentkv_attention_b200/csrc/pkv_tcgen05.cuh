// pkv_tcgen05.cuh -- sm_100a tensor-core primitives: TMEM allocation and
// access, tcgen05.mma with operands in shared memory or TMEM, descriptors.
#pragma once

#include "pkv_device.cuh"

namespace pkv {

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " elect.sync _|p, 0xffffffff;\n"
        " selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(one));
    return one != 0;
}

// ---------------------------------------------------------------- TMEM
// Whole-warp; writes the base address to *slot (shared memory).
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(slot)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns)
                 : "memory");
}

__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Arrives on `bar` once every tcgen05.mma this thread has issued is complete.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_u32(bar))
                 : "memory");
}

// ---------------------------------------------------------------- operands
// Shared-memory descriptor of a tile of 128-byte lines in the 128-byte
// swizzle (8-line, 1 KB atoms), its low word.  K-major: `lead` is unused.
// MN-major (128-byte lines run along the rows of the operand): `lead` is the
// distance of the 64-element groups along the rows.  The high word is a constant
// (groups of 8 rows, or of 8 along K, 1024 bytes apart; version 1; the swizzle), so
// that an operand costs one 32-bit add (16384 tokens: 2060 -> 2020 us).
__device__ __forceinline__ uint32_t smem_desc_sw128(uint32_t addr, uint32_t lead) {
    return ((addr & 0x3ffffu) >> 4) | ((lead >> 4) << 16);
}
constexpr uint32_t kDescHighSw128 = (1024u >> 4) | (1u << 14) | (2u << 29);

// Instruction descriptor of kind::f16 with fp32 accumulation: M x N tile,
// both operands bf16 or both fp16, B K-major or MN-major.
__host__ __device__ constexpr uint32_t mma_desc_f16(int m, int n, bool bf16, bool b_mn_major) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) |
           ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// D[tmem] (+)= A[smem] . B[smem], K = 16; one thread.
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                           bool accumulate) {
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " .reg .b64 da, db;\n"
        " mov.b64 da, {%1, %5};\n"
        " mov.b64 db, {%2, %5};\n"
        " setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHighSw128)
        : "memory");
}

// D[tmem] (+)= A[tmem] . B[smem], K = 16; one thread.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                           bool accumulate) {
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " .reg .b64 db;\n"
        " mov.b64 db, {%2, %5};\n"
        " setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHighSw128)
        : "memory");
}

// 3-D tiled TMA load (no multicast) of one box; completion as transaction
// bytes on `bar`.
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int x, int y,
                                            int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// ---------------------------------------------------------------- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}

// Barrier of all threads of the cluster; shared-memory writes before it are
// seen by the others' reads after it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The address of this CTA's shared-memory address `addr` in CTA `rank`.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                 : "=f"(v.x), "=f"(v.y)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// ---------------------------------------------------------------- launch control
// Asks for a CTA of this grid that has not started: 16 bytes of answer to
// `answer` (shared memory), as transaction bytes on `bar`.  Not asked again
// once an answer was no.
__device__ __forceinline__ void launch_cancel_async(void* answer, uint64_t* bar) {
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 "
        "[%0], [%1];" ::"r"(smem_u32(answer)),
        "r"(smem_u32(bar))
        : "memory");
}

// Whether a CTA was given, and its blockIdx.x.
__device__ __forceinline__ bool launch_cancelled(const void* answer, int& block) {
    uint32_t yes, x;
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " .reg .b128 a;\n"
        " ld.shared.b128 a, [%2];\n"
        " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n"
        " selp.u32 %0, 1, 0, p;\n"
        " mov.u32 %1, 0;\n"
        " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n"
        "}\n"
        : "=r"(yes), "=r"(x)
        : "r"(smem_u32(answer))
        : "memory");
    if (yes != 0u) block = (int)x;
    return yes != 0u;
}

#define PKV_R4(o, n) o(n), o(n + 1), o(n + 2), o(n + 3)
#define PKV_R16(o, n) PKV_R4(o, n), PKV_R4(o, n + 4), PKV_R4(o, n + 8), PKV_R4(o, n + 12)
#define PKV_R32(o, n) PKV_R16(o, n), PKV_R16(o, n + 16)

// 32 columns of the warp's 32 lanes: r[c] is this lane's column c.  The
// values are only there after tmem_wait_ld on the same registers.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
#define PKV_O(i) "=r"(r[i])
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : PKV_R32(PKV_O, 0)
        : "r"(addr));
#undef PKV_O
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
#define PKV_O(i) "=r"(r[i])
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : PKV_R16(PKV_O, 0)
        : "r"(addr));
#undef PKV_O
}

__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
#define PKV_O(i) "+r"(r[i])
    asm volatile("tcgen05.wait::ld.sync.aligned;" : PKV_R16(PKV_O, 0)::"memory");
#undef PKV_O
}

// Waits for the thread's TMEM loads; the registers pass through so that no
// use of them moves before the wait.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t* r) {
#define PKV_O(i) "+r"(r[i])
    asm volatile("tcgen05.wait::ld.sync.aligned;" : PKV_R32(PKV_O, 0)::"memory");
#undef PKV_O
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
#define PKV_O(i) "r"(r[i])
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::PKV_R16(PKV_O,
                                                                                            0),
        "r"(addr)
        : "memory");
#undef PKV_O
}

__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

}  // namespace pkv
