// The sm_100a instructions the tensor-core kernels are built from: mbarriers with bounded waits, tiled TMA loads, tensor
// memory and tcgen05.mma, each as one inline function, and the descriptors they take.
//
// Shared-memory operands are tiles of `rows` x 64 16-bit values, 128 bytes per row, in the 128-byte swizzle that the TMA
// load applies (16-byte chunk c of row r lies at chunk c ^ (r % 8)); wider rows are several such tiles behind one another.
//   K-major   (the contracted dimension runs along the 128 bytes): 8-row groups 1024 bytes apart; 16 values = 32 bytes.
//   MN-major  (the contracted dimension runs down the rows): 8-row groups 1024 bytes apart; 64-value column blocks one tile
//             (rows * 128 bytes) apart; 16 contracted rows = 2048 bytes.
#ifndef MCSPARSE_B200_TENSOR_CORE_H_
#define MCSPARSE_B200_TENSOR_CORE_H_

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mcsp_b200 {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// True in one lane of a converged warp, always the same one. (With `lane == 0` in its place a tcgen05.mma of 64 clocks of work
// took 95 to 210 clocks in a row of them.)
__device__ __forceinline__ bool elect() {
    uint32_t one = 0;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n @p mov.u32 %0, 1;\n}" : "+r"(one));
    return one != 0;
}

// A value that is the same in all lanes of a converged warp, taken over the warp. Loaded values, and loop bounds that depend on
// them, pass through it before they reach the operands of a tcgen05.mma: without it each such instruction took 75 to 100 clocks more.
__device__ __forceinline__ int uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

// ---- mbarriers

__device__ __forceinline__ void bar_init(uint32_t bar, int arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Waits until the phase of the given parity has completed, for at most `limit` SM clocks. False: it gave up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, long long limit) {
    if (bar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!bar_try(bar, parity))
        if (clock64() - t0 > limit) return false;
    return true;
}

// Limit (SM clocks, about a second) of the waits with which a block that gave up lets its copies and products end.
constexpr long long kDrain = 2000000000;
// bar_wait for a whole warp: one answer for all lanes.
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, long long limit) {
    return __all_sync(0xffffffffu, bar_wait(bar, parity, limit));
}

// ---- TMA

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// Orders this thread's ordinary shared-memory writes before later reads by TMA or tcgen05.mma.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- cluster launch control: a running block takes over a block of the grid that has not started

// Asks for one; the answer (16 bytes) completes on the barrier.
__device__ __forceinline__ void ask_block(uint32_t answer, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
// Its blockIdx.x, or -1: there is none left (and none may be asked for again).
__device__ __forceinline__ int asked_block(uint32_t answer) {
    int x;
    asm volatile(
        "{\n .reg .b128 h;\n .reg .pred p;\n ld.shared.b128 h, [%1];\n clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
        " mov.s32 %0, -1;\n @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n}"
        : "=r"(x)
        : "r"(answer)
        : "memory");
    return x;
}

// ---- tensor memory

__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, int columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base, int columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 consecutive columns of the calling thread's row (lane 32 * (warp % 4) + lane of the tensor memory).
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// Keeps the compiler from using loaded registers before wait_loads(): the load's outputs carry no such dependence themselves.
__device__ __forceinline__ void after_loads32(uint32_t* r) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// ---- tcgen05.mma (kind::f16: both operands fp16 or both bf16, fp32 accumulators)

// Descriptor of a swizzled shared-memory operand (see the head of the file). column_block: bytes between 64-value column
// blocks of an MN-major operand; not used by a K-major one.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t column_block = 16) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3fff);
    d |= (uint64_t)((column_block >> 4) & 0x3fff) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;  // 128-byte swizzle
    return d;
}
// The descriptor of the operand `bytes` (a multiple of 16) further on.
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }
// Instruction descriptor: D (128 x n, fp32) = A * B, bf16 or fp16; b_mn: B is MN-major; with kNegateA, A enters with its sign turned.
__host__ __device__ constexpr uint32_t mma_desc(bool bf16, int n, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
constexpr uint32_t kNegateA = 1u << 13;

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(desc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(desc), "r"((uint32_t)accumulate)
        : "memory");
}
// The barrier gets one arrival when everything this thread has issued so far is done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// ---- fp32 arithmetic

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The larger of three; NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// Two values in one register pair, one instruction for both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(lo), "f"(hi));
    return y;
}
__device__ __forceinline__ void unpair(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
// Bits 0 .. n - 1 (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

}  // namespace tc
}  // namespace mcsp_b200

#endif  // MCSPARSE_B200_TENSOR_CORE_H_
