// The few tcgen05, mbarrier and cp.async instructions that the tensor-core kernels use, and the
// shared-memory layout that their matrix descriptors state.
//
// Operands lie in panels of 64 16-bit columns: rows of 128 bytes, the 16-byte chunks of row r at
// chunk ^ (r & 7) (the 128-byte swizzle). The same panel serves as a K-major operand (its rows are
// the rows of A, or the columns of B) and as an MN-major one (its rows are k).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace oss {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- mbarrier ----------------------------------------------------------------
__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ bool mbar_try(uint32_t bar, int parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Bounded: a tile takes microseconds, the limit is about ten seconds. Once a wait of the block has run out
// (*dead), the others give up as well. False: it ran out; what it waited for is not there, and nothing may be
// issued that relies on it.
constexpr long long kWaitCycles = 20000000000ll;
[[nodiscard]] __device__ __forceinline__ bool mbar_wait(uint32_t bar, int parity, volatile int* dead) {
    if (mbar_try(bar, parity)) return true;
    const long long start = clock64();
    for (int i = 1; i < (1 << 30); ++i) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 63) == 1 && (*dead != 0 || clock64() - start > kWaitCycles)) break;
    }
    *dead = 1;
    return false;
}
// After a wait that ran out, for what is still on its way: a second at most, whatever *dead says.
__device__ __forceinline__ void mbar_settle(uint32_t bar, int parity) {
    const long long start = clock64();
    for (int i = 0; i < (1 << 28) && !mbar_try(bar, parity) && clock64() - start < kWaitCycles / 10; ++i) {
    }
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One lane of a whole warp, always the same. Products are issued under it: with a plain test of the lane
// the descriptors that reached them (they are warp-uniform registers) were not the ones computed.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one != 0;
}
// Barrier `id` among `threads` threads of the block.
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// ---- tensor copies -------------------------------------------------------------
// A box of a tensor of three axes into shared memory; completes `bar` by its bytes. x: a multiple of 8
// 16-bit elements.
__device__ __forceinline__ void tma_load(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// ---- cp.async ----------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Own shared-memory writes become visible to the tensor cores (after a barrier, everybody's).
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory -------------------------------------------------------------
template <int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t slot) {  // a whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLS) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 columns of a warp's 32 lanes: each thread its own lane's.
__device__ __forceinline__ void tmem_ld16(uint32_t at, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const float* r) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(r);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
        "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t* u) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(u[0]), "r"(u[1]),
                 "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
}

// ---- products -------------------------------------------------------------------
// Descriptor of a panel from byte address `at` (its 8-row groups 1024 bytes apart); `panel`: bytes
// to the next panel, for MN-major operands of more than 64 columns (unused otherwise).
__device__ __forceinline__ uint64_t desc(uint32_t at, uint32_t panel) {
    return static_cast<uint64_t>((at & 0x3ffff) >> 4) | (static_cast<uint64_t>(panel >> 4) << 16) | (64ull << 32) |
           (1ull << 46) | (2ull << 61);
}
// 16-bit operands of one type (bf16: 1, fp16: 0), fp32 sums, M = 128, N a multiple of 16.
__device__ __forceinline__ uint32_t idesc(int bf16, int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (static_cast<uint32_t>(bf16) << 7) | (static_cast<uint32_t>(bf16) << 10) |
           (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (8u << 24);
}
// d (+)= a b, 16 of k; one thread.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(static_cast<int>(add))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(static_cast<int>(add))
        : "memory");
}
// The barrier completes when every product issued so far by this thread has.
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// a b^T over dim16 <= DP columns: both K-major panels of ROWS_A and ROWS_B rows.
template <int DP, int ROWS_A, int ROWS_B>
__device__ __forceinline__ void mma_nt(uint32_t d, uint32_t a, uint32_t b, int dim16, uint32_t id) {
    const uint64_t da = desc(a, 16), db = desc(b, 16);
#pragma unroll
    for (int k = 0; k < DP; k += 16)
        if (k < dim16)
            mma_ss(d, da + ((k >> 6) * ROWS_A * 128 + (k & 63) * 2) / 16, db + ((k >> 6) * ROWS_B * 128 + (k & 63) * 2) / 16, id, k > 0);
}
// a b over k16 <= K rows of b (MN-major panels of K rows), a in tensor memory (two 16-bit values a column).
template <int K>
__device__ __forceinline__ void mma_tn(uint32_t d, uint32_t a, uint32_t b, int k16, uint32_t id, bool add) {
    const uint64_t db = desc(b, K * 128);
#pragma unroll
    for (int k = 0; k < K; k += 16)
        if (k < k16) mma_ts(d, a + k / 2, db + k * 128 / 16, id, add || k > 0);
}

// a^T b over K rows of MN-major panels, given their descriptors.
template <int K>
__device__ __forceinline__ void mma_tt(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
#pragma unroll
    for (int k = 0; k < K; k += 16) mma_ss(d, a + k * 128 / 16, b + k * 128 / 16, id, add || k > 0);
}

}  // namespace tc
}  // namespace oss
