// Building blocks of the tensor-core kernels, shared by the dense bipartite path and the 8-bit product: bounded mbarrier
// waits, TMA loads, tcgen05 descriptors, MMAs and tensor-memory loads, the hand-overs inside a CTA pair, and the host side's
// operand maps.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <string>

#include "tables.h"

namespace thrml {
namespace dense {

constexpr uint32_t SPIN_LIMIT = 1u << 24;  // hard cap on the number of parked waits of one mbar_wait (the time bound normally ends it first)

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Where the roles that wait on each other's barriers tell of a wait that ran out: a word in global memory, or one in the CTA's shared memory.
struct GlobalWord {
    int* p;
    __device__ __forceinline__ bool raised() const { return *reinterpret_cast<volatile int*>(p) != 0; }
    __device__ __forceinline__ void raise(int code) const { atomicCAS(p, 0, code); }
};
struct SharedWord {
    uint32_t at;
    __device__ __forceinline__ int value() const {
        int v;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
        return v;
    }
    __device__ __forceinline__ bool raised() const { return value() != 0; }
    __device__ __forceinline__ void raise(int code) const { asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(at), "r"(code) : "memory"); }
};
// mbar_wait: bounded wait on a phase parity.  Returns false (and raises the word) when the limit runs out, or another role has raised it.
// try_wait parks the thread in hardware for up to the hinted time instead of spinning: a polling loop in the producer
// or MMA warp would take issue slots from the epilogue warps that share its scheduler.  The bound is wall time
// (about two seconds on the global nanosecond timer), checked between the parked waits.
__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
constexpr uint64_t WAIT_LIMIT_NS = 2000000000ull;
__device__ __forceinline__ bool mbar_park(uint32_t bar_addr, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar_addr), "r"(parity), "r"(20000u)
        : "memory");
    return ok;
}
template <class Word>
__device__ __forceinline__ bool mbar_park_on(uint32_t bar_addr, uint32_t parity, Word word, int code) {
    uint64_t t0 = 0;
    for (uint32_t spin = 0; spin < SPIN_LIMIT; ++spin) {
        if (mbar_park(bar_addr, parity)) return true;
        if ((spin & 15u) == 15u) {
            if (word.raised()) return false;  // another role gave up
            const uint64_t now = global_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > WAIT_LIMIT_NS) break;
        }
    }
    word.raise(code);
    return false;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, int* err, int code) { return mbar_park_on(smem_u32(bar), parity, GlobalWord{err}, code); }
// The turns behind the first (20 us) out of line: few waits need any, and inside every wait they cost issue slots
// (8192 x 4096 -> 16384: 460 -> 425 us).
static __device__ __noinline__ bool mbar_park_longer(uint32_t bar_addr, uint32_t parity, SharedWord word, int code) { return mbar_park_on(bar_addr, parity, word, code); }
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, SharedWord word, int code) {
    const uint32_t addr = smem_u32(bar);
    return mbar_park(addr, parity) || mbar_park_longer(addr, parity, word, code);
}

// For what a kernel has in flight when its roles have given up: nobody to tell, and the same limit.
struct NoWord {
    __device__ __forceinline__ bool raised() const { return false; }
    __device__ __forceinline__ void raise(int) const {}
};
static __device__ __noinline__ void mbar_settle(uint64_t* bar, uint32_t parity) { mbar_park_on(smem_u32(bar), parity, NoWord{}, 0); }
// The last of `issued` loads in turn on a ring of barriers: those that no later one has waited for.
static __device__ __noinline__ void settle_loads(uint64_t* ring, int32_t stages, int32_t issued) {
    for (int32_t i = max(issued - stages, 0); i < issued; ++i) mbar_settle(ring + i % stages, i / stages & 1);
}
// Bytes that will not come count as come.
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
                 : "memory");
}

// Shared-memory matrix descriptor for a K-major tile whose rows are 128 bytes, 128-byte swizzled, groups of 8 rows
// 1024 bytes apart: start address, leading offset 16 B (unused for this layout), stride offset 1024 B, descriptor
// version 1, layout type 2 (128-byte swizzle).
__device__ __forceinline__ uint64_t make_smem_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3fffu);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// Instruction descriptor: accumulator format (1 f32, 2 s32), A/B formats, both K-major, N/8 at bit 17, M/16 at bit 24.
__host__ __device__ constexpr uint32_t make_idesc(uint32_t c_fmt, uint32_t ab_fmt, uint32_t m, uint32_t n) {
    return (c_fmt << 4) | (ab_fmt << 7) | (ab_fmt << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <int KIND_I8>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    if (KIND_I8) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Asynchronous TMEM load of 16 columns of this thread's lane; the registers are valid after tmem_ld_wait().
__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---- CTA pairs
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Address of the same shared-memory object in the CTA of the given cluster rank.
__device__ __forceinline__ uint32_t peer_addr(uint32_t local_addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local_addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// TMA load whose completion is counted on a barrier that may live in the pair's other CTA.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t smem_dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(x), "r"(y)
                 : "memory");
}
template <int KIND_I8>
__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    if (KIND_I8) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}
// Arrival (once the pair's earlier MMAs have completed) on a barrier given by its cluster address.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar_cluster_addr) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_cluster_addr) : "memory");
}

}  // namespace dense

// ---- host side
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_tiled_fn() {
    static std::atomic<EncodeTiledFn> found{nullptr};  // calls come from several threads
    EncodeTiledFn fn = found.load(std::memory_order_acquire);
    if (!fn) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            found.store(fn = reinterpret_cast<EncodeTiledFn>(sym), std::memory_order_release);
    }
    return fn;
}
// 2-D K-major operand: `rows` rows of `k_elems` contiguous elements, row pitch in bytes; box = 128 bytes of K x box_rows,
// 128-byte swizzle, out-of-range elements read as zero.
inline int32_t make_operand_map(CUtensorMap* map, void* base, bool is_u8, int64_t k_elems, int64_t rows, int64_t pitch_bytes, int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return fail(THRML_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k_elems), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(is_u8 ? 128 : 64), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, is_u8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(THRML_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(r)));
    return THRML_OK;
}

}  // namespace thrml
