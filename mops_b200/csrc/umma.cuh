// Tensor-core products with operands in shared memory and accumulators in tensor memory (tcgen05.mma), and the tiled copies
// (cp.async.bulk.tensor) that feed them. One thread issues each of them.
//
// Operand tiles are boxes of rows of 128 bytes (64 values of 16 bits), swizzled: the 16-byte chunk c of row r lies at chunk
// c ^ (r mod 8). Where the rows run along the depth of the product (K-major) a box holds `rows` rows or columns of the operand; where
// they run across it (MN-major) a box holds 64 of them, 64 deep, and boxes of further ones follow.
#ifndef MOPS_B200_UMMA_CUH
#define MOPS_B200_UMMA_CUH

#include <cuda.h>

#include "tmem.cuh"

namespace mops_b200 {

constexpr int kBoxRow = 128;               // bytes
constexpr int kBoxDepth = 64;              // values in a row, and the depth of a stage
constexpr int kBoxBytes = 64 * kBoxRow;    // of a box of 64 rows

// The shared-memory descriptor of an operand: version 1, swizzle over 128 bytes (or 64, for rows of 32 values). `across`: bytes between boxes
// of 64 rows or columns (MN-major; K-major operands ignore it). Groups of eight rows follow each other.
template <int kRowBytes = kBoxRow> __device__ __forceinline__ uint64_t operand_descriptor(uint32_t address, uint32_t across) {
    static_assert(kRowBytes == 128 || kRowBytes == 64, "swizzles");
    return static_cast<uint64_t>((address & 0x3ffff) >> 4) | static_cast<uint64_t>(across >> 4) << 16 |
           static_cast<uint64_t>(8 * kRowBytes >> 4) << 32 | uint64_t(1) << 46 | uint64_t(kRowBytes == 128 ? 2 : 4) << 61;
}
// What one step of 16 values in depth adds to a descriptor.
template <bool MN> constexpr uint64_t kDepthStep = MN ? 2048 >> 4 : 32 >> 4;

// f32 accumulators of m x n (m: 128, or 256 over a pair of SMs); both operands bf16 (or both f16).
__host__ __device__ constexpr uint32_t instruction_descriptor(bool bf16, bool a_mn, bool b_mn, int n, int m = 128) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           static_cast<uint32_t>(n / 8) << 17 | static_cast<uint32_t>(m / 16) << 24;
}

__device__ __forceinline__ void umma(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(accumulator),
                 "l"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(accumulate))
                 : "memory");
}
// With the rows' operand in tensor memory: a row to a lane, two values of depth to a column.
__device__ __forceinline__ void umma_from_tmem(uint32_t accumulator, uint32_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(accumulator),
                 "r"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(accumulate))
                 : "memory");
}
// Arrives on `bar` when the products issued so far by this thread are done.
__device__ __forceinline__ void umma_arrive(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_address(bar))
                 : "memory");
}

__device__ __forceinline__ void mbarrier_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_address(bar)) : "memory");
}

// Makes this thread's writes to shared memory visible to the copy engine and the tensor cores.
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Box at (inner, outer, slice) of an array, completion counted on `bar`.
__device__ __forceinline__ void box_in(uint32_t smem, const CUtensorMap& map, int inner, int outer, int slice, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::
                     "r"(smem),
                 "l"(&map), "r"(inner), "r"(outer), "r"(slice), "r"(smem_address(bar))
                 : "memory");
}
__device__ __forceinline__ void box_out(const CUtensorMap& map, int inner, int outer, int slice, uint32_t smem) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n" ::"l"(&map),
                 "r"(inner), "r"(outer), "r"(slice), "r"(smem)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}
// Until all but the last N boxes that this thread sent out have left shared memory.
template <int N> __device__ __forceinline__ void boxes_left() {
    asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(N) : "memory");
}
// Until all boxes that this thread sent out are in global memory, where ordinary stores may follow.
__device__ __forceinline__ void boxes_written() {
    asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
    asm volatile("fence.proxy.async;\n" ::: "memory");
}
__device__ __forceinline__ void map_prefetch(const CUtensorMap& map) {
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map) : "memory");
}

__device__ __forceinline__ void smem_store16(uint32_t address, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(address), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ uint16_t smem_load2(uint32_t address) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(v) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t smem_load4(uint32_t address) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ uint4 smem_load16(uint32_t address) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
    return v;
}

// ---- work that is handed out while the kernel runs: the grid has a block (or a pair) for each piece of work; those that run take over the places of
// those that have not begun. The answer (16 bytes of shared memory, of both blocks of a pair) is counted on `bar`.
template <bool kPair> __device__ __forceinline__ void take_over(void* answer, uint64_t* bar) {
    if constexpr (kPair)
        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.multicast::cluster::all.b128 [%0], [%1];\n" ::
                         "r"(smem_address(answer)),
                     "r"(smem_address(bar))
                     : "memory");
    else
        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(smem_address(answer)),
                     "r"(smem_address(bar))
                     : "memory");
}
// Index of the (first) block whose place was taken over, or -1 if there is none left.
__device__ __forceinline__ int taken_over(const void* answer) {
    uint32_t taken, x;
    asm volatile("{\n .reg .b128 a;\n .reg .pred p;\n .reg .b32 y, z, w;\n"
                 " ld.shared.b128 a, [%2];\n"
                 " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n"
                 " selp.u32 %0, 1, 0, p;\n"
                 " mov.b32 %1, 0;\n"
                 " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, a;\n}\n"
                 : "=r"(taken), "=r"(x)
                 : "r"(smem_address(answer))
                 : "memory");
    return taken ? static_cast<int>(x) : -1;
}

// ---- pairs of blocks (clusters of two), whose SMs multiply together: each has half of the rows of the accumulator in its tensor memory, and half of
// either operand in its shared memory, at the same addresses. The first block of the pair issues the products.
__device__ __forceinline__ unsigned pair_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
// Both blocks, all threads.
__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The address of the first block's copy of something in shared memory.
__device__ __forceinline__ uint32_t first_of_pair(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(a) : "r"(smem_address(p)));
    return a;
}
__device__ __forceinline__ void pair_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pair_arrive_expect(uint32_t bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
// Sees what the other block wrote before it arrived, too (which costs hundreds of clocks: not for barriers that only copies and products are
// counted on).
__device__ __forceinline__ bool mbarrier_try_wait_pair(uint64_t* bar, unsigned parity) {
    unsigned done;
    asm volatile("{\n .reg .pred p;\n"
                 " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
                 " selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(smem_address(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}
// Into this block's shared memory, completion counted on a barrier of either block.
__device__ __forceinline__ void pair_box_in(uint32_t smem, const CUtensorMap& map, int inner, int outer, int slice, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];\n" ::
                     "r"(smem),
                 "l"(&map), "r"(inner), "r"(outer), "r"(slice), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void pair_umma(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(accumulator),
                 "l"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(accumulate))
                 : "memory");
}
// Arrives on the barrier at this address of both blocks.
__device__ __forceinline__ void pair_umma_arrive(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(smem_address(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* smem_address_out, unsigned columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_address(smem_address_out)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_free(uint32_t address, unsigned columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(address), "r"(columns) : "memory");
}

} // namespace mops_b200

#endif
