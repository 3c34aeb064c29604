// PTX of the fifth-generation tensor cores shared by the e4m3 product and the cross attention: mbarriers with bounded
// waits, TMA tile loads, tensor memory, and the host's tensor maps.
#pragma once

#include <cuda.h>

#include <atomic>
#include <mutex>

#include "common.cuh"

namespace krea2 {

constexpr uint64_t kTensorWaitLimitNs = 2000000000ull;  // every wait gives up after two seconds

__device__ __forceinline__ uint32_t smem_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint64_t clock_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// ---------------------------------------------------------------- mbarriers
__device__ __forceinline__ void barrier_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_address(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_init_done() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_address(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_address(bar)) : "memory");
}
__device__ __forceinline__ bool barrier_test(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(smem_address(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// The same without the time that a try_wait may spend before it answers no.
__device__ __forceinline__ bool barrier_peek(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(smem_address(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// How a CTA's roles give up together: the CTA's flag, the device's status word and the bit to raise there.
struct Abort {
    volatile int *flag;
    int *status;
    int bit;
};
// What a wait that has not been met does between its tests: every 64th time it looks whether the CTA gives up or the time
// is over.  (The global timer takes longer to read than most waits last.)
struct Patience {
    uint64_t start = 0;
    uint32_t spins = 0;
    __device__ __forceinline__ bool over(const Abort &abort) {
        if ((++spins & 63u) != 0u) return false;
        if (*abort.flag) return true;
        const uint64_t now = clock_ns();
        if (start == 0) start = now;
        if (now - start <= kTensorWaitLimitNs) return false;
        *abort.flag = 1;
        atomicOr(abort.status, abort.bit);
        return true;
    }
};
// Waits for the phase of `parity`.  False when the CTA is giving up, or when this wait ran out (it raises both flags).
__device__ __forceinline__ bool barrier_wait(uint64_t *bar, uint32_t parity, const Abort &abort) {
    Patience patience;
    while (!barrier_test(bar, parity))
        if (patience.over(abort)) return false;
    return true;
}
// The same for a converged warp, whose lanes leave together.  `ready` is what an earlier barrier_peek() of this phase said: a
// loop that peeks at its next barriers before the work at hand has their answers when it comes back (a wait that is met takes
// some 130 clocks, as long as the tensor cores take for a quarter of a block).
__device__ __forceinline__ bool barrier_wait_warp(uint64_t *bar, uint32_t parity, const Abort &abort, bool ready = false) {
    if (__all_sync(0xffffffffu, ready)) return true;
    Patience patience;
    while (!__all_sync(0xffffffffu, barrier_test(bar, parity)))
        if (__any_sync(0xffffffffu, patience.over(abort))) return false;
    return true;
}
// After a wait that gave up: waits (bounded) until the loads armed on this phase have landed, so that none still writes
// this CTA's shared memory when it exits.
__device__ __forceinline__ void barrier_drain(uint64_t *bar, uint32_t parity, uint64_t start) {
    while (!barrier_test(bar, parity))
        if (clock_ns() - start > kTensorWaitLimitNs) return;
}

// A value that all lanes hold alike, taken from lane 0: what depends on it is compiled as uniform, and the products' operands
// need not be moved to uniform registers one by one.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// True in one lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_lane() {
    uint32_t elected;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(elected));
    return elected != 0;
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
// The shared::cluster address of `p` (in this CTA's shared memory) inside CTA `rank`.
__device__ __forceinline__ uint32_t cluster_address(const void *p, uint32_t rank) {
    uint32_t out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_address(p)), "r"(rank));
    return out;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_store(uint32_t address, uint32_t value) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(address), "r"(value) : "memory");
}
__device__ __forceinline__ float4 cluster_load(uint32_t address) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ float2 cluster_load_pair(uint32_t address) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(address) : "memory");
    return v;
}
// Arrives in another CTA of the cluster, for what this CTA has read from tensor memory: there is no global or shared
// memory to publish, and a release at cluster scope would wait for every load in flight (860 instead of 490 us for the
// e4m3 product of 4608 x 15360 x 6144, once per block of 128 channels).
__device__ __forceinline__ void barrier_arrive_at(uint32_t address) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(address) : "memory");
}

// ---------------------------------------------------------------- tile loads
__device__ __forceinline__ void load_tile(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_address(dst)), "l"(map), "r"(smem_address(bar)), "r"(c0), "r"(c1)
        : "memory");
}
// For a pair of CTAs: the completion is counted on a barrier that may live in the other CTA.
__device__ __forceinline__ void load_tile_pair(void *dst, const CUtensorMap *map, uint32_t bar_address, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_address(dst)), "l"(map), "r"(bar_address), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void load_tile_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_address(dst)), "l"(map), "r"(smem_address(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
// Shared memory to a tile; what lies outside the tensor is left out.  The caller commits and waits for the group.
__device__ __forceinline__ void store_tile_4d(const void *src, const CUtensorMap *map, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map), "r"(smem_address(src)), "r"(c0), "r"(c1),
                 "r"(c2), "r"(c3)
                 : "memory");
}

// ---------------------------------------------------------------- tensor memory
template <int kCtas>
__device__ __forceinline__ void tensor_alloc(uint32_t *dst, uint32_t columns) {
    if constexpr (kCtas == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(dst)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(dst)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int kCtas>
__device__ __forceinline__ void tensor_free(uint32_t address, uint32_t columns) {
    if constexpr (kCtas == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_stores_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Once the products issued so far have completed, arrives on the barrier (of both CTAs of a pair).
__device__ __forceinline__ void tensor_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_address(bar)) : "memory");
}
__device__ __forceinline__ void tensor_commit_pair(uint64_t *bar) {
    const uint16_t both = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_address(bar)), "h"(both)
                 : "memory");
}
// 32 lanes x 16 or 32 consecutive 32-bit columns: thread i of the warp receives (or stores) lane base + i.  The loads
// return before the values are there: a tensor_loads_done completes all that were issued.
__device__ __forceinline__ void tensor_load_16(uint32_t address, float *r) {
    uint32_t *u = reinterpret_cast<uint32_t *>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]),
          "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(address));
}
__device__ __forceinline__ void tensor_load_32(uint32_t address, float *r) {
    uint32_t *u = reinterpret_cast<uint32_t *>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]),
          "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]),
          "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]),
          "=r"(u[31])
        : "r"(address));
}
// Waits for all loads that were issued; tied to the values, so that nothing that uses them can be moved in front of it.
__device__ __forceinline__ void tensor_loads_done_16(float *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                   "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tensor_loads_done_32(float *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                   "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]),
                   "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]),
                   "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :
                 : "memory");
}
// 16 lanes x 16 columns in the fragment order: r[4 j + 0], r[4 j + 1] are columns 8 j + 2 (lane % 4) and the one after it of
// lane base + lane / 4, r[4 j + 2], r[4 j + 3] the same columns eight lanes below.  A thread meets a quarter of the columns.
__device__ __forceinline__ void tensor_load_fragment(uint32_t address, float *r) {
    uint32_t *u = reinterpret_cast<uint32_t *>(r);
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
                 : "r"(address));
}
__device__ __forceinline__ void tensor_store_32(uint32_t address, const uint32_t *u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(address),
        "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]),
        "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]),
        "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
        : "memory");
}
// K-major operand tile of 128-byte rows, 128-byte swizzled, eight rows (1024 bytes) per swizzle atom.
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t address) {
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// (a.x, a.y) * (b.x, b.y) + (c.x, c.y), one rounding per lane, in one issue slot.
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{ .reg .b64 p, q, r, s;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n mov.b64 r, {%6, %7};\n"
        " fma.rn.f32x2 s, p, q, r;\n mov.b64 {%0, %1}, s;\n }"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
    float2 d;
    asm("{ .reg .b64 p, q, r;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n add.rn.f32x2 r, p, q;\n mov.b64 {%0, %1}, r;\n }"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// ---------------------------------------------------------------- host side
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                   const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn() {
    static const EncodeTiledFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// A row-major tensor of `rank` dimensions (innermost first) as boxes with the 128-byte swizzle; what lies outside reads
// as zero.  `strides` are the bytes between neighbours in dimensions 1 and up.
inline int make_tensor_map(CUtensorMap *map, CUtensorMapDataType type, uint32_t rank, const void *base, const cuuint64_t *dims,
                           const cuuint64_t *strides, const cuuint32_t *box) {
    const EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return fail(KREA2_RUNTIME, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint32_t element_strides[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(map, type, rank, const_cast<void *>(base), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(KREA2_RUNTIME, "cuTensorMapEncodeTiled failed with code %d", static_cast<int>(r));
    return KREA2_OK;
}

// The current device's number of SMs.
inline int multiprocessors() {
    static std::atomic<int> cached[64];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 148;
    int n = cached[device].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) n = 148;
        cached[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Raises a kernel's dynamic shared-memory limit, once per device and kernel (`once` and `status` belong to the kernel).
struct Prepared {
    std::once_flag once[64];
    cudaError_t status[64] = {};
};
template <typename Kernel>
int prepare_kernel(Prepared &prepared, Kernel kernel, int shared_bytes) {
    int device = 0;
    KREA2_CUDA(cudaGetDevice(&device));
    if (device < 0 || device >= 64) return fail(KREA2_INTERNAL, "device index %d out of range", device);
    std::call_once(prepared.once[device], [&] {
        prepared.status[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes);
    });
    if (prepared.status[device] != cudaSuccess)
        return fail(KREA2_RUNTIME, "cannot reserve %d bytes of shared memory: %s", shared_bytes, cudaGetErrorString(prepared.status[device]));
    return KREA2_OK;
}

}  // namespace krea2
