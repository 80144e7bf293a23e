// Tensor-core, TMA and barrier pieces of the dense kernels (sm_100a inline PTX), beside those of
// spmm_device.cuh: tiled TMA loads, block-scaled and bf16 MMAs from shared memory, scale copies
// into tensor memory, and bounded waits with a status word of this translation unit.
#pragma once
#include "dense8.hpp"
#include "spmm_device.cuh"

#include <cuda.h>

namespace tcc {
namespace {

__device__ unsigned int gDenseStatus = 0; // bit 0: a bounded wait ran out (merged into tcc_device_status)
constexpr uint64_t kDenseWaitNs = 2000000000ull;

// Wait for a phase of an mbarrier, at most about two seconds; false when it ran out.
__device__ __forceinline__ bool waitPhase(uint32_t bar, uint32_t parity) {
    if (dev::mbarTryWait(bar, parity))
        return true;
    uint64_t start = 0;
    for (uint32_t attempt = 1;; ++attempt) {
        if (dev::mbarTryWaitSuspend(bar, parity, 2000u))
            return true;
        if ((attempt & 63u) == 0) {
            const uint64_t now = dev::globalTimerNs();
            if (start == 0) {
                start = now;
            } else if (now - start > kDenseWaitNs) {
                atomicOr(&gDenseStatus, 1u);
                return false;
            }
        }
    }
}

// Box of a 2-D tensor map at (x, y) (x along the row, in elements) into shared memory. x is a
// multiple of 16 bytes in every call: the maps' boxes are 128 bytes wide and x steps by them.
__device__ __forceinline__ void tmaLoad2d(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tmaPrefetchMap(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Shared-memory matrix descriptor of a 128-byte swizzled operand (start address, leading and stride
// byte offsets in units of 16; bits 46-47 = 1; bits 61-63 = 2 for the 128-byte swizzle).
//  K-major: rows of 128 bytes of k, 8-row groups `stride` bytes apart (the leading offset is unused).
//  MN-major: rows of 128 bytes of m or n, one row per k; `leading` bytes between 128-byte column
//  groups, `stride` bytes between groups of 8 rows.
__device__ __forceinline__ uint64_t swizzledDesc(uint32_t addr, uint32_t leading, uint32_t stride) {
    return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t((leading >> 4) & 0x3FFFu) << 16) |
           (uint64_t((stride >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
// Descriptor of 32 rows of 16 bytes (8-row groups 128 bytes apart, no swizzle): a scale slab.
__device__ __forceinline__ uint64_t slabDesc(uint32_t addr) {
    return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(128 >> 4) << 32) | (1ull << 46);
}

// 32 rows x 16 bytes from shared memory to 4 tensor-memory columns, repeated in the four lane
// quarters: row i's word c lands in lanes i, i + 32, i + 64 and i + 96 of column c. In every CTA of a
// pair, from its own shared memory.
template <int CG> __device__ __forceinline__ void tcCopyScales(uint32_t elected, uint32_t taddr, uint64_t desc) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
                     "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(elected)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
                     "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(elected)
                     : "memory");
}

// The MMA issuing warps run in uniform control flow, so that the operands stay in uniform registers
// (an MMA issued inside a one-lane branch moves each operand there first, which took longer than the
// MMA itself), and one elected lane issues.
__device__ __forceinline__ uint32_t electLane() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}
// D(tmem) (+)= A x B from shared memory, 8-bit floats with E8M0 scales in tensor memory (one per 32
// elements of k), by the lane with `elected`.
template <int CG>
__device__ __forceinline__ void mmaScaled8(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                           uint32_t scaleA, uint32_t scaleB, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %7, 0;\n\t"
                     "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scaleA), "r"(scaleB), "r"(accumulate), "r"(elected)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %7, 0;\n\t"
                     "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scaleA), "r"(scaleB), "r"(accumulate), "r"(elected)
                     : "memory");
}

// Warp load of 32 TMEM lanes x 8 columns: thread t reads lane t, r[j] = column j.
__device__ __forceinline__ void tcLoad32x32bx8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
// The same for 32 columns: thread t reads lane t, r[j] = column j.
__device__ __forceinline__ void tcLoad32x32bx32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
}

// ---- clusters of one or two CTAs (CG) ----------------------------------------------------------
__device__ __forceinline__ uint32_t clusterRank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// All threads of the CTAs of the cluster.
__device__ __forceinline__ void clusterBarrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CG> __device__ __forceinline__ void clusterSync() {
    if constexpr (CG == 1)
        __syncthreads();
    else
        clusterBarrier();
}
// A float at this shared-memory address of another CTA of the cluster.
__device__ __forceinline__ float ldClusterF32(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
                 : "=f"(v)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}
// Arrive on the barrier at this address of the cluster's first CTA. No cluster-wide release, which
// took about 1300 cycles and held the MMAs up: nothing that one CTA wrote is read by the other. Each
// SM's tensor core reads its own CTA's shared and tensor memory, whose writers have fenced and
// arrived before; the arrival only tells the issuing thread so.
template <int CG> __device__ __forceinline__ void arriveLeader(uint32_t bar) {
    if constexpr (CG == 1)
        dev::mbarArrive(bar);
    else
        asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
                     "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar)
                     : "memory");
}
// One arrival on the barrier at this address in every CTA of the cluster, once the tcgen05
// operations that the elected lane issued are done.
template <int CG> __device__ __forceinline__ void commitCluster(uint32_t elected, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
                     "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                     ::"r"(bar), "r"(elected)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
                     "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}"
                     ::"r"(bar), "r"(elected), "h"(static_cast<unsigned short>(3))
                     : "memory");
}
template <int CG> __device__ __forceinline__ void tmemAllocGroup(uint32_t dst, uint32_t cols) {
    if constexpr (CG == 1) {
        dev::tmemAlloc(dst, cols);
        dev::tmemRelinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG> __device__ __forceinline__ void tmemDeallocGroup(uint32_t taddr, uint32_t cols) {
    if constexpr (CG == 1)
        dev::tmemDealloc(taddr, cols);
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}

// Warp store of 16 TMEM lanes x 8 columns: thread t writes lane t / 4 (r0, r1) and lane t / 4 + 8
// (r2, r3) at columns 2 (t % 4) and 2 (t % 4) + 1.
__device__ __forceinline__ void tcStore16x256b(uint32_t taddr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r0), "r"(r1), "r"(r2),
                 "r"(r3)
                 : "memory");
}
template <int N> __device__ __forceinline__ void registersUp() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void registersDown() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// A 2-D map of rows x cols bytes-or-wider elements and zeros outside, swizzled unless told otherwise.
inline CUtensorMap tensorMap2d(const void* base, CUtensorMapDataType type, uint32_t elementBytes, uint64_t rows,
                               uint64_t cols, uint64_t stride, uint32_t boxRows, uint32_t boxCols,
                               CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found{};
        checkCudaCall(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
        if (fn == nullptr || found != cudaDriverEntryPointSuccess)
            throw CudaError("the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<Encode>(fn);
    }();
    CUtensorMap map;
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {stride * elementBytes};
    const cuuint32_t box[2] = {boxCols, boxRows}, steps[2] = {1, 1};
    if (encode(&map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) !=
        CUDA_SUCCESS)
        throw CudaError("cuTensorMapEncodeTiled refused a matrix");
    return map;
}

inline uint32_t denseStatus(bool reset) {
    uint32_t s = 0;
    checkCudaCall(cudaMemcpyFromSymbol(&s, gDenseStatus, sizeof s));
    if (reset && s != 0) {
        const uint32_t zero = 0;
        checkCudaCall(cudaMemcpyToSymbol(gDenseStatus, &zero, sizeof zero));
    }
    return s;
}

} // namespace
} // namespace tcc
