// Host-side pieces shared by the 8-bit block-scaled dense operators (blocks8.cu, matmul_fp8.cu,
// weight_grad.cu): argument checks and the launch check.
#pragma once
#include "common.hpp"

#include <atomic>

#include <cuda_runtime.h>

namespace tcc {

inline void checkCudaCall(cudaError_t s) {
    if (s != cudaSuccess)
        throw CudaError(cudaGetErrorString(s));
}
inline void require(bool ok, const char* message) {
    if (!ok)
        throw std::invalid_argument(message);
}
inline bool alignedTo(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
// Whether every row of a matrix starts on `a` bytes.
inline bool rowsAlignedTo(const void* p, uint64_t strideBytes, uintptr_t a) {
    return alignedTo(p, a) && strideBytes % a == 0;
}
inline bool isFloatType(int t) { return t == TCC_F32 || t == TCC_BF16 || t == TCC_F16; }
inline bool isFp8Type(int t) { return t == TCC_E4M3 || t == TCC_E5M2; }
inline uint32_t typeBytes(int t) { return t == TCC_F32 ? 4 : (t == TCC_BF16 || t == TCC_F16) ? 2 : 1; }
template <typename T> T ceilDiv(T a, T b) { return (a + b - 1) / b; }
// The largest number of rows or columns: sizes are rounded up to whole tiles of up to 256 in 32 bits.
constexpr uint32_t kLargestSize = 0xFFFFFF00u;
// The matrix's bytes do not reach over the end of the address space, nor its sizes over kLargestSize
// (rows, cols > 0).
inline bool extentFits(uint64_t rows, uint64_t cols, uint64_t stride, uint64_t elementBytes) {
    return rows <= kLargestSize && cols <= kLargestSize && stride <= (uint64_t(1) << 60) / elementBytes / rows && cols <= stride;
}
inline int currentDevice() {
    int device = 0;
    checkCudaCall(cudaGetDevice(&device));
    return device;
}
// Multiprocessors of the current device (asked once per device).
inline int multiprocessors() {
    static std::atomic<int> known[64] = {};
    const int device = currentDevice();
    int sms = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
    if (sms == 0) {
        checkCudaCall(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        if (device < 64)
            known[device].store(sms, std::memory_order_relaxed);
    }
    return sms;
}
// Lets a kernel use `bytes` of dynamic shared memory on the current device (set once per device).
template <auto Kernel> void allowSharedMemory(int bytes) {
    static std::atomic<bool> done[64] = {};
    const int device = currentDevice();
    if (device < 64 && done[device].load(std::memory_order_acquire))
        return;
    checkCudaCall(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (device < 64)
        done[device].store(true, std::memory_order_release);
}

// Status words of the dense kernels' bounded waits, merged into tcc_device_status. Each lives in
// its kernels' translation unit.
uint32_t matmulDeviceStatus(bool reset);
uint32_t weightGradDeviceStatus(bool reset);

} // namespace tcc
