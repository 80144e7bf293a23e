// Product of two 8-bit block-scaled matrices on sm_100a:
//   Y[m, n] = sum over k of a[m, k] 2^ea[m, k / 128] * b[n, k] 2^eb[n, k / 128]  (+ bias[n])
#include "dense8.cuh"
#include "dense8.hpp"

namespace tcc {
namespace {

using namespace blk;

struct Operand {
    const uint8_t* data;
    const uint8_t* scales;
    uint64_t stride;
    int type;
    uint32_t rowShift; // rows per scale block: 1 << rowShift
};
struct Product {
    Operand a, b;
    bool kn; // b is [k, n] instead of [n, k]
    const float* bias;
    void* out;
    uint64_t outStride;
    int outType;
    uint32_t m, n, k;
    cudaStream_t stream;
};

__device__ __forceinline__ float fp8Value(uint8_t v, bool e4m3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(v, e4m3 ? __NV_E4M3 : __NV_E5M2);
    return __half2float(__half(h));
}

// ---- any strides and alignment ----------------------------------------------------------------
// 64 x 64 outputs per CTA, 4 x 4 per thread, FP32 FMA from operands dequantized into shared memory.
// For matrices whose rows do not start on 16 bytes, which the tensor-core kernels' copies cannot read.
constexpr int kTile = 64, kStep = 32;

template <typename T>
__global__ void __launch_bounds__(256) productGeneric(const Operand a, const Operand b, bool kn, const float* __restrict__ bias,
                                                      T* __restrict__ out, uint64_t outStride, uint32_t m, uint32_t n,
                                                      uint32_t k, uint32_t tilesN) {
    __shared__ float as[kStep][kTile + 1], bs[kStep][kTile + 1];
    const uint32_t m0 = blockIdx.x / tilesN * kTile, n0 = blockIdx.x % tilesN * kTile;
    const uint32_t kBlocks = (k + kBlock - 1) / kBlock, nBlocks = (n + kBlock - 1) / kBlock;
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < k; k0 += kStep) {
        for (uint32_t i = threadIdx.x; i < kStep * kTile; i += 256) {
            {
                const uint32_t kk = i % kStep, r = i / kStep;
                const uint32_t row = m0 + r, col = k0 + kk;
                float v = 0.0f;
                if (row < m && col < k)
                    v = fp8Value(a.data[row * a.stride + col], a.type == TCC_E4M3) *
                        scaleValue(a.scales[uint64_t(row >> a.rowShift) * kBlocks + col / kBlock]);
                as[kk][r] = v;
            }
            const uint32_t kk = kn ? i / kTile : i % kStep, r = kn ? i % kTile : i / kStep;
            const uint32_t row = n0 + r, col = k0 + kk;
            float v = 0.0f;
            if (row < n && col < k) {
                if (kn)
                    v = fp8Value(b.data[col * b.stride + row], b.type == TCC_E4M3) *
                        scaleValue(b.scales[uint64_t(col >> b.rowShift) * nBlocks + row / kBlock]);
                else
                    v = fp8Value(b.data[row * b.stride + col], b.type == TCC_E4M3) *
                        scaleValue(b.scales[uint64_t(row >> b.rowShift) * kBlocks + col / kBlock]);
            }
            bs[kk][r] = v;
        }
        __syncthreads();
#pragma unroll 8
        for (int kk = 0; kk < kStep; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fmaf(as[kk][ty * 4 + i], bs[kk][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t row = m0 + ty * 4 + i, col = n0 + tx + 16 * j;
            if (row < m && col < n)
                out[row * outStride + col] = fromFloat<T>(acc[i][j] + (bias ? bias[col] : 0.0f));
        }
}

template <typename T> void launchGeneric(const Product& p) {
    const uint32_t tilesN = ceilDiv<uint32_t>(p.n, kTile);
    const uint64_t grid = uint64_t(ceilDiv<uint32_t>(p.m, kTile)) * tilesN;
    require(grid <= 0x7FFFFFFFull, "too many output tiles for one call");
    productGeneric<T><<<uint32_t(grid), 256, 0, p.stream>>>(p.a, p.b, p.kn, p.bias, static_cast<T*>(p.out), p.outStride,
                                                            p.m, p.n, p.k, tilesN);
    checkCudaCall(cudaGetLastError());
}

void launchProduct(const Product& p) {
    switch (p.outType) {
    case TCC_F32: launchGeneric<float>(p); break;
    case TCC_BF16: launchGeneric<__nv_bfloat16>(p); break;
    default: launchGeneric<__half>(p); break;
    }
}

} // namespace

uint32_t matmulDeviceStatus(bool) { return 0; }

} // namespace tcc

extern "C" {

int tcc_matmul_fp8_blocks(const void* a, int a_type, uint64_t a_stride, const uint8_t* a_scales, uint32_t a_block_rows,
                          const void* b, int b_type, uint64_t b_stride, const uint8_t* b_scales, uint32_t b_block_rows,
                          int b_layout, const float* bias, void* output, int output_type, uint64_t output_stride,
                          uint32_t m, uint32_t n, uint32_t k, tcc_stream_t stream) {
    using namespace tcc;
    return guarded([&] {
        require(isFp8Type(a_type) && isFp8Type(b_type), "matmul_fp8_blocks multiplies e4m3 or e5m2");
        require(isFloatType(output_type), "matmul_fp8_blocks writes fp32, bf16 or fp16");
        require((a_block_rows == 1 || a_block_rows == 128) && (b_block_rows == 1 || b_block_rows == 128),
                "block rows must be 1 or 128");
        require(b_layout == TCC_B_NK || b_layout == TCC_B_KN, "unknown layout of b");
        require(b_layout == TCC_B_NK || b_block_rows == 128, "a [k, n] operand needs blocks of 128 x 128");
        if (m == 0 || n == 0)
            return;
        const bool kn = b_layout == TCC_B_KN;
        require(output != nullptr, "matmul_fp8_blocks requires an output");
        require(extentFits(m, n, output_stride, typeBytes(output_type)), "output: stride below n, or too large");
        require(alignedTo(output, typeBytes(output_type)) && alignedTo(bias, 4), "a matrix must be aligned to its element type");
        if (k != 0) {
            require(a != nullptr && b != nullptr && a_scales != nullptr && b_scales != nullptr,
                    "matmul_fp8_blocks requires both operands and their scales");
            require(extentFits(m, k, a_stride, 1), "a: stride below k, or too large");
            require(extentFits(kn ? k : n, kn ? n : k, b_stride, 1), "b: stride below its width, or too large");
        }
        Product p{};
        p.a = {static_cast<const uint8_t*>(a), a_scales, a_stride, a_type, a_block_rows == 128 ? 7u : 0u};
        p.b = {static_cast<const uint8_t*>(b), b_scales, b_stride, b_type, b_block_rows == 128 ? 7u : 0u};
        p.kn = kn;
        p.bias = bias;
        p.out = output;
        p.outStride = output_stride;
        p.outType = output_type;
        p.m = m, p.n = n, p.k = k;
        p.stream = reinterpret_cast<cudaStream_t>(stream);
        launchProduct(p);
    });
}

} // extern "C"
