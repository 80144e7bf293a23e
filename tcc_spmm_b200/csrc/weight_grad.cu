// Weight gradient of a linear layer whose input was kept as an INT8 checkpoint, on sm_100a:
//   dW[n, k] (+)= sum over rows r of dy[r, n] * q[r, k] 2^e[r, k / 128]
#include "dense8.cuh"
#include "dense8.hpp"

namespace tcc {
namespace {

using namespace blk;

struct Grad {
    const void* dy;
    uint64_t dyStride;
    int type;
    const uint8_t* q;
    uint64_t qStride;
    const uint8_t* scales;
    float* dw;
    uint64_t dwStride;
    uint32_t rows, n, k;
    bool accumulate;
    float* partials;
    cudaStream_t stream;
};

// How the sum over the rows is split: `splits` ranges of rowsPerSplit rows, one CTA per range and
// output tile. More than one range leaves partial matrices, which sumPartials adds in order.
struct Plan {
    uint32_t tilesN, tilesK, splits, rowsPerSplit;
};
constexpr uint32_t kTile = 64, kRowStep = 32;

Plan planOf(uint32_t rows, uint32_t n, uint32_t k) {
    Plan p{};
    p.tilesN = ceilDiv(n, kTile);
    p.tilesK = ceilDiv(k, kTile);
    const uint64_t tiles = uint64_t(p.tilesN) * p.tilesK;
    const uint32_t steps = std::max(1u, ceilDiv(rows, kRowStep));
    const uint64_t want = std::max<uint64_t>(1, 592 / tiles);
    const uint32_t stepsPerSplit = std::max<uint32_t>(4, ceilDiv<uint64_t>(steps, want));
    p.rowsPerSplit = stepsPerSplit * kRowStep;
    p.splits = ceilDiv(steps, stepsPerSplit);
    return p;
}
uint64_t workspaceBytes(const Plan& p, uint32_t n, uint32_t k) {
    return p.splits > 1 ? uint64_t(p.splits) * n * k * 4 : 0;
}

template <typename T>
__global__ void __launch_bounds__(256)
    gradGeneric(const T* __restrict__ dy, uint64_t dyStride, const uint8_t* __restrict__ q, uint64_t qStride,
                const uint8_t* __restrict__ scales, float* out, uint64_t outStride, uint64_t splitStride, uint32_t rows,
                uint32_t n, uint32_t k, uint32_t tilesN, uint32_t tilesK, uint32_t rowsPerSplit, bool accumulate) {
    __shared__ float as[kRowStep][kTile + 1], bs[kRowStep][kTile + 1];
    const uint32_t split = blockIdx.x / (tilesN * tilesK), tile = blockIdx.x % (tilesN * tilesK);
    const uint32_t n0 = tile / tilesK * kTile, k0 = tile % tilesK * kTile;
    const uint32_t kBlocks = (k + kBlock - 1) / kBlock;
    const uint64_t begin = uint64_t(split) * rowsPerSplit;
    const uint64_t end = min(uint64_t(rows), begin + rowsPerSplit);
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (uint64_t r0 = begin; r0 < end; r0 += kRowStep) {
        for (uint32_t i = threadIdx.x; i < kRowStep * kTile; i += 256) {
            const uint32_t rr = i / kTile, c = i % kTile;
            const uint64_t r = r0 + rr;
            as[rr][c] = r < end && n0 + c < n ? toFloat(dy[r * dyStride + n0 + c]) : 0.0f;
            bs[rr][c] = r < end && k0 + c < k ? float(int8_t(q[r * qStride + k0 + c])) *
                                                    scaleValue(scales[r * kBlocks + (k0 + c) / kBlock])
                                              : 0.0f;
        }
        __syncthreads();
#pragma unroll 8
        for (uint32_t rr = 0; rr < kRowStep; ++rr)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fmaf(as[rr][ty * 4 + i], bs[rr][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    float* o = out + split * splitStride;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t r = n0 + ty * 4 + i, c = k0 + tx + 16 * j;
            if (r < n && c < k)
                o[r * outStride + c] = acc[i][j] + (accumulate ? o[r * outStride + c] : 0.0f);
        }
}

// dW (+)= the partial matrices, added in the order of their row ranges.
__global__ void __launch_bounds__(256) sumPartials(const float* __restrict__ partials, uint32_t splits, uint64_t count,
                                                   float* __restrict__ dw, uint64_t dwStride, uint32_t k, bool accumulate) {
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += uint64_t(gridDim.x) * 256) {
        float sum = 0.0f;
        for (uint32_t s = 0; s < splits; ++s)
            sum += partials[s * count + i];
        float* o = dw + i / k * dwStride + i % k;
        *o = accumulate ? *o + sum : sum;
    }
}

template <typename T> void launchGeneric(const Grad& g, const Plan& p) {
    const uint64_t grid = uint64_t(p.tilesN) * p.tilesK * p.splits;
    require(grid <= 0x7FFFFFFFull, "too many output tiles for one call");
    const uint64_t count = uint64_t(g.n) * g.k;
    const bool split = p.splits > 1;
    gradGeneric<T><<<uint32_t(grid), 256, 0, g.stream>>>(
        static_cast<const T*>(g.dy), g.dyStride, g.q, g.qStride, g.scales, split ? g.partials : g.dw,
        split ? uint64_t(g.k) : g.dwStride, split ? count : 0, g.rows, g.n, g.k, p.tilesN, p.tilesK, p.rowsPerSplit,
        !split && g.accumulate);
    checkCudaCall(cudaGetLastError());
    if (split) {
        sumPartials<<<uint32_t(std::min<uint64_t>(ceilDiv<uint64_t>(count, 256), 1184)), 256, 0, g.stream>>>(
            g.partials, p.splits, count, g.dw, g.dwStride, g.k, g.accumulate);
        checkCudaCall(cudaGetLastError());
    }
}

} // namespace

uint32_t weightGradDeviceStatus(bool) { return 0; }

} // namespace tcc

extern "C" {

int tcc_weight_grad_int8_workspace_size(uint32_t rows, uint32_t n, uint32_t k, uint64_t* bytes) {
    using namespace tcc;
    return guarded([&] {
        require(bytes != nullptr, "workspace size requires an output");
        *bytes = n == 0 || k == 0 ? 0 : workspaceBytes(planOf(rows, n, k), n, k);
    });
}

int tcc_weight_grad_int8(const void* grad_y, int type, uint64_t grad_y_stride, const int8_t* q, uint64_t q_stride,
                         const uint8_t* scales, float* grad_w, uint64_t grad_w_stride, uint32_t rows, uint32_t n,
                         uint32_t k, int accumulate, void* workspace, uint64_t workspace_bytes, tcc_stream_t stream) {
    using namespace tcc;
    return guarded([&] {
        require(isFloatType(type), "weight_grad_int8 reads a gradient in fp32, bf16 or fp16");
        if (n == 0 || k == 0)
            return;
        require(grad_w != nullptr && alignedTo(grad_w, 4), "weight_grad_int8 requires an aligned grad_w");
        require(extentFits(n, k, grad_w_stride, 4), "grad_w: stride below k, or too large");
        if (rows != 0) {
            require(grad_y != nullptr && q != nullptr && scales != nullptr,
                    "weight_grad_int8 requires grad_y and the checkpoint");
            require(alignedTo(grad_y, typeBytes(type)), "a matrix must be aligned to its element type");
            require(extentFits(rows, n, grad_y_stride, typeBytes(type)), "grad_y: stride below n, or too large");
            require(extentFits(rows, k, q_stride, 1), "q: stride below k, or too large");
        }
        const Plan p = planOf(rows, n, k);
        require(workspaceBytes(p, n, k) == 0 ||
                    (workspace != nullptr && workspace_bytes >= workspaceBytes(p, n, k) && alignedTo(workspace, 16)),
                "weight_grad_int8 needs a 16-byte aligned workspace of weight_grad_int8_workspace_size bytes");
        const Grad g{grad_y, grad_y_stride, type, reinterpret_cast<const uint8_t*>(q), q_stride, scales, grad_w,
                     grad_w_stride, rows, n, k, accumulate != 0, static_cast<float*>(workspace),
                     reinterpret_cast<cudaStream_t>(stream)};
        switch (type) {
        case TCC_F32: launchGeneric<float>(g, p); break;
        case TCC_BF16: launchGeneric<__nv_bfloat16>(g, p); break;
        default: launchGeneric<__half>(g, p); break;
        }
    });
}

} // extern "C"
