// Elementwise operators over 8-bit blocks on sm_100a: the quantizer to 8-bit floating point, the
// INT8 checkpoint of an activation function's input, and the function's gradient from it.
//
// All three read their input once and write their outputs once, so HBM bounds them. In the kernels
// over rows 8 lanes own one block of 128 columns: lane j takes its 16-byte pieces j, j + 8, ..., so
// that every load and store of a warp covers whole sectors, the block stays in registers between
// the absmax (three shuffles) and the rounding, and nothing is read twice. The 128 x 128 blocks of
// weights take one CTA each, held in registers the same way.
//
// Measured on 8192 x 4096 (bytes read and written once per second; a plain copy reaches 6.5 TB/s): fp32
// checkpoints and gradients 6.2 to 6.4 TB/s for every function; in bf16, where a third of the bytes
// carries as much arithmetic, ReLU 6.2 and 5.8 TB/s, SiLU 5.8 and 5.5, GELU 4.7 and 4.8 (35 us each way),
// which the arithmetic pipes bound; quantizers 5.4 to 7.4 (fp32 rows) TB/s.
#include "dense8.cuh"
#include "dense8.hpp"

namespace tcc {
namespace {

using namespace blk;

constexpr uint32_t kThreads = 256;
constexpr uint32_t kGroup = 8;                         // lanes per block of 128 columns
constexpr uint32_t kGroups = kThreads / kGroup;        // blocks per CTA

// The row and column block of a CTA's group. blocks = rows * column blocks; 32-bit arithmetic
// wherever it reaches.
struct Place {
    uint64_t row;
    uint32_t col;
    bool active;
};
__device__ __forceinline__ Place placeOf(uint64_t blocks, uint32_t colBlocks) {
    const uint64_t g = uint64_t(blockIdx.x) * kGroups + threadIdx.x / kGroup;
    Place p;
    p.active = g < blocks;
    uint32_t c;
    if (blocks <= 0xFFFFFFFFull) {
        const uint32_t r = uint32_t(g) / colBlocks;
        p.row = r;
        c = uint32_t(g) - r * colBlocks;
    } else {
        p.row = g / colBlocks;
        c = uint32_t(g - p.row * colBlocks);
    }
    p.col = c * kBlock;
    return p;
}

// 16 bytes from or to an address that is `align` bytes aligned (16, 8 or 4; the same in every thread).
__device__ __forceinline__ uint4 loadWords16(const void* p, uint32_t align) {
    if (align >= 16)
        return __ldcs(reinterpret_cast<const uint4*>(p));
    if (align == 8) {
        const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p)), b = __ldcs(reinterpret_cast<const uint2*>(p) + 1);
        return make_uint4(a.x, a.y, b.x, b.y);
    }
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
    return make_uint4(__ldcs(w), __ldcs(w + 1), __ldcs(w + 2), __ldcs(w + 3));
}
__device__ __forceinline__ void storeWords16(void* p, uint4 v, uint32_t align) {
    if (align >= 16) {
        __stcs(reinterpret_cast<uint4*>(p), v);
    } else if (align == 8) {
        __stcs(reinterpret_cast<uint2*>(p), make_uint2(v.x, v.y));
        __stcs(reinterpret_cast<uint2*>(p) + 1, make_uint2(v.z, v.w));
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(p);
        __stcs(w, v.x), __stcs(w + 1, v.y), __stcs(w + 2, v.z), __stcs(w + 3, v.w);
    }
}

// One lane's share of a block of x: pieces of 16 bytes (kPer16 elements), piece i at column
// kPer16 * (8 i + lane), as they were loaded. Columns at or beyond `left` read as zero.
template <typename T> struct Share {
    static constexpr int kElems = kPer16<T>;
    static constexpr int kPieces = kBlock / kGroup / kElems;
    uint4 raw[kPieces];
    static __device__ __forceinline__ uint32_t column(int i, uint32_t lane) { return kElems * (kGroup * i + lane); }
    __device__ __forceinline__ void load(const T* row, uint32_t left, uint32_t lane, uint32_t align) {
        if (align >= 16 && left >= kBlock) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                raw[i] = __ldcs(reinterpret_cast<const uint4*>(row + column(i, lane)));
            return;
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint32_t c = column(i, lane);
            if (align >= 4 && c + kElems <= left) {
                raw[i] = loadWords16(row + c, align);
            } else {
                float v[kElems];
#pragma unroll
                for (int e = 0; e < kElems; ++e)
                    v[e] = c + e < left ? toFloat(row[c + e]) : 0.0f;
                raw[i] = pack16<T>(v); // exact: the values have type T
            }
        }
    }
    // Piece i of a row of T.
    static __device__ __forceinline__ void store(T* row, int i, const float (&v)[kElems], uint32_t left, uint32_t lane,
                                                 uint32_t align) {
        const uint32_t c = column(i, lane);
        if (align >= 16 && left >= kBlock) {
            __stcs(reinterpret_cast<uint4*>(row + c), pack16<T>(v));
        } else if (align >= 4 && c + kElems <= left) {
            storeWords16(row + c, pack16<T>(v), align);
        } else {
#pragma unroll
            for (int e = 0; e < kElems; ++e)
                if (c + e < left)
                    row[c + e] = fromFloat<T>(v[e]);
        }
    }
};

// Stores the 8-bit elements of one piece (4 or 8 of them) at q.
template <int N>
__device__ __forceinline__ void storeBytes(uint8_t* q, const uint32_t (&w)[N / 4], uint32_t left, bool vector) {
    if (vector && left >= uint32_t(N)) {
        if constexpr (N == 8)
            *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(q) = w[0];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (uint32_t(e) < left)
                q[e] = uint8_t(w[e / 4] >> (8 * (e % 4)));
    }
}

// Blocks of 128 columns of a row: q and the scale of x and, with A != kNone, y = f(x).
template <typename T, int Q, int A>
__global__ void __launch_bounds__(kThreads)
    quantizeRowBlocks(const T* x, uint64_t xStride, T* y, uint64_t yStride, uint8_t* __restrict__ q, uint64_t qStride,
                      uint8_t* __restrict__ scales, uint64_t blocks, uint32_t cols, uint32_t colBlocks, uint32_t alignX,
                      uint32_t alignY, bool vectorQ) {
    const uint32_t lane = threadIdx.x % kGroup;
    const Place p = placeOf(blocks, colBlocks);
    const uint32_t left = p.active ? cols - p.col : 0u;
    Share<T> s;
    s.load(x + p.row * xStride + p.col, left, lane, alignX);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < Share<T>::kPieces; ++i)
        top = absmax16<T>(s.raw[i], top);
    top = absmaxBits<T>(top);
#pragma unroll
    for (int offset = kGroup / 2; offset > 0; offset >>= 1)
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
    if (!p.active)
        return;
    const uint32_t byte = scaleByte<Q>(top);
    const float inverse = inverseScale(byte);
    uint8_t* qRow = q + p.row * qStride + p.col;
    if (lane == 0)
        scales[p.row * colBlocks + p.col / kBlock] = uint8_t(byte);
#pragma unroll
    for (int i = 0; i < Share<T>::kPieces; ++i) {
        constexpr int kE = Share<T>::kElems;
        float v[kE];
        unpack16<T>(s.raw[i], v);
        uint32_t w[kE / 4];
#pragma unroll
        for (int h = 0; h < kE / 4; ++h)
            w[h] = byte == 255u ? nanBytes<Q>()
                                : quantize4<Q>(v[4 * h] * inverse, v[4 * h + 1] * inverse, v[4 * h + 2] * inverse,
                                               v[4 * h + 3] * inverse);
        const uint32_t c = Share<T>::column(i, lane);
        storeBytes<kE>(qRow + c, w, left > c ? left - c : 0u, vectorQ);
        if constexpr (A != kNone) {
#pragma unroll
            for (int e = 0; e < kE; e += 2)
                activation<A>(v[e], v[e + 1]);
            Share<T>::store(y + p.row * yStride + p.col, i, v, left, lane, alignY);
        }
    }
}

// Blocks of 128 x 128 elements: one CTA each. Lane groups of a row's 128 columns (16 bytes per
// lane) walk down the block's rows; the raw words stay in registers.
template <typename T, int Q>
__global__ void __launch_bounds__(kThreads)
    quantizeSquareBlocks(const T* __restrict__ x, uint64_t xStride, uint8_t* __restrict__ q, uint64_t qStride,
                         uint8_t* __restrict__ scales, uint32_t rows, uint32_t cols, uint32_t colBlocks, uint32_t alignX,
                         bool vectorQ) {
    constexpr int kE = kPer16<T>;
    constexpr uint32_t kLanes = kBlock / kE;               // lanes per row: 32 (fp32) or 16
    constexpr uint32_t kRowsPerPass = kThreads / kLanes;
    constexpr int kPasses = kBlock / kRowsPerPass;
    const uint32_t rowBlock = blockIdx.x / colBlocks, colBlock = blockIdx.x % colBlocks;
    const uint32_t c = colBlock * kBlock + (threadIdx.x % kLanes) * kE;
    const uint32_t r0 = rowBlock * kBlock + threadIdx.x / kLanes;
    uint4 raw[kPasses];
    uint32_t top = 0;
    if (alignX >= 16 && (rowBlock + 1) * uint64_t(kBlock) <= rows && (colBlock + 1) * uint64_t(kBlock) <= cols) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i)
            raw[i] = __ldcs(reinterpret_cast<const uint4*>(x + (uint64_t(r0) + i * kRowsPerPass) * xStride + c));
    } else {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const uint64_t r = uint64_t(r0) + i * kRowsPerPass;
            const T* src = x + r * xStride + c;
            if (r < rows && alignX >= 4 && c + kE <= cols) {
                raw[i] = loadWords16(src, alignX);
            } else {
                float v[kE];
#pragma unroll
                for (int e = 0; e < kE; ++e)
                    v[e] = r < rows && c + e < cols ? toFloat(src[e]) : 0.0f;
                raw[i] = pack16<T>(v); // exact: the values have type T
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
        top = absmax16<T>(raw[i], top);
    top = absmaxBits<T>(top);
    __shared__ uint32_t tops[kThreads / 32];
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (threadIdx.x % 32 == 0)
        tops[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kThreads / 32; ++i)
        top = max(top, tops[i]);
    const uint32_t byte = scaleByte<Q>(top);
    const float inverse = inverseScale(byte);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const uint64_t r = uint64_t(r0) + i * kRowsPerPass;
        float v[kE];
        unpack16<T>(raw[i], v);
        uint32_t w[kE / 4];
#pragma unroll
        for (int h = 0; h < kE / 4; ++h)
            w[h] = byte == 255u ? nanBytes<Q>()
                                : quantize4<Q>(v[4 * h] * inverse, v[4 * h + 1] * inverse, v[4 * h + 2] * inverse,
                                               v[4 * h + 3] * inverse);
        if (r < rows)
            storeBytes<kE>(q + r * qStride + c, w, cols > c ? cols - c : 0u, vectorQ);
    }
    if (threadIdx.x == 0)
        scales[blockIdx.x] = uint8_t(byte);
}

// dx = dy * f'(q 2^e), blocks of 128 columns of a row. dx may be dy itself.
template <typename T, int A>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 8 : 6) // warps for latency: 37 -> 35 us with 8 in bf16
    activationBackward(const T* dy, uint64_t dyStride, const uint8_t* __restrict__ q, uint64_t qStride,
                       const uint8_t* __restrict__ scales, T* dx, uint64_t dxStride, uint64_t blocks, uint32_t cols,
                       uint32_t colBlocks, uint32_t alignDy, uint32_t alignDx, bool vectorQ) {
    constexpr int kE = Share<T>::kElems;
    const uint32_t lane = threadIdx.x % kGroup;
    const Place p = placeOf(blocks, colBlocks);
    if (!p.active)
        return;
    const uint32_t left = cols - p.col;
    const float scale = scaleValue(scales[p.row * colBlocks + p.col / kBlock]);
    const uint8_t* qRow = q + p.row * qStride + p.col;
    uint32_t w[Share<T>::kPieces][kE / 4];
#pragma unroll
    for (int i = 0; i < Share<T>::kPieces; ++i) {
        const uint32_t c = kE * (kGroup * i + lane);
        if (vectorQ && c + kE <= left) {
            if constexpr (kE == 8) {
                const uint2 t = __ldcs(reinterpret_cast<const uint2*>(qRow + c));
                w[i][0] = t.x, w[i][1] = t.y;
            } else {
                w[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(qRow + c));
            }
        } else {
#pragma unroll
            for (int h = 0; h < kE / 4; ++h) {
                w[i][h] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + 4 * h + e < left)
                        w[i][h] |= uint32_t(qRow[c + 4 * h + e]) << (8 * e);
            }
        }
    }
    Share<T> s;
    s.load(dy + p.row * dyStride + p.col, left, lane, alignDy);
#pragma unroll
    for (int i = 0; i < Share<T>::kPieces; ++i) {
        float v[kE];
        unpack16<T>(s.raw[i], v);
#pragma unroll
        for (int e = 0; e < kE; e += 2) {
            const uint32_t flipped = w[i][e / 4] ^ 0x80808080u;
            float f = int8At(flipped, e % 4) * scale, g = int8At(flipped, e % 4 + 1) * scale;
            activationSlope<A>(f, g);
            v[e] *= f, v[e + 1] *= g;
        }
        Share<T>::store(dx + p.row * dxStride + p.col, i, v, left, lane, alignDx);
    }
}

uint32_t rowGrid(uint64_t blocks) {
    const uint64_t grid = ceilDiv<uint64_t>(blocks, kGroups);
    require(grid <= 0x7FFFFFFFull, "too many blocks for one call");
    return uint32_t(grid);
}

// Bytes (16, 8, 4, or 0 for less) on which every row of a matrix starts.
uint32_t alignmentOf(const void* p, uint64_t strideBytes) {
    return rowsAlignedTo(p, strideBytes, 16) ? 16 : rowsAlignedTo(p, strideBytes, 8) ? 8 : rowsAlignedTo(p, strideBytes, 4) ? 4 : 0;
}

// Bytes that a lane stores or loads of q at once: 4 (fp32) or 8.
uint32_t pieceBytes(int type) { return type == TCC_F32 ? 4 : 8; }

struct RowArgs {
    const void* x;
    uint64_t xStride;
    void* y;
    uint64_t yStride;
    uint8_t* q;
    uint64_t qStride;
    uint8_t* scales;
    uint32_t rows, cols;
    cudaStream_t stream;
};

template <typename T, int Q, int A> void launchRows(const RowArgs& a, int type) {
    const uint32_t colBlocks = ceilDiv(a.cols, kBlock);
    const uint64_t blocks = uint64_t(a.rows) * colBlocks;
    const uint64_t size = typeBytes(type);
    quantizeRowBlocks<T, Q, A><<<rowGrid(blocks), kThreads, 0, a.stream>>>(
        static_cast<const T*>(a.x), a.xStride, static_cast<T*>(a.y), a.yStride, a.q, a.qStride, a.scales, blocks, a.cols,
        colBlocks, alignmentOf(a.x, a.xStride * size), alignmentOf(a.y, a.yStride * size),
        rowsAlignedTo(a.q, a.qStride, pieceBytes(type)));
    checkCudaCall(cudaGetLastError());
}

template <typename T, int Q> void launchSquares(const RowArgs& a, int type) {
    const uint32_t colBlocks = ceilDiv(a.cols, kBlock);
    const uint64_t blocks = uint64_t(ceilDiv(a.rows, kBlock)) * colBlocks;
    require(blocks <= 0x7FFFFFFFull, "too many blocks for one call");
    quantizeSquareBlocks<T, Q><<<uint32_t(blocks), kThreads, 0, a.stream>>>(
        static_cast<const T*>(a.x), a.xStride, a.q, a.qStride, a.scales, a.rows, a.cols, colBlocks,
        alignmentOf(a.x, a.xStride * typeBytes(type)), rowsAlignedTo(a.q, a.qStride, pieceBytes(type)));
    checkCudaCall(cudaGetLastError());
}

// Calls f(T{}) with the element type of a tcc_type.
template <typename F> void withType(int type, F&& f) {
    switch (type) {
    case TCC_F32: f(float{}); break;
    case TCC_BF16: f(__nv_bfloat16{}); break;
    default: f(__half{}); break;
    }
}
template <int V> struct Const { static constexpr int value = V; };
template <typename F> void withActivation(int activation, F&& f) {
    switch (activation) {
    case TCC_RELU: f(Const<kRelu>{}); break;
    case TCC_GELU: f(Const<kGelu>{}); break;
    case TCC_GELU_TANH: f(Const<kGeluTanh>{}); break;
    case TCC_SILU: f(Const<kSilu>{}); break;
    default: f(Const<kNone>{}); break;
    }
}

void checkMatrix(const void* p, uint64_t stride, uint32_t rows, uint32_t cols, uint32_t elementBytes, const char* null,
                 const char* extent) {
    require(p != nullptr, null);
    require(extentFits(rows, cols, stride, elementBytes), extent);
    require(alignedTo(p, elementBytes), "a matrix must be aligned to its element type");
}

} // namespace
} // namespace tcc

extern "C" {

int tcc_quantize_blocks_fp8(const void* x, int x_type, uint64_t x_stride, void* q, int q_type, uint64_t q_stride,
                            uint8_t* scales, uint32_t rows, uint32_t cols, uint32_t block_rows, tcc_stream_t stream) {
    using namespace tcc;
    return guarded([&] {
        require(isFloatType(x_type), "quantize_blocks_fp8 reads fp32, bf16 or fp16");
        require(isFp8Type(q_type), "quantize_blocks_fp8 writes e4m3 or e5m2");
        require(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128");
        if (rows == 0 || cols == 0)
            return;
        checkMatrix(x, x_stride, rows, cols, typeBytes(x_type), "quantize_blocks_fp8 requires x", "x: stride below cols, or too large");
        checkMatrix(q, q_stride, rows, cols, 1, "quantize_blocks_fp8 requires q", "q: stride below cols, or too large");
        require(scales != nullptr, "quantize_blocks_fp8 requires scales");
        const RowArgs a{x, x_stride, nullptr, 0, static_cast<uint8_t*>(q), q_stride, scales, rows, cols,
                        reinterpret_cast<cudaStream_t>(stream)};
        withType(x_type, [&](auto t) {
            using T = decltype(t);
            if (block_rows == 1)
                q_type == TCC_E4M3 ? launchRows<T, kE4M3, kNone>(a, x_type) : launchRows<T, kE5M2, kNone>(a, x_type);
            else
                q_type == TCC_E4M3 ? launchSquares<T, kE4M3>(a, x_type) : launchSquares<T, kE5M2>(a, x_type);
        });
    });
}

int tcc_activation_checkpoint_int8(const void* x, uint64_t x_stride, void* y, uint64_t y_stride, int type, int8_t* q,
                                   uint64_t q_stride, uint8_t* scales, uint32_t rows, uint32_t cols, int activation,
                                   tcc_stream_t stream) {
    using namespace tcc;
    return guarded([&] {
        require(isFloatType(type), "activation_checkpoint_int8 takes fp32, bf16 or fp16");
        require(activation >= TCC_RELU && activation <= TCC_IDENTITY, "unknown activation");
        if (rows == 0 || cols == 0)
            return;
        checkMatrix(x, x_stride, rows, cols, typeBytes(type), "activation_checkpoint_int8 requires x", "x: stride below cols, or too large");
        checkMatrix(q, q_stride, rows, cols, 1, "activation_checkpoint_int8 requires q", "q: stride below cols, or too large");
        require(scales != nullptr, "activation_checkpoint_int8 requires scales");
        if (activation == TCC_IDENTITY)
            require(y == nullptr, "the identity writes no y: pass a null y");
        else
            checkMatrix(y, y_stride, rows, cols, typeBytes(type), "activation_checkpoint_int8 requires y", "y: stride below cols, or too large");
        const RowArgs a{x, x_stride, y, y_stride, reinterpret_cast<uint8_t*>(q), q_stride, scales, rows, cols,
                        reinterpret_cast<cudaStream_t>(stream)};
        withType(type, [&](auto t) {
            withActivation(activation, [&](auto f) { launchRows<decltype(t), kInt8, decltype(f)::value>(a, type); });
        });
    });
}

int tcc_activation_backward_int8(const void* grad_y, uint64_t grad_y_stride, int type, const int8_t* q,
                                 uint64_t q_stride, const uint8_t* scales, void* grad_x, uint64_t grad_x_stride,
                                 uint32_t rows, uint32_t cols, int activation, tcc_stream_t stream) {
    using namespace tcc;
    return guarded([&] {
        require(isFloatType(type), "activation_backward_int8 takes fp32, bf16 or fp16");
        require(activation >= TCC_RELU && activation < TCC_IDENTITY, "unknown activation");
        if (rows == 0 || cols == 0)
            return;
        checkMatrix(grad_y, grad_y_stride, rows, cols, typeBytes(type), "activation_backward_int8 requires grad_y", "grad_y: stride below cols, or too large");
        checkMatrix(grad_x, grad_x_stride, rows, cols, typeBytes(type), "activation_backward_int8 requires grad_x", "grad_x: stride below cols, or too large");
        checkMatrix(q, q_stride, rows, cols, 1, "activation_backward_int8 requires q", "q: stride below cols, or too large");
        require(scales != nullptr, "activation_backward_int8 requires scales");
        const uint32_t colBlocks = ceilDiv(cols, kBlock);
        const uint64_t blocks = uint64_t(rows) * colBlocks, size = typeBytes(type);
        withType(type, [&](auto t) {
            using T = decltype(t);
            withActivation(activation, [&](auto f) {
                if constexpr (decltype(f)::value != kNone) {
                    activationBackward<T, decltype(f)::value><<<rowGrid(blocks), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                        static_cast<const T*>(grad_y), grad_y_stride, reinterpret_cast<const uint8_t*>(q), q_stride,
                        scales, static_cast<T*>(grad_x), grad_x_stride, blocks, cols, colBlocks,
                        alignmentOf(grad_y, grad_y_stride * size), alignmentOf(grad_x, grad_x_stride * size),
                        rowsAlignedTo(q, q_stride, pieceBytes(type)));
                    checkCudaCall(cudaGetLastError());
                }
            });
        });
    });
}

} // extern "C"
