// Elementwise operators over 8-bit blocks on sm_100a: the quantizer to 8-bit floating point, the
// INT8 checkpoint of an activation function's input, and the function's gradient from it.
//
// All three read their input once and write their outputs once, so HBM bounds them. In the kernels
// over rows 8 lanes own one block of 128 columns: lane j takes its 16-byte pieces j, j + 8, ... (or
// shorter runs, where rows are not aligned to 16 bytes), so that a warp's loads and stores cover whole
// sectors, the block stays in registers between
// the absmax (three shuffles) and the rounding, and nothing is read twice. The 128 x 128 blocks of
// weights take one CTA each, held in registers the same way.
//
// Measured on 8192 x 4096 (bytes read and written once per second; a plain copy reaches 6.5 TB/s): fp32
// checkpoints and gradients 6.2 to 6.4 TB/s for every function; in bf16, where a third of the bytes
// carries as much arithmetic, ReLU 6.2 and 5.8 TB/s, SiLU 5.8 and 5.5, GELU 4.7 and 4.8 (35 us each way). No pipe is
// full there: a CTA's loads, arithmetic and stores follow one another, instructions issue in 75% of the active cycles
// and 11% of the time an SM has no CTA. Quantizers 5.4 to 7.4 (fp32 rows) TB/s.
#include "dense8.cuh"
#include "dense8.hpp"

#include <type_traits>

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

// A lane's N elements of a row of a block: runs of W neighbouring elements, run i at column
// W * (LANES * i + lane), so that a warp's stores stay together whatever W is. W is the most that the
// alignment of the rows that are written allows, 16 bytes of T at best: storing 16 neighbouring bytes per
// lane element by element took the checkpoint of 8192 x 4101 bf16 177 us, runs of one element take 79 us.
template <typename T, int W, int LANES, int N> struct Runs {
    static constexpr int kElems = kPer16<T>, kBytes = W * int(sizeof(T)), kWords = N * int(sizeof(T)) / 4;
    static constexpr int kPerPiece = kElems / W; // runs of 16 bytes of T, in which the kernels compute
    using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, unsigned short>;
    static __device__ __forceinline__ uint32_t column(int run, uint32_t lane) { return W * (LANES * run + lane); }
    // Element n of `words`.
    template <int WORDS> static __device__ __forceinline__ void put(uint32_t (&words)[WORDS], int n, uint32_t bits) {
        if constexpr (sizeof(T) == 4)
            words[n] = bits;
        else
            words[n / 2] = n % 2 == 0 ? bits : words[n / 2] | (bits << 16);
    }
    // The elements of a row of which `left` columns are inside, zeros behind them. whole: all are inside.
    // The row starts on `align` bytes; a run comes in accesses as wide as that allows.
    static __device__ __forceinline__ void load(const T* row, uint32_t left, bool whole, uint32_t lane, uint32_t align,
                                                uint32_t (&raw)[kWords]) {
        if (align >= uint32_t(kBytes))
            loadAll<kBytes>(row, left, whole, lane, raw);
        else if (kBytes > 8 && align == 8)
            loadAll<(kBytes > 8 ? 8 : kBytes)>(row, left, whole, lane, raw);
        else if (kBytes > 4 && align == 4)
            loadAll<(kBytes > 4 ? 4 : kBytes)>(row, left, whole, lane, raw);
        else
            loadAll<int(sizeof(T))>(row, left, whole, lane, raw);
    }
    template <int ACCESS>
    static __device__ __forceinline__ void loadAll(const T* row, uint32_t left, bool whole, uint32_t lane, uint32_t (&raw)[kWords]) {
        if (whole) { // all loads in flight together
#pragma unroll
            for (int run = 0; run < N / W; ++run)
                loadRun<ACCESS>(row + column(run, lane), run, raw);
        } else {
#pragma unroll
            for (int w = 0; w < kWords; ++w)
                raw[w] = 0;
#pragma unroll
            for (int run = 0; run < N / W; ++run)
                if (column(run, lane) + W <= left)
                    loadRun<ACCESS>(row + column(run, lane), run, raw);
            if (W > 1 && left % W != 0) // the run in which the row ends
#pragma unroll
                for (int run = 0; run < N / W; ++run) {
                    const uint32_t c = column(run, lane);
                    if (c < left && left < c + W)
#pragma unroll
                        for (int e = 0; e < W; ++e)
                            put(raw, run * W + e, c + e < left ? uint32_t(reinterpret_cast<const Bits*>(row)[c + e]) : 0u);
                }
        }
    }
    template <int ACCESS> static __device__ __forceinline__ void loadRun(const T* at, int run, uint32_t (&raw)[kWords]) {
#pragma unroll
        for (int a = 0; a < kBytes / ACCESS; ++a) {
            const uint8_t* from = reinterpret_cast<const uint8_t*>(at) + a * ACCESS;
            const int word = (run * kBytes + a * ACCESS) / 4;
            if constexpr (ACCESS == 16) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4*>(from));
                raw[word] = v.x, raw[word + 1] = v.y, raw[word + 2] = v.z, raw[word + 3] = v.w;
            } else if constexpr (ACCESS == 8) {
                const uint2 v = __ldcs(reinterpret_cast<const uint2*>(from));
                raw[word] = v.x, raw[word + 1] = v.y;
            } else if constexpr (ACCESS == 4) {
                raw[word] = __ldcs(reinterpret_cast<const uint32_t*>(from));
            } else {
                put(raw, run * W + a, __ldcs(reinterpret_cast<const unsigned short*>(from)));
            }
        }
    }
    // Whether piece i lies behind the row's end.
    static __device__ __forceinline__ bool behind(int i, uint32_t left) { return column(i * kPerPiece, 0) >= left; }
    static __device__ __forceinline__ uint4 piece(const uint32_t (&raw)[kWords], int i) {
        return make_uint4(raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]);
    }
    // 16 bytes of T (piece i) to a row.
    static __device__ __forceinline__ void store(T* row, uint32_t left, bool whole, uint32_t lane, int i, uint4 v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < kPerPiece; ++j) {
            const uint32_t c = column(i * kPerPiece + j, lane);
            if (whole || c + W <= left) {
                if constexpr (kBytes == 16)
                    __stcs(reinterpret_cast<uint4*>(row + c), v);
                else if constexpr (kBytes == 8)
                    __stcs(reinterpret_cast<uint2*>(row + c), make_uint2(w[2 * j], w[2 * j + 1]));
                else if constexpr (kBytes == 4)
                    __stcs(reinterpret_cast<uint32_t*>(row + c), w[j]);
                else
                    __stcs(reinterpret_cast<unsigned short*>(row + c), static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2))));
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if (c + e < left)
                        reinterpret_cast<Bits*>(row)[c + e] =
                            Bits(sizeof(T) == 4 ? w[(j * W + e) % 4] : w[(j * W + e) / 2 % 4] >> (16 * ((j * W + e) % 2)));
            }
        }
    }
    // The 8-bit elements of piece i, one word per four.
    static __device__ __forceinline__ void storeBytes(uint8_t* row, uint32_t left, bool whole, uint32_t lane, int i,
                                                      const uint32_t (&w)[kElems / 4]) {
#pragma unroll
        for (int j = 0; j < kPerPiece; ++j) {
            const uint32_t c = column(i * kPerPiece + j, lane);
            if (whole || c + W <= left) {
                if constexpr (W == 8)
                    *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
                else if constexpr (W == 4)
                    *reinterpret_cast<uint32_t*>(row + c) = w[j];
                else if constexpr (W == 2)
                    *reinterpret_cast<unsigned short*>(row + c) = static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2)));
                else
                    row[c] = uint8_t(w[j / 4] >> (8 * (j % 4)));
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if (c + e < left)
                        row[c + e] = uint8_t(w[(j * W + e) / 4] >> (8 * ((j * W + e) % 4)));
            }
        }
    }
    static __device__ __forceinline__ void loadBytes(const uint8_t* row, uint32_t left, bool whole, uint32_t lane, int i,
                                                     uint32_t (&w)[kElems / 4]) {
#pragma unroll
        for (int h = 0; h < kElems / 4; ++h)
            w[h] = 0;
#pragma unroll
        for (int j = 0; j < kPerPiece; ++j) {
            const uint32_t c = column(i * kPerPiece + j, lane);
            if (whole || c + W <= left) {
                if constexpr (W == 8) {
                    const uint2 t = __ldcs(reinterpret_cast<const uint2*>(row + c));
                    w[0] = t.x, w[1] = t.y;
                } else if constexpr (W == 4) {
                    w[j] = __ldcs(reinterpret_cast<const uint32_t*>(row + c));
                } else if constexpr (W == 2) {
                    w[j / 2] |= uint32_t(__ldcs(reinterpret_cast<const unsigned short*>(row + c))) << (16 * (j % 2));
                } else {
                    w[j / 4] |= uint32_t(__ldcs(row + c)) << (8 * (j % 4));
                }
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if (c + e < left)
                        w[(j * W + e) / 4] |= uint32_t(row[c + e]) << (8 * ((j * W + e) % 4));
            }
        }
    }
};
template <typename T, int W> using RowRuns = Runs<T, W, int(kGroup), int(kBlock / kGroup)>;

// Blocks of 128 columns of a row: q and the scale of x and, with A != kNone, y = f(x).
template <typename T, int W, int Q, int A>
// GELU in bf16 would take 44 registers: 37 us, 35 us with 40; the quantizer of 8192 x 4096 bf16 takes 19.1 us
// with 40 registers, 17.6 us with 32.
__global__ void __launch_bounds__(kThreads, A == kGelu || sizeof(T) == 4 ? 6 : 8)
    quantizeRowBlocks(const T* x, uint64_t xStride, T* y, uint64_t yStride, uint8_t* __restrict__ q, uint64_t qStride,
                      uint8_t* __restrict__ scales, uint64_t blocks, uint32_t cols, uint32_t colBlocks, uint32_t alignX) {
    using R = RowRuns<T, W>;
    constexpr int kE = R::kElems, kPieces = kBlock / kGroup / kE;
    const uint32_t lane = threadIdx.x % kGroup;
    const Place p = placeOf(blocks, colBlocks);
    const uint32_t left = p.active ? cols - p.col : 0u;
    const bool whole = left >= kBlock;
    uint32_t raw[R::kWords];
    R::load(x + p.row * xStride + p.col, left, whole, lane, alignX, raw);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        top = absmax16<T>(R::piece(raw, i), top);
    top = absmaxBits<T>(top);
#pragma unroll
    for (int offset = kGroup / 2; offset > 0; offset >>= 1)
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
    if (!p.active)
        return;
    const uint32_t byte = scaleByte<Q>(top);
    const float inverse = inverseScale(byte);
    if (lane == 0)
        scales[p.row * colBlocks + p.col / kBlock] = uint8_t(byte);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        if (!whole && R::behind(i, left))
            break;
        float v[kE];
        unpack16<T>(R::piece(raw, i), v);
        uint32_t w[kE / 4];
#pragma unroll
        for (int h = 0; h < kE / 4; ++h)
            w[h] = byte == 255u ? nanBytes<Q>()
                                : quantize4<Q>(v[4 * h] * inverse, v[4 * h + 1] * inverse, v[4 * h + 2] * inverse,
                                               v[4 * h + 3] * inverse);
        R::storeBytes(q + p.row * qStride + p.col, left, whole, lane, i, w);
        if constexpr (A != kNone) {
#pragma unroll
            for (int e = 0; e < kE; e += 2)
                activation<A>(v[e], v[e + 1]);
            R::store(y + p.row * yStride + p.col, left, whole, lane, i, pack16<T>(v));
        }
    }
}

// Blocks of 128 x 128 elements: one CTA each. Lane groups of a row's 128 columns (16 bytes per
// lane) walk down the block's rows; the raw words stay in registers.
template <typename T, int W, int Q>
__global__ void __launch_bounds__(kThreads)
    quantizeSquareBlocks(const T* __restrict__ x, uint64_t xStride, uint8_t* __restrict__ q, uint64_t qStride,
                         uint8_t* __restrict__ scales, uint32_t rows, uint32_t cols, uint32_t colBlocks) {
    constexpr int kE = kPer16<T>;
    constexpr uint32_t kLanes = kBlock / kE;               // lanes per row: 32 (fp32) or 16
    constexpr uint32_t kRowsPerPass = kThreads / kLanes;
    constexpr int kPasses = kBlock / kRowsPerPass;
    using R = Runs<T, W, int(kLanes), kE>;
    const uint32_t rowBlock = blockIdx.x / colBlocks, colBlock = blockIdx.x % colBlocks;
    const uint32_t c = colBlock * kBlock, left = cols - c, lane = threadIdx.x % kLanes;
    const uint32_t r0 = rowBlock * kBlock + threadIdx.x / kLanes;
    const bool wide = left >= kBlock;
    uint32_t raw[kPasses][4], top = 0;
    if (wide && (rowBlock + 1) * uint64_t(kBlock) <= rows) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i)
            R::template loadAll<R::kBytes>(x + (uint64_t(r0) + i * kRowsPerPass) * xStride + c, left, true, lane, raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const uint64_t r = uint64_t(r0) + i * kRowsPerPass;
            R::template loadAll<R::kBytes>(x + r * xStride + c, r < rows ? min(left, kBlock) : 0u, false, lane, raw[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
        top = absmax16<T>(R::piece(raw[i], 0), top);
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
        unpack16<T>(R::piece(raw[i], 0), v);
        uint32_t w[kE / 4];
#pragma unroll
        for (int h = 0; h < kE / 4; ++h)
            w[h] = byte == 255u ? nanBytes<Q>()
                                : quantize4<Q>(v[4 * h] * inverse, v[4 * h + 1] * inverse, v[4 * h + 2] * inverse,
                                               v[4 * h + 3] * inverse);
        if (r < rows)
            R::storeBytes(q + r * qStride + c, left, wide, lane, 0, w);
    }
    if (threadIdx.x == 0)
        scales[blockIdx.x] = uint8_t(byte);
}

// dx = dy * f'(q 2^e), blocks of 128 columns of a row. dx may be dy itself.
template <typename T, int W, int A>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 8 : 6) // warps for latency: 37 -> 35 us with 8 in bf16
    activationBackward(const T* dy, uint64_t dyStride, const uint8_t* __restrict__ q, uint64_t qStride,
                       const uint8_t* __restrict__ scales, T* dx, uint64_t dxStride, uint64_t blocks, uint32_t cols,
                       uint32_t colBlocks, uint32_t alignDy) {
    using R = RowRuns<T, W>;
    constexpr int kE = R::kElems, kPieces = kBlock / kGroup / kE;
    const uint32_t lane = threadIdx.x % kGroup;
    const Place p = placeOf(blocks, colBlocks);
    if (!p.active)
        return;
    const uint32_t left = cols - p.col;
    const bool whole = left >= kBlock;
    const float scale = slopeScale(scales[p.row * colBlocks + p.col / kBlock]);
    uint32_t w[kPieces][kE / 4], raw[R::kWords];
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        R::loadBytes(q + p.row * qStride + p.col, left, whole, lane, i, w[i]);
    R::load(dy + p.row * dyStride + p.col, left, whole, lane, alignDy, raw);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        if (!whole && R::behind(i, left))
            break;
        float v[kE];
        unpack16<T>(R::piece(raw, i), v);
#pragma unroll
        for (int e = 0; e < kE; e += 2) {
            const uint32_t flipped = w[i][e / 4] ^ 0x80808080u;
            float f = int8At(flipped, e % 4) * scale, g = int8At(flipped, e % 4 + 1) * scale;
            activationSlope<A>(f, g);
            v[e] *= f, v[e + 1] *= g;
        }
        R::store(dx + p.row * dxStride + p.col, left, whole, lane, i, pack16<T>(v));
    }
}

uint32_t rowGrid(uint64_t blocks) {
    const uint64_t grid = ceilDiv<uint64_t>(blocks, kGroups);
    require(grid <= 0x7FFFFFFFull, "too many blocks for one call");
    return uint32_t(grid);
}

template <int V> struct Const { static constexpr int value = V; };

// Bytes (16, 8, 4 or 2) on which every row of a matrix starts.
uint32_t alignmentOf(const void* p, uint64_t strideBytes) {
    uint32_t a = 16;
    while (a > 2 && !rowsAlignedTo(p, strideBytes, a))
        a /= 2;
    return a;
}
// The longest run (16 bytes of T, or 4, 2 or 1 elements) on which every row of y (null: no matter) and of the
// 8-bit q starts. Where x is off 16 bytes it is at most 4, and no shorter for x alone: the quantizer of
// 8192 x 4101 bf16 takes 27.1 us with runs of 4 in loads of one element, 42 us with runs of 1. (Blocks of
// 128 x 128 hold more of x at once and take their runs from x and q alike.)
template <typename T> int runOf(const void* y, uint64_t yStride, const void* q, uint64_t qStride, uint32_t alignX) {
    int w = alignX < 16 ? 4 : kPer16<T>;
    while (w > 1 && !((y == nullptr || rowsAlignedTo(y, yStride * sizeof(T), w * sizeof(T))) && rowsAlignedTo(q, qStride, w)))
        w /= 2;
    return w;
}
// Calls f(Const<run>{}).
template <typename T, typename F> void withRun(int run, F&& f) {
    if constexpr (kPer16<T> == 8)
        if (run == 8)
            return f(Const<8>{});
    run == 4 ? f(Const<4>{}) : run == 2 ? f(Const<2>{}) : f(Const<1>{});
}

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

template <typename T, int Q, int A> void launchRows(const RowArgs& a) {
    const uint32_t colBlocks = ceilDiv(a.cols, kBlock);
    const uint64_t blocks = uint64_t(a.rows) * colBlocks;
    const uint32_t grid = rowGrid(blocks);
    const uint32_t alignX = alignmentOf(a.x, a.xStride * sizeof(T));
    withRun<T>(runOf<T>(a.y, a.yStride, a.q, a.qStride, alignX), [&](auto run) {
        quantizeRowBlocks<T, decltype(run)::value, Q, A><<<grid, kThreads, 0, a.stream>>>(
            static_cast<const T*>(a.x), a.xStride, static_cast<T*>(a.y), a.yStride, a.q, a.qStride, a.scales, blocks, a.cols,
            colBlocks, alignX);
    });
    checkCudaCall(cudaGetLastError());
}

template <typename T, int Q> void launchSquares(const RowArgs& a) {
    const uint32_t colBlocks = ceilDiv(a.cols, kBlock);
    const uint64_t blocks = uint64_t(ceilDiv(a.rows, kBlock)) * colBlocks;
    require(blocks <= 0x7FFFFFFFull, "too many blocks for one call");
    withRun<T>(runOf<T>(a.x, a.xStride, a.q, a.qStride, 16), [&](auto run) {
        quantizeSquareBlocks<T, decltype(run)::value, Q><<<uint32_t(blocks), kThreads, 0, a.stream>>>(
            static_cast<const T*>(a.x), a.xStride, a.q, a.qStride, a.scales, a.rows, a.cols, colBlocks);
    });
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
                q_type == TCC_E4M3 ? launchRows<T, kE4M3, kNone>(a) : launchRows<T, kE5M2, kNone>(a);
            else
                q_type == TCC_E4M3 ? launchSquares<T, kE4M3>(a) : launchSquares<T, kE5M2>(a);
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
            withActivation(activation, [&](auto f) { launchRows<decltype(t), kInt8, decltype(f)::value>(a); });
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
        const uint64_t blocks = uint64_t(rows) * colBlocks;
        const uint32_t grid = rowGrid(blocks);
        withType(type, [&](auto t) {
            using T = decltype(t);
            withActivation(activation, [&](auto f) {
                if constexpr (decltype(f)::value != kNone) {
                    const uint32_t alignDy = alignmentOf(grad_y, grad_y_stride * sizeof(T));
                    withRun<T>(runOf<T>(grad_x, grad_x_stride, q, q_stride, alignDy), [&](auto run) {
                        activationBackward<T, decltype(run)::value, decltype(f)::value>
                            <<<grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                                static_cast<const T*>(grad_y), grad_y_stride, reinterpret_cast<const uint8_t*>(q), q_stride,
                                scales, static_cast<T*>(grad_x), grad_x_stride, blocks, cols, colBlocks, alignDy);
                    });
                    checkCudaCall(cudaGetLastError());
                }
            });
        });
    });
}

} // extern "C"
