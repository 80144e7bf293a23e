// Product of two 8-bit block-scaled matrices on sm_100a:
//   Y[m, n] = sum over k of a[m, k] 2^ea[m, k / 128] * b[n, k] 2^eb[n, k / 128]  (+ bias[n])
#include "dense8.cuh"
#include "dense8_tc.cuh"

#include <mutex>

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

// A scale 2^e (NaN for the byte 255) as two factors of about half its exponent, the larger first. The product
// of two scales may be beyond the floats where a sum times it is none (zero times infinity) or is one; so a sum
// is multiplied by a.large * b.small and then by a.small * b.large, which are floats for all bytes and both
// on one side of 1.
struct Halves {
    float large, small;
};
__device__ __forceinline__ Halves halves(uint32_t byte) { // exponents byte - byte / 2 - 63 and byte / 2 - 64
    return {__uint_as_float(byte == 255u ? 0x7FC00000u : (byte - byte / 2 + 64u) << 23), __uint_as_float((byte / 2 + 63u) << 23)};
}
__device__ __forceinline__ float timesScales(float sum, Halves a, Halves b) {
    return sum * (a.large * b.small) * (a.small * b.large);
}

// ---- any strides and alignment ----------------------------------------------------------------
// 64 x 64 outputs per CTA, 4 x 4 per thread, FP32 FMA from elements widened into shared memory; the sum over a
// block of 128 is multiplied by its two scales.
// For matrices whose rows do not start on 16 bytes, which the tensor-core kernels' copies cannot read.
// FMA and shared-memory bound: 12.2 ms for 8192 x 4096 x 4100 on rows of 4101 bytes, 22.6 TFLOP/s.
constexpr int kTile = 64, kStep = 32;

template <typename T>
__global__ void __launch_bounds__(256) productGeneric(const Operand a, const Operand b, bool kn, const float* __restrict__ bias,
                                                      T* __restrict__ out, uint64_t outStride, uint32_t m, uint32_t n,
                                                      uint32_t k, uint32_t tilesN) {
    static_assert(kBlock % kStep == 0, "a step lies in one block");
    __shared__ float as[kStep][kTile + 1], bs[kStep][kTile + 1];
    __shared__ Halves aScale[kTile], bScale[kTile];
    const uint32_t m0 = blockIdx.x / tilesN * kTile, n0 = blockIdx.x % tilesN * kTile;
    const uint32_t kBlocks = (k + kBlock - 1) / kBlock, nBlocks = (n + kBlock - 1) / kBlock;
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {}, part[4][4] = {};
    for (uint32_t k0 = 0; k0 < k; k0 += kStep) {
        const uint32_t block = k0 / kBlock;
        if (k0 % kBlock == 0 && threadIdx.x < 2 * kTile) { // rows and columns outside: their sums go nowhere
            const uint32_t i = threadIdx.x % kTile, row = min(m0 + i, m - 1), col = min(n0 + i, n - 1);
            if (threadIdx.x < kTile)
                aScale[i] = halves(a.scales[uint64_t(row >> a.rowShift) * kBlocks + block]);
            else
                bScale[i] = halves(kn ? b.scales[uint64_t(block) * nBlocks + col / kBlock]
                                      : b.scales[uint64_t(col >> b.rowShift) * kBlocks + block]);
        }
        for (uint32_t i = threadIdx.x; i < kStep * kTile; i += 256) {
            {
                const uint32_t kk = i % kStep, r = i / kStep;
                const uint32_t row = m0 + r, col = k0 + kk;
                float v = 0.0f;
                if (row < m && col < k)
                    v = fp8Value(a.data[row * a.stride + col], a.type == TCC_E4M3);
                as[kk][r] = v;
            }
            const uint32_t kk = kn ? i / kTile : i % kStep, r = kn ? i % kTile : i / kStep;
            const uint32_t row = n0 + r, col = k0 + kk;
            float v = 0.0f;
            if (row < n && col < k)
                v = fp8Value(kn ? b.data[col * b.stride + row] : b.data[row * b.stride + col], b.type == TCC_E4M3);
            bs[kk][r] = v;
        }
        __syncthreads();
#pragma unroll 8
        for (int kk = 0; kk < kStep; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    part[i][j] = fmaf(as[kk][ty * 4 + i], bs[kk][tx + 16 * j], part[i][j]);
        if (k0 % kBlock == kBlock - kStep || k - k0 <= kStep)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] += timesScales(part[i][j], aScale[ty * 4 + i], bScale[tx + 16 * j]);
                    part[i][j] = 0.0f;
                }
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

// ---- few rows of a ------------------------------------------------------------------------------
// With up to 16 rows of a the product is a read of b. A CTA takes 16 rows of b; its warps take blocks of
// 128 of k in turn, each with a ring of its own of asynchronous copies (no barrier between warps, and
// all of a 4096-wide row in flight at once), and their sums are added up in shared memory at the end, in
// a fixed order. The order of k in mma.m16n8k32 may be any that both operands share, so a lane reads 16
// bytes of k of two rows of b and of MT rows of a at a time: two MMAs per 64 of k and 8 rows of a. The sum
// over a block is multiplied by the two scales, powers of two (see Halves). 6.9 us for 1 x 4096 x 4096 out of
// HBM (2.4 TB/s; 2.4 us of it launch and drain), 19.0 us for 1 x 8192 x 8192 (3.5 TB/s: its 512 CTAs are 1.73 rounds on
// 296 places, and each begins with an empty ring).
template <int MT_> struct Few {
    static constexpr int MT = MT_;
    static constexpr int kWarps = 8, kRows = 16;         // rows of b per CTA
    static constexpr int kStages = MT == 1 ? 4 : 3;
    static constexpr int kStageBytes = (kRows + 8 * MT) * 128;
    static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
    static constexpr uint32_t kMostBlocks = 512;         // blocks of k whose scales fit beside the rings
    static int bytes(uint32_t kBlocks) { return kRingBytes + int(kRows + 8 * MT) * int(kBlocks); }
};

// Rows of 8-bit floats from the row-major operand; which is which in mma.m16n8k32 follows the types.
template <bool TA5, bool TB5>
__device__ __forceinline__ void mmaFp8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
#define TCC_MMA(TA, TB)                                                                                             \
    asm("mma.sync.aligned.m16n8k32.row.col.f32." TA "." TB ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                            \
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
    if constexpr (TA5 && TB5)
        TCC_MMA("e5m2", "e5m2");
    else if constexpr (TA5)
        TCC_MMA("e5m2", "e4m3");
    else if constexpr (TB5)
        TCC_MMA("e4m3", "e5m2");
    else
        TCC_MMA("e4m3", "e4m3");
#undef TCC_MMA
}
// 16 bytes to shared memory, the last 16 - bytes of them zero.
__device__ __forceinline__ void cpAsync16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int MT, bool A5, bool B5, typename T>
__global__ void __launch_bounds__(32 * Few<MT>::kWarps)
    productFew(const Operand a, const Operand b, const float* __restrict__ bias, T* __restrict__ out, uint64_t outStride,
               uint32_t m, uint32_t n, uint32_t k) {
    using L = Few<MT>;
    extern __shared__ __align__(128) unsigned char smem[];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint64_t n0 = uint64_t(blockIdx.x) * L::kRows;
    const uint32_t kBlocks = (k + kBlock - 1) / kBlock;
    const uint32_t ring = dev::smemAddr(smem) + warp * L::kStages * L::kStageBytes;
    // Copies of a block: a lane's 16-byte piece of rows lane / 8, + 4, ... Rows outside are not copied:
    // their sums go nowhere. Odd rows swap their 64-byte halves, for the banks.
    const uint32_t piece = lane % 8, row0 = lane / 8;
    auto copy = [&](uint32_t kb, uint32_t stage) {
        const uint32_t to = ring + stage * L::kStageBytes + ((piece ^ ((row0 & 1) << 2)) * 16) + row0 * 128;
        const uint32_t c = kb * kBlock + 16 * piece;
        const uint32_t bytes = c < k ? min(16u, k - c) : 0u, at = c < k ? c : 0u;
#pragma unroll
        for (int i = 0; i < L::kRows / 4; ++i)
            if (n0 + row0 + 4 * i < n)
                cpAsync16(to + 512 * i, b.data + (n0 + row0 + 4 * i) * b.stride + at, bytes);
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
            if (row0 + 4 * i < m)
                cpAsync16(to + L::kRows * 128 + 512 * i, a.data + uint64_t(row0 + 4 * i) * a.stride + at, bytes);
    };
#pragma unroll
    for (int i = 0; i < L::kStages; ++i) {
        if (warp + i * L::kWarps < kBlocks)
            copy(warp + i * L::kWarps, i);
        dev::cpAsyncCommit();
    }
    // Scale bytes of the CTA's rows of b, then of a: [row][block].
    unsigned char* scales = smem + L::kRingBytes;
    for (uint32_t i = threadIdx.x; i < (L::kRows + 8 * MT) * kBlocks; i += 32 * L::kWarps) {
        const uint32_t row = i / kBlocks, kb = i - row * kBlocks;
        scales[i] = row < L::kRows ? __ldg(b.scales + (min(n0 + row, uint64_t(n - 1)) >> b.rowShift) * kBlocks + kb)
                                   : __ldg(a.scales + uint64_t(min(row - L::kRows, m - 1) >> a.rowShift) * kBlocks + kb);
    }
    __syncthreads();
    float acc[MT][4] = {};
    uint32_t stage = 0;
    for (uint32_t kb = warp; kb < kBlocks; kb += L::kWarps) {
        dev::cpAsyncWaitGroup<L::kStages - 1>();
        __syncwarp();
        const uint32_t from = ring + stage * L::kStageBytes + g * 128;
        float part[MT][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = from + (((4 * h + t) ^ ((g & 1) << 2)) * 16);
            const uint4 u = dev::ldsV4(at), v = dev::ldsV4(at + 1024);
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const uint4 x = dev::ldsV4(at + L::kRows * 128 + 1024 * j);
                mmaFp8<B5, A5>(part[j], u.x, v.x, u.y, v.y, x.x, x.y);
                mmaFp8<B5, A5>(part[j], u.z, v.z, u.w, v.w, x.z, x.w);
            }
        }
        const Halves sb[2] = {halves(scales[g * kBlocks + kb]), halves(scales[(g + 8) * kBlocks + kb])};
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const unsigned char* sa = scales + (L::kRows + 8 * j + 2 * t) * kBlocks + kb;
            const Halves s[2] = {halves(sa[0]), halves(sa[kBlocks])};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                acc[j][i] += timesScales(part[j][i], s[i % 2], sb[i / 2]);
        }
        __syncwarp(); // every lane has read the stage
        if (kb + L::kStages * L::kWarps < kBlocks)
            copy(kb + L::kStages * L::kWarps, stage);
        dev::cpAsyncCommit();
        stage = stage + 1 == L::kStages ? 0 : stage + 1;
    }
    dev::cpAsyncWaitAll();
    __syncthreads(); // the rings become the sums
    float(*sums)[L::kRows][8 * MT + 1] = reinterpret_cast<float(*)[L::kRows][8 * MT + 1]>(smem);
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            sums[warp][g + 8 * (i / 2)][8 * j + 2 * t + i % 2] = acc[j][i];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < L::kRows * 8 * MT; i += 32 * L::kWarps) {
        const uint32_t row = i / L::kRows, c = i % L::kRows; // row of a, row of b within the CTA's
        if (row < m && n0 + c < n) {
            float sum = bias ? bias[n0 + c] : 0.0f;
#pragma unroll
            for (int w = 0; w < L::kWarps; ++w)
                sum += sums[w][c][row];
            out[row * outStride + n0 + c] = fromFloat<T>(sum);
        }
    }
}

template <int MT, bool A5, bool B5, typename T> void launchFewTo(const Product& p) {
    using L = Few<MT>;
    allowSharedMemory<productFew<MT, A5, B5, T>>(L::bytes(L::kMostBlocks));
    productFew<MT, A5, B5, T><<<ceilDiv<uint32_t>(p.n, L::kRows), 32 * L::kWarps, L::bytes(ceilDiv(p.k, kBlock)), p.stream>>>(
        p.a, p.b, p.bias, static_cast<T*>(p.out), p.outStride, p.m, p.n, p.k);
    checkCudaCall(cudaGetLastError());
}
template <int MT, bool A5, bool B5> void launchFewTyped(const Product& p) {
    switch (p.outType) {
    case TCC_F32: launchFewTo<MT, A5, B5, float>(p); break;
    case TCC_BF16: launchFewTo<MT, A5, B5, __nv_bfloat16>(p); break;
    default: launchFewTo<MT, A5, B5, __half>(p); break;
    }
}
template <int MT> void launchFew(const Product& p) {
    if (p.a.type == TCC_E5M2)
        p.b.type == TCC_E5M2 ? launchFewTyped<MT, true, true>(p) : launchFewTyped<MT, true, false>(p);
    else
        p.b.type == TCC_E5M2 ? launchFewTyped<MT, false, true>(p) : launchFewTyped<MT, false, false>(p);
}

// ---- tensor cores -------------------------------------------------------------------------------
// Persistent clusters of CG CTAs (one per SM) compute tiles of 128 CG x BN outputs. A warp issues TMA
// copies of 128 bytes of k per stage (128-byte swizzle); one thread issues tcgen05.mma kind::mxf8f6f4,
// over the pair where CG = 2 (each CTA brings half of b's rows, which halves what an SM reads). Its
// E8M0 scales are the blocks' own bytes: the hardware takes one scale per 32 elements of k, and a
// block's four groups take the same one, so no scale is applied outside the tensor core and the sum
// over k stays in one FP32 accumulator in tensor memory. The tensor core cuts off what an addition
// shifts out below the accumulator's last bit: measured, 1.4e-6 of the sum of absolute values after 128 MMAs on
// operands of either sign, and 2.4e-3 after 32768 (7e-8 for every MMA) where all terms have one sign. So a long sum
// is emptied into registers, which round to nearest, every kPass blocks (mostBlocks says which sums are long); that
// also bounds how long the epilogue waits. Scales travel as words of four
// consecutive blocks per row, loaded by warps of their own, copied to tensor memory by the MMA thread
// and picked by the byte selector of the instruction descriptor. Eight warps bring finished tiles into
// registers, release the accumulator, and write them by TMA through 4 KB of shared memory each.
//
// Large products run at the power limit: 8192 x 4096 x 4096 bf16 takes 93 us (2.95 PFLOP/s) on operands of
// few distinct exponents and 116 to 124 us on normal ones, 8192^3 351 us (3.13 PFLOP/s). Few columns are
// bound by HBM: 1M x 128 x 256 fp32 145 us (5.5 TB/s), bf16 88 us (6.1 TB/s).
template <int BN_, int CG_> struct Tile {
    static constexpr int BN = BN_, CG = CG_;
    static constexpr int kStages = BN == 256 ? 5 : BN == 128 ? 4 : 6;
    static constexpr int kAcc = BN == 256 ? 1 : 2;       // accumulators in tensor memory
    static constexpr int kSlots = 6;                     // groups of four blocks' scales
    static constexpr int kSlabs = 1 + (BN + 127) / 128;  // of 512 bytes: A's rows, B's rows
    static constexpr int kBRows = BN / CG;               // rows of b in this CTA
    static constexpr int kABytes = 128 * 128, kBBytes = kBRows * 128;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kHalf = BN / 2;                 // columns per epilogue warp
    static constexpr int kOutBufs = BN == 256 ? 1 : 2;   // of 4 KB per epilogue warp
    static constexpr int kEpilogueWarps = 8;
    static constexpr int kOutOff = kStages * kStageBytes;
    static constexpr int kScaleOff = kOutOff + kEpilogueWarps * kOutBufs * 4096;
    static constexpr int kBiasOff = kScaleOff + kSlots * kSlabs * 512; // kHalf floats per epilogue warp
    static constexpr int kBarOff = kBiasOff + kEpilogueWarps * kHalf * 4;
    // full, empty, peerFull [kStages]; scaleFull, scaleEmpty [kSlots]; accFull, accEmpty [kAcc]; TMEM address
    static constexpr int kBars = 3 * kStages + 2 * kSlots + 2 * kAcc;
    static constexpr int kNeed = kBarOff + 8 * kBars + 16 + 1024; // + alignment to 1024
    // At least half of the shared memory: a second CTA on the SM would wait for tensor memory.
    static constexpr int kBytes = kNeed > 120 * 1024 ? kNeed : 120 * 1024;
    static constexpr uint32_t kPass = 16;                // blocks of k (64 MMAs); a multiple of 4, as scales come
    static constexpr int kScaleCols = 4 * kSlabs;
    static constexpr int kTmemCols = 512;
    static constexpr int kTmaWarp = 8, kMmaWarp = 9, kScaleWarp = 10;
    static constexpr int kScaleWarps = BN == 256 ? 2 : 3; // 13 warps would leave the epilogue 128 registers
    static constexpr int kThreads = 32 * (kScaleWarp + kScaleWarps);
    static_assert(kSlots % kScaleWarps == 0, "a slot belongs to one scale warp");
    static_assert(kAcc * BN + kSlots * kScaleCols <= kTmemCols && kBytes <= 232448, "resources");
};

// Instruction descriptor of kind::mxf8f6f4 without the byte selectors: types (0 e4m3, 1 e5m2) in
// bits 7-9 and 10-12, B MN-major in bit 16, N / 8 in bits 17-22, E8M0 scales in bit 23, M / 128 in
// bits 27-28. The selectors are bits 29-30 (A) and 4-5 (B).
__host__ __device__ constexpr uint32_t scaledIdesc(bool aE5m2, bool bE5m2, bool kn, uint32_t m, uint32_t n) {
    return (uint32_t(aE5m2) << 7) | (uint32_t(bE5m2) << 10) | (uint32_t(kn) << 16) | ((n >> 3) << 17) | (1u << 23) |
           ((m >> 7) << 27);
}

struct ScaleView {
    const uint8_t* data;
    uint32_t rows, rowShift; // rows of the operand; rows per block = 1 << rowShift
    uint32_t width;          // bytes per row of scales
    bool words;              // rows of scales start on 4 bytes
};
struct ProductArgs {
    ScaleView a, b;
    const float* bias;
    void* out;
    uint64_t outStride;
    int outType;
    bool outTma;   // output rows start and end on 16 bytes: written by TMA
    bool outWords; // output rows start and end on 4 bytes
    uint32_t aBytes, bBytes; // what a stage's two copies bring
    bool keepB; // one column of tiles, and a stage always holds the same block of k: its b stays
    uint32_t m, n, k, tilesM, tilesN;
    uint32_t idesc;
    uint32_t splits; // of SPLIT: CTAs per tile (2, 4 or 8)
};

// Scale bytes of blocks 4g .. 4g + 3 of one row; 1.0 for rows and blocks outside.
__device__ __forceinline__ uint32_t scaleWord(const ScaleView& s, uint64_t row, uint32_t g) {
    if (row >= s.rows)
        return 0x7F7F7F7Fu;
    const uint8_t* p = s.data + (row >> s.rowShift) * s.width + 4 * g;
    if (s.words)
        return __ldg(reinterpret_cast<const uint32_t*>(p));
    uint32_t w = 0x7F7F7F7Fu;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (4 * g + i < s.width)
            w = (w & ~(0xFFu << (8 * i))) | (uint32_t(__ldg(p + i)) << (8 * i));
    return w;
}
// The same for column n of a [k, n] operand with blocks of 128 x 128.
__device__ __forceinline__ uint32_t scaleWordKn(const ScaleView& s, uint32_t kBlocks, uint32_t n, uint32_t g) {
    uint32_t w = 0x7F7F7F7Fu;
    const uint32_t c = min(n / kBlock, s.width - 1);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (4 * g + i < kBlocks)
            w = (w & ~(0xFFu << (8 * i))) | (uint32_t(__ldg(s.data + uint64_t(4 * g + i) * s.width + c)) << (8 * i));
    return w;
}

// Tiles in groups of 16 rows of tiles, so that the tiles in flight share operands in L2.
template <typename L> __device__ __forceinline__ void tilePlace(const ProductArgs& p, uint32_t t, uint64_t& m0, uint32_t& n0) {
    const uint32_t span = 16 * p.tilesN;
    const uint32_t first = t / span * 16, local = t % span;
    const uint32_t height = min(16u, p.tilesM - first);
    m0 = uint64_t(first + local % height) * (128 * L::CG);
    n0 = local / height * L::BN;
}

// A tensor-memory row's columns [c, c + N) with the bias added, to 16 bytes of T each.
template <typename T>
__device__ __forceinline__ uint4 outputPiece(const uint32_t* acc, uint32_t bias) {
    constexpr int kE = kPer16<T>;
    float v[kE];
#pragma unroll
    for (int i = 0; i < kE; i += 4) {
        const uint4 b = dev::ldsV4(bias + 4 * i);
        v[i] = __uint_as_float(acc[i]) + __uint_as_float(b.x), v[i + 1] = __uint_as_float(acc[i + 1]) + __uint_as_float(b.y);
        v[i + 2] = __uint_as_float(acc[i + 2]) + __uint_as_float(b.z), v[i + 3] = __uint_as_float(acc[i + 3]) + __uint_as_float(b.w);
    }
    return pack16<T>(v);
}

__device__ __forceinline__ void tmaStore2d(const CUtensorMap* map, uint32_t src, uint32_t x, uint32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(map), "r"(x), "r"(y), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int LEFT> __device__ __forceinline__ void tmaStoreWaitRead() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}

// Up to 32 rows of a box of WIDTH bytes a row to the output, `bytes` of each, in pieces of W bytes:
// neighbouring lanes on neighbouring pieces, several rounds of loads before their stores (701999 x 21 x 256 fp32
// 93 -> 46 us).
template <int WIDTH, int W>
__device__ __forceinline__ void copyRows(uint32_t at, void* out, uint64_t step, uint32_t rows, uint32_t bytes, uint32_t lane) {
    constexpr uint32_t kLanes = WIDTH / W < 32 ? WIDTH / W : 32, kRows = 32 / kLanes, kPieces = WIDTH / W / kLanes;
    constexpr uint32_t kBatch = kRows > 4 ? 32 / kRows : 8 / kPieces;
    static_assert(32 % (kRows * kBatch) == 0, "rounds end with the box");
    const uint32_t sub = lane / kLanes, byte0 = lane % kLanes * W;
    uint8_t* to = static_cast<uint8_t*>(out) + sub * step + byte0;
    for (uint32_t row0 = 0; row0 < rows; row0 += kRows * kBatch) {
        uint32_t v[kBatch][kPieces];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b)
#pragma unroll
            for (uint32_t i = 0; i < kPieces; ++i) {
                const uint32_t row = row0 + b * kRows + sub, byte = byte0 + i * kLanes * W;
                const uint32_t piece = WIDTH == 128 ? (byte / 16) ^ (row & 7) : byte / 16;
                const uint32_t from = at + row * WIDTH + piece * 16 + byte % 16;
                if constexpr (W == 4)
                    v[b][i] = dev::ldsU32(from);
                else
                    asm volatile("{ .reg .u16 t; ld.shared.u16 t, [%1]; cvt.u32.u16 %0, t; }" : "=r"(v[b][i]) : "r"(from) : "memory");
            }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b, to += kRows * step)
#pragma unroll
            for (uint32_t i = 0; i < kPieces; ++i)
                if (row0 + b * kRows + sub < rows && byte0 + i * kLanes * W < bytes) {
                    if constexpr (W == 4)
                        *reinterpret_cast<uint32_t*>(to + i * kLanes * W) = v[b][i];
                    else
                        *reinterpret_cast<unsigned short*>(to + i * kLanes * W) = static_cast<unsigned short>(v[b][i]);
                }
    }
}

// One warp's 32 rows x kHalf columns of a finished tile: lane = row. Boxes of 32 rows x 128 bytes (or
// the whole width, if less) go through shared memory, swizzled as the map says, to the output by TMA, or,
// where rows do not start and end on 16 bytes, row by row with neighbouring lanes on neighbouring
// columns (straight from the registers, a column of 32 rows at a time, took four times as long).
template <typename L, typename T>
__device__ __forceinline__ void storeTile(const ProductArgs& p, const CUtensorMap* map, const uint32_t (&r)[L::kHalf],
                                          uint32_t buf, uint32_t& turn, uint32_t bias, uint64_t row0, uint32_t n0, uint32_t lane) {
    constexpr int kWidth = L::kHalf * int(sizeof(T)) < 128 ? L::kHalf * int(sizeof(T)) : 128;
    constexpr int kPerBox = kWidth / int(sizeof(T)), kBoxes = L::kHalf / kPerBox;
#pragma unroll
    for (int box = 0; box < kBoxes; ++box) {
        const uint32_t c0 = n0 + box * kPerBox;
        if (c0 >= p.n)
            break;
        const uint32_t at = buf + turn * 4096;
        turn = turn + 1 == L::kOutBufs ? 0 : turn + 1;
        if (p.outTma && lane == 0) // the box that was last stored from here, kOutBufs boxes ago, has been read
            tmaStoreWaitRead<L::kOutBufs - 1>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kWidth / 16; ++j) {
            const uint4 w = outputPiece<T>(r + box * kPerBox + j * kPer16<T>, bias + 4 * (box * kPerBox + j * kPer16<T>));
            const uint32_t piece = kWidth == 128 ? j ^ (lane & 7) : j;
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                         ::"r"(at + lane * kWidth + piece * 16), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                         : "memory");
        }
        if (p.outTma) {
            dev::fenceProxyAsyncShared();
            __syncwarp();
            if (lane == 0)
                tmaStore2d(map, at, c0, uint32_t(row0));
        } else {
            __syncwarp();
            const uint32_t rows = uint32_t(min(uint64_t(32), p.m - row0));
            const uint32_t bytes = min(uint32_t(kPerBox), p.n - c0) * uint32_t(sizeof(T));
            T* out = static_cast<T*>(p.out) + row0 * p.outStride + c0;
            if (sizeof(T) == 4 || p.outWords)
                copyRows<kWidth, 4>(at, out, p.outStride * sizeof(T), rows, bytes, lane);
            else
                copyRows<kWidth, 2>(at, out, p.outStride * sizeof(T), rows, bytes, lane);
        }
    }
}

// Eight columns from column c on of one row of a split tile.
template <typename T>
__device__ __forceinline__ void storeEight(const ProductArgs& p, uint64_t row, uint32_t c, const float (&v)[8], uint32_t bias) {
    T* out = static_cast<T*>(p.out) + row * p.outStride + c;
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = __float_as_uint(v[i]);
    if (p.outTma && c + 8 <= p.n) {
#pragma unroll
        for (int i = 0; i < 8; i += kPer16<T>)
            *reinterpret_cast<uint4*>(out + i) = outputPiece<T>(w + i, bias + 4 * i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < p.n)
                out[i] = fromFloat<T>(v[i] + __uint_as_float(dev::ldsU32(bias + 4 * i)));
    }
}

// The first block of k of one of the CTAs that share a tile: groups of four blocks, as their scales come, dealt out
// evenly.
__host__ __device__ constexpr uint32_t firstBlock(uint32_t kBlocks, uint32_t part, uint32_t parts) {
    return (kBlocks + 3) / 4 * part / parts * 4;
}

// LONG: more blocks of k than mostBlocks, whose accumulators are summed in registers.
// SPLIT: few tiles: the cluster's CTAs share one tile's blocks of k (see firstBlock); each leaves its
// sums in its shared memory and adds up an equal part of the columns of all of them, in the order of k.
template <int BN, int CG, bool KN, bool LONG, bool SPLIT>
__global__ void __launch_bounds__(Tile<BN, CG>::kThreads, 1)
    productTiles(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                 const __grid_constant__ CUtensorMap mapOut, const ProductArgs p) {
    using L = Tile<BN, CG>;
    extern __shared__ unsigned char smemRaw[];
    const uint32_t base = (dev::smemAddr(smemRaw) + 1023u) & ~1023u;
    unsigned char* smem = smemRaw + (base - dev::smemAddr(smemRaw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = base + L::kBarOff, empty = full + 8 * L::kStages;
    const uint32_t peerFull = empty + 8 * L::kStages; // in the first CTA: the second's stage and scales are there
    const uint32_t scaleFull = peerFull + 8 * L::kStages, scaleEmpty = scaleFull + 8 * L::kSlots;
    const uint32_t accFull = scaleEmpty + 8 * L::kSlots, accEmpty = accFull + 8 * L::kAcc;
    const uint32_t tmemSlot = accEmpty + 8 * L::kAcc;
    const uint32_t rank = CG == 1 ? 0 : clusterRank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i)
            dev::mbarInit(full + 8 * i, 1), dev::mbarInit(empty + 8 * i, 1), dev::mbarInit(peerFull + 8 * i, 1);
        for (int i = 0; i < L::kSlots; ++i)
            dev::mbarInit(scaleFull + 8 * i, 1), dev::mbarInit(scaleEmpty + 8 * i, 1);
        for (int i = 0; i < L::kAcc; ++i)
            dev::mbarInit(accFull + 8 * i, 1), dev::mbarInit(accEmpty + 8 * i, L::kEpilogueWarps * CG);
        dev::fenceBarrierInit();
    }
    if (warp == L::kMmaWarp)
        tmemAllocGroup<CG>(tmemSlot, L::kTmemCols);
    dev::tcFenceBefore();
    clusterSync<CG>();
    dev::tcFenceAfter();
    const uint32_t tmem = dev::ldsU32(tmemSlot);
    const uint32_t scaleTmem = tmem + L::kAcc * BN;
    static_assert(!SPLIT || CG == 1, "a split tile belongs to single CTAs");
    const uint32_t kBlocks = (p.k + kBlock - 1) / kBlock;
    const uint32_t part = SPLIT ? clusterRank() : 0, parts = SPLIT ? p.splits : 1;
    const uint32_t kbFirst = SPLIT ? firstBlock(kBlocks, part, parts) : 0;
    const uint32_t kbLast = SPLIT ? min(firstBlock(kBlocks, part + 1, parts), kBlocks) : kBlocks;
    const uint32_t groups = (kbLast - kbFirst + 3) / 4; // kbFirst is a multiple of 4
    const uint32_t tiles = p.tilesM * p.tilesN, firstTile = blockIdx.x / (SPLIT ? parts : CG),
                   tileStep = gridDim.x / (SPLIT ? parts : CG);

    if (warp == L::kTmaWarp) {
        if (lane == 0) {
            tmaPrefetchMap(&mapA);
            tmaPrefetchMap(&mapB);
            uint32_t it = 0, stage = 0, phase = 1; // a stage's first turn does not wait
            bool ok = true;
            for (uint32_t t = firstTile; t < tiles && ok; t += tileStep) {
                uint64_t m0;
                uint32_t n0;
                tilePlace<L>(p, t, m0, n0);
                m0 += 128 * rank, n0 += L::kBRows * rank;
                for (uint32_t kb = kbFirst; kb < kbLast; ++kb, ++it) {
                    if (!waitPhase(empty + 8 * stage, phase)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a = base + stage * L::kStageBytes, b = a + L::kABytes, bar = full + 8 * stage;
                    const bool bringB = !p.keepB || it < L::kStages;
                    dev::mbarArriveExpectTx(bar, p.aBytes + (bringB ? p.bBytes : 0u));
                    tmaLoad2d(a, &mapA, kb * kBlock, uint32_t(m0), bar);
                    if (!bringB)
                        ;
                    else if constexpr (KN)
                        tmaLoad2d(b, &mapB, n0, kb * kBlock, bar);
                    else
                        tmaLoad2d(b, &mapB, kb * kBlock, n0, bar);
                    if (++stage == L::kStages)
                        stage = 0, phase ^= 1;
                }
            }
            // After a wait that ran out, no copy may still be on its way when the CTA exits.
            if (!ok)
                for (uint32_t i = it < L::kStages ? 0 : it - L::kStages; i < it; ++i)
                    waitPhase(full + 8 * (i % L::kStages), (i / L::kStages) & 1);
        }
        __syncwarp();
    } else if (warp == L::kMmaWarp && rank == 0) {
        // The whole warp in uniform control flow; one elected lane issues.
        const uint32_t elected = electLane();
        uint32_t stage = 0, phase = 0, slot = 0, slotPhase = 0, acc = 0, accPhase = 1;
        bool ok = true;
        for (uint32_t t = firstTile; t < tiles && ok; t += tileStep) {
            uint32_t passEnd = kbFirst, d = 0; // the block of k before which the accumulator changes
            for (uint32_t kb = kbFirst; kb < kbLast; ++kb) {
                const bool fresh = kb == passEnd;
                if (fresh) {
                    if (!waitPhase(accEmpty + 8 * acc, accPhase)) {
                        ok = false;
                        break;
                    }
                    dev::tcFenceAfter();
                    d = tmem + acc * BN;
                    passEnd = LONG ? min(kb + L::kPass, kbLast) : kbLast;
                }
                const uint32_t sa = scaleTmem + slot * L::kScaleCols, sb = sa + 4, byte = kb & 3;
                if (byte == 0 && !waitPhase(scaleFull + 8 * slot, slotPhase)) {
                    ok = false;
                    break;
                }
                if (!waitPhase(full + 8 * stage, phase) || (CG == 2 && !waitPhase(peerFull + 8 * stage, phase))) {
                    ok = false;
                    break;
                }
                dev::tcFenceAfter();
                if (byte == 0) {
                    const uint32_t slab = base + L::kScaleOff + slot * L::kSlabs * 512;
#pragma unroll
                    for (int i = 0; i < L::kSlabs; ++i)
                        tcCopyScales<CG>(elected, sa + 4 * i, slabDesc(slab + 512 * i));
                }
                const uint32_t a = base + stage * L::kStageBytes, b = a + L::kABytes;
                const uint64_t descA = swizzledDesc(a, 16, 1024), descB = swizzledDesc(b, 16, 1024);
                const uint32_t idesc = p.idesc | (byte << 29) | (byte << 4);
                if (p.k - kb * kBlock >= kBlock) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mmaScaled8<CG>(elected, d, descA + 2 * j, descB + (KN ? 256 : 2) * j, idesc, sa, sb,
                                       j != 0 ? 1u : uint32_t(!fresh));
                } else { // the last block ends inside
                    const uint32_t steps = (p.k - kb * kBlock + 31) / 32;
                    for (uint32_t j = 0; j < steps; ++j)
                        mmaScaled8<CG>(elected, d, descA + 2 * j, descB + (KN ? 256 : 2) * j, idesc, sa, sb,
                                       j != 0 || !fresh);
                }
                commitCluster<CG>(elected, empty + 8 * stage);
                if (++stage == L::kStages)
                    stage = 0, phase ^= 1;
                if (byte == 3 || kb + 1 == kbLast) {
                    commitCluster<CG>(elected, scaleEmpty + 8 * slot);
                    if (++slot == L::kSlots)
                        slot = 0, slotPhase ^= 1;
                }
                if (kb + 1 == passEnd) {
                    commitCluster<CG>(elected, accFull + 8 * acc);
                    if (++acc == L::kAcc)
                        acc = 0, accPhase ^= 1;
                }
            }
        }
    } else if (warp == L::kMmaWarp) {
        // The second CTA of a pair tells the first that its stages and scales are there.
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, slot = 0, slotPhase = 0;
            bool ok = true;
            for (uint32_t t = firstTile; t < tiles && ok; t += tileStep)
                for (uint32_t kb = 0; kb < kBlocks; ++kb) {
                    if ((kb % 4 == 0 && !waitPhase(scaleFull + 8 * slot, slotPhase)) || !waitPhase(full + 8 * stage, phase)) {
                        ok = false;
                        break;
                    }
                    arriveLeader<CG>(peerFull + 8 * stage);
                    if (++stage == L::kStages)
                        stage = 0, phase ^= 1;
                    if ((kb % 4 == 3 || kb + 1 == kBlocks) && ++slot == L::kSlots)
                        slot = 0, slotPhase ^= 1;
                }
        }
        __syncwarp();
    } else if (warp >= L::kScaleWarp) {
        // Lane i holds rows i, i + 32, i + 64 and i + 96 of a slab, 16 bytes in shared memory: A's 128
        // rows of this CTA, all of B's.
        // The warps take groups in turn: one warp's loads, whose latency under a full memory bus is 2.6
        // us, set the pace of short products. A slot always belongs to the same warp (kSlots is a
        // multiple of their number), so no warp can be two of its phases away from another.
        constexpr int kWords = 4 * L::kSlabs;
        const uint32_t first = warp - L::kScaleWarp;
        const uint64_t total = firstTile < tiles ? uint64_t((tiles - firstTile - 1) / tileStep + 1) * groups : 0;
        uint32_t slot = first, phase = 1;
        for (uint64_t i = first; i < total; i += L::kScaleWarps) {
            const uint32_t turn = uint32_t(i / groups), g = uint32_t(i - uint64_t(turn) * groups) + kbFirst / 4;
            uint64_t m0;
            uint32_t n0, w[kWords];
            tilePlace<L>(p, firstTile + turn * tileStep, m0, n0);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                w[c] = scaleWord(p.a, m0 + 128 * rank + 32 * c + lane, g);
#pragma unroll
            for (int c = 0; c < kWords - 4; ++c) {
                if (32 * c >= BN)
                    w[4 + c] = 0x7F7F7F7Fu;
                else if constexpr (KN)
                    w[4 + c] = scaleWordKn(p.b, kBlocks, n0 + 32 * c + lane, g);
                else
                    w[4 + c] = scaleWord(p.b, n0 + 32 * c + lane, g);
            }
            if (!waitPhase(scaleEmpty + 8 * slot, phase))
                break;
            unsigned char* slab = smem + L::kScaleOff + slot * L::kSlabs * 512 + 16 * lane;
#pragma unroll
            for (int j = 0; j < L::kSlabs; ++j)
                *reinterpret_cast<uint4*>(slab + 512 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            dev::fenceProxyAsyncShared();
            __syncwarp();
            if (lane == 0)
                dev::mbarArrive(scaleFull + 8 * slot);
            slot += L::kScaleWarps;
            if (slot >= L::kSlots)
                slot = first, phase ^= 1;
        }
    } else {
        const uint32_t quarter = warp % 4, half = warp / 4; // two warps share a lane quarter
        const uint32_t buf = base + L::kOutOff + warp * L::kOutBufs * 4096;
        const uint32_t bias = base + L::kBiasOff + warp * L::kHalf * 4;
        uint32_t acc = 0, phase = 0, turn = 0, biasAt = 0xFFFFFFFFu;
        for (uint32_t t = firstTile; t < tiles; t += tileStep) {
            uint64_t m0;
            uint32_t n0;
            tilePlace<L>(p, t, m0, n0);
            n0 += half * L::kHalf;
            if (n0 != biasAt) { // the warp's columns of the bias, zero where there is none
                __syncwarp();
                for (uint32_t i = lane; i < uint32_t(L::kHalf); i += 32) {
                    const float v = p.bias != nullptr && n0 + i < p.n ? __ldg(p.bias + n0 + i) : 0.0f;
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(bias + 4 * i), "f"(v) : "memory");
                }
                __syncwarp();
                biasAt = n0;
            }
            uint32_t r[L::kHalf];
            bool ok = true;
            for (uint32_t kb = kbFirst; kb < (LONG ? kbLast : kbFirst + 1); kb += L::kPass) {
                if (!waitPhase(accFull + 8 * acc, phase)) {
                    ok = false;
                    break;
                }
                dev::tcFenceAfter();
                const uint32_t from = tmem + acc * BN + half * L::kHalf + (quarter << 21); // lanes in bits 16-31
                if (!LONG || kb == kbFirst) {
                    if constexpr (L::kHalf == 16) {
                        dev::tcLoad32x32bx16(from, r);
                    } else {
#pragma unroll
                        for (int i = 0; i < L::kHalf / 32; ++i)
                            tcLoad32x32bx32(from + 32 * i, *reinterpret_cast<uint32_t(*)[32]>(r + 32 * i));
                    }
                    dev::tcWaitLd();
                } else {
#pragma unroll
                    for (int i = 0; i < L::kHalf; i += 8) {
                        uint32_t more[8];
                        tcLoad32x32bx8(from + i, more);
                        dev::tcWaitLd();
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            r[i + j] = __float_as_uint(__uint_as_float(r[i + j]) + __uint_as_float(more[j]));
                    }
                }
                dev::tcFenceBefore();
                __syncwarp();
                if (lane == 0)
                    arriveLeader<CG>(accEmpty + 8 * acc);
                if (++acc == L::kAcc)
                    acc = 0, phase ^= 1;
            }
            const uint64_t row0 = m0 + 128 * rank + 32 * quarter;
            if constexpr (SPLIT) {
                // The stages' memory is free: every MMA of this CTA is done.
                const uint32_t mine = base + warp * (L::kHalf * 128) + 4 * lane; // [column][row]
                if (ok)
#pragma unroll
                    for (int i = 0; i < L::kHalf; ++i)
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(mine + 128 * i), "r"(r[i]) : "memory");
                __syncwarp();
                clusterBarrier();
                const uint32_t width = L::kHalf / parts;
                if (ok)
                    for (uint32_t c = part * width; c < (part + 1) * width; c += 8) {
                        float v[8] = {};
                        for (uint32_t s = 0; s < parts; ++s)
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                v[j] += ldClusterF32(mine + 128 * (c + j), s);
                        if (row0 + lane < p.m && n0 + c < p.n) {
                            if (p.outType == TCC_BF16)
                                storeEight<__nv_bfloat16>(p, row0 + lane, n0 + c, v, bias + 4 * c);
                            else if (p.outType == TCC_F32)
                                storeEight<float>(p, row0 + lane, n0 + c, v, bias + 4 * c);
                            else
                                storeEight<__half>(p, row0 + lane, n0 + c, v, bias + 4 * c);
                        }
                    }
                break; // a cluster has one tile
            }
            if (!ok)
                break;
            if (row0 < p.m && n0 < p.n) {
                if (p.outType == TCC_BF16)
                    storeTile<L, __nv_bfloat16>(p, &mapOut, r, buf, turn, bias, row0, n0, lane);
                else if (p.outType == TCC_F32)
                    storeTile<L, float>(p, &mapOut, r, buf, turn, bias, row0, n0, lane);
                else
                    storeTile<L, __half>(p, &mapOut, r, buf, turn, bias, row0, n0, lane);
            }
        }
        if (!SPLIT && lane == 0) // shared memory stays until the stores have read it
            tmaStoreWaitRead<0>();
    }
    __syncwarp();
    if (SPLIT && warp >= L::kEpilogueWarps)
        clusterBarrier(); // the one at which the epilogue's sums are there
    dev::tcFenceBefore();
    // No CTA of a cluster leaves while another may still arrive on its barriers or read its sums.
    SPLIT ? clusterBarrier() : clusterSync<CG>();
    dev::tcFenceAfter();
    if (warp == L::kMmaWarp)
        tmemDeallocGroup<CG>(tmem, L::kTmemCols);
}

ScaleView scaleView(const Operand& o, uint32_t rows, uint32_t width) {
    return {o.scales, rows, o.rowShift, width, width % 4 == 0 && alignedTo(o.scales, 4)};
}

// How many CTAs share k where there are `tiles` tiles of 128 x 128: one to eight, as long as all the tiles' clusters
// run at once and each CTA has four blocks of k. clusters: how many of 2, 4 and 8 CTAs run at once, which is less
// than the SMs would hold since a cluster stays within a GPC (33 of 4 and 15 of 8 on a B200; 16 tiles at k = 8192
// take 18.6 us with eight CTAs each and 10.9 with four, 14 tiles 10.3 and 10.9).
constexpr uint32_t ctasPerTile(uint64_t tiles, uint32_t kBlocks, const uint32_t (&clusters)[3]) {
    uint32_t parts = 1;
    for (int i = 0; i < 3 && tiles <= clusters[i] && kBlocks >= 8 * parts; ++i)
        parts *= 2;
    return parts;
}
// The most blocks of k that one accumulator sums: kPass for fp32 outputs, and so many for the 16-bit types that the
// loss of 7e-8 for each of a block's four MMAs stays below a tenth of a half step (fp16 3.7e-5 of 4.9e-4, bf16
// 2.9e-4 of 3.9e-3). Emptying it takes 8192 x 4096 x 16512 from 385 us (bf16, one accumulator) to 407 (fp16).
template <typename L> constexpr uint32_t mostBlocks(int outType) {
    return outType == TCC_F32 ? L::kPass : outType == TCC_F16 ? 128u : 1024u;
}

template <int BN, int CG, bool KN, bool SPLIT = false> void launchTiles(const Product& p, uint32_t splits = 1) {
    using L = Tile<BN, CG>;
    static_assert(!KN || L::kBRows == 128, "rows of a [k, n] operand are copied 128 bytes at a time");
    const uint32_t kBlocks = ceilDiv(p.k, kBlock), outBytes = typeBytes(p.outType);
    ProductArgs args{};
    args.a = scaleView(p.a, p.m, kBlocks);
    args.b = KN ? ScaleView{p.b.scales, p.k, 7, ceilDiv(p.n, kBlock), false} : scaleView(p.b, p.n, kBlocks);
    args.bias = p.bias;
    args.out = p.out;
    args.outStride = p.outStride;
    args.outType = p.outType;
    // A TMA store writes whole 16-byte pieces of a row: n has to end one, or the next columns change.
    args.outTma = rowsAlignedTo(p.out, p.outStride * outBytes, 16) && p.n * uint64_t(outBytes) % 16 == 0 && p.outStride < (1ull << 38);
    args.outWords = rowsAlignedTo(p.out, p.outStride * outBytes, 4) && p.n * uint64_t(outBytes) % 4 == 0;
    args.m = p.m, args.n = p.n, args.k = p.k;
    args.tilesM = ceilDiv<uint32_t>(p.m, 128 * CG);
    args.tilesN = ceilDiv<uint32_t>(p.n, BN);
    require(uint64_t(args.tilesM) * args.tilesN <= 0x3FFFFFFFull, "too many output tiles for one call");
    args.idesc = scaledIdesc(p.a.type == TCC_E5M2, p.b.type == TCC_E5M2, KN, 128 * CG, BN);
    const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    // A box ends with a matrix of fewer rows than a tile: filling rows up with zeros takes a copy longer than
    // loading them (17 x 4096 x 4096 17.2 -> 11.2 us), and what is left in their place only reaches outputs
    // that are not there.
    const uint32_t aRows = std::min(128u, p.m), bRows = KN ? 128u : std::min<uint32_t>(L::kBRows, p.n);
    args.aBytes = aRows * 128, args.bBytes = bRows * 128;
    // 701999 x 21 x 65 fp32 72 -> 48 us, 1M x 128 x 256 fp32 149 -> 145 us.
    args.keepB = args.tilesN == 1 && L::kStages % kBlocks == 0;
    const CUtensorMap mapA = tensorMap2d(p.a.data, u8, 1, p.m, p.k, p.a.stride, aRows, 128);
    const CUtensorMap mapB = KN ? tensorMap2d(p.b.data, u8, 1, p.k, p.n, p.b.stride, 128, 128)
                                : tensorMap2d(p.b.data, u8, 1, p.n, p.k, p.b.stride, bRows, 128);
    CUtensorMap mapOut{};
    if (args.outTma) {
        const uint32_t width = std::min<uint32_t>(128, L::kHalf * outBytes);
        mapOut = tensorMap2d(p.out,
                             p.outType == TCC_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                             : p.outType == TCC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                             outBytes, p.m, p.n, p.outStride, std::min(32u, p.m), width / outBytes,
                             width == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE);
    }
    args.splits = splits;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(SPLIT ? args.tilesM * args.tilesN * splits
                                : CG * std::min<uint32_t>(args.tilesM * args.tilesN, multiprocessors() / CG));
    config.blockDim = dim3(L::kThreads);
    config.dynamicSmemBytes = L::kBytes;
    config.stream = p.stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = SPLIT ? splits : CG, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    if ((SPLIT ? ceilDiv(ceilDiv(kBlocks, 4u), splits) * 4 : kBlocks) > mostBlocks<L>(p.outType)) {
        allowSharedMemory<productTiles<BN, CG, KN, true, SPLIT>>(L::kBytes);
        checkCudaCall(cudaLaunchKernelEx(&config, productTiles<BN, CG, KN, true, SPLIT>, mapA, mapB, mapOut, args));
    } else {
        allowSharedMemory<productTiles<BN, CG, KN, false, SPLIT>>(L::kBytes);
        checkCudaCall(cudaLaunchKernelEx(&config, productTiles<BN, CG, KN, false, SPLIT>, mapA, mapB, mapOut, args));
    }
}

// The clusters of 2, 4 and 8 CTAs that share a tile which run at once on the current device (asked once per device).
struct SharingClusters {
    std::atomic<bool> known;
    uint32_t count[3];
};
const uint32_t (&sharingClusters())[3] {
    static SharingClusters devices[64] = {};
    static std::mutex asking;
    static constexpr uint32_t none[3] = {};
    const int device = currentDevice();
    if (device >= 64)
        return none;
    SharingClusters& d = devices[device];
    if (!d.known.load(std::memory_order_acquire)) {
        using L = Tile<128, 1>;
        const std::lock_guard<std::mutex> lock(asking);
        if (d.known.load(std::memory_order_relaxed))
            return d.count;
        allowSharedMemory<productTiles<128, 1, true, false, true>>(L::kBytes);
        for (uint32_t i = 0; i < 3; ++i) {
            cudaLaunchAttribute attr{};
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 2u << i, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
            cudaLaunchConfig_t config{};
            config.gridDim = dim3(8 * multiprocessors());
            config.blockDim = dim3(L::kThreads);
            config.dynamicSmemBytes = L::kBytes;
            config.attrs = &attr;
            config.numAttrs = 1;
            int count = 0;
            checkCudaCall(cudaOccupancyMaxActiveClusters(&count, productTiles<128, 1, true, false, true>, &config));
            d.count[i] = uint32_t(count);
        }
        d.known.store(true, std::memory_order_release);
    }
    return d.count;
}

void launchProduct(const Product& p) {
    const bool tma = p.k != 0 && rowsAlignedTo(p.a.data, p.a.stride, 16) && rowsAlignedTo(p.b.data, p.b.stride, 16) &&
                     p.a.stride < (1ull << 40) && p.b.stride < (1ull << 40) &&
                     std::max({p.m, p.n, p.k}) <= 0x7FFFFF00u; // coordinates of a copy are signed
    if (!tma) {
        switch (p.outType) {
        case TCC_F32: launchGeneric<float>(p); break;
        case TCC_BF16: launchGeneric<__nv_bfloat16>(p); break;
        default: launchGeneric<__half>(p); break;
        }
        return;
    }
    if (p.m <= 16 && !p.kn && ceilDiv(p.k, kBlock) <= Few<1>::kMostBlocks) {
        p.m <= 8 ? launchFew<1>(p) : launchFew<2>(p);
        return;
    }
    const uint64_t rowTiles = ceilDiv(p.m, 128u), sms = multiprocessors();
    const uint32_t splits = ctasPerTile(rowTiles * ceilDiv(p.n, 128u), ceilDiv(p.k, kBlock), sharingClusters());
    // One row of tiles of [n, k] weights runs as fast or faster in narrower tiles where those fill the SMs (128 x 4096
    // x 4096 11.1 us either way, 64 x 2048 x 8192 17.4 us against 20.4; not measured for few columns, which leave most
    // SMs idle), two rows gain (256 x 4096 x 4096 18.0 -> 13.1 us), and so do [k, n] weights, which have no narrower
    // tiles (128 x 4096 x 4096 14.4 -> 11.2 us).
    if (splits > 1 && (p.kn || rowTiles > 1)) {
        p.kn ? launchTiles<128, 1, true, true>(p, splits) : launchTiles<128, 1, false, true>(p, splits);
        return;
    }
    // The narrowest tile that holds n (701999 x 24 x 128 fp32 39 -> 35 us); of wider n the widest tile
    // that leaves few SMs idle.
    if (!p.kn && p.n <= 32)
        launchTiles<32, 1, false>(p);
    else if (!p.kn && p.n <= 64)
        launchTiles<64, 1, false>(p);
    else if (p.n > 128 && ceilDiv(p.m, 256u) * uint64_t(ceilDiv(p.n, 256u)) * 2 >= sms)
        p.kn ? launchTiles<256, 2, true>(p) : launchTiles<256, 2, false>(p);
    else if (p.kn || rowTiles * ceilDiv(p.n, 128u) >= sms)
        p.kn ? launchTiles<128, 1, true>(p) : launchTiles<128, 1, false>(p);
    else if (rowTiles * ceilDiv(p.n, 64u) >= sms)
        launchTiles<64, 1, false>(p);
    else
        launchTiles<32, 1, false>(p);
}

} // namespace

uint32_t matmulDeviceStatus(bool reset) { return denseStatus(reset); }

} // namespace tcc

extern "C" {

// Test hook: the CTAs that share a tile (returned) and the first block of k of each, with the end behind the last.
uint32_t tcc_test_product_parts(uint64_t tiles, uint32_t k_blocks, const uint32_t clusters[3], uint32_t first[9]) {
    const uint32_t parts = tcc::ctasPerTile(tiles, k_blocks, {clusters[0], clusters[1], clusters[2]});
    for (uint32_t i = 0; i <= parts; ++i)
        first[i] = std::min(tcc::firstBlock(k_blocks, i, parts), k_blocks);
    return parts;
}

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
