// Weight gradient of a linear layer whose input was kept as an INT8 checkpoint, on sm_100a:
//   dW[n, k] (+)= sum over rows r of dy[r, n] * q[r, k] 2^e[r, k / 128]
//
// The sum runs on the tensor cores in bf16 with FP32 accumulators, and no operand is rounded: an
// INT8 element times a power of two has at most 8 significant bits, which bf16 holds (at half its
// value, since an element may stand for 2^128; what leaves the accumulator is doubled), and dy is
// split into P bf16 parts that add up to it (P = 1 for bf16, 2 for fp16: 8 + 3 bits, 3 for fp32:
// 8 + 8 + 8 bits), each multiplied on its own into the same accumulator.
//
// A cluster of CG CTAs computes 128 CG rows (n) by 256 columns (k) of dW over a range of rows r, with
// tcgen05.mma over the pair where CG = 2: each CTA brings 128 columns of dy and half of the columns
// of q^, which halves the conversions and the shared-memory reads of an SM. CG = 1 where dW has at
// most 128 rows.
//
// Raw rows arrive by TMA in a ring of stages. Eight warps turn dy into operand A in tensor memory: a
// thread takes four neighbouring columns of a row at a time and pairs rows with byte permutes. Eight
// warps turn q into operand B in shared memory, row-major as it comes (MN-major, 128-byte swizzle).
// One thread issues the MMAs.
//
// The tensor core cuts off what an addition shifts out below the accumulator's last bit, about
// 1.5e-8 of the sum for every MMA (measured; 2.1e-5 after 1300; more where all terms have one sign), so
// the accumulator is emptied every 60 MMAs into the fp32 registers of eight warps, which round to
// nearest. The MMAs wait meanwhile: halves of the accumulator that take turns need MMAs of 128
// columns, which ran at 91 cycles instead of 64.
//
// 8192 x 4096 x 2048 bf16 takes 129 us (1.07 PFLOP/s; 128 tiles on 74 pairs are two rounds for 1.73),
// bound by shared memory's bandwidth in this layout (80 KB a stage and SM for 512 cycles of MMAs, 32 of
// them for the widened q; as operand A, in tensor memory, it would take none of it, and dy no copy). 1M
// rows x 128 x 256 takes 106 us in bf16 (5.1 TB/s) and 177 to 220 us in fp32, whose three parts run at the
// power limit (SM clock 1.2 GHz).
#include "dense8.cuh"
#include "dense8_tc.cuh"

#include <cmath>

namespace tcc {
namespace {

using namespace blk;

struct GradArgs {
    const void* dy;
    uint64_t dyStride;
    const uint8_t* q;
    uint64_t qStride;
    const uint8_t* scales;
    float* dw;
    uint64_t dwStride;
    float* partials; // [split][tile][CTA][64][128][4], null when the rows are not split
    uint32_t rows, n, k;
    uint32_t tilesN, tilesK, rowsPerSplit;
    bool accumulate;
    int dyAlign, qAlign; // bytes (up to 8 and 4) that every row of dy and of q starts on, read where TMA is not used
    bool dwTma; // rows of dw start and end on 16 bytes: written by TMA
};

template <uint32_t V> struct Const { static constexpr uint32_t value = V; };

template <typename T> constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
template <> constexpr int kParts<__half> = 2;

template <typename T, int CG> struct GradTile {
    static constexpr int kP = kParts<T>;
    static constexpr int kRows = kP == 3 || CG == 1 ? 32 : 64; // rows per stage
    static constexpr int kBk = 256, kBCols = kBk / CG; // columns of dW: of the cluster, of q in this CTA
    // Raw and operand stages: an operand stage takes about a microsecond from its conversion over the
    // MMAs' completion to its next use, so that much has to be in flight.
    static constexpr int kRaw = kP == 3 ? (CG == 1 ? 6 : 8) : CG == 1 || kP == 2 ? 6 : 4;
    static constexpr int kStages = kP == 3 || (kP == 2 && CG == 2) ? 4 : 6;
    // Two sets of producer warps take alternate stages. In an even ring a place always belongs to the
    // same set; in an odd one a set could run two of the place's phases ahead of the other, where a
    // barrier's parity no longer tells done from not yet begun.
    static_assert(kRaw % 2 == 0 && kStages % 2 == 0, "even rings");
    static constexpr int kABoxes = int(sizeof(T)), kBBoxes = kBCols / 128; // of 128 bytes x kRows
    static constexpr int kBox = kRows * 128;
    static constexpr int kRawBytes = (kABoxes + kBBoxes) * kBox;
    static constexpr int kBBytes = kRows * kBCols * 2;
    static constexpr int kACols = kP * kRows / 2;       // tensor-memory columns of a stage of A
    static constexpr int kSteps = kP * kRows / 16;      // MMAs per stage
    static constexpr uint32_t kFlush = 60 / kSteps;     // stages between two flushes
    static constexpr int kRawOff = kStages * kBBytes;
    static constexpr int kScaleOff = kRawOff + kRaw * kRawBytes; // halves of a raw stage's scales as bf16 pairs, by box and row
    static constexpr int kScaleBytes = kRows * kBBoxes * 4;
    static constexpr int kBarOff = kScaleOff + kRaw * kScaleBytes;
    // rawFull, rawEmpty [kRaw]; full, empty, peerFull [kStages]; accFull, accEmpty; TMEM address
    static constexpr int kBytes = kBarOff + 8 * (2 * kRaw + 3 * kStages + 2) + 16 + 1024;
    static constexpr int kCols = kBk + kStages * kACols;
    static constexpr int kEpilogueWarps = 8, kBWarp = 16, kLoadWarp = 24, kMmaWarp = 27;
    static constexpr int kThreads = 32 * 28;
    // Registers: 72 per thread at launch (seven warpgroups); the warpgroups then share them out, 152 for the
    // epilogue's 128 sums.
    static constexpr int kRegsEpilogue = 152, kRegsA = 40, kRegsB = 40, kRegsIssue = 40;
    // Whether a kernel that was built with `regs` registers per thread, which a launch rounds up to a multiple of 8,
    // has the shares to give: a warpgroup would wait for ever for registers that the launch did not get.
    static constexpr bool sharesFit(int regs) {
        const int held = (regs + 7) / 8 * 8;
        return kRegsA <= held && kRegsB <= held && kRegsIssue <= held && held <= kRegsEpilogue &&
               2 * kRegsEpilogue + 2 * kRegsA + 2 * kRegsB + kRegsIssue <= 7 * held;
    }
    static_assert(sharesFit(65) && sharesFit(72) && !sharesFit(64) && !sharesFit(160), "shares of 72 registers per thread");
    static_assert(kRaw * kRawBytes >= 8 * 4096 && kCols <= 512 && kBytes <= 232448 && kBytes > 116 * 1024, "resources: one CTA per SM");
};

// kind::f16 with FP32 accumulators (bits 4-5 = 1), bf16 A and B (bits 7-9 and 10-12 = 1), B
// MN-major (bit 16), N / 8 in bits 17-22 and M / 16 in bits 24-28.
__host__ __device__ constexpr uint32_t bf16Idesc(uint32_t m, uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// D(tmem) (+)= A(tmem, bf16) x B(shared memory, bf16).
template <int CG>
__device__ __forceinline__ void mmaBf16Ts(uint32_t elected, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
                     "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                     ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
                     "@e tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                     ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected)
                     : "memory");
}

// Four neighbouring columns of one row of dy, from a raw stage.
template <typename T> struct Quad { uint32_t w[sizeof(T)]; };
template <typename T> __device__ __forceinline__ Quad<T> loadQuad(uint32_t addr) {
    Quad<T> v;
    if constexpr (sizeof(T) == 4) {
        const uint4 u = dev::ldsV4(addr);
        v.w[0] = u.x, v.w[1] = u.y, v.w[2] = u.z, v.w[3] = u.w;
    } else {
        const uint2 u = dev::ldsV2(addr);
        v.w[0] = u.x, v.w[1] = u.y;
    }
    return v;
}

// The upper halves of two floats (their bf16 parts, cut off) as a pair, and what is left of them: a
// float's 24 bits are three such parts of 8, and every difference is exact.
__device__ __forceinline__ uint32_t upperPair(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}
__device__ __forceinline__ float withoutUpper(float v) {
    return v - __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
}

// Column c (0..3) of two rows' quads as P bf16 pairs (row u in the low half). CHECK: a value that is
// not finite leaves its later parts zero (infinity minus infinity would make them NaN).
template <typename T, bool CHECK>
__device__ __forceinline__ void splitPair(const Quad<T>& u, const Quad<T>& v, int c, uint32_t (&part)[kParts<T>]) {
    if constexpr (kParts<T> == 1) {
        part[0] = __byte_perm(u.w[c / 2], v.w[c / 2], c % 2 ? 0x7632 : 0x5410);
    } else {
        float a, b;
        if constexpr (sizeof(T) == 4) {
            a = __uint_as_float(u.w[c]), b = __uint_as_float(v.w[c]);
        } else {
            const uint32_t pair = __byte_perm(u.w[c / 2], v.w[c / 2], c % 2 ? 0x7632 : 0x5410);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
            a = f.x, b = f.y;
        }
        part[0] = upperPair(a, b);
        if constexpr (CHECK) { // a NaN whose upper half says infinity still has to stay one
            part[0] |= (a != a ? 0x7FFFu : 0u) | (b != b ? 0x7FFF0000u : 0u);
            a = fabsf(a) < INFINITY ? a : 0.0f, b = fabsf(b) < INFINITY ? b : 0.0f;
        }
        a = withoutUpper(a), b = withoutUpper(b);
        part[1] = upperPair(a, b);
        if constexpr (kParts<T> == 3)
            part[2] = upperPair(withoutUpper(a), withoutUpper(b));
    }
}
// Whether any of a warp's quads may hold a value that is not finite: exponents are looked at together,
// so large finite ones can raise it too, which only costs the checks.
template <typename T> __device__ __forceinline__ bool mayNotBeFinite(const Quad<T> (&q)[4]) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < int(sizeof(T)); ++j)
            any |= q[i].w[j];
    const bool raised = sizeof(T) == 4 ? (any & 0x7F800000u) == 0x7F800000u
                                       : (any & 0x7C00u) == 0x7C00u || (any & 0x7C000000u) == 0x7C000000u;
    return __any_sync(0xFFFFFFFFu, raised);
}

// Four INT8 elements times a power of two (a bf16 pair) in bf16: low 7 bits under the exponent
// of 128, minus 128 or, for negative elements, 256. Every step is exact.
__device__ __forceinline__ void int8ToBf16(uint32_t w, uint32_t scale, uint32_t& lo, uint32_t& hi) {
    const uint32_t x[2] = {__byte_perm(w, 0u, 0x4140), __byte_perm(w, 0u, 0x4342)};
    uint32_t out[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = (x[i] & 0x007F007Fu) | 0x43004300u, c = (x[i] & 0x00800080u) | 0xC300C300u;
        const __nv_bfloat162 f = __hmul2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                                 *reinterpret_cast<const __nv_bfloat162*>(&c)),
                                         *reinterpret_cast<const __nv_bfloat162*>(&scale));
        out[i] = *reinterpret_cast<const uint32_t*>(&f);
    }
    lo = out[0], hi = out[1];
}
// Half the 2^e of a scale byte as a bf16 pair (NaN for 255, subnormal for 1 and 0). With the whole of it
// the elements that stand for 2^128 were infinite and made every sum that a zero of dy met them in NaN.
__device__ __forceinline__ uint32_t halfScalePair(uint32_t byte) {
    return (byte == 255u ? 0x7FC0u : byte <= 1u ? 0x0020u << byte : (byte - 1u) << 7) * 0x10001u;
}

// Lane of a 32-lane quarter of A and D -> column of dy within the quarter's 32: the 16-lane store
// writes lanes t / 4 and t / 4 + 8 from thread t, which holds columns 4 (t / 4) .. + 3; the first
// half of the quarter takes columns 0 and 1 of each four, the second half 2 and 3.
__device__ __forceinline__ uint32_t laneColumn(uint32_t l) { return 4 * (l % 8) + 2 * (l / 16) + (l / 8) % 2; }

__device__ __forceinline__ void stsU32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void stsU8(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Row of a raw stage whose values stand at row k of the operands. Any order will do that A and B
// share; this one lets the four threads that read one column group of dy take rows two apart, which
// the TMA swizzle puts into distinct banks.
__device__ __forceinline__ uint32_t operandRow(uint32_t r) { // its inverse: raw row -> operand row
    return (r & ~15u) | ((r & 6u) << 1) | ((r & 8u) >> 2) | (r & 1u);
}

// One row's pieces of W bytes (8, 4, 2 or 1), 32 W apart, to shared memory at place(byte of the row);
// `have` bytes exist from the lane's first piece on, and zeros go behind them. 8 and 4 bytes go by
// asynchronous copies, whose address has to be valid even where nothing is read; 2 and 1 through
// registers, all loads before the stores.
template <int W, int PIECES, typename Place>
__device__ __forceinline__ void copyRow(const uint8_t* src, const void* valid, int have, uint32_t lane, Place place) {
    if constexpr (W >= 4) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const uint32_t bytes = uint32_t(max(0, min(W, have - 32 * i * W)));
            const void* from = bytes != 0 ? static_cast<const void*>(src + 32 * i * W) : valid;
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(place((32 * i + lane) * W)), "l"(from), "n"(W),
                         "r"(bytes)
                         : "memory");
        }
    } else {
        uint32_t v[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const uint8_t* at = src + 32 * i * W;
            v[i] = have - 32 * i * W < W ? 0u : W == 2 ? uint32_t(__ldg(reinterpret_cast<const unsigned short*>(at))) : uint32_t(__ldg(at));
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const uint32_t to = place((32 * i + lane) * W);
            if constexpr (W == 2)
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(static_cast<unsigned short>(v[i])) : "memory");
            else
                stsU8(to, v[i]);
        }
    }
}
// One of the three warps that fill raw stages without TMA: rows warp, warp + 3, ..., pieces of WA bytes
// of dy and WB bytes of q. Every lane arrives on the stage's barrier once its asynchronous copies have landed; that
// arrival does not publish the lane's ordinary stores (scales, pieces of 2 and 1 bytes), so a warp arrives once
// more, after them.
template <typename T, int CG, int WA, int WB>
__device__ __forceinline__ void loadRaw(const GradArgs& p, uint32_t base, uint32_t rawFull, uint32_t rawEmpty, uint32_t warp,
                                        uint32_t lane, uint64_t begin, uint64_t end, uint32_t stages, uint32_t n0,
                                        uint32_t kMine) {
    using L = GradTile<T, CG>;
    constexpr int kPiecesA = 128 * int(sizeof(T)) / (32 * WA), kPiecesB = L::kBCols / (32 * WB);
    const uint32_t kBlocks = (p.k + kBlock - 1) / kBlock, col = kMine / kBlock;
    const uint32_t scaleRow = warp + 3 * lane; // the lane's row for the scales
    const int bytesA = n0 < p.n ? int(min(p.n - n0, 128u) * sizeof(T)) - int(lane) * WA : 0;
    const int bytesB = kMine < p.k ? int(min(p.k - kMine, uint32_t(L::kBCols))) - int(lane) * WB : 0;
    const uint8_t* dy = static_cast<const uint8_t*>(p.dy) + uint64_t(n0) * sizeof(T) + lane * WA;
    const uint8_t* q = p.q + kMine + lane * WB;
    uint32_t raw = 0, phase = 1;
    for (uint32_t it = 0; it < stages; ++it) {
        if (!waitPhase(rawEmpty + 8 * raw, phase))
            break;
        const uint32_t to = base + L::kRawOff + raw * L::kRawBytes, scales = base + L::kScaleOff + raw * L::kScaleBytes;
        const uint64_t row0 = begin + uint64_t(it) * L::kRows;
        uint32_t scale[L::kBBoxes];
#pragma unroll
        for (int box = 0; box < L::kBBoxes; ++box)
            scale[box] = scaleRow < uint32_t(L::kRows) && row0 + scaleRow < end && col + box < kBlocks
                             ? uint32_t(__ldg(p.scales + (row0 + scaleRow) * kBlocks + col + box)) : 127u;
        for (uint32_t r = warp; r < uint32_t(L::kRows); r += 3) {
            const uint64_t row = row0 + r;
            const bool in = row < end;
            copyRow<WA, kPiecesA>(dy + row * p.dyStride * sizeof(T), p.dy, in ? bytesA : 0, lane, [&](uint32_t byte) {
                return to + byte / 128 * L::kBox + r * 128 + ((byte % 128) ^ ((r & 7) << 4));
            });
            copyRow<WB, kPiecesB>(q + row * p.qStride, p.q, in ? bytesB : 0, lane, [&](uint32_t byte) {
                return to + (L::kABoxes + byte / 128) * L::kBox + r * 128 + byte % 128;
            });
        }
#pragma unroll
        for (int box = 0; box < L::kBBoxes; ++box)
            if (scaleRow < uint32_t(L::kRows))
                stsU32(scales + 4 * (box * L::kRows + scaleRow), halfScalePair(scale[box]));
        dev::cpAsyncArriveNoinc(rawFull + 8 * raw);
        __syncwarp();
        if (lane == 0)
            dev::mbarArrive(rawFull + 8 * raw);
        if (++raw == L::kRaw)
            raw = 0, phase ^= 1;
    }
    dev::cpAsyncWaitAll(); // none may be on its way when the CTA exits
}

template <typename T, int CG, bool TMA>
__global__ void __launch_bounds__(GradTile<T, CG>::kThreads, 1)
    gradTiles(const __grid_constant__ CUtensorMap mapDy, const __grid_constant__ CUtensorMap mapQ,
              const __grid_constant__ CUtensorMap mapDw, const GradArgs p) {
    using L = GradTile<T, CG>;
    extern __shared__ unsigned char smemRaw[];
    const uint32_t base = (dev::smemAddr(smemRaw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rawFull = base + L::kBarOff, rawEmpty = rawFull + 8 * L::kRaw;
    const uint32_t full = rawEmpty + 8 * L::kRaw, empty = full + 8 * L::kStages;
    const uint32_t peerFull = empty + 8 * L::kStages; // in the first CTA: the second's stage is full
    const uint32_t accFull = peerFull + 8 * L::kStages, accEmpty = accFull + 8, tmemSlot = accEmpty + 8;
    const uint32_t rank = CG == 1 ? 0 : clusterRank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kRaw; ++i)
            dev::mbarInit(rawFull + 8 * i, TMA ? 2 : 3 * (32 + 1)), dev::mbarInit(rawEmpty + 8 * i, 8); // 4 warps of A, 4 of B
        for (int i = 0; i < L::kStages; ++i)
            dev::mbarInit(full + 8 * i, 8), dev::mbarInit(empty + 8 * i, 1), dev::mbarInit(peerFull + 8 * i, 1);
        dev::mbarInit(accFull, 1), dev::mbarInit(accEmpty, 8 * CG);
        dev::fenceBarrierInit();
    }
    if (warp == L::kMmaWarp)
        tmemAllocGroup<CG>(tmemSlot, 512);
    dev::tcFenceBefore();
    clusterSync<CG>();
    dev::tcFenceAfter();
    const uint32_t tmem = dev::ldsU32(tmemSlot), tmemA = tmem + L::kBk;
    const uint32_t unit = blockIdx.x / CG, tiles = p.tilesN * p.tilesK;
    const uint32_t tile = unit % tiles, split = unit / tiles;
    const uint32_t n0 = (tile % p.tilesN * CG + rank) * 128;
    const uint32_t k0 = tile / p.tilesN * L::kBk, kMine = k0 + rank * L::kBCols;
    const uint64_t begin = uint64_t(split) * p.rowsPerSplit;
    const uint64_t end = min(uint64_t(p.rows), begin + p.rowsPerSplit);
    const uint32_t stages = uint32_t((end - begin + L::kRows - 1) / L::kRows);
    if (warp < L::kEpilogueWarps) {
        registersUp<L::kRegsEpilogue>();
        const uint32_t quarter = warp % 4, half = warp / 4;
        float sum[128];
#pragma unroll
        for (int i = 0; i < 128; ++i)
            sum[i] = 0.0f;
        bool ok = true;
        const uint32_t flushes = (stages + L::kFlush - 1) / L::kFlush;
        for (uint32_t e = 0; e < flushes; ++e) {
            if (!waitPhase(accFull, e & 1)) {
                ok = false;
                break;
            }
            dev::tcFenceAfter();
#pragma unroll
            for (int c = 0; c < 128; c += 8) {
                uint32_t r[8];
                tcLoad32x32bx8(tmem + half * 128 + c + (quarter << 21), r);
                dev::tcWaitLd();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sum[c + i] = fmaf(__uint_as_float(r[i]), 2.0f, sum[c + i]); // B holds half of q^
            }
            dev::tcFenceBefore();
            __syncwarp();
            if (lane == 0)
                arriveLeader<CG>(accEmpty);
        }
        if (ok && p.partials != nullptr) {
            float4* out = reinterpret_cast<float4*>(p.partials) + uint64_t(blockIdx.x) * (128 * L::kBk / 4) + half * 32 * 128 +
                          32 * quarter + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i)
                out[128 * i] = make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
        } else if (ok) {
            // Boxes of 32 x 32 through the raw ring, which nothing uses any more, swizzled as the map says:
            // by TMA, which adds them where they go for accumulate, or, where rows do not start and end on
            // 16 bytes, row by row with neighbouring lanes on neighbouring columns.
            const uint32_t buf = base + L::kRawOff + warp * 4096, r = laneColumn(lane);
#pragma unroll
            for (int box = 0; box < 4; ++box) {
                const uint32_t x = k0 + 128 * half + 32 * box, y = n0 + 32 * quarter;
                if (p.dwTma && lane == 0)
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};"
                                 ::"r"(buf + r * 128 + ((j ^ r) & 7) * 16), "f"(sum[32 * box + 4 * j]),
                                 "f"(sum[32 * box + 4 * j + 1]), "f"(sum[32 * box + 4 * j + 2]),
                                 "f"(sum[32 * box + 4 * j + 3])
                                 : "memory");
                if (p.dwTma) {
                    dev::fenceProxyAsyncShared();
                    __syncwarp();
                    if (lane == 0 && x < p.k && y < p.n) {
                        if (p.accumulate)
                            asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];"
                                         ::"l"(&mapDw), "r"(x), "r"(y), "r"(buf)
                                         : "memory");
                        else
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                                         ::"l"(&mapDw), "r"(x), "r"(y), "r"(buf)
                                         : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    __syncwarp();
                    if (x + lane < p.k)
                        for (uint32_t i = 0; i < 32 && y + i < p.n; ++i) {
                            float* out = p.dw + uint64_t(y + i) * p.dwStride + x + lane;
                            const float v = __uint_as_float(dev::ldsU32(buf + i * 128 + (((lane / 4) ^ i) & 7) * 16 + lane % 4 * 4));
                            *out = v + (p.accumulate ? *out : 0.0f);
                        }
                }
            }
            if (p.dwTma && lane == 0) // shared memory stays until the copies have read it
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
        }
    } else if (warp < L::kBWarp) {
        registersDown<L::kRegsA>();
        // ---- A: the warp's quarter of the 128 columns of dy; two sets of warps take alternate stages,
        // since a warp spends more time on a stage's waits and fences than on its values ----
        constexpr int kJ = L::kRows / 32; // 16 kJ rows at a time, for the registers
        const uint32_t quarter = warp % 4, q4 = lane % 4;
        const uint32_t byte = (32 * quarter + 4 * (lane / 4)) * sizeof(T); // of the thread's columns in a raw row
        const uint32_t from = base + L::kRawOff + byte / 128 * L::kBox, within = byte % 128;
        for (uint32_t it = warp / 4 % 2; it < stages; it += 2) {
            const uint32_t raw = it % L::kRaw, s = it % L::kStages;
            if (!waitPhase(rawFull + 8 * raw, it / L::kRaw & 1) || !waitPhase(empty + 8 * s, (it / L::kStages + 1) & 1))
                break;
            dev::tcFenceAfter();
            const uint32_t src = from + raw * L::kRawBytes;
            const uint32_t to = tmemA + s * L::kACols + (quarter << 21);
            // Loads in batches: the compiler keeps the order of these accesses, and a load behind a store
            // would wait for what the store needs.
#pragma unroll
            for (int j0 = 0; j0 < L::kRows / 16; j0 += kJ) {
            Quad<T> quads[kJ][4]; // operand rows 16 (j0 + j) + 4 q4 + i
#pragma unroll
            for (int j = 0; j < kJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t r = 16 * (j0 + j) + 8 * (i / 2) + 2 * q4 + i % 2;
                    quads[j][i] = loadQuad<T>(src + r * 128 + (within ^ ((r & 7) << 4)));
                }
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                const Quad<T>(&q)[4] = quads[j];
                auto put = [&](auto check) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t out[4][L::kP];
#pragma unroll
                        for (int x = 0; x < 4; ++x) // lane t / 4 + 8 (x / 2), column 8 j + 2 q4 + x % 2
                            splitPair<T, decltype(check)::value != 0>(q[2 * (x % 2)], q[2 * (x % 2) + 1], 2 * half + x / 2,
                                                                      out[x]);
#pragma unroll
                        for (int m = 0; m < L::kP; ++m)
                            tcStore16x256b(to + m * (L::kRows / 2) + 8 * (j0 + j) + (half << 20), out[0][m], out[1][m],
                                           out[2][m], out[3][m]);
                    }
                };
                if (L::kP > 1 && mayNotBeFinite<T>(q))
                    put(Const<1>{});
                else
                    put(Const<0>{});
            }
            }
            dev::tcWaitSt();
            dev::tcFenceBefore();
            __syncwarp();
            if (lane == 0) {
                dev::mbarArrive(rawEmpty + 8 * raw);
                dev::mbarArrive(full + 8 * s);
            }
        }
    } else if (warp < L::kLoadWarp) {
        registersDown<L::kRegsB>();
        // ---- B: a quarter of the stage's rows per warp, 16 lanes of 8 columns per row and box; two sets
        // of warps, as for A ----
        constexpr uint32_t kWarpRows = L::kRows / 4;
        const uint32_t c = lane % 16, row0 = warp % 4 * kWarpRows + lane / 16;
        // No load from global memory here: the proxy fence below would wait for it.
        for (uint32_t it = warp / 4 % 2; it < stages; it += 2) {
            const uint32_t raw = it % L::kRaw, s = it % L::kStages;
            if (!waitPhase(rawFull + 8 * raw, it / L::kRaw & 1) || !waitPhase(empty + 8 * s, (it / L::kStages + 1) & 1))
                break;
            const uint32_t scales = base + L::kScaleOff + raw * L::kScaleBytes;
            const uint32_t src = base + L::kRawOff + raw * L::kRawBytes + L::kABoxes * L::kBox;
            const uint32_t to = base + s * L::kBBytes;
#pragma unroll
            for (int batch = 0; batch < L::kBBoxes * int(kWarpRows) / 8; ++batch) {
                const uint32_t box = batch / (kWarpRows / 8), r0 = row0 + batch % (kWarpRows / 8) * 8;
                uint2 w[4];
                uint32_t scale[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    w[i] = dev::ldsV2(src + box * L::kBox + (r0 + 2 * i) * 128 + 8 * c);
                    scale[i] = dev::ldsU32(scales + 4 * (box * L::kRows + r0 + 2 * i));
                }
                // Rows r0 + 2 i stand at operand rows k + 4 i, k = operandRow(r0), so their pieces lie 512
                // bytes apart, in one of two swizzled places.
                const uint32_t k = operandRow(r0), piece = (c ^ k) & 7;
                const uint32_t at = to + (2 * box + c / 8) * L::kBox + k * 128;
                const uint32_t even = at + piece * 16, odd = at + 512 + (piece ^ 4) * 16;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    uint32_t o[4];
                    int8ToBf16(w[i].x, scale[i], o[0], o[1]);
                    int8ToBf16(w[i].y, scale[i], o[2], o[3]);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                                 ::"r"((i % 2 ? odd : even) + i / 2 * 1024), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                                 : "memory");
                }
            }
            dev::fenceProxyAsyncShared();
            __syncwarp();
            if (lane == 0) {
                dev::mbarArrive(rawEmpty + 8 * raw);
                dev::mbarArrive(full + 8 * s);
            }
        }
    } else {
        registersDown<L::kRegsIssue>();
        if (warp == L::kMmaWarp) {
            if (rank == 0) {
                // ---- MMA issue, by the whole warp in uniform control flow ----
                const uint32_t elected = electLane();
                uint32_t slot = 0, phase = 0, untilFlush = L::kFlush, flushes = 0;
                bool fresh = true; // the next MMA overwrites the accumulator
                for (uint32_t x = 0; x < stages; ++x) {
                    if (!waitPhase(full + 8 * slot, phase) || (CG == 2 && !waitPhase(peerFull + 8 * slot, phase)))
                        break;
                    if (fresh && flushes != 0 && !waitPhase(accEmpty, (flushes - 1) & 1))
                        break;
                    dev::tcFenceAfter();
                    const uint32_t a = tmemA + slot * L::kACols;
                    const uint64_t desc = swizzledDesc(base + slot * L::kBBytes, L::kBox, 1024);
#pragma unroll
                    for (int j = 0; j < L::kRows / 16; ++j)
#pragma unroll
                        for (int m = 0; m < L::kP; ++m)
                            mmaBf16Ts<CG>(elected, tmem, a + m * (L::kRows / 2) + 8 * j, desc + 128 * j,
                                          bf16Idesc(128 * CG, 256), j + m != 0 ? 1u : uint32_t(!fresh));
                    fresh = false;
                    commitCluster<CG>(elected, empty + 8 * slot);
                    if (++slot == L::kStages)
                        slot = 0, phase ^= 1;
                    if (--untilFlush == 0 || x + 1 == stages) {
                        commitCluster<CG>(elected, accFull);
                        untilFlush = L::kFlush;
                        fresh = true;
                        ++flushes;
                    }
                }
            } else if (lane == 0) {
                // ---- the second CTA of a pair passes its full stages on ----
                uint32_t s = 0, phase = 0;
                for (uint32_t it = 0; it < stages; ++it) {
                    if (!waitPhase(full + 8 * s, phase))
                        break;
                    arriveLeader<CG>(peerFull + 8 * s);
                    if (++s == L::kStages)
                        s = 0, phase ^= 1;
                }
            }
        } else if constexpr (TMA) {
            if (warp == L::kLoadWarp && lane == 0) {
                tmaPrefetchMap(&mapDy);
                tmaPrefetchMap(&mapQ);
                uint32_t raw = 0, phase = 1, it = 0;
                bool ok = true;
                for (; it < stages; ++it) {
                    if (!waitPhase(rawEmpty + 8 * raw, phase)) {
                        ok = false;
                        break;
                    }
                    const uint32_t to = base + L::kRawOff + raw * L::kRawBytes, bar = rawFull + 8 * raw;
                    const uint32_t r = uint32_t(begin) + it * L::kRows;
                    dev::mbarArriveExpectTx(bar, L::kRawBytes);
#pragma unroll
                    for (int i = 0; i < L::kABoxes; ++i)
                        tmaLoad2d(to + i * L::kBox, &mapDy, n0 + i * (128 / uint32_t(sizeof(T))), r, bar);
#pragma unroll
                    for (int i = 0; i < L::kBBoxes; ++i)
                        tmaLoad2d(to + (L::kABoxes + i) * L::kBox, &mapQ, kMine + 128 * i, r, bar);
                    if (++raw == L::kRaw)
                        raw = 0, phase ^= 1;
                }
                // After a wait that ran out, no copy may still be on its way when the CTA exits.
                if (!ok)
                    for (uint32_t i = it < L::kRaw ? 0 : it - L::kRaw; i < it; ++i)
                        waitPhase(rawFull + 8 * (i % L::kRaw), (i / L::kRaw) & 1);
            } else if (warp != L::kLoadWarp) {
                // ---- scale bytes: two warps take alternate stages, loaded two of their stages ahead and
                // brought into L2 before; rows and blocks outside count 1.0 ----
                constexpr int kLoads = L::kRows * L::kBBoxes / 32;
                constexpr uint32_t kEarly = 12; // stages
                const uint32_t kBlocks = (p.k + kBlock - 1) / kBlock;
                uint32_t held[2][kLoads];
                auto place = [&](uint32_t it, int i, const uint8_t*& at) {
                    const uint32_t item = 32 * i + lane, col = kMine / kBlock + item / L::kRows;
                    const uint64_t r = begin + uint64_t(it) * L::kRows + item % L::kRows;
                    at = p.scales + r * kBlocks + col;
                    return r < end && col < kBlocks;
                };
                auto fetch = [&](uint32_t it, uint32_t (&v)[kLoads]) {
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        const uint8_t* at;
                        v[i] = place(it, i, at) ? uint32_t(__ldg(at)) : 127u;
                    }
                };
                const uint32_t first = warp - L::kLoadWarp - 1;
                fetch(first, held[0]);
                fetch(first + 2, held[1]);
                bool ok = true;
                for (uint32_t it = first; it < stages && ok; it += 4)
#pragma unroll
                    for (uint32_t u = 0; u < 2; ++u) {
                        const uint32_t stage = it + 2 * u, raw = stage % L::kRaw;
                        if (ok && stage < stages) {
                            ok = waitPhase(rawEmpty + 8 * raw, (stage / L::kRaw + 1) & 1);
#pragma unroll
                            for (int i = 0; i < kLoads; ++i)
                                stsU32(base + L::kScaleOff + raw * L::kScaleBytes + 4 * (32 * i + lane), halfScalePair(held[u][i]));
                            __syncwarp();
                            if (lane == 0)
                                dev::mbarArrive(rawFull + 8 * raw);
                            fetch(stage + 4, held[u]);
#pragma unroll
                            for (int i = 0; i < kLoads; ++i) {
                                const uint8_t* at;
                                if (place(stage + kEarly, i, at))
                                    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
                            }
                        }
                    }
            }
        } else {
            // ---- raw stages by three warps, for rows that do not start on 16 bytes: pieces of dy and of q
            // as wide as their rows' alignment allows ----
            if (p.dyAlign >= 8)
                p.qAlign >= 4 ? loadRaw<T, CG, 8, 4>(p, base, rawFull, rawEmpty, warp - L::kLoadWarp, lane, begin, end, stages, n0, kMine)
                              : loadRaw<T, CG, 8, 1>(p, base, rawFull, rawEmpty, warp - L::kLoadWarp, lane, begin, end, stages, n0, kMine);
            else if (p.dyAlign >= 4)
                p.qAlign >= 4 ? loadRaw<T, CG, 4, 4>(p, base, rawFull, rawEmpty, warp - L::kLoadWarp, lane, begin, end, stages, n0, kMine)
                              : loadRaw<T, CG, 4, 1>(p, base, rawFull, rawEmpty, warp - L::kLoadWarp, lane, begin, end, stages, n0, kMine);
            else if constexpr (sizeof(T) == 2)
                p.qAlign >= 4 ? loadRaw<T, CG, 2, 4>(p, base, rawFull, rawEmpty, warp - L::kLoadWarp, lane, begin, end, stages, n0, kMine)
                              : loadRaw<T, CG, 2, 1>(p, base, rawFull, rawEmpty, warp - L::kLoadWarp, lane, begin, end, stages, n0, kMine);
        }
    }
    __syncwarp();
    dev::tcFenceBefore();
    clusterSync<CG>(); // no CTA of a pair leaves while the other may still arrive on its barriers
    dev::tcFenceAfter();
    if (warp == L::kMmaWarp)
        tmemDeallocGroup<CG>(tmem, 512);
}

// dW (+)= the partial tiles, added in the order of their row ranges, where there are many within eight
// interleaved sums that are then added in order: the result does not depend on timing. 256 / PARTS float4
// columns of a CTA's partial tile per block, PARTS threads each. (8192 x 1024 x 1024 bf16, four ranges: 35
// -> 26 us for both kernels with PARTS = 1 instead of 8 and stores of 16 bytes.)
template <int CG, int PARTS> __global__ void __launch_bounds__(256) sumPartials(const GradArgs p, uint32_t splits) {
    constexpr uint32_t kPerCta = 128 * 256 / 4, kColumns = 256 / PARTS;
    const uint64_t item = uint64_t(blockIdx.x) * kColumns + threadIdx.x % kColumns;
    const uint32_t cta = uint32_t(item / kPerCta), within = uint32_t(item % kPerCta);
    const uint32_t part = threadIdx.x / kColumns;
    const uint64_t step = uint64_t(p.tilesN) * p.tilesK * CG * kPerCta;
    const float4* in = reinterpret_cast<const float4*>(p.partials) + item;
    float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (uint32_t s = part; s < splits; s += PARTS) {
        const float4 v = __ldcs(in + s * step);
        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
    }
    if constexpr (PARTS > 1) {
        __shared__ float4 sums[PARTS][kColumns];
        sums[part][threadIdx.x % kColumns] = sum;
        __syncthreads();
        if (part != 0)
            return;
        for (int i = 1; i < PARTS; ++i) {
            const float4 v = sums[i][threadIdx.x];
            sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
        }
    }
    const uint32_t l = within % 128, c = within / 128 * 4, tile = cta / CG;
    const uint32_t row = (tile % p.tilesN * CG + cta % CG) * 128 + l / 32 * 32 + laneColumn(l % 32);
    const uint32_t col = tile / p.tilesN * 256 + c;
    if (row >= p.n || col >= p.k)
        return;
    float* out = p.dw + row * p.dwStride + col;
    if (p.dwTma) { // rows start and end on 16 bytes
        float4* to = reinterpret_cast<float4*>(out);
        if (p.accumulate) {
            const float4 v = *to;
            sum = make_float4(v.x + sum.x, v.y + sum.y, v.z + sum.z, v.w + sum.w);
        }
        *to = sum;
        return;
    }
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < p.k)
            out[i] = p.accumulate ? out[i] + v[i] : v[i];
}

// How the sum over the rows is split: `splits` ranges of rowsPerSplit rows, one CTA per range and
// tile of dW. More than one range leaves partial tiles, which sumPartials adds. The number of
// ranges is the cheapest by an estimate for 148 SMs: waves of CTAs, each row of a range at the MMA
// rate and each CTA with a fixed start and end, against the partial tiles' traffic through L2 (2048 x 1024 x
// 1024 bf16: 22.6 us in one range, 14.7 us in four).
struct Plan {
    int cg;
    uint32_t tilesN, tilesK, splits, rowsPerSplit;
};
Plan planOf(uint32_t rows, uint32_t n, uint32_t k) {
    constexpr double kSms = 148, kFixedUs = 5, kSumUs = 3;
    Plan p{};
    p.cg = n <= 128 ? 1 : 2;
    p.tilesN = ceilDiv(n, 128u * p.cg);
    p.tilesK = ceilDiv(k, 256u);
    const double tiles = double(p.tilesN) * p.tilesK;
    const uint32_t steps = std::max(1u, ceilDiv(rows, 64u));
    const double stepUs = 0.4, tileUs = p.cg * 128.0 * 256 * 4 * 2 / 1e7; // 64 rows; a partial tile out and in
    double best = 0;
    const uint32_t most = uint32_t(std::min(double(steps), std::max(4.0, 2 * kSms / (tiles * p.cg))));
    for (uint32_t splits = 1; splits <= most; ++splits) {
        const uint32_t per = ceilDiv(steps, splits);
        if (ceilDiv(steps, per) != splits)
            continue;
        const double waves = std::ceil(tiles * splits * p.cg / kSms);
        const double us = waves * (per * stepUs + kFixedUs) + (splits > 1 ? kSumUs + splits * tiles * tileUs : 0);
        if (splits == 1 || us < best) {
            best = us;
            p.splits = splits;
            p.rowsPerSplit = per * 64;
        }
    }
    return p;
}
uint64_t workspaceBytes(const Plan& p) {
    return p.splits > 1 ? uint64_t(p.splits) * p.tilesN * p.tilesK * p.cg * 128 * 256 * 4 : 0;
}

template <typename T, int CG, bool TMA>
void launchTiles(const GradArgs& g, const Plan& p, int type, cudaStream_t stream) {
    using L = GradTile<T, CG>;
    constexpr auto kernel = gradTiles<T, CG, TMA>;
    static const int regs = [] {
        cudaFuncAttributes attr{};
        checkCudaCall(cudaFuncGetAttributes(&attr, gradTiles<T, CG, TMA>));
        return attr.numRegs;
    }();
    if (!L::sharesFit(regs))
        throw CudaError("weight_grad_int8 was built with an unexpected register count");
    const uint64_t grid = uint64_t(p.tilesN) * p.tilesK * p.splits * CG;
    require(grid <= 0x7FFFFFFFull, "too many output tiles for one call");
    CUtensorMap mapDy{}, mapQ{}, mapDw{};
    if (g.dwTma)
        mapDw = tensorMap2d(g.dw, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, g.n, g.k, g.dwStride, 32, 32);
    if constexpr (TMA) {
        const auto t = type == TCC_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == TCC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        mapDy = tensorMap2d(g.dy, t, sizeof(T), g.rows, g.n, g.dyStride, L::kRows, 128 / sizeof(T));
        mapQ = tensorMap2d(g.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.rows, g.k, g.qStride, L::kRows, 128,
                           CU_TENSOR_MAP_SWIZZLE_NONE);
    }
    allowSharedMemory<gradTiles<T, CG, TMA>>(L::kBytes);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(uint32_t(grid));
    config.blockDim = dim3(L::kThreads);
    config.dynamicSmemBytes = L::kBytes;
    config.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CG, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    checkCudaCall(cudaLaunchKernelEx(&config, kernel, mapDy, mapQ, mapDw, g));
    if (p.splits > 1) {
        // Few ranges: one thread's loads of a column are in flight together. Many: the columns are few.
        const uint32_t columns = p.tilesN * p.tilesK * CG * (128 * 256 / 4);
        if (p.splits <= 8)
            sumPartials<CG, 1><<<columns / 256, 256, 0, stream>>>(g, p.splits);
        else
            sumPartials<CG, 8><<<columns / 32, 256, 0, stream>>>(g, p.splits);
        checkCudaCall(cudaGetLastError());
    }
}
template <typename T> void launchGrad(const GradArgs& g, const Plan& p, int type, bool tma, cudaStream_t stream) {
    if (p.cg == 1)
        tma ? launchTiles<T, 1, true>(g, p, type, stream) : launchTiles<T, 1, false>(g, p, type, stream);
    else
        tma ? launchTiles<T, 2, true>(g, p, type, stream) : launchTiles<T, 2, false>(g, p, type, stream);
}

} // namespace

uint32_t weightGradDeviceStatus(bool reset) { return denseStatus(reset); }

} // namespace tcc

extern "C" {

int tcc_weight_grad_int8_workspace_size(uint32_t rows, uint32_t n, uint32_t k, uint64_t* bytes) {
    using namespace tcc;
    return guarded([&] {
        require(bytes != nullptr, "workspace size requires an output");
        require(std::max({rows, n, k}) <= kLargestSize, "weight_grad_int8: a size is too large");
        *bytes = n == 0 || k == 0 ? 0 : workspaceBytes(planOf(rows, n, k));
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
        const uint64_t need = workspaceBytes(p);
        require(need == 0 || (workspace != nullptr && workspace_bytes >= need && alignedTo(workspace, 16)),
                "weight_grad_int8 needs a 16-byte aligned workspace of weight_grad_int8_workspace_size bytes");
        GradArgs g{};
        g.dy = grad_y, g.dyStride = grad_y_stride;
        g.q = reinterpret_cast<const uint8_t*>(q), g.qStride = q_stride;
        g.scales = scales;
        g.dw = grad_w, g.dwStride = grad_w_stride;
        g.partials = need != 0 ? static_cast<float*>(workspace) : nullptr;
        g.rows = rows, g.n = n, g.k = k;
        g.tilesN = p.tilesN, g.tilesK = p.tilesK, g.rowsPerSplit = p.rowsPerSplit;
        g.accumulate = accumulate != 0;
        const uint64_t dyBytes = grad_y_stride * typeBytes(type);
        g.dyAlign = rowsAlignedTo(grad_y, dyBytes, 8) ? 8 : rowsAlignedTo(grad_y, dyBytes, 4) ? 4 : 2;
        g.qAlign = rowsAlignedTo(q, q_stride, 4) ? 4 : 1;
        // A TMA store writes whole 16-byte pieces of a row: k has to end one, or the next columns change.
        g.dwTma = rowsAlignedTo(grad_w, grad_w_stride * 4, 16) && k % 4 == 0 && grad_w_stride < (1ull << 38) &&
                  std::max(n, k) <= 0x7FFFFF00u;
        const bool tma = rows != 0 && rowsAlignedTo(grad_y, grad_y_stride * typeBytes(type), 16) &&
                         rowsAlignedTo(q, q_stride, 16) && grad_y_stride < (1ull << 38) && q_stride < (1ull << 40) &&
                         std::max({rows, n, k}) <= 0x7FFFFF00u; // coordinates of a copy are signed
        auto s = reinterpret_cast<cudaStream_t>(stream);
        switch (type) {
        case TCC_F32: launchGrad<float>(g, p, type, tma, s); break;
        case TCC_BF16: launchGrad<__nv_bfloat16>(g, p, type, tma, s); break;
        default: launchGrad<__half>(g, p, type, tma, s); break;
        }
    });
}

} // extern "C"
