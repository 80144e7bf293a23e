// Weight gradient of a linear layer whose input was kept as an INT8 checkpoint, on sm_100a:
//   dW[n, k] (+)= sum over rows r of dy[r, n] * q[r, k] 2^e[r, k / 128]
//
// The sum runs on the tensor cores in bf16 with FP32 accumulators, and no operand is rounded: an
// INT8 element times a power of two has at most 8 significant bits, which bf16 holds, and dy is
// split into P bf16 parts that add up to it (P = 1 for bf16, 2 for fp16: 8 + 3 bits, 3 for fp32:
// 8 + 8 + 8 bits), each multiplied on its own into the same accumulator.
//
// A CTA computes 128 rows of dW (n) by BK columns (k) over a range of rows r. dy^T is operand A in
// tensor memory: a thread loads four neighbouring columns of a row at a time and pairs rows with
// byte permutes, so A never passes through shared memory, whose bandwidth the B side needs. q^ is
// operand B in shared memory, row-major as it comes (MN-major, 128-byte swizzle), converted on the
// way by warps of their own. Two sets of producer warps take alternate stages, so the global loads
// of one run under the conversions of the other; one thread issues the MMAs.
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
    float* partials; // [split][tile][BK / 4][128][4], null when the rows are not split
    uint32_t rows, n, k;
    uint32_t tilesN, tilesK, rowsPerSplit;
    bool accumulate, vectorDy, vectorQ;
    int dwAlign; // 32, 16 or 0 bytes that every row of dw starts on
};

template <typename T> constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
template <> constexpr int kParts<__half> = 2;

template <typename T, int BK> struct GradTile {
    static constexpr int kP = kParts<T>;
    static constexpr int kRows = kP == 3 ? 32 : 64; // rows per stage
    static constexpr int kStages = 4;
    static constexpr int kBBytes = kRows * BK * 2;
    static constexpr int kACols = kP * kRows / 2;   // tensor-memory columns of a stage of A
    static constexpr int kBarOff = kStages * kBBytes;
    static constexpr int kNeed = kBarOff + 8 * (2 * kStages + 1) + 16 + 1024;
    // At least half of the shared memory: a second CTA on the SM would wait for tensor memory.
    static constexpr int kBytes = kNeed > 120 * 1024 ? kNeed : 120 * 1024;
    static constexpr int kCols = BK + kStages * kACols;
    static constexpr int kTmemCols = kCols <= 256 ? 256 : 512;
    static constexpr int kAWarps = 8, kBWarps = 8, kMmaWarp = 16;
    static constexpr int kThreads = 32 * 17;
    static_assert(kCols <= 512 && kBytes <= 232448, "resources");
};

// kind::f16 with FP32 accumulators (bits 4-5 = 1), bf16 A and B (bits 7-9 and 10-12 = 1), B
// MN-major (bit 16), N / 8 in bits 17-22 and M / 16 in bits 24-28.
__host__ __device__ constexpr uint32_t bf16Idesc(uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// D(tmem) (+)= A(tmem, bf16) x B(shared memory, bf16).
__device__ __forceinline__ void mmaBf16Ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}

// Four neighbouring columns of one row of dy, as loaded.
template <typename T> struct Quad { uint32_t w[sizeof(T)]; };

template <typename T> __device__ __forceinline__ Quad<T> loadQuad(const T* p, uint32_t left, bool vector) {
    Quad<T> v;
    if (vector && left >= 4) {
        if constexpr (sizeof(T) == 4) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            v.w[0] = u.x, v.w[1] = u.y, v.w[2] = u.z, v.w[3] = u.w;
        } else {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
            v.w[0] = u.x, v.w[1] = u.y;
        }
    } else {
        const uint32_t zero = 0;
#pragma unroll
        for (int i = 0; i < int(sizeof(T)); ++i) {
            if constexpr (sizeof(T) == 4) {
                v.w[i] = uint32_t(i) < left ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : zero;
            } else {
                const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
                v.w[i] = (uint32_t(2 * i) < left ? uint32_t(__ldg(h + 2 * i)) : zero) |
                         (uint32_t(2 * i + 1) < left ? uint32_t(__ldg(h + 2 * i + 1)) << 16 : zero);
            }
        }
    }
    return v;
}

__device__ __forceinline__ uint32_t packBf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What is left of a pair after its bf16 rounding (exact).
__device__ __forceinline__ void subtractBf16(float& lo, float& hi, uint32_t packed) {
    lo -= __uint_as_float(packed << 16);
    hi -= __uint_as_float(packed & 0xFFFF0000u);
}

// Column c (0..3) of two rows' quads as P bf16 pairs (row u in the low half). A part that is not
// finite because the value is not leaves the later parts zero.
template <typename T> __device__ __forceinline__ void splitPair(const Quad<T>& u, const Quad<T>& v, int c, uint32_t (&part)[kParts<T>]) {
    if constexpr (sizeof(T) == 4) {
        float a = __uint_as_float(u.w[c]), b = __uint_as_float(v.w[c]);
        part[0] = packBf16(a, b);
        subtractBf16(a, b, part[0]);
        a = fabsf(a) < INFINITY ? a : 0.0f, b = fabsf(b) < INFINITY ? b : 0.0f;
        part[1] = packBf16(a, b);
        subtractBf16(a, b, part[1]);
        part[2] = packBf16(a, b);
    } else {
        const uint32_t pair = __byte_perm(u.w[c / 2], v.w[c / 2], c % 2 ? 0x7632 : 0x5410);
        if constexpr (kParts<T> == 1) {
            part[0] = pair;
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
            float a = f.x, b = f.y;
            part[0] = packBf16(a, b);
            subtractBf16(a, b, part[0]);
            a = fabsf(a) < INFINITY ? a : 0.0f, b = fabsf(b) < INFINITY ? b : 0.0f;
            part[1] = packBf16(a, b);
        }
    }
}

// Four INT8 elements times a power of two (as a bf16 pair) in bf16: low 7 bits under the exponent
// of 128, minus 128 or, for negative elements, 256. Every step is exact.
__device__ __forceinline__ void int8ToBf16(uint32_t w, __nv_bfloat162 scale, uint32_t& lo, uint32_t& hi) {
    const uint32_t x[2] = {__byte_perm(w, 0u, 0x4140), __byte_perm(w, 0u, 0x4342)};
    uint32_t out[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = (x[i] & 0x007F007Fu) | 0x43004300u, c = (x[i] & 0x00800080u) | 0xC300C300u;
        const __nv_bfloat162 f = __hmul2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                                 *reinterpret_cast<const __nv_bfloat162*>(&c)), scale);
        out[i] = *reinterpret_cast<const uint32_t*>(&f);
    }
    lo = out[0], hi = out[1];
}
// 2^e of a scale byte as a bf16 pair (NaN for 255, a subnormal for 0).
__device__ __forceinline__ __nv_bfloat162 scalePair(uint32_t byte) {
    const uint32_t h = byte == 255u ? 0x7FC0u : byte == 0u ? 0x0040u : byte << 7;
    const uint32_t w = h * 0x10001u;
    return *reinterpret_cast<const __nv_bfloat162*>(&w);
}

// Lane of a 32-lane quarter of A and D -> column of dy within the quarter's 32: the 16-lane store
// writes lanes t / 4 and t / 4 + 8 from thread t, which holds columns 4 (t / 4) .. + 3; the first
// half of the quarter takes columns 0 and 1 of each four, the second half 2 and 3.
__device__ __forceinline__ uint32_t laneColumn(uint32_t l) { return 4 * (l % 8) + 2 * (l / 16) + (l / 8) % 2; }

template <int REPEAT> __device__ __forceinline__ void storeA(uint32_t taddr, const uint32_t (&r)[4 * REPEAT]) {
    if constexpr (REPEAT == 4)
        dev::tcStore16x256bx4(taddr, r);
    else
        dev::tcStore16x256bx2(taddr, r);
}

template <typename T, int BK>
__global__ void __launch_bounds__(GradTile<T, BK>::kThreads, 1) gradTiles(const GradArgs p) {
    using L = GradTile<T, BK>;
    extern __shared__ unsigned char smemRaw[];
    const uint32_t base = (dev::smemAddr(smemRaw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = base + L::kBarOff, empty = full + 8 * L::kStages, done = empty + 8 * L::kStages;
    const uint32_t tmemSlot = done + 8;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i)
            dev::mbarInit(full + 8 * i, 8), dev::mbarInit(empty + 8 * i, 1); // 4 warps of A, 4 of B
        dev::mbarInit(done, 1);
        dev::fenceBarrierInit();
    }
    if (warp == L::kMmaWarp) {
        dev::tmemAlloc(tmemSlot, L::kTmemCols);
        dev::tmemRelinquish();
    }
    dev::tcFenceBefore();
    __syncthreads();
    dev::tcFenceAfter();
    const uint32_t tmem = dev::ldsU32(tmemSlot);
    const uint32_t tiles = p.tilesN * p.tilesK;
    const uint32_t tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
    const uint32_t n0 = tile % p.tilesN * 128, k0 = tile / p.tilesN * BK;
    const uint64_t begin = uint64_t(split) * p.rowsPerSplit;
    const uint64_t end = min(uint64_t(p.rows), begin + p.rowsPerSplit);
    const uint32_t stages = uint32_t((end - begin + L::kRows - 1) / L::kRows);

    if (warp < L::kAWarps) {
        // ---- A: stages warp / 4, + 2, ...; the warp's quarter of the 128 columns of dy ----
        const uint32_t quarter = warp % 4, q4 = lane % 4;
        const uint32_t col = n0 + 32 * quarter + 4 * (lane / 4);
        const uint32_t left = col < p.n ? p.n - col : 0u;
        const T* dy = static_cast<const T*>(p.dy);
        constexpr int kJ = L::kRows / 16;
        Quad<T> held[kJ][4]; // rows 16 j + 4 q4 + i
        auto fetch = [&](uint32_t it) {
            const uint64_t r0 = begin + uint64_t(it) * L::kRows + 4 * q4;
#pragma unroll
            for (int j = 0; j < kJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint64_t r = r0 + 16 * j + i;
                    held[j][i] = loadQuad<T>(dy + r * p.dyStride + col, r < end ? left : 0u, p.vectorDy);
                }
        };
        uint32_t it = warp / 4;
        if (it < stages)
            fetch(it);
        for (; it < stages; it += 2) {
            const uint32_t s = it % L::kStages, turn = it / L::kStages;
            if (turn != 0 && !waitPhase(empty + 8 * s, (turn - 1) & 1))
                break;
            dev::tcFenceAfter();
            const uint32_t to = tmem + BK + s * L::kACols + (quarter << 21);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t out[L::kP][4 * kJ];
#pragma unroll
                for (int j = 0; j < kJ; ++j)
#pragma unroll
                    for (int x = 0; x < 4; ++x) { // lane t / 4 + 8 (x / 2), column 8 j + 2 q4 + x % 2
                        uint32_t part[L::kP];
                        splitPair<T>(held[j][2 * (x % 2)], held[j][2 * (x % 2) + 1], 2 * half + x / 2, part);
#pragma unroll
                        for (int m = 0; m < L::kP; ++m)
                            out[m][4 * j + x] = part[m];
                    }
#pragma unroll
                for (int m = 0; m < L::kP; ++m)
                    storeA<kJ>(to + m * (L::kRows / 2) + (half << 20), out[m]);
            }
            dev::tcWaitSt();
            dev::tcFenceBefore();
            __syncwarp();
            if (lane == 0)
                dev::mbarArrive(full + 8 * s);
            if (it + 2 < stages)
                fetch(it + 2);
        }
    } else if (warp < L::kAWarps + L::kBWarps) {
        // ---- B: stages (warp - 8) / 4, + 2, ...; a quarter of the stage's rows per warp ----
        constexpr int kLanes = BK / 8;              // lanes per row, 8 elements each
        constexpr int kRowsAtOnce = 32 / kLanes;
        constexpr int kWarpRows = L::kRows / 4;
        constexpr int kLoads = kWarpRows / kRowsAtOnce;
        constexpr int kKb = BK / 128;
        const uint32_t w = warp % 4;
        const uint32_t kk = lane % kLanes * 8, k = k0 + kk;
        const uint32_t left = k < p.k ? p.k - k : 0u;
        const uint32_t kBlocks = (p.k + kBlock - 1) / kBlock;
        const uint32_t scaleRow = lane / kKb, scaleCol = k0 / kBlock + lane % kKb;
        uint2 held[kLoads];
        uint32_t heldScale = 127;
        auto fetch = [&](uint32_t it) {
            const uint64_t r0 = begin + uint64_t(it) * L::kRows + w * kWarpRows;
            heldScale = scaleRow < uint32_t(kWarpRows) && r0 + scaleRow < end && scaleCol < kBlocks
                            ? __ldg(p.scales + (r0 + scaleRow) * kBlocks + scaleCol) : 127u;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint64_t r = r0 + i * kRowsAtOnce + lane / kLanes;
                const uint8_t* src = p.q + r * p.qStride + k;
                const uint32_t have = r < end ? left : 0u;
                if (p.vectorQ && have >= 8) {
                    held[i] = __ldg(reinterpret_cast<const uint2*>(src));
                } else {
                    uint32_t b[2] = {0, 0};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (uint32_t(e) < have)
                            b[e / 4] |= uint32_t(__ldg(src + e)) << (8 * (e % 4));
                    held[i] = make_uint2(b[0], b[1]);
                }
            }
        };
        uint32_t it = (warp - L::kAWarps) / 4;
        if (it < stages)
            fetch(it);
        for (; it < stages; it += 2) {
            const uint32_t s = it % L::kStages, turn = it / L::kStages;
            if (turn != 0 && !waitPhase(empty + 8 * s, (turn - 1) & 1))
                break;
            // Column group kk / 64: kRows rows of 128 bytes; 16-byte pieces swizzled by the row.
            const uint32_t to = base + s * L::kBBytes + kk / 64 * (L::kRows * 128);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t row = i * kRowsAtOnce + lane / kLanes;
                const __nv_bfloat162 scale =
                    scalePair(__shfl_sync(0xFFFFFFFFu, heldScale, row * kKb + kk / 128));
                uint32_t o[4];
                int8ToBf16(held[i].x, scale, o[0], o[1]);
                int8ToBf16(held[i].y, scale, o[2], o[3]);
                const uint32_t r = w * kWarpRows + row;
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                             ::"r"(to + r * 128 + (((kk / 8) ^ r) & 7) * 16), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                             : "memory");
            }
            dev::fenceProxyAsyncShared();
            __syncwarp();
            if (lane == 0)
                dev::mbarArrive(full + 8 * s);
            if (it + 2 < stages)
                fetch(it + 2);
        }
    } else if (lane == 0) {
        // ---- MMA issue ----
        bool ok = true;
        for (uint32_t it = 0; it < stages; ++it) {
            const uint32_t s = it % L::kStages;
            if (!waitPhase(full + 8 * s, (it / L::kStages) & 1)) {
                ok = false;
                break;
            }
            dev::tcFenceAfter();
            const uint32_t a = tmem + BK + s * L::kACols;
            const uint64_t b = swizzledDesc(base + s * L::kBBytes, L::kRows * 128, 1024);
#pragma unroll
            for (int j = 0; j < L::kRows / 16; ++j)
#pragma unroll
                for (int m = 0; m < L::kP; ++m)
                    mmaBf16Ts(tmem, a + m * (L::kRows / 2) + 8 * j, b + 128 * j, bf16Idesc(BK), (it | j | m) != 0);
            dev::tcCommit(empty + 8 * s);
        }
        if (ok)
            dev::tcCommit(done);
    }
    __syncwarp();
    // ---- dW or a partial tile: eight warps, half of the columns each ----
    if (warp < 8 && (stages == 0 || waitPhase(done, 0))) {
        dev::tcFenceAfter();
        const uint32_t quarter = warp % 4, half = warp / 4;
        const uint32_t row = n0 + 32 * quarter + laneColumn(lane);
#pragma unroll
        for (int c = 0; c < BK / 2; c += 32) {
            const uint32_t col = half * (BK / 2) + c;
            uint32_t r[32];
            if (stages != 0) {
                tcLoad32x32bx32(tmem + col + (quarter << 21), r);
                dev::tcWaitLd();
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    r[i] = 0u;
            }
            if (p.partials != nullptr) {
                float4* out = reinterpret_cast<float4*>(p.partials) + uint64_t(blockIdx.x) * (128 * BK / 4) +
                              (col / 4) * 128 + 32 * quarter + lane;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    out[128 * i] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                               __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
            } else if (row < p.n) {
                float* out = p.dw + row * p.dwStride + k0 + col;
                if (p.dwAlign != 0 && k0 + col + 32 <= p.k) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float4 v = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                               __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
                        float4* o = reinterpret_cast<float4*>(out) + i;
                        if (p.accumulate) {
                            const float4 was = *o;
                            v = make_float4(v.x + was.x, v.y + was.y, v.z + was.z, v.w + was.w);
                        }
                        *o = v;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (k0 + col + i < p.k)
                            out[i] = __uint_as_float(r[i]) + (p.accumulate ? out[i] : 0.0f);
                }
            }
        }
    }
    dev::tcFenceBefore();
    __syncthreads();
    dev::tcFenceAfter();
    if (warp == L::kMmaWarp)
        dev::tmemDealloc(tmem, L::kTmemCols);
}

// dW (+)= the partial tiles, added in the order of their row ranges within eight interleaved sums
// that are then added in order: the result does not depend on timing. 32 float4 columns of a
// partial tile per CTA, eight threads each.
__global__ void __launch_bounds__(256) sumPartials(const GradArgs p, uint32_t splits, uint32_t bk) {
    __shared__ float4 sums[8][32];
    const uint32_t perTile = 128 * bk / 4;
    const uint64_t item = uint64_t(blockIdx.x) * 32 + threadIdx.x % 32;
    const uint32_t tile = uint32_t(item / perTile), within = uint32_t(item % perTile);
    const uint32_t part = threadIdx.x / 32;
    const uint64_t step = uint64_t(p.tilesN) * p.tilesK * perTile;
    const float4* in = reinterpret_cast<const float4*>(p.partials) + item;
    float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (uint32_t s = part; s < splits; s += 8) {
        const float4 v = __ldcs(in + s * step);
        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
    }
    sums[part][threadIdx.x % 32] = sum;
    __syncthreads();
    if (part != 0)
        return;
    for (int i = 1; i < 8; ++i) {
        const float4 v = sums[i][threadIdx.x];
        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
    }
    const uint32_t l = within % 128, row = tile % p.tilesN * 128 + l / 32 * 32 + laneColumn(l % 32);
    const uint32_t col = tile / p.tilesN * bk + within / 128 * 4;
    if (row >= p.n || col >= p.k)
        return;
    float* out = p.dw + row * p.dwStride + col;
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < p.k)
            out[i] = p.accumulate ? out[i] + v[i] : v[i];
}

// How the sum over the rows is split: `splits` ranges of rowsPerSplit rows, one CTA per range and
// tile of dW. More than one range leaves partial tiles, which sumPartials adds. The number of
// ranges is the cheapest by an estimate for 148 SMs: waves of CTAs, each row of a range at the MMA
// rate and each CTA with a fixed start and end, against the partial tiles' traffic.
struct Plan {
    uint32_t bk, tilesN, tilesK, splits, rowsPerSplit;
};
Plan planOf(uint32_t rows, uint32_t n, uint32_t k) {
    constexpr double kSms = 148, kFixedUs = 4, kSumUs = 4;
    Plan p{};
    p.bk = k <= 128 ? 128 : 256;
    p.tilesN = ceilDiv(n, 128u);
    p.tilesK = ceilDiv(k, p.bk);
    const double tiles = double(p.tilesN) * p.tilesK;
    const uint32_t steps = std::max(1u, ceilDiv(rows, 64u));
    const double stepUs = 0.35 * p.bk / 256, tileUs = 128.0 * p.bk * 4 * 2 / 5e6; // a partial tile out and in
    double best = 0;
    for (uint32_t splits = 1; splits <= steps && splits <= 296; ++splits) {
        const uint32_t per = ceilDiv(steps, splits);
        if (ceilDiv(steps, per) != splits)
            continue;
        const double waves = std::ceil(tiles * splits / kSms);
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
    return p.splits > 1 ? uint64_t(p.splits) * p.tilesN * p.tilesK * 128 * p.bk * 4 : 0;
}

template <typename T, int BK> void launchTiles(const GradArgs& g, const Plan& p, cudaStream_t stream) {
    using L = GradTile<T, BK>;
    const uint64_t grid = uint64_t(p.tilesN) * p.tilesK * p.splits;
    require(grid <= 0x7FFFFFFFull, "too many output tiles for one call");
    allowSharedMemory<gradTiles<T, BK>>(L::kBytes);
    gradTiles<T, BK><<<uint32_t(grid), L::kThreads, L::kBytes, stream>>>(g);
    checkCudaCall(cudaGetLastError());
    if (p.splits > 1) {
        sumPartials<<<p.tilesN * p.tilesK * (128 * BK / 4 / 32), 256, 0, stream>>>(g, p.splits, BK);
        checkCudaCall(cudaGetLastError());
    }
}
template <typename T> void launchGrad(const GradArgs& g, const Plan& p, cudaStream_t stream) {
    p.bk == 128 ? launchTiles<T, 128>(g, p, stream) : launchTiles<T, 256>(g, p, stream);
}

} // namespace

uint32_t weightGradDeviceStatus(bool reset) { return denseStatus(reset); }

} // namespace tcc

extern "C" {

int tcc_weight_grad_int8_workspace_size(uint32_t rows, uint32_t n, uint32_t k, uint64_t* bytes) {
    using namespace tcc;
    return guarded([&] {
        require(bytes != nullptr, "workspace size requires an output");
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
        g.vectorDy = rowsAlignedTo(grad_y, grad_y_stride * typeBytes(type), 4 * typeBytes(type));
        g.vectorQ = rowsAlignedTo(q, q_stride, 8);
        const uint64_t rowBytes = grad_w_stride * 4;
        g.dwAlign = rowsAlignedTo(grad_w, rowBytes, 16) ? 16 : 0;
        auto s = reinterpret_cast<cudaStream_t>(stream);
        switch (type) {
        case TCC_F32: launchGrad<float>(g, p, s); break;
        case TCC_BF16: launchGrad<__nv_bfloat16>(g, p, s); break;
        default: launchGrad<__half>(g, p, s); break;
        }
    });
}

} // extern "C"
