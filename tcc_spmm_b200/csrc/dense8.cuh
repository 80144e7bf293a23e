// Device pieces of the 8-bit block-scaled dense operators: element loads and stores, the scale
// rule, and the activation functions.
//
// A block (128 columns of a row, or of 128 x 128 elements) has one power-of-two scale 2^e, kept as
// the byte e + 127 (E8M0). e is the least exponent with absmax <= 2^e * largest, so x * 2^-e is
// exact and rounding to the 8-bit type is the only rounding; a power of two also makes the
// dequantized int8 value exact in bf16, and is what the tensor core's block-scaled MMA takes.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace tcc {
namespace blk {

constexpr uint32_t kBlock = 128;

enum Elem8 { kInt8 = 0, kE4M3 = 1, kE5M2 = 2 };
enum Act { kRelu = 0, kGelu = 1, kGeluTanh = 2, kSilu = 3, kNone = 4 };

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float toFloat(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T fromFloat(float v);
template <> __device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }

template <typename T> constexpr bool isHalf = false;
template <> constexpr bool isHalf<__half> = true;

// 16 bytes of T as floats, and back.
template <typename T> constexpr int kPer16 = 16 / int(sizeof(T));
template <typename T> __device__ __forceinline__ void unpack16(uint4 w, float (&v)[kPer16<T>]);
template <> __device__ __forceinline__ void unpack16<float>(uint4 w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
}
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(uint4 w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}
template <> __device__ __forceinline__ void unpack16<__half>(uint4 w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
template <typename T> __device__ __forceinline__ uint4 pack16(const float (&v)[kPer16<T>]);
template <> __device__ __forceinline__ uint4 pack16<float>(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <> __device__ __forceinline__ uint4 pack16<__nv_bfloat16>(const float (&v)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
template <> __device__ __forceinline__ uint4 pack16<__half>(const float (&v)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// Running absmax of 16 bytes of T as unsigned words, and its final value as the bits of a float. The
// 16-bit types compare two elements at a time in their own bits, which order as the floats do.
template <typename T> __device__ __forceinline__ uint32_t absmax16(uint4 w, uint32_t top) {
    if constexpr (sizeof(T) == 4) {
        return max(max(max(top, w.x & 0x7FFFFFFFu), max(w.y & 0x7FFFFFFFu, w.z & 0x7FFFFFFFu)), w.w & 0x7FFFFFFFu);
    } else {
        constexpr uint32_t m = 0x7FFF7FFFu;
        return __vmaxu2(__vmaxu2(top, w.x & m), __vmaxu2(__vmaxu2(w.y & m, w.z & m), w.w & m));
    }
}
template <typename T> __device__ __forceinline__ uint32_t absmaxBits(uint32_t top) {
    if constexpr (sizeof(T) == 4)
        return top;
    const uint32_t h = max(top & 0xFFFFu, top >> 16);
    if constexpr (sizeof(T) == 2 && !isHalf<T>)
        return h << 16;
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
}

// ---- scale of a block -------------------------------------------------------------------------
// The scale byte from the bits of the block's absmax (compared as unsigned integers, which order
// non-negative floats, infinity and NaN). largest = 1.75 * 2^8 (E4M3), 1.75 * 2^15 (E5M2) or
// 1.984375 * 2^6 (INT8): adding 2^23 - 1 minus its mantissa carries into the exponent exactly when
// the absmax's mantissa is above it. At least 2^-126, so that the scale and its inverse are normal
// floats; 1 for a block of zeros; 255 (E8M0's NaN) for a block that holds an infinity or NaN.
template <int Q> __device__ __forceinline__ uint32_t scaleByte(uint32_t absmaxBits) {
    constexpr uint32_t carry = Q == kInt8 ? 0x01FFFFu : 0x1FFFFFu;
    constexpr int below = Q == kInt8 ? 6 : Q == kE4M3 ? 8 : 15;
    const int e = max(int((absmaxBits + carry) >> 23) - below, 1);
    return absmaxBits == 0u ? 127u : absmaxBits >= 0x7F800000u ? 255u : uint32_t(e);
}
// 2^-e of a scale byte (byte <= 249 when finite; the NaN byte gives some finite number).
__device__ __forceinline__ float inverseScale(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }
// 2^e of a scale byte, NaN for 255. A byte of 0 (2^-127, which the quantizers do not write) is a
// subnormal float.
__device__ __forceinline__ float scaleValue(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23);
}

// Four floats, already divided by the scale, as 8-bit elements.
template <int Q> __device__ __forceinline__ uint32_t quantize4(float a, float b, float c, float d) {
    if constexpr (Q == kInt8) {
        // 1.5 * 2^23 + v rounds v to a whole number, ties to even, in the low bits.
        const float magic = 12582912.0f;
        const uint32_t ab = __byte_perm(__float_as_uint(a + magic), __float_as_uint(b + magic), 0x0040);
        const uint32_t cd = __byte_perm(__float_as_uint(c + magic), __float_as_uint(d + magic), 0x0040);
        return __byte_perm(ab, cd, 0x5410);
    } else {
        constexpr __nv_fp8_interpretation_t kind = Q == kE4M3 ? __NV_E4M3 : __NV_E5M2;
        const uint32_t ab = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, kind);
        const uint32_t cd = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, kind);
        return ab | (cd << 16);
    }
}
// The bytes of a block whose scale is NaN.
template <int Q> __device__ __forceinline__ uint32_t nanBytes() { return Q == kInt8 ? 0u : 0x7F7F7F7Fu; }

// Byte i of a word of INT8 elements that were flipped to unsigned (word ^ 0x80808080) as a float: the
// byte under the exponent of 2^23, minus 2^23 + 128 (exact; no conversion instruction).
__device__ __forceinline__ float int8At(uint32_t flipped, int i) {
    return __uint_as_float(__byte_perm(flipped, 0x4B000000u, 0x7540 + i)) - 8388736.0f;
}

// ---- activation functions -----------------------------------------------------------------------
// All forms keep the relative accuracy of the left tail, which 1 + erf and 1 + tanh lose, as far as the exponential
// is a normal float. They work
// on pairs, with the packed FP32 instructions (two lanes per issue) where there is a polynomial.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    return (uint64_t(__float_as_uint(b)) << 32) | __float_as_uint(a);
}
__device__ __forceinline__ float2 unpair2(uint64_t v) {
    return make_float2(__uint_as_float(uint32_t(v)), __uint_as_float(uint32_t(v >> 32)));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// The hardware's approximations (2^-22 relative), results below 2^-126 as zero: without the steps
// that keep subnormal results. SiLU is zero below about -87 for it, where it is |x| 2^-126 and less.
__device__ __forceinline__ float exp2Approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocalApprox(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The normal distribution's tail Phi(-|x|) and its density's factor exp(-x^2 / 2), of two values.
// Phi(-a) exp(a^2 / 2) is a smooth function of t = 1 / (1 + 0.3 a): t times a polynomial of degree 7
// fitted to the least largest relative error over 0 <= a <= 14 (1.5e-7; 5e-7 with fp32 arithmetic).
// Beyond a = 16 both are below the smallest float.
struct Tail {
    float2 phi, density;
};
__device__ __forceinline__ Tail normalTail(float x0, float x1) {
    const float a0 = fminf(fabsf(x0), 16.0f), a1 = fminf(fabsf(x1), 16.0f);
    const uint64_t a = pair2(a0, a1);
    const float2 d = unpair2(fma2(a, pair2(0.3f, 0.3f), pair2(1.0f, 1.0f)));
    const uint64_t t = pair2(reciprocalApprox(d.x), reciprocalApprox(d.y));
    const float c[8] = {0.11962928622961044f, 0.12075415253639221f, 0.09991224855184555f, 0.1285656988620758f,
                        -0.053691279143095016f, 0.20636169612407684f, -0.15720775723457336f, 0.03567587584257126f};
    uint64_t s = pair2(c[7], c[7]);
#pragma unroll
    for (int i = 6; i >= 0; --i)
        s = fma2(s, t, pair2(c[i], c[i]));
    const float2 e = unpair2(mul2(mul2(a, a), pair2(-0.72134752044448170f, -0.72134752044448170f))); // -log2(e) / 2
    const uint64_t density = pair2(exp2Approx(e.x), exp2Approx(e.y));
    return {unpair2(mul2(mul2(s, t), density)), unpair2(density)};
}

// 1 / (1 + exp(-x)) by exp(-|x|), so that the divisor stays within [1, 2] and nothing overflows.
__device__ __forceinline__ float logistic(float x) {
    const float t = exp2Approx(-1.4426950408889634f * fabsf(x));
    return (x < 0.0f ? t : 1.0f) * reciprocalApprox(1.0f + t);
}
__device__ __forceinline__ float tanhArgument(float x) { // 2 sqrt(2/pi) (x + 0.044715 x^3)
    return x * (1.5957691216057308f + 0.0713548162726009f * x * x);
}

// f of two values, in place.
template <int A> __device__ __forceinline__ void activation(float& x, float& y) {
    if constexpr (A == kRelu) {
        x = x < 0.0f ? 0.0f : x, y = y < 0.0f ? 0.0f : y;
    } else if constexpr (A == kGelu) { // max(x, 0) - |x| Phi(-|x|)
        const Tail t = normalTail(x, y);
        x = (x < 0.0f ? 0.0f : x) - fminf(fabsf(x), 16.0f) * t.phi.x;
        y = (y < 0.0f ? 0.0f : y) - fminf(fabsf(y), 16.0f) * t.phi.y;
    } else if constexpr (A == kGeluTanh) {
        x *= logistic(tanhArgument(x)), y *= logistic(tanhArgument(y));
    } else if constexpr (A == kSilu) {
        x *= logistic(x), y *= logistic(y);
    }
}
// The scale of a checkpoint's block for the slopes below: 2^e up to 2^20, NaN for 255. From there on every
// element but 0 is beyond 2^20 in size, where a slope is exactly 0 or 1 whatever the size; kept to that, x^ stays
// a float (an element may stand for 2^128) and its square does not overflow (infinity times a factor of 0).
__device__ __forceinline__ float slopeScale(uint32_t byte) { return scaleValue(byte == 255u ? byte : min(byte, 147u)); }

// f' of two values, in place: NaN, or below 2^60 in size.
template <int A> __device__ __forceinline__ void activationSlope(float& x, float& y) {
    if constexpr (A == kRelu) {
        x = x > 0.0f ? 1.0f : x == x ? 0.0f : x, y = y > 0.0f ? 1.0f : y == y ? 0.0f : y;
    } else if constexpr (A == kGelu) { // Phi(x) + x phi(x)
        const Tail t = normalTail(x, y);
        x = (x < 0.0f ? t.phi.x : 1.0f - t.phi.x) + x * (0.3989422804014327f * t.density.x);
        y = (y < 0.0f ? t.phi.y : 1.0f - t.phi.y) + y * (0.3989422804014327f * t.density.y);
    } else if constexpr (A == kGeluTanh) {
        const float s = logistic(tanhArgument(x)), u = logistic(tanhArgument(y));
        x = s + x * s * (1.0f - s) * (1.5957691216057308f + 0.2140644488178027f * x * x);
        y = u + y * u * (1.0f - u) * (1.5957691216057308f + 0.2140644488178027f * y * y);
    } else {
        const float s = logistic(x), u = logistic(y);
        x = s + x * s * (1.0f - s), y = u + y * u * (1.0f - u);
    }
}

} // namespace blk
} // namespace tcc
