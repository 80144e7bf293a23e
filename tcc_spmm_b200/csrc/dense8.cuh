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

__device__ __forceinline__ float int8At(uint32_t word, int i) { return float(int8_t(word >> (8 * i))); }

// ---- activation functions -----------------------------------------------------------------------
// Phi(x) = erfc(-x / sqrt 2) / 2 and the logistic forms keep the relative accuracy of the left tail,
// which 1 + erf and 1 + tanh lose.
__device__ __forceinline__ float normalCdf(float x) { return 0.5f * erfcf(-0.70710678118654752f * x); }
// 1 / (1 + exp(-x)) by exp(-|x|), so that the divisor stays within [1, 2] and nothing overflows.
__device__ __forceinline__ float logistic(float x) {
    const float t = __expf(-fabsf(x));
    return __fdividef(x < 0.0f ? t : 1.0f, 1.0f + t);
}
__device__ __forceinline__ float tanhArgument(float x) { // 2 sqrt(2/pi) (x + 0.044715 x^3)
    return x * (1.5957691216057308f + 0.0713548162726009f * x * x);
}

template <int A> __device__ __forceinline__ float activation(float x) {
    if constexpr (A == kRelu)
        return x < 0.0f ? 0.0f : x;
    else if constexpr (A == kGelu)
        return x * normalCdf(x);
    else if constexpr (A == kGeluTanh)
        return x * logistic(tanhArgument(x));
    else if constexpr (A == kSilu)
        return x * logistic(x);
    else
        return x;
}
template <int A> __device__ __forceinline__ float activationSlope(float x) {
    if constexpr (A == kRelu) {
        return x > 0.0f ? 1.0f : x == x ? 0.0f : x;
    } else if constexpr (A == kGelu) {
        return normalCdf(x) + x * 0.3989422804014327f * __expf(-0.5f * x * x);
    } else if constexpr (A == kGeluTanh) {
        const float s = logistic(tanhArgument(x));
        return s + x * s * (1.0f - s) * (1.5957691216057308f + 0.2140644488178027f * x * x);
    } else {
        const float s = logistic(x);
        return s + x * s * (1.0f - s);
    }
}

} // namespace blk
} // namespace tcc
