// 8-bit KV pools: codes (int8 or e4m3) in one layer's pool [num_blocks, block_size, n_kv_heads, head_dim] and one fp32
// scale per block and KV head (K and V apart): value = code * scale.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace ns {

// Storage kinds of a pool element. kMaxMant / kMaxExp: the largest code's mantissa bits and exponent (127 = 1.984375 * 2^6,
// 448 = 1.75 * 2^8), from which the smallest power-of-two scale that holds a magnitude follows without a division.
// encode: nearest code, ties to even, saturating; NaN gives code 0. encode4: four finite values within the code range, packed.
struct KvInt8 {
    static constexpr uint32_t kMaxMant = 0x7E0000u;
    static constexpr int kMaxExp = 6;
    static __device__ __forceinline__ uint32_t encode(float x) {
        return x == x ? (uint32_t)__float2int_rn(fminf(fmaxf(x, -127.f), 127.f)) & 0xffu : 0u;
    }
    static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
        // adding 1.5 * 2^23 rounds to an integer (to even) and leaves its two's complement in the low byte
        const float r = 12582912.f;
        const uint32_t x = __float_as_uint(__fadd_rn(a, r)), y = __float_as_uint(__fadd_rn(b, r)), z = __float_as_uint(__fadd_rn(c, r)),
                       w = __float_as_uint(__fadd_rn(d, r));
        return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
    }
    static __device__ __forceinline__ float decode(uint32_t byte) { return (float)(int8_t)byte; }
    static __device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
        const uint32_t u = w ^ 0x80808080u;                // 0 .. 255: under the exponent of 2^23, less 2^23 + 128
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 | j)) - 8388736.f;
    }
    static __device__ __forceinline__ uint32_t without_nan(uint32_t w) { return w; }
};
struct KvE4m3 {
    static constexpr uint32_t kMaxMant = 0x600000u;
    static constexpr int kMaxExp = 8;
    static __device__ __forceinline__ uint32_t encode(float x) {
        return x == x ? (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : 0u;
    }
    static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
        uint32_t w;
        asm("{.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};}"
            : "=r"(w)
            : "f"(a), "f"(b), "f"(c), "f"(d));
        return w;
    }
    static __device__ __forceinline__ float decode(uint32_t byte) {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
    }
    static __device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
        uint32_t lo, hi;
        asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(lo), "=r"(hi) : "r"(w));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
    // NaN codes (0x7f under either sign) become code 0.
    static __device__ __forceinline__ uint32_t without_nan(uint32_t w) {
        return w & ~(((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu);
    }
};

// Smallest scale = power of two >= 2^-100 whose largest code reaches the magnitude with these bits (sign cleared); NaN for an
// infinity or a NaN. Powers of two make x / scale exact, so a code has one rounding, and growing a scale shifts the block's
// older codes by whole binary places: e4m3 codes survive it unchanged (down to its subnormals), int8 codes round once
// per doubling. (A scale of exactly A / 127 would leave int8 up to one bit finer, but would round all older codes of the
// block again for every token that sets a new maximum, 2 to 3 times in a block of 16.)
template <typename KV> __device__ __forceinline__ float pow2_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __int_as_float(0x7fffffff);
    int e = (int)(amax_bits >> 23) - 127 - KV::kMaxExp + ((amax_bits & 0x7fffffu) > KV::kMaxMant ? 1 : 0);
    e = e < -100 ? -100 : e;
    return __int_as_float((e + 127) << 23);
}

}  // namespace ns
