// The 8-bit form in which activations are held for the backward pass: codes of 8 bits and one exponent byte for each 32 consecutive
// elements (include/rt_hip.h has the definition).  Device helpers shared by the kernels that write and that read it.
#pragma once

#include "rt_common.h"

constexpr uint32_t kP8Group = RT_PACK8_GROUP;
constexpr uint32_t kP8LowByte = 8;        // exponent -119: every restored value is 0 or a normal f32 (and a normal bf16) number
constexpr uint32_t kP8NotFinite = 255;

// 2^(byte - 127), and NaN for byte 255: the exponent field of all ones with a mantissa bit set.
template <class T> __device__ __forceinline__ T p8_step(uint32_t byte) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, byte << 23 | (byte + 1) >> 8 << 22);
    else return byte == kP8NotFinite ? __builtin_nan("") : __builtin_bit_cast(double, (uint64_t)(byte + 896u) << 52);
}
template <class T> __device__ __forceinline__ T p8_value(int32_t code, uint32_t byte) { return (T)code * p8_step<T>(byte); }

// Bits of |x|: as unsigned integers they are ordered like the magnitudes, infinities above all numbers and NaN above infinities, so a
// group's maximum by integer comparison also says whether the group is finite.
__device__ __forceinline__ uint32_t p8_magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }
__device__ __forceinline__ uint64_t p8_magnitude(double x) { return __builtin_bit_cast(uint64_t, x) & 0x7fffffffffffffffull; }

// The exponent byte of a group with this largest magnitude M = 1.f * 2^q: q - 6 puts M * 2^-e into [64, 128); from 127.5 on it would
// round to 128, and the next exponent is taken.
__device__ __forceinline__ uint32_t p8_byte_of(uint32_t top) {
    const uint32_t ex = top >> 23;
    if (ex == 255u) return kP8NotFinite;
    const int32_t b = (int32_t)ex - 6 + ((top & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
    return b < (int32_t)kP8LowByte ? kP8LowByte : (uint32_t)b;
}
__device__ __forceinline__ uint32_t p8_byte_of(uint64_t top) {
    const uint32_t ex = (uint32_t)(top >> 52);
    const int32_t b = (int32_t)ex - 1023 + 127 - 6 + ((top & 0xfffffffffffffull) >= 0xfe00000000000ull ? 1 : 0);
    if (b > 254) return kP8NotFinite;                           // infinities, NaN, and magnitudes that no exponent byte reaches
    return b < (int32_t)kP8LowByte ? kP8LowByte : (uint32_t)b;
}
// 2^-(byte - 127); byte != 255
template <class T> __device__ __forceinline__ T p8_inverse_step(uint32_t byte) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, (254u - byte) << 23);
    else return __builtin_bit_cast(double, (uint64_t)(1150u - byte) << 52);
}
// rint(x / step): the scaling by a power of two is exact (or underflows to less than half a step), so one rounding remains, the one to
// an integer.  byte != 255.
__device__ __forceinline__ int32_t p8_code(float x, float inv) { return (int32_t)__builtin_rintf(x * inv); }
__device__ __forceinline__ int32_t p8_code(double x, double inv) { return (int32_t)__builtin_rint(x * inv); }
