// lowbits.hpp — what the kernels on rows held in few bits share (rows4.hip, kv_append.hip, kv_attend.hip): element types,
// exact splits of f32 / f16 values into bf16 parts, and the conversions of 4- and 8-bit codes.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace vdb {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) int32_t i32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

enum { kF32 = 0, kF16 = 1, kBF16 = 2 };  // vdb_dtype

template <int T>
struct Elem;
template <>
struct Elem<kF32> {
    typedef float type;
    static constexpr int splits = 3;  // bf16 parts that hold a value exactly: 24 significand bits in three times 8
};
template <>
struct Elem<kF16> {
    typedef _Float16 type;
    static constexpr int splits = 2;  // 11 bits
};
template <>
struct Elem<kBF16> {
    typedef __bf16 type;
    static constexpr int splits = 1;
};

__device__ __forceinline__ uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float float_of(uint32_t x) { return __builtin_bit_cast(float, x); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return float_of((uint32_t)__builtin_bit_cast(uint16_t, x) << 16); }

// Part `s` of x = part 0 + part 1 + part 2, each a bf16 (given as the f32 with its lower 16 bits zero): the leading bits are cut
// off, not rounded, so no part overflows and every remainder is exact.  What lies below 2^-133, bf16's least number, is in no part
// (of f32 values below 2^-110 that can be bits that count).  An infinity or a NaN stays whole in part 0.
__device__ __forceinline__ float bf16_part(float x, int s) {
    const uint32_t b = bits_of(x);
    if ((b & 0x7F800000u) == 0x7F800000u) return s == 0 ? ((b & 0x007FFFFFu) ? float_of(0x7FC00000u) : x) : 0.0f;
    float hi = float_of(b & 0xFFFF0000u);
    if (s == 0) return hi;
    float r = x - hi;
    hi = float_of(bits_of(r) & 0xFFFF0000u);
    return s == 1 ? hi : r - hi;
}

// Two f32 whose lower halves are zero -> the pair of bf16, `a` in the lower half.
__device__ __forceinline__ uint32_t pack_hi16(float a, float b) { return __builtin_amdgcn_perm(bits_of(b), bits_of(a), 0x07060302u); }

}  // namespace vdb
