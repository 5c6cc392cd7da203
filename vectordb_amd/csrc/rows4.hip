// rows4.hip — base rows held in 4 bits: packing, unpacking and the products of a few queries with every row.
//
// A row of d values is ceil(d / 32) groups of 32; a group is 16 bytes of e2m1 codes (even columns in the low nibbles; sign, two
// exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one byte e, and stands for code * 2^(e - 127).  That is the
// block-scaled 4-bit format of the matrix units: v_cvt_scalef32_pk_bf16_fp4 turns a byte of codes into two scaled bf16 in ONE
// instruction, and exactly (two significand bits times a power of two), so a row costs 17 bytes per 32 columns of HBM and half a
// vector instruction per column.
#include <hip/hip_runtime.h>

#include <string>

#include "launch.hpp"
#include "lowbits.hpp"

namespace vdb {

namespace {

struct ProductArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    const void* x;
    float* out;
    uint64_t x_stride;  // elements between two queries
    uint32_t n, dim, groups, nq;
};

// The columns [c0, c0 + 32) of a query as bf16 part `split`, zero beyond `dim`: four matrix operands of 8 columns.
template <int T>
__device__ __forceinline__ void load_parts(const typename Elem<T>::type* x, uint32_t c0, uint32_t dim, int split, uint32_t out[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t c = c0 + 2 * i;
        const float a = c < dim ? to_f32(x[c]) : 0.0f;
        const float b = c + 1 < dim ? to_f32(x[c + 1]) : 0.0f;
        out[i] = pack_hi16(bf16_part(a, split), bf16_part(b, split));
    }
}

// y[m][r] = sum_c x[m][c] * value[r][c] on the matrix units: 16 rows are the A operand; the 16 columns of B are (query, part)
// pairs, a query in f32 being three bf16 parts (f16: two) that sum to it exactly.  So no bit of a query is lost, and the f32
// accumulators see exact products.
template <int T>
__global__ __launch_bounds__(256) void rows4_products(ProductArgs a) {
    constexpr int S = Elem<T>::splits, Q = 16 / S;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m = lane & 15, q4 = lane >> 4;
    const uint32_t row0 = (blockIdx.x * 4u + wave) * 16u;
    if (row0 >= a.n) return;
    const uint32_t row = min(row0 + m, a.n - 1);
    const uint32_t query = blockIdx.y * Q + m / S;
    const bool live = m < Q * S && query < a.nq;
    const typename Elem<T>::type* x = (const typename Elem<T>::type*)a.x + (live ? query : 0) * a.x_stride;
    const uint8_t* codes = a.codes + (uint64_t)row * a.groups * 16u;
    const uint8_t* scales = a.scales + (uint64_t)row * a.groups;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t g0 = 0; g0 < a.groups; g0 += 4) {
        const uint32_t g = g0 + q4;
        u32x4 w = {0, 0, 0, 0};
        uint32_t e = 127;
        if (g < a.groups) {
            w = *(const u32x4*)(codes + (uint64_t)g * 16u);
            e = scales[g];
        }
        uint32_t b[16];
        load_parts<T>(x, g * 32u, live ? a.dim : 0, m % S, b);
        const float scale = float_of(e == 0 ? 0x00400000u : e << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x8 av;
            uint32_t* ap = (uint32_t*)&av;
            ap[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 0));
            ap[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 1));
            ap[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 2));
            ap[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 3));
            u32x4 bv = {b[4 * j], b[4 * j + 1], b[4 * j + 2], b[4 * j + 3]};
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(bf16x8, bv), acc, 0, 0, 0);
        }
    }
    // lane (m, q4) holds rows row0 + 4 q4 + i of column m; the parts of a query sit in neighbouring columns
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] += __shfl(acc[i], (lane & 48) | ((m * S + s) & 15));
    }
    const uint32_t oq = blockIdx.y * Q + m;
    if (m < Q && oq < a.nq) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = row0 + 4 * q4 + i;
            if (r < a.n) a.out[(uint64_t)oq * a.n + r] = y[i];
        }
    }
}

struct PackArgs {
    const void* rows;
    uint8_t* codes;
    uint8_t* scales;
    uint64_t row_stride;
    uint64_t total;  // rows * groups
    uint32_t dim, groups;
};

// One thread per group of 32 columns.  The group's scale is the smallest power of two under which its largest magnitude is at
// most 6, the largest code; codes round to nearest, ties to even.  A group that holds an infinity or a NaN becomes NaN (e = 255).
// The scale stops at 2^125, where 6 is the largest finite f32 code * scale: magnitudes above 6 * 2^125 saturate there.
template <int T>
__global__ __launch_bounds__(256) void rows4_pack(PackArgs a) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < a.total; i += (uint64_t)gridDim.x * 256u) {
        const uint64_t row = i / a.groups;
        const uint32_t g = (uint32_t)(i - row * a.groups);
        const typename Elem<T>::type* x = (const typename Elem<T>::type*)a.rows + row * a.row_stride + g * 32u;
        const uint32_t left = a.dim - g * 32u;
        float v[32];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            v[c] = (uint32_t)c < left ? to_f32(x[c]) : 0.0f;
            top = max(top, bits_of(v[c]) & 0x7FFFFFFFu);
        }
        int e = 127;
        if (top >= 0x7F800000u) {
            e = 255;
        } else if (top) {
            int ex;
            const float f = frexpf(float_of(top), &ex);
            e = min(max(127 + ex - (f <= 0.75f ? 3 : 2), 1), 252);
        }
        u32x4 w;
        const float scale = float_of((uint32_t)e << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t d = 0;
            if (e != 255) {
                d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * j + 0], v[8 * j + 1], scale, 0);
                d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * j + 2], v[8 * j + 3], scale, 1);
                d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * j + 4], v[8 * j + 5], scale, 2);
                d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[8 * j + 6], v[8 * j + 7], scale, 3);
            }
            w[j] = d;
        }
        *(u32x4*)(a.codes + i * 16u) = w;
        a.scales[i] = (uint8_t)e;
    }
}

__global__ __launch_bounds__(256) void rows4_unpack(const uint8_t* codes, const uint8_t* scales, float* out, uint64_t total, uint32_t dim, uint32_t groups) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256u) {
        const uint64_t row = i / groups;
        const uint32_t g = (uint32_t)(i - row * groups), e = scales[i];
        const u32x4 w = *(const u32x4*)(codes + i * 16u);
        const float scale = float_of(e == 0 ? 0x00400000u : e == 255 ? 0x7FC00000u : e << 23);
        float* o = out + row * dim + g * 32u;
        for (uint32_t c = 0; c < 32 && c < dim - g * 32u; ++c) {
            const uint32_t code = w[c >> 3] >> (4 * (c & 7)) & 15u, mag = code & 7u;
            const float v = mag < 2 ? 0.5f * mag : (1.0f + 0.5f * (mag & 1u)) * (float)(1u << ((mag >> 1) - 1));
            o[c] = (code & 8u ? -v : v) * scale;
        }
    }
}

int done(const char* what, std::string* err) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    if (err) *err = std::string(what) + ": " + hipGetErrorString(e);
    return 3;
}

}  // namespace

int launch_rows4_products(const uint8_t* d_codes, const uint8_t* d_scales, uint32_t n, uint32_t dim, const void* d_x, int dtype, uint32_t nq,
                          uint64_t x_stride, float* d_out, hipStream_t stream, std::string* err) {
    const ProductArgs a{d_codes, d_scales, d_x, d_out, x_stride, n, dim, (dim + 31) / 32, nq};
    const uint32_t bx = (n + 63) / 64;
    auto go = [&](auto t) {
        constexpr int T = decltype(t)::value, Q = 16 / Elem<T>::splits;
        hipLaunchKernelGGL((rows4_products<T>), dim3(bx, (nq + Q - 1) / Q), dim3(256), 0, stream, a);
    };
    if (dtype == kF32) go(std::integral_constant<int, kF32>());
    else if (dtype == kF16) go(std::integral_constant<int, kF16>());
    else go(std::integral_constant<int, kBF16>());
    return done("rows4_products", err);
}

int launch_rows4_pack(const void* d_rows, int dtype, uint64_t n, uint32_t dim, uint64_t row_stride, uint8_t* d_codes, uint8_t* d_scales,
                      hipStream_t stream, std::string* err) {
    PackArgs a{d_rows, d_codes, d_scales, row_stride, n * ((dim + 31) / 32), dim, (dim + 31) / 32};
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.total + 255) / 256, 1u << 16);
    if (dtype == kF32) hipLaunchKernelGGL((rows4_pack<kF32>), dim3(blocks), dim3(256), 0, stream, a);
    else if (dtype == kF16) hipLaunchKernelGGL((rows4_pack<kF16>), dim3(blocks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rows4_pack<kBF16>), dim3(blocks), dim3(256), 0, stream, a);
    return done("rows4_pack", err);
}

int launch_rows4_unpack(const uint8_t* d_codes, const uint8_t* d_scales, uint64_t n, uint32_t dim, float* d_out, hipStream_t stream, std::string* err) {
    const uint32_t groups = (dim + 31) / 32;
    const uint64_t total = n * groups;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((total + 255) / 256, 1u << 16);
    hipLaunchKernelGGL(rows4_unpack, dim3(blocks), dim3(256), 0, stream, d_codes, d_scales, d_out, total, dim, groups);
    return done("rows4_unpack", err);
}

}  // namespace vdb
