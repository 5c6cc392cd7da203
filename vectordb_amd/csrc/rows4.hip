// rows4.hip — base rows held in 4 bits: packing, unpacking and the products of a few queries with every row.
//
// A row of d values is ceil(d / 32) groups of 32; a group is 16 bytes of e2m1 codes (even columns in the low nibbles; sign, two
// exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one byte e, and stands for code * 2^(e - 127).  That is the
// block-scaled 4-bit format of the matrix units: v_cvt_scalef32_pk_bf16_fp4 turns a byte of codes into two scaled bf16 in ONE
// instruction, and exactly (two significand bits times a power of two), so a row costs 17 bytes per 32 columns of HBM and half a
// vector instruction per column.
#include <hip/hip_runtime.h>

#include <algorithm>
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
    uint32_t chunk;  // blocks of 128 columns whose queries are in LDS at once
};

// y[m][r] = sum_c x[m][c] * value[r][c] on the matrix units: 16 rows are the A operand, 16 queries the B operand.  A query in
// f32 is three bf16 parts (f16: two) that sum to it exactly, one matrix instruction each into the same accumulator: the f32
// accumulators see exact products (of all but what lies below 2^-133 in an f32 query).
//
// What bounds it is the rows' bytes.  The queries go to LDS once per block, as parts and in operand order; the blocks are
// persistent, and a wave takes RT tiles of 16 rows by KB blocks of 128 columns at a time (16 bytes of codes and one scale a lane
// for each), the next ones on their way while these are multiplied.  Four neighbouring lanes load 64 consecutive bytes of a row (a lane 32
// columns, of which each of the four matrix steps takes 8) and the lanes then exchange what they hold for the order that the
// matrix units want: loaded in that order, every lane touches a cache line of its own (1M x 128 x 16: 50 us instead of 30, with the stores).
// The rows are the B operand, so that 16 lanes hold results of one query for neighbouring rows and store them side by side.
// Queries whose parts are too large for LDS are taken in ranges of columns, each added to the results of the one before.
// Blocks that a compute unit holds, by registers.
constexpr int products_blocks(int pieces, int nct) { return pieces == 1 ? 6 : nct == 1 ? 4 : 3; }

template <int T, int RT, int KB, int NCT, bool SPLIT>
__global__ __launch_bounds__(256, products_blocks(RT * KB, NCT)) void rows4_products(ProductArgs a) {
    constexpr int S = Elem<T>::splits;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, q4 = lane >> 4;
    const uint32_t q0 = blockIdx.y * (16 * NCT), nq = min(a.nq - q0, 16u * NCT);
    const uint32_t nblk = (a.groups + 3) / 4, plane = a.chunk * nq * 256;  // bytes of one part of the queries
    const uint32_t tiles = (a.n + 16 * RT - 1) / (16 * RT);
    const uint32_t first = SPLIT ? blockIdx.x : blockIdx.x * 4 + wave, step = SPLIT ? gridDim.x : gridDim.x * 4;
    // where a lane finds its query among nq of them (operands: [block][step][query][quarter] of 16 bytes)
    uint32_t at[NCT];
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) at[ct] = (min((uint32_t)(ct * 16 + m), nq - 1) * 4 + q4) * 16;

    for (uint32_t b0 = 0; b0 < nblk; b0 += a.chunk) {
        const uint32_t b1 = min(b0 + a.chunk, nblk);
        __syncthreads();
        for (uint32_t u = threadIdx.x; u < (b1 - b0) * 16 * nq; u += 256) {  // 8 columns of one query
            const uint32_t quarter = u & 3, query = (u >> 2) % nq, bs = (u >> 2) / nq;  // bs = block * 4 + step
            const uint32_t c0 = (b0 + (bs >> 2)) * 128 + quarter * 32 + (bs & 3) * 8;
            const typename Elem<T>::type* x = (const typename Elem<T>::type*)a.x + (uint64_t)(q0 + query) * a.x_stride;
            float v[8];
            if (c0 + 8 <= a.dim) {
                typedef __attribute__((ext_vector_type(8), aligned(sizeof(typename Elem<T>::type)))) typename Elem<T>::type vec;
                const vec y = *(const vec*)(x + c0);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = to_f32((typename Elem<T>::type)y[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = c0 + i < a.dim ? to_f32(x[c0 + i]) : 0.0f;
            }
#pragma unroll
            for (int s = 0; s < S; ++s)
                *(u32x4*)(lds + s * plane + u * 16) =
                    u32x4{pack_hi16(bf16_part(v[0], s), bf16_part(v[1], s)), pack_hi16(bf16_part(v[2], s), bf16_part(v[3], s)),
                          pack_hi16(bf16_part(v[4], s), bf16_part(v[5], s)), pack_hi16(bf16_part(v[6], s), bf16_part(v[7], s))};
        }
        __syncthreads();

        u32x4 w[2][RT * KB];
        uint32_t e[2][RT * KB];
        auto fetch = [&](uint32_t tile, uint32_t blk, u32x4 cw[RT * KB], uint32_t ce[RT * KB]) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const uint32_t row = min(tile * (16 * RT) + r * 16 + (lane >> 2), a.n - 1);
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const uint32_t g = (blk + k) * 4 + (lane & 3);
                    const uint64_t at = (uint64_t)row * a.groups + min(g, a.groups - 1);
                    cw[r * KB + k] = *(const u32x4*)(a.codes + at * 16);
                    ce[r * KB + k] = a.scales[at];
                }
            }
        };
        f32x4 acc[RT][NCT];
        const int from = (m * 4 + q4) * 4;  // the lane that loaded this lane's piece
        auto multiply = [&](uint32_t blk, u32x4 cw[RT * KB], uint32_t ce[RT * KB]) {
            if ((blk + KB) * 128 > a.dim) {  // codes past the last column are taken for 0 (scaled, they may be infinite in bf16)
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const int left = (int)a.dim - (int)((blk + k) * 4 + (lane & 3)) * 32;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        if (left <= 0) ce[r * KB + k] = 127;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int n = left - 8 * j;
                            cw[r * KB + k][j] &= n >= 8 ? 0xFFFFFFFFu : n > 0 ? (1u << 4 * n) - 1 : 0u;
                        }
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < RT * KB; ++p) {
#pragma unroll
                for (int j = 0; j < 4; ++j) cw[p][j] = __builtin_amdgcn_ds_bpermute(from, cw[p][j]);
                ce[p] = __builtin_amdgcn_ds_bpermute(from, ce[p]);
            }
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                if (KB > 1 && blk + k >= b1) break;
                const unsigned char* here = lds + (blk + k - b0) * nq * 256;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u32x4 bv[NCT][S];
#pragma unroll
                    for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                        for (int s = 0; s < S; ++s) bv[ct][s] = *(const u32x4*)(here + s * plane + j * nq * 64 + at[ct]);
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint32_t code = cw[r * KB + k][j], x = ce[r * KB + k];
                        const float scale = float_of(x == 0 ? 0x00400000u : x << 23);
                        const u32x4 av = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 0)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 1)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 2)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 3))};
#pragma unroll
                        for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                            for (int s = S - 1; s >= 0; --s)
                                acc[r][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, bv[ct][s]), __builtin_bit_cast(bf16x8, av), acc[r][ct], 0, 0, 0);
                    }
                }
            }
        };
        // (tile, block) pairs of this wave in order; with SPLIT the block's waves share a tile and take every fourth block of it
        const uint32_t start = b0 + (SPLIT ? wave * KB : 0), stride = SPLIT ? 4 * KB : KB;
        uint32_t tile = first, blk = start, ntile = first, nblkk = start;
        auto next = [&](uint32_t& t, uint32_t& b) {
            b += stride;
            if (b >= b1) b = start, t += step;
        };
        auto clear = [&] {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int ct = 0; ct < NCT; ++ct) acc[r][ct] = f32x4{0, 0, 0, 0};
        };
        // lane (m, q4) holds row m of queries 4 q4 + i
        auto finish = [&](uint32_t t) {
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t query = ct * 16 + q4 * 4 + i;
                    if (query < nq) {
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            const uint32_t row = t * (16 * RT) + r * 16 + m;
                            float* o = a.out + (uint64_t)(q0 + query) * a.n + row;
                            if (row < a.n) *o = b0 ? *o + acc[r][ct][i] : acc[r][ct][i];
                        }
                    }
                }
        };
        if constexpr (!SPLIT) {
            clear();
            if (ntile < tiles) fetch(ntile, nblkk, w[0], e[0]);
            while (tile < tiles) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (tile < tiles) {
                        next(ntile, nblkk);
                        if (ntile < tiles) fetch(ntile, nblkk, w[k ^ 1], e[k ^ 1]);
                        multiply(blk, w[k], e[k]);
                        const uint32_t t = tile;
                        next(tile, blk);
                        if (tile != t) {
                            finish(t);
                            clear();
                        }
                    }
                }
            }
        } else {
            float* red = (float*)(lds + S * plane);  // [4][RT * NCT * 4][64]
            for (uint32_t t = first; t < tiles; t += step) {
                clear();
                uint32_t b = start;
                if (b < b1) fetch(t, b, w[0], e[0]);
                while (b < b1) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (b < b1) {
                            if (b + stride < b1) fetch(t, b + stride, w[k ^ 1], e[k ^ 1]);
                            multiply(b, w[k], e[k]);
                            b += stride;
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                        for (int i = 0; i < 4; ++i) red[((wave * RT + r) * NCT + ct) * 256 + i * 64 + lane] = acc[r][ct][i];
                __syncthreads();
                if (wave == 0) {
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float y = 0.0f;
#pragma unroll
                                for (int v = 0; v < 4; ++v) y += red[((v * RT + r) * NCT + ct) * 256 + i * 64 + lane];
                                acc[r][ct][i] = y;
                            }
                    finish(t);
                }
                __syncthreads();
            }
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
    ProductArgs a{d_codes, d_scales, d_x, d_out, x_stride, n, dim, (dim + 31) / 32, nq, 0};
    auto go = [&](auto t) {
        constexpr int T = decltype(t)::value, S = Elem<T>::splits;
        const uint32_t nblk = (a.groups + 3) / 4, tiles = (n + 15) / 16;
        const bool two = nq > 16;  // two column tiles: 17 to 32 queries a pass over the rows
        const uint32_t per = std::min(nq, two ? 32u : 16u), ys = (nq + (two ? 31 : 15)) / (two ? 32 : 16);
        const uint32_t block = per * 256 * S;  // bytes of LDS for 128 columns
        a.chunk = std::max(1u, std::min(nblk, (64u << 10) / block));
        auto launch = [&](auto kernel, uint32_t rt, uint32_t kb, bool split) {
            const uint32_t groups = (tiles + rt - 1) / rt;
            const size_t lds = (size_t)a.chunk * block + (split ? 4 * rt * (two ? 2 : 1) * 1024 : 0);
            const uint32_t fit = std::max<uint32_t>(1, std::min<uint32_t>(products_blocks(rt * kb, two ? 2 : 1), (uint32_t)((160u << 10) / lds)));
            const uint32_t blocks = std::min(split ? groups : (groups + 3) / 4, 256 * fit);
            hipLaunchKernelGGL(kernel, dim3(blocks, ys), dim3(256), lds, stream, a);
        };
        auto pick = [&](auto n_ct) {
            constexpr int NCT = decltype(n_ct)::value;
            // Few rows: the waves of a block share the columns of a tile (4000 x 2000: 10.5 -> 6.0 us, 16 000 x 960: 7.9 -> 6.3), with
            // more than a few queries only where there are very few (16 000 x 960 x 16: 9.6 -> 11.9 us: a block's LDS is filled for less).
            // Many rows: 4 KB a wave at a time, of rows of more than 128 columns whole cache lines at once (1M x 960: four tiles by 128
            // columns 169 us and 1.7 times the bytes, two by 256 119 us, one by 512 121, four by 256 138).
            if (tiles <= (nq <= 4 ? 1024 : 512) && nblk >= 4) launch(rows4_products<T, 1, 1, NCT, true>, 1, 1, true);
            else if (tiles < 8192) launch(rows4_products<T, 1, 1, NCT, false>, 1, 1, false);
            else if (nblk == 1) launch(rows4_products<T, 4, 1, NCT, false>, 4, 1, false);
            else launch(rows4_products<T, 2, 2, NCT, false>, 2, 2, false);
        };
        if (two) pick(std::integral_constant<int, 2>());
        else pick(std::integral_constant<int, 1>());
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
