// kv_attend.hip — attention over the 8-bit memory of kv_append.hip.
//
//   o = sum_t p_t v_t,  p = softmax(scale * q . k_t) over the tokens t that the query sees,
// with k_t, v_t = code * the scale of the token's page and head.  Codes (4 significand bits) are exact in bf16 and in f16,
// so the matrix units multiply them as they are; the scales are applied to the scores and to p.
//
// One wave works on 32 tokens at a time and on 16 query rows (the query heads that share a key head, times the new tokens):
//   S^T = K Q^T   A = 16 tokens x 32 dims, B = 32 dims x 16 rows: a lane holds scores of ONE row for 8 tokens, and
//   O^T += V^T P^T  takes exactly these as its B operand, with no exchange between lanes: the token that stands at
//                   row m of score tile t is number (m >> 2) * 8 + t * 4 + (m & 3) of the 32.
// V^T wants 8 tokens of one dimension in a lane; a lane loads 8 tokens x w dimensions and transposes the bytes in registers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "launch.hpp"
#include "lowbits.hpp"

namespace vdb {

namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNone = -3.0e38f;  // the running maximum before a row has seen a token

template <int T>
using E = typename Elem<T>::type;

// bf16 parts of p: bf16 results need one (rounded to nearest: 2^-9 of each p, of either sign), f16 two, f32 three
template <int T>
struct Parts {
    static constexpr int value = T == kBF16 ? 1 : T == kF16 ? 2 : 3;
};

// 8 codes (two words) -> 8 elements of the type that scores are computed in
template <bool HALF>
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) {
    u32x4 r;
    if constexpr (HALF) {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    }
    return r;
}

template <bool HALF>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// rows a[0..3] of 4 bytes -> columns
__device__ __forceinline__ void transpose4(const uint32_t a[4], uint32_t out[4]) {
    const uint32_t l01 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), h01 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u);
    const uint32_t l23 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u), h23 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return ~(((x & 0x7F7F7F7Fu) ^ 0x7F7F7F7Fu) + 0x7F7F7F7Fu) & 0x80808080u; }

template <int T, int DS>
struct Shape {
    static constexpr int D = DS * 32, ND = DS * 2, LDO = D + 4;
    static constexpr size_t lds = (size_t)4 * 16 * LDO * 4 + 2 * 4 * 16 * 4;
};

// The dimensions are cut into chunks of 128, 64 and 32, of which a lane holds 8, 4 and 2 neighbours: chunk c of DS.
template <int DS>
struct Chunks {
    static constexpr int count = DS / 4 + (DS >> 1 & 1) + (DS & 1);
    static constexpr int width(int c) { return c < DS / 4 ? 8 : (c == DS / 4 && (DS & 2)) ? 4 : 2; }
    static constexpr int offset(int c) { return c <= DS / 4 ? c * 128 : DS / 4 * 128 + 64; }
    static constexpr int tile(int c) { return offset(c) / 16; }
};

template <int T, int DS, bool SEL>
__global__ __launch_bounds__(256) void kv_attend(KvAttendArgs a) {
    constexpr bool HALF = T == kF16;
    constexpr int NQ = T == kF32 ? 3 : 1, NP = Parts<T>::value, D = DS * 32, ND = DS * 2, LDO = Shape<T, DS>::LDO;
    extern __shared__ float smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, q4 = lane >> 4;
    const uint32_t b = blockIdx.z, head = blockIdx.y, H = a.mem.heads, P = a.mem.page_tokens, G = a.q_heads / H;
    const int64_t first = a.batch.offsets ? a.batch.offsets[b] : b;
    const int64_t n_new = a.batch.offsets ? (int64_t)a.batch.offsets[b + 1] - first : 1;
    if (n_new <= 0 || first < 0 || first + n_new > (int64_t)a.batch.tokens) return;
    const int64_t len = min((int64_t)a.batch.lengths[b], (int64_t)a.batch.table_width * P);
    const int64_t start = (int64_t)a.batch.lengths[b] - n_new;
    const int32_t* table = a.batch.table + (uint64_t)b * a.batch.table_width;
    const int64_t* select = SEL ? a.select + ((uint64_t)b * H + head) * a.n_select : nullptr;
    const int64_t rows = n_new * G;
    const uint8_t* kc = (const uint8_t*)a.mem.k;
    const uint8_t* vc = (const uint8_t*)a.mem.v;

    for (int64_t row0 = (int64_t)blockIdx.x * 16; row0 < rows; row0 += (int64_t)gridDim.x * 16) {
        const int64_t r = row0 + m;
        const bool live = r < rows;
        const int64_t tok = live ? r / G : 0;
        const uint32_t qh = head * G + (live ? (uint32_t)(r - tok * G) : 0);
        const int64_t pos = live ? start + tok : -1;
        u32x4 qf[NQ][DS];
        {
            const E<T>* q = (const E<T>*)a.q + (uint64_t)(first + tok) * a.q_token + (uint64_t)qh * a.q_head + q4 * 8 * DS;
#pragma unroll
            for (int j = 0; j < DS; ++j) {
                if constexpr (T == kF32) {
                    const f32x4 x = live ? *(const f32x4*)(q + j * 8) : f32x4{0, 0, 0, 0};
                    const f32x4 y = live ? *(const f32x4*)(q + j * 8 + 4) : f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < NQ; ++s)
                        qf[s][j] = u32x4{pack_hi16(bf16_part(x[0], s), bf16_part(x[1], s)), pack_hi16(bf16_part(x[2], s), bf16_part(x[3], s)),
                                         pack_hi16(bf16_part(y[0], s), bf16_part(y[1], s)), pack_hi16(bf16_part(y[2], s), bf16_part(y[3], s))};
                } else {
                    qf[0][j] = live ? *(const u32x4*)(q + j * 8) : u32x4{0, 0, 0, 0};
                }
            }
        }
        // positions of the tile's first and last row; tokens [lo, hi) are seen by some row, [lo_all, hi_all) by every row
        const int64_t pos0 = start + row0 / G, pos1 = start + min(row0 + 15, rows - 1) / G;
        const int64_t hi = SEL ? (int64_t)a.n_select : max((int64_t)0, min(pos1 + 1, len));
        const int64_t lo = SEL || a.window == 0 ? 0 : max((int64_t)0, pos0 - a.window + 1);
        const bool same = SEL || pos0 == pos1;
        const int64_t lo_all = a.window == 0 ? 0 : max((int64_t)0, pos1 - a.window + 1), hi_all = pos0 + 1;

        f32x4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = f32x4{0, 0, 0, 0};
        float top = kNone, sum = 0.0f;

        for (int64_t kb = (lo & ~31ll) + wave * 32; kb < hi; kb += 128) {
            // ---- where the tokens lie: two for the scores (row m of either tile), eight for the values
            float ks[8], vs[8];
            bool have[8];
            int64_t koff[2];
            int64_t voff[8];
            auto place = [&](int64_t t) -> int64_t {  // row number of token t, or -1
                if (t < 0 || t >= len) return -1;
                const int32_t pid = table[t >> a.mem.page_shift];
                if (pid < 0 || (uint64_t)pid >= a.mem.pages) return -1;
                return (((int64_t)pid * H + head) << a.mem.page_shift) + (t & (P - 1));
            };
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int64_t i = kb + (m >> 2) * 8 + t * 4 + (m & 3);
                koff[t] = i >= lo && i < hi ? place(SEL ? select[i] : i) : -1;
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const int64_t i = kb + q4 * 8 + t;
                voff[t] = i >= lo && i < hi ? place(SEL ? select[i] : i) : -1;
                have[t] = voff[t] >= 0;
                const uint64_t page = have[t] ? (uint64_t)voff[t] >> a.mem.page_shift : 0;
                ks[t] = have[t] ? a.mem.k_scale[page] : 0.0f;
                vs[t] = have[t] ? a.mem.v_scale[page] : 0.0f;
            }
            f32x4 sc[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[t] = f32x4{0, 0, 0, 0};
                const uint8_t* kp = kc + (koff[t] < 0 ? 0 : koff[t]) * D + q4 * 8 * DS;
#pragma unroll
                for (int j = 0; j < DS; ++j) {
                    const u32x2 w = koff[t] >= 0 ? *(const u32x2*)(kp + j * 8) : u32x2{0, 0};
                    const u32x4 kf = widen<HALF>(w[0], w[1]);
#pragma unroll
                    for (int s = 0; s < NQ; ++s) sc[t] = mfma<HALF>(kf, qf[s][j], sc[t]);
                }
            }
            // ---- softmax over what the lane's row sees of its 8 tokens
            float p[8];
            bool seen[8];
            float now = top;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const int64_t i = kb + q4 * 8 + t;
                seen[t] = live && have[t] && (SEL || (i <= pos && (a.window == 0 || i > pos - a.window)));
                p[t] = sc[t >> 2][t & 3] * (ks[t] * (a.scale * kLog2e));
                if (seen[t] && !(p[t] <= now)) now = p[t];
            }
            now = __builtin_fmaxf(now, __shfl_xor(now, 16));
            now = __builtin_fmaxf(now, __shfl_xor(now, 32));
            const float shrink = exp2f(top - now);
            top = now;
            sum *= shrink;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                p[t] = seen[t] ? exp2f(p[t] - now) : 0.0f;
                sum += p[t];
                p[t] *= vs[t];
            }
            u32x4 pf[NP];
#pragma unroll
            for (int s = 0; s < NP; ++s) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if constexpr (NP == 1) {
                        bf16x2 w = {(__bf16)p[2 * t], (__bf16)p[2 * t + 1]};
                        pf[s][t] = __builtin_bit_cast(uint32_t, w);
                    } else {
                        pf[s][t] = pack_hi16(bf16_part(p[2 * t], s), bf16_part(p[2 * t + 1], s));
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= shrink;
            // ---- values: chunks of w dimensions a lane
#pragma unroll
            for (int c = 0; c < Chunks<DS>::count; ++c) {
                const int w = Chunks<DS>::width(c), off = Chunks<DS>::offset(c) + m * w;
                uint32_t col[8][2];  // [dimension][tokens 0-3, 4-7]
                uint32_t odd = 0;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t x[4][2];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint8_t* vp = vc + (have[hf * 4 + t] ? voff[hf * 4 + t] : 0) * D + off;
                        x[t][0] = x[t][1] = 0;
                        if (have[hf * 4 + t]) {
                            if (w == 8) {
                                const u32x2 y = *(const u32x2*)vp;
                                x[t][0] = y[0], x[t][1] = y[1];
                            } else if (w == 4) {
                                x[t][0] = *(const uint32_t*)vp;
                            } else {
                                x[t][0] = *(const uint16_t*)vp;
                            }
                        }
                        odd |= nan_bytes(x[t][0]) | nan_bytes(x[t][1]);
                    }
#pragma unroll
                    for (int g = 0; g < (w + 3) / 4; ++g) {
                        const uint32_t in[4] = {x[0][g], x[1][g], x[2][g], x[3][g]};
                        uint32_t out[4];
                        transpose4(in, out);
#pragma unroll
                        for (int e = 0; e < 4 && g * 4 + e < w; ++e) col[g * 4 + e][hf] = out[e];
                    }
                }
                // a NaN among values that some rows of the tile do not see must not reach those (0 * NaN)
                const bool mixed = !same && (kb < lo_all || kb + 32 > hi_all) && __any(odd != 0);
#pragma unroll
                for (int e = 0; e < w; ++e) {
                    const int d = Chunks<DS>::tile(c) + e;
                    uint32_t x = col[e][0], y = col[e][1];
                    if (mixed) {
                        const uint32_t nx = nan_bytes(x) >> 7, ny = nan_bytes(y) >> 7;  // 1 in the bytes that are NaN
                        x &= ~(nx * 255u);
                        y &= ~(ny * 255u);
                        const u32x4 is_nan = widen<false>(nx * 0x38u, ny * 0x38u);  // 0x38 = 1.0
                        u32x4 sees;
#pragma unroll
                        for (int t = 0; t < 4; ++t) sees[t] = (seen[2 * t] ? 0x3F80u : 0u) | (seen[2 * t + 1] ? 0x3F800000u : 0u);
                        const f32x4 n = mfma<false>(is_nan, sees, f32x4{0, 0, 0, 0});
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n[i] > 0.0f) o[d][i] = float_of(0x7FC00000u);
                    }
                    const u32x4 vf = widen<false>(x, y);
#pragma unroll
                    for (int s = 0; s < NP; ++s) o[d] = mfma<false>(vf, pf[s], o[d]);
                }
            }
        }
        // ---- join the four waves: each row's maximum, then sums and outputs in wave order
        float* so = smem;                    // [4][16][LDO]
        float* st = smem + 4 * 16 * LDO;     // [4][16] maxima
        float* ss = st + 64;                 // [4][16] sums
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (q4 == 0) st[wave * 16 + m] = top, ss[wave * 16 + m] = sum;
#pragma unroll
        for (int c = 0; c < Chunks<DS>::count; ++c) {
            const int w = Chunks<DS>::width(c);
#pragma unroll
            for (int e = 0; e < w; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    so[(wave * 16 + m) * LDO + Chunks<DS>::offset(c) + (q4 * 4 + i) * w + e] = o[Chunks<DS>::tile(c) + e][i];
        }
        __syncthreads();
        const int row = threadIdx.x >> 4, part = threadIdx.x & 15;
        float best = kNone;
#pragma unroll
        for (int w = 0; w < 4; ++w) best = fmaxf(best, st[w * 16 + row]);
        float f[4], total = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            f[w] = exp2f(st[w * 16 + row] - best);
            total += f[w] * ss[w * 16 + row];
        }
        if (row0 + row < rows) {
            const int64_t ot = (row0 + row) / G;
            const uint64_t orow = (uint64_t)(first + ot) * a.q_heads + head * G + (uint32_t)(row0 + row - ot * G);
            const bool none = total == 0.0f;  // (a NaN is something)
            const float inv = none ? 0.0f : 1.0f / total;
            E<T>* out = (E<T>*)a.out + orow * D + part * ND;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) v += f[w] * so[(w * 16 + row) * LDO + part * ND + d];
                out[d] = (E<T>)(none ? 0.0f : v * inv);
            }
            if (a.lse && part == 0) a.lse[orow] = none ? -__builtin_inff() : (best + log2f(total)) * kLn2;
        }
        __syncthreads();
    }
}

template <int T, int DS>
hipError_t launch_one(const KvAttendArgs& a, uint32_t max_new, hipStream_t stream) {
    const uint32_t G = a.q_heads / a.mem.heads;
    const uint32_t tiles = (uint32_t)std::min<uint64_t>(((uint64_t)max_new * G + 15) / 16, 65535);
    const dim3 grid(tiles, a.mem.heads, a.batch.count);
    if (a.select) hipLaunchKernelGGL((kv_attend<T, DS, true>), grid, dim3(256), (Shape<T, DS>::lds), stream, a);
    else hipLaunchKernelGGL((kv_attend<T, DS, false>), grid, dim3(256), (Shape<T, DS>::lds), stream, a);
    return hipGetLastError();
}

}  // namespace

#ifndef VDB_PART
#define VDB_PART 0
#endif
#define VDB_CAT2(a, b) a##b
#define VDB_CAT(a, b) VDB_CAT2(a, b)

// compiled once per element type (-DVDB_PART = vdb_dtype)
hipError_t VDB_CAT(kv_attend_launch_, VDB_PART)(const KvAttendArgs& a, uint32_t max_new, hipStream_t stream) {
    switch (a.mem.dim / 32) {
        case 1: return launch_one<VDB_PART, 1>(a, max_new, stream);
        case 2: return launch_one<VDB_PART, 2>(a, max_new, stream);
        case 3: return launch_one<VDB_PART, 3>(a, max_new, stream);
        case 4: return launch_one<VDB_PART, 4>(a, max_new, stream);
        case 5: return launch_one<VDB_PART, 5>(a, max_new, stream);
        case 6: return launch_one<VDB_PART, 6>(a, max_new, stream);
        case 7: return launch_one<VDB_PART, 7>(a, max_new, stream);
        case 8: return launch_one<VDB_PART, 8>(a, max_new, stream);
    }
    return hipErrorInvalidValue;
}

#if VDB_PART == 0
hipError_t kv_attend_launch_1(const KvAttendArgs&, uint32_t, hipStream_t);
hipError_t kv_attend_launch_2(const KvAttendArgs&, uint32_t, hipStream_t);

size_t kv_attend_workspace_bytes(const KvAttendArgs&, uint32_t) { return 0; }

int launch_kv_attend(const KvAttendArgs& a, int dtype, uint32_t max_new, void*, hipStream_t stream, std::string* err) {
    const hipError_t e = dtype == kF32 ? kv_attend_launch_0(a, max_new, stream)
                         : dtype == kF16 ? kv_attend_launch_1(a, max_new, stream)
                                         : kv_attend_launch_2(a, max_new, stream);
    if (e == hipSuccess) return 0;
    if (err) *err = std::string("kv_attend: ") + hipGetErrorString(e);
    return 3;
}
#endif

}  // namespace vdb
