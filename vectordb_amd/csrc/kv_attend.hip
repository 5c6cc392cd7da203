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

// bf16 parts of p: f32 results need three; two, rounded, are off by 2^-16 of each p at most, so that a bf16 result is off by its own
// rounding alone (64 sequences of up to 8192 tokens: 122 us with one part, 124 with two).  MANY: kv_attend_many takes one for bf16 results, off
// by 2^-8 of each p at most, of either sign.  That is a choice for speed: four chunks of up to 2048 rows 294 us, with two parts 370, and
// a mean error against 64 bits 1.33 times that of rounding the result alone (1.52e-4 against 1.14e-4, of results of 0.069 in the
// mean square).  (f16 weights, as fast, would lose those below 2^-24 of the largest, which a number of a value may consist of.)
template <int T, bool MANY = false>
struct Parts {
    static constexpr int value = T == kBF16 && MANY ? 1 : T == kF32 ? 3 : 2;
};

// 8 codes (two words) -> 8 elements of the type that scores are computed in
template <bool HALF>
__device__ __forceinline__ u32x2 widen4(uint32_t x) {
    u32x2 r;
    if constexpr (HALF) {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true));
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true));
    }
    return r;
}

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
    static constexpr size_t lds(int waves) { return (size_t)waves * 16 * LDO * 4 + 2 * waves * 16 * 4; }
};

// The dimensions are cut into chunks of 128, 64 and 32, of which a lane holds 8, 4 and 2 neighbours: chunk c of DS.
template <int DS>
struct Chunks {
    static constexpr int count = DS / 4 + (DS >> 1 & 1) + (DS & 1);
    static constexpr int width(int c) { return c < DS / 4 ? 8 : (c == DS / 4 && (DS & 2)) ? 4 : 2; }
    static constexpr int offset(int c) { return c <= DS / 4 ? c * 128 : DS / 4 * 128 + 64; }
    static constexpr int tile(int c) { return offset(c) / 16; }
};

// Work of one launch.  The tokens of a row tile are cut into `splits` ranges of `chunk` (a multiple of 128), one block each;
// where more than one range holds tokens, the blocks leave (maximum, sum, output) in the workspace and kv_join_* adds them up
// in the order of the ranges.
struct Plan {
    uint32_t tiles;   // row tiles of 16 that have blocks of their own (more than that are walked by the blocks of range 0)
    uint32_t splits;
    uint32_t chunk;
    float* part;      // [sequence][head][tile][split][16][D + 2]
    uint32_t max_new;
    bool wide;        // blocks of eight waves instead of four
    bool many;        // kv_attend_many, which needs none of the above
};

typedef const __attribute__((address_space(4))) int32_t* UniformI32;  // read through scalar registers
typedef const __attribute__((address_space(4))) float* UniformF32;

// Token numbers fit 32 bits with room to step past the end (the host checks the table's width and the list's length).
struct Sequence {
    int64_t first;
    int32_t n_new, start, len;  // start: position of the first new token, negative if the length counts fewer tokens
};

__device__ __forceinline__ bool sequence_of(const KvAttendArgs& a, uint32_t b, Sequence& s) {
    s.first = a.batch.offsets ? a.batch.offsets[b] : b;
    const int64_t n = a.batch.offsets ? (int64_t)a.batch.offsets[b + 1] - s.first : 1;
    if (n <= 0 || s.first < 0 || s.first + n > (int64_t)a.batch.tokens) return false;
    const int32_t held = max(a.batch.lengths[b], 0);
    s.n_new = (int32_t)n;
    s.start = held - s.n_new;
    s.len = (int32_t)min((int64_t)held, (int64_t)a.batch.table_width << a.mem.page_shift);
    return true;
}

// Tokens (or places of the list of selected ones) [lo, hi) that rows row0 .. row1 see; lo is rounded down to the tiles of 32.
template <bool SEL>
__device__ __forceinline__ void range_of(const KvAttendArgs& a, const Sequence& s, int32_t pos0, int32_t pos1, int32_t& lo, int32_t& hi) {
    hi = SEL ? (int32_t)a.n_select : max(0, min(pos1, s.len - 1) + 1);
    lo = SEL || a.window == 0 ? 0 : (int32_t)max((int64_t)0, pos0 - a.window + 1);
}

__device__ __forceinline__ float max_of_quarters(float x) {  // over the lanes m, m + 16, m + 32, m + 48
    auto r = __builtin_amdgcn_permlane16_swap(bits_of(x), bits_of(x), false, false);
    x = __builtin_fmaxf(float_of(r[0]), float_of(r[1]));
    r = __builtin_amdgcn_permlane32_swap(bits_of(x), bits_of(x), false, false);
    return __builtin_fmaxf(float_of(r[0]), float_of(r[1]));
}

// The bytes of a key that a lane holds for matrix step j (8 of them) start at this place of the row: pairs of steps lie side by
// side, so that four lanes read 64 contiguous bytes at once.
template <int DS>
__device__ __forceinline__ constexpr int key_byte(int q4, int j) {
    return j == DS - 1 && (DS & 1) ? (DS - 1) * 32 + q4 * 8 : (j >> 1) * 64 + q4 * 16 + (j & 1) * 8;
}

// What a query sees: the tokens up to its own (chunks of several tokens), the same for all rows of a block (one new token per
// sequence), or a list of tokens.
enum { kChunks = 0, kSingle = 1, kSelected = 2 };

// Waves a SIMD that the registers allow (512 / waves each, without spilling).
constexpr int attend_waves(int t, int ds, int mode) {
    if (t == kF32) return ds <= 2 ? 3 : ds <= 5 ? 2 : 1;
    if (mode == kSingle) return ds <= 2 ? 4 : ds <= 4 ? 3 : 2;
    return ds <= 2 ? 4 : ds <= 4 ? 3 : ds <= 6 || mode == kSelected ? 2 : 1;
}

template <int T, int DS, int MODE, int WAVES>
__global__ __launch_bounds__(WAVES * 64, attend_waves(T, DS, MODE)) void kv_attend(KvAttendArgs a, Plan plan) {
    constexpr bool HALF = T == kF16, SEL = MODE == kSelected;
    constexpr int NQ = T == kF32 ? 3 : 1, NP = Parts<T>::value, D = DS * 32, ND = DS * 2, LDO = Shape<T, DS>::LDO;
    constexpr int VW = DS / 4 * 2 + (DS >> 1 & 1) + (DS & 1);  // words of a value that a lane holds
    constexpr int STEP = WAVES * 32;  // tokens that a block takes at a time
    extern __shared__ float smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, q4 = lane >> 4;
    const uint32_t H = a.mem.heads, P = a.mem.page_tokens, G = a.q_heads / H;
    uint32_t b = blockIdx.z, head = blockIdx.y, x = blockIdx.x;
    // Blocks go to the eight dies in turn.
    if constexpr (SEL) {
        // The heads of a sequence find their places in the same pages, whose scales and numbers lie side by side: all of a
        // sequence's blocks go to one die (100 sequences x 8 heads x 1000 tokens in bf16: 65 us without, 57 with).
        const uint64_t each = (uint64_t)gridDim.x * H, i = x + (uint64_t)gridDim.x * head + each * b;
        if (i < gridDim.z / 8 * 8 * each) {
            const uint64_t of = i / 8 % each;
            b = (uint32_t)(i % 8 + i / (8 * each) * 8), head = (uint32_t)(of / gridDim.x), x = (uint32_t)(of % gridDim.x);
        }
    }
    // With four or eight ranges a die would get one and the same range of every sequence, the last one of which only the long
    // sequences have: the ranges rotate from head to head (64 sequences of 1 000 to 8 192 tokens: 147 us without, 125 with).
    const uint32_t split = (x + head + b * H) % plan.splits;
    Sequence s;
    if (!sequence_of(a, b, s)) return;
    const UniformI32 table = (UniformI32)(a.batch.table + (uint64_t)b * a.batch.table_width);
    const int64_t* select = SEL ? a.select + ((uint64_t)b * H + head) * a.n_select : nullptr;
    const int64_t rows = (int64_t)s.n_new * G;
    const uint8_t* kc = (const uint8_t*)a.mem.k;
    const uint8_t* vc = (const uint8_t*)a.mem.v;
    const float to_log2 = a.scale * kLog2e;

    for (int64_t rt = x / plan.splits; rt * 16 < rows; rt += plan.tiles) {
        const int64_t row0 = rt * 16, row1 = min(row0 + 15, rows - 1);
        // positions of the tile's first and last row; tokens [lo, hi) are seen by some row, [lo_all, hi_all) by every row
        const int32_t pos0 = s.start + (int32_t)(row0 / G), pos1 = s.start + (int32_t)(row1 / G);
        int32_t lo, hi;
        range_of<SEL>(a, s, pos0, pos1, lo, hi);
        const bool same = MODE != kChunks || pos0 == pos1;
        const int32_t lo_all = a.window == 0 ? 0 : (int32_t)max((int64_t)0, pos1 - a.window + 1), hi_all = SEL ? hi : min(max(pos0, -1) + 1, hi);
        int32_t kb0 = lo & ~31, kb1 = hi;
        bool whole = true;  // this block sees all of the tile's tokens
        if (plan.splits > 1) {
            if (rt < plan.tiles) {
                whole = kb1 - kb0 <= (int32_t)plan.chunk;
                const int64_t at = kb0 + (int64_t)split * plan.chunk;
                if (split && at >= kb1) continue;
                kb0 = (int32_t)at;
                kb1 = (int32_t)min((int64_t)kb1, at + plan.chunk);
            } else if (split) {
                continue;
            }
        }
        const int64_t r = row0 + m;
        const bool live = r < rows;
        const int32_t tok = live ? (int32_t)(r / G) : 0;
        const uint32_t qh = head * G + (live ? (uint32_t)(r - (int64_t)tok * G) : 0);
        const int32_t pos = live ? s.start + tok : -1;

        // ---- where tokens lie
        // Not selected: a tile of 32 lies in one page or two, whose numbers are the same for the whole wave.  Pages that are
        // not there count as page 0 for the loads, and their tokens are masked.
        auto page_of = [&](int32_t t) -> int32_t {  // -1: none
            int32_t page = t < s.len ? table[t >> a.mem.page_shift] : -1;
            return (uint32_t)page < (uint32_t)a.mem.pages ? page : -1;
        };
        // Selected: lane l (and l + 32) looks place kb + (l & 31) of the list up, in three steps one tile apart, so that none
        // of the loads is waited for: token number, page number, then row and scales into the wave's table (two, in turn).
        int64_t* rows_s = (int64_t*)smem + wave * 128;       // [2][32] first bytes of rows (of row 0 for tokens that are not there)
        float* scales_s = (float*)smem + wave * 256 + 128;   // [2][64] key scales, value scales
        auto listed = [&](int32_t kb) -> int64_t {
            const int32_t i = kb + (lane & 31);
            return i < kb1 ? select[i] : -1;
        };
        auto paged = [&](int64_t t) -> int32_t { return t >= 0 && t < s.len ? a.batch.table[(uint64_t)b * a.batch.table_width + (t >> a.mem.page_shift)] : -1; };
        auto placed = [&](int64_t t, int32_t page, int slot) -> uint32_t {
            const bool there = (uint32_t)page < (uint32_t)a.mem.pages;
            const int64_t ph = (int64_t)page * H + head;
            if (lane < 32) rows_s[slot * 32 + lane] = there ? ((ph << a.mem.page_shift) + (t & (P - 1))) * D : 0;
            scales_s[slot * 64 + lane] = there ? (lane < 32 ? a.mem.k_scale : a.mem.v_scale)[ph] : 0.0f;
            return (uint32_t)__ballot(there);  // bit t: token t of the tile is there
        };

        u32x2 kw[2][DS];
        uint32_t vw[8][VW];
        auto load_keys = [&](int32_t kb, int32_t p0, int32_t p1, int slot) {
            int64_t row[2];
            if constexpr (SEL) {
                row[0] = rows_s[slot * 32 + (m >> 2) * 8 + (m & 3)];
                row[1] = rows_s[slot * 32 + (m >> 2) * 8 + 4 + (m & 3)];
            } else {
                const int64_t r0 = (((int64_t)max(p0, 0) * H + head) << a.mem.page_shift) + (kb & (P - 1));
                const int64_t r1 = (((int64_t)max(p1, 0) * H + head) << a.mem.page_shift) + ((kb + 16) & (P - 1)) - 16;
                row[0] = ((m < 8 ? r0 : r1) + (m >> 2) * 8 + (m & 3)) * D;
                row[1] = row[0] + 4 * D;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint8_t* p = kc + row[t] + (DS > 1 ? q4 * 16 : 0);
#pragma unroll
                for (int j = 0; j + 1 < DS; j += 2) {
                    const u32x4 w = *(const u32x4*)(p + j * 32);
                    kw[t][j] = u32x2{w[0], w[1]};
                    kw[t][j + 1] = u32x2{w[2], w[3]};
                }
                if constexpr (DS & 1) kw[t][DS - 1] = *(const u32x2*)(kc + row[t] + key_byte<DS>(q4, DS - 1));
            }
        };
        auto load_values = [&](int32_t kb, int32_t p0, int32_t p1, int slot) {
            int64_t first = 0;
            if constexpr (!SEL) {
                const int64_t r0 = (((int64_t)max(p0, 0) * H + head) << a.mem.page_shift) + (kb & (P - 1));
                const int64_t r1 = (((int64_t)max(p1, 0) * H + head) << a.mem.page_shift) + ((kb + 16) & (P - 1)) - 16;
                first = ((q4 < 2 ? r0 : r1) + q4 * 8) * D;
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const uint8_t* p = vc + (SEL ? rows_s[slot * 32 + q4 * 8 + t] : first + t * D);
#pragma unroll
                for (int c = 0; c < DS / 4; ++c) {
                    const u32x2 y = *(const u32x2*)(p + c * 128 + m * 8);
                    vw[t][2 * c] = y[0];
                    vw[t][2 * c + 1] = y[1];
                }
                if constexpr (DS & 2) vw[t][DS / 4 * 2] = *(const uint32_t*)(p + DS / 4 * 128 + m * 4);
                if constexpr (DS & 1) vw[t][VW - 1] = *(const uint16_t*)(p + DS / 2 * 64 + m * 2);
            }
        };

        u32x4 qf[NQ][DS];
        {
            const E<T>* q = (const E<T>*)a.q + (uint64_t)(s.first + tok) * a.q_token + (uint64_t)qh * a.q_head;
#pragma unroll
            for (int j = 0; j < DS; ++j) {
                const E<T>* qj = q + key_byte<DS>(q4, j);
                if constexpr (T == kF32) {
                    const f32x4 x = live ? *(const f32x4*)qj : f32x4{0, 0, 0, 0};
                    const f32x4 y = live ? *(const f32x4*)(qj + 4) : f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
                        qf[n][j] = u32x4{pack_hi16(bf16_part(x[0], n), bf16_part(x[1], n)), pack_hi16(bf16_part(x[2], n), bf16_part(x[3], n)),
                                         pack_hi16(bf16_part(y[0], n), bf16_part(y[1], n)), pack_hi16(bf16_part(y[2], n), bf16_part(y[3], n))};
                } else {
                    qf[0][j] = live ? *(const u32x4*)qj : u32x4{0, 0, 0, 0};
                }
            }
        }

        f32x4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = f32x4{0, 0, 0, 0};
        float top = kNone, sum = 0.0f;

        int32_t kb = kb0 + wave * 32;
        int32_t p0 = -1, p1 = -1, n0 = -1, n1 = -1;  // pages of this tile and of the next
        int64_t t1 = -1, t2 = -1;                    // selected: tokens of the next tile and of the one after it
        int32_t g1 = -1;                             // page of the next tile's token
        int slot = 0;
        uint32_t here = 0, next = 0;                 // selected: which tokens of this tile, and of the next, are there
        if (kb < kb1) {
            if constexpr (SEL) {
                const int64_t t0 = listed(kb);
                t1 = listed(kb + STEP);
                t2 = listed(kb + 2 * STEP);
                const int32_t g0 = paged(t0);
                g1 = paged(t1);
                here = placed(t0, g0, 0);
                __builtin_amdgcn_wave_barrier();
            } else {
                p0 = page_of(kb), p1 = page_of(kb + 16);
                n0 = page_of(kb + STEP), n1 = page_of(kb + STEP + 16);
            }
            load_keys(kb, p0, p1, 0);
        }
        for (; kb < kb1; kb += STEP) {
            const bool more = kb + STEP < kb1;
            load_values(kb, p0, p1, slot);
            float ks[SEL ? 8 : 1], vs[SEL ? 8 : 1];
            uint32_t have = 0;  // bit t: token t of the lane's 8 is there, and in the range that some row sees
            bool full;          // every row sees every token of the tile
            if constexpr (SEL) {
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    ks[t] = scales_s[slot * 64 + q4 * 8 + t];
                    vs[t] = scales_s[slot * 64 + 32 + q4 * 8 + t];
                }
                have = here >> (q4 * 8) & 255u;
                full = here == 0xFFFFFFFFu;
                if (more) {
                    next = placed(t1, g1, slot ^ 1);
                    g1 = paged(t2);
                    t1 = t2;
                    t2 = listed(kb + 3 * STEP);
                }
                __builtin_amdgcn_wave_barrier();
            } else {
                const int64_t x0 = (int64_t)max(p0, 0) * H + head, x1 = (int64_t)max(p1, 0) * H + head;
                const float ks0 = ((UniformF32)a.mem.k_scale)[x0], ks1 = ((UniformF32)a.mem.k_scale)[x1];
                const float vs0 = ((UniformF32)a.mem.v_scale)[x0], vs1 = ((UniformF32)a.mem.v_scale)[x1];
                ks[0] = q4 < 2 ? ks0 : ks1;
                vs[0] = q4 < 2 ? vs0 : vs1;
                full = kb >= lo_all && kb + 32 <= hi_all && p0 >= 0 && p1 >= 0;
                if (!full) {
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        const int32_t i = kb + q4 * 8 + t;
                        have |= (i >= lo && i < hi && (q4 < 2 ? p0 : p1) >= 0 ? 1u : 0u) << t;
                    }
                }
            }
            f32x4 sc[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < DS; ++j) {
                    const u32x4 kf = widen<HALF>(kw[t][j][0], kw[t][j][1]);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) sc[t] = mfma<HALF>(kf, qf[n][j], sc[t]);
                }
            }
            // the keys of the next tile travel while the values of this one are worked on
            if (more) load_keys(kb + STEP, n0, n1, slot ^ 1);
            // ---- softmax over what the lane's row sees of its 8 tokens
            float p[8];
#pragma unroll
            for (int t = 0; t < 8; ++t) p[t] = sc[t >> 2][t & 3] * (ks[SEL ? t : 0] * to_log2);
            uint32_t seen = 255;
            if (!full) {
                seen = live ? have : 0;
                if constexpr (MODE == kChunks) {
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        const int32_t i = kb + q4 * 8 + t;
                        if (!(i <= pos && (a.window == 0 || i > (int64_t)pos - a.window))) seen &= ~(1u << t);
                    }
                }
#pragma unroll
                for (int t = 0; t < 8; ++t) p[t] = seen >> t & 1 ? p[t] : -__builtin_inff();
                // what no row sees may hold anything: it is taken for zeros
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int w = 0; w < VW; ++w) vw[t][w] = have >> t & 1 ? vw[t][w] : 0;
            }
            float now = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(p[0], p[1]), __builtin_fmaxf(p[2], p[3])),
                                        __builtin_fmaxf(__builtin_fmaxf(p[4], p[5]), __builtin_fmaxf(p[6], p[7])));
            now = max_of_quarters(now);
            if (__any(now > top)) {
                now = __builtin_fmaxf(now, top);
                const float shrink = __builtin_amdgcn_exp2f(top - now);
                top = now;
                sum *= shrink;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] *= shrink;
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                p[t] = __builtin_amdgcn_exp2f(p[t] - top);
                sum += p[t];
                p[t] *= vs[SEL ? t : 0];
            }
            if (!full) {  // (a scale that belongs to no token may hold anything)
#pragma unroll
                for (int t = 0; t < 8; ++t) p[t] = seen >> t & 1 ? p[t] : 0.0f;
            }
            u32x4 pf[NP];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if constexpr (NP == 2) {  // rounded, and what is left of it (weights are finite or NaN)
                    const bf16x2 w = {(__bf16)p[2 * t], (__bf16)p[2 * t + 1]};
                    pf[0][t] = __builtin_bit_cast(uint32_t, w);
                    const bf16x2 r = {(__bf16)(p[2 * t] - float_of(pf[0][t] << 16)), (__bf16)(p[2 * t + 1] - float_of(pf[0][t] & 0xFFFF0000u))};
                    pf[1][t] = __builtin_bit_cast(uint32_t, r);
                } else {
#pragma unroll
                    for (int n = 0; n < NP; ++n) pf[n][t] = pack_hi16(bf16_part(p[2 * t], n), bf16_part(p[2 * t + 1], n));
                }
            }
            // a NaN among values that some rows of the tile do not see must not reach those (0 * NaN)
            bool mixed = false;
            if (MODE == kChunks && !full && !same) {
                uint32_t odd = 0;
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int w = 0; w < VW; ++w) odd |= nan_bytes(vw[t][w]);
                mixed = __any(odd != 0);
            }
            // ---- values: chunks of w dimensions a lane
            auto values = [&](auto is_mixed) {
            constexpr bool MIXED = decltype(is_mixed)::value;
#pragma unroll
            for (int c = 0; c < Chunks<DS>::count; ++c) {
                const int w = Chunks<DS>::width(c), word = c <= DS / 4 ? 2 * c : 2 * (DS / 4) + 1;
                uint32_t col[8][2];  // [dimension][tokens 0-3, 4-7]
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
                    for (int g = 0; g < (w + 3) / 4; ++g) {
                        const uint32_t in[4] = {vw[hf * 4][word + g], vw[hf * 4 + 1][word + g], vw[hf * 4 + 2][word + g], vw[hf * 4 + 3][word + g]};
                        uint32_t out[4];
                        transpose4(in, out);
#pragma unroll
                        for (int e = 0; e < 4 && g * 4 + e < w; ++e) col[g * 4 + e][hf] = out[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < w; ++e) {
                    const int d = Chunks<DS>::tile(c) + e;
                    uint32_t y = col[e][0], z = col[e][1];
                    if constexpr (MIXED) {
                        const uint32_t ny = nan_bytes(y) >> 7, nz = nan_bytes(z) >> 7;  // 1 in the bytes that are NaN
                        y &= ~(ny * 255u);
                        z &= ~(nz * 255u);
                        const u32x4 is_nan = widen<false>(ny * 0x38u, nz * 0x38u);  // 0x38 = 1.0
                        u32x4 sees;
#pragma unroll
                        for (int t = 0; t < 4; ++t) sees[t] = (seen >> (2 * t) & 1 ? 0x3F80u : 0u) | (seen >> (2 * t + 1) & 1 ? 0x3F800000u : 0u);
                        const f32x4 n = mfma<false>(is_nan, sees, f32x4{0, 0, 0, 0});
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n[i] > 0.0f) o[d][i] = float_of(0x7FC00000u);
                    }
                    const u32x4 vf = widen<false>(y, z);
#pragma unroll
                    for (int n = 0; n < NP; ++n) o[d] = mfma<false>(vf, pf[n], o[d]);
                }
            }
            };
            if constexpr (MODE == kChunks) {
                if (mixed) values(std::true_type());
                else values(std::false_type());
            } else {
                values(std::false_type());
            }
            p0 = n0, p1 = n1;
            if constexpr (!SEL) n0 = page_of(kb + 2 * STEP), n1 = page_of(kb + 2 * STEP + 16);
            slot ^= 1;
            here = next;
        }

        // ---- join the waves: each row's maximum, then sums and outputs in wave order
        float* so = smem;                     // [WAVES][16][LDO]
        float* st = smem + WAVES * 16 * LDO;  // [WAVES][16] maxima
        float* ss = st + WAVES * 16;          // [WAVES][16] sums
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (SEL) __syncthreads();  // the look-up tables of the waves lie there as well
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
        if (row < 16 && row0 + row < rows) {  // (16 threads a row: the first four waves; the others have no row in LDS)
            float best = kNone;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) best = __builtin_fmaxf(best, st[w * 16 + row]);
            float f[WAVES], total = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                f[w] = __builtin_amdgcn_exp2f(st[w * 16 + row] - best);
                total += f[w] * ss[w * 16 + row];
            }
            float v[ND];
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                v[d] = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) v[d] += f[w] * so[(w * 16 + row) * LDO + part * ND + d];
            }
            if (whole) {
                const int64_t ot = (row0 + row) / G;
                const uint64_t orow = (uint64_t)(s.first + ot) * a.q_heads + head * G + (uint32_t)(row0 + row - ot * G);
                const bool none = total == 0.0f;  // (a NaN is something)
                const float inv = none ? 0.0f : 1.0f / total;
                E<T>* out = (E<T>*)a.out + orow * D + part * ND;
#pragma unroll
                for (int d = 0; d < ND; ++d) out[d] = (E<T>)(none ? 0.0f : v[d] * inv);
                if (a.lse && part == 0) a.lse[orow] = none ? -__builtin_inff() : (best + __builtin_amdgcn_logf(total)) * kLn2;
            } else {
                float* w = plan.part + (((((uint64_t)b * H + head) * plan.tiles + rt) * plan.splits + split) * 16 + row) * (D + 2);
#pragma unroll
                for (int d = 0; d < ND; d += 2) *(f32x2*)(w + part * ND + d) = f32x2{v[d], v[d + 1]};
                if (part == 0) *(f32x2*)(w + D) = f32x2{best, total};
            }
        }
        __syncthreads();
    }
}

// ---- many rows: chunks of prompts ---------------------------------------------------------------------
//
// Four or eight waves of NT tiles of 16 rows go through the tokens together, 64 at a time.  What bounds this is, next to the
// matrix units (256 cycles for 32 tokens x 16 rows at 128 dimensions), the softmax on the vector units (about as long: an exp2
// costs four instructions) and the reads of LDS; so
//   - codes are widened to bf16 (f16) once per block, into LDS in the order in which lanes hold matrix operands; a wave uses
//     each operand it reads for its NT row tiles;
//   - the scale of a page's values is folded into the exponent: w = exp2(score + log2 v_scale - M) with M the running
//     maximum of just that, and the softmax's sum takes w / v_scale; so a score costs one fma, one exp2, one add.  (Where the
//     scales of a head's pages lie so far apart that w could underflow and w / v_scale count - pages of zeros beside values of
//     thousands do - the weight is w / v_scale from the start, and costs a product more.)
//   - the loads of the tile after next are under way while one is computed and the next is being widened.
// Measured: four chunks of 30 to 2048 tokens, the longest sequence 6 000, 32 heads on 8, 128 dimensions, bf16: 284 us, 325 in the first
// launches, before the clock has risen (its matrix products at the rate of a large product: 182); then, of a block's 45 to 240 us, 2.3 a tile, 4 one at an edge, and some 25 to start
// and end.  Left out in turn, the loads, the exp2, either product, the barrier or the widening save 5 to 15 % each: nothing of it
// alone is what takes the time.
template <int T, int DS>
struct Many {
    static constexpr int NT = T == kF32 || DS > 5 ? 1 : 2;  // (192 dimensions: 511 us with one, 627 with two; 160: 473, 380)
    // Two blocks of four waves or one of eight a CU (waves of one block wait for each other, but it widens its tokens for twice
    // the rows).  Four: 32 dimensions 166 us against 193, 64 202 against 228, 128 in f16 428 against 454, in f32 642 against 695;
    // eight: 96 261 against 297, 128 in bf16 325 against 339, 160 380 against 640, 256 611 against 1014, but in f32 1990 against 1609,
    // where three parts of the queries would not fit the registers.
    static constexpr bool four = DS <= 2 || (T != kBF16 && DS == 4) || (T == kF32 && DS > 6);
    static constexpr int kThreads = four ? 256 : 512, occupancy = DS <= 2 ? 3 : DS > 6 && four ? 1 : 2;  // occupancy: waves a SIMD
    static constexpr int rows = kThreads / 64 * NT * 16;
    static constexpr int D = DS * 32, ND = DS * 2;
    static constexpr int side = 64 * D * 2;                // bytes of 64 keys (or values) in bf16
    static constexpr size_t lds = 4 * side + 80;           // two buffers of both, of the scales of four pages each, and of a tile's number
    static constexpr int units = (D * 4 + kThreads - 1) / kThreads;  // 16 bytes of keys, and 4 tokens x 4 dimensions of values, that a thread widens; D * 4 of each in all
};

// Which rows a block takes.  An item is `rows` rows of one sequence (for one head); its cost is the number of tokens that its last
// row sees.  Items go to the blocks by falling cost, over all sequences: blocks start in the order of their numbers, so the
// long ones are under way first and the short ones fill up the end.  (Found by every wave for itself: 4 us a block.)
struct Items {
    Sequence mine;  // sequence `lane`
    int32_t seen;   // tokens that its last row sees
    int32_t items;

    __device__ __forceinline__ Items(const KvAttendArgs& a, int lane, uint32_t G, uint32_t rows) {
        mine.n_new = mine.start = mine.len = seen = items = 0;
        mine.first = 0;
        if ((uint32_t)lane < a.batch.count && sequence_of(a, lane, mine)) {
            seen = (int32_t)min((int64_t)mine.len, a.window == 0 ? (int64_t)0x7FFFFFFF : a.window + rows);
            items = (int32_t)(((uint64_t)mine.n_new * G + rows - 1) / rows);
        } else {
            mine.n_new = 0;
        }
    }
    // items of sequence b that see at least `tokens`
    __device__ __forceinline__ int32_t at_least(int b, uint32_t tokens, uint32_t G, uint32_t rows) const {
        const uint32_t n = __builtin_amdgcn_readlane(items, b);
        // (rows before the first token, of a length that counts fewer tokens than there are new ones, see 0)
        const int32_t more = tokens ? (int32_t)tokens - 1 - max(__builtin_amdgcn_readlane(mine.start, b), -(1 << 30)) : 0;
        const uint32_t before = (uint32_t)min((uint64_t)(uint32_t)max(more, 0) * G / rows, (uint64_t)0xFFFFFFFF);
        return tokens > (uint32_t)__builtin_amdgcn_readlane(seen, b) ? 0 : (int32_t)(n - min(before, max(n, 1u) - 1));
    }
    // Item k by falling cost (in steps of 64 tokens): 64 costs are looked at at once, one a lane.
    __device__ __forceinline__ bool find(uint32_t count, int lane, int64_t k, uint32_t G, uint32_t rows, Sequence& s, uint32_t& b, int32_t& block) const {
        int32_t most = 0;
        int64_t all = 0;
        for (uint32_t i = 0; i < count; ++i) most = max(most, __builtin_amdgcn_readlane(seen, i)), all += __builtin_amdgcn_readlane(items, i);
        if (k >= all) return false;
        int32_t lo = 0, end = most / 64 + 1;
        while (end - lo > 1) {
            const int32_t step = (end - lo + 63) / 64;
            const int32_t here = min(lo + lane * step, most / 64 + 1);
            int64_t n = 0;
            for (uint32_t i = 0; i < count; ++i) n += at_least(i, here * 64u, G, rows);
            const uint64_t yes = __ballot(here < end && n > k);  // lane 0 always
            lo += (63 - __builtin_clzll(yes)) * step;
            end = min(end, lo + step);
        }
        // those of that cost, sequence by sequence
        for (uint32_t i = 0; i < count; ++i) k -= at_least(i, (lo + 1) * 64u, G, rows);
        for (b = 0; b < count; ++b) {
            const int32_t more = at_least(b, (lo + 1) * 64u, G, rows), here = at_least(b, lo * 64u, G, rows) - more;
            if (k < here) {
                block = __builtin_amdgcn_readlane(items, b) - more - 1 - (int32_t)k;
                s.first = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int32_t)(mine.first >> 32), b) << 32 | (uint32_t)__builtin_amdgcn_readlane((int32_t)mine.first, b));
                s.n_new = __builtin_amdgcn_readlane(mine.n_new, b);
                s.start = __builtin_amdgcn_readlane(mine.start, b);
                s.len = __builtin_amdgcn_readlane(mine.len, b);
                return true;
            }
            k -= here;
        }
        return false;
    }
};

// Places for the items of all sequences together: no fewer than there are.
__host__ __device__ __forceinline__ int64_t many_items(const KvBatch& t, uint32_t G, uint32_t rows) { return (int64_t)(t.tokens * G / rows + t.count); }

// x, but computed where it is used: what follows from it is not kept in registers through the loops.
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// x is computed here, and not moved to where it is next used (with all that it is computed from).
__device__ __forceinline__ void keep(float& x) { asm volatile("" : "+v"(x)); }

template <int T, int DS>
__global__ __launch_bounds__((Many<T, DS>::kThreads), (Many<T, DS>::occupancy)) void kv_attend_many(KvAttendArgs a) {
    typedef Many<T, DS> M;
    constexpr bool HALF = T == kF16;
    constexpr int NQ = T == kF32 ? 3 : 1, NP = Parts<T, true>::value, D = M::D, ND = M::ND, NT = M::NT, side = M::side;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, q4 = lane >> 4;
    const uint32_t H = a.mem.heads, head = blockIdx.x % H, P = a.mem.page_tokens, G = a.q_heads / H;
    float* scales_s = (float*)(lds + 4 * side);  // [2][8]: of keys, of values
    const uint8_t* kc = (const uint8_t*)a.mem.k;
    const uint8_t* vc = (const uint8_t*)a.mem.v;
    const float to_log2 = __builtin_fabsf(a.scale) * kLog2e;
    const uint32_t flip = a.scale < 0.0f ? (T == kF32 ? 0x80000000u : 0x80008000u) : 0u;  // the scale's sign goes into the queries
    Sequence s;
    const int32_t* table = nullptr;
    // Page numbers: 64 of them in a register of the wave, refilled every 64 pages.  (Scalar loads would do, but a wait for LDS is
    // a wait for them as well.)
    int32_t held = -1, held_from = 0;
    auto page_of = [&](int32_t t) -> int32_t {  // -1: none
        return t < s.len ? __builtin_amdgcn_readlane(held, (t >> a.mem.page_shift) - held_from) : -1;
    };
    auto pages = [&](int32_t kb) {  // of a tile, one for every 16 tokens
        if (kb < s.len && ((kb + 63) >> a.mem.page_shift) - held_from > 63) {
            held_from = kb >> a.mem.page_shift;
            const uint32_t at = held_from + lane;
            const int32_t page = at < a.batch.table_width ? table[at] : -1;
            held = (uint32_t)page < (uint32_t)a.mem.pages ? page : -1;
        }
        return i32x4{page_of(kb), page_of(kb + 16), page_of(kb + 32), page_of(kb + 48)};
    };

    for (int64_t k = blockIdx.x / H;; k += gridDim.x / H) {
        uint32_t b = 0;
        int32_t rb = 0;
        if (a.batch.count <= 64) {
            if (!Items(a, lane, G, M::rows).find(a.batch.count, lane, k, G, M::rows, s, b, rb)) break;
        } else {
            // More sequences: in their order.  Sequence b has places for its items, and one at most that stays empty, from here on.
            if (k >= many_items(a.batch, G, M::rows)) break;
            auto base = [&](uint32_t i) { return (int64_t)(a.batch.offsets ? max(a.batch.offsets[i], 0) : (int32_t)i) * G / M::rows + i; };
            uint32_t end = a.batch.count;
            while (end - b > 1) {
                const uint32_t mid = (b + end) / 2;
                if (base(mid) <= k) b = mid;
                else end = mid;
            }
            if (!sequence_of(a, b, s)) continue;
            const int64_t n = ((int64_t)s.n_new * G + M::rows - 1) / M::rows, at = k - base(b);
            if (at < 0 || at >= n) continue;
            rb = (int32_t)(n - 1 - at);
        }
        const int64_t rows = (int64_t)s.n_new * G;
        table = a.batch.table + (uint64_t)b * a.batch.table_width;
        const int64_t row0 = (int64_t)rb * M::rows;
        const int32_t here = (int32_t)min(rows - row0, (int64_t)M::rows);  // rows of the item
        const int32_t tok0 = (int32_t)(row0 / G);
        const uint32_t qh0 = (uint32_t)(row0 - (int64_t)tok0 * G);
        auto token = [&](int32_t r) { return tok0 + (int32_t)((qh0 + r) / G); };             // of row r of the item
        auto q_head = [&](int32_t r) { return head * G + (qh0 + r) % G; };
        const int32_t pos0 = s.start + tok0, pos1 = s.start + token(here - 1);
        int32_t lo, hi;
        range_of<false>(a, s, pos0, pos1, lo, hi);
        // this wave's rows
        const int32_t wrow0 = wave * NT * 16;
        const bool idle = wrow0 >= here;
        const int32_t wpos0 = s.start + token(min(wrow0, here - 1)), wpos1 = s.start + token(min(wrow0 + NT * 16, here) - 1);
        const int32_t w_lo = a.window == 0 ? 0 : (int32_t)max((int64_t)0, wpos0 - a.window + 1);
        // the tokens [lo_all, hi_all) are seen by all rows of the block, [w_lo_all, w_hi_all) by all of the wave
        const int32_t w_lo_all = a.window == 0 ? 0 : (int32_t)max((int64_t)0, wpos1 - a.window + 1), w_hi_all = idle ? 0 : min(max(wpos0, -1) + 1, hi);
        const int32_t lo_all = a.window == 0 ? 0 : (int32_t)max((int64_t)0, pos1 - a.window + 1), hi_all = min(max(pos0, -1) + 1, hi);
        f32x4 o[NT][ND];
        float top[NT], sum[NT];
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            top[ct] = wrow0 + ct * 16 + m < here ? kNone : -kNone, sum[ct] = 0.0f;  // (a row that does not exist has no weights)
#pragma unroll
            for (int d = 0; d < ND; ++d) o[ct][d] = f32x4{0, 0, 0, 0};
        }

        // Places in LDS, in bytes, apart from multiples of 1 KB (a matrix operand) that go into the instructions.  Operand rows are
        // exchanged by j (keys) and d (values), so that the pieces that neighbouring threads write lie in different banks.
        uint32_t key_at[4], value_at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            key_at[j] = (q4 * 16 + (m ^ ((j * 2 + (q4 >> 1)) & 7))) * 16;
            value_at[j] = side + (q4 * 16 + (m ^ j)) * 16;
        }
        // ---- staging: a thread widens `pieces` 16-byte pieces of keys, and `units` of 8 tokens x 4 dimensions of values
        float scale_r = 1.0f;  // of threads 0-7
        constexpr int kThreads = M::kThreads;
        u32x4 kr[M::units];
        uint32_t vr[M::units][4];
        const uint64_t page_bytes = (uint64_t)H * P * D;
        const uint8_t* const kh = kc + (uint64_t)head * P * D;
        const uint8_t* const vh = vc + (uint64_t)head * P * D;
        auto pick = [&](i32x4 pg, int i) { return i < 2 ? (i == 0 ? pg[0] : pg[1]) : (i == 2 ? pg[2] : pg[3]); };
        auto load = [&](int32_t kb, i32x4 pg) {
            if (tid < 8) {  // (a page of which no row sees a token may have any scale: it is taken for 0)
                const int32_t page = pick(pg, tid & 3), t = kb + (tid & 3) * 16;
                scale_r = page >= 0 && t < hi && t + 16 > lo ? (tid < 4 ? a.mem.k_scale : a.mem.v_scale)[(int64_t)page * H + head] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < M::units; ++i) {
                const int piece = tid + i * kThreads;
                if (D * 4 % kThreads == 0 || piece < D * 4) {
                    const int tok = piece / (D / 16), c = piece % (D / 16);
                    const uint32_t page = (uint32_t)max(pick(pg, tok >> 4), 0);
                    kr[i] = *(const u32x4*)(kh + page * page_bytes + ((kb + tok) & (P - 1)) * (uint32_t)D + c * 16);
                }
            }
#pragma unroll
            for (int i = 0; i < M::units; ++i) {
                const int unit = tid + i * kThreads;
                if (D * 4 % kThreads == 0 || unit < D * 4) {
                    const int grp = unit / (D / 4), c = unit % (D / 4);
                    const uint32_t page = (uint32_t)max(pick(pg, grp >> 2), 0);
                    const uint8_t* p = vh + page * page_bytes + ((kb + grp * 4) & (P - 1)) * (uint32_t)D + c * 4;
#pragma unroll
                    for (int t = 0; t < 4; ++t) vr[i][t] = *(const uint32_t*)(p + t * D);
                }
            }
        };
        // every row of the block sees every token of the tile
        auto plain = [&](int32_t kb, i32x4 pg) {
            return kb >= lo_all && kb + 64 <= hi_all && (pg[0] | pg[1] | pg[2] | pg[3]) >= 0;
        };
        auto plain_here = [&](int32_t kb, i32x4 pg) {  // of the wave
            return kb >= w_lo_all && kb + 64 <= w_hi_all && (pg[0] | pg[1] | pg[2] | pg[3]) >= 0;
        };
        // What no row sees may hold anything: it is taken for zeros.  Of NaN among the rest, nan_s[] tells the tile's waves.
        int32_t* nan_s = (int32_t*)(scales_s + 16);
        auto hide = [&](int32_t kb, i32x4 pg, int buf) {
            if (!plain(kb, pg)) {
                uint32_t nan = 0;
                const int tid = fresh((int)threadIdx.x);
#pragma unroll
                for (int i = 0; i < M::units; ++i) {
                    const int grp = (tid + i * kThreads) / (D / 4), t0 = kb + grp * 4;
                    const bool there = pick(pg, (grp >> 2) & 3) >= 0;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        vr[i][t] = there && t0 + t >= lo && t0 + t < hi ? vr[i][t] : 0;
                        if (D * 4 % kThreads == 0 || tid + i * kThreads < D * 4) nan |= nan_bytes(vr[i][t]);
                    }
                }
                if (nan) nan_s[buf] = kb;
            }
        };
        auto store_keys = [&](int buf) {
            unsigned char* ks = lds + buf * 2 * side;
            if (tid < 8) scales_s[buf * 8 + tid] = scale_r;
#pragma unroll
            for (int i = 0; i < M::units; ++i) {
                const int piece = tid + i * kThreads;
                if (D * 4 % kThreads == 0 || piece < D * 4) {
                    // token x of 32: row (x >> 3) * 4 + (x & 3) of score tile (x >> 2) & 1.  Bytes 16 c .. + 15: quarters
                    // 2 (c & 1), 2 (c & 1) + 1 of step c / 2.  Rows are exchanged by c, so that pieces of one token go to other banks.
                    const int tok = piece / (D / 16), c = piece % (D / 16), x = tok & 31;
                    const int tile = (tok >> 5) * 2 + (x >> 2 & 1), row = ((x >> 3) * 4 + (x & 3)) ^ (c & 7);
                    unsigned char* w = ks + ((tile * DS + (c >> 1)) * 64 + (c & 1) * 32 + row) * 16;
                    *(u32x4*)w = widen<HALF>(kr[i][0], kr[i][1]);
                    *(u32x4*)(w + 256) = widen<HALF>(kr[i][2], kr[i][3]);
                }
            }
        };
        auto store_values = [&](int buf) {
            unsigned char* vs = lds + buf * 2 * side + side;
#pragma unroll
            for (int i = 0; i < M::units; ++i) {
                const int unit = tid + i * kThreads;
                if (D * 4 % kThreads == 0 || unit < D * 4) {
                    const int grp = unit / (D / 4), c = unit % (D / 4);
                    uint32_t x[4];
                    transpose4(vr[i], x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = c * 4 + e, dt = d >> 4;
                        *(u32x2*)(vs + ((dt * 2 + (grp >> 3)) * 64 + (grp >> 1 & 3) * 16 + ((d & 15) ^ (dt & 3))) * 16 + (grp & 1) * 8) = widen4<false>(x[e]);
                    }
                }
            }
        };

        const int32_t kb0 = lo & ~63;
        i32x4 pa, pb, pc;  // pages of this tile, of the next, of the one after it
        if (kb0 < hi) {
            held_from = -64;
            pa = pages(kb0);
            pb = pages(kb0 + 64);
            pc = pages(kb0 + 128);
            load(kb0, pa);
        }
        // (the queries travel beside the first tokens)
        u32x4 qf[NT][NQ][DS];
        int32_t pos[NT];
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            const int32_t r = wrow0 + ct * 16 + m;
            const bool live = r < here;
            const int32_t tok = live ? token(r) : 0;
            const uint32_t qh = live ? q_head(r) : 0;
            pos[ct] = live ? s.start + tok : -1;
            const E<T>* q = (const E<T>*)a.q + (uint64_t)(s.first + tok) * a.q_token + (uint64_t)qh * a.q_head + q4 * 8;
#pragma unroll
            for (int j = 0; j < DS; ++j) {
                if constexpr (T == kF32) {
                    u32x4 x = live ? *(const u32x4*)(q + j * 32) : u32x4{0, 0, 0, 0};
                    u32x4 y = live ? *(const u32x4*)(q + j * 32 + 4) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] ^= flip, y[i] ^= flip;
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            qf[ct][n][j][i] = pack_hi16(bf16_part(float_of(x[2 * i]), n), bf16_part(float_of(x[2 * i + 1]), n));
                            qf[ct][n][j][2 + i] = pack_hi16(bf16_part(float_of(y[2 * i]), n), bf16_part(float_of(y[2 * i + 1]), n));
                        }
                } else {
                    qf[ct][0][j] = live ? *(const u32x4*)(q + j * 32) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[ct][0][j][i] ^= flip;
                }
            }
        }
        if (tid < 2) nan_s[tid] = -1;
        __syncthreads();  // (of the last rows, too, that all waves are done)
        if (kb0 < hi) {
            hide(kb0, pa, 0);
            store_keys(0);
            store_values(0);
            if (kb0 + 64 < hi) load(kb0 + 64, pb);
        }
        __syncthreads();
        int32_t kb = kb0;
        int buf = 0;
        float c[2], lv[2], inv[2], vs[2];  // of the tile's pages: scale of the scores, log2, inverse and scale of the values
        float v_least = 0.0f;  // 2^-60 of the largest scale of values that the softmax's reference can have come from
        auto read_scales = [&] {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                c[h] = scales_s[buf * 8 + 2 * h + (q4 >> 1)] * to_log2;
                vs[h] = __builtin_fmaxf(scales_s[buf * 8 + 4 + 2 * h + (q4 >> 1)], 0x1p-120f);
                lv[h] = __builtin_amdgcn_logf(vs[h]), inv[h] = __builtin_amdgcn_rcpf(vs[h]);
            }
        };
        u32x4 ring[4];  // operands are read three products ahead
        auto read_key = [&](int e) { ring[e & 3] = *(const u32x4*)(lds + buf * 2 * side + key_at[e % DS & 3] + e * 1024); };
        auto read_value = [&](int e) { ring[e & 3] = *(const u32x4*)(lds + buf * 2 * side + value_at[e % ND & 3] + (e % ND * 2 + e / ND) * 1024); };
        auto pack_weights = [&](float p, float r, u32x4 (&w)[NP], int t) {
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                if constexpr (NP == 1) {
                    bf16x2 x = {(__bf16)p, (__bf16)r};
                    w[n][t] = __builtin_bit_cast(uint32_t, x);
                } else {
                    w[n][t] = pack_hi16(bf16_part(p, n), bf16_part(r, n));
                }
            }
        };
        // A tile at an edge, the first ones, and where the softmax's reference has to move: 32 tokens at a time, so that the scores
        // take no more registers than in the other loop.
        auto careful = [&] {
            read_scales();
#pragma unroll
            for (int i = 0; i < 4; ++i) v_least = __builtin_fmaxf(v_least, scales_s[buf * 8 + 4 + i] * 0x1p-60f);
            const bool nan_here = __builtin_amdgcn_readfirstlane(nan_s[buf]) == kb;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x4 sc[NT][2];
#pragma unroll
                for (int e = 0; e < 3 && e < 2 * DS; ++e) read_key(h * 2 * DS + e);
#pragma unroll
                for (int e = 0; e < 2 * DS; ++e) {
                    if (e + 3 < 2 * DS) read_key(h * 2 * DS + e + 3);
#pragma unroll
                    for (int ct = 0; ct < NT; ++ct) {
                        if (e % DS == 0) sc[ct][e / DS] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int n = 0; n < NQ; ++n) sc[ct][e / DS] = mfma<HALF>(ring[(h * 2 * DS + e) & 3], qf[ct][n][e % DS], sc[ct][e / DS]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                u32x4 pf[NT][NP];
                uint32_t seen[NT];
#pragma unroll
                for (int ct = 0; ct < NT; ++ct) {
                    // the row sees the tokens first + [from, to) of the lane's 8 (a window reaches below 0 by 2^63 at most)
                    const int32_t first = kb + h * 32 + (fresh(lane) >> 4) * 8, at = fresh(pos[ct]);
                    const bool there = (q4 < 2 ? pa[2 * h] : pa[2 * h + 1]) >= 0;
                    const int64_t least = a.window == 0 ? 0 : (int64_t)at - a.window + 1;
                    const int32_t to = there ? min(max(min(at, s.len - 1) + 1 - first, 0), 8) : 0;
                    const int32_t from = (int32_t)min(max(least - first, (int64_t)0), (int64_t)8);
                    seen[ct] = ((1u << to) - 1) & ~((1u << from) - 1);
                    float now = top[ct], p[8];
#pragma unroll
                    for (int t = 0; t < 8; ++t) now = __builtin_fmaxf(now, seen[ct] >> t & 1 ? __builtin_fmaf(sc[ct][t >> 2][t & 3], c[h], lv[h]) : -__builtin_inff());
                    now = max_of_quarters(now);
                    const float shrink = __builtin_amdgcn_exp2f(top[ct] - now);
                    top[ct] = now;
#pragma unroll
                    for (int d = 0; d < ND; ++d) o[ct][d] *= shrink;
#pragma unroll
                    for (int t = 0; t < 8; ++t) p[t] = seen[ct] >> t & 1 ? __builtin_amdgcn_exp2f(__builtin_fmaf(sc[ct][t >> 2][t & 3], c[h], -now)) : 0.0f;
                    sum[ct] = __builtin_fmaf(sum[ct], shrink, ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
#pragma unroll
                    for (int t = 0; t < 8; ++t) p[t] *= vs[h];
                    keep(sum[ct]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) pack_weights(p[2 * t], p[2 * t + 1], pf[ct], t);
                    __builtin_amdgcn_sched_barrier(0);
                }
                auto products = [&](auto has_nan) {
#pragma unroll
                    for (int e = 0; e < 3; ++e) read_value(h * ND + e);
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        if (d + 3 < ND) read_value(h * ND + d + 3);
                        u32x4 x = ring[(h * ND + d) & 3];
                        if constexpr (decltype(has_nan)::value) {
                            // A NaN among values that some rows do not see must not reach those (0 * NaN): it is taken out,
                            // and counted for each row by a product of its own.
                            u32x4 is_nan;
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const uint32_t n = ((x[t] & 0x7FFFu) > 0x7F80u ? 0xFFFFu : 0u) | ((x[t] & 0x7FFF0000u) > 0x7F800000u ? 0xFFFF0000u : 0u);
                                is_nan[t] = n & 0x3F803F80u;
                                x[t] &= ~n;
                            }
#pragma unroll
                            for (int ct = 0; ct < NT; ++ct) {
                                u32x4 sees;
#pragma unroll
                                for (int t = 0; t < 4; ++t)
                                    sees[t] = (seen[ct] >> (2 * t) & 1 ? 0x3F80u : 0u) | (seen[ct] >> (2 * t + 1) & 1 ? 0x3F800000u : 0u);
                                const f32x4 n = mfma<false>(is_nan, sees, f32x4{0, 0, 0, 0});
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[ct][d][i] = n[i] > 0.0f ? float_of(0x7FC00000u) : o[ct][d][i];
                            }
                        }
#pragma unroll
                        for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                            for (int n = 0; n < NP; ++n) o[ct][d] = mfma<false>(x, pf[ct][n], o[ct][d]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                if (nan_here) products(std::true_type());
                else products(std::false_type());
            }
        };
        // A tile of which every row of the wave sees every token, against the running reference as it is.  That need not be the
        // maximum: no score is compared with another while the sums of the weights stay below 2^11.  Where one does not (rarely:
        // in the first tiles) the answer is false, nothing has been added up, and the tile is done again by `careful`.  (One loop
        // that does both holds every output twice, and so does one with a second branch beside `careful`: what is spilled then
        // comes back from HBM, 12 us a tile instead of 4.)
        auto simple = [&]() -> bool {
            read_scales();
            // scores; the next tile is widened beside them
            f32x4 sc[2][NT][2];
#pragma unroll
            for (int e = 0; e < 3 && e < 4 * DS; ++e) read_key(e);
#pragma unroll
            for (int e = 0; e < 4 * DS; ++e) {
                const int i = e / DS, j = e % DS;
                if (e + 3 < 4 * DS) read_key(e + 3);
                if (e == DS) store_keys(buf ^ 1);
                if (e == 2 * DS) store_values(buf ^ 1);
#pragma unroll
                for (int ct = 0; ct < NT; ++ct) {
                    if (j == 0) sc[i >> 1][ct][i & 1] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int n = 0; n < NQ; ++n) sc[i >> 1][ct][i & 1] = mfma<HALF>(ring[e & 3], qf[ct][n][j], sc[i >> 1][ct][i & 1]);
                }
                if (j == DS - 1) __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);  // a wave in its products goes before one in its softmax: 317 us against 327
            u32x4 pf[2][NT][NP];
            float more[NT];
            // (where a page's scale is that far below, a weight times it could underflow though it counts in the sum)
            bool over = __builtin_fminf(vs[0], vs[1]) < v_least;
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) {
                more[ct] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float off = lv[h] - top[ct];
                    float p[8];
#pragma unroll
                    for (int t = 0; t < 8; ++t) p[t] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[h][ct][t >> 2][t & 3], c[h], off));
                    const float part = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                    over |= part > 2048.0f;
                    more[ct] = __builtin_fmaf(part, inv[h], more[ct]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) pack_weights(p[2 * t], p[2 * t + 1], pf[h][ct], t);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (__any(over)) return false;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) sum[ct] += more[ct];
            if (kb + 128 < hi) load(kb + 128, pc);
#pragma unroll
            for (int e = 0; e < 3; ++e) read_value(e);
#pragma unroll
            for (int e = 0; e < 2 * ND; ++e) {
                const int h = e / ND, d = e % ND;
                if (e + 3 < 2 * ND) read_value(e + 3);
#pragma unroll
                for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                    for (int n = 0; n < NP; ++n) o[ct][d] = mfma<false>(ring[e & 3], pf[h][ct][n], o[ct][d]);
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
            return true;
        };
        auto advance = [&] {
            pa = pb, pb = pc, pc = pages(kb + 192);
            kb += 64;
            buf ^= 1;
            __syncthreads();
        };
        // (behind the last tile the other buffer is filled with what the registers hold, and read by nobody)
        // Every wave passes the same barriers, one a tile, from whichever of the two loops.
        while (kb < hi) {
            if (kb + 64 < hi) hide(kb + 64, pb, buf ^ 1);
            store_keys(buf ^ 1);
            store_values(buf ^ 1);
            if (!idle && kb <= wpos1 && kb + 63 >= w_lo) careful();
            if (kb + 128 < hi) load(kb + 128, pc);
            advance();
            bool again = false;
            while (kb < hi && plain_here(kb, pa) && !again) {
                if (kb + 64 < hi) hide(kb + 64, pb, buf ^ 1);
                again = !simple();
                if (!again) advance();
            }
        }
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            float total = sum[ct];
            total += __shfl_xor(total, 16);
            total += __shfl_xor(total, 32);
            const int32_t r = wrow0 + ct * 16 + fresh(m);
            if (r < here) {
                const uint64_t orow = (uint64_t)(s.first + token(r)) * a.q_heads + q_head(r);
                const bool none = total == 0.0f;
                const float inv = none ? 0.0f : 1.0f / total;
                E<T>* out = (E<T>*)a.out + orow * D + q4 * 4;
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    typedef __attribute__((ext_vector_type(4))) E<T> vec;
                    vec v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = (E<T>)(none ? 0.0f : o[ct][d][i] * inv);
                    *(vec*)(out + d * 16) = v;
                }
                if (a.lse && q4 == 0) a.lse[orow] = none ? -__builtin_inff() : (top[ct] + __builtin_amdgcn_logf(total)) * kLn2;
            }
        }
    }
}

// Adds up the ranges of a row, of which there are at most 16: a wave a row, lane i weighs range i, then each lane adds up two or
// four dimensions, in the order of the ranges.
template <int T, bool SEL>
__global__ __launch_bounds__(256) void kv_join_few(KvAttendArgs a, Plan plan) {
    const uint32_t b = blockIdx.z, head = blockIdx.y, H = a.mem.heads, G = a.q_heads / H, D = a.mem.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Sequence s;
    if (!sequence_of(a, b, s)) return;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave, rows = min((int64_t)s.n_new * G, (int64_t)plan.tiles * 16), rt = row / 16;
    if (row >= rows) return;
    int32_t lo, hi;
    range_of<SEL>(a, s, s.start + (int32_t)(rt * 16 / G), s.start + (int32_t)(min(rt * 16 + 15, (int64_t)s.n_new * G - 1) / G), lo, hi);
    lo &= ~31;
    if (hi - lo <= (int32_t)plan.chunk) return;  // written by kv_attend
    const uint32_t used = min(((uint32_t)(hi - lo) + plan.chunk - 1) / plan.chunk, plan.splits);
    const uint64_t step = 16 * (D + 2);
    const float* part = plan.part + ((((uint64_t)b * H + head) * plan.tiles + rt) * plan.splits * 16 + row % 16) * (D + 2);
    const f32x2 mine = (uint32_t)lane < used ? *(const f32x2*)(part + lane * step + D) : f32x2{kNone, 0.0f};
    float best = mine[0];
#pragma unroll
    for (int o = 32; o; o >>= 1) best = __builtin_fmaxf(best, __shfl_xor(best, o));
    const float f = (uint32_t)lane < used ? __builtin_amdgcn_exp2f(mine[0] - best) : 0.0f;
    float sum = f * mine[1];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    const uint32_t per = D > 128 ? 4 : 2, d = lane * per;
    if (d >= D) return;
    f32x2 acc[2] = {{0, 0}, {0, 0}};
    for (uint32_t i = 0; i < used; i += 8) {
        f32x2 x[8][2];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float* w = part + (uint64_t)min(i + u, used - 1) * step + d;
            x[u][0] = *(const f32x2*)w;
            x[u][1] = per == 4 ? *(const f32x2*)(w + 2) : f32x2{0, 0};
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i + u < used) {
                const float g = float_of(__builtin_amdgcn_readlane(bits_of(f), i + u));
                acc[0] += x[u][0] * g;
                acc[1] += x[u][1] * g;
            }
    }
    const int64_t ot = row / G;
    const uint64_t orow = (uint64_t)(s.first + ot) * a.q_heads + head * G + (uint32_t)(row - ot * G);
    const bool none = sum == 0.0f;
    const float inv = none ? 0.0f : 1.0f / sum;
    E<T>* out = (E<T>*)a.out + orow * D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < (int)per) out[i] = (E<T>)(none ? 0.0f : acc[i >> 1][i & 1] * inv);
    if (a.lse && lane == 0) a.lse[orow] = none ? -__builtin_inff() : (best + __builtin_amdgcn_logf(sum)) * kLn2;
}

// The same for many ranges: a block takes 32 dimensions of a row, eight threads a range, so that 64 ranges are under way at a time.
template <int T, bool SEL>
__global__ __launch_bounds__(512) void kv_join_long(KvAttendArgs a, Plan plan) {
    __shared__ float mx[8], sums[8];
    __shared__ f32x4 red[8][8];
    const uint32_t b = blockIdx.z, head = blockIdx.y, H = a.mem.heads, G = a.q_heads / H, D = a.mem.dim, cuts = D / 32;
    Sequence s;
    if (!sequence_of(a, b, s)) return;
    const int64_t row = blockIdx.x / cuts, rows = (int64_t)s.n_new * G, rt = row / 16;
    if (row >= rows) return;
    int32_t lo, hi;
    range_of<SEL>(a, s, s.start + (int32_t)(rt * 16 / G), s.start + (int32_t)(min(rt * 16 + 15, rows - 1) / G), lo, hi);
    lo &= ~31;
    if (hi - lo <= (int32_t)plan.chunk) return;  // written by kv_attend
    const uint32_t used = min(((uint32_t)(hi - lo) + plan.chunk - 1) / plan.chunk, plan.splits);
    const uint64_t step = 16 * (D + 2);
    const float* part = plan.part + ((((uint64_t)b * H + head) * plan.tiles + rt) * plan.splits * 16 + row % 16) * (D + 2);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float best = kNone;
    for (uint32_t i = threadIdx.x; i < used; i += 512) best = __builtin_fmaxf(best, part[i * step + D]);
#pragma unroll
    for (int o = 32; o; o >>= 1) best = __builtin_fmaxf(best, __shfl_xor(best, o));
    if (lane == 0) mx[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) best = __builtin_fmaxf(best, mx[w]);
    const uint32_t g = threadIdx.x >> 3, d = blockIdx.x % cuts * 32 + (threadIdx.x & 7) * 4;
    f32x4 acc = {0, 0, 0, 0};
    float total = 0.0f;
    for (uint32_t i = g; i < used; i += 4 * 64) {
        f32x2 x[4], y[4], z[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float* w = part + (uint64_t)min(i + u * 64, used - 1) * step;
            x[u] = *(const f32x2*)(w + d), y[u] = *(const f32x2*)(w + d + 2), z[u] = *(const f32x2*)(w + D);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (i + u * 64 < used) {
                const float f = __builtin_amdgcn_exp2f(z[u][0] - best);
                total += f * z[u][1];
                acc += f32x4{x[u][0], x[u][1], y[u][0], y[u][1]} * f;
            }
        }
    }
#pragma unroll
    for (int o = 32; o >= 8; o >>= 1) {
        total += __shfl_xor(total, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o);
    }
    if (lane < 8) red[wave][lane] = acc;
    if (lane == 0) sums[wave] = total;
    __syncthreads();
    if (threadIdx.x < 8) {
        float sum = 0.0f;
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += sums[w], v += red[w][threadIdx.x];
        const int64_t ot = row / G;
        const uint64_t orow = (uint64_t)(s.first + ot) * a.q_heads + head * G + (uint32_t)(row - ot * G);
        const bool none = sum == 0.0f;
        const float inv = none ? 0.0f : 1.0f / sum;
        E<T>* out = (E<T>*)a.out + orow * D + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = (E<T>)(none ? 0.0f : v[i] * inv);
        if (a.lse && d == 0) a.lse[orow] = none ? -__builtin_inff() : (best + __builtin_amdgcn_logf(sum)) * kLn2;
    }
}

template <int T, int DS>
hipError_t launch_one(const KvAttendArgs& a, const Plan& plan, hipStream_t stream) {
    if (plan.many) {
        // blocks a head: as many as there can be items (fewer than 2^32 threads; the rest is walked)
        const uint64_t G = a.q_heads / a.mem.heads, rows = Many<T, DS>::rows, count = a.batch.count;
        const uint64_t items = (uint64_t)many_items(a.batch, (uint32_t)G, (uint32_t)rows);
        const uint64_t blocks = std::min<uint64_t>(count <= 64 ? std::min<uint64_t>(items, plan.max_new * count * G / rows + count) : items, (1u << 22) / a.mem.heads);
        hipLaunchKernelGGL((kv_attend_many<T, DS>), dim3((uint32_t)blocks * a.mem.heads), dim3(Many<T, DS>::kThreads), (Many<T, DS>::lds), stream, a);
        return hipGetLastError();
    }
    const dim3 grid(plan.tiles * plan.splits, a.mem.heads, a.batch.count);
    auto launch = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, grid, dim3(waves * 64), (Shape<T, DS>::lds(waves)), stream, a, plan); };
    if constexpr (T != kF32 || DS <= 5) {  // (f32 in more dimensions: 256 registers a lane are too few)
        if (plan.wide) {
            launch(kv_attend<T, DS, kSelected, 8>, 8);
            return hipGetLastError();
        }
    }
    if (a.select) launch(kv_attend<T, DS, kSelected, 4>, 4);
    else if (!a.batch.offsets) launch(kv_attend<T, DS, kSingle, 4>, 4);
    else launch(kv_attend<T, DS, kChunks, 4>, 4);
    return hipGetLastError();
}

template <int T, bool SEL>
void launch_join_of(const KvAttendArgs& a, const Plan& plan, const dim3& grid, hipStream_t stream) {
    // (a block of 256 threads a row: 6 ranges 6.9 us, a wave 5.2; 384 ranges 17, of 512 threads 9.7, cut into 32 dimensions 6.7; 32 of
    // them, with the attention: 25.3 us with 256 threads a row, 23.2)
    if (plan.splits <= 16) hipLaunchKernelGGL((kv_join_few<T, SEL>), dim3((grid.x + 3) / 4, grid.y, grid.z), dim3(256), 0, stream, a, plan);
    else hipLaunchKernelGGL((kv_join_long<T, SEL>), dim3(grid.x * (a.mem.dim / 32), grid.y, grid.z), dim3(512), 0, stream, a, plan);
}

template <int T>
hipError_t launch_join(const KvAttendArgs& a, const Plan& plan, uint32_t rows, hipStream_t stream) {  // rows: of one new token
    // (every row of a cut tile left partial results: with offsets a sequence may have more new tokens than the caller said)
    const dim3 grid(a.batch.offsets ? plan.tiles * 16 : rows, a.mem.heads, a.batch.count);
    if (a.select) launch_join_of<T, true>(a, plan, grid, stream);
    else launch_join_of<T, false>(a, plan, grid, stream);
    return hipGetLastError();
}

// How a launch is cut, from what the host knows (sizes only, so that the workspace asked for is the one used): the table's width (or the list's length, or the window) bounds the tokens.
Plan plan_of(const KvAttendArgs& a, uint32_t max_new) {
    const uint32_t G = a.q_heads / a.mem.heads;
    Plan p{};
    p.max_new = max_new;
    p.splits = 1;
    // Chunks that fill half of the chip at least with blocks of 128 rows, and whose rows fill them at least by half, are walked from
    // end to end (us, cut into ranges / walked, memories of 2000 tokens, 32 heads on 8, bf16, 128 dimensions: one chunk of 256 new
    // tokens 60 / 85, of 512 96 / 86, of 1024 100 / 89; 32 of 4 42 / 80, of 16 116 / 85; 100 of 8 132 / 238, of 32 488 / 270;
    // in f32 one of 256 80 / 84, of 512 133 / 87).
    const uint64_t rows = (uint64_t)max_new * G;
    p.many = !a.n_select && rows >= 64 && (rows + 127) / 128 * a.mem.heads * a.batch.count >= 128;
    if (p.many) return p;
    p.tiles = (uint32_t)std::min<uint64_t>(((uint64_t)max_new * G + 15) / 16, 65535);
    uint64_t tokens = a.n_select ? a.n_select : (uint64_t)a.batch.table_width << a.mem.page_shift;
    // (what a tile can see: the 16 rows may be as many tokens, whatever max_new says, and the first is rounded down to 32)
    if (!a.n_select && a.window) tokens = std::min<uint64_t>(tokens, (uint64_t)a.window + (a.batch.offsets ? 15 : 0) + 31);
    const uint64_t blocks = std::max<uint64_t>(1, (uint64_t)p.tiles * a.mem.heads * a.batch.count);
    // As many ranges as give some 12 blocks a CU, four times what the chip holds at once: sequences of different lengths even out
    // (64 of 1 000 to 8 192 tokens, 8 heads: 147 us at 4 a CU, 130 at 6, 121 at 12, 125 at 16).  But no range shorter than 512
    // tokens, where a block's start and end begin to count (500 tokens in one block 9.4 us, in four 6.0 and 4 for the join), and
    // at most 384 of one row, or the join counts (two sequences of 500 003: 384 ranges 103 us, 768 104, 256 109, and the join 6.7 at 384).
    // Selected tokens, whose rows and places take longer to come: where there are few rows, blocks of eight waves and ranges of
    // 2048, or 1024 if that leaves half of the chip idle (32 sequences x 8 heads x 2048 tokens in f32: 37 us in two ranges of
    // four waves and a join, 32 in one of eight; 1 x 8 x 2048 22.8, 24.4 in one range of eight, 19.0 in two; 64 x 8 x 2048 in bf16 76 and
    // 66, but 48 x 8 x 2048 49 and 57: one and a half rounds of blocks).
    const uint64_t want = std::min<uint64_t>(384, std::max<uint64_t>(1, 12 * 256 / blocks));
    p.wide = a.n_select && blocks <= 512;
    uint64_t chunk = std::max<uint64_t>(!a.n_select ? 512 : blocks >= 128 && p.wide ? 2048 : 1024, (tokens + want - 1) / want);
    chunk = (chunk + 127) / 128 * 128;
    p.chunk = (uint32_t)std::min<uint64_t>(chunk, 1u << 30);
    p.splits = (uint32_t)std::max<uint64_t>(1, (tokens + p.chunk - 1) / p.chunk);
    return p;
}

}  // namespace

#ifndef VDB_PART
#define VDB_PART 0
#endif
#define VDB_CAT2(a, b) a##b
#define VDB_CAT(a, b) VDB_CAT2(a, b)

// compiled once per element type (-DVDB_PART = vdb_dtype)
hipError_t VDB_CAT(kv_attend_launch_, VDB_PART)(const KvAttendArgs& a, uint32_t max_new, void* workspace, hipStream_t stream) {
    Plan plan = plan_of(a, max_new);
    plan.part = (float*)workspace;
    hipError_t e = hipErrorInvalidValue;
    switch (a.mem.dim / 32) {
        case 1: e = launch_one<VDB_PART, 1>(a, plan, stream); break;
        case 2: e = launch_one<VDB_PART, 2>(a, plan, stream); break;
        case 3: e = launch_one<VDB_PART, 3>(a, plan, stream); break;
        case 4: e = launch_one<VDB_PART, 4>(a, plan, stream); break;
        case 5: e = launch_one<VDB_PART, 5>(a, plan, stream); break;
        case 6: e = launch_one<VDB_PART, 6>(a, plan, stream); break;
        case 7: e = launch_one<VDB_PART, 7>(a, plan, stream); break;
        case 8: e = launch_one<VDB_PART, 8>(a, plan, stream); break;
    }
    if (e == hipSuccess && plan.splits > 1) e = launch_join<VDB_PART>(a, plan, a.q_heads / a.mem.heads, stream);
    return e;
}

#if VDB_PART == 0
hipError_t kv_attend_launch_1(const KvAttendArgs&, uint32_t, void*, hipStream_t);
hipError_t kv_attend_launch_2(const KvAttendArgs&, uint32_t, void*, hipStream_t);

size_t kv_attend_workspace_bytes(const KvAttendArgs& a, uint32_t max_new) {
    const Plan p = plan_of(a, max_new);
    return p.splits > 1 ? (size_t)a.batch.count * a.mem.heads * p.tiles * p.splits * 16 * (a.mem.dim + 2) * 4 : 0;
}

int launch_kv_attend(const KvAttendArgs& a, int dtype, uint32_t max_new, void* workspace, hipStream_t stream, std::string* err) {
    const hipError_t e = dtype == kF32 ? kv_attend_launch_0(a, max_new, workspace, stream)
                         : dtype == kF16 ? kv_attend_launch_1(a, max_new, workspace, stream)
                                         : kv_attend_launch_2(a, max_new, workspace, stream);
    if (e == hipSuccess) return 0;
    if (err) *err = std::string("kv_attend: ") + hipGetErrorString(e);
    return 3;
}
#endif

}  // namespace vdb
