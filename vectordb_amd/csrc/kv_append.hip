// kv_append.hip — new keys and values into the pages of an 8-bit memory, positions rotated on the way.
//
// A page holds P tokens of one head as e4m3 codes with one scale, a power of two.  New rows raise the scale if they must
// (smallest power of two under which the largest magnitude is at most 448, the largest code); the rows that the page held
// before are then re-expressed in it, which is exact but for codes that fall among the subnormals (below 2^-6).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "launch.hpp"
#include "lowbits.hpp"

namespace vdb {

namespace {

template <int T>
using E = typename Elem<T>::type;

// 8 consecutive elements, 16-byte aligned (f32: two loads)
template <int T>
__device__ __forceinline__ void load8(const E<T>* p, float v[8]) {
    if constexpr (T == kF32) {
        const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
        typedef __attribute__((ext_vector_type(8))) E<T> vec;
        const vec a = *(const vec*)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32((E<T>)a[i]);
    }
}

template <int T>
__device__ __forceinline__ void store8(E<T>* p, const float v[8]) {
    if constexpr (T == kF32) {
        *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        typedef __attribute__((ext_vector_type(8))) E<T> vec;
        vec a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (E<T>)v[i];
        *(vec*)p = a;
    }
}

// A head's row is cut into units that turn by themselves: 8 dimensions and the 8 that pair with them (rot / 16 units), or 8
// neighbours where pairs are neighbours (rot / 8), and then the 8 dimensions at a time that do not turn.
struct Units {
    uint32_t turning, count, half;  // half: distance of a pair's members, 0: neighbours (or nothing turns)
};

template <bool NEXT>  // pairs are neighbours
__device__ __forceinline__ Units units_of(uint32_t dim, uint32_t rot) {
    Units u;
    u.half = NEXT ? 0 : rot / 2;
    u.turning = NEXT ? rot / 8 : rot / 16;
    u.count = u.turning + (dim - rot) / 8;
    return u;
}

// First dimension of unit u; a second piece of 8 lies n.half behind it if it turns.
__device__ __forceinline__ uint32_t unit_start(const Units& n, uint32_t u, uint32_t rot) {
    return u < n.turning ? u * 8 : rot + (u - n.turning) * 8;
}

// (a, b) -> (a cos - b sin, b cos + a sin), each operation rounded; cs, sn: the angles of the unit's position.
template <bool NEXT>
__device__ __forceinline__ void load_turn(const float* cs, const float* sn, uint32_t u, float c[8], float s[8]) {
    if constexpr (NEXT) {
        const f32x4 x = *(const f32x4*)(cs + u * 4), y = *(const f32x4*)(sn + u * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = x[i], s[i] = y[i], c[4 + i] = s[4 + i] = 0.0f;
    } else {
        load8<kF32>(cs + u * 8, c);
        load8<kF32>(sn + u * 8, s);
    }
}

template <bool NEXT>
__device__ __forceinline__ void turn_unit(const float c[8], const float s[8], float a[8], float b[8]) {
    if constexpr (NEXT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = a[2 * i], y = a[2 * i + 1];
            a[2 * i] = x * c[i] - y * s[i];
            a[2 * i + 1] = y * c[i] + x * s[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * c[i] - y * s[i];
            b[i] = y * c[i] + x * s[i];
        }
    }
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

__device__ __forceinline__ void unpack_e4m3(uint32_t w, float v[4]) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
}

// The smallest power of two s with top <= 448 s (448 = 0.875 * 2^9); never below 2^-100.
__device__ __forceinline__ float scale_for(uint32_t top_bits) {
    int ex;
    const float top = float_of(top_bits), f = frexpf(top, &ex);
    ex = max(top > 0.0f ? ex - (f <= 0.875f ? 9 : 8) : -100, -100);
    return float_of((uint32_t)(ex + 127) << 23);
}

struct Span {
    int64_t first;  // row of the new tokens' arrays that holds the sequence's first new token
    int64_t start, end;  // positions start .. end - 1 are new
};

__device__ __forceinline__ Span span_of(const KvBatch& t, uint32_t b) {
    Span s;
    s.first = t.offsets ? t.offsets[b] : b;
    const int64_t n = t.offsets ? (int64_t)t.offsets[b + 1] - s.first : 1;
    s.end = t.lengths[b];
    s.start = s.end - n;
    // offsets beyond the arrays hold nothing that may be read
    if (n <= 0 || s.first < 0 || s.first + n > (int64_t)t.tokens) s.end = s.start;
    return s;
}

template <int NT>
__device__ __forceinline__ uint32_t block_max(uint32_t x, uint32_t* red) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = max(x, (uint32_t)__shfl_xor(x, o));
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) x = max(x, red[w]);
        __syncthreads();
    }
    return x;
}

__device__ __forceinline__ uint32_t top_of(uint32_t top, const float v[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, bits_of(v[i]) & 0x7FFFFFFFu);
    return top;
}

// The same over finite values only.
__device__ __forceinline__ uint32_t finite_top_of(uint32_t top, const float v[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t m = bits_of(v[i]) & 0x7FFFFFFFu;
        top = m < 0x7F800000u ? max(top, m) : top;
    }
    return top;
}

// 8 values over the scale, rounded (an infinity, like a NaN, becomes NaN: e4m3 has none).
__device__ __forceinline__ void store_codes(uint8_t* p, const float v[8], float scale, float inverse, bool exact) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = exact ? v[i] * inverse : v[i] / scale;
    *(u32x2*)p = u32x2{pack_e4m3(x[0], x[1], x[2], x[3]), pack_e4m3(x[4], x[5], x[6], x[7])};
}

// The new rows of one page and head (keys or values).  One block owns a page of a head, so nothing is shared and no order of
// atomics enters the result.  Rows that fit the block's registers (8 pieces of 8 numbers a thread: 128 tokens of 128 dimensions)
// are read once, all loads under way together (no branch between them: places past the end read the last one again); longer
// ones are read a second time for their codes.
template <int T, int NT, int NP8, bool NEXT, bool TURN>
__device__ __forceinline__ void store_page(const KvAppendArgs& a, const E<T>* src, uint64_t token_stride, int64_t at0, uint32_t r0, uint32_t r1,
                                           uint8_t* page, float* scale, uint32_t* red) {
    constexpr bool PAIR = TURN && !NEXT;
    constexpr int NP = PAIR ? 2 : 1, NU = (NP8 + NP - 1) / NP;
    const uint32_t D = a.mem.dim, rot = TURN ? a.rot : 0;
    const Units n = units_of<NEXT>(D, rot);
    const uint32_t total = (r1 - r0) * n.count;
    // unit i of the page: its row and first dimension
    auto place = [&](uint32_t i, uint32_t& r, uint32_t& u, uint32_t& d, bool& pair) {
        r = r0 + i / n.count;
        u = i % n.count;
        d = unit_start(n, u, rot);
        pair = PAIR && u < n.turning;
    };
    auto load = [&](uint32_t i, float v[NP][8]) {
        uint32_t r, u, d;
        bool pair;
        place(i, r, u, d, pair);
        const E<T>* row = src + (uint64_t)(r - r0) * token_stride + d;
        load8<T>(row, v[0]);
        if constexpr (PAIR) load8<T>(row + (pair ? n.half : 0), v[NP - 1]);
    };
    auto turn = [&](uint32_t i, float v[NP][8]) {
        if constexpr (TURN) {
            uint32_t r, u, d;
            bool pair;
            place(i, r, u, d, pair);
            float c[8], s[8];
            const int64_t at = (at0 + r) * (rot / 2);
            load_turn<NEXT>(a.cos + at, a.sin + at, u < n.turning ? u : 0, c, s);
#pragma unroll
            for (int k = 0; k < 8; ++k) c[k] = u < n.turning ? c[k] : 1.0f, s[k] = u < n.turning ? s[k] : 0.0f;
            // (x * 1 - y * 0 is x, also for an infinite y's sake: a number that does not turn is kept as it was)
            float x[8], y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = v[0][k], y[k] = v[NP - 1][k];
            turn_unit<NEXT>(c, s, x, y);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[0][k] = u < n.turning ? x[k] : v[0][k];
                if constexpr (PAIR) v[NP - 1][k] = u < n.turning ? y[k] : v[NP - 1][k];
            }
        }
    };
    auto store = [&](uint32_t i, const float v[NP][8], float now, float inverse, bool exact) {
        uint32_t r, u, d;
        bool pair;
        place(i, r, u, d, pair);
        store_codes(page + (uint64_t)r * D + d, v[0], now, inverse, exact);
        if (pair) store_codes(page + (uint64_t)r * D + d + n.half, v[NP - 1], now, inverse, exact);
    };
    float v[NU][NP][8];
    const bool resident = total <= NU * NT;
    uint32_t top = 0;
    const float was = *scale;
    if (resident) {
#pragma unroll
        for (int k = 0; k < NU; ++k) load(min(threadIdx.x + k * NT, total - 1), v[k]);
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            turn(min(threadIdx.x + k * NT, total - 1), v[k]);
#pragma unroll
            for (int p = 0; p < NP; ++p) top = top_of(top, v[k][p]);
        }
    } else {
        for (uint32_t i = threadIdx.x; i < total; i += NT) {
            load(i, v[0]);
            turn(i, v[0]);
#pragma unroll
            for (int p = 0; p < NP; ++p) top = top_of(top, v[0][p]);
        }
    }
    top = block_max<NT>(top, red);
    if (top >= 0x7F800000u) {  // infinities or NaN among them: once more without
        top = 0;
        for (uint32_t i = threadIdx.x; i < total; i += NT) {
            float x[NP][8];
            load(i, x);
            turn(i, x);
#pragma unroll
            for (int p = 0; p < NP; ++p) top = finite_top_of(top, x[p]);
        }
        top = block_max<NT>(top, red);
    }
    float now = scale_for(top);
    if (r0 && was > now) now = was;
    if (r0 && now != was) {
        const float f = was / now;
        for (uint32_t i = threadIdx.x; i < r0 * D / 16; i += NT) {
            u32x4 w = *((u32x4*)page + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float x[4];
                unpack_e4m3(w[k], x);
                w[k] = pack_e4m3(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
            }
            *((u32x4*)page + i) = w;
        }
    }
    const bool exact = (bits_of(now) & 0x007FFFFFu) == 0;  // a power of two: its inverse is one (a scale set by hand need not be)
    const float inverse = 1.0f / now;
    if (resident) {
#pragma unroll
        for (int k = 0; k < NU; ++k)
            if (threadIdx.x + k * NT < total) store(threadIdx.x + k * NT, v[k], now, inverse, exact);
    } else {
        for (uint32_t i = threadIdx.x; i < total; i += NT) {
            load(i, v[0]);
            turn(i, v[0]);
            store(i, v[0], now, inverse, exact);
        }
    }
    if (threadIdx.x == 0 && now != was) *scale = now;
}

// The queries of new tokens, turned: a wave takes a token, holds its angles and goes through the heads.
template <int T, bool NEXT>
__device__ __forceinline__ void turn_queries(const KvAppendArgs& a, uint64_t wave, uint64_t waves) {
    const int lane = threadIdx.x & 63;
    const uint32_t D = a.mem.dim;
    const Units n = units_of<NEXT>(D, a.rot);
    const uint32_t side_by_side = 64 / n.count, first = lane / n.count, u = lane % n.count;
    const uint32_t d = unit_start(n, u, a.rot);
    const bool pair = n.half != 0 && u < n.turning;
    if (first >= side_by_side) return;
    for (uint64_t t = wave; t < a.batch.tokens; t += waves) {
        uint32_t b = (uint32_t)t;
        if (a.batch.offsets) {  // the last sequence that begins at or before t
            uint32_t lo = 0, hi = a.batch.count;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (a.batch.offsets[mid] <= (int64_t)t) lo = mid;
                else hi = mid;
            }
            b = lo;
        }
        const Span s = span_of(a.batch, b);
        const int64_t at = s.start + (int64_t)t - s.first;
        const bool any = (int64_t)t >= s.first && at < s.end;  // a row of no sequence is copied
        const bool known = any && at >= 0 && at < (int64_t)a.positions;
        float c[8] = {}, s8[8] = {};  // (of unit 0 where nothing turns; a position that the tables lack has none, and they may have no rows)
        if (known) load_turn<NEXT>(a.cos + at * (a.rot / 2), a.sin + at * (a.rot / 2), u < n.turning ? u : 0, c, s8);
        const E<T>* q = (const E<T>*)a.q + t * a.q_token + d;
        E<T>* out = (E<T>*)a.q_out + t * a.q_heads * D + d;
#pragma unroll 4
        for (uint32_t h = first; h < a.q_heads; h += side_by_side) {
            float x[8], y[8];
            load8<T>(q + (uint64_t)h * a.q_head, x);
            load8<T>(q + (uint64_t)h * a.q_head + (pair ? n.half : 0), y);
            if (known && u < n.turning) turn_unit<NEXT>(c, s8, x, y);
            if (any && !known) {  // no such position: not a number, so that it shows
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = y[i] = float_of(0x7FC00000u);
            }
            store8<T>(out + (uint64_t)h * D, x);
            if (pair) store8<T>(out + (uint64_t)h * D + n.half, y);
        }
    }
}

template <int T, bool NEXT>
__global__ __launch_bounds__(256) void kv_turn(KvAppendArgs a) {
    turn_queries<T, NEXT>(a, blockIdx.x * 4ull + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), gridDim.x * 4ull);
}

// Queries of a call without sequences: copied.  (The test for it in turn_queries cost kv_append up to 19 registers, and spills.)
template <int T>
__global__ __launch_bounds__(256) void kv_copy(KvAppendArgs a) {
    const uint32_t D8 = a.mem.dim / 8;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < a.batch.tokens * a.q_heads * D8; i += gridDim.x * 256ull) {
        const uint64_t row = i / D8, t = row / a.q_heads;
        float x[8];
        load8<T>((const E<T>*)a.q + t * a.q_token + (row - t * a.q_heads) * a.q_head + i % D8 * 8, x);
        store8<T>((E<T>*)a.q_out + i * 8, x);
    }
}

enum { kBoth = 0, kKeys = 1, kValues = 2 };  // sides that a launch stores (kKeys: turned)

// Slots of pages, where a launch has as many for all sequences as their rows can need: those of sequence b begin here.  (n tokens
// touch n / P + 2 pages at most, which is no more than what lies between two of these.)
__device__ __forceinline__ uint32_t slot_base(const KvBatch& t, uint32_t b, uint32_t page_shift) { return ((uint32_t)max(t.offsets[b], 0) >> page_shift) + 2 * b; }

// One launch for all: a sequence has blocks of (slot, side and head), a slot being one of the pages that its new tokens touch, or
// several; the blocks from store_blocks on turn queries, of whatever sequence.  With SHARED the slots are those of all sequences
// together, and a block looks up whose its own is.
template <int T, int NT, int NP8, bool NEXT, int SIDES, bool SHARED>
__global__ __launch_bounds__(NT, SIDES == kValues ? 6 : 4) void kv_append(KvAppendArgs a, uint32_t slots, uint32_t store_blocks) {
    __shared__ uint32_t red[NT / 64];
    if (blockIdx.x >= store_blocks) {
        const uint64_t per = NT / 64;
        turn_queries<T, NEXT>(a, (blockIdx.x - store_blocks) * per + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), (gridDim.x - store_blocks) * per);
        return;
    }
    const uint32_t sides = (SIDES == kBoth ? 2 : 1) * a.mem.heads, rest = blockIdx.x / slots;
    uint32_t slot = blockIdx.x % slots, step = slots, b = rest / sides;
    const uint32_t head = (rest % sides) >> (SIDES == kBoth);
    const bool is_v = SIDES == kBoth ? rest % sides & 1 : SIDES == kValues;
    if constexpr (SHARED) {
        uint32_t lo = 0, hi = a.batch.count;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (slot_base(a.batch, mid, a.mem.page_shift) <= slot) lo = mid;
            else hi = mid;
        }
        const uint32_t base = slot_base(a.batch, lo, a.mem.page_shift);
        if (slot < base) return;
        b = lo, slot -= base, step = slot_base(a.batch, lo + 1, a.mem.page_shift) - base;
    }
    const Span s = span_of(a.batch, b);
    if (s.end <= s.start) return;
    const uint32_t P = a.mem.page_tokens, D = a.mem.dim;
    const int64_t begin = s.start < 0 ? 0 : s.start;
    const E<T>* src = (const E<T>*)(is_v ? a.v : a.k) + (uint64_t)head * (is_v ? a.v_head : a.k_head);
    const uint64_t token_stride = is_v ? a.v_token : a.k_token;
    const bool turn = !is_v && a.rot != 0;
    for (int64_t p = (begin >> a.mem.page_shift) + slot; p * P < s.end && p < (int64_t)a.batch.table_width; p += step) {
        const int32_t pid = a.batch.table[(uint64_t)b * a.batch.table_width + p];
        if (pid < 0 || (uint64_t)pid >= a.mem.pages) continue;
        const uint32_t r0 = p * P < begin ? (uint32_t)(begin - p * P) : 0;
        uint32_t r1 = s.end - p * P < P ? (uint32_t)(s.end - p * P) : P;
        if (turn) {  // a position without a row in the tables is not stored
            const int64_t known = (int64_t)a.positions - p * P;
            if (known < (int64_t)r1) r1 = known > (int64_t)r0 ? (uint32_t)known : r0;
        }
        if (r1 <= r0) continue;
        uint8_t* page = (uint8_t*)(is_v ? a.mem.v : a.mem.k) + ((uint64_t)pid * a.mem.heads + head) * P * D;
        float* scale = (is_v ? a.mem.v_scale : a.mem.k_scale) + (uint64_t)pid * a.mem.heads + head;
        const E<T>* rows = src + (uint64_t)(s.first + p * P + r0 - s.start) * token_stride;
        if constexpr (SIDES != kValues) {
            if (turn) {
                store_page<T, NT, NP8, NEXT, true>(a, rows, token_stride, p * P, r0, r1, page, scale, red);
                continue;
            }
        }
        if constexpr (SIDES != kKeys) store_page<T, NT, NP8, NEXT, false>(a, rows, token_stride, p * P, r0, r1, page, scale, red);
    }
}

}  // namespace

int launch_kv_append(const KvAppendArgs& a, int dtype, uint32_t max_new, hipStream_t stream, std::string* err) {
    // A sequence's max_new tokens touch at most this many pages; more of them (a wrong max_new) are walked by the same blocks.
    const uint64_t P = a.mem.page_tokens, sides = 2ull * a.mem.heads, count = a.batch.count, total = a.batch.tokens / P + 2 * count;
    const uint64_t each = std::min<uint64_t>(a.batch.table_width, ((uint64_t)max_new + 2 * P - 2) / P), most = (1u << 22) / sides;  // (fewer than 2^32 threads)
    // Where that is more than twice what all rows together can need, blocks look for their sequences (a block without work costs
    // 5 ns: a prompt of 9000 tokens beside 299 of 3, 8 heads of 128, pages of 64: 2.4 -> 0.10 ms;
    // a thousand of 4, without max_new, 5.1 -> 0.25).
    const bool shared = a.batch.offsets && each * count > 2 * total && total <= most;
    const uint32_t slots = (uint32_t)(shared ? total : std::max<uint64_t>(1, std::min(each, most / std::max<uint64_t>(count, 1))));
    const uint64_t store_blocks = slots * sides * (shared ? 1 : count);
    // By the pieces of 8 numbers that a page can get: a wave with one each (a step of decoding), a wave with four, eight waves
    // with four (8 x 8192 tokens, pages of 128 x 128: 142 us; four waves with eight pieces 152, sixteen with two 209; read
    // twice instead of held 164).  Where there are many pages, values, which do not turn, have a launch of their own with fewer
    // registers and so more of them under way (143 us -> 80 + 51; with 64 registers, spilled, 74).
    const uint64_t pieces = (uint64_t)std::min(max_new, a.mem.page_tokens) * a.mem.dim / 8;
    if (store_blocks > 0xFFFFFFFFu / (pieces <= 256 ? 64 : 512) - 65536) {
        if (err) *err = "kv_append: too many sequences times heads in one call";
        return 1;
    }
    auto go = [&](auto t) {
        constexpr int T = decltype(t)::value;
        auto launch = [&](auto next, auto is_shared) {
            constexpr bool NEXT = decltype(next)::value, SHARED = decltype(is_shared)::value;
            // Few queries go along with the keys and values, in one launch (64 tokens: 5.0 us instead of 5.4 + 3.2; 5 x 700: 15.7 instead of 15.2 + 6.9); many have
            // one of their own, with a third of the registers and so more loads on their way (8 x 8192 tokens: 436 -> 327 us).
            const bool along = a.q && a.batch.tokens * a.q_heads <= 65536;
            auto store = [&](auto kernel, uint32_t threads, uint64_t stores, bool turning) {
                const uint64_t per = threads / 64, blocks = stores + (turning ? (a.batch.tokens + per - 1) / per : 0);
                hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(threads), 0, stream, a, slots, (uint32_t)stores);
            };
            if (pieces <= 64) {
                store(kv_append<T, 64, 1, NEXT, kBoth, SHARED>, 64, store_blocks, along);
            } else if (pieces <= 256) {
                store(kv_append<T, 64, 4, NEXT, kBoth, SHARED>, 64, store_blocks, along);
            } else if (a.rot && store_blocks >= 4096) {
                store(kv_append<T, 512, 4, NEXT, kKeys, SHARED>, 512, store_blocks / 2, along);
                store(kv_append<T, 512, 4, NEXT, kValues, SHARED>, 512, store_blocks / 2, false);
            } else {
                store(kv_append<T, 512, 4, NEXT, kBoth, SHARED>, 512, store_blocks, along);
            }
            if (a.q && !along)
                hipLaunchKernelGGL((kv_turn<T, NEXT>), dim3((uint32_t)std::min<uint64_t>((a.batch.tokens + 3) / 4, 8192)), dim3(256), 0, stream, a);
        };
        if (!count) {
            hipLaunchKernelGGL(kv_copy<T>, dim3((uint32_t)std::min<uint64_t>((a.batch.tokens * a.q_heads * (a.mem.dim / 8) + 255) / 256, 8192)), dim3(256), 0, stream, a);
        } else if (a.interleaved) {
            if (shared) launch(std::true_type(), std::true_type());
            else launch(std::true_type(), std::false_type());
        } else {
            if (shared) launch(std::false_type(), std::true_type());
            else launch(std::false_type(), std::false_type());
        }
    };
    if (dtype == kF32) go(std::integral_constant<int, kF32>());
    else if (dtype == kF16) go(std::integral_constant<int, kF16>());
    else go(std::integral_constant<int, kBF16>());
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    if (err) *err = std::string("kv_append: ") + hipGetErrorString(e);
    return 3;
}

}  // namespace vdb
