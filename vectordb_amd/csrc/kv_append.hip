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

// Dimensions d0 .. d0 + 7 of a head's row, rotated by the tables' row of its position: the pair (a, b) becomes
// (a cos - b sin, b cos + a sin), three f32 roundings each.  Pairs are (d, d + rot / 2), or (2 i, 2 i + 1) if interleaved.
template <int T>
__device__ __forceinline__ void load_rotated(const E<T>* row, uint32_t d0, const float* cs, const float* sn, uint32_t rot, bool interleaved, float v[8]) {
    load8<T>(row + d0, v);
    if (d0 >= rot) return;
    if (interleaved) {
        const f32x4 c = *(const f32x4*)(cs + d0 / 2), s = *(const f32x4*)(sn + d0 / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[2 * i], b = v[2 * i + 1];
            v[2 * i] = a * c[i] - b * s[i];
            v[2 * i + 1] = b * c[i] + a * s[i];
        }
        return;
    }
    const uint32_t half = rot / 2;
    const bool first = d0 < half;
    float o[8], c[8], s[8];
    load8<T>(row + (first ? d0 + half : d0 - half), o);
    load8<kF32>(cs + (first ? d0 : d0 - half), c);
    load8<kF32>(sn + (first ? d0 : d0 - half), s);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = first ? v[i] * c[i] - o[i] * s[i] : v[i] * c[i] + o[i] * s[i];
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

__device__ __forceinline__ void unpack_e4m3(uint32_t w, float v[4]) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
}

// A NaN or an infinity has no code but NaN: both become NaN.
__device__ __forceinline__ float finite_or_nan(float x) { return (bits_of(x) & 0x7F800000u) == 0x7F800000u ? float_of(0x7FC00000u) : x; }

// The smallest power of two s with top <= 448 s (448 = 0.875 * 2^9); never below 2^-100.
__device__ __forceinline__ float scale_for(float top) {
    int ex;
    const float f = frexpf(top, &ex);
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

// Block (slot, side and head, sequence): the pages that the sequence's new tokens touch, slot by slot.  One block owns a page
// of a head, so nothing is shared and no order of atomics enters the result.
template <int T>
__global__ __launch_bounds__(256) void kv_store(KvAppendArgs a) {
    __shared__ float red[4];
    const uint32_t b = blockIdx.z, head = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const Span s = span_of(a.batch, b);
    if (s.end <= s.start) return;
    const uint32_t P = a.mem.page_tokens, D = a.mem.dim, chunks = D / 8;
    const int64_t begin = s.start < 0 ? 0 : s.start;
    const E<T>* src = (const E<T>*)(is_v ? a.v : a.k) + (uint64_t)head * (is_v ? a.v_head : a.k_head);
    const uint64_t token_stride = is_v ? a.v_token : a.k_token;
    const bool turn = !is_v && a.rot != 0;
    for (int64_t p = (begin >> a.mem.page_shift) + blockIdx.x; p * P < s.end && p < (int64_t)a.batch.table_width; p += gridDim.x) {
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
        auto fetch = [&](uint32_t r, uint32_t c, float v[8]) {
            const int64_t at = p * P + r;
            const E<T>* row = src + (uint64_t)(s.first + at - s.start) * token_stride;
            if (turn) load_rotated<T>(row, c * 8, a.cos + at * (a.rot / 2), a.sin + at * (a.rot / 2), a.rot, a.interleaved, v);
            else load8<T>(row + c * 8, v);
        };
        float top = 0.0f;
        for (uint32_t i = threadIdx.x; i < (r1 - r0) * chunks; i += 256) {
            float v[8];
            fetch(r0 + i / chunks, i % chunks, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float m = fabsf(finite_or_nan(v[j]));
                top = m > top ? m : top;
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
        const float was = *scale;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        float now = scale_for(top);
        if (r0 && was > now) now = was;
        if (r0 && now != was) {
            const float f = was / now;
            for (uint32_t i = threadIdx.x; i < r0 * D / 4; i += 256) {
                uint32_t* w = (uint32_t*)page + i;
                float v[4];
                unpack_e4m3(*w, v);
                *w = pack_e4m3(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
            }
        }
        for (uint32_t i = threadIdx.x; i < (r1 - r0) * chunks; i += 256) {
            const uint32_t r = r0 + i / chunks, c = i % chunks;
            float v[8];
            fetch(r, c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = finite_or_nan(v[j]) / now;
            *(u32x2*)(page + (uint64_t)r * D + c * 8) = u32x2{pack_e4m3(v[0], v[1], v[2], v[3]), pack_e4m3(v[4], v[5], v[6], v[7])};
        }
        if (threadIdx.x == 0 && now != was) *scale = now;
        __syncthreads();  // red is free again
    }
}

// The queries of the new tokens, rotated: one thread per 8 dimensions.
template <int T>
__global__ __launch_bounds__(256) void kv_rotate_queries(KvAppendArgs a) {
    const uint32_t chunks = a.mem.dim / 8;
    const uint64_t total = (uint64_t)a.batch.tokens * a.q_heads * chunks;
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256u) {
        const uint32_t c = (uint32_t)(i % chunks);
        const uint64_t th = i / chunks;
        const uint32_t h = (uint32_t)(th % a.q_heads);
        const int64_t t = (int64_t)(th / a.q_heads);
        uint32_t b = (uint32_t)t;
        if (a.batch.offsets) {  // the last sequence that begins at or before t
            uint32_t lo = 0, hi = a.batch.count;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (a.batch.offsets[mid] <= t) lo = mid;
                else hi = mid;
            }
            b = lo;
        }
        const Span s = span_of(a.batch, b);
        const int64_t at = s.start + t - s.first;
        const bool any = t >= s.first && at < s.end;  // a row of no sequence is copied
        const bool known = at >= 0 && at < (int64_t)a.positions;
        float v[8];
        const E<T>* row = (const E<T>*)a.q + (uint64_t)t * a.q_token + (uint64_t)h * a.q_head;
        if (any && known) {
            load_rotated<T>(row, c * 8, a.cos + at * (a.rot / 2), a.sin + at * (a.rot / 2), a.rot, a.interleaved, v);
        } else if (any) {  // no such position: not a number, so that it shows
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = float_of(0x7FC00000u);
        } else {
            load8<T>(row + c * 8, v);
        }
        store8<T>((E<T>*)a.q_out + i * 8, v);
    }
}

}  // namespace

int launch_kv_append(const KvAppendArgs& a, int dtype, uint32_t max_new, hipStream_t stream, std::string* err) {
    // a sequence's max_new tokens touch at most this many pages; more of them (a wrong max_new) are walked by the same blocks
    const uint32_t slots = std::min<uint32_t>(a.batch.table_width, (max_new + 2 * a.mem.page_tokens - 2) / a.mem.page_tokens);
    auto go = [&](auto t) {
        constexpr int T = decltype(t)::value;
        hipLaunchKernelGGL((kv_store<T>), dim3(slots, 2 * a.mem.heads, a.batch.count), dim3(256), 0, stream, a);
        if (a.q) {
            const uint64_t total = (uint64_t)a.batch.tokens * a.q_heads * (a.mem.dim / 8);
            hipLaunchKernelGGL((kv_rotate_queries<T>), dim3((uint32_t)std::min<uint64_t>((total + 255) / 256, 1u << 16)), dim3(256), 0, stream, a);
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
