// The paged key/value cache: new keys and values into their slots, as 16-bit values or as 8-bit codes with a scale
// for each (token, head), and back.
//
// scale = largest |x| of the row / the largest code (127, or 448 for 8-bit floats), code = x * largest code / largest
// |x|, rounded to nearest even.  The quotient is the correctly rounded one: with y = 1 / b rounded, one correction
// q + fma(-q, b, a) * y of q = a * y gives the rounded a / b, so that exact ties between two codes are seen as ties.
// Bound by memory: a lane moves 8 or 16 elements in 16-byte accesses, a row takes neighbouring lanes, and the keys' and
// values' rows of a (token, head) go together, so that every lane has two to four loads in flight.  Measured: 65536 tokens of
// 32 heads of 128 dims from bf16 into int8 300 us and back 293, 5.4 and 5.6 TB/s (a copy of large tensors: 4.9); 2047
// tokens of 64 heads of 96 dims from fp16 into fp8 16 and back 13.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_kernels.hpp"

namespace neox {

struct CacheArgs {
    char *k, *v;                      // rows outside the cache, 16-bit
    char *kc, *vc;                    // the cache
    float *ks, *vs;                   // its scales (4 bits: bytes)
    const void* slots;
    int64_t k_st[2], v_st[2];         // token, head
    int64_t kc_st[3], vc_st[3], ks_st[3], vs_st[3];  // token within a page, page, head
    int64_t slot_count;               // slots of the cache; page = slot / page size
    int64_t rows;                     // tokens * heads
    int heads, d, page;
    FastDiv by_heads, by_page;
    bool wide;                        // 64-bit slots
};

// One row's share of a lane (16 elements in two words of 8) as codes; *scale gets the row's.
template <typename T, int SRC, int G>
__device__ __forceinline__ u32x4 encode16(const u32x4 (&w)[2], float* scale) {
    constexpr float kTop = SRC == kPagedI8 ? 127.f : 448.f;
    // the largest magnitude, on the bits: an infinity is larger than every number, a NaN larger still
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[h][i] & 0x7fffu, (w[h][i] >> 16) & 0x7fffu));
    top = group_largest<G>(top);
    float b, unused;
    Elem<T>::unpack(top, b, unused);
    const bool finite = b < __builtin_inff();
    *scale = finite ? b / kTop : __builtin_nanf("");
    // values whose product with the largest code or whose reciprocal would leave the range are moved into it
    const float shift = b > 0x1p100f ? 0x1p-100f : b < 0x1p-100f ? 0x1p100f : 1.f;
    b *= shift;
    const float y = b > 0.f ? 1.f / b : 0.f;
    u32x4 out;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float x[8];
        unpack8<T>(w[h], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = x[i] * (shift * kTop);
            const float q = a * y;
            x[i] = __builtin_fmaf(__builtin_fmaf(-q, b, a), y, q);
        }
        if constexpr (SRC == kPagedI8) {
            // 1.5 * 2^23 more rounds to a whole number, whose low byte is the code
            uint32_t code[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) code[i] = __builtin_bit_cast(uint32_t, x[i] + 12582912.f);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t lo = __builtin_amdgcn_perm(code[4 * i + 1], code[4 * i], 0x0c0c0400);
                out[2 * h + i] = lo | __builtin_amdgcn_perm(code[4 * i + 3], code[4 * i + 2], 0x04000c0c);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
                out[2 * h + i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], c, true);
            }
        }
    }
    return finite ? out : u32x4{0, 0, 0, 0};
}

template <typename T, int SRC>
__device__ __forceinline__ u32x4 scaled8(const u32x2& c, float scale) {
    float f[8];
    decode8<SRC>(c, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= scale;
    return pack8<T>(f);
}

// Elements of a lane: 16 where codes are made, so that their stores have 16 bytes too (65536 tokens of 32 heads of 128
// dims in int8: 426 us with 8, 306 with 16); 8 otherwise, so that the 16-bit side is dense (reading them back: 306, 342).
template <int SRC, bool WRITE>
__host__ __device__ constexpr int cache_elems() { return SRC != kPaged16 && WRITE ? 16 : 8; }

// G: lanes of a row, a power of two.
template <typename T, int SRC, int G, bool WRITE>
__global__ __launch_bounds__(256) void cache_kernel(CacheArgs a) {
    constexpr bool kCodes = SRC != kPaged16;
    constexpr int kElems = cache_elems<SRC, WRITE>(), kBytes = kCodes ? 1 : 2;
    const uint32_t row = (uint32_t)(((uint64_t)blockIdx.x * 256 + threadIdx.x) / G);  // (below 2^30 + 256)
    const int part = threadIdx.x % G;
    const bool mine = row < (uint32_t)a.rows && part * kElems < a.d;
    const uint32_t token = a.by_heads.div(min(row, (uint32_t)a.rows - 1)), head = min(row, (uint32_t)a.rows - 1) - token * a.heads;
    const int64_t slot = a.wide ? static_cast<const int64_t*>(a.slots)[token] : static_cast<const int32_t*>(a.slots)[token];
    const bool held = slot >= 0 && slot < a.slot_count;
    // (page numbers and slots of a page are below 2^30, slots themselves may not be)
    const int64_t page = held ? (a.slot_count <= 0x7fffffff ? (int64_t)a.by_page.div((uint32_t)slot) : slot / a.page) : 0;
    const int64_t in = held ? slot - page * a.page : 0;
    char* const kp = a.k + (token * a.k_st[0] + head * a.k_st[1] + part * kElems) * 2;
    char* const vp = a.v + (token * a.v_st[0] + head * a.v_st[1] + part * kElems) * 2;
    char* const kc = a.kc + (in * a.kc_st[0] + page * a.kc_st[1] + head * a.kc_st[2] + part * kElems) * kBytes;
    char* const vc = a.vc + (in * a.vc_st[0] + page * a.vc_st[1] + head * a.vc_st[2] + part * kElems) * kBytes;
    u32x4 none = {0, 0, 0, 0};
    if constexpr (!kCodes) {
        if (!mine) return;
        if constexpr (WRITE) {
            if (!held) return;
            const u32x4 k = *reinterpret_cast<const u32x4*>(kp), v = *reinterpret_cast<const u32x4*>(vp);
            *reinterpret_cast<u32x4*>(kc) = k;
            *reinterpret_cast<u32x4*>(vc) = v;
        } else {
            const u32x4 k = load8(kc, held), v = load8(vc, held);
            *reinterpret_cast<u32x4*>(kp) = k;
            *reinterpret_cast<u32x4*>(vp) = v;
        }
    } else {
        float* const ks = a.ks + in * a.ks_st[0] + page * a.ks_st[1] + head * a.ks_st[2];
        float* const vs = a.vs + in * a.vs_st[0] + page * a.vs_st[1] + head * a.vs_st[2];
        if constexpr (WRITE) {
            u32x4 k[2] = {none, none}, v[2] = {none, none};
            if (mine) {
                k[0] = *reinterpret_cast<const u32x4*>(kp);
                k[1] = *reinterpret_cast<const u32x4*>(kp + 16);
                v[0] = *reinterpret_cast<const u32x4*>(vp);
                v[1] = *reinterpret_cast<const u32x4*>(vp + 16);
            }
            float k_scale, v_scale;
            const u32x4 x = encode16<T, SRC, G>(k, &k_scale), y = encode16<T, SRC, G>(v, &v_scale);
            if (mine && held) {
                *reinterpret_cast<u32x4*>(kc) = x;
                *reinterpret_cast<u32x4*>(vc) = y;
                if (part == 0) {
                    *ks = k_scale;
                    *vs = v_scale;
                }
            }
        } else {
            if (!mine) return;
            u32x4 k = none, v = none;
            if (held) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(kc), y = *reinterpret_cast<const u32x2*>(vc);
                const float k_scale = *ks, v_scale = *vs;
                k = scaled8<T, SRC>(x, k_scale);
                v = scaled8<T, SRC>(y, v_scale);
            }
            // (streaming: 306 us become 300 at the size above, and the codes that were just written stay in the caches)
            st128(kp, k);
            st128(vp, v);
        }
    }
}

}  // namespace neox
