// The paged key/value cache: new keys and values into their slots, as 16-bit values or as 8-bit codes with a scale
// for each (token, head), and back.
//
// scale = largest |x| of the row / the largest code (127, or 448 for 8-bit floats), code = x * largest code / largest
// |x|, rounded to nearest even.  The quotient is the correctly rounded one: with y = 1 / b rounded, one correction
// q + fma(-q, b, a) * y of q = a * y gives the rounded a / b, so that exact ties between two codes are seen as ties.
// Bound by memory: a lane moves 8 elements, a row takes d / 8 neighbouring lanes, and the keys' and values' rows of a
// (token, head) go together, two loads in flight for every lane.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_kernels.hpp"

namespace neox {

struct CacheArgs {
    char *k, *v;                      // rows outside the cache, 16-bit
    char *kc, *vc;                    // the cache
    float *ks, *vs;                   // its scales
    const void* slots;
    int64_t k_st[2], v_st[2];         // token, head
    int64_t kc_st[3], vc_st[3], ks_st[3], vs_st[3];  // token within a page, page, head
    int64_t slot_count;               // slots of the cache; page = slot / page size
    int64_t rows;                     // tokens * heads
    int heads, d, page;
    bool wide;                        // 64-bit slots
};

// largest of the 16 lanes' (8, 32) values of a row, lane groups of G; values are non-negative integers
template <int G>
__device__ __forceinline__ uint32_t group_largest(uint32_t x) {
#pragma unroll
    for (int i = 1; i < G; i *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, i));
    return x;
}

// One row's share of a lane (8 elements in w) as codes; *scale gets the row's.
template <typename T, int SRC, int G>
__device__ __forceinline__ u32x2 encode8(const u32x4& w, float* scale) {
    constexpr float kTop = SRC == kPagedI8 ? 127.f : 448.f;
    // the largest magnitude, on the bits: an infinity is larger than every number, a NaN larger still
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
    top = group_largest<G>(top);
    float b, unused;
    Elem<T>::unpack(top, b, unused);
    const bool finite = b < __builtin_inff();
    *scale = finite ? b / kTop : __builtin_nanf("");
    // values whose product with the largest code or whose reciprocal would leave the range are moved into it
    const float shift = b > 0x1p100f ? 0x1p-100f : b < 0x1p-100f ? 0x1p100f : 1.f;
    b *= shift;
    const float y = 1.f / b;
    float x[8];
    unpack8<T>(w, x);
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = x[i] * shift * kTop;
        float q = a * y;
        q = __builtin_fmaf(__builtin_fmaf(-q, b, a), y, q);
        x[i] = finite && b > 0.f ? q : 0.f;
        if constexpr (SRC == kPagedI8) code[i] = __builtin_bit_cast(uint32_t, x[i] + 12582912.f) & 0xffu;  // 1.5 * 2^23: rounds to a whole number
    }
    if constexpr (SRC == kPagedI8) {
        return u32x2{code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24};
    } else {
        int lo = 0, hi = 0;
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], hi, true);
        return u32x2{(uint32_t)lo, (uint32_t)hi};
    }
}

// G: lanes of a row, the power of two from d / 8 on.
template <typename T, int SRC, int G, bool WRITE>
__global__ __launch_bounds__(256) void cache_kernel(CacheArgs a) {
    constexpr bool kCodes = SRC != kPaged16;
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
    const int part = threadIdx.x % G;
    const bool mine = row < a.rows && part * 8 < a.d;
    const int64_t token = row < a.rows ? row / a.heads : 0, head = row < a.rows ? row - token * a.heads : 0;
    int64_t slot = -1;
    if (row < a.rows) slot = a.wide ? static_cast<const int64_t*>(a.slots)[token] : static_cast<const int32_t*>(a.slots)[token];
    const bool held = slot >= 0 && slot < a.slot_count;
    const int64_t page = held ? slot / a.page : 0, in = held ? slot - page * a.page : 0;
    char* const kp = a.k + (token * a.k_st[0] + head * a.k_st[1] + part * 8) * 2;
    char* const vp = a.v + (token * a.v_st[0] + head * a.v_st[1] + part * 8) * 2;
    constexpr int kBytes = kCodes ? 1 : 2;
    char* const kc = a.kc + (in * a.kc_st[0] + page * a.kc_st[1] + head * a.kc_st[2] + part * 8) * kBytes;
    char* const vc = a.vc + (in * a.vc_st[0] + page * a.vc_st[1] + head * a.vc_st[2] + part * 8) * kBytes;
    float *ks = nullptr, *vs = nullptr;
    if constexpr (kCodes) {
        ks = a.ks + in * a.ks_st[0] + page * a.ks_st[1] + head * a.ks_st[2];
        vs = a.vs + in * a.vs_st[0] + page * a.vs_st[1] + head * a.vs_st[2];
    }
    if constexpr (WRITE) {
        const u32x4 k = load8(kp, mine), v = load8(vp, mine);
        if constexpr (kCodes) {
            float k_scale, v_scale;
            const u32x2 x = encode8<T, SRC, G>(k, &k_scale), y = encode8<T, SRC, G>(v, &v_scale);
            if (mine && held) {
                *reinterpret_cast<u32x2*>(kc) = x;
                *reinterpret_cast<u32x2*>(vc) = y;
                if (part == 0) {
                    *ks = k_scale;
                    *vs = v_scale;
                }
            }
        } else if (mine && held) {
            *reinterpret_cast<u32x4*>(kc) = k;
            *reinterpret_cast<u32x4*>(vc) = v;
        }
    } else {
        u32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
        if (mine && held) {
            if constexpr (kCodes) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(kc), y = *reinterpret_cast<const u32x2*>(vc);
                const float k_scale = *ks, v_scale = *vs;
                float f[8];
                decode8<SRC>(x, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] *= k_scale;
                k = pack8<T>(f);
                decode8<SRC>(y, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] *= v_scale;
                v = pack8<T>(f);
            } else {
                k = *reinterpret_cast<const u32x4*>(kc);
                v = *reinterpret_cast<const u32x4*>(vc);
            }
        }
        if (mine) {
            *reinterpret_cast<u32x4*>(kp) = k;
            *reinterpret_cast<u32x4*>(vp) = v;
        }
    }
}

}  // namespace neox
