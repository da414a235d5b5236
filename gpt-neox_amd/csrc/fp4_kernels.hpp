// The paged cache in 4 bits: e2m1 codes, 32 neighbouring values of a row under one power of two (a byte, its exponent + 127).
// The kernels that make the codes and take them back, and attention of single tokens over them; chunks of
// prompts are the forward kernel's (Stage4 in attention_kernels.hpp).  The machine makes and widens two codes an
// instruction, with the scale, and rounds to nearest even and saturates as the format says.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_kernels.hpp"
#include "cache_kernels.hpp"

namespace neox {

// ---- the cache ------------------------------------------------------------------------------------------
// exponent of the largest of 32 values, less 2, or less 1 where it is above 7/4 of its power: the least of which seven times is
// no less.  The smallest keeps its codes normal numbers of both types' exponents; the largest keeps six times finite.
constexpr uint32_t kScaleLeast = 127 - 125;
template <typename T>
constexpr uint32_t scale_most() { return __is_same(T, BF16) ? 127 + 125 : 127 + 13; }

template <typename T>
__device__ __forceinline__ uint32_t scale_of(uint32_t largest16) {
    float b, unused;
    Elem<T>::unpack(largest16, b, unused);
    const int e = (int)((__builtin_bit_cast(uint32_t, b) + 0x1fffffu) >> 23) - 2;
    return (uint32_t)min(max(e, (int)kScaleLeast), (int)scale_most<T>());
}

// two values of 16 bits as codes, into byte SEL of `word`
template <typename T, int SEL>
__device__ __forceinline__ uint32_t narrow2(uint32_t word, uint32_t pair, float scale) {
    if constexpr (__is_same(T, BF16)) return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(bf16x2, pair), scale, SEL);
    else return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(f16x2, pair), scale, SEL);
}
template <typename T>
__device__ __forceinline__ uint32_t narrow8(const u32x4& w, float scale) {
    uint32_t c = narrow2<T, 0>(0, w.x, scale);
    c = narrow2<T, 1>(c, w.y, scale);
    c = narrow2<T, 2>(c, w.z, scale);
    return narrow2<T, 3>(c, w.w, scale);
}

// A lane's 16 values (half of a scale's 32, the other half its neighbour's) as codes; G lanes to a row.
template <typename T, int G>
__device__ __forceinline__ u32x2 encode4(const u32x4 (&w)[2], uint32_t* scale) {
    uint32_t top = 0;  // the largest magnitude, on the bits: an infinity is larger than every number, a NaN larger still
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[h][i] & 0x7fffu, (w[h][i] >> 16) & 0x7fffu));
    constexpr uint32_t kInf = __is_same(T, BF16) ? 0x7f80u : 0x7c00u;
    const bool finite = group_largest<G>(top) < kInf;
    const uint32_t e = scale_of<T>(group_largest<2>(top));
    *scale = finite ? e : kScaleNan;
    const float f = scale_bits(e);
    return finite ? u32x2{narrow8<T>(w[0], f), narrow8<T>(w[1], f)} : u32x2{0, 0};
}

// G: lanes of a row, a power of two; 16 values a lane.
template <typename T, int G, bool WRITE>
__global__ __launch_bounds__(256) void cache4_kernel(CacheArgs a) {
    const uint32_t row = (uint32_t)(((uint64_t)blockIdx.x * 256 + threadIdx.x) / G);  // (below 2^30 + 256)
    const int part = threadIdx.x % G;
    const bool mine = row < (uint32_t)a.rows && part * 16 < a.d;
    const uint32_t token = a.by_heads.div(min(row, (uint32_t)a.rows - 1)), head = min(row, (uint32_t)a.rows - 1) - token * a.heads;
    const int64_t slot = a.wide ? static_cast<const int64_t*>(a.slots)[token] : static_cast<const int32_t*>(a.slots)[token];
    const bool held = slot >= 0 && slot < a.slot_count;
    // (page numbers and slots of a page are below 2^30, slots themselves may not be)
    const int64_t page = held ? (a.slot_count <= 0x7fffffff ? (int64_t)a.by_page.div((uint32_t)slot) : slot / a.page) : 0;
    const int64_t in = held ? slot - page * a.page : 0;
    char* const kp = a.k + (token * a.k_st[0] + head * a.k_st[1] + part * 16) * 2;
    char* const vp = a.v + (token * a.v_st[0] + head * a.v_st[1] + part * 16) * 2;
    char* const kc = a.kc + in * a.kc_st[0] + page * a.kc_st[1] + head * a.kc_st[2] + part * 8;
    char* const vc = a.vc + in * a.vc_st[0] + page * a.vc_st[1] + head * a.vc_st[2] + part * 8;
    uint8_t* const ks = reinterpret_cast<uint8_t*>(a.ks) + in * a.ks_st[0] + page * a.ks_st[1] + head * a.ks_st[2] + part / 2;
    uint8_t* const vs = reinterpret_cast<uint8_t*>(a.vs) + in * a.vs_st[0] + page * a.vs_st[1] + head * a.vs_st[2] + part / 2;
    const u32x4 none = {0, 0, 0, 0};
    if constexpr (WRITE) {
        u32x4 k[2] = {none, none}, v[2] = {none, none};
        if (mine) {
            k[0] = *reinterpret_cast<const u32x4*>(kp);
            k[1] = *reinterpret_cast<const u32x4*>(kp + 16);
            v[0] = *reinterpret_cast<const u32x4*>(vp);
            v[1] = *reinterpret_cast<const u32x4*>(vp + 16);
        }
        uint32_t k_scale, v_scale;
        const u32x2 x = encode4<T, G>(k, &k_scale), y = encode4<T, G>(v, &v_scale);
        if (mine && held) {
            *reinterpret_cast<u32x2*>(kc) = x;
            *reinterpret_cast<u32x2*>(vc) = y;
            if (part % 2 == 0) {
                *ks = (uint8_t)k_scale;
                *vs = (uint8_t)v_scale;
            }
        }
    } else {
        if (!mine) return;
        u32x4 k[2] = {none, none}, v[2] = {none, none};
        if (held) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(kc), y = *reinterpret_cast<const u32x2*>(vc);
            const float fk = scale_bits(*ks), fv = scale_bits(*vs);
            k[0] = widen4<T>(x.x, fk);
            k[1] = widen4<T>(x.y, fk);
            v[0] = widen4<T>(y.x, fv);
            v[1] = widen4<T>(y.y, fv);
        }
        st128(kp, k[0]);
        st128(kp + 16, k[1]);
        st128(vp, v[0]);
        st128(vp + 16, v[1]);
    }
}

// ---- single tokens ----------------------------------------------------------------------------------------
// As attn_token_kernel in attention_kernels.hpp: at most 16 rows per key head, every wave streams 32 keys at a time of its own,
// 16x16x32 tiles, the values through LDS of the wave's own for the transposing reads.  A lane fetches pieces of keys l % 16
// and 16 + l % 16 of which one scale holds all: 32 dims from 128 s + 32 (l / 16), at 64 and 96 dims 16 from 64 s + 16 (l / 16).  Codes
// take their scale along as bf16, exactly.  fp16 queries and the probabilities that go with them have 11 bits where
// bf16 has 8: they are the sum of two bf16 numbers and take two instructions each, so that nothing leaves fp16's range.
template <int DP>
struct Piece4 {
    static constexpr int kWords = DP >= 128 ? 4 : 2;   // of 8 codes
    static constexpr int kDims = 8 * kWords;           // of a lane
    static constexpr int kLoads = (DP + 4 * kDims - 1) / (4 * kDims);
    typedef std::conditional_t<kWords == 4, u32x4, u32x2> Codes;
};

template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(256, DP <= 128 ? 3 : 2) void attn_token4_kernel(AttnArgs a) {
    typedef Piece4<DP> P;
    typedef typename P::Codes Codes;
    constexpr bool kTwo = __is_same(T, F16);
    constexpr int kKeys = 32, kLoads = P::kLoads, kWords = P::kWords;
    constexpr int kWaveBytes = kKeys * Tile<DP>::kRow;
    __shared__ __attribute__((aligned(512))) char lds[4 * kWaveBytes];
    __shared__ float wave_m[4][16], wave_l[4][16];

    // The heads of one part of a sequence run on one XCD at about the same time: their rows are neighbours in memory.
    const uint32_t turn = blockIdx.x >> 3, at = a.by_kv.div(turn), item = at * 8 + (blockIdx.x & 7);
    const int g = turn - at * a.kv;
    if (item >= (uint32_t)a.b * a.splits) return;
    const int b = SPLIT ? a.by_splits.div(item) : item, split = SPLIT ? item - b * a.splits : 0;
    int token0, tokens, keys;
    paged_sample(a, b, token0, tokens, keys);
    const int rows = min(tokens * a.group, 16);
    if (rows == 0) return;
    const int position0 = keys - tokens;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, quad = lane >> 4, col = lane & 15;
    const bool there = col < rows;
    const int row = min(col, rows - 1);
    const int token = a.by_group.div(row), head = g * a.group + row - token * a.group;
    const int position = position0 + token;

    const KeyTiles tiles = key_tiles<kKeys>(position0, position0 + tokens - 1, keys, a.window, a.sinks);
    int first = 0, end = tiles.count;
    if constexpr (SPLIT) {
        const int each = ((tiles.count + a.splits - 1) / a.splits + 3) / 4 * 4;
        first = min(split * each, tiles.count);
        end = min(first + each, tiles.count);
    }

    auto dim_of = [&](int s) { return 4 * P::kDims * s + P::kDims * quad; };
    u32x4 q[kLoads * kWords], q_low[kTwo ? kLoads * kWords : 1];
    {
        const char* p = a.q + ((int64_t)(token0 + token) * a.q_st[0] + (int64_t)head * a.q_st[2]) * 2;
#pragma unroll
        for (int s = 0; s < kLoads; ++s)
#pragma unroll
            for (int t = 0; t < kWords; ++t) {
                const int dim = dim_of(s) + 8 * t;
                u32x4 x = load8(p + dim * 2, there && dim < a.d);
                x ^= a.flip;
                if constexpr (kTwo) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float lo, hi;
                        uint32_t rest;
                        Elem<F16>::unpack(x[i], lo, hi);
                        q[s * kWords + t][i] = pack_with_rest<BF16>(lo, hi, rest);
                        // (nothing is left of an infinity)
                        if (__builtin_fabsf(lo) == __builtin_inff()) rest &= 0xffff0000u;
                        if (__builtin_fabsf(hi) == __builtin_inff()) rest &= 0x0000ffffu;
                        q_low[s * kWords + t][i] = rest;
                    }
                } else {
                    q[s * kWords + t] = x;
                }
            }
    }

    char* const vt = lds + wave * kWaveBytes;
    uint32_t put_at, get_at;
    {
        put_at = lds_byte(vt) + (col * Tile<DP>::kRow | (Tile<DP>::turn(col) ^ (kWords * quad)) << 4);
        const uint32_t j = col, r = 4 * quad + (j >> 2);
        get_at = lds_byte(vt) + (r * Tile<DP>::kRow | (Tile<DP>::turn(r) ^ ((j >> 1) & 1)) << 4 | (j & 1) * 8);
    }
    const int32_t* const table = a.table + (int64_t)b * a.table_stride;
    Codes kw[2][kLoads], vw[2][kLoads];
    uint32_t ke[2][kLoads], ve[2][kLoads];
    // Where pages hold whole blocks, a block has one page and its addresses are a scalar and a lane's own offset;
    // otherwise every lane looks up the pages of its two keys.
    const bool even = a.by_page.d % kKeys == 0 && a.k_st[0] < kSmallStride && a.v_st[0] < kSmallStride && a.ks_st[0] < kSmallStride &&
                      a.vs_st[0] < kSmallStride;
    uint32_t block_page = 0;
    int pages[2];
    auto look_up = [&](int i) {
        if (even) {
            const int key = tiles.tile(i) * kKeys;
            block_page = i < end ? __builtin_amdgcn_readfirstlane(table[a.by_page.div(key)]) : ~0u;
            return;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int key = tiles.tile(i) * kKeys + 16 * kb + col;
            pages[kb] = i < end && key < keys ? table[a.by_page.div(key)] : -1;
        }
    };
    const uint32_t k_row = (uint32_t)a.k_st[0], v_row = (uint32_t)a.v_st[0], ks_row = (uint32_t)a.ks_st[0], vs_row = (uint32_t)a.vs_st[0];
    const char* const kbase = a.k + (int64_t)g * a.k_st[2];
    const char* const vbase = a.v + (int64_t)g * a.v_st[2];
    const char* const ksbase = reinterpret_cast<const char*>(a.k_scale) + (int64_t)g * a.ks_st[2];
    const char* const vsbase = reinterpret_cast<const char*>(a.v_scale) + (int64_t)g * a.vs_st[2];
    const uint32_t code0 = dim_of(0) / 2, scale0 = dim_of(0) / 32;
    auto codes_at = [](const char* p, bool ok) {
        Codes c = {};
        if (ok) c = *reinterpret_cast<const Codes*>(p);
        return c;
    };
    auto scale_at = [](const char* p, bool ok) { return ok ? (uint32_t)*reinterpret_cast<const uint8_t*>(p) : 0u; };
    auto fetch = [&](int i) {
        const int key0 = tiles.tile(i) * kKeys;
        if (even && key0 + kKeys <= keys && block_page < (uint32_t)a.pages) {
            const uint32_t in = a.by_page.mod(key0);
            const char* const kp = step_to(step_to(kbase, block_page, (uint32_t)a.k_st[1]), in, k_row);
            const char* const vp = step_to(step_to(vbase, block_page, (uint32_t)a.v_st[1]), in, v_row);
            const char* const kf = step_to(step_to(ksbase, block_page, (uint32_t)a.ks_st[1]), in, ks_row);
            const char* const vf = step_to(step_to(vsbase, block_page, (uint32_t)a.vs_st[1]), in, vs_row);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int s = 0; s < kLoads; ++s) {
                    const bool ok = dim_of(s) < a.d;
                    kw[kb][s] = codes_at(kp + (uint64_t)(16 * kb) * k_row + s * 2 * P::kDims + (col * k_row + code0), ok);
                    vw[kb][s] = codes_at(vp + (uint64_t)(16 * kb) * v_row + s * 2 * P::kDims + (col * v_row + code0), ok);
                    ke[kb][s] = scale_at(kf + (uint64_t)(16 * kb) * ks_row + s * P::kDims / 8 + (col * ks_row + scale0), ok);
                    ve[kb][s] = scale_at(vf + (uint64_t)(16 * kb) * vs_row + s * P::kDims / 8 + (col * vs_row + scale0), ok);
                }
            return;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int key = key0 + 16 * kb + col;
            const uint32_t page = even ? block_page : pages[kb], in = a.by_page.mod(key);
            const bool is = key < keys && page < (uint32_t)a.pages;
            const char* const kp = step_to(step_to(kbase, page, (uint32_t)a.k_st[1]), in, k_row) + code0;
            const char* const vp = step_to(step_to(vbase, page, (uint32_t)a.v_st[1]), in, v_row) + code0;
            const char* const kf = step_to(step_to(ksbase, page, (uint32_t)a.ks_st[1]), in, ks_row) + scale0;
            const char* const vf = step_to(step_to(vsbase, page, (uint32_t)a.vs_st[1]), in, vs_row) + scale0;
#pragma unroll
            for (int s = 0; s < kLoads; ++s) {
                const bool ok = is && dim_of(s) < a.d;
                kw[kb][s] = codes_at(kp + s * 2 * P::kDims, ok);
                vw[kb][s] = codes_at(vp + s * 2 * P::kDims, ok);
                ke[kb][s] = scale_at(kf + s * P::kDims / 8, ok);
                ve[kb][s] = scale_at(vf + s * P::kDims / 8, ok);
            }
        }
    };

    f32x4 acc[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.f;

    look_up(first + wave);
    if (first + wave < end) fetch(first + wave);
    look_up(first + wave + 4);
    for (int i = first + wave; i < end; i += 4) {
        const int key0 = tiles.tile(i) * kKeys;
        asm("" : "+v"(put_at), "+v"(get_at));
        typedef __attribute__((address_space(3))) u32x4 lds16;
        typedef __attribute__((address_space(3))) s16x4 lds4;
        f32x4 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            s[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < kLoads; ++st) {
                const float f = scale_bits(ke[kb][st]);
#pragma unroll
                for (int t = 0; t < kWords; ++t) {
                    const u32x4 w = widen4<BF16>(kw[kb][st][t], f);
                    s[kb] = Mma<BF16>::op16(w, q[st * kWords + t], s[kb]);
                    if constexpr (kTwo) s[kb] = Mma<BF16>::op16(w, q_low[st * kWords + t], s[kb]);
                }
            }
        }
        // A NaN scale among the values: their codes go without, and the probabilities that are not zero become NaN.
        // bits: key l % 16 of either half; rare
        uint32_t nan_keys[2] = {0, 0};
        bool nan = false;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int st = 0; st < kLoads; ++st) nan |= ve[kb][st] == kScaleNan;
        const bool any_nan = __any(nan);
        if (any_nan) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int st = 0; st < kLoads; ++st) {
                    const uint64_t of = __ballot(ve[kb][st] == kScaleNan);
                    nan_keys[kb] |= (uint32_t)(of | of >> 16 | of >> 32 | of >> 48) & 0xffffu;
                    ve[kb][st] = ve[kb][st] == kScaleNan ? 0 : ve[kb][st];
                }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int st = 0; st < kLoads; ++st) {
                const float f = scale_bits(ve[kb][st]);
                if (DP % (4 * P::kDims) == 0 || dim_of(st) < DP) {
#pragma unroll
                    for (int t = 0; t < kWords; ++t)
                        *(lds16*)(uintptr_t)((put_at ^ (st * 4 * kWords + t) << 4) + 16 * kb * Tile<DP>::kRow) = widen4<BF16>(vw[kb][st][t], f);
                }
            }
        if (i + 4 < end) {
            fetch(i + 4);
            look_up(i + 8);
        }
        __builtin_amdgcn_wave_barrier();
        // (the last token sees furthest ahead, the first least; a window's near end moves with both)
        const bool all = key0 + kKeys - 1 <= position0 && key0 + kKeys <= keys &&
                         (a.window < 0 || key0 >= position0 + tokens - 1 - a.window || key0 + kKeys <= a.sinks);
        if (!all) {
            const int lo = a.window < 0 ? 0 : position - a.window, hi = min(position, keys - 1);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = key0 + 16 * kb + 4 * quad + r;
                    const bool sees = key <= hi && (key >= lo || key < a.sinks);
                    s[kb][r] = sees ? s[kb][r] : kNegInf;
                }
        }
        float top = kNegInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[kb][r]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = both_halves_max(top) * a.scale_log2;
        if (__any(top > m + 8.f)) {
            const float higher = fmaxf(m, top);
            const float f = __builtin_amdgcn_exp2f(m - (higher == kNegInf ? 0.f : higher));
            m = higher;
            l *= f;
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) acc[j] *= f;
        }
        const float base = m == kNegInf ? 0.f : m;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.scale_log2, -base));
                l += s[kb][r];
            }
        if (any_nan) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[kb][r] = (nan_keys[kb] >> (4 * quad + r) & 1) && s[kb][r] != 0.f ? nan_value() : s[kb][r];
        }
        u32x4 p, p_low = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (kTwo) {
                uint32_t rest;
                p[e] = pack_with_rest<BF16>(s[e >> 1][2 * (e & 1)], s[e >> 1][2 * (e & 1) + 1], rest);
                p_low[e] = rest;
            } else {
                p[e] = Elem<BF16>::pack(s[e >> 1][2 * (e & 1)], s[e >> 1][2 * (e & 1) + 1]);
            }
        }
#pragma unroll
        for (int db = 0; db < DP / 16; ++db) {
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(get_at ^ (db << 5)));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)((get_at ^ (db << 5)) + 16 * Tile<DP>::kRow));
            const u32x2 u = __builtin_bit_cast(u32x2, x), v = __builtin_bit_cast(u32x2, y);
            acc[db] = Mma<BF16>::op16(u32x4{u.x, u.y, v.x, v.y}, p, acc[db]);
            if constexpr (kTwo) acc[db] = Mma<BF16>::op16(u32x4{u.x, u.y, v.x, v.y}, p_low, acc[db]);
        }
        __builtin_amdgcn_wave_barrier();
    }

    // the four waves' results: rows of DP values in each wave's own LDS, joined by the whole workgroup
    l += __shfl_xor(l, 16);
    l = both_halves_sum(l);
    float* const mine = reinterpret_cast<float*>(vt);
#pragma unroll
    for (int db = 0; db < DP / 16; ++db) *reinterpret_cast<f32x4*>(mine + col * DP + 16 * db + 4 * quad) = acc[db];
    if (quad == 0) {
        wave_m[wave][col] = m;
        wave_l[wave][col] = l;
    }
    __syncthreads();
    for (int at = threadIdx.x * 8; at < rows * DP; at += 256 * 8) {
        const int r = at / DP, dim = at % DP;
        if (dim >= a.d) continue;
        float high = wave_m[0][r];
#pragma unroll
        for (int w = 1; w < 4; ++w) high = fmaxf(high, wave_m[w][r]);
        const float base = high == kNegInf ? 0.f : high;
        float total = 0.f, x[8] = {};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(wave_m[w][r] - base);
            total += wave_l[w][r] * f;
            const float* from = reinterpret_cast<const float*>(lds + w * kWaveBytes) + r * DP + dim;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] += from[e] * f;
        }
        const float inverse = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= inverse;
        const int t = a.by_group.div(r), h = g * a.group + r - t * a.group;
        if constexpr (SPLIT) {
            const int64_t slot = (int64_t)split * a.part_rows + (int64_t)(token0 + t) * a.kv * a.group + h;
            float* p = a.part_o + slot * a.d + dim;
            *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
            if (dim == 0) a.part_lse[slot] = total == 0.f ? kNegInf : high + __builtin_amdgcn_logf(total);
        } else {
            *reinterpret_cast<u32x4*>(a.o + ((int64_t)(token0 + t) * a.o_st[0] + (int64_t)h * a.o_st[2] + dim) * 2) = pack8<T>(x);
        }
    }
}

}  // namespace neox
