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
constexpr uint32_t scale_most() { return __is_same(T, BF16) ? kScaleMost : 127 + 13; }

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

// Values of a lane: 16 where codes are made; 8 on the way back, so that the 16-bit side is dense (with 16, whose lanes store
// every other 16 bytes, 65536 tokens of 32 heads of 128 dims take 461 us).
template <bool WRITE>
__host__ __device__ constexpr int cache4_elems() { return WRITE ? 16 : 8; }

// G: lanes of a row, a power of two.  Bound by memory: 65536 tokens of 32 heads of 128 dims in bf16 take 253 us into the cache and 260 back,
// 5.3 TB/s; a few tokens 2.6 and 3.1, a launch.
template <typename T, int G, bool WRITE>
__global__ __launch_bounds__(256) void cache4_kernel(CacheArgs a) {
    const uint32_t row = (uint32_t)(((uint64_t)blockIdx.x * 256 + threadIdx.x) / G);  // (below 2^30 + 256)
    const int part = threadIdx.x % G;
    const bool mine = row < (uint32_t)a.rows && part * cache4_elems<WRITE>() < a.d;
    const uint32_t token = a.by_heads.div(min(row, (uint32_t)a.rows - 1)), head = min(row, (uint32_t)a.rows - 1) - token * a.heads;
    const int64_t slot = a.wide ? static_cast<const int64_t*>(a.slots)[token] : static_cast<const int32_t*>(a.slots)[token];
    const bool held = slot >= 0 && slot < a.slot_count;
    // (page numbers and slots of a page are below 2^30, slots themselves may not be)
    const int64_t page = held ? (a.slot_count <= 0x7fffffff ? (int64_t)a.by_page.div((uint32_t)slot) : slot / a.page) : 0;
    const int64_t in = held ? slot - page * a.page : 0;
    constexpr int kElems = cache4_elems<WRITE>();
    char* const kp = a.k + (token * a.k_st[0] + head * a.k_st[1] + part * kElems) * 2;
    char* const vp = a.v + (token * a.v_st[0] + head * a.v_st[1] + part * kElems) * 2;
    char* const kc = a.kc + in * a.kc_st[0] + page * a.kc_st[1] + head * a.kc_st[2] + part * (kElems / 2);
    char* const vc = a.vc + in * a.vc_st[0] + page * a.vc_st[1] + head * a.vc_st[2] + part * (kElems / 2);
    uint8_t* const ks = reinterpret_cast<uint8_t*>(a.ks) + in * a.ks_st[0] + page * a.ks_st[1] + head * a.ks_st[2] + part * kElems / 32;
    uint8_t* const vs = reinterpret_cast<uint8_t*>(a.vs) + in * a.vs_st[0] + page * a.vs_st[1] + head * a.vs_st[2] + part * kElems / 32;
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
        u32x4 k = none, v = none;
        if (held) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(kc), y = *reinterpret_cast<const uint32_t*>(vc);
            const float fk = scale_bits(known_scale(*ks)), fv = scale_bits(known_scale(*vs));
            k = widen4<T>(x, fk);
            v = widen4<T>(y, fv);
        }
        st128(kp, k);
        st128(vp, v);
    }
}

// ---- single tokens ----------------------------------------------------------------------------------------
// As attn_token_kernel in attention_kernels.hpp: 16 rows of a key head to a workgroup, every wave streams blocks of 32 keys of its own,
// 16x16x32 tiles, the values through LDS of the wave's own for the transposing reads.  A lane fetches pieces of keys l % 16 and
// 16 + l % 16 of which one scale holds all: 32 dims from 128 s + 32 (l / 16), at 64 and 96 dims 16 from 64 s + 16 (l / 16).
// Codes take their scale along as bf16, exactly.  fp16 queries and the probabilities that go with them have 11 bits where
// bf16 has 8: they are the sum of two bf16 numbers and take two instructions each, so that nothing leaves fp16's range.
//
// A wave works on HEADS neighbouring key heads at once, whose rows share the 16 columns of its tiles: a column takes the
// scores of its own head's product and meets its own head's values, the others' with probabilities of zero.  The loads are the
// bound, and two heads of a row are next to each other.  us with one and two heads to a wave, bf16, 128 dims, 32 heads on 8: 64
// sequences of 8192 tokens 104, 93 (with nothing but the loads 80, 77); one of 131001 45, 38; 16 of 8192 35, 35; four with 64 dims
// no less than two; but four sequences of 4099 with 8 heads 17.4, 18.6: two take CUs that have work enough.
//
// Measured: 64 sequences of 2048 to 8192 tokens, a token each, 32 heads on 8 of 128 dims, bf16, 84 us, 4.2 TB/s; one of 131001 28.9, 4.9; the launch
// that joins the parts 4.7 to 4.9.  At 4 sequences of 517 tokens 7.5 us are the latency of one block of keys after the other.  In fp16, whose two-head
// kernels of 96 and 128 dims spill 3 registers, the 64 sequences take 93.6 with the join, in bf16 89.0.
// With bf16 queries the probabilities are rounded to bf16 for the second product, half an ulp of each as in the other kernels: outputs are off by 1.2
// times their own rounding.  Two instructions each, as in fp16, would take that away; the sums stay in 32 bits either way.
//
// Scales come by rows, lanes 0-31 the keys' and 32-63 the values', and go to the lanes that need them from there: loads of a byte for
// each lane cost as much as those of its 16 bytes of codes (64 sequences of 2048 to 8192 tokens: 98 us, so 85).
template <int DP>
struct Piece4 {
    static constexpr int kWords = DP >= 128 ? 4 : 2;   // of 8 codes
    static constexpr int kDims = 8 * kWords;           // of a lane
    static constexpr int kLoads = (DP + 4 * kDims - 1) / (4 * kDims);
    typedef std::conditional_t<kWords == 4, u32x4, u32x2> Codes;
};

// the scales of a row of DP dims: as many bytes as a load takes, one by one at 96 and 160
template <int DP>
struct Scales4 {
    typedef std::conditional_t<DP == 64, uint16_t, std::conditional_t<DP == 96 || DP == 160, uint8_t, uint32_t>> Unit;
    static constexpr int kUnits = DP == 96 ? 3 : DP == 160 ? 5 : DP == 256 ? 2 : 1;
};

// the larger of the values of lane l and of lane l ^ 16
__device__ __forceinline__ float both_quads_max(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

template <typename C>
__device__ __forceinline__ C buf_codes(rsrc_t r, uint32_t at) {
    if constexpr (sizeof(C) == 16) return buf_ld128<false>(r, (int)at, 0);
    else return buf_ld64(r, (int)at, 0);
}

// The head dims that the kernels over 4 bits are built for.  (160: for chunks, whose figures are at the forward kernel; 64 sequences of 2048 to 8192
// tokens of 16 heads on 8, a token each, take 138 us there and padded to 256.)
inline int padded4(int d) { return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 160 ? 160 : 256; }

// How the kernel may fetch: half a block, 16 keys, through one buffer if pages hold whole halves, keys and values are laid out alike,
// and a row's bytes lie before the next row's (kFetchHalves); and the scales of a row at once if there are DP dims and these are
// aligned (kFetchRows).  Otherwise every lane goes by itself (kFetchOwn).
enum Fetch4 { kFetchOwn = 0, kFetchHalves = 1, kFetchRows = 2 };
inline Fetch4 token4_fetch(const AttnArgs& a, int dp) {
    const int64_t row = a.d / 2, scales = a.d / 32;
    int64_t bits = reinterpret_cast<intptr_t>(a.k_scale) | reinterpret_cast<intptr_t>(a.v_scale);
    for (int i = 0; i < 3; ++i) {
        if (a.k_st[i] != a.v_st[i] || a.ks_st[i] != a.vs_st[i]) return kFetchOwn;
        bits |= a.ks_st[i];
    }
    if (a.by_page.d % 16 != 0 || a.k_st[0] < row || a.ks_st[0] < scales || a.k_st[0] >= kSmallStride || a.ks_st[0] >= kSmallStride) return kFetchOwn;
    return a.d == dp && (dp == 96 || dp == 160 || bits % (dp / 32) == 0) ? kFetchRows : kFetchHalves;
}

template <typename T, int DP, int HEADS, bool SPLIT, int FETCH, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 2 : DP <= 128 ? 3 : 2) void attn_token4_kernel(AttnArgs a) {
    typedef Piece4<DP> P;
    typedef typename P::Codes Codes;
    constexpr bool kTwo = __is_same(T, F16), EVEN = FETCH != kFetchOwn, kScaleRows = FETCH == kFetchRows;
    constexpr int kKeys = 32, kLoads = P::kLoads, kWords = P::kWords, kColumns = 16 / HEADS;  // columns of a head
    constexpr int kWaveBytes = kKeys * Tile<DP>::kRow;
    __shared__ __attribute__((aligned(512))) char lds[WAVES * kWaveBytes];
    __shared__ float wave_m[WAVES][16], wave_l[WAVES][16];

    // The heads of one part of a sequence, and the blocks of 16 rows of a head, run on one XCD at about the same time: what they read is
    // in the same lines.  (by_kv: by the groups of HEADS heads, times the blocks)
    const uint32_t turn = blockIdx.x >> 3, at = a.by_kv.div(turn), item = at * 8 + (blockIdx.x & 7);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, quad = lane >> 4, col = lane & 15;
    const uint32_t sub = turn - at * a.by_kv.d, group_of = a.by_row_tiles.div(sub);
    const int g0 = group_of * HEADS, row0 = (sub - group_of * a.row_tiles) * 16;
    if (item >= (uint32_t)a.b * a.splits) return;
    const int b = SPLIT ? a.by_splits.div(item) : item, split = SPLIT ? item - b * a.splits : 0;
    int token0, tokens, keys;
    paged_sample(a, b, token0, tokens, keys);
    const int rows = min(tokens * a.group - row0, kColumns);
    if (rows <= 0) return;
    const int position0 = keys - tokens;
    const int first_position = position0 + (int)a.by_group.div(row0), last_position = position0 + (int)a.by_group.div(row0 + rows - 1);

    const int mine = col / kColumns;  // of the heads
    const bool there = col % kColumns < rows;
    const int row = row0 + min(col % kColumns, rows - 1);
    const int token = a.by_group.div(row), head = (g0 + mine) * a.group + row - token * a.group;
    const int position = position0 + token;

    const KeyTiles tiles = key_tiles<kKeys>(first_position, last_position, keys, a.window, a.sinks);
    int first = 0, end = tiles.count;
    if constexpr (SPLIT) {
        const int each = ((tiles.count + a.splits - 1) / a.splits + WAVES - 1) / WAVES * WAVES;
        first = min(split * each, tiles.count);
        end = min(first + each, tiles.count);
    }
    first += wave;

    auto dim_of = [&](int s) { return 4 * P::kDims * s + P::kDims * quad; };
    char* const vt = lds + wave * kWaveBytes;
    uint32_t put_at, get_at;
    {
        put_at = lds_byte(vt) + (col * Tile<DP>::kRow | (Tile<DP>::turn(col) ^ (kWords * quad)) << 4);
        const uint32_t j = col, r = 4 * quad + (j >> 2);
        get_at = lds_byte(vt) + (r * Tile<DP>::kRow | (Tile<DP>::turn(r) ^ ((j >> 1) & 1)) << 4 | (j & 1) * 8);
    }
    const int32_t* const table = a.table + (int64_t)b * a.table_stride;
    Codes kw[HEADS][2][kLoads], vw[HEADS][2][kLoads];
    typename Scales4<DP>::Unit rows_of[HEADS][Scales4<DP>::kUnits];
    uint8_t ke[HEADS][2][kLoads], ve[HEADS][2][kLoads];  // (bytes: as words they would be cut to bytes, and waited for, where they are loaded)
    const uint32_t code0 = dim_of(0) / 2, scale0 = dim_of(0) / 32;
    // The pages of this wave's next blocks.  EVEN: lane 2 n + h has that of half h of the n-th block of 32, looked up 32 blocks ahead;
    // otherwise those of a lane's own two keys, one block ahead.
    uint32_t page_set[2];
    auto look_up = [&](int n) {  // n: blocks from the wave's first one
        const int i = first + WAVES * (n + (lane >> 1)), key = tiles.tile(i) * kKeys + 16 * (lane & 1);
        return i < end && key < keys ? (uint32_t)table[a.by_page.div(key)] : ~0u;
    };
    auto look_up_own = [&](int n) {
        const int i = first + WAVES * n;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int key = tiles.tile(i) * kKeys + 16 * kb + col;
            page_set[kb] = i < end && key < keys ? (uint32_t)table[a.by_page.div(key)] : ~0u;
        }
    };
    const uint32_t k_row = (uint32_t)a.k_st[0], v_row = (uint32_t)a.v_st[0], ks_row = (uint32_t)a.ks_st[0], vs_row = (uint32_t)a.vs_st[0];
    const char* const kbase = a.k + (int64_t)g0 * a.k_st[2];
    const char* const vbase = a.v + (int64_t)g0 * a.v_st[2];
    const char* const ksbase = reinterpret_cast<const char*>(a.k_scale) + (int64_t)g0 * a.ks_st[2];
    const char* const vsbase = reinterpret_cast<const char*>(a.v_scale) + (int64_t)g0 * a.vs_st[2];
    // kFetchRows: lanes 0-31 have the scales of the block's keys, 32-63 those of its values
    const char* const own_scales = (lane & 32 ? vsbase : ksbase) + col * ks_row;
    // A lane's place in 16 rows; what lies behind the last key, in no page or behind d is outside the buffer, and zero.
    uint32_t code_at[kLoads], scale_at[kLoads];
    if constexpr (EVEN) {
#pragma unroll
        for (int s = 0; s < kLoads; ++s) {
            const bool ok = dim_of(s) < a.d;
            code_at[s] = ok ? col * k_row + code0 + s * 2 * P::kDims : kOutOfRange;
            scale_at[s] = ok ? col * ks_row + scale0 + s * P::kDims / 8 : kOutOfRange;
        }
    }
    int ahead = 0;  // blocks fetched so far
    bool key_there[2];
    auto fetch = [&](int i) {
        const int key0 = tiles.tile(i) * kKeys;
        if constexpr (EVEN) {
            const int at = 2 * (ahead & 31);
            if (ahead && at == 0) {
                page_set[0] = page_set[1];
                page_set[1] = look_up(ahead + 32);
            }
            uint64_t code_off[2], scale_off[2];
            uint32_t count[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const uint32_t page = __builtin_amdgcn_readlane(page_set[0], at + kb), in = a.by_page.mod(key0 + 16 * kb);
                // (a vector instruction where the compiler sees a median: it is told that all lanes have the same)
                count[kb] = __builtin_amdgcn_readfirstlane(page < (uint32_t)a.pages ? (uint32_t)max(0, min(16, keys - key0 - 16 * kb)) : 0);
                code_off[kb] = (uint64_t)page * (uint32_t)a.k_st[1] + (uint64_t)in * k_row;
                scale_off[kb] = (uint64_t)page * (uint32_t)a.ks_st[1] + (uint64_t)in * ks_row;
            }
            if constexpr (kScaleRows) {
                const uint64_t off = lane & 16 ? scale_off[1] : scale_off[0];
                const bool ok = col < (int)(lane & 16 ? count[1] : count[0]);
                typedef Scales4<DP> S;
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    const auto* from = reinterpret_cast<const typename S::Unit*>(own_scales + (off + (uint64_t)h * (uint32_t)a.ks_st[2]));
#pragma unroll
                    for (int u = 0; u < S::kUnits; ++u) rows_of[h][u] = 0;
                    if (ok) {
#pragma unroll
                        for (int u = 0; u < S::kUnits; ++u) rows_of[h][u] = from[u];
                    }
                }
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    const rsrc_t codes = make_rsrc(kbase + (code_off[kb] + (uint64_t)h * (uint32_t)a.k_st[2]), count[kb] * k_row);
                    const rsrc_t scales = make_rsrc(ksbase + (scale_off[kb] + (uint64_t)h * (uint32_t)a.ks_st[2]), count[kb] * ks_row);
#pragma unroll
                    for (int s = 0; s < kLoads; ++s) {
                        kw[h][kb][s] = buf_codes<Codes>(codes, code_at[s]);
                        if constexpr (!kScaleRows) ke[h][kb][s] = __builtin_amdgcn_raw_buffer_load_b8(scales, scale_at[s], 0, 0);
                    }
                }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    const rsrc_t codes = make_rsrc(vbase + (code_off[kb] + (uint64_t)h * (uint32_t)a.v_st[2]), count[kb] * v_row);
                    const rsrc_t scales = make_rsrc(vsbase + (scale_off[kb] + (uint64_t)h * (uint32_t)a.vs_st[2]), count[kb] * vs_row);
#pragma unroll
                    for (int s = 0; s < kLoads; ++s) {
                        vw[h][kb][s] = buf_codes<Codes>(codes, code_at[s]);
                        if constexpr (!kScaleRows) ve[h][kb][s] = __builtin_amdgcn_raw_buffer_load_b8(scales, scale_at[s], 0, 0);
                    }
                }
        } else {
            // Lanes with nothing to fetch read the head's first piece instead, and throw it away when its turn comes.
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int key = key0 + 16 * kb + col;
                key_there[kb] = key < keys && page_set[kb] < (uint32_t)a.pages;
                const uint32_t page = key_there[kb] ? page_set[kb] : 0, in = key_there[kb] ? a.by_page.mod(key) : 0;
                const char* kp = step_to(step_to(kbase, page, (uint32_t)a.k_st[1]), in, k_row);
                const char* vp = step_to(step_to(vbase, page, (uint32_t)a.v_st[1]), in, v_row);
                const char* kf = step_to(step_to(ksbase, page, (uint32_t)a.ks_st[1]), in, ks_row);
                const char* vf = step_to(step_to(vsbase, page, (uint32_t)a.vs_st[1]), in, vs_row);
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
#pragma unroll
                    for (int s = 0; s < kLoads; ++s) {
                        const bool ok = dim_of(s) < a.d;
                        const uint32_t code = ok ? code0 + s * 2 * P::kDims : 0, scale = ok ? scale0 + s * P::kDims / 8 : 0;
                        kw[h][kb][s] = *reinterpret_cast<const Codes*>(kp + code);
                        vw[h][kb][s] = *reinterpret_cast<const Codes*>(vp + code);
                        ke[h][kb][s] = reinterpret_cast<const uint8_t*>(kf)[scale];
                        ve[h][kb][s] = reinterpret_cast<const uint8_t*>(vf)[scale];
                    }
                    kp += a.k_st[2];
                    vp += a.v_st[2];
                    kf += a.ks_st[2];
                    vf += a.vs_st[2];
                }
            }
            look_up_own(ahead + 1);
        }
        ++ahead;
    };

    // the first block is on its way before the queries are waited for
    if constexpr (EVEN) {
        page_set[0] = look_up(0);
        page_set[1] = look_up(32);
    } else {
        look_up_own(0);
    }
    if (first < end) fetch(first);
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
                if constexpr (kTwo) q[s * kWords + t] = two_bf16(x, q_low[s * kWords + t]);
                else q[s * kWords + t] = x;
            }
    }

    f32x4 acc[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.f;

    for (int i = first; i < end; i += WAVES) {
        const int key0 = tiles.tile(i) * kKeys;
        asm("" : "+v"(put_at), "+v"(get_at));
        typedef __attribute__((address_space(3))) u32x4 lds16;
        typedef __attribute__((address_space(3))) s16x4 lds4;
        if constexpr (!EVEN) {
            // zeros where a key is behind the last one or its page outside the cache, and behind d
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int st = 0; st < kLoads; ++st) {
                        const bool ok = key_there[kb] && dim_of(st) < a.d;
                        ke[h][kb][st] = ok ? ke[h][kb][st] : (uint8_t)0;
                        ve[h][kb][st] = ok ? ve[h][kb][st] : (uint8_t)0;
#pragma unroll
                        for (int t = 0; t < kWords; ++t) {
                            kw[h][kb][st][t] = ok ? kw[h][kb][st][t] : 0;
                            vw[h][kb][st][t] = ok ? vw[h][kb][st][t] : 0;
                        }
                    }
        }
        uint32_t kf[HEADS][2][kLoads], vf[HEADS][2][kLoads];  // scales
        if constexpr (kScaleRows) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                uint32_t w[Scales4<DP>::kUnits];
#pragma unroll
                for (int u = 0; u < Scales4<DP>::kUnits; ++u) w[u] = rows_of[h][u];
                if constexpr (DP == 96) w[0] |= w[1] << 8 | w[2] << 16;
                if constexpr (DP == 160) {
                    w[0] |= w[1] << 8 | w[2] << 16 | w[3] << 24;
                    w[1] = w[4];
                }
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int st = 0; st < kLoads; ++st) {
                        // (of a lane's 8, 16 or 32 dims: byte dim / 32)
                        const uint32_t word = w[DP > 128 ? st : 0], byte = DP >= 128 ? quad : DP == 96 && st == 1 ? 2 : quad >> 1;
                        kf[h][kb][st] = (uint32_t)__shfl((int)word, col + 16 * kb) >> 8 * byte & 0xff;
                        vf[h][kb][st] = (uint32_t)__shfl((int)word, col + 16 * kb + 32) >> 8 * byte & 0xff;
                    }
            }
        } else {
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int st = 0; st < kLoads; ++st) {
                        kf[h][kb][st] = ke[h][kb][st];
                        vf[h][kb][st] = ve[h][kb][st];
                    }
        }
        f32x4 s[2];
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            f32x4 x[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) x[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < kLoads; ++st)
#pragma unroll
                for (int t = 0; t < kWords; ++t)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        const u32x4 w = widen4<BF16>(kw[h][kb][st][t], scale_bits(known_scale(kf[h][kb][st])));
                        x[kb] = Mma<BF16>::op16(w, q[st * kWords + t], x[kb]);
                        if constexpr (kTwo) x[kb] = Mma<BF16>::op16(w, q_low[st * kWords + t], x[kb]);
                    }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[kb][r] = h == 0 || mine == h ? x[kb][r] : s[kb][r];
        }
        // A NaN scale among the values: their codes go without, and the probabilities that are not zero become NaN.  Bits: key l % 16
        // of each half; rare.
        uint32_t nan_keys[2] = {0, 0}, top_scale = 0;
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int st = 0; st < kLoads; ++st) top_scale = max(top_scale, vf[h][kb][st]);
        const bool any_nan = __any(top_scale > kScaleMost);
        if (any_nan) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int st = 0; st < kLoads; ++st) {
                        const uint64_t of = __ballot(vf[h][kb][st] > kScaleMost);
                        nan_keys[kb] |= mine == h ? (uint32_t)(of | of >> 16 | of >> 32 | of >> 48) & 0xffffu : 0;
                        vf[h][kb][st] = vf[h][kb][st] > kScaleMost ? 0 : vf[h][kb][st];
                    }
        }
        // a head's values into LDS
        auto put = [&](int h) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int st = 0; st < kLoads; ++st) {
                    const float f = scale_bits(vf[h][kb][st]);
                    if (DP % (4 * P::kDims) == 0 || dim_of(st) < DP) {
#pragma unroll
                        for (int t = 0; t < kWords; ++t)
                            *(lds16*)(uintptr_t)((put_at ^ (st * 4 * kWords + t) << 4) + 16 * kb * Tile<DP>::kRow) = widen4<BF16>(vw[h][kb][st][t], f);
                    }
                }
            __builtin_amdgcn_wave_barrier();
        };
        put(0);
        if (HEADS == 1 && i + WAVES < end) fetch(i + WAVES);
        // (the last token sees furthest ahead, the first least; a window's near end moves with both)
        const bool all = key0 + kKeys - 1 <= first_position && key0 + kKeys <= keys &&
                         (a.window < 0 || key0 >= last_position - a.window || key0 + kKeys <= a.sinks);
        if (!all) {
            const int lo = a.window < 0 ? 0 : position - a.window, hi = min(position, keys - 1);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = key0 + 16 * kb + 4 * quad + r;
                    const bool sees = (key <= hi) & ((key >= lo) | (key < a.sinks));
                    s[kb][r] = sees ? s[kb][r] : kNegInf;
                }
        }
        float top = kNegInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) top = max3(max3(top, s[kb][0], s[kb][1]), s[kb][2], s[kb][3]);
        top = both_quads_max(top);
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
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.scale_log2, -base));
            l += (s[kb][0] + s[kb][1]) + (s[kb][2] + s[kb][3]);
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
        for (int h = 0; h < HEADS; ++h) {
            if (h > 0) put(h);
            if (HEADS > 1 && h == HEADS - 1 && i + WAVES < end) fetch(i + WAVES);
            u32x4 mine_p, mine_low;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                mine_p[e] = HEADS == 1 || mine == h ? p[e] : 0;
                mine_low[e] = HEADS == 1 || mine == h ? p_low[e] : 0;
            }
#pragma unroll
            for (int db = 0; db < DP / 16; ++db) {
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(get_at ^ (db << 5)));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)((get_at ^ (db << 5)) + 16 * Tile<DP>::kRow));
                const u32x2 u = __builtin_bit_cast(u32x2, x), v = __builtin_bit_cast(u32x2, y);
                acc[db] = Mma<BF16>::op16(u32x4{u.x, u.y, v.x, v.y}, mine_p, acc[db]);
                if constexpr (kTwo) acc[db] = Mma<BF16>::op16(u32x4{u.x, u.y, v.x, v.y}, mine_low, acc[db]);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }

    // the waves' results: rows of DP values in each wave's own LDS, joined by the whole workgroup
    l = both_halves_sum(l + __shfl_xor(l, 16));
    float* const own = reinterpret_cast<float*>(vt);
#pragma unroll
    for (int db = 0; db < DP / 16; ++db) *reinterpret_cast<f32x4*>(own + col * DP + 16 * db + 4 * quad) = acc[db];
    if (quad == 0) {
        wave_m[wave][col] = m;
        wave_l[wave][col] = l;
    }
    __syncthreads();
    for (int at = threadIdx.x * 8; at < 16 * DP; at += 64 * WAVES * 8) {
        const int c = at / DP, r = c % kColumns, dim = at % DP;
        if (r >= rows || dim >= a.d) continue;
        float high = wave_m[0][c];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) high = fmaxf(high, wave_m[w][c]);
        const float base = high == kNegInf ? 0.f : high;
        float total = 0.f, x[8] = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(wave_m[w][c] - base);
            total += wave_l[w][c] * f;
            const float* from = reinterpret_cast<const float*>(lds + w * kWaveBytes) + c * DP + dim;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] += from[e] * f;
        }
        const float inverse = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= inverse;
        const int t = a.by_group.div(row0 + r), h = (g0 + c / kColumns) * a.group + row0 + r - t * a.group;
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
