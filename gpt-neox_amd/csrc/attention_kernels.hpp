// Attention without stored scores: the device code shared by the forward kernel (training, evaluation,
// prompts over a paged cache) and the two backward kernels.
//
// One (sample, key head) at a time.  Its queries are "rows": row = token * group + head in the group, so
// that the heads that share keys share the tiles of those keys too.  All products run on the matrix cores as
// 32x32x16 tiles with the row (or, for the key gradients, the key) in the column of the result: lane l then
// holds the results of column l % 32, sixteen of the 32 along the other axis, and the maximum and sum of a
// softmax row stay within a lane and its partner l ^ 32.
//   forward:   S^T = K Q^T;  O^T  += V^T P^T
//   queries:   S^T = K Q^T;  dP^T = V dO^T;  dQ^T += K^T dS^T
//   keys:      S   = Q K^T;  dP   = dO V^T;  dV^T += dO^T P;  dK^T += Q^T dS
// The result of the first product of each chain is the second operand of the last without a move: result
// register 8 t + e of a lane is what k-slot e of step t takes, if the other operand numbers its k-slots by
// element key_of(t, half, e) -- two transposing LDS reads of four consecutive elements each.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave.hpp"

namespace neox {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();
constexpr int kTileRows = 128;  // rows of a workgroup of the forward and the query-gradient kernel: 32 for each of its four waves
constexpr int kTileKeys = 64;   // keys of one step of the query-gradient kernel
constexpr int kStepRows = 32;   // rows of one step of the key-gradient kernel
constexpr int kGradKeys = 128;  // keys of a workgroup there: 32 for each of its four waves

// p + i * bytes in one instruction (strides are below 2^31 elements, which the entry points see to)
__device__ __forceinline__ const char* step_to(const char* p, uint32_t i, uint32_t bytes) { return p + (uint64_t)i * bytes; }

// where keys and values come from
enum KvSource { kStrided = 0, kPaged16 = 1, kPagedI8 = 2, kPagedF8 = 3 };

struct AttnArgs {
    const char *q, *k, *v;       // 16-bit elements (k, v: 8-bit codes for the last two sources)
    char* o;
    char* o_low;                 // null, or what rounding the output to 16 bits took away, laid out like the output
    float* lse;                  // log2 of every row's sum of exponentials, less gradient_bits(), +inf for an empty row; [b, kv, rows]
    const float *k_scale, *v_scale;
    // element strides.  q, o: token, sample (strided only), head.  k, v: token, sample, head; for pages the token
    // stride within a page, the page stride and the head stride
    int64_t q_st[3], o_st[3], k_st[3], v_st[3];
    int64_t ks_st[3], vs_st[3];  // the scales': token within a page, page, head
    const int32_t* lengths;      // keys of every sample (null, strided only: all of them)
    const int32_t* starts;       // paged: first token of every sequence in q, and the end
    const int32_t* table;        // paged: [b, table_stride] page numbers
    int64_t table_stride;
    int table_keys;              // keys that a row of the table can name
    int64_t pages;
    int tokens;                  // paged: rows of q
    float scale_log2;            // |scale| * log2(e)
    uint32_t flip;               // 0x80008000: the queries change sign on their way in (a negative scale)
    int d, kv, group;
    int sq, sk;                  // strided: queries and keys of a sample; paged: the most new tokens of a sequence
    int b;
    int window;                  // < 0: none
    int sinks;
    int row_tiles;               // of the longest sample
    int splits;                  // parts of the key axis; with more than one, o and lse are partial results:
    float* part_o;               //   [split][row slot][d] and
    float* part_lse;             //   [split][row slot], row slot = (token * kv + key head) * group + head in the group
    int64_t part_rows;           //   row slots of one split
    FastDiv by_group, by_page, by_row_tiles, by_kv, by_splits;
    // backward
    const char *dout;            // [token, sample, head] like q
    const char* out;
    int64_t do_st[3];
    char *dq, *dk, *dv;
    int64_t dq_st[3], dk_st[3], dv_st[3];
    float* delta;                // minus the sum over d of dO * O of every row, [b, kv, rows]
    float scale;
    int key_tiles;
    // The key-gradient kernel's work: every key tile's near rows (those whose window reaches it) in up to near_parts
    // pieces of piece_rows; for the first sink_tiles tiles, the rows behind in far_parts pieces.  A tile in more than one piece
    // leaves fp32 sums in part_o, [b, kv][such a tile][piece][dk, dv][key][d]; near pieces have kGradKeys keys, far pieces
    // far_keys, which those below `sinks` are among.
    int near_parts, far_parts, sink_tiles, units;
    int far_keys;
    int piece_rows;              // of a piece of near rows
    FastDiv by_units, by_near_parts, by_far_parts;
};

// While a wave feeds the matrix cores it goes before the waves that compute exponentials (8192 tokens of 128-dim
// heads, window 4096, us: forward 510 -> 474, queries' gradient 696 -> 678).  It also keeps the compiler from moving
// work in or out, which costs the kernels that have no registers to spare: the key gradients (960 -> 1580) and codes
// (242 -> 250) go without.
__device__ __forceinline__ void matrix_first(bool on) {
    if (on) __builtin_amdgcn_s_setprio(1);
}
__device__ __forceinline__ void matrix_done(bool on) {
    if (on) __builtin_amdgcn_s_setprio(0);
}

template <typename T>
struct Mma;
template <>
struct Mma<BF16> {
    static __device__ __forceinline__ f32x16 op(const u32x4& a, const u32x4& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 op16(const u32x4& a, const u32x4& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<F16> {
    static __device__ __forceinline__ f32x16 op(const u32x4& a, const u32x4& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 op16(const u32x4& a, const u32x4& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// One head dim class: DP is the padded head dim.  A tile row in LDS has kRow bytes (a power of two), cut into
// 16-byte pieces whose order is permuted by the row number, so that both kinds of read spread over all banks:
// 16 rows at one piece (row operand), 4 rows at 4 neighbouring pieces (transposing reads of 32 dims) and 8 rows at 2 (of
// 16 dims).
template <int DP>
struct Tile {
    static constexpr int kRow = DP <= 64 ? 128 : DP <= 128 ? 256 : 512;
    static constexpr int kPieces = DP / 8;  // of a row that hold data
    static __device__ __forceinline__ uint32_t turn(uint32_t row) {
        const uint32_t low = ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
        if constexpr (kRow == 128) return ((row >> 1) & 1) << 2 | low;
        return (row & 3) << 2 | low;
    }
    static __device__ __forceinline__ uint32_t at(uint32_t row, uint32_t piece) {
        return row * kRow + ((piece ^ turn(row)) << 4);
    }
};

// Where in LDS the lanes of a wave find the operands of a tile at byte `at` of LDS.  Of the permuted address only
// an exclusive or with a constant changes from operand to operand, so two registers serve a whole tile; they are hidden
// from the compiler, which would otherwise keep an address for every operand in a register of its own.
template <int DP>
struct Operands {
    uint32_t straight, turned;
    __device__ __forceinline__ explicit Operands(uint32_t at) {
        const uint32_t lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
        straight = at + (row * Tile<DP>::kRow | (Tile<DP>::turn(row) ^ half) << 4);
        const uint32_t i = lane & 15, trow = 4 * half + (i >> 2);
        turned = at + (trow * Tile<DP>::kRow | (Tile<DP>::turn(trow) ^ (2 * ((lane >> 4) & 1) + ((i >> 1) & 1))) << 4 | (i & 1) * 8);
        asm("" : "+v"(straight), "+v"(turned));
    }
    // 32 tile rows from row0 and the 16 dims of step s, row-major: lane l has row l % 32, dims 8 (l / 32) ..
    __device__ __forceinline__ u32x4 rows(int row0, int s) const {
        typedef const __attribute__((address_space(3))) u32x4* from;
        return *(from)(uintptr_t)((straight ^ (s << 5)) + row0 * Tile<DP>::kRow);
    }
    // 32 dims from 32 * db and 16 tile rows from row0, transposed: lane l has dim l % 32 and, in slot e, row
    // row0 + 8 (e / 4) + 4 (l / 32) + e % 4.
    __device__ __forceinline__ u32x4 columns(int row0, int db) const {
        typedef __attribute__((address_space(3))) s16x4* from;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((from)(uintptr_t)((turned ^ (db << 6)) + row0 * Tile<DP>::kRow));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((from)(uintptr_t)((turned ^ (db << 6) ^ 16) + (row0 + 8) * Tile<DP>::kRow));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        return u32x4{a.x, a.y, b.x, b.y};
    }
};
__device__ __forceinline__ uint32_t lds_byte(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
// four floats at a byte of LDS (where a copy into another part of the same array may be in flight, which the compiler
// would wait for if it knew the array)
__device__ __forceinline__ f32x4 lds_floats(uint32_t at) {
    return *(const __attribute__((address_space(3))) f32x4*)(uintptr_t)at;
}

// The values of lane l and of lane l ^ 32, combined.  (The results go through integers of their own: a bit cast of
// a vector's element takes the first element, whichever is asked for.)
struct HalfPair {
    float a, b;
};
__device__ __forceinline__ HalfPair both_halves(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ float both_halves_max(float x) {
    const HalfPair p = both_halves(x);
    return fmaxf(p.a, p.b);
}
__device__ __forceinline__ float both_halves_sum(float x) {
    const HalfPair p = both_halves(x);
    return p.a + p.b;
}

// the largest of three, in one instruction.  (Written for the compiler to see: behind a matrix instruction it puts the
// wait states that a reader of the result needs only before instructions that it knows, and not before inline assembly.)
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// the largest magnitude of a lane's results
__device__ __forceinline__ float largest(const f32x16& x) {
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) top = max3(top, __builtin_fabsf(x[r]), __builtin_fabsf(x[r + 1]));
    return top;
}

// the largest of a wave's numbers, none below zero, as a scalar
__device__ __forceinline__ float wave_largest(float x) { return wave_reduce<OpMax>(x); }

// the element of a 32-long result axis that register r of a lane in this half holds
__device__ __forceinline__ int element_of(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// 8 elements at p, or zeros
__device__ __forceinline__ u32x4 load8(const char* p, bool there) {
    u32x4 z = {0, 0, 0, 0};
    return there ? *reinterpret_cast<const u32x4*>(p) : z;
}

// two values rounded to 16 bits, and what the rounding took from them, rounded too
template <typename T>
__device__ __forceinline__ uint32_t pack_with_rest(float x, float y, uint32_t& rest) {
    const uint32_t w = Elem<T>::pack(x, y);
    float a, b;
    Elem<T>::unpack(w, a, b);
    rest = Elem<T>::pack(x - a, y - b);
    return w;
}
// Writes the 32 columns' results of one wave (lane: column, registers: 32 dims per block) times f as rows of 16-bit
// elements, and with LOW at `low` what the rounding took from them.  The halves exchange registers, so that every lane
// stores 16 bytes.
template <typename T, int DP, bool LOW = false>
__device__ __forceinline__ void store_rows(char* row, const f32x16 (&acc)[DP / 32], float f, int d, bool there, char* low = nullptr) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            uint32_t w[4], rest[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = acc[b][8 * p + 2 * i] * f, y = acc[b][8 * p + 2 * i + 1] * f;
                if constexpr (LOW) w[i] = pack_with_rest<T>(x, y, rest[i]);
                else w[i] = Elem<T>::pack(x, y);
            }
            const int dim = 32 * b + 16 * p + 8 * half;
            const bool ok = there && dim < d;
            const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
            if (ok) *reinterpret_cast<u32x4*>(row + dim * 2) = u32x4{x[0], y[0], x[1], y[1]};
            if constexpr (LOW) {
                const auto u = __builtin_amdgcn_permlane32_swap(rest[0], rest[2], false, false);
                const auto v = __builtin_amdgcn_permlane32_swap(rest[1], rest[3], false, false);
                if (ok) *reinterpret_cast<u32x4*>(low + dim * 2) = u32x4{u[0], v[0], u[1], v[1]};
            }
        }
    }
}

// eight 8-bit codes as numbers
template <int SRC>
__device__ __forceinline__ void decode8(const u32x2& w, float (&f)[8]) {
    if constexpr (SRC == kPagedI8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int word = (int)(i ? w.y : w.x);
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false);
            const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
            f[4 * i] = lo[0];
            f[4 * i + 1] = lo[1];
            f[4 * i + 2] = hi[0];
            f[4 * i + 3] = hi[1];
        }
    }
}
// two 8-bit floats of a word, the lower or the upper, as 16-bit values
template <typename T>
__device__ __forceinline__ uint32_t widen2(uint32_t word, bool upper) {
    if constexpr (__is_same(T, BF16)) {
        const auto x = upper ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, false);
        return __builtin_bit_cast(uint32_t, x);
    } else {
        const auto x = upper ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, false);
        return __builtin_bit_cast(uint32_t, x);
    }
}
// eight codes as 16-bit values, exactly: no code has more than 7 bits of significand
template <typename T, int SRC>
__device__ __forceinline__ u32x4 widen8(const u32x2& w) {
    if constexpr (SRC == kPagedF8) {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = widen2<T>(i < 2 ? w.x : w.y, i & 1);
        return x;
    }
    float f[8];
    decode8<SRC>(w, f);
    return pack8<T>(f);
}

// Where a probability is multiplied by its value's scale before it is rounded to fp16, the product can be anything: scales
// are the values' own size, over the largest code, and the largest of them may belong to keys that are hardly looked at.
// The accumulators of a row therefore hold their sums times a power of two of the row's own, which brings the largest
// product so far to 2^10 .. 2^15: what is then below fp16's normal numbers is less than 2^-24 of it.  bf16 has the
// range of fp32, and goes without.  4 x 512 tokens over 8192 keys, 32 heads on 8, window 4096, us without it and with: int8 64
// dims 169, 177, 128 dims 223, 230, 256 dims 647, 713; 64 single tokens over 4096: as before, within 1 %.
struct Lift {
    static constexpr uint32_t kField = 0x7f800000u;  // the exponent of a float
    float times = 0x1p60f;                           // the most, for rows whose products are all zero as yet
    static __device__ __forceinline__ uint32_t bits(float x) { return __builtin_bit_cast(uint32_t, x); }
    static __device__ __forceinline__ float power(uint32_t field) { return __builtin_bit_cast(float, field); }
    static __device__ __forceinline__ float inverse(float p) { return power((254u << 23) - bits(p)); }  // of a power of two
    __device__ __forceinline__ bool short_of(float most) const { return most * times > 0x1p15f; }
    // The running maximum has moved and the sums are to be multiplied by f <= 1, as the products that are behind them
    // are: the power may rise by as much.  Returns the sums' factor.
    __device__ __forceinline__ float follow(float f) {
        const uint32_t room = (126u << 23) - min(bits(f) & kField, 126u << 23);  // 1 / f, rounded down, without its bias
        const float before = times;
        times = power(min(bits(times) + room, bits(0x1p60f)));
        return f * (times * inverse(before));
    }
    // The power for products up to `most`, no larger than the present one.  Returns the sums' factor.
    __device__ __forceinline__ float lower(float most) {
        const float before = times;
        times = power(min(bits(times), (264u << 23) - max(bits(most) & kField, 77u << 23)));
        return times * inverse(before);
    }
    // The same where `most` has been multiplied by the power already.
    __device__ __forceinline__ float lower_by(float most) {
        const float f = power(min(127u << 23, (264u << 23) - max(bits(most) & kField, 77u << 23)));
        times *= f;
        return f;
    }
    __device__ __forceinline__ float undone() const { return inverse(times); }
    __device__ __forceinline__ float log2() const { return (float)((int)(bits(times) >> 23) - 127); }
};

// Probabilities that meet 16-bit values are rounded to the type as they are: up to 2^8, which is what the running maximum
// may lag behind.  In fp16 they are 2^7 times that, so that one is a subnormal number only 2^-21 below the largest.
template <typename T, bool CODES>
constexpr float probability_bits() { return __is_same(T, F16) && !CODES ? 7.f : 0.f; }
// The backward pass knows the rows' sums, so that no probability is above one: in fp16 it takes 2^14 times each.  The
// forward pass leaves the rows' logarithms less by as much.
template <typename T>
constexpr float gradient_bits() { return __is_same(T, F16) ? 14.f : 0.f; }

// The tiles of keys that rows with positions first .. last look at: some at the front for the sinks, then those of
// the window.
struct KeyTiles {
    int front, from, count;
    __device__ __forceinline__ int tile(int i) const { return i < front ? i : from + (i - front); }
};
template <int TILE>
__device__ __forceinline__ KeyTiles key_tiles(int first, int last, int keys, int window, int sinks) {
    const int end = min(last + 1, keys);
    if (end <= 0) return {0, 0, 0};
    int lo = window < 0 ? 0 : max(0, first - window);
    lo = min(lo, end);
    const int from = lo / TILE, to = (end + TILE - 1) / TILE;
    const int front = min((min(sinks, end) + TILE - 1) / TILE, from);
    return {front, from, front + max(0, to - from)};
}

// One sequence of a paged call.  What the device's tables say is kept inside what the tensors hold.
__device__ __forceinline__ void paged_sample(const AttnArgs& a, int b, int& token0, int& tokens, int& keys) {
    token0 = max(0, min(a.starts[b], a.tokens));
    tokens = max(0, min(a.starts[b + 1], a.tokens) - token0);
    tokens = min(tokens, a.sq);
    keys = max(0, min(a.lengths[b], a.table_keys));
}

// Which of the 16 keys whose scores a lane has (element_of: first + 8 (r / 4) + 4 half + r % 4) its row sees: those
// from lo to hi and, where sinks reach this far, the first ones.  One subtraction and one comparison each: an offset
// below zero is a large unsigned number.
struct Sight {
    int lo, width, front;  // front: the last of the sinks that the row sees
    __device__ __forceinline__ Sight(int position, int keys, int window, int sinks, int first, int half) {
        const int base = first + 4 * half;
        const int hi = min(position, keys - 1) - base;
        lo = window < 0 ? -base : position - window - base;
        width = hi - lo;
        if (width < 0) {  // nothing: no offset from here is small enough
            lo = 1 << 30;
            width = 0;
        }
        front = min(sinks - 1 - base, hi);
    }
    static __device__ __forceinline__ constexpr int offset(int r) { return 8 * (r >> 2) + (r & 3); }
    __device__ __forceinline__ bool window(int r) const { return (uint32_t)(offset(r) - lo) <= (uint32_t)width; }
    __device__ __forceinline__ bool any(int r) const { return window(r) | (offset(r) <= front); }
};

// ---- staging -----------------------------------------------------------------------------------------
// One tile of ROWS rows of codes on its way from memory to LDS through registers, where they become 16-bit values: 256
// threads, 8 codes at a time.  Rows behind the last key and dims behind d come as zeros: what lies there may be anything.
template <typename T, int DP, int SRC, int ROWS>
struct Stage {
    static constexpr int kRowsAtOnce = 256 / Tile<DP>::kPieces;  // DP = 96: 21, the last threads idle
    static constexpr int kSteps = (ROWS + kRowsAtOnce - 1) / kRowsAtOnce;
    u32x2 codes[kSteps];

    static __device__ __forceinline__ int row(int step) { return (int)(threadIdx.x / Tile<DP>::kPieces) + step * kRowsAtOnce; }
    static __device__ __forceinline__ int piece() { return (int)(threadIdx.x % Tile<DP>::kPieces); }
    static __device__ __forceinline__ bool works(int step) {
        return (int)threadIdx.x < kRowsAtOnce * Tile<DP>::kPieces && row(step) < ROWS;
    }

    __device__ __forceinline__ void load(int step, const char* at, bool there) {
        codes[step] = u32x2{0, 0};
        if (there) codes[step] = *reinterpret_cast<const u32x2*>(at);
    }
    __device__ __forceinline__ void put(char* tile) const {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (!works(s)) continue;
            u32x2 c = codes[s];
            asm("" : "+v"(c.x), "+v"(c.y));  // (or the compiler takes the words apart where they are loaded, and waits for them there)
            *reinterpret_cast<u32x4*>(tile + Tile<DP>::at(row(s), piece())) = widen8<T, SRC>(c);
            __builtin_amdgcn_sched_barrier(0);  // one step after the other: their values together would not fit the registers
        }
    }
};

// 16-bit rows get there without registers in between: every lane names the 16 bytes that go to its place of the
// tile (256 threads, a wave 1 KiB at a time), or writes zeros there.  The copies are in flight until landed().
template <int DP, int ROWS>
struct Flight {
    static constexpr int kSteps = ROWS * Tile<DP>::kRow / 4096;
    static_assert(kSteps * 4096 == ROWS * Tile<DP>::kRow, "whole steps");
    static constexpr int kPlaces = Tile<DP>::kRow / 16;
    uint32_t thread = threadIdx.x;
    // The compiler forgets where the thread's number came from: what follows from it is computed again for every tile
    // and not kept in registers, which the accumulators need.
    __device__ __forceinline__ void again() { asm("" : "+v"(thread)); }
    __device__ __forceinline__ uint32_t place(int step) const { return step * 256 + thread; }
    __device__ __forceinline__ int row(int step) const { return (int)(place(step) / kPlaces); }
    __device__ __forceinline__ int piece(int step) const { return (int)((place(step) % kPlaces) ^ Tile<DP>::turn(row(step))); }
    static __device__ __forceinline__ void load(int step, const char* from, char* tile) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                         (__attribute__((address_space(3))) void*)(tile + step * 4096 + wave * 1024), 16, 0, 0);
    }
    // Whole tiles of rows a fixed stride apart: the addresses are a scalar for the step and a lane's own offset, which
    // stays the same from step to step (but for the permutation, which repeats every 16 rows) and from tile to tile.
    static constexpr int kRowsAtOnce = 4096 / Tile<DP>::kRow;
    __device__ __forceinline__ uint32_t offset(uint32_t row_bytes) const { return row(0) * row_bytes + piece(0) * 16; }
    static __device__ __forceinline__ void load(int step, const char* first, uint32_t row_bytes, uint32_t offset, uint32_t piece, char* tile) {
        if constexpr (kRowsAtOnce < 16) offset += ((piece ^ (step & 1)) - piece) * 16;
        load(step, first + (uint64_t)(step * kRowsAtOnce) * row_bytes + offset, tile);
    }
    __device__ __forceinline__ void zero(int step, char* tile) const {
        *reinterpret_cast<u32x4*>(tile + place(step) * 16) = u32x4{0, 0, 0, 0};
    }
};
constexpr int64_t kSmallStride = 1 << 25;  // elements: a tile's offsets fit 32 bits
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- forward --------------------------------------------------------------------------------------------
// O = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m), x = scale log2(e) q.k over the keys that a row sees, in one pass over
// them with the running maximum m and the running sum in registers; lse = m + log2(sum).  A workgroup has 128 rows of one
// (sample, key head), 32 in each wave, and steps over the tiles of keys that any of them sees, copied into one half of LDS
// while the other is worked on.  The probabilities are rounded to the 16-bit type, as the second product takes them; what
// that costs is half an ulp of each, as where they are stored.
// Bound by the matrix cores and by the exponentials and the mask around them, about half as long: a wave does one after
// the other, and two waves of a SIMD that are at different places overlap little.  Measured (medians of 100 launches in a row), us and
// what its two products reach: 8192 tokens, 32 heads of 128 dims, window 4096 (bf16) 470, 877 TFLOP/s; 2 x 2048 tokens, 64 heads of 96
// dims, window 512 (fp16) 99, 457 TFLOP/s, of which a quarter of the columns are padding and the edges of the window are
// computed and masked.  Chunks of 512 tokens of four sequences over 16384 keys, window 4096, 32 heads on 8, fp8: 200, 513
// TFLOP/s, the widening of codes being work of its own.
// Over codes at 256 dims the fp16 kernels spill 6 to 11 registers.
template <typename T, int DP, int SRC, bool SPLIT>
__global__ __launch_bounds__(256, DP <= 128 ? (SRC == kStrided || SRC == kPaged16 ? 3 : 2) : 1) void attn_fwd_kernel(AttnArgs a) {
    constexpr bool kPages = SRC != kStrided;
    constexpr bool kCodes = SRC == kPagedI8 || SRC == kPagedF8;
    constexpr int kBytes = kCodes ? 1 : 2;
    // Keys of one step.  32 leave registers and LDS for a third workgroup on a CU (measured with 64 and 32, us: 2 x 64
    // heads of 96 dims, 2048 keys, window 512: 126, 105; 32 heads of 128 dims, 8192 keys, window 4096: 562, 539); with
    // codes, whose widening takes the registers anyway, 64 save barriers (chunks of 512 over 16384 in fp8: 251, 275).
    constexpr int kFwdKeys = kCodes ? 64 : 32;
    constexpr int kTile = kFwdKeys * Tile<DP>::kRow;
    __shared__ __attribute__((aligned(512))) char lds[2 * 2 * kTile + (kCodes ? 2 * 2 * kFwdKeys * 4 : 0)];

    // block -> (sample, key head), row tile, part: neighbours in time on one XCD (blocks go to the 8 XCDs in
    // turn) are the row tiles of one key head, whose keys they share
    uint32_t block = blockIdx.x;
    const uint32_t split = SPLIT ? blockIdx.y : 0;
    const uint32_t heads = a.b * a.kv;
    uint32_t bh, mt;
    if (heads % 8 == 0) {
        const uint32_t xcd = block & 7, k = block >> 3;
        const uint32_t part = a.by_row_tiles.div(k);
        bh = part * 8 + xcd;
        mt = k - part * a.row_tiles;
    } else {
        bh = a.by_row_tiles.div(block);
        mt = block - bh * a.row_tiles;
    }
    mt = a.row_tiles - 1 - mt;  // the later rows, which see most keys, first
    const int b = a.by_kv.div(bh), g = bh - b * a.kv;

    int token0 = 0, tokens = a.sq, keys = a.sk, position0 = a.sk - a.sq;
    if constexpr (kPages) {
        paged_sample(a, b, token0, tokens, keys);
        position0 = keys - tokens;
    } else if (a.lengths) {
        keys = max(0, min(a.lengths[b], a.sk));
    }
    const int rows = tokens * a.group, row0 = mt * kTileRows;
    if (row0 >= rows) return;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5;
    const int row = row0 + wave * 32 + (lane & 31);
    const bool there = row < rows;
    const int token = a.by_group.div(min(row, rows - 1)), head = g * a.group + (min(row, rows - 1) - token * a.group);
    const int position = position0 + token;
    // positions of the workgroup's and of the wave's rows
    const int wg_first = position0 + (int)a.by_group.div(row0), wg_last = position0 + (int)a.by_group.div(min(row0 + kTileRows, rows) - 1);
    const int wave_row0 = min(row0 + wave * 32, rows - 1);
    const int wv_first = __builtin_amdgcn_readfirstlane(position0 + (int)a.by_group.div(wave_row0));
    const int wv_last = __builtin_amdgcn_readfirstlane(position0 + (int)a.by_group.div(min(row0 + wave * 32 + 32, rows) - 1));
    const bool wave_works = row0 + wave * 32 < rows;

    KeyTiles tiles = key_tiles<kFwdKeys>(wg_first, wg_last, keys, a.window, a.sinks);
    int first_tile = 0, end_tile = tiles.count;
    if constexpr (SPLIT) {
        const int each = (tiles.count + a.splits - 1) / a.splits;
        first_tile = min((int)split * each, tiles.count);
        end_tile = min(first_tile + each, tiles.count);
    }

    // One tile of keys and values into one of the buffers: 16-bit rows are copied there as they are; codes come through
    // registers and are widened on the way, which put() does when the tile's turn is near.
    typedef Stage<T, DP, kCodes ? SRC : kPagedI8, kFwdKeys> St;
    typedef Flight<DP, kFwdKeys> Fl;
    Fl fl;
    constexpr int kSteps = kCodes ? St::kSteps : Fl::kSteps;
    St ks, vs;
    auto row_of = [&](int s) { return kCodes ? St::row(s) : fl.row(s); };
    int page_of[kPages ? kSteps : 1];   // the pages of the next tile's rows, looked up one step ahead
    int page_at = -1;                   // the same for the scale that this thread fetches
    const int32_t* table = kPages ? a.table + (int64_t)b * a.table_stride : nullptr;
    // Whether whole tiles have their rows a fixed stride apart (for pages: a page holds whole tiles), and this lane's
    // part in that.  Its places beyond d are zeros from the start and stay so.
    const bool even = !kCodes && a.k_st[0] < kSmallStride && a.v_st[0] < kSmallStride && (!kPages || a.by_page.d % kFwdKeys == 0) &&
                      (Fl::kRowsAtOnce >= 16 || a.d == DP);
    const uint32_t k_row = (uint32_t)a.k_st[0] * 2, v_row = (uint32_t)a.v_st[0] * 2;
    const uint32_t k_offset = fl.offset(k_row), v_offset = fl.offset(v_row), lane_piece = fl.piece(0);
    const bool has_dims = (int)lane_piece * 8 < a.d;
    if (even && !has_dims) {
#pragma unroll
        for (int s = 0; s < 2 * 2 * Fl::kSteps; ++s) fl.zero(s, lds);
    }
    uint32_t tile_page = 0;
    auto look_up = [&](int tile) {
        if constexpr (kPages) {
            if (even) {
                const int key = tile * kFwdKeys;
                tile_page = key < keys ? __builtin_amdgcn_readfirstlane(table[a.by_page.div(key)]) : ~0u;
                return;
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int key = tile * kFwdKeys + row_of(s);
                page_of[s] = key < keys ? table[a.by_page.div(key)] : -1;
            }
            if constexpr (kCodes) {
                const int key = tile * kFwdKeys + lane;
                page_at = (wave < 2 && key < keys) ? table[a.by_page.div(key)] : -1;
            }
        }
    };
    const char* const kbase = a.k + ((kPages ? 0 : (int64_t)b * a.k_st[1]) + (int64_t)g * a.k_st[2]) * kBytes;
    const char* const vbase = a.v + ((kPages ? 0 : (int64_t)b * a.v_st[1]) + (int64_t)g * a.v_st[2]) * kBytes;
    float scale_of_key = 0.f;  // waves 0 and 1: the scales of the tile's keys and of its values
    auto fetch = [&](int tile, int buffer) {
        char* const kt = lds + buffer * 2 * kTile;
        if constexpr (!kCodes) {
            const int key = tile * kFwdKeys;
            if (even && key + kFwdKeys <= keys && (!kPages || tile_page < (uint32_t)a.pages)) {
                const char *kp = kbase, *vp = vbase;
                uint32_t first = key;
                if constexpr (kPages) {
                    kp = step_to(kp, tile_page, (uint32_t)a.k_st[1] * 2);
                    vp = step_to(vp, tile_page, (uint32_t)a.v_st[1] * 2);
                    first = a.by_page.mod(key);
                }
                kp = step_to(kp, first, k_row);
                vp = step_to(vp, first, v_row);
                if (has_dims) {
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) {
                        Fl::load(s, kp, k_row, k_offset, lane_piece, kt);
                        Fl::load(s, vp, v_row, v_offset, lane_piece, kt + kTile);
                    }
                }
                return;
            }
        }
        fl.again();
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int key = tile * kFwdKeys + row_of(s), piece = kCodes ? St::piece() : fl.piece(s);
            bool ok = key < keys && piece * 8 < a.d;
            const char *kp = kbase + piece * 8 * kBytes, *vp = vbase + piece * 8 * kBytes;
            if constexpr (kPages) {
                const uint32_t page = even ? tile_page : page_of[s], in = a.by_page.mod(key);
                ok = ok && page < (uint32_t)a.pages;
                kp = step_to(step_to(kp, page, (uint32_t)a.k_st[1] * kBytes), in, (uint32_t)a.k_st[0] * kBytes);
                vp = step_to(step_to(vp, page, (uint32_t)a.v_st[1] * kBytes), in, (uint32_t)a.v_st[0] * kBytes);
            } else {
                kp = step_to(kp, key, (uint32_t)a.k_st[0] * 2);
                vp = step_to(vp, key, (uint32_t)a.v_st[0] * 2);
            }
            if constexpr (kCodes) {
                ks.load(s, kp, ok && St::works(s));
                vs.load(s, vp, ok && St::works(s));
            } else if (ok) {
                Fl::load(s, kp, kt);
                Fl::load(s, vp, kt + kTile);
            } else {
                fl.zero(s, kt);
                fl.zero(s, kt + kTile);
            }
        }
        if constexpr (kCodes) {
            scale_of_key = 0.f;
            if (wave < 2 && (uint32_t)page_at < (uint32_t)a.pages) {
                const int64_t in = a.by_page.mod(tile * kFwdKeys + lane);
                if (wave) scale_of_key = a.v_scale[page_at * a.vs_st[1] + in * a.vs_st[0] + (int64_t)g * a.vs_st[2]];
                else scale_of_key = a.k_scale[page_at * a.ks_st[1] + in * a.ks_st[0] + (int64_t)g * a.ks_st[2]];
            }
        }
    };
    float* const scales = reinterpret_cast<float*>(lds + 2 * 2 * kTile);  // [buffer][keys, values][64]
    auto put = [&](int buffer) {
        if constexpr (kCodes) {
            ks.put(lds + buffer * 2 * kTile);
            vs.put(lds + buffer * 2 * kTile + kTile);
            if (wave < 2) scales[(buffer * 2 + wave) * kFwdKeys + lane] = scale_of_key;
        } else {
            landed();
        }
    };

    f32x16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    float m = kNegInf, l = 0.f;
    constexpr bool kLifted = kCodes && __is_same(T, F16);
    constexpr float kBits = probability_bits<T, kCodes>();
    Lift lift;

    // the first tile is on its way before the queries are waited for
    if (first_tile < end_tile) {
        look_up(tiles.tile(first_tile));
        fetch(tiles.tile(first_tile), 0);
        if (first_tile + 1 < end_tile) look_up(tiles.tile(first_tile + 1));
    }

    // queries, the second operand of the scores
    u32x4 q[DP / 16];
    {
        const char* p = a.q + ((int64_t)(token0 + token) * a.q_st[0] + (kPages ? 0 : (int64_t)b * a.q_st[1]) + (int64_t)head * a.q_st[2]) * 2;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int dim = 16 * s + 8 * half;
            q[s] = load8(p + dim * 2, there && dim < a.d);
            q[s] ^= a.flip;
        }
    }

    if (first_tile < end_tile) put(0);
    __syncthreads();

    for (int it = first_tile; it < end_tile; ++it) {
        const int buffer = (it - first_tile) & 1, next = buffer ^ 1;
        const Operands<DP> kt_ops(lds_byte(lds) + buffer * 2 * kTile), vt_ops(lds_byte(lds) + buffer * 2 * kTile + kTile);
        const int key0 = tiles.tile(it) * kFwdKeys;
        if (it + 1 < end_tile) {
            fetch(tiles.tile(it + 1), next);
            if (it + 2 < end_tile) look_up(tiles.tile(it + 2));
        }
        // what of the tile this wave's rows see: nothing, all, or some of it
        const int key_end = key0 + kFwdKeys;
        const bool none = !wave_works || key0 > wv_last || key0 >= keys ||
                          (a.window >= 0 && key_end - 1 < wv_first - a.window && key0 >= a.sinks);
        const bool all = key_end - 1 <= wv_first && key_end <= keys &&
                         (a.window < 0 || key0 >= wv_last - a.window || key_end <= a.sinks);
        if (!none) {
            f32x16 s[kFwdKeys / 32];
#pragma unroll
            for (int kb = 0; kb < kFwdKeys / 32; ++kb) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
                matrix_first(!kCodes);
#pragma unroll
                for (int st = 0; st < DP / 16; ++st) s[kb] = Mma<T>::op(kt_ops.rows(32 * kb, st), q[st], s[kb]);
                matrix_done(!kCodes);
            }
            if constexpr (kCodes) {
                const float* f = scales + buffer * 2 * kFwdKeys;
#pragma unroll
                for (int kb = 0; kb < kFwdKeys / 32; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f32x4 c = *reinterpret_cast<const f32x4*>(f + 32 * kb + 8 * (r >> 2) + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kb][r + i] *= c[i];
                    }
            }
            if (!all) {
#pragma unroll
                for (int kb = 0; kb < kFwdKeys / 32; ++kb) {
                    const Sight sight(position, keys, a.window, a.sinks, key0 + 32 * kb, half);
                    if (key0 < a.sinks) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[kb][r] = sight.any(r) ? s[kb][r] : kNegInf;
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[kb][r] = sight.window(r) ? s[kb][r] : kNegInf;
                    }
                }
            }
            float top = kNegInf;
#pragma unroll
            for (int kb = 0; kb < kFwdKeys / 32; ++kb)
#pragma unroll
                for (int r = 0; r < 16; r += 2) top = max3(top, s[kb][r], s[kb][r + 1]);
            top = both_halves_max(top) * a.scale_log2;
            // The running maximum follows only where a row has outgrown it by 2^8: until then its exponentials stay
            // below 256 and the accumulators need no rescaling.
            if (__any(top > m + 8.f)) {
                const float higher = fmaxf(m, top);
                float f = __builtin_amdgcn_exp2f(m - (higher == kNegInf ? 0.f : higher));
                m = higher;
                l *= f;
                if constexpr (kLifted) f = lift.follow(f);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][r] *= f;
            }
            const float base = (m == kNegInf ? 0.f : m) - kBits;
            float sum = 0.f;
#pragma unroll
            for (int kb = 0; kb < kFwdKeys / 32; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.scale_log2, -base));
                    sum += s[kb][r];
                }
            l += sum;
            if (kCodes && !all) {  // a hidden value's scale may be anything
#pragma unroll
                for (int kb = 0; kb < kFwdKeys / 32; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f32x4 c = *reinterpret_cast<const f32x4*>(scales + (buffer * 2 + 1) * kFwdKeys + 32 * kb + 2 * r + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kb][r + i] = s[kb][r + i] != 0.f ? s[kb][r + i] * c[i] : 0.f;
                    }
            } else if constexpr (kCodes) {
                const float* f = scales + (buffer * 2 + 1) * kFwdKeys;
#pragma unroll
                for (int kb = 0; kb < kFwdKeys / 32; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f32x4 c = *reinterpret_cast<const f32x4*>(f + 32 * kb + 8 * (r >> 2) + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kb][r + i] *= c[i];
                    }
            }
            if constexpr (kLifted) {
                float most = 0.f;
#pragma unroll
                for (int kb = 0; kb < kFwdKeys / 32; ++kb) most = fmaxf(most, largest(s[kb]));
                most = both_halves_max(most);
                if (__any(lift.short_of(most))) {
                    const float f = lift.lower(most);
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
                }
#pragma unroll
                for (int kb = 0; kb < kFwdKeys / 32; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] *= lift.times;
            }
#pragma unroll
            for (int t = 0; t < kFwdKeys / 16; ++t) {
                u32x4 p;
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = Elem<T>::pack(s[t >> 1][8 * (t & 1) + 2 * e], s[t >> 1][8 * (t & 1) + 2 * e + 1]);
                matrix_first(!kCodes);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) acc[i] = Mma<T>::op(vt_ops.columns(16 * t, i), p, acc[i]);
                matrix_done(!kCodes);
            }
        }
        if (it + 1 < end_tile) put(next);
        __syncthreads();
    }

    const float total = both_halves_sum(l);
    float inverse = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);  // (a NaN stays one)
    if constexpr (kLifted) inverse *= lift.undone();
    if constexpr (SPLIT) {
        const int64_t slot = (int64_t)split * a.part_rows + ((int64_t)(token0 + token) * a.kv + g) * a.group + (head - g * a.group);
        float* p = a.part_o + slot * a.d;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int dim = 32 * i + element_of(r, half);
                const f32x4 x = {acc[i][r] * inverse, acc[i][r + 1] * inverse, acc[i][r + 2] * inverse, acc[i][r + 3] * inverse};
                if (there && dim < a.d) *reinterpret_cast<f32x4*>(p + dim) = x;
            }
        if (there && half == 0) a.part_lse[slot] = total == 0.f ? kNegInf : m - kBits + __builtin_amdgcn_logf(total);
    } else {
        const int64_t at = ((int64_t)(token0 + token) * a.o_st[0] + (kPages ? 0 : (int64_t)b * a.o_st[1]) + (int64_t)head * a.o_st[2]) * 2;
        if (!kPages && a.o_low) store_rows<T, DP, true>(a.o + at, acc, inverse, a.d, there, a.o_low + at);
        else store_rows<T, DP>(a.o + at, acc, inverse, a.d, there);
        if (!kPages && a.lse && there && half == 0)
            a.lse[(int64_t)bh * rows + row] = total == 0.f ? __builtin_inff() : m - kBits + __builtin_amdgcn_logf(total) - gradient_bits<T>();
    }
}

// ---- single tokens ----------------------------------------------------------------------------------------
// At most 16 rows per key head: the bytes of the keys and values bound it, so every wave streams keys of its own,
// 32 at a time, with no barrier before the end.  16x16x32 tiles.  A lane fetches, of keys l % 16 and 16 + l % 16, the
// 16-byte pieces that go into its first operands as they are (16-bit: 8 dims from 32 s + 8 (l / 16); codes: 16 dims from
// 64 s + 16 (l / 16)); the same pieces of the values go through LDS of the wave's own for the transposing reads.
// Measured, 32 heads on 8 of 128 dims: one token of each of 64 sequences of 2048 to 8192 keys, int8, 158 us, 4.4 TB/s, in
// 4096 workgroups of unequal length; one token over 131001 keys in bf16, 112 us, 4.8 TB/s (a copy of large tensors reaches
// 4.9, and a kernel that does nothing but read such rows 5.3 to 5.7).  At 256 dims over 16-bit pages two blocks of keys and
// values do not fit beside the sums: 35 registers are spilled inside the loop (one sequence of 65536 keys on 8 key heads 144 us, 3.7 TB/s).
template <typename T, int DP, int SRC, bool SPLIT>
__global__ __launch_bounds__(256, DP <= 128 ? 3 : 2) void attn_token_kernel(AttnArgs a) {
    constexpr bool kCodes = SRC == kPagedI8 || SRC == kPagedF8;
    constexpr int kBytes = kCodes ? 1 : 2;
    constexpr int kKeys = 32;
    constexpr int kLoads = kCodes ? (DP + 63) / 64 : DP / 32;  // 16-byte pieces of one key per lane
    constexpr int kWaveBytes = kKeys * Tile<DP>::kRow;
    __shared__ __attribute__((aligned(512))) char lds[4 * kWaveBytes];
    __shared__ __attribute__((aligned(16))) float scales[4][2][kKeys];
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

    // dim of the first element of step s's (first half of the) operand
    auto dim_of = [&](int s) { return kCodes ? 64 * s + 16 * quad : 32 * s + 8 * quad; };
    u32x4 q[kCodes ? 2 * kLoads : kLoads];
    {
        const char* p = a.q + ((int64_t)(token0 + token) * a.q_st[0] + (int64_t)head * a.q_st[2]) * 2;
#pragma unroll
        for (int s = 0; s < kLoads; ++s) {
#pragma unroll
            for (int t = 0; t < (kCodes ? 2 : 1); ++t) {
                const int dim = dim_of(s) + 8 * t;
                u32x4 x = load8(p + dim * 2, there && dim < a.d);
                x ^= a.flip;
                q[kCodes ? 2 * s + t : s] = x;
            }
        }
    }

    char* const vt = lds + wave * kWaveBytes;
    // Where this lane's pieces of the values go, and where the transposing reads find dims 16 db + l % 16 of keys
    // 4 (l / 16) ..: as in Operands, an exclusive or with a constant away from one register each.
    uint32_t put_at, get_at;
    {
        put_at = lds_byte(vt) + (col * Tile<DP>::kRow | (Tile<DP>::turn(col) ^ (kCodes ? 2 * quad : quad)) << 4);
        const uint32_t j = col, r = 4 * quad + (j >> 2);
        get_at = lds_byte(vt) + (r * Tile<DP>::kRow | (Tile<DP>::turn(r) ^ ((j >> 1) & 1)) << 4 | (j & 1) * 8);
    }
    const int32_t* const table = a.table + (int64_t)b * a.table_stride;
    u32x4 kw[2][kLoads], vw[2][kLoads];
    float k_scale = 0.f, v_scale = 0.f;
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
    const uint32_t k_row = (uint32_t)a.k_st[0] * kBytes, v_row = (uint32_t)a.v_st[0] * kBytes;
    const char* const kbase = a.k + (int64_t)g * a.k_st[2] * kBytes;
    const char* const vbase = a.v + (int64_t)g * a.v_st[2] * kBytes;
    const uint32_t k_offset = col * k_row + dim_of(0) * kBytes, v_offset = col * v_row + dim_of(0) * kBytes;
    auto fetch = [&](int i) {
        const int key0 = tiles.tile(i) * kKeys;
        if (even && key0 + kKeys <= keys && block_page < (uint32_t)a.pages) {
            const uint32_t in = a.by_page.mod(key0);
            const char* const kp = step_to(step_to(kbase, block_page, (uint32_t)a.k_st[1] * kBytes), in, k_row);
            const char* const vp = step_to(step_to(vbase, block_page, (uint32_t)a.v_st[1] * kBytes), in, v_row);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int s = 0; s < kLoads; ++s) {
                    kw[kb][s] = load8(kp + (uint64_t)(16 * kb) * k_row + s * 64 + k_offset, dim_of(s) < a.d);
                    vw[kb][s] = load8(vp + (uint64_t)(16 * kb) * v_row + s * 64 + v_offset, dim_of(s) < a.d);
                }
            if constexpr (kCodes) {
                if (quad < 2) {
                    const float* const kf = a.k_scale + ((int64_t)block_page * a.ks_st[1] + (int64_t)in * a.ks_st[0] + (int64_t)g * a.ks_st[2]);
                    const float* const vf = a.v_scale + ((int64_t)block_page * a.vs_st[1] + (int64_t)in * a.vs_st[0] + (int64_t)g * a.vs_st[2]);
                    k_scale = kf[(uint32_t)lane * (uint32_t)a.ks_st[0]];
                    v_scale = vf[(uint32_t)lane * (uint32_t)a.vs_st[0]];
                }
            }
            return;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int key = key0 + 16 * kb + col;
            const uint32_t page = even ? block_page : pages[kb], in = a.by_page.mod(key);
            const bool ok = key < keys && page < (uint32_t)a.pages;
            const char* const kp = step_to(step_to(kbase, page, (uint32_t)a.k_st[1] * kBytes), in, k_row) + dim_of(0) * kBytes;
            const char* const vp = step_to(step_to(vbase, page, (uint32_t)a.v_st[1] * kBytes), in, v_row) + dim_of(0) * kBytes;
#pragma unroll
            for (int s = 0; s < kLoads; ++s) {
                kw[kb][s] = load8(kp + s * 64, ok && dim_of(s) < a.d);
                vw[kb][s] = load8(vp + s * 64, ok && dim_of(s) < a.d);
            }
            if constexpr (kCodes) {
                if (quad == kb) {
                    k_scale = ok ? a.k_scale[(int64_t)page * a.ks_st[1] + (int64_t)in * a.ks_st[0] + (int64_t)g * a.ks_st[2]] : 0.f;
                    v_scale = ok ? a.v_scale[(int64_t)page * a.vs_st[1] + (int64_t)in * a.vs_st[0] + (int64_t)g * a.vs_st[2]] : 0.f;
                }
            }
        }
    };

    f32x4 acc[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.f;
    constexpr bool kLifted = kCodes && __is_same(T, F16);
    constexpr float kBits = probability_bits<T, kCodes>();
    Lift lift;

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
                if constexpr (kCodes) {
                    s[kb] = Mma<T>::op16(widen8<T, SRC>(u32x2{kw[kb][st].x, kw[kb][st].y}), q[2 * st], s[kb]);
                    s[kb] = Mma<T>::op16(widen8<T, SRC>(u32x2{kw[kb][st].z, kw[kb][st].w}), q[2 * st + 1], s[kb]);
                } else {
                    s[kb] = Mma<T>::op16(kw[kb][st], q[st], s[kb]);
                }
            }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int st = 0; st < kLoads; ++st) {
                const u32x4 w = vw[kb][st];
                if constexpr (kCodes) {
                    if (DP % 64 == 0 || dim_of(st) < DP) {
                        *(lds16*)(uintptr_t)((put_at ^ (st << 7)) + 16 * kb * Tile<DP>::kRow) = widen8<T, SRC>(u32x2{w.x, w.y});
                        *(lds16*)(uintptr_t)((put_at ^ (st << 7) ^ 16) + 16 * kb * Tile<DP>::kRow) = widen8<T, SRC>(u32x2{w.z, w.w});
                    }
                } else {
                    *(lds16*)(uintptr_t)((put_at ^ (st << 6)) + 16 * kb * Tile<DP>::kRow) = w;
                }
            }
        if constexpr (kCodes) {
            if (quad < 2) {
                scales[wave][0][lane] = k_scale;
                scales[wave][1][lane] = v_scale;
            }
        }
        if (i + 4 < end) {
            fetch(i + 4);
            look_up(i + 8);
        }
        __builtin_amdgcn_wave_barrier();
        if constexpr (kCodes) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[kb] *= *reinterpret_cast<const f32x4*>(&scales[wave][0][16 * kb + 4 * quad]);
        }
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
            float f = __builtin_amdgcn_exp2f(m - (higher == kNegInf ? 0.f : higher));
            m = higher;
            l *= f;
            if constexpr (kLifted) f = lift.follow(f);
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) acc[j] *= f;
        }
        const float base = (m == kNegInf ? 0.f : m) - kBits;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.scale_log2, -base));
                l += s[kb][r];
            }
        if constexpr (kCodes) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const f32x4 c = *reinterpret_cast<const f32x4*>(&scales[wave][1][16 * kb + 4 * quad]);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[kb][r] = s[kb][r] != 0.f ? s[kb][r] * c[r] : 0.f;  // a hidden value's scale may be anything
            }
        }
        if constexpr (kLifted) {
            float most = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 4; r += 2) most = max3(most, __builtin_fabsf(s[kb][r]), __builtin_fabsf(s[kb][r + 1]));
            most = fmaxf(most, __shfl_xor(most, 16));
            most = both_halves_max(most);
            if (__any(lift.short_of(most))) {
                const float f = lift.lower(most);
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) acc[j] *= f;
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[kb] *= lift.times;
        }
        const u32x4 p = {Elem<T>::pack(s[0][0], s[0][1]), Elem<T>::pack(s[0][2], s[0][3]),
                         Elem<T>::pack(s[1][0], s[1][1]), Elem<T>::pack(s[1][2], s[1][3])};
#pragma unroll
        for (int db = 0; db < DP / 16; ++db) {
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(get_at ^ (db << 5)));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)((get_at ^ (db << 5)) + 16 * Tile<DP>::kRow));
            const u32x2 u = __builtin_bit_cast(u32x2, x), v = __builtin_bit_cast(u32x2, y);
            acc[db] = Mma<T>::op16(u32x4{u.x, u.y, v.x, v.y}, p, acc[db]);
        }
        __builtin_amdgcn_wave_barrier();
    }

    // the four waves' results: rows of DP values in each wave's own LDS, joined by the whole workgroup
    l += __shfl_xor(l, 16);
    l = both_halves_sum(l);
    float* const mine = reinterpret_cast<float*>(vt);
#pragma unroll
    for (int db = 0; db < DP / 16; ++db) {
        if constexpr (kLifted) acc[db] *= lift.undone();
        *reinterpret_cast<f32x4*>(mine + col * DP + 16 * db + 4 * quad) = acc[db];
    }
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
            if (dim == 0) a.part_lse[slot] = total == 0.f ? kNegInf : high - kBits + __builtin_amdgcn_logf(total);
        } else {
            *reinterpret_cast<u32x4*>(a.o + ((int64_t)(token0 + t) * a.o_st[0] + (int64_t)h * a.o_st[2] + dim) * 2) = pack8<T>(x);
        }
    }
}

// Joins the parts of a split key axis: a workgroup per row, 64 threads for the dims (four each), four groups of them for
// every fourth part.  O = sum_s 2^(lse_s - m) O_s / sum_s 2^(lse_s - m), m the largest lse.  Latency: 3 to 6 us for 16 to
// 4096 rows, the launch among them.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) f32x4 sums[4][64];
    __shared__ float weights[128];
    const int64_t slot = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, dim = lane * 4;
    // every wave reduces the parts' logarithms by itself: at most 128 of them
    float lse[2], high = kNegInf;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = i * 64 + lane;
        lse[i] = s < a.splits ? a.part_lse[s * a.part_rows + slot] : kNegInf;
        high = fmaxf(high, lse[i]);
    }
    high = wave_reduce<OpMax>(high);  // (a NaN is not the largest; it reaches the total)
    const float base = high == kNegInf ? 0.f : high;
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float f = __builtin_amdgcn_exp2f(lse[i] - base);
        total += f;
        if (wave == 0) weights[i * 64 + lane] = f;
    }
    total = wave_reduce<OpSum>(total);
    __syncthreads();
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (dim < a.d) {
        const float* from = a.part_o + slot * a.d + dim;
#pragma unroll 4
        for (int s = wave; s < a.splits; s += 4) sum += *reinterpret_cast<const f32x4*>(from + s * a.part_rows * a.d) * weights[s];
    }
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave || dim >= a.d) return;
    sum = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    const float inverse = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
    const int64_t token = slot / (a.kv * a.group), head = slot - token * (a.kv * a.group);
    const u32x2 w = {Elem<T>::pack(sum[0] * inverse, sum[1] * inverse), Elem<T>::pack(sum[2] * inverse, sum[3] * inverse)};
    *reinterpret_cast<u32x2*>(a.o + (token * a.o_st[0] + head * a.o_st[2] + dim) * 2) = w;
}

// The same with a wave for each row, whose lanes hold a part's logarithm each (launched for at most 16 parts): 32 lanes for the dims up to 128 (then the halves take every other
// part), 64 above.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_rows_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63, lanes = a.d <= 128 ? 32 : 64, groups = 64 / lanes, part = lane / lanes, dim = lane % lanes * 4;
    const int64_t slot = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (slot >= a.part_rows) return;
    const float lse = lane < a.splits ? a.part_lse[lane * a.part_rows + slot] : kNegInf;
    const float high = wave_reduce<OpMax>(lse);  // (a NaN is not the largest; it reaches the total)
    const float f = __builtin_amdgcn_exp2f(lse - (high == kNegInf ? 0.f : high));
    const float total = wave_reduce<OpSum>(f);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    const float* from = a.part_o + slot * a.d + dim;
#pragma unroll 4
    for (int s0 = 0; s0 < a.splits; s0 += groups) {
        const int s = s0 + part;
        const float weight = __shfl(f, s);  // (0 behind the last part)
        if (s < a.splits && dim < a.d) sum += *reinterpret_cast<const f32x4*>(from + s * a.part_rows * a.d) * weight;
    }
    if (groups == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = both_halves_sum(sum[i]);
    }
    if (part || dim >= a.d) return;
    const float inverse = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
    const int64_t token = slot / (a.kv * a.group), head = slot - token * (a.kv * a.group);
    const u32x2 w = {Elem<T>::pack(sum[0] * inverse, sum[1] * inverse), Elem<T>::pack(sum[2] * inverse, sum[3] * inverse)};
    *reinterpret_cast<u32x2*>(a.o + (token * a.o_st[0] + head * a.o_st[2] + dim) * 2) = w;
}

// ---- backward: the queries' gradient, and the rows' sums of dO * O -----------------------------------------
// P = 2^(x - lse), dS = P (dO.v - delta), delta = sum_d dO O, dQ = scale sum_j dS_j k_j: the scores once more, row by row as
// in the forward kernel, with no maximum to keep.  Queries and dO stay in registers, delta is left for the keys' kernel.
// dS is rounded to the 16-bit type for the last product; in fp16, times a power of two that follows the largest of its row
// (Lift), since it is as small as the incoming gradient over the number of keys.  That the scores are computed here and again there (7 products for
// 5) buys gradients that are summed in registers, in a fixed order, without atomics.
// Bound by the matrix cores as the forward kernel is.  Measured: 8192 tokens, 32 heads of 128 dims, window 4096: 688 us, 900
// TFLOP/s for its three products; 8 x 1001 tokens, 16 heads of 64 dims, window 256 (fp16): 50 us.  At 256 dims the fp16 kernel spills 19
// registers.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attn_bwd_q_kernel(AttnArgs a) {
    constexpr int kTile = kTileKeys * Tile<DP>::kRow;
    __shared__ __attribute__((aligned(512))) char lds[2 * 2 * kTile];

    const uint32_t block = blockIdx.x, heads = a.b * a.kv;
    uint32_t bh, mt;
    if (heads % 8 == 0) {
        const uint32_t xcd = block & 7, k = block >> 3, part = a.by_row_tiles.div(k);
        bh = part * 8 + xcd;
        mt = k - part * a.row_tiles;
    } else {
        bh = a.by_row_tiles.div(block);
        mt = block - bh * a.row_tiles;
    }
    mt = a.row_tiles - 1 - mt;
    const int b = a.by_kv.div(bh), g = bh - b * a.kv;
    const int keys = a.lengths ? max(0, min(a.lengths[b], a.sk)) : a.sk, position0 = a.sk - a.sq;
    const int rows = a.sq * a.group, row0 = mt * kTileRows;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5;
    const int row = row0 + wave * 32 + (lane & 31);
    const bool there = row < rows;
    const int token = a.by_group.div(min(row, rows - 1)), head = g * a.group + (min(row, rows - 1) - token * a.group);
    const int position = position0 + token;
    const int wg_first = position0 + (int)a.by_group.div(row0), wg_last = position0 + (int)a.by_group.div(min(row0 + kTileRows, rows) - 1);
    const int wv_first = __builtin_amdgcn_readfirstlane(position0 + (int)a.by_group.div(min(row0 + wave * 32, rows - 1)));
    const int wv_last = __builtin_amdgcn_readfirstlane(position0 + (int)a.by_group.div(min(row0 + wave * 32 + 32, rows) - 1));
    const bool wave_works = row0 + wave * 32 < rows;
    const KeyTiles tiles = key_tiles<kTileKeys>(wg_first, wg_last, keys, a.window, a.sinks);

    typedef Flight<DP, kTileKeys> Fl;
    Fl fl;
    const char* const kbase = a.k + ((int64_t)b * a.k_st[1] + (int64_t)g * a.k_st[2]) * 2;
    const char* const vbase = a.v + ((int64_t)b * a.v_st[1] + (int64_t)g * a.v_st[2]) * 2;
    const bool even = a.k_st[0] < kSmallStride && a.v_st[0] < kSmallStride && (Fl::kRowsAtOnce >= 16 || a.d == DP);
    const uint32_t k_row = (uint32_t)a.k_st[0] * 2, v_row = (uint32_t)a.v_st[0] * 2;
    const uint32_t k_offset = fl.offset(k_row), v_offset = fl.offset(v_row), lane_piece = fl.piece(0);
    const bool has_dims = (int)lane_piece * 8 < a.d;
    if (even && !has_dims) {
#pragma unroll
        for (int s = 0; s < 4 * Fl::kSteps; ++s) fl.zero(s, lds);
    }
    auto fetch = [&](int tile, int buffer) {
        char* const kt = lds + buffer * 2 * kTile;
        if (even && tile * kTileKeys + kTileKeys <= keys) {
            const char* const kp = step_to(kbase, tile * kTileKeys, k_row);
            const char* const vp = step_to(vbase, tile * kTileKeys, v_row);
            if (has_dims) {
#pragma unroll
                for (int s = 0; s < Fl::kSteps; ++s) {
                    Fl::load(s, kp, k_row, k_offset, lane_piece, kt);
                    Fl::load(s, vp, v_row, v_offset, lane_piece, kt + kTile);
                }
            }
            return;
        }
        fl.again();
#pragma unroll
        for (int s = 0; s < Fl::kSteps; ++s) {
            const int key = tile * kTileKeys + fl.row(s), piece = fl.piece(s);
            if (key < keys && piece * 8 < a.d) {
                Fl::load(s, step_to(kbase + piece * 16, key, (uint32_t)a.k_st[0] * 2), kt);
                Fl::load(s, step_to(vbase + piece * 16, key, (uint32_t)a.v_st[0] * 2), kt + kTile);
            } else {
                fl.zero(s, kt);
                fl.zero(s, kt + kTile);
            }
        }
    };

    if (tiles.count) fetch(tiles.tile(0), 0);
    u32x4 q[DP / 16], dout[DP / 16];
    float delta = 0.f, lse = __builtin_inff();
    {
        const char* qp = a.q + ((int64_t)token * a.q_st[0] + (int64_t)b * a.q_st[1] + (int64_t)head * a.q_st[2]) * 2;
        const char* dp = a.dout + ((int64_t)token * a.do_st[0] + (int64_t)b * a.do_st[1] + (int64_t)head * a.do_st[2]) * 2;
        const int64_t o_at = ((int64_t)token * a.o_st[0] + (int64_t)b * a.o_st[1] + (int64_t)head * a.o_st[2]) * 2;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int dim = 16 * s + 8 * half;
            const bool ok = there && dim < a.d;
            q[s] = load8(qp + dim * 2, ok);
            dout[s] = load8(dp + dim * 2, ok);
            float x[8], y[8];
            unpack8<T>(dout[s], x);
            unpack8<T>(load8(a.out + o_at + dim * 2, ok), y);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(x[e], y[e], delta);
            if (a.o_low) {
                unpack8<T>(load8(a.o_low + o_at + dim * 2, ok), y);
#pragma unroll
                for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(x[e], y[e], delta);
            }
        }
        delta = both_halves_sum(delta);
        if (there) {
            lse = a.lse[(int64_t)bh * rows + row];
            if (half == 0) a.delta[(int64_t)bh * rows + row] = -delta;
        }
    }

    f32x16 minus_delta;  // where the sums of dP start: held in registers of its own, so that no tile has to set it up
#pragma unroll
    for (int r = 0; r < 16; ++r) minus_delta[r] = -delta;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    const float scale_log2 = a.scale * kLog2e;
    // fp16: dS times a power of two of the row's own, which is part of the exponent
    constexpr bool kLifted = __is_same(T, F16);
    Lift lift;
    auto lifted_lse = [&] { return kLifted ? lse + gradient_bits<T>() - lift.log2() : lse; };
    float row_lse = lifted_lse();

    landed();
    __syncthreads();
    for (int it = 0; it < tiles.count; ++it) {
        const int buffer = it & 1;
        const Operands<DP> ops(lds_byte(lds) + buffer * 2 * kTile);  // the keys' tile, and kTileKeys rows behind it the values'
        const int key0 = tiles.tile(it) * kTileKeys;
        if (it + 1 < tiles.count) fetch(tiles.tile(it + 1), buffer ^ 1);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int k0 = key0 + 32 * kb, k1 = k0 + 32;
            const bool none = !wave_works || k0 > wv_last || k0 >= keys ||
                              (a.window >= 0 && k1 - 1 < wv_first - a.window && k0 >= a.sinks);
            const bool all = k1 - 1 <= wv_first && k1 <= keys &&
                             (a.window < 0 || k0 >= wv_last - a.window || k1 <= a.sinks);
            if (none) continue;
            f32x16 s, dp = minus_delta;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
            matrix_first(true);
#pragma unroll
            for (int st = 0; st < DP / 16; ++st) s = Mma<T>::op(ops.rows(32 * kb, st), q[st], s);
            matrix_done(true);
            matrix_first(true);
#pragma unroll
            for (int st = 0; st < DP / 16; ++st) dp = Mma<T>::op(ops.rows(kTileKeys + 32 * kb, st), dout[st], dp);
            matrix_done(true);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale_log2, -row_lse)) * dp[r];
            if (!all) {
                const Sight sight(position, keys, a.window, a.sinks, k0, half);
                if (k0 < a.sinks) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = sight.any(r) ? s[r] : 0.f;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = sight.window(r) ? s[r] : 0.f;
                }
            }
            if constexpr (kLifted) {
                const float most = both_halves_max(largest(s));
                if (__any(most > 0x1p15f)) {
                    const float f = lift.lower_by(most);
                    row_lse = lifted_lse();
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] *= f;
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                u32x4 p;
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = Elem<T>::pack(s[8 * t + 2 * e], s[8 * t + 2 * e + 1]);
                matrix_first(true);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) acc[i] = Mma<T>::op(ops.columns(32 * kb + 16 * t, i), p, acc[i]);
                matrix_done(true);
            }
        }
        landed();
        __syncthreads();
    }
    char* p = a.dq + ((int64_t)token * a.dq_st[0] + (int64_t)b * a.dq_st[1] + (int64_t)head * a.dq_st[2]) * 2;
    store_rows<T, DP>(p, acc, kLifted ? a.scale * lift.undone() : a.scale, a.d, there);
}

// The partial sums of a key head, in keys: those of the tiles that are done in more than one piece.  Where near rows are in
// one piece, these are the first sink_tiles, and none without far pieces.
__host__ __device__ __forceinline__ int64_t grad_part_keys(int key_tiles, int near_parts, int sink_tiles, int far_parts, int far_keys) {
    return (int64_t)(near_parts > 1 ? key_tiles : sink_tiles) * near_parts * kGradKeys + (int64_t)sink_tiles * far_parts * far_keys;
}
// the first key of a tile's partial sums: near_parts pieces of kGradKeys, and for a tile with sinks far_parts of far_keys
__device__ __forceinline__ int64_t grad_part(const AttnArgs& a, uint32_t bh, int tile) {
    return bh * grad_part_keys(a.key_tiles, a.near_parts, a.sink_tiles, a.far_parts, a.far_keys) + (int64_t)tile * a.near_parts * kGradKeys +
           (int64_t)min(tile, a.sink_tiles) * a.far_parts * a.far_keys;
}

// The rows that see some key of a tile: those from its first position to the end of its last one's window, and where
// it holds sinks, whose rows behind are not work of their own, all.
struct KeyRows {
    int begin, end;
    __device__ __forceinline__ int pieces(const AttnArgs& a) const { return (end - begin + a.piece_rows - 1) / a.piece_rows; }
};
__device__ __forceinline__ KeyRows key_rows(const AttnArgs& a, int tile, int keys, bool far_apart) {
    const int key0 = tile * kGradKeys, position0 = a.sk - a.sq;
    if (key0 >= keys) return {0, 0};
    const int last = min(key0 + kGradKeys, keys) - 1;
    const int t0 = min(max(0, key0 - position0), a.sq);
    int t1 = a.window < 0 ? a.sq : (int)min((int64_t)a.sq, (int64_t)last + a.window - position0 + 1);
    if (key0 < a.sinks && !far_apart) t1 = a.sq;
    return {t0 * a.group, max(t0, t1) * a.group};
}

// ---- backward: the gradients of keys and values -------------------------------------------------------------
// dV_j = sum_i P_ij dO_i, dK_j = scale sum_i dS_ij q_i.  A workgroup has 128 keys of one (sample, key head), 32 in each wave,
// whose keys and values stay in registers, and steps over 32 rows at a time of all the heads that share them: the sum over
// the group is part of the same chain.  P and dS are rounded to the 16-bit type for the products, in fp16 times a power
// of two: the row's logarithm has it for P, and dS takes one that follows the largest of the wave's 32 keys, a scalar (a
// power for each key is a register more, and spilled 56 at 128 dims).  4096 tokens, 32 heads, window 1024, forward and
// backward in fp16, us, both gradients as they were and with the powers: 64 dims 276, 287, 128 dims 458, 480, 256 dims 1416, 1482.
// P is packed before dP is summed, which frees its registers.  One wave's accumulators
// are 2 x 64 registers at 128 dims, which with the operands leaves two workgroups on a CU.
// Bound by the matrix cores and the waits of a CU's few waves.  Measured: 8192 tokens, 32 heads of 128 dims, window 4096: 852
// us, 969 TFLOP/s for its four products; 4096 tokens, 32 heads on 8, window 1024: 164 us and 18 of the join.
// Head dims over 128 take two launches, one for each gradient (DK, DV): together their accumulators, keys and values
// are 384 registers of a lane, and the compiler spilled 330.  Of the two, the keys' spills 8 in bf16.
template <typename T, int DP, bool DK, bool DV>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) void attn_bwd_kv_kernel(AttnArgs a) {
    constexpr int kTile = kStepRows * Tile<DP>::kRow;
    __shared__ __attribute__((aligned(512))) char lds[2 * 2 * kTile];
    __shared__ __attribute__((aligned(16))) float row_sums[2][2][kStepRows];  // lse and delta of the tile's rows
    __shared__ __attribute__((aligned(16))) int row_at[2][kStepRows];         // and where they stand

    const uint32_t block = blockIdx.x, heads = a.b * a.kv;
    uint32_t bh, unit;
    if (heads % 8 == 0) {
        const uint32_t xcd = block & 7, k = block >> 3, part = a.by_units.div(k);
        bh = part * 8 + xcd;
        unit = k - part * a.units;
    } else {
        bh = a.by_units.div(block);
        unit = block - bh * a.units;
    }
    const int far_units = a.sink_tiles * a.far_parts;  // short, and first
    const bool far = (int)unit < far_units;
    const int kt = far ? a.by_far_parts.div(unit) : a.by_near_parts.div(unit - far_units);
    const int part = far ? unit - kt * a.far_parts : unit - far_units - kt * a.near_parts;
    const int far_of_tile = kt < a.sink_tiles ? a.far_parts : 0;
    const int b = a.by_kv.div(bh), g = bh - b * a.kv;
    const int keys = a.lengths ? max(0, min(a.lengths[b], a.sk)) : a.sk, position0 = a.sk - a.sq;
    const int rows = a.sq * a.group, key0 = kt * kGradKeys;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
    const int key = key0 + wave * 32 + (lane & 31);
    const int wv_first = __builtin_amdgcn_readfirstlane(key0 + wave * 32), wv_last = wv_first + 31;

    const KeyRows seen = key_rows(a, kt, keys, far_of_tile != 0);
    int row_begin, row_end;
    if (far) {
        const int each = ((a.sq * a.group - seen.end + kStepRows - 1) / kStepRows + a.far_parts - 1) / a.far_parts * kStepRows;
        row_begin = min(seen.end + part * each, a.sq * a.group);
        row_end = min(row_begin + each, a.sq * a.group);
        if (key0 >= keys) row_end = row_begin;
    } else {
        if (part >= seen.pieces(a) && a.near_parts + far_of_tile > 1) return;  // the join knows
        row_begin = min(seen.begin + part * a.piece_rows, seen.end);
        row_end = min(row_begin + a.piece_rows, seen.end);
    }

    typedef Flight<DP, kStepRows> Fl;
    Fl fl;
    const char* const qbase = a.q + ((int64_t)b * a.q_st[1] + (int64_t)g * a.group * a.q_st[2]) * 2;
    const char* const dbase = a.dout + ((int64_t)b * a.do_st[1] + (int64_t)g * a.group * a.do_st[2]) * 2;
    // half a wave each fetches the rows' lse and delta; rows behind the end see nothing
    // Steps begin at a token's first head where the group divides them; a lane then keeps its place in the step, as in
    // the kernels above.
    const bool even = kStepRows % a.group == 0 && (Fl::kRowsAtOnce >= 16 || a.d == DP) &&
                      a.q_st[0] < kSmallStride && a.do_st[0] < kSmallStride && a.q_st[2] < kSmallStride && a.do_st[2] < kSmallStride &&
                      (Fl::kRowsAtOnce % a.group == 0);
    if (even && fl.piece(0) * 8 >= a.d) {
#pragma unroll
        for (int s = 0; s < 4 * Fl::kSteps; ++s) fl.zero(s, lds);
    }
    const uint32_t step_tokens = even ? a.by_group.div(Fl::kRowsAtOnce) : 0;
    auto fetch_rows = [&](int row0, int buffer) {
        fl.again();
        if (even && row0 + kStepRows <= row_end) {
            const uint32_t lane_token = a.by_group.div(fl.row(0)), lane_head = fl.row(0) - lane_token * a.group, lane_piece = fl.piece(0);
            const uint32_t q_offset = (lane_token * (uint32_t)a.q_st[0] + lane_head * (uint32_t)a.q_st[2] + lane_piece * 8) * 2;
            const uint32_t d_offset = (lane_token * (uint32_t)a.do_st[0] + lane_head * (uint32_t)a.do_st[2] + lane_piece * 8) * 2;
            const uint32_t token = a.by_group.div(row0);
            const char* const qp = step_to(qbase, token, (uint32_t)a.q_st[0] * 2);
            const char* const dp = step_to(dbase, token, (uint32_t)a.do_st[0] * 2);
            if ((int)lane_piece * 8 < a.d) {
#pragma unroll
                for (int s = 0; s < Fl::kSteps; ++s) {
                    uint32_t qo = q_offset, dof = d_offset;
                    if constexpr (Fl::kRowsAtOnce < 16) {
                        const uint32_t other = ((lane_piece ^ (s & 1)) - lane_piece) * 16;
                        qo += other;
                        dof += other;
                    }
                    Fl::load(s, step_to(qp, s * step_tokens, (uint32_t)a.q_st[0] * 2) + qo, lds + buffer * 2 * kTile);
                    Fl::load(s, step_to(dp, s * step_tokens, (uint32_t)a.do_st[0] * 2) + dof, lds + buffer * 2 * kTile + kTile);
                }
            }
            return;
        }
#pragma unroll
        for (int s = 0; s < Fl::kSteps; ++s) {
            const int row = row0 + fl.row(s), piece = fl.piece(s);
            if (row < row_end && piece * 8 < a.d) {
                const uint32_t token = a.by_group.div(row), h = row - token * a.group;
                Fl::load(s, step_to(step_to(qbase + piece * 16, token, (uint32_t)a.q_st[0] * 2), h, (uint32_t)a.q_st[2] * 2),
                         lds + buffer * 2 * kTile);
                Fl::load(s, step_to(step_to(dbase + piece * 16, token, (uint32_t)a.do_st[0] * 2), h, (uint32_t)a.do_st[2] * 2),
                         lds + buffer * 2 * kTile + kTile);
            } else {
                fl.zero(s, lds + buffer * 2 * kTile);
                fl.zero(s, lds + buffer * 2 * kTile + kTile);
            }
        }
    };
    auto fetch = [&](int row0, int buffer) {
        fetch_rows(row0, buffer);
        if (wave == 0) {
            const int row = row0 + (int)(fl.thread & 31);
            const float* const sums = (fl.thread & 32 ? a.delta : a.lse) + (int64_t)bh * rows;
            if (row < row_end)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(sums + row),
                                                 (__attribute__((address_space(3))) void*)row_sums[buffer], 4, 0, 0);
            else
                row_sums[buffer][0][fl.thread] = fl.thread & 32 ? 0.f : __builtin_inff();
        } else if (wave == 1 && fl.thread < 64 + kStepRows) {
            row_at[buffer][fl.thread - 64] = position0 + (int)a.by_group.div(row0 + (int)fl.thread - 64);
        }
    };

    f32x16 dk[DP / 32], dv[DP / 32];  // (the one that is not wanted never comes to be)
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[i][r] = dv[i][r] = 0.f;
    const float scale_log2 = a.scale * kLog2e;
    // fp16: P is 2^14 times itself (as its logarithms are less), and dS that times a power of two of the wave's own
    constexpr bool kLifted = __is_same(T, F16);
    Lift lift;

    if (row_begin < row_end) fetch(row_begin, 0);
    u32x4 kreg[DP / 16], vreg[DK ? DP / 16 : 1];
    {
        const char* kp = a.k + ((int64_t)key * a.k_st[0] + (int64_t)b * a.k_st[1] + (int64_t)g * a.k_st[2]) * 2;
        const char* vp = a.v + ((int64_t)key * a.v_st[0] + (int64_t)b * a.v_st[1] + (int64_t)g * a.v_st[2]) * 2;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int dim = 16 * s + 8 * half;
            kreg[s] = load8(kp + dim * 2, key < keys && dim < a.d);
            if constexpr (DK) vreg[s] = load8(vp + dim * 2, key < keys && dim < a.d);
        }
    }

    landed();
    __syncthreads();
    int buffer = 0;
    for (int row0 = row_begin; row0 < row_end; row0 += kStepRows, buffer ^= 1) {
        const Operands<DP> ops(lds_byte(lds) + buffer * 2 * kTile);  // the queries' tile, and kStepRows rows behind it dO's
        uint32_t sums_at = lds_byte(row_sums) + buffer * 8 * kStepRows + 16 * half;
        asm("" : "+v"(sums_at));
        if (row0 + kStepRows < row_end) fetch(row0 + kStepRows, buffer ^ 1);
        const int at_first = position0 + (int)a.by_group.div(row0);
        const int at_last = position0 + (int)a.by_group.div(min(row0 + kStepRows, row_end) - 1);
        const bool none = at_last < wv_first || wv_first >= keys ||
                          (a.window >= 0 && wv_last < at_first - a.window && wv_first >= a.sinks);
        const bool all = at_first >= wv_last && wv_last < keys &&
                         (a.window < 0 || wv_first >= at_last - a.window || wv_last < a.sinks);
        if (!none) {
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
            for (int st = 0; st < DP / 16; ++st) s = Mma<T>::op(ops.rows(0, st), kreg[st], s);
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 c = lds_floats(sums_at + 32 * (r >> 2));
#pragma unroll
                for (int i = 0; i < 4; ++i) s[r + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + i], scale_log2, -c[i]));
            }
            if (!all) {
                // a row sees this lane's key from `reach` positions behind it at most; a key behind the end stands behind
                // every row
                const int mine = wv_first + (int)(fl.thread & 31), key_at = mine < keys ? mine : 1 << 30;
                const uint32_t reach = a.window < 0 || mine < a.sinks ? 0x7fffffffu : (uint32_t)a.window;
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int* at = &row_at[buffer][8 * (r >> 2) + 4 * half];
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[r + i] = (uint32_t)(at[i] - key_at) <= reach ? s[r + i] : 0.f;
                }
            }
            if constexpr (DK) {
#pragma unroll
                for (int r = 0; r < 16; r += 4) {  // dP - delta: the sum starts at -delta, which is what memory holds
                    const f32x4 c = lds_floats(sums_at + 4 * kStepRows + 32 * (r >> 2));
#pragma unroll
                    for (int i = 0; i < 4; ++i) dp[r + i] = c[i];
                }
#pragma unroll
                for (int st = 0; st < DP / 16; ++st) dp = Mma<T>::op(ops.rows(kStepRows, st), vreg[st], dp);
            }
            u32x4 prob[DV ? 2 : 1];  // P, rounded
            if constexpr (DV) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) prob[t][e] = Elem<T>::pack(s[8 * t + 2 * e], s[8 * t + 2 * e + 1]);
            }
            if constexpr (DK) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= dp[r];
                if constexpr (kLifted) {
                    const float most = largest(s);
                    if (__any(lift.short_of(most))) {
                        const float f = lift.lower(wave_largest(most));
#pragma unroll
                        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                            for (int r = 0; r < 16; ++r) dk[i][r] *= f;
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] *= lift.times;
                }
            }
            if constexpr (DV) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) dv[i] = Mma<T>::op(ops.columns(kStepRows + 16 * t, i), prob[t], dv[i]);
            }
            if constexpr (DK) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    u32x4 p;
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = Elem<T>::pack(s[8 * t + 2 * e], s[8 * t + 2 * e + 1]);
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) dk[i] = Mma<T>::op(ops.columns(16 * t, i), p, dk[i]);
                }
            }
        }
        landed();
        __syncthreads();
    }
    const float dk_times = kLifted ? lift.undone() * 0x1p-14f : 1.f, dv_times = kLifted ? 0x1p-14f : 1.f;
    static_assert(!kLifted || gradient_bits<T>() == 14.f, "2^-14");
    if (a.near_parts + far_of_tile == 1) {
        const bool there = key < a.sk;
        if constexpr (DK) store_rows<T, DP>(a.dk + ((int64_t)key * a.dk_st[0] + (int64_t)b * a.dk_st[1] + (int64_t)g * a.dk_st[2]) * 2, dk, a.scale * dk_times, a.d, there);
        if constexpr (DV) store_rows<T, DP>(a.dv + ((int64_t)key * a.dv_st[0] + (int64_t)b * a.dv_st[1] + (int64_t)g * a.dv_st[2]) * 2, dv, dv_times, a.d, there);
        return;
    }
    const int piece_keys = far ? a.far_keys : kGradKeys;
    float* const to = a.part_o + (grad_part(a, bh, kt) + (far ? a.near_parts * kGradKeys : 0) + part * piece_keys) * 2 * a.d + (key - key0) * a.d;
    if (!far || (key < a.sinks && key - key0 < a.far_keys)) {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int dim = 32 * i + element_of(r, half);
                if (dim < a.d) {
                    if constexpr (DK) *reinterpret_cast<f32x4*>(to + dim) = f32x4{dk[i][r], dk[i][r + 1], dk[i][r + 2], dk[i][r + 3]} * dk_times;
                    if constexpr (DV) *reinterpret_cast<f32x4*>(to + piece_keys * a.d + dim) = f32x4{dv[i][r], dv[i][r + 1], dv[i][r + 2], dv[i][r + 3]} * dv_times;
                }
            }
    }
}

// Sums the pieces of the key tiles that were done in several, in order: a thread per four dims of a key.  Bound by memory, 4
// to 19 us.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_join_kernel(AttnArgs a) {
    const int quads = a.d / 4, tile = blockIdx.y;
    const uint32_t bh = blockIdx.x / (kGradKeys / 32), slice = blockIdx.x % (kGradKeys / 32);
    const int b = a.by_kv.div(bh), g = bh - b * a.kv;
    const int keys = a.lengths ? max(0, min(a.lengths[b], a.sk)) : a.sk;
    const int near = key_rows(a, tile, keys, tile < a.sink_tiles && a.far_parts > 0).pieces(a);  // those that were written
    for (int at = threadIdx.x; at < 32 * quads; at += 256) {
        const int row = slice * 32 + at / quads, dim = at % quads * 4, key = tile * kGradKeys + row;
        if (key >= a.sk) return;
        const float* from = a.part_o + grad_part(a, bh, tile) * 2 * a.d + row * a.d + dim;
        f32x4 dk = {0.f, 0.f, 0.f, 0.f}, dv = dk;
        auto add = [&](const float* x, int count, int piece_keys) {
            for (int p = 0; p < count; ++p, x += (int64_t)2 * piece_keys * a.d) {
                dk += *reinterpret_cast<const f32x4*>(x);
                dv += *reinterpret_cast<const f32x4*>(x + piece_keys * a.d);
            }
        };
        add(from, near, kGradKeys);
        if (tile < a.sink_tiles && key < a.sinks && row < a.far_keys) add(from + (int64_t)a.near_parts * 2 * kGradKeys * a.d, a.far_parts, a.far_keys);
        dk *= a.scale;
        *reinterpret_cast<u32x2*>(a.dk + ((int64_t)key * a.dk_st[0] + (int64_t)b * a.dk_st[1] + (int64_t)g * a.dk_st[2] + dim) * 2) =
            u32x2{Elem<T>::pack(dk[0], dk[1]), Elem<T>::pack(dk[2], dk[3])};
        *reinterpret_cast<u32x2*>(a.dv + ((int64_t)key * a.dv_st[0] + (int64_t)b * a.dv_st[1] + (int64_t)g * a.dv_st[2] + dim) * 2) =
            u32x2{Elem<T>::pack(dv[0], dv[1]), Elem<T>::pack(dv[2], dv[3])};
    }
}

}  // namespace neox
