// extern "C" entry points of the attention kernels and of the paged cache: argument validation, the choice of the
// kernel and of the parts of a split key axis, and the launches.  As in api.hip, validation finishes before the
// first HIP call.
#include <algorithm>

#include "internal.hpp"

namespace neox {

// ---- launches whose kernels do not depend on the head dim ------------------------------------------------
// A wave for each row where there are many rows in few parts, else a workgroup (bf16, 128 dims, us: 32768 rows in 2 parts
// 24 with a workgroup, 11 with a wave; 16384 in 4 14, 9; 4096 in 16 8.6, 7.2; 2048 in 4 4.4, 4.5; 512 in 16 4.8, 6.4).
static bool join_by_waves(const AttnArgs& a) { return a.splits <= 16 && a.part_rows >= 4096; }
static int64_t join_blocks(const AttnArgs& a) { return join_by_waves(a) ? (a.part_rows + 3) / 4 : a.part_rows; }
hipError_t launch_attn_join(const AttnArgs& a, int dtype, hipStream_t stream) {
    const uint32_t blocks = (uint32_t)join_blocks(a);
    if (join_by_waves(a)) {
        if (dtype == NEOX_BF16) attn_join_rows_kernel<BF16><<<blocks, 256, 0, stream>>>(a);
        else attn_join_rows_kernel<F16><<<blocks, 256, 0, stream>>>(a);
        return hipGetLastError();
    }
    if (dtype == NEOX_BF16) attn_join_kernel<BF16><<<blocks, 256, 0, stream>>>(a);
    else attn_join_kernel<F16><<<blocks, 256, 0, stream>>>(a);
    return hipGetLastError();
}

// Threads of a row: a power of two, for as many elements each as the kernels take.
static int cache_lanes(int d, int source, bool write) {
    const int elems = write && source != kPaged16 ? 16 : 8;
    int lanes = write && source == kPagedF4 ? 2 : 4;
    while (lanes * elems < d) lanes *= 2;
    return lanes;
}
template <typename T, int SRC, bool WRITE>
static void cache_rows(const CacheArgs& a, hipStream_t stream) {
    constexpr int kElems = cache_elems<SRC, WRITE>();
    const int lanes = cache_lanes(a.d, SRC, WRITE);
    const uint32_t blocks = (uint32_t)((a.rows * lanes + 255) / 256);
    switch (lanes) {
        case 4: cache_kernel<T, SRC, 4, WRITE><<<blocks, 256, 0, stream>>>(a); break;
        case 8: cache_kernel<T, SRC, 8, WRITE><<<blocks, 256, 0, stream>>>(a); break;
        case 16: cache_kernel<T, SRC, 16, WRITE><<<blocks, 256, 0, stream>>>(a); break;
        default:
            if constexpr (kElems == 8) cache_kernel<T, SRC, 32, WRITE><<<blocks, 256, 0, stream>>>(a);
    }
}
template <typename T, bool WRITE>
static void cache_source(const CacheArgs& a, int source, hipStream_t stream) {
    if (source == kPagedI8) cache_rows<T, kPagedI8, WRITE>(a, stream);
    else if (source == kPagedF8) cache_rows<T, kPagedF8, WRITE>(a, stream);
    else cache_rows<T, kPaged16, WRITE>(a, stream);
}
template <typename T, bool WRITE>
static void cache4_rows(const CacheArgs& a, hipStream_t stream) {
    const int lanes = cache_lanes(a.d, kPagedF4, WRITE);
    const uint32_t blocks = (uint32_t)((a.rows * lanes + 255) / 256);
    switch (lanes) {
        case 2: if constexpr (WRITE) cache4_kernel<T, 2, WRITE><<<blocks, 256, 0, stream>>>(a); break;  // (32 dims)
        case 4: cache4_kernel<T, 4, WRITE><<<blocks, 256, 0, stream>>>(a); break;
        case 8: cache4_kernel<T, 8, WRITE><<<blocks, 256, 0, stream>>>(a); break;
        case 16: cache4_kernel<T, 16, WRITE><<<blocks, 256, 0, stream>>>(a); break;
        default: if constexpr (!WRITE) cache4_kernel<T, 32, WRITE><<<blocks, 256, 0, stream>>>(a);  // (above 128)
    }
}
hipError_t launch_cache(const CacheArgs& a, int source, int dtype, bool write, hipStream_t stream) {
    if (source == kPagedF4) {
        if (dtype == NEOX_BF16) write ? cache4_rows<BF16, true>(a, stream) : cache4_rows<BF16, false>(a, stream);
        else write ? cache4_rows<F16, true>(a, stream) : cache4_rows<F16, false>(a, stream);
        return hipGetLastError();
    }
    if (dtype == NEOX_BF16) write ? cache_source<BF16, true>(a, source, stream) : cache_source<BF16, false>(a, source, stream);
    else write ? cache_source<F16, true>(a, source, stream) : cache_source<F16, false>(a, source, stream);
    return hipGetLastError();
}

// ---- validation ------------------------------------------------------------------------------------------------
constexpr int kMost = 1 << 30;  // sizes and positions stay below, so that sums of two stay in 32 bits

// A launch has less than 2^32 threads in one direction.  (Workgroups of 512 there are 256 at most.)
static bool launches(int64_t blocks) { return blocks * 256 < (int64_t)1 << 32; }

static int check_heads(int h, int h_kv, int d, const char* what) {
    if (h < 1 || h_kv < 1 || h % h_kv != 0)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: h=%d must be a positive multiple of h_kv=%d", what, h, h_kv);
    if (d < 8 || d > 256 || d % 8 != 0)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: head dim %d must be a multiple of 8 from 8 to 256", what, d);
    return NEOX_OK;
}

// Strides of a tensor whose last axis is dense: not negative, rows on 16-byte boundaries (unit: elements in 16 bytes),
// heads at least d apart.
static int check_strides(const int64_t* st, int n, int heads, int d, int unit, const char* what, const char* name) {
    if (!st) return fail(NEOX_ERR_NULL_POINTER, "%s: %s strides are null", what, name);
    for (int i = 0; i < n; ++i) {
        if (st[i] < 0) return fail(NEOX_ERR_BAD_STRIDE, "%s: %s stride[%d]=%lld is negative", what, name, i, (long long)st[i]);
        if (st[i] >= (int64_t)1 << 31)
            return fail(NEOX_ERR_BAD_STRIDE, "%s: %s stride[%d]=%lld is not below 2^31", what, name, i, (long long)st[i]);
        if (unit && st[i] % unit != 0)
            return fail(NEOX_ERR_BAD_STRIDE, "%s: %s stride[%d]=%lld is not a multiple of %d elements", what, name, i, (long long)st[i], unit);
    }
    if (heads > 1 && st[n - 1] < d)
        return fail(NEOX_ERR_BAD_STRIDE, "%s: %s head stride %lld is smaller than d=%d", what, name, (long long)st[n - 1], d);
    return NEOX_OK;
}

static int check_pointer(const void* p, int bytes, const char* what, const char* name) {
    if (!p) return fail(NEOX_ERR_NULL_POINTER, "%s: %s is null", what, name);
    if (!aligned(p, bytes)) return fail(NEOX_ERR_MISALIGNED, "%s: %s must be %d-byte aligned", what, name, bytes);
    return NEOX_OK;
}

#define NEOX_TRY(call) \
    if (int status = (call)) return status

template <int N>
static void copy_strides(int64_t (&to)[N], const int64_t* from) {
    for (int i = 0; i < N; ++i) to[i] = from[i];
}

static int check_scale_window(float scale, int sinks, const char* what) {
    if (!(scale >= -__FLT_MAX__ && scale <= __FLT_MAX__)) return fail(NEOX_ERR_BAD_SHAPE, "%s: scale must be finite", what);
    if (sinks < 0) return fail(NEOX_ERR_BAD_SHAPE, "%s: sinks=%d is negative", what, sinks);
    return NEOX_OK;
}

static void set_scale_window(AttnArgs& a, float scale, int window, int sinks) {
    a.scale = scale;
    // (never 0: a hidden key's score is minus infinity before it is multiplied)
    a.scale_log2 = __builtin_fmaxf((scale < 0.f ? -scale : scale) * kLog2e, __FLT_MIN__);
    a.flip = scale < 0.f ? 0x80008000u : 0u;
    a.window = window < 0 || window >= kMost ? -1 : window;
    a.sinks = sinks < kMost ? sinks : kMost;
}

static int padded(int d) { return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : 256; }

static hipError_t run_fwd(const AttnArgs& a, int source, int dtype, hipStream_t stream) {
    switch (padded(a.d)) {
        case 64: return launch_attn_fwd<64>(a, source, dtype, stream);
        case 96: return launch_attn_fwd<96>(a, source, dtype, stream);
        case 128: return launch_attn_fwd<128>(a, source, dtype, stream);
        default: return launch_attn_fwd<256>(a, source, dtype, stream);
    }
}
static hipError_t run_token(const AttnArgs& a, int source, int dtype, hipStream_t stream) {
    switch (padded(a.d)) {
        case 64: return launch_attn_token<64>(a, source, dtype, stream);
        case 96: return launch_attn_token<96>(a, source, dtype, stream);
        case 128: return launch_attn_token<128>(a, source, dtype, stream);
        default: return launch_attn_token<256>(a, source, dtype, stream);
    }
}
static hipError_t run_bwd(const AttnArgs& a, int dtype, hipStream_t stream) {
    switch (padded(a.d)) {
        case 64: return launch_attn_bwd<64>(a, dtype, stream);
        case 96: return launch_attn_bwd<96>(a, dtype, stream);
        case 128: return launch_attn_bwd<128>(a, dtype, stream);
        default: return launch_attn_bwd<256>(a, dtype, stream);
    }
}

// sizes of a window-attention call
static int check_window_sizes(int b, int sq, int sk, int h, int h_kv, int d, const char* what) {
    if (b < 1 || sq < 1 || sk < 1 || sq >= kMost || sk >= kMost)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: b=%d sq=%d sk=%d must be at least 1 (and sq, sk below 2^30)", what, b, sq, sk);
    NEOX_TRY(check_heads(h, h_kv, d, what));
    const int64_t rows = (int64_t)sq * (h / h_kv), tiles = (rows + kTileRows - 1) / kTileRows, units = (int64_t)b * h_kv;
    if (rows >= kMost || units * tiles >= kMost || units * (((int64_t)sk + 127) / 128) * 128 >= kMost || sk > 65535 * 128)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: b=%d sq=%d sk=%d h=%d is too large for one call", what, b, sq, sk, h);
    return NEOX_OK;
}

static void set_window_sizes(AttnArgs& a, int b, int sq, int sk, int h, int h_kv, int d) {
    a.b = b;
    a.sq = sq;
    a.sk = sk;
    a.kv = h_kv;
    a.group = h / h_kv;
    a.d = d;
    a.splits = 1;
    a.row_tiles = (sq * a.group + kTileRows - 1) / kTileRows;
    a.by_group = FastDiv::by((uint32_t)a.group);
    a.by_kv = FastDiv::by((uint32_t)h_kv);
    a.by_row_tiles = FastDiv::by((uint32_t)a.row_tiles);
    a.by_page = FastDiv::by(1);
}

// how the key gradients' work is cut into pieces, and the scratch it needs: fp32 sums of pieces, then delta
struct GradPlan {
    int key_tiles, near_parts, piece_rows, sink_tiles, far_parts, far_keys;
    int64_t parts_bytes, bytes;
};

// Pieces of a tile's near rows, of one size for all tiles: so many that two workgroups run on every CU, or under a bare
// causal mask, whose first tiles have twice the rows of the average, so that no piece is longer than a CU's share; 256
// rows or more for each.  Rows behind the window of a tile that holds sinks come in pieces of 512 rows, or longer
// ones where those would be more than two for every workgroup that fits (many sinks are many such tiles, and every piece is
// scratch).  Where they are no more than 128, and would be the only reason to join pieces, the tile takes them along: apart and
// with their tile, bf16, forward and backward, us: 28 rows (256 tokens, window 100), 8 heads of 64 dims 75, 72, 2 samples of 128
// dims 74, 70; 64 rows 75, 71; 128 rows 74, 71; 256 rows (512 tokens, 8 heads of 128 dims) 73, 71, but 640 tokens, 32 heads 77, 82;
// 512 rows (768 tokens, 32 heads of 64 dims) 74, 70.
static GradPlan plan_grad(int b, int sq, int sk, int h, int h_kv, int d, int window, int sinks) {
    GradPlan p{};
    const int64_t group = h / h_kv, units = (int64_t)b * h_kv;
    p.key_tiles = (sk + kGradKeys - 1) / kGradKeys;
    const bool all = window < 0 || (int64_t)window + kGradKeys >= sq;
    const int64_t near = all ? sq : (int64_t)window + kGradKeys;
    const int64_t tiles = units * p.key_tiles, most = near * group / 256;
    int64_t parts = ((all ? 1024 : 512) + tiles - 1) / tiles;
    if (parts > most) parts = most;
    p.near_parts = parts < 1 ? 1 : parts > 64 ? 64 : (int)parts;
    // (a single piece holds whatever a tile has: with sinks that may be more than the near rows)
    p.piece_rows = p.near_parts == 1 ? kMost : (int)((near * group + p.near_parts * kStepRows - 1) / (p.near_parts * kStepRows) * kStepRows);
    const int64_t last = (sinks < sk ? sinks : sk);
    // the last position whose window reaches the first tile is kGradKeys - 1 + window
    const int64_t behind = window < 0 || last < 1 ? 0 : (int64_t)sk - kGradKeys - window;
    const int64_t rows = (behind < sq ? behind : sq) * group;
    if (behind > 0 && (p.near_parts > 1 || rows > 128)) {
        p.sink_tiles = (int)((last + kGradKeys - 1) / kGradKeys);
        const int64_t far = (rows + 511) / 512, enough = (1024 + units * p.sink_tiles - 1) / (units * p.sink_tiles);
        p.far_parts = (int)(far < enough ? far : enough);
        if (p.far_parts > 64) p.far_parts = 64;
        p.far_keys = last < kGradKeys ? (int)last : kGradKeys;
    }
    p.parts_bytes = units * grad_part_keys(p.key_tiles, p.near_parts, p.sink_tiles, p.far_parts, p.far_keys) * 2 * d * (int64_t)sizeof(float);
    p.bytes = p.parts_bytes + (int64_t)b * h * sq * (int64_t)sizeof(float);
    return p;
}

// how a call over pages is cut: single tokens or row tiles, and how many parts of the key axis
struct PagedPlan {
    bool token;
    int row_tiles, splits;
    int waves;  // of a workgroup: single tokens over 4 bits
    int64_t bytes;
};

// Single tokens are calls of at most 16 rows to a key head, which is what that kernel's instructions hold; what has more goes to
// row tiles of 128, mostly empty at first.  128 dims, us, 8 rows (one token of 32 heads on 4), 16, 24 and 40: 16 sequences of
// 8192 keys in int8 41, 44, 52, 59, in bf16 55, 62, 50, 56; one of 65536 in int8 24, 25, 32, 37, in bf16 33, 34, 35, 37; a single key
// head, 16 and 17 rows, one of 65536: int8 18 and 29, bf16 20 and 30.
// Parts: so many that every CU has workgroups enough, with at least 256 keys for each part and 128 parts at most.  Row
// tiles: two that widen codes fit a CU, three that read 16 bits.  Measured in bf16 pages with two and with three, us: 1 x 512 tokens
// over 8192, 32 heads on 8: 113, 102; 2 x 512 over 4096: 111, 100; 1 x 2048 over 8192, 12 heads of 64 dims: 131, 105; 4 x 64 over
// 8192: 65, 63; but 2 x 1000 over 3000, 32 heads on 32: 137, 162; 4 x 512 with a window of 4096: 186, 214; 1 x 256 over 32768, 16
// heads of 256 dims: 372, 391: a second part costs calls whose tiles nearly fill the card.  In int8 with two and with three: 115, 130; 117,
// 132; 161, 127; 68, 78; 147, 173; 205, 232; 328, 355.  Single tokens: eight, twice what fits, because sequences differ in length and
// the host does not know by how much: 64 sequences of 2048 to 8192 tokens, int8, take 191 us with four (170 before four fitted),
// 158 with eight, 169 with sixteen; one of 131001 tokens in bf16 takes 125 us with 128 parts and 128 with 256.
//
// Single tokens over 4 bits take up to 48 rows in blocks of 16 (64 above 160 dims), whose workgroups read the same keys: a few tokens of
// a draft would leave row tiles of 128 mostly empty.  us in row tiles and in blocks: bf16, 128 dims, 16 sequences of 8000 tokens, 4 key heads, 20
// rows 39, 28, 40 rows 47, 35, 48 rows 47, 39, 64 rows 49, 44; 64 of 4000, 8 key heads, 64 rows 115, 125; one of 30000, 64 rows 33, 37; 256 dims, fp16, 64 of
// 2000, 20 rows 231, 78; 64 of 4000, 64 rows 492, 241.
//
// They have less to read for each key, and parts cost them more: no more of them than that, one up to 640 keys and up
// to eight for each workgroup of a single round; else a workgroup to a CU, two where parts are longer than 640 keys then, eight where they are longer than
// 1024 (and a single one than 2048), of 1024 keys at least.  One part of more than 256 keys, and no more workgroups than CUs: eight waves,
// which are slower wherever workgroups share a CU (us with four and eight: four sequences of 517 tokens, 12 heads of 64 dims, 8.5, 7.5; 16 of 517
// 7.7, 7.0; 16 of 1000 of 8 heads of 128 12.3, 11.3; 64 of 1000 15.3, 16.4; one of 120 5.5, 6.0).  us by parts, bf16, 128 dims, 8 key heads: 16 sequences of 517 tokens 1: 9.1, 2: 10.3, 4: 10.4; 64 of
// 1000 1: 15.1, 2: 19.9, 4: 22.7; 64 of 2000 1: 24.4, 2: 27.9; 16 of 2000 2: 16.9, 4: 15.0, 8: 16.5, 16: 19.7; 1 of 4000 16: 10.8, 32: 9.3; 4 of
// 2000 4: 12.0, 8: 10.4, 16: 11.9; 4 of 32000 16: 28.1, 32: 26.6, 64: 28.8; 64 of 8192 1: 116, 2: 98, 4: 88, 8: 88, 12: 95; 256 dims, fp16, 16 drafts of 5
// tokens in a window of 1024 1: 24.0, 2: 23.2, 3: 24.5.
// Next to the rule's borders: those drafts, 128 units, with windows of 880 1: 23.3, 2: 21.4, of 1014 1: 23.8, 2: 23.2; 16 sequences of 1024 tokens of 8 heads of 128
// 1: 12.6, 2: 12.9, of 1060 1: 12.7, 2: 13.8, of 1280 2: 14.1, 4: 14.4, of 1300 2: 14.9, 4: 14.5; 4 of 640 1: 9.4, 3: 9.6, of 660 1: 10.2, 3: 9.6; 64 of 2048
// 1: 36.7, 2: 33.5, 3: 35.1, of 2060 1: 36.8, 2: 35.0, 3: 36.0; 32 of 2048 1: 18.8, 2: 21.5, of 2100 1: 18.5, 3: 22.5, of 3000 1: 23.9, 3: 27.6.  The
// rule is within 10 % of the better side but for those 256 units of equal length above 2048 keys, 15 to 22 %; unequal ones need the parts.
static int parts_token4(int64_t units, int64_t keys, int64_t most) {
    int64_t parts = std::min(most, (256 + units - 1) / units);
    if (keys <= std::max((int64_t)640, 8 * std::min(units, (int64_t)256))) return 1;
    if (keys > 640 * parts) parts = std::min(most, (512 + units - 1) / units);
    if (keys > (parts == 1 ? 2048 : 1024 * parts)) parts = std::min({most, (2048 + units - 1) / units, (keys + 1023) / 1024});
    return (int)parts;
}
static PagedPlan plan_paged(int b, int tokens, int max_query, int max_context, int h, int h_kv, int d, int window, int sinks, int source) {
    const bool codes = source != kPaged16;
    PagedPlan p{};
    const int64_t group = h / h_kv, rows = max_query * group;
    p.token = rows <= 16;
    p.row_tiles = p.token ? 1 : (int)((rows + kTileRows - 1) / kTileRows);
    int64_t keys = max_context;
    if (window >= 0) {
        const int64_t seen = (int64_t)window + max_query + sinks;
        if (seen < keys) keys = seen;
    }
    const bool blocks = source == kPagedF4 && rows <= (d <= 160 ? 48 : 64);
    const int64_t units = (int64_t)b * h_kv * p.row_tiles, target = 256 * (p.token ? 8 : codes && !blocks ? 2 : 3);
    int64_t splits = (target + units - 1) / units;
    const int64_t most = (keys + 255) / 256;
    if (splits > most) splits = most;
    if (splits > kMostParts) splits = kMostParts;
    if (splits < 1) splits = 1;
    p.splits = (int)splits;
    if (blocks) {
        p.token = true;
        p.row_tiles = (int)((rows + 15) / 16);
        const int64_t groups = (int64_t)b * h_kv * p.row_tiles;
        p.splits = parts_token4(groups, keys, splits);
        p.waves = p.splits == 1 && groups <= 256 && keys > 256 ? 8 : 4;
    }
    p.bytes = p.splits > 1 ? (int64_t)p.splits * tokens * h * (d + 1) * (int64_t)sizeof(float) : 0;
    return p;
}

// Key heads to a wave of the single tokens over 4 bits: two, where a row's scales are fetched at once, their rows fit the columns
// and half the workgroups are two to a CU.
static int token4_heads(const AttnArgs& a) {
    const bool two = token4_fetch(a, padded4(a.d)) == kFetchRows && a.d <= 128 && a.kv % 2 == 0 && 2 * a.sq * a.group <= 16;
    return two && (int64_t)a.b * a.kv * a.splits >= 1024 ? 2 : 1;
}

static int check_paged_sizes(int b, int tokens, int max_query, int max_context, int h, int h_kv, int d, const char* what) {
    if (b < 1 || tokens < 1 || max_query < 1 || max_context < 1 || max_query >= kMost || max_context >= kMost)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: b=%d tokens=%d max_query=%d max_context=%d must be at least 1 (the maxima below 2^30)", what, b,
                    tokens, max_query, max_context);
    NEOX_TRY(check_heads(h, h_kv, d, what));
    const int64_t rows = (int64_t)max_query * (h / h_kv);
    if (rows >= kMost || (int64_t)b * h_kv * ((rows + kTileRows - 1) / kTileRows) >= kMost || (int64_t)tokens * h >= kMost)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: b=%d tokens=%d max_query=%d h=%d is too large for one call", what, b, tokens, max_query, h);
    return NEOX_OK;
}

static int cache_source_of(int cache_dtype, int dtype) {
    if (cache_dtype == dtype) return kPaged16;
    if (cache_dtype == NEOX_I8) return kPagedI8;
    if (cache_dtype == NEOX_F8) return kPagedF8;
    if (cache_dtype == NEOX_F4) return kPagedF4;
    return -1;
}

// The cache's own part of a call: pointers, strides {page, token in the page, head}, sizes.
static int check_cache(const void* kc, const void* vc, const void* ks, const void* vs, const int64_t* kc_st, const int64_t* vc_st,
                       const int64_t* ks_st, const int64_t* vs_st, int64_t pages, int page_size, int h_kv, int d, int dtype,
                       int cache_dtype, const char* what) {
    const int source = cache_source_of(cache_dtype, dtype);
    if (source < 0)
        return fail(NEOX_ERR_BAD_DTYPE, "%s: the cache must hold int8, fp8 (e4m3), fp4 (e2m1) or the dtype of the call (code %d)", what, cache_dtype);
    const bool codes = source != kPaged16, nibbles = source == kPagedF4;
    NEOX_TRY(check_pointer(kc, 16, what, "k_cache"));
    NEOX_TRY(check_pointer(vc, 16, what, "v_cache"));
    if (pages < 1 || pages >= kMost || page_size < 1 || page_size >= kMost)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: pages=%lld page_size=%d must be at least 1 and below 2^30", what, (long long)pages, page_size);
    if (nibbles && d % 32 != 0) return fail(NEOX_ERR_BAD_SHAPE, "%s: head dim %d of a 4-bit cache must be a multiple of 32", what, d);
    if (codes && d % 16 != 0) return fail(NEOX_ERR_BAD_SHAPE, "%s: head dim %d of an 8-bit cache must be a multiple of 16", what, d);
    const int unit = codes ? 16 : 8;
    const int row = nibbles ? d / 2 : d, scales = nibbles ? d / 32 : 1;
    NEOX_TRY(check_strides(kc_st, 3, h_kv, row, unit, what, "k_cache"));
    NEOX_TRY(check_strides(vc_st, 3, h_kv, row, unit, what, "v_cache"));
    if (codes) {
        NEOX_TRY(check_pointer(ks, nibbles ? 1 : 4, what, "k_scales"));
        NEOX_TRY(check_pointer(vs, nibbles ? 1 : 4, what, "v_scales"));
        NEOX_TRY(check_strides(ks_st, 3, h_kv, scales, 0, what, "k_scales"));
        NEOX_TRY(check_strides(vs_st, 3, h_kv, scales, 0, what, "v_scales"));
    }
    return NEOX_OK;
}

// {page, token, head} as the kernels have them: token, page, head
static void page_strides(int64_t (&to)[3], const int64_t* from) {
    to[0] = from[1];
    to[1] = from[0];
    to[2] = from[2];
}

static int cache_call(const char* what, void* k, void* v, const void* kc, const void* vc, const void* ks, const void* vs, const void* slots,
                      int slots_64, int64_t tokens, int h_kv, int d, int64_t pages, int page_size, const int64_t* k_st, const int64_t* v_st,
                      const int64_t* kc_st, const int64_t* vc_st, const int64_t* ks_st, const int64_t* vs_st, int dtype, int cache_dtype,
                      bool write, void* stream) {
    NEOX_TRY(check_dtype(dtype, what));
    NEOX_TRY(check_heads(h_kv, h_kv, d, what));
    NEOX_TRY(check_pointer(k, 16, what, "k"));
    NEOX_TRY(check_pointer(v, 16, what, "v"));
    NEOX_TRY(check_pointer(slots, slots_64 ? 8 : 4, what, "slots"));
    if (tokens < 1 || tokens >= kMost || tokens * h_kv >= kMost)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: %lld tokens of %d heads: must be at least 1 and below 2^30 rows", what, (long long)tokens, h_kv);
    NEOX_TRY(check_strides(k_st, 2, h_kv, d, 8, what, "k"));
    NEOX_TRY(check_strides(v_st, 2, h_kv, d, 8, what, "v"));
    NEOX_TRY(check_cache(kc, vc, ks, vs, kc_st, vc_st, ks_st, vs_st, pages, page_size, h_kv, d, dtype, cache_dtype, what));
    const int source = cache_source_of(cache_dtype, dtype);
    if (!launches((tokens * h_kv * cache_lanes(d, source, write) + 255) / 256))
        return fail(NEOX_ERR_BAD_SHAPE, "%s: %lld tokens of %d heads of %d dims are too large for one call", what, (long long)tokens, h_kv, d);
    CacheArgs a{};
    a.k = static_cast<char*>(k);
    a.v = static_cast<char*>(v);
    a.kc = static_cast<char*>(const_cast<void*>(kc));
    a.vc = static_cast<char*>(const_cast<void*>(vc));
    a.slots = slots;
    a.wide = slots_64 != 0;
    copy_strides(a.k_st, k_st);
    copy_strides(a.v_st, v_st);
    page_strides(a.kc_st, kc_st);
    page_strides(a.vc_st, vc_st);
    if (source != kPaged16) {
        a.ks = static_cast<float*>(const_cast<void*>(ks));
        a.vs = static_cast<float*>(const_cast<void*>(vs));
        page_strides(a.ks_st, ks_st);
        page_strides(a.vs_st, vs_st);
    }
    a.slot_count = pages * page_size;
    a.rows = tokens * h_kv;
    a.heads = h_kv;
    a.d = d;
    a.page = page_size;
    a.by_heads = FastDiv::by((uint32_t)h_kv);
    a.by_page = FastDiv::by((uint32_t)page_size);
    return check_launch(launch_cache(a, source, dtype, write, (hipStream_t)stream), what);
}

}  // namespace neox

using namespace neox;

#pragma GCC visibility push(default)
extern "C" {

int neox_window_attention_fwd(void* out, void* out_low, float* lse, const void* q, const void* k, const void* v, const int32_t* key_lengths, int32_t b,
                              int32_t sq, int32_t sk, int32_t h, int32_t h_kv, int32_t d, const int64_t q_strides[3],
                              const int64_t k_strides[3], const int64_t v_strides[3], const int64_t out_strides[3], float scale,
                              int32_t window, int32_t sinks, int32_t dtype, void* stream) {
    static const char* what = "neox_window_attention_fwd";
    NEOX_TRY(check_dtype(dtype, what));
    NEOX_TRY(check_pointer(out, 16, what, "out"));
    NEOX_TRY(check_pointer(q, 16, what, "q"));
    NEOX_TRY(check_pointer(k, 16, what, "k"));
    NEOX_TRY(check_pointer(v, 16, what, "v"));
    if (!aligned(out_low, 16) || !aligned(lse, 4) || !aligned(key_lengths, 4)) return fail(NEOX_ERR_MISALIGNED, "%s: misaligned pointer", what);
    NEOX_TRY(check_window_sizes(b, sq, sk, h, h_kv, d, what));
    NEOX_TRY(check_strides(q_strides, 3, h, d, 8, what, "q"));
    NEOX_TRY(check_strides(k_strides, 3, h_kv, d, 8, what, "k"));
    NEOX_TRY(check_strides(v_strides, 3, h_kv, d, 8, what, "v"));
    NEOX_TRY(check_strides(out_strides, 3, h, d, 8, what, "out"));
    NEOX_TRY(check_scale_window(scale, sinks, what));
    AttnArgs a{};
    set_window_sizes(a, b, sq, sk, h, h_kv, d);
    set_scale_window(a, scale, window, sinks);
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k);
    a.v = static_cast<const char*>(v);
    a.o = static_cast<char*>(out);
    a.o_low = static_cast<char*>(out_low);
    a.lse = lse;
    a.lengths = key_lengths;
    copy_strides(a.q_st, q_strides);
    copy_strides(a.k_st, k_strides);
    copy_strides(a.v_st, v_strides);
    copy_strides(a.o_st, out_strides);
    return check_launch(run_fwd(a, kStrided, dtype, (hipStream_t)stream), what);
}

int neox_window_attention_bwd_workspace(int64_t* bytes, int32_t b, int32_t sq, int32_t sk, int32_t h, int32_t h_kv, int32_t d, int32_t window,
                                        int32_t sinks) {
    static const char* what = "neox_window_attention_bwd_workspace";
    if (!bytes) return fail(NEOX_ERR_NULL_POINTER, "%s: bytes is null", what);
    NEOX_TRY(check_window_sizes(b, sq, sk, h, h_kv, d, what));
    NEOX_TRY(check_scale_window(1.f, sinks, what));
    *bytes = plan_grad(b, sq, sk, h, h_kv, d, window, sinks).bytes;
    return NEOX_OK;
}

int neox_window_attention_bwd(void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes, const void* dout, const void* out, const void* out_low, const float* lse, const void* q,
                              const void* k, const void* v, const int32_t* key_lengths, int32_t b, int32_t sq, int32_t sk, int32_t h,
                              int32_t h_kv, int32_t d, const int64_t dq_strides[3], const int64_t dk_strides[3],
                              const int64_t dv_strides[3], const int64_t dout_strides[3], const int64_t out_strides[3],
                              const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3], float scale,
                              int32_t window, int32_t sinks, int32_t dtype, void* stream) {
    static const char* what = "neox_window_attention_bwd";
    NEOX_TRY(check_dtype(dtype, what));
    struct Given {
        const void* p;
        const int64_t* st;
        bool grouped;
        const char* name;
    };
    const Given given[] = {{dq, dq_strides, false, "dq"},       {dk, dk_strides, true, "dk"},    {dv, dv_strides, true, "dv"},
                           {dout, dout_strides, false, "dout"}, {out, out_strides, false, "out"}, {q, q_strides, false, "q"},
                           {k, k_strides, true, "k"},           {v, v_strides, true, "v"}};
    for (const Given& g : given) NEOX_TRY(check_pointer(g.p, 16, what, g.name));
    NEOX_TRY(check_pointer(lse, 4, what, "lse"));
    NEOX_TRY(check_pointer(workspace, 16, what, "workspace"));
    if (!aligned(out_low, 16) || !aligned(key_lengths, 4)) return fail(NEOX_ERR_MISALIGNED, "%s: misaligned pointer", what);
    NEOX_TRY(check_window_sizes(b, sq, sk, h, h_kv, d, what));
    for (const Given& g : given) NEOX_TRY(check_strides(g.st, 3, g.grouped ? h_kv : h, d, 8, what, g.name));
    NEOX_TRY(check_scale_window(scale, sinks, what));
    const GradPlan plan = plan_grad(b, sq, sk, h, h_kv, d, window, sinks);
    if (workspace_bytes < plan.bytes)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: workspace of %lld bytes, needs %lld", what, (long long)workspace_bytes, (long long)plan.bytes);
    AttnArgs a{};
    set_window_sizes(a, b, sq, sk, h, h_kv, d);
    set_scale_window(a, scale, window, sinks);
    a.key_tiles = plan.key_tiles;
    a.near_parts = plan.near_parts;
    a.piece_rows = plan.piece_rows;
    a.sink_tiles = plan.sink_tiles;
    a.far_parts = plan.far_parts;
    a.far_keys = plan.far_keys;
    a.units = plan.key_tiles * plan.near_parts + plan.sink_tiles * plan.far_parts;
    a.by_units = FastDiv::by((uint32_t)a.units);
    a.by_near_parts = FastDiv::by((uint32_t)a.near_parts);
    a.by_far_parts = FastDiv::by((uint32_t)(a.far_parts > 0 ? a.far_parts : 1));
    a.part_o = static_cast<float*>(workspace);
    a.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.parts_bytes);
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k);
    a.v = static_cast<const char*>(v);
    a.out = static_cast<const char*>(out);
    a.o_low = static_cast<char*>(const_cast<void*>(out_low));
    a.dout = static_cast<const char*>(dout);
    a.dq = static_cast<char*>(dq);
    a.dk = static_cast<char*>(dk);
    a.dv = static_cast<char*>(dv);
    a.lse = const_cast<float*>(lse);
    a.lengths = key_lengths;
    copy_strides(a.q_st, q_strides);
    copy_strides(a.k_st, k_strides);
    copy_strides(a.v_st, v_strides);
    copy_strides(a.o_st, out_strides);
    copy_strides(a.do_st, dout_strides);
    copy_strides(a.dq_st, dq_strides);
    copy_strides(a.dk_st, dk_strides);
    copy_strides(a.dv_st, dv_strides);
    return check_launch(run_bwd(a, dtype, (hipStream_t)stream), what);
}

int neox_paged_attention_workspace(int64_t* bytes, int32_t b, int32_t tokens, int32_t max_query, int32_t max_context, int32_t h, int32_t h_kv,
                                   int32_t d, int32_t window, int32_t sinks) {
    static const char* what = "neox_paged_attention_workspace";
    if (!bytes) return fail(NEOX_ERR_NULL_POINTER, "%s: bytes is null", what);
    NEOX_TRY(check_paged_sizes(b, tokens, max_query, max_context, h, h_kv, d, what));
    NEOX_TRY(check_scale_window(1.f, sinks, what));
    *bytes = plan_paged(b, tokens, max_query, max_context, h, h_kv, d, window, sinks, kPaged16).bytes;  // (codes need no more)
    return NEOX_OK;
}

int neox_paged_attention(void* out, void* workspace, int64_t workspace_bytes, const void* q, const void* k_cache, const void* v_cache,
                         const void* k_scales, const void* v_scales, const int32_t* page_table, const int32_t* query_starts,
                         const int32_t* context_lengths, int32_t b, int32_t tokens, int32_t max_query, int32_t max_context, int32_t h,
                         int32_t h_kv, int32_t d, int64_t pages, int32_t page_size, int32_t table_columns, int64_t table_stride,
                         const int64_t out_strides[2], const int64_t q_strides[2], const int64_t k_cache_strides[3],
                         const int64_t v_cache_strides[3], const int64_t k_scale_strides[3], const int64_t v_scale_strides[3], float scale,
                         int32_t window, int32_t sinks, int32_t dtype, int32_t cache_dtype, void* stream) {
    static const char* what = "neox_paged_attention";
    NEOX_TRY(check_dtype(dtype, what));
    NEOX_TRY(check_pointer(out, 16, what, "out"));
    NEOX_TRY(check_pointer(q, 16, what, "q"));
    NEOX_TRY(check_pointer(page_table, 4, what, "page_table"));
    NEOX_TRY(check_pointer(query_starts, 4, what, "query_starts"));
    NEOX_TRY(check_pointer(context_lengths, 4, what, "context_lengths"));
    NEOX_TRY(check_paged_sizes(b, tokens, max_query, max_context, h, h_kv, d, what));
    NEOX_TRY(check_strides(out_strides, 2, h, d, 8, what, "out"));
    NEOX_TRY(check_strides(q_strides, 2, h, d, 8, what, "q"));
    NEOX_TRY(check_cache(k_cache, v_cache, k_scales, v_scales, k_cache_strides, v_cache_strides, k_scale_strides, v_scale_strides, pages,
                         page_size, h_kv, d, dtype, cache_dtype, what));
    if (table_columns < 1 || table_stride < 0)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: page_table needs a column and no negative stride (%d, %lld)", what, table_columns, (long long)table_stride);
    NEOX_TRY(check_scale_window(scale, sinks, what));
    const int source = cache_source_of(cache_dtype, dtype);
    const PagedPlan plan = plan_paged(b, tokens, max_query, max_context, h, h_kv, d, window, sinks, source);
    if (plan.bytes > 0) {
        NEOX_TRY(check_pointer(workspace, 16, what, "workspace"));
        if (workspace_bytes < plan.bytes)
            return fail(NEOX_ERR_BAD_SHAPE, "%s: workspace of %lld bytes, needs %lld", what, (long long)workspace_bytes, (long long)plan.bytes);
    }
    AttnArgs a{};
    a.b = b;
    a.sq = max_query;
    a.kv = h_kv;
    a.group = h / h_kv;
    a.d = d;
    a.tokens = tokens;
    a.row_tiles = plan.row_tiles;
    a.splits = plan.splits;
    a.waves = plan.waves;
    a.part_rows = (int64_t)tokens * h;
    a.part_o = static_cast<float*>(workspace);
    a.part_lse = a.part_o + a.splits * a.part_rows * d;
    a.by_group = FastDiv::by((uint32_t)a.group);
    a.by_kv = FastDiv::by((uint32_t)h_kv);
    a.by_row_tiles = FastDiv::by((uint32_t)a.row_tiles);
    a.by_splits = FastDiv::by((uint32_t)a.splits);
    a.by_page = FastDiv::by((uint32_t)page_size);
    set_scale_window(a, scale, window, sinks);
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k_cache);
    a.v = static_cast<const char*>(v_cache);
    a.o = static_cast<char*>(out);
    a.k_scale = static_cast<const float*>(k_scales);
    a.v_scale = static_cast<const float*>(v_scales);
    a.lengths = context_lengths;
    a.starts = query_starts;
    a.table = page_table;
    a.table_stride = table_stride;
    const int64_t named = (int64_t)table_columns * page_size;
    a.table_keys = named < max_context ? (int)named : max_context;
    a.pages = pages;
    a.q_st[0] = q_strides[0];
    a.q_st[2] = q_strides[1];
    a.o_st[0] = out_strides[0];
    a.o_st[2] = out_strides[1];
    page_strides(a.k_st, k_cache_strides);
    page_strides(a.v_st, v_cache_strides);
    if (source != kPaged16) {
        page_strides(a.ks_st, k_scale_strides);
        page_strides(a.vs_st, v_scale_strides);
    }
    a.heads = plan.token && source == kPagedF4 ? token4_heads(a) : 1;
    const int64_t blocks = (int64_t)(h_kv / a.heads) * a.row_tiles * (plan.token ? ((int64_t)b * a.splits + 7) / 8 * 8 : b);
    if (!launches(blocks) || (a.splits > 1 && !launches(join_blocks(a))))
        return fail(NEOX_ERR_BAD_SHAPE, "%s: b=%d h_kv=%d of %d rows is too large for one call", what, b, h_kv, max_query * (h / h_kv));
    hipStream_t s = (hipStream_t)stream;
    NEOX_TRY(check_launch(plan.token ? run_token(a, source, dtype, s) : run_fwd(a, source, dtype, s), what));
    return a.splits > 1 ? check_launch(launch_attn_join(a, dtype, s), what) : (int)NEOX_OK;
}

int neox_cache_write(void* k_cache, void* v_cache, void* k_scales, void* v_scales, const void* k, const void* v, const void* slots,
                     int32_t slots_64, int64_t tokens, int32_t h_kv, int32_t d, int64_t pages, int32_t page_size,
                     const int64_t k_cache_strides[3], const int64_t v_cache_strides[3], const int64_t k_scale_strides[3],
                     const int64_t v_scale_strides[3], const int64_t k_strides[2], const int64_t v_strides[2], int32_t dtype,
                     int32_t cache_dtype, void* stream) {
    return cache_call("neox_cache_write", const_cast<void*>(k), const_cast<void*>(v), k_cache, v_cache, k_scales, v_scales, slots, slots_64,
                      tokens, h_kv, d, pages, page_size, k_strides, v_strides, k_cache_strides, v_cache_strides, k_scale_strides,
                      v_scale_strides, dtype, cache_dtype, true, stream);
}

int neox_cache_read(void* k, void* v, const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                    const void* slots, int32_t slots_64, int64_t tokens, int32_t h_kv, int32_t d, int64_t pages, int32_t page_size,
                    const int64_t k_strides[2], const int64_t v_strides[2], const int64_t k_cache_strides[3],
                    const int64_t v_cache_strides[3], const int64_t k_scale_strides[3], const int64_t v_scale_strides[3], int32_t dtype,
                    int32_t cache_dtype, void* stream) {
    return cache_call("neox_cache_read", k, v, k_cache, v_cache, k_scales, v_scales, slots, slots_64, tokens, h_kv, d, pages, page_size,
                      k_strides, v_strides, k_cache_strides, v_cache_strides, k_scale_strides, v_scale_strides, dtype, cache_dtype, false,
                      stream);
}

}  // extern "C"
#pragma GCC visibility pop
