// Which pages of a cache belong to which sequence, kept in device memory: the pages and slots of new tokens from their
// numbers alone, and pages on their way back.  One workgroup of 1024 threads walks over the sequences, 1024 at a time; what
// every sequence takes follows from sums over those before it.
//   extend:   ends = cumsum(new), need_s = ceil((old + new) / page) - ceil(old / page), upto = cumsum(need);
//             page i of the call is free[left - 1 - i], slot = table[s, position / page] * page + position % page
//   truncate: the same pages in the opposite order, so that one undoes the other
// Latency bounds them, one load after the other and two sums over a workgroup: extend 4.0 us for 64 sequences of a token, 6.4 for 1000 of five, 4.7 + 6 for 256 prompts
// of 327000 tokens together; truncate 2.8, 3.1 and 6.1 for what these took.
// Sums saturate at 2^32 - 1, which keeps them sums of numbers that are not negative in any order.
#include "internal.hpp"

namespace neox {

struct PoolArgs {
    int32_t *table, *lengths, *free, *left;
    int64_t table_stride;
    const int32_t* given;  // extend: new tokens; truncate: lengths to keep
    int32_t *starts, *positions;
    int64_t* slots;
    uint8_t* granted;
    int32_t* first;  // workspace: the new pages of the sequences before; behind the last one, the pages that were free
    int sequences, columns, pages, tokens;
    FastDiv by_page;
};

constexpr int kPoolThreads = 1024, kOwnTokens = 8;

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Sums of x over the threads up to this one; *total gets that of all.  `sums` holds a word for each wave.
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t* sums, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint32_t y = __shfl_up(x, step);
        x = add_sat(x, lane >= step ? y : 0);
    }
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPoolThreads / 64; ++w) {
        if (w == wave) before = all;
        all = add_sat(all, sums[w]);
    }
    __syncthreads();
    *total = all;
    return add_sat(before, x);
}

__device__ __forceinline__ uint32_t pages_of(const PoolArgs& a, uint32_t tokens) { return a.by_page.div(tokens + a.by_page.d - 1); }

// a sequence's length, as far as its row of the table reaches
__device__ __forceinline__ uint32_t length_of(const PoolArgs& a, int s) {
    const int64_t room = (int64_t)a.columns * a.by_page.d;
    return (uint32_t)min((int64_t)max(a.lengths[s], 0), min(room, (int64_t)0x3fffffff));
}

// One new token: `inside` tokens behind the `old` ones of sequence s, whose new pages start `first` below the top of the list.
__device__ __forceinline__ void place(const PoolArgs& a, uint32_t t, int s, uint32_t old, uint32_t inside, uint32_t first, bool granted, int left) {
    const uint32_t position = old + inside, column = a.by_page.div(position), in = position - column * a.by_page.d;
    const uint32_t have = pages_of(a, old);
    int64_t slot = -1;
    if (granted) {
        int32_t* const entry = a.table + (int64_t)s * a.table_stride + column;
        int32_t page;
        if (column < have) {
            page = *entry;
        } else {
            page = a.free[left - 1 - (int)(first + column - have)];  // (granted: there are as many)
            if (in == 0) *entry = page;  // (the first token of a new page is new too)
        }
        slot = (int64_t)page * a.by_page.d + in;
    }
    a.positions[t] = (int32_t)position;
    a.slots[t] = slot;
}

// The tokens from t on of a sequence that has a few, no more than a page holds: its own thread's, whose two pages are fetched at once and which
// searches nothing (1000 sequences, 5 tokens each: 6.5 us, by the search 7.5).
__device__ __forceinline__ void place_own(const PoolArgs& a, uint32_t t, uint32_t count, int s, uint32_t old, uint32_t need, uint32_t first, bool granted,
                                          int left) {
    if (count == 0) return;
    const uint32_t size = a.by_page.d, column = a.by_page.div(old), have = pages_of(a, old);
    int32_t* const row = a.table + (int64_t)s * a.table_stride;
    int32_t pages[2] = {-1, -1};  // of `column` and the next
    if (granted) {
        const bool begun = column < have;
        if (begun) pages[0] = row[column];
        if (need) row[column + begun] = pages[begun] = a.free[left - 1 - (int)first];  // (no more than one)
    }
    for (uint32_t i = 0, in = old - column * size; i < count; ++i, ++in) {
        const bool next = in >= size;
        a.positions[t + i] = (int32_t)(old + i);
        a.slots[t + i] = granted ? (int64_t)pages[next] * size + (in - (next ? size : 0)) : -1;
    }
}

// TOKENS: the tokens' places too; otherwise they are left to place_kernel.
template <bool TOKENS>
__global__ __launch_bounds__(kPoolThreads) void extend_kernel(PoolArgs a) {
    __shared__ uint32_t sums[kPoolThreads / 64];
    __shared__ uint32_t ends[kPoolThreads], olds[kPoolThreads], firsts[kPoolThreads];
    __shared__ uint32_t taken;
    const int left = max(0, min(a.left[0], a.pages));
    const uint32_t most = (uint32_t)a.tokens;
    uint32_t tokens_before = 0, pages_before = 0;
    if (threadIdx.x == 0) taken = 0;
    __syncthreads();
    for (int s0 = 0; s0 < a.sequences; s0 += kPoolThreads) {
        const int s = s0 + threadIdx.x;
        const bool is = s < a.sequences;
        const uint32_t old = is ? length_of(a, s) : 0, count = is ? (uint32_t)max(0, min(a.given[s], 0x3fffffff)) : 0;
        uint32_t total;
        const uint32_t end = add_sat(tokens_before, scan(count, sums, &total));
        const bool fits = end <= most && (int64_t)old + count <= min((int64_t)a.columns * a.by_page.d, (int64_t)0x3fffffff);
        const uint32_t need = fits && is ? pages_of(a, old + count) - pages_of(a, old) : 0;
        uint32_t needed;
        const uint32_t upto = add_sat(pages_before, scan(need, sums, &needed));
        const bool granted = fits && (need == 0 || upto <= (uint32_t)left);
        const uint32_t first = upto - need;
        if (is) {
            if (s == 0) a.starts[0] = 0;
            a.starts[s + 1] = (int32_t)min(end, most);
            a.granted[s] = granted;
            if (granted) a.lengths[s] = (int32_t)(old + count);
            if (granted && need) atomicMax(&taken, upto);
            if (!TOKENS) a.first[s] = (int32_t)first;
        }
        if (TOKENS && !__syncthreads_or(count > kOwnTokens || kOwnTokens > a.by_page.d)) {
            place_own(a, end - count, min(count, most - min(most, end - count)), s, old, need, first, granted, left);
        } else if constexpr (TOKENS) {
            ends[threadIdx.x] = min(end, most);
            olds[threadIdx.x] = old;
            firsts[threadIdx.x] = granted ? first : ~0u;
            __syncthreads();
            const uint32_t t1 = min(add_sat(tokens_before, total), most), t0 = min(tokens_before, most);
            for (uint32_t t = t0 + threadIdx.x; t < t1; t += kPoolThreads) {
                int at = 0;  // the first sequence that ends behind t: there is one, since the last one ends at t1
#pragma unroll
                for (int step = kPoolThreads / 2; step; step /= 2)
                    if (ends[at + step - 1] <= t) at += step;
                place(a, t, s0 + at, olds[at], t - (at ? ends[at - 1] : t0), firsts[at], firsts[at] != ~0u, left);
            }
        }
        tokens_before = add_sat(tokens_before, total);
        pages_before = add_sat(pages_before, needed);
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        a.left[0] = left - (int)taken;
        if (!TOKENS) a.first[a.sequences] = left;
    }
    if constexpr (TOKENS) {
        for (uint32_t t = min(tokens_before, most) + threadIdx.x; t < most; t += kPoolThreads) {
            a.positions[t] = 0;
            a.slots[t] = -1;
        }
    }
}

__global__ __launch_bounds__(256) void place_kernel(PoolArgs a) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t >= (uint32_t)a.tokens) return;
    if ((int)t >= a.starts[a.sequences]) {
        a.positions[t] = 0;
        a.slots[t] = -1;
        return;
    }
    int lo = 0, hi = a.sequences - 1;  // the first sequence that ends behind t
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.starts[mid + 1] <= (int)t) lo = mid + 1;
        else hi = mid;
    }
    const uint32_t inside = t - a.starts[lo], count = a.starts[lo + 1] - a.starts[lo];
    const bool granted = a.granted[lo];
    const uint32_t old = granted ? (uint32_t)a.lengths[lo] - count : length_of(a, lo);
    place(a, t, lo, old, inside, (uint32_t)a.first[lo], granted, a.first[a.sequences]);
}

__global__ __launch_bounds__(kPoolThreads) void truncate_kernel(PoolArgs a) {
    __shared__ uint32_t sums[kPoolThreads / 64];
    __shared__ uint32_t ends[kPoolThreads], lasts[kPoolThreads];
    const uint32_t left = (uint32_t)max(0, min(a.left[0], a.pages)), room = (uint32_t)a.pages;
    uint32_t before = left;
    __syncthreads();
    // from the last sequence to the first, each from its last page to the first that goes
    for (int s0 = a.sequences - 1; s0 >= 0; s0 -= kPoolThreads) {
        const int s = s0 - (int)threadIdx.x;
        const bool is = s >= 0;
        const uint32_t old = is ? length_of(a, s) : 0, keep = is ? min((uint32_t)max(a.given[s], 0), old) : 0;
        const uint32_t last = pages_of(a, old);
        uint32_t total;
        const uint32_t end = scan(last - pages_of(a, keep), sums, &total);
        if (is) a.lengths[s] = (int32_t)keep;
        ends[threadIdx.x] = end;
        lasts[threadIdx.x] = last;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < total; i += kPoolThreads) {
            int at = 0;
#pragma unroll
            for (int step = kPoolThreads / 2; step; step /= 2)
                if (ends[at + step - 1] <= i) at += step;
            const uint32_t column = lasts[at] - 1 - (i - (at ? ends[at - 1] : 0));
            int32_t* const entry = a.table + (int64_t)(s0 - at) * a.table_stride + column;
            const uint32_t to = add_sat(before, i);
            if (to < room) a.free[to] = *entry;  // (a list that a caller has filled twice does not overflow)
            *entry = -1;
        }
        before = add_sat(before, total);
        __syncthreads();
    }
    if (threadIdx.x == 0) a.left[0] = (int32_t)min(before, room);
}

static int check_pool(PoolArgs& a, void* table, void* lengths, void* free_pages, void* left, const void* given, int32_t sequences, int32_t columns,
                      int64_t table_stride, int32_t pages, int32_t page_size, const char* what) {
    const struct {
        const void* p;
        const char* name;
    } words[] = {{table, "page_table"}, {lengths, "lengths"}, {free_pages, "free_pages"}, {left, "left"}, {given, "the sequences' numbers"}};
    for (const auto& w : words) {
        if (!w.p) return fail(NEOX_ERR_NULL_POINTER, "%s: %s is null", what, w.name);
        if (!aligned(w.p, 4)) return fail(NEOX_ERR_MISALIGNED, "%s: %s must be 4-byte aligned", what, w.name);
    }
    constexpr int most = 1 << 30;
    if (sequences < 1 || sequences >= most || columns < 1 || columns >= most || pages < 1 || pages >= most || page_size < 1 || page_size >= most)
        return fail(NEOX_ERR_BAD_SHAPE, "%s: sequences=%d columns=%d pages=%d page_size=%d must be at least 1 and below 2^30", what, sequences, columns,
                    pages, page_size);
    if (table_stride < (sequences > 1 ? columns : 0))
        return fail(NEOX_ERR_BAD_STRIDE, "%s: table stride %lld is smaller than its %d columns", what, (long long)table_stride, columns);
    a.table = static_cast<int32_t*>(table);
    a.lengths = static_cast<int32_t*>(lengths);
    a.free = static_cast<int32_t*>(free_pages);
    a.left = static_cast<int32_t*>(left);
    a.given = static_cast<const int32_t*>(given);
    a.table_stride = table_stride;
    a.sequences = sequences;
    a.columns = columns;
    a.pages = pages;
    a.by_page = FastDiv::by((uint32_t)page_size);
    return NEOX_OK;
}

}  // namespace neox

using namespace neox;

#pragma GCC visibility push(default)
extern "C" {

int neox_pages_extend(int32_t* query_starts, int32_t* positions, int64_t* slots, uint8_t* granted, int32_t* workspace, int32_t* page_table,
                      int32_t* lengths, int32_t* free_pages, int32_t* left, const int32_t* new_tokens, int32_t sequences, int32_t columns,
                      int64_t table_stride, int32_t pages, int32_t page_size, int32_t max_tokens, void* stream) {
    static const char* what = "neox_pages_extend";
    PoolArgs a{};
    if (int status = check_pool(a, page_table, lengths, free_pages, left, new_tokens, sequences, columns, table_stride, pages, page_size, what)) return status;
    if (max_tokens < 0 || max_tokens >= 1 << 30) return fail(NEOX_ERR_BAD_SHAPE, "%s: max_tokens=%d must be from 0 to below 2^30", what, max_tokens);
    if (!query_starts || !granted || !workspace || (max_tokens > 0 && (!positions || !slots)))
        return fail(NEOX_ERR_NULL_POINTER, "%s: an output or the workspace is null", what);
    if (!aligned(query_starts, 4) || !aligned(positions, 4) || !aligned(slots, 8) || !aligned(workspace, 4))
        return fail(NEOX_ERR_MISALIGNED, "%s: an output or the workspace is misaligned", what);
    a.starts = query_starts;
    a.positions = positions;
    a.slots = slots;
    a.granted = granted;
    a.first = workspace;
    a.tokens = max_tokens;
    hipStream_t s = (hipStream_t)stream;
    if (max_tokens <= 8 * kPoolThreads) {
        extend_kernel<true><<<1, kPoolThreads, 0, s>>>(a);
    } else {
        extend_kernel<false><<<1, kPoolThreads, 0, s>>>(a);
        place_kernel<<<((uint32_t)max_tokens + 255) / 256, 256, 0, s>>>(a);
    }
    return check_launch(hipGetLastError(), what);
}

int neox_pages_truncate(int32_t* page_table, int32_t* lengths, int32_t* free_pages, int32_t* left, const int32_t* keep, int32_t sequences,
                        int32_t columns, int64_t table_stride, int32_t pages, int32_t page_size, void* stream) {
    static const char* what = "neox_pages_truncate";
    PoolArgs a{};
    if (int status = check_pool(a, page_table, lengths, free_pages, left, keep, sequences, columns, table_stride, pages, page_size, what)) return status;
    truncate_kernel<<<1, kPoolThreads, 0, (hipStream_t)stream>>>(a);
    return check_launch(hipGetLastError(), what);
}

}  // extern "C"
#pragma GCC visibility pop
