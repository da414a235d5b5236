// The attention kernels of one padded head dim (-DNEOX_ATTN_DIM) and their launchers.
#include "internal.hpp"

namespace neox {

template <typename T, bool SPLIT>
static void forward(const AttnArgs& a, int source, hipStream_t stream) {
    constexpr int DP = NEOX_ATTN_DIM;
    const dim3 grid((uint32_t)a.b * a.kv * a.row_tiles, SPLIT ? a.splits : 1);
    switch (source) {
        case kStrided:
            if constexpr (!SPLIT) attn_fwd_kernel<T, DP, kStrided, false><<<grid, 256, 0, stream>>>(a);
            break;
        case kPaged16: attn_fwd_kernel<T, DP, kPaged16, SPLIT><<<grid, 256, 0, stream>>>(a); break;
        case kPagedI8: attn_fwd_kernel<T, DP, kPagedI8, SPLIT><<<grid, 256, 0, stream>>>(a); break;
        case kPagedF8: attn_fwd_kernel<T, DP, kPagedF8, SPLIT><<<grid, 256, 0, stream>>>(a); break;
        case kPagedF4:
            if constexpr (DP == 256) {
                if (padded4(a.d) == 160) {
                    attn_fwd_kernel<T, 160, kPagedF4, SPLIT><<<grid, 256, 0, stream>>>(a);
                    break;
                }
            }
            attn_fwd_kernel<T, DP, kPagedF4, SPLIT><<<grid, 256, 0, stream>>>(a);
            break;
    }
}

template <typename T, bool SPLIT>
static void token(const AttnArgs& a, int source, hipStream_t stream) {
    constexpr int DP = NEOX_ATTN_DIM;
    const uint32_t grid = ((uint32_t)a.b * a.splits + 7) / 8 * 8 * a.kv;
    switch (source) {
        case kPaged16: attn_token_kernel<T, DP, kPaged16, SPLIT><<<grid, 256, 0, stream>>>(a); break;
        case kPagedI8: attn_token_kernel<T, DP, kPagedI8, SPLIT><<<grid, 256, 0, stream>>>(a); break;
        case kPagedF8: attn_token_kernel<T, DP, kPagedF8, SPLIT><<<grid, 256, 0, stream>>>(a); break;
        case kPagedF4: break;  // (token4)
    }
}

template <typename T, int DP, bool SPLIT, int WAVES>
static void token4(AttnArgs a, hipStream_t stream) {
    const int fetch = token4_fetch(a, DP), groups = a.kv / a.heads * a.row_tiles;
    a.by_kv = FastDiv::by((uint32_t)groups);
    const dim3 grid(((uint32_t)a.b * a.splits + 7) / 8 * 8 * groups), threads(64 * WAVES);
    if (fetch == kFetchOwn) {
        attn_token4_kernel<T, DP, 1, SPLIT, kFetchOwn, WAVES><<<grid, threads, 0, stream>>>(a);
    } else if (fetch == kFetchHalves) {
        // (of 96 and 160 dims: always rows)
        if constexpr (DP != 96 && DP != 160) attn_token4_kernel<T, DP, 1, SPLIT, kFetchHalves, WAVES><<<grid, threads, 0, stream>>>(a);
    } else if (a.heads == 1) {
        attn_token4_kernel<T, DP, 1, SPLIT, kFetchRows, WAVES><<<grid, threads, 0, stream>>>(a);
    } else {
        if constexpr (DP <= 128 && WAVES == 4) attn_token4_kernel<T, DP, 2, SPLIT, kFetchRows, WAVES><<<grid, threads, 0, stream>>>(a);
    }
}
template <typename T, int DP>
static void token4_of(const AttnArgs& a, hipStream_t stream) {
    if (a.splits > 1) token4<T, DP, true, 4>(a, stream);
    else if (a.waves == 8) token4<T, DP, false, 8>(a, stream);
    else token4<T, DP, false, 4>(a, stream);
}
template <typename T>
static void token4(const AttnArgs& a, hipStream_t stream) {
    constexpr int DP = NEOX_ATTN_DIM;
    if constexpr (DP == 256) {
        if (padded4(a.d) == 160) return token4_of<T, 160>(a, stream);
    }
    token4_of<T, DP>(a, stream);
}

template <>
hipError_t launch_attn_fwd<NEOX_ATTN_DIM>(const AttnArgs& a, int source, int dtype, hipStream_t stream) {
    if (dtype == NEOX_BF16) a.splits > 1 ? forward<BF16, true>(a, source, stream) : forward<BF16, false>(a, source, stream);
    else a.splits > 1 ? forward<F16, true>(a, source, stream) : forward<F16, false>(a, source, stream);
    return hipGetLastError();
}

template <>
hipError_t launch_attn_token<NEOX_ATTN_DIM>(const AttnArgs& a, int source, int dtype, hipStream_t stream) {
    if (source == kPagedF4) {
        dtype == NEOX_BF16 ? token4<BF16>(a, stream) : token4<F16>(a, stream);
        return hipGetLastError();
    }
    if (dtype == NEOX_BF16) a.splits > 1 ? token<BF16, true>(a, source, stream) : token<BF16, false>(a, source, stream);
    else a.splits > 1 ? token<F16, true>(a, source, stream) : token<F16, false>(a, source, stream);
    return hipGetLastError();
}

// the queries' kernel first: it leaves the rows' sums of dO * O that the keys' kernel needs
template <typename T>
static void backward(const AttnArgs& a, hipStream_t stream) {
    constexpr int DP = NEOX_ATTN_DIM;
    const uint32_t q = (uint32_t)a.b * a.kv * a.row_tiles, kv = (uint32_t)a.b * a.kv * a.units;
    attn_bwd_q_kernel<T, DP><<<q, 256, 0, stream>>>(a);
    if constexpr (DP <= 128) {
        attn_bwd_kv_kernel<T, DP, true, true><<<kv, 256, 0, stream>>>(a);
    } else {
        attn_bwd_kv_kernel<T, DP, true, false><<<kv, 256, 0, stream>>>(a);
        attn_bwd_kv_kernel<T, DP, false, true><<<kv, 256, 0, stream>>>(a);
    }
}

template <>
hipError_t launch_attn_bwd<NEOX_ATTN_DIM>(const AttnArgs& a, int dtype, hipStream_t stream) {
    dtype == NEOX_BF16 ? backward<BF16>(a, stream) : backward<F16>(a, stream);
    if (a.near_parts > 1 || a.far_parts > 0) {
        const dim3 grid((uint32_t)a.b * a.kv * (kGradKeys / 32), a.near_parts > 1 ? a.key_tiles : a.sink_tiles);
        dtype == NEOX_BF16 ? attn_bwd_join_kernel<BF16><<<grid, 256, 0, stream>>>(a) : attn_bwd_join_kernel<F16><<<grid, 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace neox
