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
    }
}

template <>
hipError_t launch_attn_fwd<NEOX_ATTN_DIM>(const AttnArgs& a, int source, int dtype, hipStream_t stream) {
    if (dtype == NEOX_BF16) a.splits > 1 ? forward<BF16, true>(a, source, stream) : forward<BF16, false>(a, source, stream);
    else a.splits > 1 ? forward<F16, true>(a, source, stream) : forward<F16, false>(a, source, stream);
    return hipGetLastError();
}

template <>
hipError_t launch_attn_token<NEOX_ATTN_DIM>(const AttnArgs& a, int source, int dtype, hipStream_t stream) {
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
