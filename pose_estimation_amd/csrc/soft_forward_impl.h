// Launchers of the forward kernels for one arithmetic (included by the soft_forward_*.hip files).
#pragma once
#include "soft_forward.h"
#include "soft_launch.h"

namespace ispa_soft {
static_assert(kMaxSplits == kMaxSplitCount, "the join reads every part");

template <typename T, typename SRC, int DP, int WQ, int MODE>
int forward_one(Params p, hipStream_t stream) {
    static unsigned long long lds_allowed = 0;
    // codes are reference and value in one
    constexpr bool kOne = kOneBuffer<SRC, WQ>;
    constexpr int kMost = KeyTiles<Math<T, DP>, SRC>::kCodes ? lds_bytes<Math<T, DP>, DP>(true, 1, kOne) : most_lds_bytes<Math<T, DP>, DP>(1);
    const int lds = lds_bytes<Math<T, DP>, DP>(p.shared, 1, kOne);
    const unsigned grid = (unsigned)((int64_t)p.B * p.heads * p.splits * p.blocks);
    constexpr int NC = DP == 256 && !std::is_same_v<T, BF16> && !std::is_same_v<T, F32Q> ? 128 : DP;
    for (p.c0 = 0; p.c0 < p.Dv; p.c0 += NC)
        if (int rc = launch(soft_forward_kernel<T, SRC, DP, WQ, NC, MODE>, p, grid, 64 * WQ, lds, kMost, &lds_allowed, "soft_forward_kernel",
                            stream))
            return rc;
    if (p.splits == 1) return ISPA_OK;
    const unsigned bh = (unsigned)(p.B * p.heads);
    if (WQ == 1 || p.splits > kManySplits) {
        soft_join_few_kernel<T><<<dim3((unsigned)((p.nq + 7) / 8), bh, (unsigned)((p.Dv + kJoinChannels - 1) / kJoinChannels)), 256,
                                  0, stream>>>(p);
    } else {
        const int per = 32;                                   // channels of a block
        soft_join_kernel<T><<<dim3((unsigned)((p.nq + 31) / 32), bh, (unsigned)((p.Dv + per - 1) / per)), 256, 0, stream>>>(p, per);
    }
    return ispa::check_launch("soft_join_kernel");
}

template <typename T, typename SRC, int DP>
int forward_waves(const Params &p, int waves, hipStream_t stream) {
    // F32S: more than 64 queries and up to 128 channels; F32: the rest
    if constexpr (!std::is_same_v<T, F32Q> && (!std::is_same_v<T, F32> || DP == 256))
        if (waves > 1)
            return with_mode<T, DP>(p, true, [&](auto mode) { return forward_one<T, SRC, DP, 4, decltype(mode)::value>(p, stream); });
    if constexpr (!std::is_same_v<T, F32S>)
        if (waves == 1) return forward_one<T, SRC, DP, 1, kGeneral>(p, stream);
    return ispa::fail(ISPA_EUNSUPPORTED, "no forward kernel for %d waves", waves);
}

template <typename T, typename SRC>
int forward_channels(const Params &p, int waves, hipStream_t stream) {
    switch (padded_channels(p.D, p.Dv)) {
        case 32: return forward_waves<T, SRC, 32>(p, waves, stream);
        case 64: return forward_waves<T, SRC, 64>(p, waves, stream);
        case 128: return forward_waves<T, SRC, 128>(p, waves, stream);
        default:
            if constexpr (!std::is_same_v<T, F32S>) return forward_waves<T, SRC, 256>(p, waves, stream);
    }
    return ispa::fail(ISPA_EUNSUPPORTED, "no forward kernel for %d channels", p.D);
}

}  // namespace ispa_soft
