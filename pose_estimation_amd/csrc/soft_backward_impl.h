// Launchers of the backward kernels for one arithmetic (included by soft_backward_f32.hip and soft_backward_bf16.hip).
#pragma once
#include "soft_backward.h"
#include "soft_launch.h"

namespace ispa_soft {

// channels of the gradients that one launch forms
template <typename T, int DP>
constexpr int kFormed = DP == 256 && std::is_same_v<T, F32> ? 128 : DP;

template <typename T, int DP, int WQ, int MODE>
int dq_one(Params p, hipStream_t stream) {
    static unsigned long long lds_allowed = 0;
    constexpr int kMost = most_lds_bytes<Math<T, DP>, DP>(2);
    const int lds = lds_bytes<Math<T, DP>, DP>(p.shared, 2);
    const unsigned grid = (unsigned)((int64_t)p.B * p.heads * p.splits * p.blocks);
    constexpr int NC = kFormed<T, DP>;
    for (p.c0 = 0; p.c0 < p.D; p.c0 += NC)
        if (int rc = launch(soft_dq_kernel<T, DP, WQ, NC, MODE>, p, grid, 64 * WQ, lds, kMost, &lds_allowed, "soft_dq_kernel", stream))
            return rc;
    return ISPA_OK;
}

template <typename T, int DP, int WQ, int PART, int MODE>
int dkv_one(Params p, int channels, hipStream_t stream) {
    static unsigned long long lds_allowed = 0;
    constexpr int kLds = lds_bytes<Math<T, DP>, DP>(false, 2);
    const unsigned grid = (unsigned)((int64_t)p.B * p.heads * p.splits * p.blocks);
    constexpr int NC = PART == 2 ? kFormed<T, DP> : DP;
    for (p.c0 = 0; p.c0 < channels; p.c0 += NC)
        if (int rc = launch(soft_dkv_kernel<T, DP, WQ, PART, NC, MODE>, p, grid, 64 * WQ, kLds, kLds, &lds_allowed, "soft_dkv_kernel",
                            stream))
            return rc;
    return ISPA_OK;
}

template <typename T, int DP, int WQ, int MODE>
int dkv_parts(const Params &p, hipStream_t stream) {
    if constexpr (dkv_two_launches(!std::is_same_v<T, BF16>, DP, WQ)) {
        if (int rc = dkv_one<T, DP, WQ, 1, MODE>(p, p.Dv, stream)) return rc;
        return dkv_one<T, DP, WQ, 2, MODE>(p, p.D, stream);
    } else {
        return dkv_one<T, DP, WQ, 0, MODE>(p, DP, stream);
    }
}

template <typename T>
int sum_parts(const float *a, const float *b, int splits, int64_t n, float factor, void *out, hipStream_t stream) {
    soft_sum_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a, b, splits, n, factor, (typename T::elem *)out);
    return ispa::check_launch("soft_sum_kernel");
}

template <typename T, int DP>
int dq_waves(const Params &p, int waves, hipStream_t stream) {
    if constexpr (!std::is_same_v<T, F32> || DP == 256)
        if (waves > 1)
            return with_mode<T, DP>(p, true, [&](auto mode) { return dq_one<T, DP, 4, decltype(mode)::value>(p, stream); });
    if constexpr (!std::is_same_v<T, F32S>)
        if (waves == 1) return dq_one<T, DP, 1, kGeneral>(p, stream);
    return ispa::fail(ISPA_EUNSUPPORTED, "no gradient kernel for %d waves", waves);
}

template <typename T, int DP>
int dkv_waves(const Params &p, int waves, hipStream_t stream) {
    if constexpr (!std::is_same_v<T, F32> || DP == 256)
        if (waves > 1)
            return with_mode<T, DP>(p, p.query_xy == nullptr,
                                    [&](auto mode) { return dkv_parts<T, DP, 4, decltype(mode)::value>(p, stream); });
    if constexpr (!std::is_same_v<T, F32S>)
        if (waves == 1) return dkv_parts<T, DP, 1, kGeneral>(p, stream);
    return ispa::fail(ISPA_EUNSUPPORTED, "no gradient kernel for %d waves", waves);
}

// The arithmetic of each launch for float32 maps; bfloat16 has one.
template <typename T, int DP, typename F>
int with_arithmetic(int waves, F f) {
    if constexpr (std::is_same_v<T, F32> && DP <= 128)
        if (arithmetic(true, false, DP, waves) == kSplit) return f(F32S{});
    return f(T{});
}

template <typename T, int DP>
int backward_sized(Params p, const Plan &dq, const Plan &dkv, hipStream_t stream) {
    const bool f32 = !std::is_same_v<T, BF16>;
    p.splits = dq.splits;
    p.parts = dq.splits > 1;
    p.blocks = dq.blocks;
    const int64_t rows = tile_rows(arithmetic(f32, false, DP, dq.waves));
    p.tiles = p.tiles_per_view = (int)((p.cells + rows - 1) / rows);
    // without queries there is no workgroup to launch; the gradients of the maps are still to be written (zeros)
    if (p.nq > 0)
        if (int rc = with_arithmetic<T, DP>(dq.waves, [&](auto t) { return dq_waves<decltype(t), DP>(p, dq.waves, stream); })) return rc;
    const int64_t bh = (int64_t)p.B * p.heads;
    if (p.parts)
        if (int rc = sum_parts<T>(p.part_a, nullptr, p.splits, bh * p.D * p.nq, p.scale, p.dq, stream)) return rc;
    p.splits = dkv.splits;
    p.parts = dkv.splits > 1;
    p.blocks = dkv.blocks;
    if (int rc = with_arithmetic<T, DP>(dkv.waves, [&](auto t) { return dkv_waves<decltype(t), DP>(p, dkv.waves, stream); }))
        return rc;
    if (!p.parts) return ISPA_OK;
    if (p.shared) return sum_parts<T>(p.part_a, p.part_b, p.splits, bh * p.D * p.cells, 1.f, p.dk, stream);
    if (int rc = sum_parts<T>(p.part_a, nullptr, p.splits, bh * p.D * p.cells, 1.f, p.dk, stream)) return rc;
    return sum_parts<T>(p.part_b, nullptr, p.splits, bh * p.Dv * p.cells, 1.f, p.dv, stream);
}

template <typename T>
int backward_channels(const Params &p, const Plan &dq, const Plan &dkv, hipStream_t stream) {
    switch (padded_channels(p.D, p.Dv)) {
        case 32: return backward_sized<T, 32>(p, dq, dkv, stream);
        case 64: return backward_sized<T, 64>(p, dq, dkv, stream);
        case 128: return backward_sized<T, 128>(p, dq, dkv, stream);
        default: return backward_sized<T, 256>(p, dq, dkv, stream);
    }
}

}  // namespace ispa_soft
