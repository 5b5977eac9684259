// Host side of the soft-correspondence kernels: how a call is cut into workgroups, and the launchers per arithmetic.
#pragma once
#include <cmath>
#include <cstdint>

#include "soft_tile.h"

namespace ispa_soft {

inline int padded_channels(int d, int dv) {
    const int m = d > dv ? d : dv;
    return m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256;
}

// How the owned cells are dealt to workgroups of `waves` waves (32 cells each) and the streamed tiles to `splits`.
struct Plan {
    int waves, blocks, splits;
};

constexpr int kMaxSplitCount = 1024;

// Workgroups of four waves for more than 64 owned cells.  Up to that all the parallelism lies in the streamed tiles, and
// four waves would stage for one or two that have cells.
inline int waves_for(int64_t owned) { return owned <= 64 ? 1 : 4; }

// The arithmetic of a launch.  float32 maps run on bfloat16 MFMAs, six products for one (F32S), 2.7 times the rate of the
// float32 MFMAs (64x64x128: 60 us, with float32 MFMAs 95), but stream copies of three planes and keep them in registers: not
// for 256 channels, and not for few queries, which read a map once.  Codes need no copies.
enum Arithmetic { kNarrow, kSplit, kFloat };
inline Arithmetic arithmetic(bool f32, bool codes, int padded, int waves) {
    return !f32 ? kNarrow : codes || (padded <= 128 && waves > 1) ? kSplit : kFloat;
}
inline int64_t tile_rows(Arithmetic a) { return a == kFloat ? 32 : 64; }

// Whether float32 queries against codes come as columns of planes (F32Q): as many as three times fit a wave's 32 columns, with
// a free group for sums over rows of 16 lanes.  One query against 24 views of 128x128x256: 58 us, with three products
// and a wave a SIMD 90 us.
inline bool few_columns(bool f32, int64_t owned) { return f32 && owned <= 8; }

// resident: workgroups that a compute unit holds.  The tiles are split so that the rounds of
// workgroups that the 256 compute units work off, each as long as its tiles and about two more to start, are shortest; a
// split costs its workgroup about four tiles more, for writing and joining its part.
inline Plan make_plan(int64_t owned, int64_t groups, int64_t tiles, int resident) {
    Plan plan;
    plan.waves = waves_for(owned);
    plan.blocks = (int)((owned + 32 * plan.waves - 1) / (32 * plan.waves));
    plan.splits = 1;
    const int64_t base = groups * plan.blocks, room = 256 * resident;
    int64_t best = INT64_MAX;
    for (int64_t s = 1; s <= tiles && s <= kMaxSplitCount && (s == 1 || base * (s - 1) < 4 * room); ++s) {
        const int64_t cost = (base * s + room - 1) / room * ((tiles + s - 1) / s + (s > 1 ? 6 : 2));
        if (cost < best) {
            best = cost;
            plan.splits = (int)s;
        }
    }
    return plan;
}

// Whether the gradients of the reference and value maps take a launch each.
constexpr bool dkv_two_launches(bool f32, int padded, int waves) { return padded == 256 || (padded == 128 && (f32 || waves > 1)); }

// Every launcher expects p.blocks, p.splits, p.tiles and p.tiles_per_view to be set; 0 or a negative status.
int forward_f32(const Params &p, int waves, hipStream_t stream);
int forward_bf16(const Params &p, int waves, hipStream_t stream);
int forward_codes_f32(const Params &p, bool fp8, int waves, hipStream_t stream);
int forward_codes_bf16(const Params &p, bool fp8, int waves, hipStream_t stream);
int backward_f32(const Params &p, const Plan &dq, const Plan &dkv, hipStream_t stream);
int backward_bf16(const Params &p, const Plan &dq, const Plan &dkv, hipStream_t stream);

// Calls f with the mode that the kernels of four waves are built for; `grid`: the streamed cells lie on the grid.  256
// channels have the general form alone.
template <typename T, int DP, typename F>
int with_mode(const Params &p, bool grid, F f) {
    const bool cap = p.cap > 0.f, pen = p.falloff != nullptr;
    if constexpr (DP <= 128) {
        if (!cap && !pen) return f(std::integral_constant<int, kPlain>{});
        if constexpr (std::is_same_v<T, BF16>)
            if (cap && !pen && p.cap <= kFixedCap) return f(std::integral_constant<int, kCapped>{});
        if (!cap && grid && p.W % Math<T, DP>::kCells == 0 && std::fabs(p.scale) > 1e-6f)
            return f(std::integral_constant<int, kRows>{});
    }
    return f(std::integral_constant<int, kGeneral>{});
}

// most: what the kernel's calls take at most, which the first one that needs a permission asks for.
template <typename K>
int launch(K kernel, const Params &p, unsigned grid, int threads, int lds, int most, unsigned long long *lds_allowed, const char *what,
           hipStream_t stream) {
    if (lds > 65536)
        if (int rc = ispa::allow_dynamic_lds((const void *)kernel, most, lds_allowed)) return rc;
    kernel<<<grid, threads, lds, stream>>>(p);
    return ispa::check_launch(what);
}

}  // namespace ispa_soft
