// Host side of the soft-correspondence kernels: how a call is cut into workgroups, and the launchers per arithmetic.
#pragma once
#include "soft_tile.h"

namespace ispa_soft {

// Codes a template store holds, or the maps' own type.
enum Source { kSourceMap = 0, kSourceInt8 = 1, kSourceFp8 = 2 };

inline int padded_channels(int d, int dv) {
    const int m = d > dv ? d : dv;
    return m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256;
}

// How the owned cells are dealt to workgroups of `waves` waves (32 cells each) and the streamed tiles to `splits`.
struct Plan {
    int waves, blocks, splits;
};

constexpr int kMaxSplitCount = 512;

inline Plan make_plan(int64_t owned, int64_t groups, int64_t tiles) {
    Plan plan;
    plan.waves = owned <= 64 ? 1 : 4;
    plan.blocks = (int)((owned + 32 * plan.waves - 1) / (32 * plan.waves));
    const int64_t base = groups * plan.blocks, want = plan.waves == 1 ? 2048 : 512;
    int64_t s = base >= want / 2 ? 1 : (want + base - 1) / base;
    if (s > tiles / 2) s = tiles / 2;
    if (s > kMaxSplitCount) s = kMaxSplitCount;
    plan.splits = s < 1 ? 1 : (int)s;
    return plan;
}

// Whether the gradients of the reference and value maps are summed from float32 parts: where the queries are split, and
// where two launches form the two uses of a shared map of more than 128 channels (one rounding of their sum).
inline bool dkv_in_parts(int d, int dv, bool shared, int splits) {
    return splits > 1 || (shared && padded_channels(d, dv) == 256);
}

// Every launcher expects p.blocks, p.splits, p.tiles and p.tiles_per_view to be set; 0 or a negative status.
int forward_f32(const Params &p, int source, int waves, hipStream_t stream);
int forward_bf16(const Params &p, int source, int waves, hipStream_t stream);
int backward_f32(const Params &p, const Plan &dq, const Plan &dkv, hipStream_t stream);
int backward_bf16(const Params &p, const Plan &dq, const Plan &dkv, hipStream_t stream);

template <typename K>
int launch(K kernel, const Params &p, unsigned grid, int threads, int lds, unsigned long long *lds_allowed, const char *what,
           hipStream_t stream) {
    if (lds > 65536)
        if (int rc = ispa::allow_dynamic_lds((const void *)kernel, lds, lds_allowed)) return rc;
    kernel<<<grid, threads, lds, stream>>>(p);
    return ispa::check_launch(what);
}

}  // namespace ispa_soft
