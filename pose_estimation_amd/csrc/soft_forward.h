// Soft correspondence, forward: out = softmax_j(z_ij) v_j in one pass over the streamed cells (see soft_tile.h), with a
// running maximum m and sum l per query (float32, in units of log2).
//
// What bounds it (MI355X):
//   bfloat16, many queries: 64 pairs of 64x64x128 with a falloff 0.58 to 0.62 ms, by the card, 0.89 to 0.95 PFLOP/s, 64 to 69 % of
//   what a large matrix product reaches.  The matrix pipe is busy 43 % of the cycles and the vector ALU 54 %, one after the
//   other: two waves a SIMD, with unequal priorities, hide waits but not each other's issue.  Hence one operation a cell for
//   the falloff (Penalty), the lazy rescale (kSlack), the fixed maximum of kCapped.  Reading value fragments ahead, or
//   exponentials between the products, cost 3 to 5 % more cycles.
//   float32, many queries: six bfloat16 products for one, 64x64x128 58 to 62 us, 139 to 148 TFLOP/s, where a float32 matrix
//   product reaches 153; copying the maps into planes takes 4 us of it.
//   few queries: 10 against 28x28x128 in 12 us and 4 to join: a launch, a query column's loads, one tile, its stores.
#pragma once
#include "soft_tile.h"

namespace ispa_soft {

// The streamed cells of one item, tile after tile; tile t lies in view t / tiles_per_view of the item.
template <typename M, typename SRC>
struct KeyTiles {
    static constexpr bool kCodes = std::is_same_v<SRC, I8> || std::is_same_v<SRC, FP8>;
    const Params &p;
    int b, head;
    int view, left;            // of the next tile: its view, the view's tiles from it on
    int64_t map;               // the view's map in the store (-1: none); without a store the batch item's
    int cell0;                 // of the present tile
    __device__ __forceinline__ KeyTiles(const Params &p_, int b_, int head_, int t) : p(p_), b(b_), head(head_), map(b_) {
        if constexpr (kCodes) {
            view = t / p.tiles_per_view;
            left = (view + 1) * p.tiles_per_view - t;
            find();
        }
        cell0 = (kCodes ? p.tiles_per_view - left : t) * M::kRows - M::kRows;
    }
    __device__ __forceinline__ void find() {
        const int id = view < p.V ? p.views[(int64_t)b * p.V + view] : -1;
        map = id >= 0 && id < p.n_view ? id : -1;
    }
    __device__ __forceinline__ void next() {
        cell0 += M::kRows;
        if constexpr (kCodes) {
            if (left == 0) {
                ++view;
                left = p.tiles_per_view;
                cell0 = 0;
                find();
            }
            --left;
        }
    }
    __device__ __forceinline__ const typename SRC::elem *base(const void *maps, int d) const {
        return (const typename SRC::elem *)maps + ((map < 0 ? 0 : map) * p.heads + head) * (int64_t)d * p.cells;
    }
    // this lane's cell (lane % kRows) of the present tile: whether the map has it; then whether it takes part, its scale
    __device__ __forceinline__ bool inside(int lane) const { return map >= 0 && cell0 + (lane & (M::kRows - 1)) < (int)p.cells; }
    __device__ __forceinline__ uint8_t taken(int lane, bool in) const {
        return p.mask == nullptr ? (uint8_t)1 : in ? p.mask[map * p.cells + cell0 + (lane & (M::kRows - 1))] : (uint8_t)0;
    }
    __device__ __forceinline__ float scale(int lane, bool in) const {
        if constexpr (kCodes) return in ? p.kscale[map * p.cells + cell0 + (lane & (M::kRows - 1))] : 0.f;
        return 0.f;
    }
};

__device__ __forceinline__ void query_place(const Params &p, int b, int64_t i, float &x, float &y) {
    if (p.query_xy != nullptr) {
        const float *xy = p.query_xy + ((int64_t)b * p.nq + i) * 2;
        x = xy[0];
        y = xy[1];
    } else {
        x = (float)((int)i % p.W);
        y = (float)((int)i / p.W);
    }
}

// How tiles and products take turns.  Two buffers for each map, the next tile on its way during all products of the
// present one: where that fits LDS.  Else (three planes a map, reference and value apart) the value's tile is copied
// during the first products and the reference's next one during the second, with a barrier between: `phased`.
template <typename M>
constexpr bool kMayPhase = M::kPlanes == 3;

// LDS: NK times (reference tile, 3 or 4 x 64 floats per cell), then the value tiles.
constexpr int kCellBytes = 4 * 64 * (int)sizeof(float);
template <typename M, int DP>
constexpr int kTileBytes = M::kPlanes * DP * kRowBytes;
// Codes of a lone wave take one buffer: the next tile waits in registers until the present one's products are done.
template <typename SRC, int WQ>
constexpr bool kOneBuffer = WQ == 1 && (std::is_same_v<SRC, I8> || std::is_same_v<SRC, FP8>);
template <typename M, int DP>
constexpr int lds_bytes(bool shared, int phased_k, bool one = false) {
    const bool phased = kMayPhase<M> && !shared;
    return (phased ? phased_k : one ? 1 : 2) * (kTileBytes<M, DP> + kCellBytes) + (shared ? 0 : phased ? 1 : 2) * kTileBytes<M, DP>;
}
// The larger of both: a value map of its own may take less, as it is copied in phases.
template <typename M, int DP>
constexpr int most_lds_bytes(int phased_k) {
    const int shared = lds_bytes<M, DP>(true, phased_k), own = lds_bytes<M, DP>(false, phased_k);
    return shared > own ? shared : own;
}

// The tiles of one item and head: begin_* starts a tile's way into a buffer, end_* ends it.  Codes are reference and value.
// PK: buffers of the reference's tiles where phased.
template <typename T, typename SRC, int DP, int WQ, int PK>
struct Feed {
    typedef Math<T, DP> M;
    typedef KeyTiles<M, SRC> Keys;
    static constexpr bool kCodes = Keys::kCodes;
    static constexpr uint64_t kAll = M::kRows == 64 ? ~0ull : 0xffffffffull;
    static constexpr int kStage = kTileBytes<M, DP> + kCellBytes;
    typedef Loader<M, SRC, DP, 64 * WQ> L;
    typedef Direct<M, DP, WQ> D;
    struct None {
        static constexpr bool kAhead = true;
    };
    // the next tile's loads may run during the present tile's products
    static constexpr bool kAhead = std::conditional_t<kCodes, L, None>::kAhead;
    const Params &p;
    Keys keys;
    std::conditional_t<kCodes, L, None> codes;
    std::conditional_t<kCodes, None, D> dk, dv;
    bool in = false;           // of this lane's cell in the present tile, as KeyTiles says
    uint8_t taken = 0;
    float sc = 0.f;
    char *lds;
    int v_at;                  // of the first value tile
    bool phased;
    __device__ __forceinline__ Feed(const Params &p_, int b, int head, int t, char *lds_)
        : p(p_), keys(p_, b, head, t), lds(lds_) {
        phased = kMayPhase<M> && !p.shared;
        v_at = (phased ? PK : 2) * kStage;
        if constexpr (!kCodes) {
            const int64_t bh = (int64_t)b * p.heads + head;
            dk.init(p.sk, bh);
            for (int i = 0; i < (phased ? PK : 2); ++i) dk.clear_rest(lds + i * kStage);
            if (!p.shared) {
                dv.init(p.sv, bh);
                for (int i = 0; i < (phased ? 1 : 2); ++i) dv.clear_rest(lds + v_at + i * kTileBytes<M, DP>);
            }
        }
    }
    __device__ __forceinline__ char *k(int i) const { return lds + i * kStage; }
    __device__ __forceinline__ char *v(int i) const { return p.shared ? k(i) : lds + v_at + (phased ? 0 : i) * kTileBytes<M, DP>; }
    __device__ __forceinline__ const float *cell(int i) const { return reinterpret_cast<const float *>(k(i) + kTileBytes<M, DP>); }
    __device__ __forceinline__ void begin_k(int i) {           // the next tile
        const int lane = threadIdx.x & 63;
        keys.next();
        in = keys.inside(lane);
        taken = keys.taken(lane, in);
        if constexpr (kCodes) {
            sc = keys.scale(lane, in);
            codes.load(keys.base(p.k, p.D), p.cells, p.D, keys.cell0, keys.map < 0 ? 0 : p.cells);
        } else {
            dk.issue(keys.cell0, (int)p.sk.ld, k(i));
        }
    }
    __device__ __forceinline__ void begin_v(int i) {           // the tile of the last begin_k
        if constexpr (!kCodes)
            if (!p.shared) dv.issue(keys.cell0, (int)p.sv.ld, v(i));
    }
    // the tile's live cells; places: their coordinates are wanted in LDS
    __device__ __forceinline__ uint64_t end_k(int i, bool places) {
        const bool ok = in && taken != 0;
        const uint64_t live = __ballot(ok) & kAll;
        if constexpr (!kCodes) D::wait();
        if (live == 0) return live;                            // the same in every wave
        float *cell = reinterpret_cast<float *>(k(i) + kTileBytes<M, DP>);
        if constexpr (kCodes) {
            codes.store(k(i), p.cells, p.D, live);
            if (threadIdx.x < 64) cell[threadIdx.x] = ok ? sc : 0.f;
        } else if (live != kAll) {
            dk.mask(k(i), live);
        }
        if (places && threadIdx.x < M::kRows) {
            const int c = keys.cell0 + threadIdx.x;
            cell[64 + threadIdx.x] = (float)(c % p.W);
            cell[128 + threadIdx.x] = (float)(c / p.W);
        }
        return live;
    }
    __device__ __forceinline__ void end_v(int i, uint64_t live) {
        if constexpr (!kCodes) {
            if (p.shared) return;
            D::wait();
            if (live != 0 && live != kAll) dv.mask(v(i), live);
        }
    }
};

// Registers for two waves a SIMD: one's products run under the other's exponentials.
template <typename T, typename SRC, int DP, int WQ>
constexpr bool two_resident = std::is_same_v<SRC, BF16> || (kOneBuffer<SRC, WQ> && !std::is_same_v<T, F32C>)
                                  ? DP <= 128 : std::is_same_v<SRC, F32S> && DP <= 64;

// How far (in units of log2) a query's largest score may rise above the maximum that its sums are kept against before they
// are rescaled: weights stay below 2^8, and nearly all tiles leave the accumulators alone.
constexpr float kSlack = 8.f;
// A tile whose scores rise by more than this over what they were formed against is formed anew, against its own largest: their
// rounding goes by the rise, which a steep falloff makes far larger than the scores that count.
constexpr float kFar = 64.f;

// NC: value channels that one launch forms, from p.c0 on (256 float32 channels take two launches, for the registers).
template <typename T, typename SRC, int DP, int WQ, int NC, int MODE>
__global__ __launch_bounds__(64 * WQ, (two_resident<T, SRC, DP, WQ>) ? 2 : 1) void soft_forward_kernel(const Params p) {
    typedef Math<T, DP> M;
    constexpr int kBlocks = M::kRows / 32;
    constexpr uint64_t kAll = M::kRows == 64 ? ~0ull : 0xffffffffull;
    constexpr bool kCodes = KeyTiles<M, SRC>::kCodes;
    typedef Feed<T, SRC, DP, WQ, 1> F;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    out_of_step();

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    int id = die_major(blockIdx.x, gridDim.x);
    const int qblk = id % p.blocks;
    id /= p.blocks;
    const int split = id % p.splits;
    const int bh = id / p.splits;
    const int b = bh / p.heads, head = bh - b * p.heads;
    const int live_q = (int)live_queries(p, b), nq = (int)p.nq;            // fewer than 2^22
    const int q = (qblk * WQ + wave) * M::kColumns + (lane & (M::kColumns - 1));
    const bool q_ok = q < live_q;
    const bool idle = qblk * WQ * M::kColumns >= live_q;       // no live query in the whole workgroup
    const int t0 = (int)((int64_t)p.tiles * split / p.splits);
    const int t1 = idle ? t0 : (int)((int64_t)p.tiles * (split + 1) / p.splits);

    F feed(p, b, head, t0, lds);
    const bool phased = kMayPhase<M> && feed.phased;
    if (F::kAhead && t0 < t1) {                                // the first tile's loads first: the rest hides in them
        feed.begin_k(0);
        if (!phased) feed.begin_v(0);
    }
    typename M::Owned qf;
    M::load_owned(qf, (const typename T::elem *)p.q + (int64_t)bh * p.D * p.nq, q < nq ? q : 0, p.nq, p.D, q_ok, h);
    Score<T> score(p, head);
    if (MODE == kPlain && score.in < 0.f) {                        // largest product = largest score
        M::negate(qf);
        score.in = -score.in;
    }
    if (MODE == kPlain) score.in = fmaxf(score.in, 1e-37f);    // scale 0: products of a masked cell stay -inf
    const typename M::Addr addr = M::addr(lane);
    float qx = 0.f, qy = 0.f;
    if (p.falloff != nullptr && q_ok) query_place(p, b, q, qx, qy);

    f32x16 o[NC / 32];
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
    float m = -__builtin_inff(), l = 0.f;                      // l: this lane's half of the cells
    // what scores are taken relative to (m once there is one), and how far above it they may lie
    float off = 0.f, room = -__builtin_inff();

    const Penalty<M, MODE, !kCodes> penalty(p, score.fall, qx, qy);    // codes: products are yet to be scaled
    const f32x16 from = penalty.from(score.in);
    uint64_t next = 0;                                         // live cells of the next tile
    int next_cell0 = 0;
    auto finish = [&](int i) {
        next = feed.end_k(i, penalty.wants_places());
        if (!phased) feed.end_v(i, next);
        next_cell0 = feed.keys.cell0;
    };
    if (F::kAhead && t0 < t1) finish(0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        constexpr bool kOne = !F::kAhead || kOneBuffer<SRC, WQ>;
        const int i = phased || kOne ? 0 : (t - t0) & 1, j = phased || kOne ? 0 : i ^ 1;
        if constexpr (!F::kAhead) {
            feed.begin_k(0);
            finish(0);
            __syncthreads();
        } else if (phased) {
            feed.begin_v(0);
        } else if (t + 1 < t1) {
            feed.begin_k(j);
            feed.begin_v(j);
        }
        const uint64_t live = next;
        const int cell0 = next_cell0;
        const char *ktile = feed.k(i), *vtile = feed.v(i);
        const float *cell = feed.cell(i);
        f32x16 z[kBlocks] = {};
        auto form = [&]() __attribute__((always_inline)) {
            // z: scores relative to off.  kPlain: the products, scaled in the exponent.  kCapped: relative to the cap, which
            // stands for the maximum: weights are 2^(-2 cap) > 2^-93 at least.
            if constexpr (DP == 256 && kBlocks == 2) {         // block by block: fewer fragments in registers
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) {
                    f32x16 acc[1];
                    M::first(ktile, addr, k, qf, acc, from);
                    z[k] = acc[0];
                }
            } else {
                M::template first<kBlocks, M::kColumns == 32>(ktile, addr, 0, qf, z, from);
            }
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                if constexpr (M::kColumns < 32) M::fold(z[k]);
                if constexpr (kCodes) {
                    float ks[16];
                    M::per_cell(cell, k, h, ks);
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[k][i] *= ks[i];
                }
                if constexpr (MODE == kCapped) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[k][i] = score.below_cap(z[k][i]);
                } else if constexpr (MODE != kPlain) {
                    if constexpr (!std::is_same_v<T, BF16>) __builtin_amdgcn_sched_barrier(0);
                    float d[16];
                    constexpr bool kEarly = M::kColumns < 32 || (kCodes && !M::kWide);     // tanh before there is a d: registers
                    if (kEarly && score.cap) score.template bend<true>(z[k]);
                    if (MODE == kRows || penalty.on) {
                        penalty(cell + 64, cell0, k, h, -off, d);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) d[i] = -off;
                    }
                    if (MODE == kGeneral && score.cap) {
                        if constexpr (!kEarly) score.template bend<false>(z[k]);
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[k][i] = fmaf(score.top, z[k][i], d[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[k][i] = fmaf(score.in, z[k][i], d[i]);
                    }
                }
            }
            if (live != kAll) {
                stay_branch();
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) {
                    const unsigned bits = (unsigned)(live >> (32 * k)) >> M::cell(0, h);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        z[k][i] = bits & (1u << M::cell(i, 0)) ? z[k][i] : -__builtin_inff();
                }
            }
        };
        auto largest = [&]() __attribute__((always_inline)) {
            float top = -__builtin_inff();
#pragma unroll
            for (int k = 0; k < kBlocks; ++k)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, z[k][i]);
            return fmaxf(top, __shfl_xor(top, 32));
        };
        float rel = off;                                       // kPlain: what the exponents are relative to
        if (live != 0) {
            form();
            if constexpr (MODE == kCapped) {
                m = score.top;
            } else {
                const float peak = largest();
                float top = MODE == kPlain ? fmaf(peak, score.in, -off) : peak;
                if (__any(top > room)) {
                    stay_branch();
                    bool far = false;
                    if constexpr (MODE == kRows || MODE == kGeneral) {
                        far = off != 0.f && top > kFar;        // there is a maximum, and the tile lies far above it
                        if (__any(far)) {
                            stay_branch();
                            off = far ? off + top : off;                   // rounded by what a rise takes: z tells how far it is off
                            form();
                            top = largest();
                        }
                    }
                    const float m_new = fmaxf(m, top + off);
                    const bool first = m == -__builtin_inff();
                    const float fix = first ? 0.f : exp2_(m - m_new);
                    m = m_new;
                    room = m == -__builtin_inff() ? m : kSlack;
                    const float was = off;
                    off = m == -__builtin_inff() ? 0.f : m;
                    l *= fix;
#pragma unroll
                    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[c][i] *= fix;
                    // beyond 2^24 the maximum cannot follow the tile's largest score, which still is what weights go by
                    if constexpr (MODE == kPlain) {
                        rel = off;
                        const bool beyond = (first || top > 0.f) && peak > -__builtin_inff() && fabsf(fmaf(peak, score.in, -off)) > 1.f;
                        if (__any(beyond)) {
                            stay_branch();
                            rel = beyond ? 0.f : off;
#pragma unroll
                            for (int k = 0; k < kBlocks; ++k)
#pragma unroll
                                for (int i = 0; i < 16; ++i) z[k][i] -= beyond ? peak : 0.f;
                        }
                    } else {
                        const float rise = off - was, lift = (far || top > 0.f) && fabsf(top - rise) > 1.f ? top : rise;
#pragma unroll
                        for (int k = 0; k < kBlocks; ++k)
#pragma unroll
                            for (int i = 0; i < 16; ++i) z[k][i] -= lift;
                    }
                }
            }
        }
        if constexpr (kMayPhase<M>) {
            if (phased) {
                feed.end_v(0, live);
                __syncthreads();                               // the reference tile is read, the value's is there
                if (t + 1 < t1) feed.begin_k(0);
            }
        }
        if (live != 0) {
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                if constexpr (!std::is_same_v<T, BF16>) __builtin_amdgcn_sched_barrier(0);     // one block's weights at a time
                float w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    w[i] = exp2_(MODE == kPlain ? fmaf(score.in, z[k][i], -rel) : z[k][i]);
                    sum[i & 1] += w[i];
                }
                if constexpr (kCodes) {
                    float ks[16];
                    M::per_cell(cell, k, h, ks);
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] *= ks[i];
                }
                // weights are rounded to bfloat16 for the second product of bfloat16 maps, the sum l is not
                M::second(vtile + p.c0 * kRowBytes, addr, k, M::weights(w), o);
            }
            l += sum[0] + sum[1];
        }
        if (F::kAhead && t + 1 < t1) finish(j);
        __syncthreads();
    }
    l += __shfl_xor(l, 32);
    LateParams &e = late_params();
    int late_lane = lane;
    if constexpr (M::kColumns < 32) {                          // formed anew: a register less through the loop
        late_lane = threadIdx.x & 63;
        asm volatile("" : "+v"(late_lane));
    }
    const int late_h = late_lane >> 5;

    if constexpr (M::kColumns < 32) {
#pragma unroll
        for (int c = 0; c < NC / 32; ++c) M::fold(o[c]);
    }
    if (q >= e.nq || (lane & 31) >= M::kColumns) return;
    if (e.splits > 1) {
        const int64_t part = (int64_t)split * e.B * e.heads + bh;
        if (late_h == 0) {
            const float2 ml = q_ok ? make_float2(m, l) : make_float2(-__builtin_inff(), 0.f);
            *reinterpret_cast<float2 *>(e.part_ml + (part * e.nq + q) * 2) = ml;
        }
        store_columns<NC>(e.part_o + part * e.Dv * e.nq, e.nq, q, late_h, e.c0, e.Dv, o);
        return;
    }
    const bool some = q_ok && l != 0.f;                        // l is 0 only where no cell takes part (NaN is not)
    const float inv = some ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] = some ? o[c][i] * inv : 0.f;
    store_columns<NC>((typename T::elem *)e.out + (int64_t)bh * e.Dv * e.nq, e.nq, q, late_h, e.c0, e.Dv, o);
    if (e.out32 != nullptr) store_columns<NC>(e.out32 + (int64_t)bh * e.Dv * e.nq, e.nq, q, late_h, e.c0, e.Dv, o);
    if (late_h == 0 && e.lse != nullptr)
        e.lse[(int64_t)bh * e.nq + q] = some ? (m + log2f(l)) * kLn2 : -__builtin_inff();
}

// Joins the partial results of a split call: M = max m_s, out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.
// A block joins QB queries; their parts' weights lie in LDS.  The other 256 / QB threads of a query are dealt to channels
// (many queries, few parts) or, for at most 64 queries, to parts, whose sums meet in LDS in a fixed order.
constexpr int kMaxSplits = 1024, kManySplits = 64;
template <typename T>
__global__ __launch_bounds__(256) void soft_join_kernel(const Params p, int channels_per_block) {
    constexpr int QB = 32, kLanes = 256 / QB;
    __shared__ float w[kManySplits][QB], ls[kManySplits][QB];
    const int qi = threadIdx.x % QB, g = threadIdx.x / QB;
    const int bh = blockIdx.y;
    const int64_t q = (int64_t)blockIdx.x * QB + qi;
    const bool in = q < p.nq;
    const int64_t bhn = (int64_t)p.B * p.heads;
    for (int s = g; s < p.splits; s += kLanes) {
        const float2 ml = in ? *reinterpret_cast<const float2 *>(p.part_ml + ((s * bhn + bh) * p.nq + q) * 2)
                             : make_float2(-__builtin_inff(), 0.f);
        w[s][qi] = ml.x;
        ls[s][qi] = ml.y;
    }
    __syncthreads();
    float top = -__builtin_inff();
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, w[s][qi]);
    if (top == -__builtin_inff()) top = 0.f;                   // no part has a cell, or all scores are NaN
    float l = 0.f;
    for (int s = 0; s < p.splits; ++s) l = fmaf(exp2_(w[s][qi] - top), ls[s][qi], l);
    if (!in) return;
    const bool some = l != 0.f;
    const float inv = some ? 1.f / l : 0.f;
    const int c1 = min(p.Dv, ((int)blockIdx.z + 1) * channels_per_block);
    for (int c = (int)blockIdx.z * channels_per_block + g; c < c1; c += kLanes) {
        float v = 0.f;
        const float *src = p.part_o + ((int64_t)bh * p.Dv + c) * p.nq + q;
        const int64_t step = bhn * p.Dv * p.nq;
#pragma unroll 8
        for (int s = 0; s < p.splits; ++s) v = fmaf(exp2_(w[s][qi] - top), src[s * step], v);
        v = some ? v * inv : 0.f;
        const int64_t at = ((int64_t)bh * p.Dv + c) * p.nq + q;
        store_float((typename T::elem *)p.out + at, v);
        if (p.out32 != nullptr) p.out32[at] = v;
    }
    if (blockIdx.z == 0 && g == 0 && p.lse != nullptr)
        p.lse[(int64_t)bh * p.nq + q] = some ? (top + log2f(l)) * kLn2 : -__builtin_inff();
}

// 8 queries x 32 part lanes, 2 channels a block: latency is all there is, so many blocks with loads 16 at a time (1024 parts of
// 256 channels: 7 us; 8 channels a block, a part after the other: 16 us).
constexpr int kJoinChannels = 2;
template <typename T>
__global__ __launch_bounds__(256) void soft_join_few_kernel(const Params p) {
    constexpr int kPer = kMaxSplits / 32;                      // parts of a lane
    __shared__ float part[kJoinChannels][32][8];
    const int qi = threadIdx.x & 7, g = threadIdx.x >> 3;
    const int bh = blockIdx.y;
    const int64_t q = (int64_t)blockIdx.x * 8 + qi;
    const bool in = q < p.nq;
    const int64_t bhn = (int64_t)p.B * p.heads;
    const int c0 = (int)blockIdx.z * kJoinChannels;
    float m[kPer], l = 0.f, v[kJoinChannels] = {}, top = -__builtin_inff();
    float ls[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int s = g + 32 * i;
        const float2 ml = in && s < p.splits ? *reinterpret_cast<const float2 *>(p.part_ml + ((s * bhn + bh) * p.nq + q) * 2)
                                             : make_float2(-__builtin_inff(), 0.f);
        m[i] = ml.x;
        ls[i] = ml.y;
        top = fmaxf(top, ml.x);
    }
    part[0][g][qi] = top;
    __syncthreads();
    for (int i = 0; i < 32; ++i) top = fmaxf(top, part[0][i][qi]);
    if (top == -__builtin_inff()) top = 0.f;                   // no part has a cell, or all scores are NaN
    __syncthreads();
    // parts past the last one count with weight 0, from the first one's place: kBatch loads go out at once
    constexpr int kBatch = 8;
    const int cq = in ? (int)q : 0;
    const int64_t step = bhn * p.Dv * p.nq;
    const float *first = p.part_o + ((int64_t)bh * p.Dv + c0) * p.nq + cq;
    const int64_t second = c0 + 1 < p.Dv ? p.nq : 0;
#pragma unroll
    for (int i0 = 0; i0 < kPer; i0 += kBatch) {
        if (32 * i0 >= p.splits) break;                        // uniform
        float x[kBatch][kJoinChannels];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int s = g + 32 * (i0 + i);
            const float *src = first + (s < p.splits ? s : 0) * step;
            x[i][0] = src[0];
            x[i][1] = src[second];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const bool there = g + 32 * (i0 + i) < p.splits;
            const float w = there ? exp2_(m[i0 + i] - top) : 0.f;
            l = fmaf(w, ls[i0 + i], l);
#pragma unroll
            for (int c = 0; c < kJoinChannels; ++c) v[c] = there ? fmaf(w, x[i][c], v[c]) : v[c];
        }
    }
    part[0][g][qi] = l;
    __syncthreads();
    l = 0.f;
    for (int i = 0; i < 32; ++i) l += part[0][i][qi];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kJoinChannels; ++c) part[c][g][qi] = v[c];
    __syncthreads();
    const bool some = l != 0.f;
    if (in && g < kJoinChannels && c0 + g < p.Dv) {
        float x = 0.f;
        for (int i = 0; i < 32; ++i) x += part[g][i][qi];
        x = some ? x / l : 0.f;
        const int64_t at = ((int64_t)bh * p.Dv + c0 + g) * p.nq + q;
        store_float((typename T::elem *)p.out + at, x);
        if (p.out32 != nullptr) p.out32[at] = x;
    }
    if (in && blockIdx.z == 0 && g == 0 && p.lse != nullptr)
        p.lse[(int64_t)bh * p.nq + q] = some ? (top + log2f(l)) * kLn2 : -__builtin_inff();
}

}  // namespace ispa_soft
