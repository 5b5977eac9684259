// Soft correspondence, forward: out = softmax_j(z_ij) v_j in one pass over the streamed cells (see soft_tile.h), with a
// running maximum m and sum l per query (float32, in units of log2).
#pragma once
#include "soft_tile.h"

namespace ispa_soft {

// The streamed cells of one item: tile t lies in view t / tiles_per_view of the item.
template <typename M, typename SRC>
struct KeyTiles {
    static constexpr bool kCodes = std::is_same_v<SRC, I8> || std::is_same_v<SRC, FP8>;
    const Params &p;
    int b, head;
    __device__ __forceinline__ KeyTiles(const Params &p_, int b_, int head_) : p(p_), b(b_), head(head_) {}
    struct At {
        int64_t map;          // which map of the batch or store; -1 = none
        int64_t cell0;
    };
    __device__ __forceinline__ At at(int t) const {
        At a;
        if constexpr (kCodes) {
            const int view = t / p.tiles_per_view;
            const int id = p.views[(int64_t)b * p.V + view];
            a.map = id >= 0 && id < p.n_view ? id : -1;
            a.cell0 = (int64_t)(t - view * p.tiles_per_view) * M::kRows;
        } else {
            a.map = b;
            a.cell0 = (int64_t)t * M::kRows;
        }
        return a;
    }
    __device__ __forceinline__ const typename SRC::elem *base(const void *maps, const At &a, int d) const {
        return (const typename SRC::elem *)maps + ((a.map < 0 ? 0 : a.map) * p.heads + head) * (int64_t)d * p.cells;
    }
    // this lane's cell (lane % kRows) of the tile: takes part?  its scale
    __device__ __forceinline__ bool live(const At &a, int lane) const {
        const int64_t c = a.cell0 + (lane & (M::kRows - 1));
        if (a.map < 0 || c >= p.cells) return false;
        return p.mask == nullptr || p.mask[a.map * p.cells + c] != 0;
    }
    __device__ __forceinline__ float scale(const At &a, int lane, bool ok) const {
        if constexpr (kCodes) return ok ? p.kscale[a.map * p.cells + a.cell0 + (lane & (M::kRows - 1))] : 0.f;
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
template <typename M, int DP>
constexpr int lds_bytes(bool shared, int phased_k) {
    const bool phased = kMayPhase<M> && !shared;
    return (phased ? phased_k : 2) * (kTileBytes<M, DP> + kCellBytes) + (shared ? 0 : phased ? 1 : 2) * kTileBytes<M, DP>;
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
    const Keys keys;
    std::conditional_t<kCodes, L, None> codes;
    std::conditional_t<kCodes, None, D> dk, dv;
    typename Keys::At at{};
    bool ok = false;
    float sc = 0.f;
    char *lds;
    int v_at;                  // of the first value tile
    bool phased;
    __device__ __forceinline__ Feed(const Params &p_, int b, int head, char *lds_) : p(p_), keys(p_, b, head), lds(lds_) {
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
    __device__ __forceinline__ void begin_k(int t, int i) {
        const int lane = threadIdx.x & 63;
        at = keys.at(t);
        ok = keys.live(at, lane);
        if constexpr (kCodes) {
            sc = keys.scale(at, lane, ok);
            codes.load(keys.base(p.k, at, p.D), p.cells, p.D, at.cell0, at.map < 0 ? 0 : p.cells);
        } else {
            dk.issue((int)at.cell0, (int)p.sk.ld, k(i));
        }
    }
    __device__ __forceinline__ void begin_v(int i) {           // the tile of the last begin_k
        if constexpr (!kCodes)
            if (!p.shared) dv.issue((int)at.cell0, (int)p.sv.ld, v(i));
    }
    __device__ __forceinline__ uint64_t end_k(int i) {         // the tile's live cells
        const uint64_t live = __ballot(ok) & kAll;
        if constexpr (!kCodes) D::wait();
        if (live == 0) return live;                            // the same in every wave
        float *cell = reinterpret_cast<float *>(k(i) + kTileBytes<M, DP>);
        if constexpr (kCodes) {
            codes.store(k(i), p.cells, p.D, live);
            if (threadIdx.x < 64) cell[threadIdx.x] = sc;
        } else if (live != kAll) {
            dk.mask(k(i), live);
        }
        if (p.falloff != nullptr && p.W % M::kCells != 0 && threadIdx.x < M::kRows) {
            const int c = (int)at.cell0 + threadIdx.x;
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

// How far (in units of log2) a query's largest score may rise above the maximum that its sums are kept against before they
// are rescaled: weights stay below 2^8, and nearly all tiles leave the accumulators alone.
constexpr float kSlack = 8.f;

// NC: value channels that one launch forms, from p.c0 on (256 float32 channels take two launches, for the registers).
template <typename T, typename SRC, int DP, int WQ, int NC, int MODE>
__global__ __launch_bounds__(64 * WQ, (DP <= 128 && std::is_same_v<SRC, BF16>) ? 2 : 1) void soft_forward_kernel(const Params p) {
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
    const int64_t live_q = live_queries(p, b);
    const int64_t q = ((int64_t)qblk * WQ + wave) * 32 + (lane & 31);
    const bool q_ok = q < live_q;
    const bool idle = (int64_t)qblk * WQ * 32 >= live_q;       // no live query in the whole workgroup
    const int t0 = (int)((int64_t)p.tiles * split / p.splits);
    const int t1 = idle ? t0 : (int)((int64_t)p.tiles * (split + 1) / p.splits);

    typename M::Owned qf;
    M::load_owned(qf, (const typename T::elem *)p.q + (int64_t)bh * p.D * p.nq + (q < p.nq ? q : 0), p.nq, p.D, q_ok, h);
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

    F feed(p, b, head, lds);
    const bool phased = kMayPhase<M> && feed.phased;
    const Penalty<M, MODE> penalty(p, score.fall, qx, qy, true);
    const f32x16 from = penalty.from(score.in);
    uint64_t next = 0;                                         // live cells of the next tile
    int next_cell0 = 0;
    auto finish = [&](int i) {
        next = feed.end_k(i);
        if (!phased) feed.end_v(i, next);
        next_cell0 = (int)feed.at.cell0;
    };
    if (F::kAhead && t0 < t1) {
        feed.begin_k(t0, 0);
        if (!phased) feed.begin_v(0);
        finish(0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int i = phased || !F::kAhead ? 0 : (t - t0) & 1, j = phased || !F::kAhead ? 0 : i ^ 1;
        if constexpr (!F::kAhead) {
            feed.begin_k(t, 0);
            finish(0);
            __syncthreads();
        } else if (phased) {
            feed.begin_v(0);
        } else if (t + 1 < t1) {
            feed.begin_k(t + 1, j);
            feed.begin_v(j);
        }
        const uint64_t live = next;
        const int cell0 = next_cell0;
        const char *ktile = feed.k(i), *vtile = feed.v(i);
        const float *cell = feed.cell(i);
        f32x16 z[kBlocks];
        if (live != 0) {
            // z: scores relative to off.  kPlain: the products, scaled in the exponent.  kCapped: relative to the cap, which
            // stands for the maximum: weights are 2^(-2 cap) > 2^-93 at least.
            M::first(ktile, addr, 0, qf, z, from);
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                if constexpr (kCodes) {
                    float ks[16];
                    M::per_cell(cell, k, h, ks);
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[k][i] *= ks[i];
                }
                if constexpr (MODE == kCapped) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[k][i] = (-2.f * score.top) * score.r(z[k][i]);
                } else if constexpr (MODE != kPlain) {
                    float d[16];
                    if (MODE == kRows || penalty.on) {
                        penalty(cell + 64, cell0, k, h, -off, d);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) d[i] = -off;
                    }
                    if (MODE == kGeneral && score.cap) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[k][i] = fmaf(score.top, score.bend(z[k][i]), d[i]);
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
            if constexpr (MODE == kCapped) {
                m = score.top;
            } else {
                float top = -__builtin_inff();
#pragma unroll
                for (int k = 0; k < kBlocks; ++k)
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, z[k][i]);
                if (MODE == kPlain) top = fmaf(top, score.in, -off);
                top = fmaxf(top, __shfl_xor(top, 32));
                if (__any(top > room)) {
                    stay_branch();
                    const float m_new = fmaxf(m, top + off);
                    const float fix = m == -__builtin_inff() ? 0.f : exp2_(m - m_new);
                    m = m_new;
                    room = m == -__builtin_inff() ? m : kSlack;
                    const float was = off;
                    off = m == -__builtin_inff() ? 0.f : m;
                    l *= fix;
#pragma unroll
                    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[c][i] *= fix;
                    if constexpr (MODE != kPlain)
#pragma unroll
                        for (int k = 0; k < kBlocks; ++k)
#pragma unroll
                            for (int i = 0; i < 16; ++i) z[k][i] -= off - was;
                }
            }
        }
        if constexpr (kMayPhase<M>) {
            if (phased) {
                feed.end_v(0, live);
                __syncthreads();                               // the reference tile is read, the value's is there
                if (t + 1 < t1) feed.begin_k(t + 1, 0);
            }
        }
        if (live != 0) {
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                float w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    w[i] = exp2_(MODE == kPlain ? fmaf(score.in, z[k][i], -off) : z[k][i]);
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

    if (q >= p.nq) return;
    if (p.splits > 1) {
        const int64_t part = (int64_t)split * p.B * p.heads + bh;
        if (h == 0) {
            const float2 ml = q_ok ? make_float2(m, l) : make_float2(-__builtin_inff(), 0.f);
            *reinterpret_cast<float2 *>(p.part_ml + (part * p.nq + q) * 2) = ml;
        }
        store_columns<NC>(p.part_o + part * p.Dv * p.nq, p.nq, q, h, p.c0, p.Dv, o);
        return;
    }
    const bool some = q_ok && l != 0.f;                        // l is 0 only where no cell takes part (NaN is not)
    const float inv = some ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] = some ? o[c][i] * inv : 0.f;
    store_columns<NC>((typename T::elem *)p.out + (int64_t)bh * p.Dv * p.nq, p.nq, q, h, p.c0, p.Dv, o);
    if (p.out32 != nullptr) store_columns<NC>(p.out32 + (int64_t)bh * p.Dv * p.nq, p.nq, q, h, p.c0, p.Dv, o);
    if (h == 0 && p.lse != nullptr)
        p.lse[(int64_t)bh * p.nq + q] = some ? (m + log2f(l)) * kLn2 : -__builtin_inff();
}

// Joins the partial results of a split call: M = max m_s, out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.
// A block joins QB queries; their parts' weights lie in LDS.
constexpr int kMaxSplits = 512;
template <typename T, int QB>
__global__ __launch_bounds__(256) void soft_join_kernel(const Params p, int channels_per_block) {
    constexpr int kMost = QB == 8 ? kMaxSplits : kMaxSplits / 8, kLanes = 256 / QB;
    __shared__ float w[kMost][QB], ls[kMost][QB];
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
    __syncthreads();
    if (top == -__builtin_inff()) top = 0.f;                   // no part has a cell, or all scores are NaN
    for (int s = g; s < p.splits; s += kLanes) w[s][qi] = exp2_(w[s][qi] - top);
    __syncthreads();
    float l = 0.f;
    for (int s = 0; s < p.splits; ++s) l = fmaf(w[s][qi], ls[s][qi], l);
    if (!in) return;
    const bool some = l != 0.f;
    const float inv = some ? 1.f / l : 0.f;
    const int c1 = min(p.Dv, ((int)blockIdx.z + 1) * channels_per_block);
    for (int c = (int)blockIdx.z * channels_per_block + g; c < c1; c += kLanes) {
        float v = 0.f;
        const float *src = p.part_o + ((int64_t)bh * p.Dv + c) * p.nq + q;
        const int64_t step = bhn * p.Dv * p.nq;
#pragma unroll 8
        for (int s = 0; s < p.splits; ++s) v = fmaf(w[s][qi], src[s * step], v);
        v = some ? v * inv : 0.f;
        const int64_t at = ((int64_t)bh * p.Dv + c) * p.nq + q;
        store_float((typename T::elem *)p.out + at, v);
        if (p.out32 != nullptr) p.out32[at] = v;
    }
    if (blockIdx.z == 0 && g == 0 && p.lse != nullptr)
        p.lse[(int64_t)bh * p.nq + q] = some ? (top + log2f(l)) * kLn2 : -__builtin_inff();
}

}  // namespace ispa_soft
