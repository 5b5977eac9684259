// Soft correspondence, backward.  With P recomputed from the stored log-sum (see soft_tile.h for the tile scheme):
//   delta_i = sum_c do_ci o_ci - dlse_i      dP_ij = sum_c do_ci v_cj      dx_ij = P_ij (dP_ij - delta_i) (1 - tanh^2)
//   dq_ci = scale sum_j dx_ij k_cj           dk_cj = scale sum_i dx_ij q_ci           dv_cj = sum_i P_ij do_ci
// Two kernels, one per owned side: scores and dP are formed twice (7 products instead of 5; 8 where the gradients of reference
// and value take a launch each, see dkv_two_launches: scores three times), and in exchange no gradient is summed with
// atomics - every sum has a fixed order and two runs agree bit for bit.  P and dx are rounded to bfloat16 for the products of
// bfloat16 maps (2^-9 of a weight on average, beside the result's own rounding; in two terms of bfloat16 the kernels of up to
// 64 channels took 30 to 40 % longer).
//
// What bounds it (MI355X): 16 pairs of 64x64x128, bfloat16, reference and value one map: forward 0.16, query gradient 0.19,
// value's part 0.16, reference's 0.22 ms; in the gradients the matrix pipe is 38 to 47 % busy, the vector ALU 44 to 54 %,
// together 89 to 92 %.
// float32, 8 pairs of 28x28x128: 0.21 ms for all, two to four tiles a workgroup, half of it the start and end of workgroups.
#pragma once
#include "soft_forward.h"

namespace ispa_soft {

// Registers for two waves a SIMD: one's products run under the other's exponentials.
template <typename T, int DP, int WQ>
constexpr bool two_waves = DP <= 128 && WQ > 1 && std::is_same_v<T, BF16>;

// delta (B,heads,nq); 0 for queries that are not live or have no cell.
template <typename T>
__global__ __launch_bounds__(256) void soft_delta_kernel(const Params p, const float *o32, const float *d_lse,
                                                         float *delta) {
    __shared__ float part[8][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int64_t per = (p.nq + 31) / 32;
    const int64_t bh = blockIdx.x / per;
    const int64_t q = (blockIdx.x - bh * per) * 32 + lane;
    const bool in = q < p.nq && q < live_queries(p, (int)(bh / p.heads));
    float s = 0.f;
    if (in) {
        const typename T::elem *a = (const typename T::elem *)p.d_out + bh * p.Dv * p.nq + q;
        const float *o = o32 + bh * p.Dv * p.nq + q;
#pragma unroll 8
        for (int c = g; c < p.Dv; c += 8) s = fmaf(load_float(a + c * p.nq), o[c * p.nq], s);
    }
    part[g][lane] = s;
    __syncthreads();
    if (g != 0 || q >= p.nq) return;
    s = ((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane])) +
        ((part[4][lane] + part[5][lane]) + (part[6][lane] + part[7][lane]));
    const bool some = in && p.lse[bh * p.nq + q] != -__builtin_inff();
    if (d_lse != nullptr && in) s -= d_lse[bh * p.nq + q];
    delta[bh * p.nq + q] = some ? s : 0.f;
}

// A weight from its log in units of log2.  The log-sum is off by its own rounding, 2^-24 of itself: scores beyond 2^31 would
// overflow without the bound (which costs nothing: a modifier of the instruction).
__device__ __forceinline__ float probability(float x) { return __builtin_amdgcn_fmed3f(exp2_(x), 0.f, 1.f); }

// From products `acc` and w = -(falloff d^2) + minus_lse: w = P and the slope 1 - tanh^2, or at once dx / scale with dP in `dp`.
template <typename T, int MODE>
__device__ __forceinline__ void probabilities(const Score<T> &score, const f32x16 &acc, float (&w)[16], float (&slope)[16]) {
    if (MODE == kPlain || MODE == kRows || (MODE == kGeneral && !score.cap)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = probability(fmaf(score.in, acc[i], w[i]));
    } else if (Score<T>::kExact || (MODE == kGeneral && score.exact)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float th = score.bend(acc[i], slope[i]);
            w[i] = probability(fmaf(score.top, th, w[i]));
        }
    } else {
        // tanh = 1 - 2 r; the cap itself is in w
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = score.two_r(acc[i], slope[i]);
            w[i] = probability(fmaf(-score.top, x, w[i]));
        }
    }
}
template <typename T, int MODE>
__device__ __forceinline__ void weights(const Score<T> &score, const f32x16 &acc, float (&w)[16], const f32x16 &dp,
                                        float delta) {
    if (MODE == kPlain || MODE == kRows || (MODE == kGeneral && !score.cap)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = probability(fmaf(score.in, acc[i], w[i])) * (dp[i] - delta);
    } else if (Score<T>::kExact || (MODE == kGeneral && score.exact)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float slope;
            const float th = score.bend(acc[i], slope);
            w[i] = probability(fmaf(score.top, th, w[i])) * ((dp[i] - delta) * slope);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float slope;
            const float x = score.two_r(acc[i], slope);
            w[i] = probability(fmaf(-score.top, x, w[i])) * ((dp[i] - delta) * slope);
        }
    }
}
// -lse in log2 units, with what probabilities() expects beside: the cap where tanh is taken as 1 - 2 r.
template <typename T, int MODE>
__device__ __forceinline__ float minus_lse(const Score<T> &score, float lse) {
    if (lse == -__builtin_inff()) return -__builtin_inff();    // no cells: weights 0
    const bool cap = MODE == kCapped || (MODE == kGeneral && score.cap);
    return fmaf(-kLog2e, lse, !Score<T>::kExact && cap && !(MODE == kGeneral && score.exact) ? score.top : 0.f);
}

// Both kernels can form their gradients for NC channels at a time, from p.c0 on.  A launch per half is what 256 float32
// channels take: two owned operands and a whole accumulator would need more than a lane's 512 registers.
//
// Gradient of the queries: owned = queries, streamed = cells.
template <typename T, int DP, int WQ, int NC, int MODE>
__global__ __launch_bounds__(64 * WQ, (two_waves<T, DP, WQ>) ? 2 : 1) void soft_dq_kernel(const Params p) {
    typedef Math<T, DP> M;
    constexpr int kBlocks = M::kRows / 32;
    constexpr int kUnroll = DP == 256 ? 1 : kBlocks;           // registers
    constexpr uint64_t kAll = M::kRows == 64 ? ~0ull : 0xffffffffull;
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
    const int q = (qblk * WQ + wave) * 32 + (lane & 31);
    const bool q_ok = q < live_q;
    const bool idle = qblk * WQ * 32 >= live_q;
    const int t0 = (int)((int64_t)p.tiles * split / p.splits);
    const int t1 = idle ? t0 : (int)((int64_t)p.tiles * (split + 1) / p.splits);

    typename M::Owned qf, of;
    M::load_owned(qf, (const typename T::elem *)p.q + (int64_t)bh * p.D * p.nq, q < nq ? q : 0, p.nq, p.D, q_ok, h);
    M::load_owned(of, (const typename T::elem *)p.d_out + (int64_t)bh * p.Dv * p.nq, q < nq ? q : 0, p.nq, p.Dv, q_ok, h);
    const typename M::Addr addr = M::addr(lane);
    const Score<T> score(p, head);
    float qx = 0.f, qy = 0.f;
    if (p.falloff != nullptr && q_ok) query_place(p, b, q, qx, qy);
    float minus = -__builtin_inff(), delta = 0.f;
    if (q_ok) {
        minus = minus_lse<T, MODE>(score, p.lse[(int64_t)bh * p.nq + q]);
        delta = p.delta[(int64_t)bh * p.nq + q];
    }
    f32x16 g[NC / 32];
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) g[c][i] = 0.f;

    Feed<T, T, DP, WQ, 2> feed(p, b, head, t0, lds);
    const bool phased = kMayPhase<M> && feed.phased;
    const Penalty<M, MODE, false> penalty(p, score.fall, qx, qy);
    const f32x16 from = penalty.from(score.in);
    uint64_t next = 0;                                         // live cells of the next tile
    int next_cell0 = 0;
    auto finish = [&](int i) {
        next = feed.end_k(i, penalty.wants_places());
        if (!phased) feed.end_v(i, next);
        next_cell0 = feed.keys.cell0;
    };
    if (t0 < t1) {
        feed.begin_k(0);
        if (!phased) feed.begin_v(0);
        finish(0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int i = (t - t0) & 1, j = i ^ 1;
        if (phased) {
            feed.begin_v(0);
        } else if (t + 1 < t1) {
            feed.begin_k(j);
            feed.begin_v(j);
        }
        const uint64_t live = next;
        const int cell0 = next_cell0;
        const char *ktile = feed.k(i), *vtile = feed.v(i);
        const float *cell = feed.cell(i);
        f32x16 ahead[kMayPhase<M> ? kBlocks : 1];              // products of the first map, where they come a phase before
        if constexpr (kMayPhase<M>) {
            if (live != 0) M::first(ktile, addr, 0, qf, ahead);
            if (phased) {
                feed.end_v(0, live);
                __syncthreads();                               // the value's tile is there
                if (t + 1 < t1) feed.begin_k(j);
            }
        }
        if (live != 0) {
#pragma unroll kUnroll
            for (int k = 0; k < kBlocks; ++k) {
                if (DP == 256) __builtin_amdgcn_sched_barrier(0);
                f32x16 acc[1], dp[1];
                if constexpr (kMayPhase<M>) acc[0] = ahead[k];
                else M::first(ktile, addr, k, qf, acc, from);
                M::first(vtile, addr, k, of, dp);
                float w[16];
                if (MODE == kRows || penalty.on) {
                    penalty(cell + 64, cell0, k, h, minus, w);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = minus;
                }
                weights<T, MODE>(score, acc[0], w, dp[0], delta);
                if (live != kAll) {
                    stay_branch();
                    const unsigned bits = (unsigned)(live >> (32 * k)) >> M::cell(0, h);
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = bits & (1u << M::cell(i, 0)) ? w[i] : 0.f;
                }
                M::second(ktile + p.c0 * kRowBytes, addr, k, M::weights(w), g);
            }
        }
        if (t + 1 < t1) finish(j);
        __syncthreads();
    }
    LateParams &e = late_params();
    if (q >= e.nq) return;
    if (e.parts) {
#pragma unroll
        for (int c = 0; c < NC / 32; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) g[c][i] = q_ok ? g[c][i] : 0.f;
        store_columns<NC>(e.part_a + ((int64_t)split * e.B * e.heads + bh) * e.D * e.nq, e.nq, q, h, e.c0, e.D, g);
        return;
    }
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) g[c][i] = q_ok ? g[c][i] * e.scale : 0.f;
    store_columns<NC>((typename T::elem *)e.dq + (int64_t)bh * e.D * e.nq, e.nq, q, h, e.c0, e.D, g);
}

// Gradients of the reference and value maps: owned = cells, streamed = queries.  PART 0: both; 1: the value's, 2: the
// reference's alone: two launches and a fifth product, which pays where it brings two waves to a SIMD, and which the
// registers ask for above 128 channels.
template <typename T, int DP, int WQ, int PART, int NC, int MODE>
__global__ __launch_bounds__(64 * WQ, (two_waves<T, DP, WQ> && (DP <= 64 || PART != 0)) ? 2 : 1) void soft_dkv_kernel(const Params p) {
    typedef Math<T, DP> M;
    constexpr int kBlocks = M::kRows / 32;
    constexpr int kUnroll = !kMayPhase<M> && (DP == 256 || (DP == 128 && PART == 2)) ? 1 : kBlocks;           // registers
    constexpr bool kDv = PART != 2, kDk = PART != 1;
    constexpr uint64_t kAll = M::kRows == 64 ? ~0ull : 0xffffffffull;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    out_of_step();

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    int id = die_major(blockIdx.x, gridDim.x);
    const int blk = id % p.blocks;
    id /= p.blocks;
    const int split = id % p.splits;
    const int bh = id / p.splits;
    const int b = bh / p.heads, head = bh - b * p.heads;
    const int live_q = (int)live_queries(p, b);                // fewer than 2^22
    const int tiles = (live_q + M::kRows - 1) / M::kRows;
    const int t0 = (int)((int64_t)tiles * split / p.splits), t1 = (int)((int64_t)tiles * (split + 1) / p.splits);
    const int cell = (blk * WQ + wave) * 32 + (lane & 31), cells = (int)p.cells;   // fewer than 2^22
    const bool c_ok = cell < cells && (p.mask == nullptr || p.mask[(int64_t)b * p.cells + cell] != 0);
    const float cx = (float)(cell % p.W), cy = (float)(cell / p.W);

    typename M::Owned kf, vf;
    M::load_owned(kf, (const typename T::elem *)p.k + (int64_t)bh * p.D * p.cells, cell < cells ? cell : 0, p.cells, p.D,
                  c_ok, h);
    if constexpr (kDk)
        M::load_owned(vf, (const typename T::elem *)p.v + (int64_t)bh * p.Dv * p.cells, cell < cells ? cell : 0, p.cells, p.Dv,
                      c_ok, h);
    const typename M::Addr addr = M::addr(lane);
    const Score<T> score(p, head);
    f32x16 gk[kDk ? NC / 32 : 1], gv[kDv ? NC / 32 : 1];
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (kDk) gk[c][i] = 0.f;
            if constexpr (kDv) gv[c][i] = 0.f;
        }

    const Penalty<M, MODE, std::is_same_v<T, BF16>> penalty(p, score.fall, cx, cy);
    const f32x16 from = penalty.from(score.in);
    // buffers as in Feed: twice (query tile, per query -log-sum, -delta and place), then the gradient's tiles, of which
    // three planes leave room for one
    typedef Direct<M, DP, WQ> Copy;
    constexpr bool phased = kMayPhase<M>;
    constexpr int kTile = kTileBytes<M, DP>, kStage = kTile + kCellBytes;
    Copy cq, co;
    cq.init(p.sq, bh);
    co.init(p.so, bh);
    for (int i = 0; i < 2; ++i) {
        cq.clear_rest(lds + i * kStage);
        if (i == 0 || !phased) co.clear_rest(lds + 2 * kStage + i * kTile);
    }
    float minus = 0.f, delta = 0.f, px = 0.f, py = 0.f;
    auto live_of = [&](int t) {                                // what lies behind the live queries counts as zeros
        const int left = live_q - t * M::kRows;
        return left < M::kRows ? (1ull << left) - 1 : kAll;
    };
    auto begin_q = [&](int t, int i) {
        const int q0 = t * M::kRows;
        if (threadIdx.x < M::kRows) {
            const int q = q0 + (int)threadIdx.x;
            minus = -__builtin_inff();
            delta = 0.f;
            if (q < live_q) {
                minus = minus_lse<T, MODE>(score, p.lse[(int64_t)bh * p.nq + q]);
                delta = p.delta[(int64_t)bh * p.nq + q];
                if (penalty.wants_places()) query_place(p, b, q, px, py);
            }
        }
        cq.issue(q0, (int)p.sq.ld, lds + i * kStage);
    };
    auto begin_o = [&](int t, int i) { co.issue(t * M::kRows, (int)p.so.ld, lds + 2 * kStage + i * kTile); };
    auto end_q = [&](int t, int i) {
        Copy::wait();
        const uint64_t live = live_of(t);
        if (live != kAll) cq.mask(lds + i * kStage, live);
        if (threadIdx.x < M::kRows) {
            float *cell = reinterpret_cast<float *>(lds + i * kStage + kTile) + threadIdx.x;
            cell[0] = minus;
            cell[64] = -delta;
            cell[128] = px;
            cell[192] = py;
        }
    };
    auto end_o = [&](int t, int i) {
        Copy::wait();
        const uint64_t live = live_of(t);
        if (live != kAll) co.mask(lds + 2 * kStage + i * kTile, live);
    };
    if (t0 < t1) {
        begin_q(t0, 0);
        if (!phased) begin_o(t0, 0);
        end_q(t0, 0);
        if (!phased) end_o(t0, 0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int i = (t - t0) & 1, j = i ^ 1;
        const char *qtile = lds + i * kStage, *otile = lds + 2 * kStage + (phased ? 0 : i) * kTile;
        const float *larr = reinterpret_cast<const float *>(qtile + kTile);
        const float *darr = larr + 64, *xarr = larr + 128;
        auto minus_delta = [&](int k) {                        // what dP is added to
            float v[16];
            M::per_cell(darr, k, h, v);
            f32x16 x;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = v[i];
            return x;
        };
        f32x16 ahead[phased ? kBlocks : 1];                    // scores, where they come a phase before the rest
        if constexpr (phased) {
            begin_o(t, 0);
            if constexpr (PART == 2) {                         // block by block: fewer fragments in registers
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) {
                    f32x16 acc[1];
                    M::template first<1, MODE != kGeneral>(qtile, addr, k, kf, acc, from);
                    ahead[k] = acc[0];
                }
            } else {
                M::first(qtile, addr, 0, kf, ahead, from);
            }
            end_o(t, 0);
            __syncthreads();                                   // the gradient's tile is there
            if (t + 1 < t1) begin_q(t + 1, j);
        } else if (t + 1 < t1) {
            begin_q(t + 1, j);
            begin_o(t + 1, j);
        }
#pragma unroll kUnroll
        for (int k = 0; k < kBlocks; ++k) {
            if constexpr (phased) __builtin_amdgcn_sched_barrier(0);
            f32x16 acc[1];
            if constexpr (phased) acc[0] = ahead[k];
            else M::first(qtile, addr, k, kf, acc, from);
            float w[16];
            if (MODE == kRows || penalty.on) {
                penalty(xarr, t * M::kRows, k, h, 0.f, w);
                float minus_l[16];
                M::per_cell(larr, k, h, minus_l);
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] += minus_l[i];
            } else {
                M::per_cell(larr, k, h, w);
            }
            if constexpr (kDv) {
                float slope[16];
                probabilities<T, MODE>(score, acc[0], w, slope);
                M::second(otile + p.c0 * kRowBytes, addr, k, M::weights(w), gv);
                if constexpr (kDk) {
                    f32x16 dp[1];
                    M::first(otile, addr, k, vf, dp, minus_delta(k));
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] *= dp[0][i];
                    if (MODE == kCapped || (MODE == kGeneral && score.cap))
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] *= slope[i];
                }
            } else {
                f32x16 dp[1];
                M::template first<1, !(phased && MODE == kGeneral)>(otile, addr, k, vf, dp, minus_delta(k));
                weights<T, MODE>(score, acc[0], w, dp[0], 0.f);
            }
            if constexpr (kDk) M::second(qtile + p.c0 * kRowBytes, addr, k, M::weights(w), gk);
        }
        if (t + 1 < t1) {
            end_q(t + 1, j);
            if (!phased) end_o(t + 1, j);
        }
        __syncthreads();
    }
    LateParams &e = late_params();
    if (cell >= e.cells) return;
    // masked cells take no part: their columns hold zeros' products and are dropped here
    const int64_t part = (int64_t)split * e.B * e.heads + bh;
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (kDk) gk[c][i] = c_ok ? gk[c][i] * e.scale : 0.f;
            if constexpr (kDv) gv[c][i] = c_ok ? gv[c][i] : 0.f;
        }
    typedef typename T::elem elem;
    float *pv = e.part_b + part * e.Dv * e.cells;
    elem *dk = (elem *)e.dk + (int64_t)bh * e.D * e.cells, *dv = (elem *)e.dv + (int64_t)bh * e.Dv * e.cells;
    if (e.parts) {
        if constexpr (kDk) store_columns<NC>(e.part_a + part * e.D * e.cells, e.cells, cell, h, e.c0, e.D, gk);
        if constexpr (kDv) store_columns<NC>(pv, e.cells, cell, h, e.c0, e.Dv, gv);
    } else if (!e.shared) {
        if constexpr (kDk) store_columns<NC>(dk, e.cells, cell, h, e.c0, e.D, gk);
        if constexpr (kDv) store_columns<NC>(dv, e.cells, cell, h, e.c0, e.Dv, gv);
    } else if constexpr (PART == 1) {                          // shared: the sum of both uses, rounded once
        store_columns<NC>(pv, e.cells, cell, h, e.c0, e.Dv, gv);       // float32, for the launch that forms the other one
    } else {
#pragma unroll
        for (int c = 0; c < NC / 32; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int ch = e.c0 + 32 * c + out_channel(i, h);
                if constexpr (PART == 2) gk[c][i] += ch < e.D ? pv[ch * e.cells + cell] : 0.f;
                else gk[c][i] += gv[c][i];
            }
        store_columns<NC>(dk, e.cells, cell, h, e.c0, e.D, gk);
    }
}

// out[i] = factor * sum_s a[s][i] (+ sum_s b[s][i]), in the order of s, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void soft_sum_kernel(const float *a, const float *b, int splits, int64_t n, float factor,
                                                       typename T::elem *out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float x = 0.f, y = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) x += a[s * n + i];
    x *= factor;
    if (b != nullptr) {
#pragma unroll 4
        for (int s = 0; s < splits; ++s) y += b[s * n + i];
        x += y;
    }
    store_float(out + i, x);
}

}  // namespace ispa_soft
