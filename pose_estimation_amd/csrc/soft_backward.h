// Soft correspondence, backward.  With P recomputed from the stored log-sum (see soft_tile.h for the tile scheme):
//   delta_i = sum_c do_ci o_ci - dlse_i      dP_ij = sum_c do_ci v_cj      dx_ij = P_ij (dP_ij - delta_i) (1 - tanh^2)
//   dq_ci = scale sum_j dx_ij k_cj           dk_cj = scale sum_i dx_ij q_ci           dv_cj = sum_i P_ij do_ci
// Two kernels, one per owned side: scores and dP are formed twice (7 products instead of 5), and in exchange no gradient
// is summed with atomics - every sum has a fixed order and two runs agree bit for bit.
#pragma once
#include "soft_forward.h"

namespace ispa_soft {

// delta (B,heads,nq); 0 for queries that are not live or have no cell.
template <typename T>
__global__ __launch_bounds__(256) void soft_delta_kernel(const Params p, const float *o32, const float *d_lse,
                                                         float *delta) {
    __shared__ float part[4][64];
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int64_t per = (p.nq + 63) / 64;
    const int64_t bh = blockIdx.x / per;
    const int64_t q = (blockIdx.x - bh * per) * 64 + lane;
    const bool in = q < p.nq && q < live_queries(p, (int)(bh / p.heads));
    float s = 0.f;
    if (in) {
        const typename T::elem *a = (const typename T::elem *)p.d_out + bh * p.Dv * p.nq + q;
        const float *o = o32 + bh * p.Dv * p.nq + q;
#pragma unroll 4
        for (int c = g; c < p.Dv; c += 4) s = fmaf(load_float(a + c * p.nq), o[c * p.nq], s);
    }
    part[g][lane] = s;
    __syncthreads();
    if (g != 0 || q >= p.nq) return;
    s = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    const bool some = in && p.lse[bh * p.nq + q] != -__builtin_inff();
    if (d_lse != nullptr && in) s -= d_lse[bh * p.nq + q];
    delta[bh * p.nq + q] = some ? s : 0.f;
}

// Both kernels can form their gradients for NC channels at a time, from p.c0 on.  A launch per half is what 256 float32
// channels take: two owned operands and a whole accumulator would need more than a lane's 512 registers.
//
// Gradient of the queries: owned = queries, streamed = cells.
template <typename T, int DP, int WQ, int NC>
__global__ __launch_bounds__(64 * WQ) void soft_dq_kernel(const Params p) {
    typedef Math<T, DP> M;
    constexpr int NT = 64 * WQ;
    constexpr int kBlocks = M::kRows / 32;
    constexpr int kUnroll = DP == 256 ? 1 : kBlocks;           // registers
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char *ktile = lds;
    char *vtile = p.shared ? lds : lds + DP * kRowBytes;
    float *xarr = reinterpret_cast<float *>(vtile + DP * kRowBytes), *yarr = xarr + 64;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    int id = blockIdx.x;
    const int qblk = id % p.blocks;
    id /= p.blocks;
    const int split = id % p.splits;
    const int bh = id / p.splits;
    const int b = bh / p.heads, head = bh - b * p.heads;
    const int t0 = (int)((int64_t)p.tiles * split / p.splits), t1 = (int)((int64_t)p.tiles * (split + 1) / p.splits);
    const int64_t live_q = live_queries(p, b);
    const int64_t q = ((int64_t)qblk * WQ + wave) * 32 + (lane & 31);
    const bool q_ok = q < live_q;
    const bool idle = (int64_t)qblk * WQ * 32 >= live_q;

    typename M::Owned qf, of;
    M::load_owned(qf, (const typename T::elem *)p.q + (int64_t)bh * p.D * p.nq + (q < p.nq ? q : 0), p.nq, p.D, q_ok, h);
    M::load_owned(of, (const typename T::elem *)p.d_out + (int64_t)bh * p.Dv * p.nq + (q < p.nq ? q : 0), p.nq, p.Dv, q_ok, h);
    const typename M::Addr addr = M::addr(lane);
    const Score<T> score(p, head);
    float qx = 0.f, qy = 0.f;
    if (p.falloff != nullptr && q_ok) query_place(p, b, q, qx, qy);
    float lse2 = __builtin_inff(), delta = 0.f;                // a query without cells has weights 0
    if (q_ok) {
        const float x = p.lse[(int64_t)bh * p.nq + q];
        lse2 = x == -__builtin_inff() ? __builtin_inff() : x * kLog2e;
        delta = p.delta[(int64_t)bh * p.nq + q];
    }
    f32x16 g[NC / 32];
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) g[c][i] = 0.f;

    const KeyTiles<M, T> keys(p, b, head);
    for (int t = t0; t < (idle ? t0 : t1); ++t) {
        const typename KeyTiles<M, T>::At at = keys.at(t);
        uint64_t live = __ballot(keys.live(at, lane));
        if constexpr (M::kRows == 32) live &= 0xffffffffull;
        if (live == 0) continue;                               // the same in every wave
        __syncthreads();
        Loader<M, T, DP, NT> kl, vl;
        kl.load(keys.base(p.k, at, p.D), p.cells, p.D, at.cell0, p.cells);
        kl.store(ktile, p.cells, p.D, live, 0.f);
        if (!p.shared) {
            vl.load(keys.base(p.v, at, p.Dv), p.cells, p.Dv, at.cell0, p.cells);
            vl.store(vtile, p.cells, p.Dv, live, 0.f);
        }
        if (p.falloff != nullptr && threadIdx.x < M::kRows) {
            const int c = (int)at.cell0 + threadIdx.x;
            xarr[threadIdx.x] = (float)(c % p.W);
            yarr[threadIdx.x] = (float)(c / p.W);
        }
        __syncthreads();
#pragma unroll kUnroll
        for (int k = 0; k < kBlocks; ++k) {
            const f32x16 acc = M::first(ktile, addr, k, qf);
            const f32x16 dp = M::first(vtile, addr, k, of);
            const unsigned bits = (unsigned)(live >> (32 * k));
            float w[16];
            if (p.falloff != nullptr) {
                M::per_cell(xarr, k, h, w);
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = (w[i] - qx) * (w[i] - qx);
                float cy[16];
                M::per_cell(yarr, k, h, cy);
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = fmaf(-score.fall, fmaf(cy[i] - qy, cy[i] - qy, w[i]), -lse2);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = -lse2;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float ds = dp[i] - delta;
                if (score.cap) {
                    const float th = score.bend(acc[i]);
                    w[i] = fmaf(score.top, th, w[i]);
                    ds *= fmaf(-th, th, 1.f);
                } else {
                    w[i] = fmaf(score.in, acc[i], w[i]);
                }
                ds *= exp2_(w[i]);
                w[i] = (bits >> M::cell(i, h)) & 1u ? ds : 0.f;
            }
            M::second(ktile + p.c0 * kRowBytes, addr, k, M::weights(w), g);
        }
    }
    if (q >= p.nq) return;
    if (p.parts) {
        float *dst = p.part_a + ((int64_t)split * p.B * p.heads + bh) * p.D * p.nq + q;
#pragma unroll
        for (int c = 0; c < NC / 32; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int ch = p.c0 + 32 * c + out_channel(i, h);
                if (ch < p.D) dst[ch * p.nq] = q_ok ? g[c][i] : 0.f;
            }
        return;
    }
    typename T::elem *dst = (typename T::elem *)p.dq + (int64_t)bh * p.D * p.nq + q;
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int ch = p.c0 + 32 * c + out_channel(i, h);
            if (ch < p.D) store_float(dst + ch * p.nq, q_ok ? g[c][i] * p.scale : 0.f);
        }
}

// Gradients of the reference and value maps: owned = cells, streamed = queries.  PART 0: both; 1: the value's, 2: the
// reference's alone (maps of more than 128 channels, for the registers).
template <typename T, int DP, int WQ, int PART, int NC>
__global__ __launch_bounds__(64 * WQ) void soft_dkv_kernel(const Params p) {
    typedef Math<T, DP> M;
    constexpr int NT = 64 * WQ;
    constexpr int kBlocks = M::kRows / 32;
    constexpr int kUnroll = DP == 256 ? 1 : kBlocks;           // registers
    constexpr bool kDv = PART != 2, kDk = PART != 1;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char *qtile = lds, *otile = lds + DP * kRowBytes;
    float *larr = reinterpret_cast<float *>(otile + DP * kRowBytes);
    float *darr = larr + 64, *xarr = larr + 128, *yarr = larr + 192;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    int id = blockIdx.x;
    const int blk = id % p.blocks;
    id /= p.blocks;
    const int split = id % p.splits;
    const int bh = id / p.splits;
    const int b = bh / p.heads, head = bh - b * p.heads;
    const int64_t live_q = live_queries(p, b);
    const int tiles = (int)((live_q + M::kRows - 1) / M::kRows);
    const int t0 = (int)((int64_t)tiles * split / p.splits), t1 = (int)((int64_t)tiles * (split + 1) / p.splits);
    const int64_t cell = ((int64_t)blk * WQ + wave) * 32 + (lane & 31);
    const bool c_ok = cell < p.cells && (p.mask == nullptr || p.mask[(int64_t)b * p.cells + cell] != 0);
    const float cx = (float)((int)cell % p.W), cy = (float)((int)cell / p.W);

    typename M::Owned kf, vf;
    M::load_owned(kf, (const typename T::elem *)p.k + (int64_t)bh * p.D * p.cells + (cell < p.cells ? cell : 0), p.cells, p.D,
                  c_ok, h);
    if constexpr (kDk)
        M::load_owned(vf, (const typename T::elem *)p.v + (int64_t)bh * p.Dv * p.cells + (cell < p.cells ? cell : 0), p.cells, p.Dv,
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

    const typename T::elem *qmap = (const typename T::elem *)p.q + (int64_t)bh * p.D * p.nq;
    const typename T::elem *omap = (const typename T::elem *)p.d_out + (int64_t)bh * p.Dv * p.nq;
    for (int t = t0; t < t1; ++t) {
        const int64_t q0 = (int64_t)t * M::kRows;
        __syncthreads();
        Loader<M, T, DP, NT> ql, ol;
        ql.load(qmap, p.nq, p.D, q0, live_q);
        ql.store(qtile, p.nq, p.D, ~0ull, 0.f);
        ol.load(omap, p.nq, p.Dv, q0, live_q);
        ol.store(otile, p.nq, p.Dv, ~0ull, 0.f);
        if (threadIdx.x < M::kRows) {
            const int64_t q = q0 + threadIdx.x;
            float lse2 = __builtin_inff(), delta = 0.f, x = 0.f, y = 0.f;      // no weight without cells
            if (q < live_q) {
                const float l = p.lse[(int64_t)bh * p.nq + q];
                lse2 = l == -__builtin_inff() ? __builtin_inff() : l * kLog2e;
                delta = p.delta[(int64_t)bh * p.nq + q];
                if (p.falloff != nullptr) query_place(p, b, q, x, y);
            }
            larr[threadIdx.x] = lse2;
            darr[threadIdx.x] = delta;
            xarr[threadIdx.x] = x;
            yarr[threadIdx.x] = y;
        }
        __syncthreads();
#pragma unroll kUnroll
        for (int k = 0; k < kBlocks; ++k) {
            const f32x16 acc = M::first(qtile, addr, k, kf);
            float w[16], slope[16], ls[16];
            M::per_cell(larr, k, h, ls);
            if (score.cap) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float th = score.bend(acc[i]);
                    w[i] = score.top * th;
                    slope[i] = fmaf(-th, th, 1.f);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    w[i] = score.in * acc[i];
                    slope[i] = 1.f;
                }
            }
            if (p.falloff != nullptr) {
                float qx[16], qy[16];
                M::per_cell(xarr, k, h, qx);
                M::per_cell(yarr, k, h, qy);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float dx = cx - qx[i], dy = cy - qy[i];
                    w[i] = fmaf(-score.fall, fmaf(dx, dx, dy * dy), w[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = exp2_(w[i] - ls[i]);
            if constexpr (kDv) M::second(otile + p.c0 * kRowBytes, addr, k, M::weights(w), gv);
            if constexpr (kDk) {
                const f32x16 dp = M::first(otile, addr, k, vf);
                float dl[16];
                M::per_cell(darr, k, h, dl);
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = w[i] * (dp[i] - dl[i]) * slope[i];
                M::second(qtile + p.c0 * kRowBytes, addr, k, M::weights(w), gk);
            }
        }
    }
    if (cell >= p.cells) return;
    // masked cells take no part: their columns hold zeros' products and are dropped here
    const int64_t part = ((int64_t)split * p.B * p.heads + bh);
#pragma unroll
    for (int c = 0; c < NC / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int ch = p.c0 + 32 * c + out_channel(i, h);
            float a = 0.f, v = 0.f;
            if constexpr (kDk) a = c_ok ? gk[c][i] * p.scale : 0.f;
            if constexpr (kDv) v = c_ok ? gv[c][i] : 0.f;
            if (p.parts) {
                if constexpr (kDk)
                    if (ch < p.D) p.part_a[(part * p.D + ch) * p.cells + cell] = a;
                if constexpr (kDv)
                    if (ch < p.Dv) p.part_b[(part * p.Dv + ch) * p.cells + cell] = v;
                continue;
            }
            typename T::elem *dk = (typename T::elem *)p.dk + ((int64_t)bh * p.D + ch) * p.cells + cell;
            if (p.shared) {                                    // PART 0 only: the parts of a shared map go to part_a, part_b
                if (ch < p.D) store_float(dk, a + v);
                continue;
            }
            if constexpr (kDk)
                if (ch < p.D) store_float(dk, a);
            if constexpr (kDv)
                if (ch < p.Dv) store_float((typename T::elem *)p.dv + ((int64_t)bh * p.Dv + ch) * p.cells + cell, v);
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
