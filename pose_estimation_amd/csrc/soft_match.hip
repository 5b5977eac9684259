// Soft correspondence: C entry points (argument checks, workgroup plans, workspace layout).
#include <cmath>

#include "soft_backward.h"
#include "soft_launch.h"

namespace {
using namespace ispa_soft;

bool sizes_ok(int dtype, int B, int heads, int D, int Dv, int64_t nq, int V, int64_t cells) {
    return (dtype == ISPA_F32 || dtype == ISPA_BF16) && B >= 0 && heads >= 1 && D >= 1 && D <= ISPA_SOFT_MAX_CHANNELS && Dv >= 1 &&
           Dv <= ISPA_SOFT_MAX_CHANNELS && nq >= 0 && nq < (1ll << 22) && V >= 0 && cells >= 1 && cells < (1ll << 22) &&
           (int64_t)B * heads < 65536 && V * ((cells + 31) / 32) < (1ll << 30) &&
           (int64_t)B * heads * ((nq > cells ? nq : cells) / 32 + 1) < (1ll << 24);       // threads of a launch: 2^32
}

int check_sizes(int dtype, int B, int heads, int D, int Dv, int64_t nq, int V, int64_t cells) {
    ISPA_REQUIRE(dtype == ISPA_F32 || dtype == ISPA_BF16, "dtype %d is neither float32 nor bfloat16", dtype);
    ISPA_REQUIRE(heads >= 1 && D >= 1 && Dv >= 1 && D <= ISPA_SOFT_MAX_CHANNELS && Dv <= ISPA_SOFT_MAX_CHANNELS,
                 "heads %d of %d query and %d value channels (1 to %d each)", heads, D, Dv, ISPA_SOFT_MAX_CHANNELS);
    ISPA_REQUIRE(sizes_ok(dtype, B, heads, D, Dv, nq, V, cells),
                 "sizes out of range: batch %d, heads %d, %lld queries, %d views of %lld cells", B, heads, (long long)nq, V,
                 (long long)cells);
    return ISPA_OK;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Maps (maps, d, n) to be copied into the form Direct wants: rows of `segs` 16-byte segments, d8 rows with d8 the next multiple of
// 8, zeros beside; for kSplit three planes of bfloat16 numbers, (maps, 3, d8, ld).  One launch copies all maps of a call
// that take the same arithmetic: its copies are a few us each, launches as much again (a float32 training step of 8 pairs of
// 28x28x128 makes four copies, one of ragged bfloat16 maps six).
constexpr int kMostCopies = 4;
struct CopyJob {
    const void *src;
    void *dst;
    int d, d8, n, segs;
    int64_t total;             // segments of the copy (kSplit: of one plane)
};
struct CopyJobs {
    CopyJob job[kMostCopies];
    unsigned until[kMostCopies];       // the first block behind each job
    int count;
};

// 16 bytes a thread, read as they lie.
template <Arithmetic A>
__global__ __launch_bounds__(256) void soft_copy_kernel(const CopyJobs jobs) {
    int k = 0;
    while (k + 1 < jobs.count && blockIdx.x >= jobs.until[k]) ++k;
    const CopyJob &job = jobs.job[k];
    const unsigned block = blockIdx.x - (k > 0 ? jobs.until[k - 1] : 0);
    const int64_t i = (int64_t)block * 256 + threadIdx.x;
    if (i >= job.total) return;
    typedef std::conditional_t<A == kNarrow, unsigned short, float> elem;
    constexpr int kN = A == kFloat ? 4 : 8;
    const int row = (int)(i / job.segs), seg = (int)(i - (int64_t)row * job.segs), cell = seg * kN;
    const int map = row / job.d8, c = row - map * job.d8;
    elem e[kN] = {};
    if (c < job.d) {
        const elem *at = (const elem *)job.src + ((int64_t)map * job.d + c) * job.n + cell;
        if (cell + kN <= job.n) {
            __builtin_memcpy(e, at, sizeof(e));
        } else {
#pragma unroll
            for (int j = 0; j < kN; ++j)
                if (cell + j < job.n) e[j] = at[j];
        }
    }
    u32x4 *dst = (u32x4 *)job.dst;
    if constexpr (A == kSplit) {
        u32x4 v[3];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned x[3], y[3];
            split3(e[2 * j], x[0], x[1], x[2]);
            split3(e[2 * j + 1], y[0], y[1], y[2]);
#pragma unroll
            for (int p = 0; p < 3; ++p) v[p][j] = uppers(x[p], y[p]);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) dst[(((int64_t)map * 3 + p) * job.d8 + c) * job.segs + seg] = v[p];
    } else {
        u32x4 v;
        __builtin_memcpy(&v, e, 16);
        dst[i] = v;
    }
}

// Copies of maps in the workspace: three planes for kSplit; else only maps whose rows do not start on 16-byte borders or
// whose channels are no multiple of 8.
struct Copies {
    int64_t ld;
    int d8;
    size_t bytes;              // 0: the map is streamed as it is
};

Copies copies(Arithmetic a, int64_t maps, int d, int64_t n) {
    const int64_t unit = a == kFloat ? 4 : 8;
    Copies c;
    c.ld = (n + unit - 1) / unit * unit;
    c.d8 = (d + 7) & ~7;
    const size_t numbers = (size_t)maps * c.d8 * c.ld;
    c.bytes = a == kSplit ? align256(numbers * 6) : c.ld == n && c.d8 == d ? 0 : align256(numbers * (a == kFloat ? 4 : 2));
    return c;
}

// The copies of a call: add() settles how a map is streamed, launch() makes the copies that were asked for.
class Copier {
public:
    explicit Copier(char *workspace) : at(workspace) {}
    int add(Stream *s, Arithmetic a, const void *map, int64_t maps, int d, int64_t n) {
        const Copies c = copies(a, maps, d, n);
        s->ld = c.ld;
        s->d = c.d8;
        s->map = map;
        if (c.bytes == 0) return ISPA_OK;
        const int segs = (int)(c.ld / (a == kFloat ? 4 : 8));
        const int64_t rows = maps * c.d8, total = rows * segs;
        CopyJobs &j = jobs[a];
        const int64_t before = j.count > 0 ? j.until[j.count - 1] : 0, blocks = before + (total + 255) / 256;
        ISPA_REQUIRE(rows < (1ll << 31) && blocks < (1ll << 32) / 256, "maps of %lld rows are too large for one call", (long long)rows);
        j.job[j.count] = CopyJob{map, at, d, c.d8, (int)n, segs, total};
        j.until[j.count++] = (unsigned)blocks;
        s->map = at;
        at += c.bytes;
        return ISPA_OK;
    }
    int launch(hipStream_t stream) const {
        if (int rc = one<kNarrow>(stream)) return rc;
        if (int rc = one<kSplit>(stream)) return rc;
        return one<kFloat>(stream);
    }
    char *at;                  // of the workspace, behind the copies

private:
    template <Arithmetic A>
    int one(hipStream_t stream) const {
        const CopyJobs &j = jobs[A];
        if (j.count == 0) return ISPA_OK;
        soft_copy_kernel<A><<<j.until[j.count - 1], 256, 0, stream>>>(j);
        return ispa::check_launch("soft_copy_kernel");
    }
    CopyJobs jobs[3] = {};
};

// Workgroups a compute unit holds: two waves a SIMD where a lane's registers allow it, else one.
int resident(int dtype, bool codes, bool backward, int D, int Dv, int64_t owned) {
    if (waves_for(owned) == 1)
        return codes && padded_channels(D, Dv) <= 128 && (dtype == ISPA_BF16 || few_columns(true, owned)) ? 8 : 4;
    backward |= codes;
    return padded_channels(D, Dv) <= (dtype == ISPA_BF16 ? 128 : backward ? 0 : 64) ? 2 : 1;
}

Arithmetic arithmetic_of(int dtype, bool codes, int D, int Dv, int64_t owned) {
    return arithmetic(dtype == ISPA_F32, codes, padded_channels(D, Dv), waves_for(owned));
}

Plan plan_of(int dtype, bool codes, bool backward, int64_t groups, int D, int Dv, int64_t owned, int V, int64_t streamed) {
    const int64_t r = tile_rows(arithmetic_of(dtype, codes, D, Dv, owned));
    return make_plan(owned, groups, (streamed + r - 1) / r * V, resident(dtype, codes, backward, D, Dv, owned));
}

size_t forward_bytes(const Plan &plan, int B, int heads, int Dv, int64_t nq) {
    return plan.splits == 1 ? 0 : (size_t)plan.splits * B * heads * nq * (Dv + 2) * sizeof(float);
}

void backward_plans(int dtype, int B, int heads, int D, int Dv, int64_t nq, int64_t cells, Plan *dq, Plan *dkv) {
    *dq = plan_of(dtype, false, true, (int64_t)B * heads, D, Dv, nq, 1, cells);
    *dkv = plan_of(dtype, false, true, (int64_t)B * heads, D, Dv, cells, 1, nq);
}

// Channels of float32 parts per cell: every split's, or what the first of two launches leaves for the second (a map that is
// reference and value; the size does not say which, so any map of equal channels).
size_t dkv_parts(int dtype, const Plan &dkv, int D, int Dv) {
    if (dkv.splits > 1) return (size_t)dkv.splits * (D + Dv);
    return D == Dv && dkv_two_launches(dtype == ISPA_F32, padded_channels(D, Dv), dkv.waves) ? Dv : 0;
}

size_t backward_bytes(int dtype, const Plan &dq, const Plan &dkv, int B, int heads, int D, int Dv, int64_t nq, int64_t cells) {
    const size_t bh = (size_t)B * heads;
    const Arithmetic aq = arithmetic_of(dtype, false, D, Dv, nq), akv = arithmetic_of(dtype, false, D, Dv, cells);
    const size_t copied = copies(aq, bh, D, cells).bytes + copies(aq, bh, Dv, cells).bytes + copies(akv, bh, D, nq).bytes +
                          copies(akv, bh, Dv, nq).bytes;
    const size_t a = dq.splits > 1 ? dq.splits * bh * D * nq : 0, k = dkv_parts(dtype, dkv, D, Dv) * bh * cells;
    return copied + align256(bh * nq * sizeof(float)) + (a > k ? a : k) * sizeof(float);
}

int check_score(float scale, float cap, const float *falloff, int W) {
    ISPA_REQUIRE(std::isfinite(scale) && std::isfinite(cap) && cap >= 0.f, "scale %g, cap %g: finite, cap >= 0 wanted", scale, cap);
    ISPA_REQUIRE(cap == 0.f || (cap >= 1e-30f && std::fabs(scale) <= 1e30 * cap), "cap %g is too small for scale %g", cap, scale);
    ISPA_REQUIRE(falloff == nullptr || W >= 1, "falloff needs the map's width");
    return ISPA_OK;
}

size_t forward_copies(int dtype, int B, int heads, int D, int Dv, int64_t nq, int64_t cells, bool shared) {
    const Arithmetic a = arithmetic_of(dtype, false, D, Dv, nq);
    return copies(a, (int64_t)B * heads, D, cells).bytes + (shared ? 0 : copies(a, (int64_t)B * heads, Dv, cells).bytes);
}

enum Source { kMaps, kInt8, kFp8 };

int run_forward(Params &p, int dtype, Source source, void *workspace, size_t workspace_bytes, hipStream_t stream) {
    const bool maps = source == kMaps;
    const int64_t bh = (int64_t)p.B * p.heads;
    const Plan plan = plan_of(dtype, !maps, false, bh, p.D, p.Dv, p.nq, p.V, p.cells);
    const Arithmetic a = arithmetic_of(dtype, !maps, p.D, p.Dv, p.nq);
    const size_t copied = maps ? forward_copies(dtype, p.B, p.heads, p.D, p.Dv, p.nq, p.cells, p.shared) : 0;
    const size_t need = copied + forward_bytes(plan, p.B, p.heads, p.Dv, p.nq);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return ispa::fail(ISPA_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    ISPA_REQUIRE(need == 0 || ((uintptr_t)workspace & 255) == 0, "the workspace must start on a 256-byte border");
    ISPA_REQUIRE(!maps || (((uintptr_t)p.k | (uintptr_t)p.v) & 15) == 0, "maps must start on 16-byte borders");
    p.tiles_per_view = (int)((p.cells + tile_rows(a) - 1) / tile_rows(a));
    p.tiles = p.tiles_per_view * p.V;
    p.blocks = plan.blocks;
    p.splits = plan.splits;
    Copier copier((char *)workspace);
    if (maps) {
        if (int rc = copier.add(&p.sk, a, p.k, bh, p.D, p.cells)) return rc;
        if (!p.shared)
            if (int rc = copier.add(&p.sv, a, p.v, bh, p.Dv, p.cells)) return rc;
        if (int rc = copier.launch(stream)) return rc;
    }
    p.part_ml = (float *)copier.at;
    p.part_o = p.part_ml + (size_t)plan.splits * bh * p.nq * 2;
    if (maps) return dtype == ISPA_F32 ? forward_f32(p, plan.waves, stream) : forward_bf16(p, plan.waves, stream);
    return dtype == ISPA_F32 ? forward_codes_f32(p, source == kFp8, plan.waves, stream)
                             : forward_codes_bf16(p, source == kFp8, plan.waves, stream);
}
}  // namespace

extern "C" size_t ispa_soft_match_workspace_bytes(int dtype, int B, int heads, int D, int Dv, int64_t nq, int views,
                                                  int64_t cells) {
    if (!sizes_ok(dtype, B, heads, D, Dv, nq, views, cells) || B == 0 || nq == 0) return 0;
    // codes may be cut into tiles of another size than maps: room for either
    size_t most = 0;
    for (int codes = 0; codes < 2; ++codes) {
        const size_t n = (codes ? 0 : forward_copies(dtype, B, heads, D, Dv, nq, cells, false)) +
                         forward_bytes(plan_of(dtype, codes, false, (int64_t)B * heads, D, Dv, nq, views, cells), B, heads, Dv, nq);
        most = n > most ? n : most;
    }
    return most;
}

extern "C" int ispa_soft_match(const void *q, const void *r, const void *v, int dtype, int B, int heads, int D, int Dv,
                               int64_t nq, int64_t cells, int W, float scale, float cap, const float *falloff,
                               const float *query_xy, const uint8_t *mask, const int32_t *num_query, void *out, float *out32,
                               float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_sizes(dtype, B, heads, D, Dv, nq, 1, cells)) return rc;
    if (int rc = check_score(scale, cap, falloff, W)) return rc;
    if (B == 0 || nq == 0) return ISPA_OK;
    ISPA_REQUIRE(q && r && out, "null pointer");
    ISPA_REQUIRE(v != nullptr || D == Dv, "without a value map the reference map is the value (%d != %d channels)", D, Dv);
    Params p = {};
    p.q = q;
    p.k = r;
    p.v = v ? v : r;
    p.shared = v == nullptr;
    p.mask = mask;
    p.falloff = falloff;
    p.query_xy = query_xy;
    p.count = num_query;
    p.out = out;
    p.out32 = out32;
    p.lse = lse;
    p.nq = nq;
    p.cells = cells;
    p.B = B;
    p.heads = heads;
    p.D = D;
    p.Dv = Dv;
    p.W = W < 1 ? 1 : W;
    p.V = 1;
    p.scale = scale;
    p.cap = cap;
    return run_forward(p, dtype, kMaps, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int ispa_store_match(const void *q, int dtype, const void *codes, const float *scales, const uint8_t *mask, int kind,
                                const int32_t *views, int V, int n_view, int B, int heads, int D, int64_t nq, int64_t cells,
                                int W, float scale, float cap, const float *falloff, const float *query_xy,
                                const int32_t *num_query, void *out, float *lse, void *workspace, size_t workspace_bytes,
                                void *stream) {
    if (int rc = check_sizes(dtype, B, heads, D, D, nq, V, cells)) return rc;
    if (int rc = check_score(scale, cap, falloff, W)) return rc;
    ISPA_REQUIRE(kind == ISPA_STORE_INT8 || kind == ISPA_STORE_FP8, "store kind %d is neither int8 nor e4m3", kind);
    ISPA_REQUIRE(n_view >= 1, "a store of %d views", n_view);
    if (B == 0 || nq == 0) return ISPA_OK;
    ISPA_REQUIRE(q && codes && scales && mask && out && (views || V == 0), "null pointer");
    Params p = {};
    p.q = q;
    p.k = p.v = codes;
    p.shared = 1;
    p.kscale = scales;
    p.views = views;
    p.n_view = n_view;
    p.mask = mask;
    p.falloff = falloff;
    p.query_xy = query_xy;
    p.count = num_query;
    p.out = out;
    p.lse = lse;
    p.nq = nq;
    p.cells = cells;
    p.B = B;
    p.heads = heads;
    p.D = p.Dv = D;
    p.W = W < 1 ? 1 : W;
    p.V = V;
    p.scale = scale;
    p.cap = cap;
    return run_forward(p, dtype, kind == ISPA_STORE_INT8 ? kInt8 : kFp8, workspace, workspace_bytes,
                       (hipStream_t)stream);
}

extern "C" size_t ispa_soft_match_backward_workspace_bytes(int dtype, int B, int heads, int D, int Dv, int64_t nq,
                                                           int64_t cells) {
    if (!sizes_ok(dtype, B, heads, D, Dv, nq, 1, cells) || B == 0) return 0;
    Plan dq, dkv;
    backward_plans(dtype, B, heads, D, Dv, nq, cells, &dq, &dkv);
    return backward_bytes(dtype, dq, dkv, B, heads, D, Dv, nq, cells);
}

extern "C" int ispa_soft_match_backward(const void *q, const void *r, const void *v, int dtype, int B, int heads, int D, int Dv,
                                        int64_t nq, int64_t cells, int W, float scale, float cap, const float *falloff,
                                        const float *query_xy, const uint8_t *mask, const int32_t *num_query,
                                        const float *out32, const float *lse, const void *d_out, const float *d_lse, void *dq,
                                        void *dr, void *dv, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_sizes(dtype, B, heads, D, Dv, nq, 1, cells)) return rc;
    if (int rc = check_score(scale, cap, falloff, W)) return rc;
    if (B == 0) return ISPA_OK;
    ISPA_REQUIRE(r && dr, "null pointer");
    ISPA_REQUIRE(nq == 0 || (q && out32 && lse && d_out && dq), "null pointer");
    ISPA_REQUIRE((v == nullptr) == (dv == nullptr), "a value map and its gradient come together");
    ISPA_REQUIRE(v != nullptr || D == Dv, "without a value map the reference map is the value (%d != %d channels)", D, Dv);
    Plan pq, pkv;
    backward_plans(dtype, B, heads, D, Dv, nq, cells, &pq, &pkv);
    const size_t need = backward_bytes(dtype, pq, pkv, B, heads, D, Dv, nq, cells);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr))
        return ispa::fail(ISPA_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    ISPA_REQUIRE(need == 0 || ((uintptr_t)workspace & 255) == 0, "the workspace must start on a 256-byte border");
    Params p = {};
    p.q = q;
    p.k = r;
    p.v = v ? v : r;
    p.shared = v == nullptr;
    p.mask = mask;
    p.falloff = falloff;
    p.query_xy = query_xy;
    p.count = num_query;
    p.lse = const_cast<float *>(lse);
    p.d_out = d_out;
    p.dq = dq;
    p.dk = dr;
    p.dv = dv;
    p.nq = nq;
    p.cells = cells;
    p.B = B;
    p.heads = heads;
    p.D = D;
    p.Dv = Dv;
    p.W = W < 1 ? 1 : W;
    p.V = 1;
    p.scale = scale;
    p.cap = cap;
    hipStream_t s = (hipStream_t)stream;
    const int64_t bh = (int64_t)B * heads;
    ISPA_REQUIRE((((uintptr_t)r | (uintptr_t)p.v | (uintptr_t)q | (uintptr_t)d_out) & 15) == 0, "maps must start on 16-byte borders");
    Copier copier((char *)workspace);
    const Arithmetic aq = arithmetic_of(dtype, false, D, Dv, nq), akv = arithmetic_of(dtype, false, D, Dv, cells);
    if (int rc = copier.add(&p.sk, aq, r, bh, D, cells)) return rc;
    if (!p.shared)
        if (int rc = copier.add(&p.sv, aq, v, bh, Dv, cells)) return rc;
    if (nq > 0) {
        if (int rc = copier.add(&p.sq, akv, q, bh, D, nq)) return rc;
        if (int rc = copier.add(&p.so, akv, d_out, bh, Dv, nq)) return rc;
    }
    if (int rc = copier.launch(s)) return rc;
    float *delta = (float *)copier.at;
    p.delta = delta;
    p.part_a = (float *)(copier.at + align256(bh * nq * sizeof(float)));
    p.part_b = p.part_a + (pkv.splits > 1 ? (size_t)pkv.splits * bh * D * cells : 0);
    if (nq > 0) {
        const unsigned grid = (unsigned)((nq + 31) / 32 * bh);
        if (dtype == ISPA_F32) soft_delta_kernel<F32><<<grid, 256, 0, s>>>(p, out32, d_lse, delta);
        else soft_delta_kernel<BF16><<<grid, 256, 0, s>>>(p, out32, d_lse, delta);
        if (int rc = ispa::check_launch("soft_delta_kernel")) return rc;
    }
    return dtype == ISPA_F32 ? backward_f32(p, pq, pkv, s) : backward_bf16(p, pq, pkv, s);
}
