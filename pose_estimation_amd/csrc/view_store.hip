// Template store: feature maps of rendered views held in 8 bits with one float32 scale per cell, written and read back.
#include "soft_tile.h"

namespace {
using namespace ispa_soft;

constexpr int kThreads = 256;
// e4m3 values end at 448, int8 codes at 127
template <typename S>
constexpr float kTop = std::is_same_v<S, I8> ? 127.f : 448.f;
template <typename S>
constexpr float kPerTop = 1.f / kTop<S>;                     // a scale is max * this float32 number

// x / s rounded to the nearest code value, ties to even, decided for the exact quotient.  The float32 quotient settles it
// but next to a border, where the sign of fma(-border, s, x) is exact.
template <typename S>
__device__ __forceinline__ float quantised(float x, float s, float inv) {
    float q = fminf(fmaxf(x * inv, -kTop<S>), kTop<S>);
    auto grid = [](float v, float &step, float &per_step) {
        step = per_step = 1.f;
        if constexpr (std::is_same_v<S, FP8>) {
            int e = (int)((__builtin_bit_cast(unsigned, v) >> 23) & 255u);      // floor(log2 |v|) + 127, -6 at least
            e = e < 121 ? 121 : e;
            step = __builtin_bit_cast(float, (unsigned)(e - 3) << 23);
            per_step = __builtin_bit_cast(float, (unsigned)(257 - e) << 23);
        }
    };
    float step, per_step;
    grid(q, step, per_step);
    float t = q * per_step, n = rintf(t);
    if (fabsf(fabsf(t - n) - 0.5f) < 1e-3f || inv == 0.f) {    // t is off by 2^-22 of itself, at most 3e-5
        stay_branch();
        if (inv == 0.f) {
            q = fminf(fmaxf(x / s, -kTop<S>), kTop<S>);
            grid(q, step, per_step);
            n = rintf(q * per_step);
        }
        const float above = fmaf(-(n + 0.5f) * step, s, x), below = fmaf(-(n - 0.5f) * step, s, x);
        const bool odd = ((int)n & 1) != 0;
        if (above > 0.f || (above == 0.f && odd)) n += 1.f;
        else if (below < 0.f || (below == 0.f && odd)) n -= 1.f;
        n = fminf(fmaxf(n * step, -kTop<S>), kTop<S>) * per_step;
    }
    return n * step;
}

template <typename S>
__device__ __forceinline__ unsigned char encode(float v) {
    if constexpr (std::is_same_v<S, I8>) return (unsigned char)(signed char)(int)v;
    return (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

// A block takes 64 cells of one view, a wave's lanes side by side, and its waves share the channels: 4 to read, 8 to write.
// 24 views of 56x56x128 float32, 48 MB either way, are written in 14.7 us (3.3 TB/s) and read in 9 to 11 us (4.4 to 5.3; a large copy:
// 4.8 TB/s).  Memory bounds the read.  The write has the vector ALU busy 66 % of the cycles with settling codes, and its waves
// wait half of theirs; 17 views of 31x47x200 bfloat16 into e4m3, 15 MB, take 20 us, with 42 % and two thirds: too few waves to
// hide the steps of a code behind each other.  (16 or 4 bytes a lane, four cells to a thread, took longer both ways: 13.7 us for 9.2 to
// read them, 23.6 us for 18.6 to write them: fewer lanes to a row.)
constexpr int kCellsPer = 64, kGroups = kThreads / kCellsPer, kWriters = 8;

// Features are read once: a thread holds its channels (HELD of them; maps of more channels read the rest again) in
// registers between the maximum and the codes.
template <typename T, typename S, int HELD>
__global__ __launch_bounds__(kWriters * kCellsPer) void store_write_kernel(const typename T::elem *__restrict__ features,
                                                               const uint8_t *__restrict__ take,
                                                               const int32_t *__restrict__ views, int n, int n_view, int C,
                                                               int64_t cells, unsigned char *__restrict__ codes,
                                                               float *__restrict__ scales, uint8_t *__restrict__ mask) {
    __shared__ float tops[kWriters][kCellsPer];
    const unsigned per = (unsigned)((cells + kCellsPer - 1) / kCellsPer);
    const int item = (int)(blockIdx.x / per);
    const int lane = threadIdx.x % kCellsPer, g = threadIdx.x / kCellsPer;
    const int64_t cell = (int64_t)(blockIdx.x - item * per) * kCellsPer + lane;
    const bool in = cell < cells;
    const typename T::elem *src = features + (int64_t)item * C * cells + (in ? cell : 0);
    float held[HELD], top = 0.f;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int c = g + kWriters * i;
        held[i] = c < C ? load_float(src + c * cells) : 0.f;
    }
    auto larger = [&](float x) {
        const float a = fabsf(x);
        top = a <= __builtin_inff() ? fmaxf(top, a) : __builtin_inff();        // NaN counts as infinite
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) larger(held[i]);
    for (int c = g + kWriters * HELD; c < C; c += kWriters) larger(load_float(src + c * cells));
    tops[g][lane] = top;
    const int id = views[item];
    // a view listed more than once keeps its last entry; an index outside is skipped
    int drop = id < 0 || id >= n_view;
    for (int i = item + 1 + (int)threadIdx.x; i < n; i += kWriters * kCellsPer) drop |= views[i] == id;
    if (__syncthreads_or(drop)) return;
#pragma unroll
    for (int i = 0; i < kWriters; ++i) top = fmaxf(top, tops[i][lane]);
    if (!in) return;
    const bool finite = top < __builtin_inff();
    const float s = finite ? top * kPerTop<S> : 0.f;
    const float inv = s > 1e-30f ? 1.f / s : 0.f;              // 1 / s may overflow below: divides there
    unsigned char *dst = codes + (int64_t)id * C * cells + cell;
    auto write = [&](int c, float x) { dst[c * cells] = s > 0.f ? encode<S>(quantised<S>(x, s, inv)) : (unsigned char)0; };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (g + kWriters * i < C) write(g + kWriters * i, held[i]);
    for (int c = g + kWriters * HELD; c < C; c += kWriters) write(c, load_float(src + c * cells));
    if (g == 0) {
        scales[(int64_t)id * cells + cell] = s;
        mask[(int64_t)id * cells + cell] = finite && (take == nullptr || take[(int64_t)item * cells + cell] != 0);
    }
}

template <typename T, typename S>
__global__ __launch_bounds__(kThreads) void store_read_kernel(const unsigned char *__restrict__ codes,
                                                              const float *__restrict__ scales,
                                                              const int32_t *__restrict__ views, int n_view, int C,
                                                              int64_t cells, typename T::elem *__restrict__ out) {
    const unsigned per = (unsigned)((cells + kCellsPer - 1) / kCellsPer);
    const int item = (int)(blockIdx.x / per);
    const int id = views[item];
    const bool have = id >= 0 && id < n_view;
    const int lane = threadIdx.x % kCellsPer, g = threadIdx.x / kCellsPer;
    const int64_t cell = (int64_t)(blockIdx.x - item * per) * kCellsPer + lane;
    if (cell >= cells) return;
    const float s = have ? scales[(int64_t)id * cells + cell] : 0.f;
    const unsigned char *src = codes + (have ? (int64_t)id : 0) * C * cells + cell;
    typename T::elem *dst = out + (int64_t)item * C * cells + cell;
#pragma unroll 8
    for (int c = g; c < C; c += kGroups) {
        float f[4];
        decode4<S>(src[c * cells], f);
        store_float(dst + c * cells, have ? f[0] * s : 0.f);
    }
}

__global__ __launch_bounds__(kThreads) void store_read_mask_kernel(const uint8_t *__restrict__ mask,
                                                                   const int32_t *__restrict__ views, int n_view, int64_t cells,
                                                                   uint8_t *__restrict__ out) {
    const unsigned per = (unsigned)((cells + 4 * kThreads - 1) / (4 * kThreads));
    const int item = (int)(blockIdx.x / per);
    const int id = views[item];
    const bool have = id >= 0 && id < n_view;
    const int64_t cell = ((int64_t)(blockIdx.x - item * per) * kThreads + threadIdx.x) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (cell + j < cells) out[item * cells + cell + j] = have && mask[(int64_t)id * cells + cell + j] != 0;
}

int check(int dtype, int kind, int n, int n_view, int C, int64_t cells) {
    ISPA_REQUIRE(dtype == ISPA_F32 || dtype == ISPA_BF16, "dtype %d is neither float32 nor bfloat16", dtype);
    ISPA_REQUIRE(kind == ISPA_STORE_INT8 || kind == ISPA_STORE_FP8, "store kind %d is neither int8 nor e4m3", kind);
    ISPA_REQUIRE(n >= 0 && n_view >= 1 && C >= 1 && cells >= 1, "store sizes out of range (n %d, views %d, channels %d)", n,
                 n_view, C);
    ISPA_REQUIRE((cells + kCellsPer - 1) / kCellsPer * (int64_t)(n > 1 ? n : 1) < (1ll << 32) / (kWriters * kCellsPer) &&
                     C * cells < 0x7fffffff,
                 "maps of %lld cells are too large for one call", (long long)cells);
    return ISPA_OK;
}

#define PICK(dtype, kind, call)                                                            \
    do {                                                                                   \
        if (dtype == ISPA_F32 && kind == ISPA_STORE_INT8) { typedef F32 T; typedef I8 S; call; }    \
        else if (dtype == ISPA_F32) { typedef F32 T; typedef FP8 S; call; }                \
        else if (kind == ISPA_STORE_INT8) { typedef BF16 T; typedef I8 S; call; }          \
        else { typedef BF16 T; typedef FP8 S; call; }                                      \
    } while (0)
}  // namespace

extern "C" int ispa_store_write(const void *features, int dtype, const uint8_t *take, const int32_t *views, int n, int kind,
                                int n_view, int C, int64_t cells, void *codes, float *scales, uint8_t *mask, void *stream) {
    if (int rc = check(dtype, kind, n, n_view, C, cells)) return rc;
    if (n == 0) return ISPA_OK;
    ISPA_REQUIRE(features && views && codes && scales && mask, "null pointer");
    const unsigned blocks = (unsigned)((cells + kCellsPer - 1) / kCellsPer * n);
#define ISPA_STORE_WRITE(HELD)                                                                                          \
    PICK(dtype, kind, (store_write_kernel<T, S, HELD><<<blocks, kWriters * kCellsPer, 0, (hipStream_t)stream>>>(                    \
                           (const T::elem *)features, take, views, n, n_view, C, cells, (unsigned char *)codes, scales, mask)))
    if (C <= 16 * kWriters) ISPA_STORE_WRITE(16);
    else ISPA_STORE_WRITE(32);
#undef ISPA_STORE_WRITE
    return ispa::check_launch("store_write_kernel");
}

extern "C" int ispa_store_read(const void *codes, const float *scales, const uint8_t *mask, const int32_t *views, int n,
                               int kind, int n_view, int C, int64_t cells, int dtype, void *out, uint8_t *mask_out,
                               void *stream) {
    if (int rc = check(dtype, kind, n, n_view, C, cells)) return rc;
    if (n == 0) return ISPA_OK;
    ISPA_REQUIRE(views && (out == nullptr || (codes && scales)) && (mask_out == nullptr || mask), "null pointer");
    if (mask_out != nullptr) {
        const unsigned blocks = (unsigned)((cells + 4 * kThreads - 1) / (4 * kThreads) * n);
        store_read_mask_kernel<<<blocks, kThreads, 0, (hipStream_t)stream>>>(mask, views, n_view, cells, mask_out);
        if (int rc = ispa::check_launch("store_read_mask_kernel")) return rc;
    }
    if (out == nullptr) return ISPA_OK;
    const unsigned blocks = (unsigned)((cells + kCellsPer - 1) / kCellsPer * n);
    PICK(dtype, kind, (store_read_kernel<T, S><<<blocks, kThreads, 0, (hipStream_t)stream>>>(
                           (const unsigned char *)codes, scales, views, n_view, C, cells, (T::elem *)out)));
    return ispa::check_launch("store_read_kernel");
}
