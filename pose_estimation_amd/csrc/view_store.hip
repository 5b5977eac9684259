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

// x / s rounded to the nearest code value, ties to even, decided for the exact quotient: n from the float32 quotient is
// off by at most one step, and only next to a border, where the sign of fma(-border, s, x) is exact.
template <typename S>
__device__ __forceinline__ float quantised(float x, float s, float inv) {
    const float y = inv > 0.f ? x * inv : x / s;
    const float q = fminf(fmaxf(y, -kTop<S>), kTop<S>);
    float step = 1.f;
    if constexpr (std::is_same_v<S, FP8>) {
        const int e = (int)((__builtin_bit_cast(unsigned, q) >> 23) & 255u) - 127;      // floor(log2 |q|)
        step = __builtin_bit_cast(float, (unsigned)(127 + (e < -6 ? -6 : e) - 3) << 23);
    }
    float n = rintf(q / step);
    const float above = fmaf(-(n + 0.5f) * step, s, x), below = fmaf(-(n - 0.5f) * step, s, x);
    const bool odd = ((int)n & 1) != 0;
    if (above > 0.f || (above == 0.f && odd)) n += 1.f;
    else if (below < 0.f || (below == 0.f && odd)) n -= 1.f;
    return fminf(fmaxf(n * step, -kTop<S>), kTop<S>);
}

template <typename S>
__device__ __forceinline__ unsigned char encode(float v) {
    if constexpr (std::is_same_v<S, I8>) return (unsigned char)(signed char)(int)v;
    return (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

// One block: kCellsPer cells of one written view; the other threads of a cell share its channels, at most kHeld each, and
// hold them in registers between the maximum and the codes, so that features are read once.  Maps of more channels read
// the rest again.
constexpr int kCellsPer = 32, kGroups = kThreads / kCellsPer, kHeld = 16;
template <typename T, typename S>
__global__ __launch_bounds__(kThreads) void store_write_kernel(const typename T::elem *__restrict__ features,
                                                               const uint8_t *__restrict__ take,
                                                               const int32_t *__restrict__ views, int n, int n_view, int C,
                                                               int64_t cells, unsigned char *__restrict__ codes,
                                                               float *__restrict__ scales, uint8_t *__restrict__ mask) {
    __shared__ float tops[kGroups][kCellsPer];
    const int64_t per = (cells + kCellsPer - 1) / kCellsPer;
    const int item = (int)(blockIdx.x / per);
    const int id = views[item];
    if (id < 0 || id >= n_view) return;                        // uniform
    const int lane = threadIdx.x % kCellsPer, g = threadIdx.x / kCellsPer;
    const int64_t cell = (blockIdx.x - item * per) * kCellsPer + lane;
    const bool in = cell < cells;
    const typename T::elem *src = features + (int64_t)item * C * cells + cell;
    float held[kHeld], top = 0.f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int c = g + kGroups * i;
        held[i] = in && c < C ? load_float(src + c * cells) : 0.f;
    }
    auto larger = [&](float x) {
        const float a = fabsf(x);
        top = a <= __builtin_inff() ? fmaxf(top, a) : __builtin_inff();        // NaN counts as infinite
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) larger(held[i]);
    if (in)
        for (int c = g + kGroups * kHeld; c < C; c += kGroups) larger(load_float(src + c * cells));
    tops[g][lane] = top;
    // a view listed more than once keeps its last entry
    int later = 0;
    for (int i = item + 1 + (int)threadIdx.x; i < n; i += kThreads) later |= views[i] == id;
    if (__syncthreads_or(later)) return;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) top = fmaxf(top, tops[i][lane]);
    if (!in) return;
    const bool finite = top < __builtin_inff();
    const float s = finite ? top * kPerTop<S> : 0.f;
    const float inv = s > 1e-30f ? 1.f / s : 0.f;              // 1 / s may overflow below: divides there
    unsigned char *dst = codes + (int64_t)id * C * cells + cell;
    auto write = [&](int c, float x) { dst[c * cells] = s > 0.f ? encode<S>(quantised<S>(x, s, inv)) : (unsigned char)0; };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (g + kGroups * i < C) write(g + kGroups * i, held[i]);
    for (int c = g + kGroups * kHeld; c < C; c += kGroups) write(c, load_float(src + c * cells));
    if (g == 0) {
        scales[(int64_t)id * cells + cell] = s;
        mask[(int64_t)id * cells + cell] = finite && (take == nullptr || take[(int64_t)item * cells + cell] != 0);
    }
}

template <typename T, typename S>
__global__ __launch_bounds__(kThreads) void store_read_kernel(const unsigned char *__restrict__ codes,
                                                              const float *__restrict__ scales,
                                                              const uint8_t *__restrict__ mask,
                                                              const int32_t *__restrict__ views, int n_view, int C,
                                                              int64_t cells, typename T::elem *__restrict__ out,
                                                              uint8_t *__restrict__ mask_out) {
    const int64_t per = (cells + 63) / 64;
    const int item = (int)(blockIdx.x / per);
    const int id = views[item];
    const bool have = id >= 0 && id < n_view;
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int64_t cell = (blockIdx.x - item * per) * 64 + lane;
    if (cell >= cells) return;
    if (mask_out != nullptr && g == 0) mask_out[item * cells + cell] = have && mask[(int64_t)id * cells + cell] != 0;
    if (out == nullptr) return;                                // uniform
    const float s = have ? scales[(int64_t)id * cells + cell] : 0.f;
    const unsigned char *src = codes + (have ? (int64_t)id : 0) * C * cells + cell;
    typename T::elem *dst = out + (int64_t)item * C * cells + cell;
#pragma unroll 8
    for (int c = g; c < C; c += 4) {
        float f[4];
        decode4<S>(src[c * cells], f);
        store_float(dst + c * cells, have ? f[0] * s : 0.f);
    }
}

int check(int dtype, int kind, int n, int n_view, int C, int64_t cells) {
    ISPA_REQUIRE(dtype == ISPA_F32 || dtype == ISPA_BF16, "dtype %d is neither float32 nor bfloat16", dtype);
    ISPA_REQUIRE(kind == ISPA_STORE_INT8 || kind == ISPA_STORE_FP8, "store kind %d is neither int8 nor e4m3", kind);
    ISPA_REQUIRE(n >= 0 && n_view >= 1 && C >= 1 && cells >= 1, "store sizes out of range (n %d, views %d, channels %d)", n,
                 n_view, C);
    ISPA_REQUIRE((cells + 31) / 32 * (int64_t)(n > 1 ? n : 1) < 0x7fffffff && C * cells < 0x7fffffff,
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
    PICK(dtype, kind, (store_write_kernel<T, S><<<blocks, kThreads, 0, (hipStream_t)stream>>>(
                           (const T::elem *)features, take, views, n, n_view, C, cells, (unsigned char *)codes, scales, mask)));
    return ispa::check_launch("store_write_kernel");
}

extern "C" int ispa_store_read(const void *codes, const float *scales, const uint8_t *mask, const int32_t *views, int n,
                               int kind, int n_view, int C, int64_t cells, int dtype, void *out, uint8_t *mask_out,
                               void *stream) {
    if (int rc = check(dtype, kind, n, n_view, C, cells)) return rc;
    if (n == 0) return ISPA_OK;
    ISPA_REQUIRE(views && (out == nullptr || (codes && scales)) && (mask_out == nullptr || mask), "null pointer");
    const unsigned blocks = (unsigned)((cells + 63) / 64 * n);
    PICK(dtype, kind, (store_read_kernel<T, S><<<blocks, kThreads, 0, (hipStream_t)stream>>>(
                           (const unsigned char *)codes, scales, mask, views, n_view, C, cells, (T::elem *)out, mask_out)));
    return ispa::check_launch("store_read_kernel");
}
