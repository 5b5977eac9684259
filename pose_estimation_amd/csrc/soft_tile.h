// Soft correspondence: the tile format, operand fragments and loaders that the forward and backward kernels share.
//
// All three kernels are the same two chained products.  One side's cells are OWNED: a wave keeps 32 of them as the
// columns of its MFMA tiles, channels in registers.  The other side's cells are STREAMED through LDS in tiles of
// kRows cells.  The first product contracts channels (scores: rows = streamed cells, columns = owned cells), the
// second contracts the streamed cells (rows = channels, columns = owned cells).  The 32x32 MFMA accumulator holds
// one owned column per lane and 16 streamed rows in its registers, which is already the second product's B operand, so
// probabilities never leave the registers.  Forward and the query gradient own queries, the key/value gradient owns
// keys.
//
// LDS tile: channel rows of 128 bytes (64 bfloat16 or 32 float32 cells), as the maps lie in memory.  The 16-byte
// segments of a row are permuted by swz(row), so that both readers are free of bank conflicts: the transposed read of
// the first product touches 4 rows x 64 bytes at a time (row bit 0 picks the bank half, bit 1 the segment half), the
// plain 16-byte read of the second one touches one segment of 16 or 32 successive rows (bits 1 to 3 pick 8 segments).
#pragma once
#include <type_traits>
#include <utility>

#include "common.h"

namespace ispa_soft {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kRowBytes = 128;

// f(0) .. f(N - 1) with constant arguments: loops over register arrays that the optimiser must not keep as loops.
template <typename F, int... I>
__device__ __forceinline__ void each(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F &&f) {
    each(f, std::make_integer_sequence<int, N>{});
}

__device__ __forceinline__ int swz(int row) { return ((row & 2) << 1) | ((row >> 2) & 3); }

__device__ __forceinline__ float bf16_to_float(unsigned short u) { return __builtin_bit_cast(float, (unsigned)u << 16); }

// Round to nearest, ties to even, two at a time (v_cvt_pk_bf16_f32).
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}

// An element whose row is the same for the wave and whose column is a lane's own: the row's address moves on in scalar
// registers, the column's bytes stay in one vector register, and no address is multiplied out.
template <typename E>
using Global = __attribute__((address_space(1))) E;
template <typename E>
__device__ __forceinline__ Global<E> *at_column(E *row, unsigned bytes) {
    typedef std::conditional_t<std::is_const_v<E>, const char, char> byte;
    return (Global<E> *)((Global<byte> *)row + bytes);
}

// The same pointer in every lane, in scalar registers.
template <typename E>
__device__ __forceinline__ E *scalar(E *p) {
    const uint64_t at = (uint64_t)p;
    return reinterpret_cast<E *>((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(uint32_t)at) |
                                 (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)) << 32);
}

// Rows are walked one after the other: not all their addresses at once.
template <typename E>
__device__ __forceinline__ void next_row(E *&row) {
    asm("" : "+s"(row));
}

// A lane's 8 channels of a 16-channel step, zeros past the last; `row` moves on by 16 rows.  whole: all 16 are there.
template <typename E>
__device__ __forceinline__ void eight_rows(const E *&row, unsigned lane, int64_t ld, bool whole, int channel, int d, E (&e)[8]) {
    const E *at = row;
    if (whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            e[j] = *at_column(at, lane);
            at += ld;
            next_row(at);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            e[j] = channel + j < d ? *at_column(at, lane) : (E)0;
            at += ld;
            next_row(at);
        }
    }
    row += 16 * ld;
    next_row(row);
}

// Keeps the code of a rare case behind its branch: turned into selects it would cost every tile three operations a cell.
__device__ __forceinline__ void stay_branch() { asm volatile(""); }

// ------------------------------------------------------------------------------------------------
// Element types of the maps in memory.
struct F32 {
    typedef float elem;
};
struct BF16 {
    typedef unsigned short elem;
};
// float32 maps and codes on bfloat16 MFMAs: a float32 number is the exact sum of three bfloat16 numbers (its 24 bits cut
// into three times 8), and six of the nine products of two such sums carry float32's precision.
struct F32S {               // streamed maps in three planes
    typedef float elem;
};
struct F32C {               // streamed codes, which one bfloat16 number holds exactly
    typedef float elem;
};
struct F32Q {               // streamed codes, up to 8 queries
    typedef float elem;
};
struct I8 {                 // codes of a template store; the value is code * scale[cell]
    typedef signed char elem;
};
struct FP8 {                // e4m3
    typedef unsigned char elem;
};

__device__ __forceinline__ float load_float(const float *p) { return *p; }
__device__ __forceinline__ float load_float(const unsigned short *p) { return bf16_to_float(*p); }
__device__ __forceinline__ void store_float(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_float(unsigned short *p, float v) { *p = (unsigned short)pack_bf16(v, 0.f); }
__device__ __forceinline__ void store_float(Global<float> *p, float v) { *p = v; }
__device__ __forceinline__ void store_float(Global<unsigned short> *p, float v) { *p = (unsigned short)pack_bf16(v, 0.f); }

template <typename S>
__device__ __forceinline__ void decode4(unsigned w, float (&f)[4]) {
    if constexpr (std::is_same_v<S, I8>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = (float)(int)(signed char)(w >> (8 * i));
    } else {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        f[0] = a[0];
        f[1] = a[1];
        f[2] = b[0];
        f[3] = b[1];
    }
}

// ------------------------------------------------------------------------------------------------
// Arithmetic of a kernel: float32 MFMAs for float32 maps, bfloat16 MFMAs (float32 accumulation) for bfloat16 maps.
template <typename T, int DP>
struct Math;

// A lane's 512 registers are two halves of 256, and the vector ALU reaches one of them: operands that only MFMAs read are
// put into the other where both are needed.
__device__ __forceinline__ bf16x8 accumulator_side(bf16x8 v) {
    asm("" : "+a"(v));
    return v;
}

template <int DP>
struct Math<BF16, DP> {
    static constexpr int kRows = 64;             // streamed cells per tile
    static constexpr int kCells = 8;             // cells of a 16-byte segment
    static constexpr int kBytes = 2;             // of a streamed number in LDS
    static constexpr int kPlanes = 1;            // LDS tiles that hold one tile of the map
    static constexpr bool kWide = false;         // float32 maps or queries
    static constexpr int kColumns = 32;          // owned cells of a wave
    struct Owned {                               // B operand of the first product: channels 16 s + 8 h .. + 7
        bf16x8 f[DP / 16];
    };
    // column `col` (always a real one) of `map`, rows of ld cells; !ok: zeros
    __device__ __forceinline__ static void load_owned(Owned &o, const unsigned short *map, int col, int64_t ld, int d, bool ok, int h) {
        const unsigned lane = (unsigned)(8 * h * (int)ld + col) * sizeof(*map);
        map = scalar(map);
        each<DP / 16>([&](auto step) {
            constexpr int s = decltype(step)::value;
            unsigned short e[8];
            const bool whole = 16 * s + 16 <= d;               // uniform
            // not eight_rows(), which sets the main loop of the forward kernel of 128 channels differently (64 pairs: 631 us for 595)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (whole) e[j] = *at_column(map, lane);
                else e[j] = 16 * s + 8 * h + j < d ? *at_column(map, lane) : (unsigned short)0;
                map += ld;
                next_row(map);
            }
            map += 8 * ld;
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = ok ? (unsigned)e[2 * j] | ((unsigned)e[2 * j + 1] << 16) : 0u;
            o.f[s] = __builtin_bit_cast(bf16x8, w);
            if constexpr (DP == 256) o.f[s] = accumulator_side(o.f[s]);
        });
    }
    __device__ __forceinline__ static void negate(Owned &o) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
            o.f[s] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, o.f[s]) ^ 0x80008000u);
    }
    // The transposed 8-byte read hands lane i of a 16-lane group element i of the group's four 8-byte pieces, for
    // 4 channel rows.  The pieces are addressed so that accumulator row 16 s + 8 e + 4 h + j belongs to streamed cell
    // 16 s + 8 h + 4 e + j: a lane then holds 8 successive cells per 16-cell step, what one plain 16-byte read of the
    // second product's A operand gives.
    struct Addr {
        int tr[2];           // first, second four channels of a 16-channel step (swz repeats every 16 rows)
        int nat;
    };
    __device__ __forceinline__ static Addr addr(int lane) {
        const int h = lane >> 5, g = (lane >> 4) & 1, p = lane & 3;
        const int seg = 2 * g + (p & 1), half = p >> 1;
        Addr a;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int row = 8 * h + ((lane & 15) >> 2) + 4 * x;
            a.tr[x] = row * kRowBytes + ((seg ^ swz(row)) << 4) + half * 8;
        }
        const int row = lane & 31;
        a.nat = row * kRowBytes + ((h ^ swz(row)) << 4);
        return a;
    }
    // Products of the owned cells with streamed cells 32 b .. 32 b + 31 of a tile, b = b0 .. b0 + N - 1.  The A fragments are
    // read kAhead steps before their MFMAs.  `from`: what the products are added to.
    template <int N, bool AHEAD = true>
    __device__ __forceinline__ static void first(const char *tile, const Addr &a, int b0, const Owned &o, f32x16 (&acc)[N],
                                 const f32x16 &from = f32x16{}) {
        typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
        constexpr int kSteps = DP / 16, kAhead = DP == 256 ? 0 : AHEAD ? 2 : 1;
        auto frag = [&](int n, int s) {
            union {
                s16x4 q[2];
                bf16x8 v;
            } u;
#pragma unroll
            for (int x = 0; x < 2; ++x)
                u.q[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_ptr)(tile + (a.tr[x] ^ ((b0 + n) << 6)) + s * 16 * kRowBytes));
            return u.v;
        };
        bf16x8 f[kAhead + 1][N];
#pragma unroll
        for (int s = 0; s < kAhead && s < kSteps; ++s)
#pragma unroll
            for (int n = 0; n < N; ++n) f[s][n] = frag(n, s);
        each<kSteps>([&](auto step) {
            constexpr int s = decltype(step)::value;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if constexpr (s + kAhead < kSteps) f[(s + kAhead) % (kAhead + 1)][n] = frag(n, s + kAhead);
                if constexpr (s == 0) acc[n] = from;
                acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[s % (kAhead + 1)][n], o.f[s], acc[n], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    struct Weights {
        bf16x8 f[2];
    };
    __device__ __forceinline__ static Weights weights(const float (&p)[16]) {
        Weights w;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = pack_bf16(p[8 * s + 2 * j], p[8 * s + 2 * j + 1]);
            w.f[s] = __builtin_bit_cast(bf16x8, v);
        }
        return w;
    }
    // out += (channels x cells 32 b .. 32 b + 31 of the tile) x weights, for the first 32 N channel rows from `tile` on
    template <int N>
    __device__ __forceinline__ static void second(const char *tile, const Addr &a, int b, const Weights &w, f32x16 (&out)[N]) {
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 v = *reinterpret_cast<const bf16x8 *>(tile + (a.nat ^ ((4 * b + 2 * s) << 4)) + c * 32 * kRowBytes);
                out[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, w.f[s], out[c], 0, 0, 0);
                if (DP == 256 && s == 1 && c % 2 == 1) __builtin_amdgcn_sched_barrier(0);   // bounds the reads in flight
            }
    }
    // Streamed cell (inside its 32) of accumulator register i, i = 0 .. 15.
    __device__ static constexpr int cell(int i, int h) { return 16 * (i >> 3) + 8 * h + (i & 7); }
    // Per-cell floats of a tile's LDS array, in register order.
    __device__ __forceinline__ static f32x4 four(const float *v, int b, int h, int t) {        // registers 4 t .. 4 t + 3
        return *reinterpret_cast<const f32x4 *>(v + 32 * b + 16 * (t >> 1) + 8 * h + 4 * (t & 1));
    }
    __device__ __forceinline__ static void per_cell(const float *v, int b, int h, float (&out)[16]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f32x4 x = four(v, b, h, t);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[4 * t + j] = x[j];
        }
    }
};

template <int DP>
struct Math<F32, DP> {
    static constexpr int kRows = 32;
    static constexpr int kCells = 4;
    static constexpr int kBytes = 4;
    static constexpr int kPlanes = 1;
    static constexpr bool kWide = true;
    static constexpr int kColumns = 32;
    struct Owned {                               // channel 2 s + h
        float f[DP / 2];
    };
    __device__ __forceinline__ static void load_owned(Owned &o, const float *map, int col, int64_t ld, int d, bool ok, int h) {
        const unsigned first = (unsigned)col * sizeof(*map), lane = first + (unsigned)(h * (int)ld) * sizeof(*map);
        map = scalar(map);
        each<DP / 2>([&](auto step) {
            constexpr int s = decltype(step)::value;
            // past the last channel the last row again: it meets zeros in LDS
            const float x = *at_column(map, 2 * s + h < d ? lane : first);
            if (2 * s + 2 < d) map += 2 * ld;
            next_row(map);
            o.f[s] = ok ? x : 0.f;
            if constexpr (DP == 256 && s % 2 == 0) asm("" : "+a"(o.f[s]));      // see accumulator_side
            if (DP == 256 && s % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        });
    }
    __device__ __forceinline__ static void negate(Owned &o) {
#pragma unroll
        for (int s = 0; s < DP / 2; ++s) o.f[s] = -o.f[s];
    }
    struct Addr {
        int one[8];          // row 2 s + h for s = 0 .. 7 (swz repeats every 16 rows)
        int nat;
    };
    __device__ __forceinline__ static Addr addr(int lane) {
        const int h = lane >> 5, cell = lane & 31;
        Addr a;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const int row = 2 * s + h;
            a.one[s] = row * kRowBytes + (((cell >> 2) ^ swz(row)) << 4) + (cell & 3) * 4;
        }
        a.nat = cell * kRowBytes + ((h ^ swz(cell)) << 4);
        return a;
    }
    template <int N, bool AHEAD = true>
    __device__ __forceinline__ static void first(const char *tile, const Addr &a, int, const Owned &o, f32x16 (&acc)[N],
                                 const f32x16 &from = f32x16{}) {
        acc[0] = from;
        each<DP / 2>([&](auto step) {
            constexpr int s = decltype(step)::value;
            const float x = *reinterpret_cast<const float *>(tile + a.one[s & 7] + (s >> 3) * 16 * kRowBytes);
            acc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, o.f[s], acc[0], 0, 0, 0);
            if (DP == 256 && s % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        });
    }
    struct Weights {
        float f[16];
    };
    __device__ __forceinline__ static Weights weights(const float (&p)[16]) {
        Weights w;
#pragma unroll
        for (int i = 0; i < 16; ++i) w.f[i] = p[i];
        return w;
    }
    template <int N>
    __device__ __forceinline__ static void second(const char *tile, const Addr &a, int, const Weights &w, f32x16 (&out)[N]) {
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {        // cells 8 i + 4 h + 0 .. 3
                const f32x4 v = *reinterpret_cast<const f32x4 *>(tile + (a.nat ^ (i << 5)) + c * 32 * kRowBytes);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    out[c] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[j], w.f[4 * i + j], out[c], 0, 0, 0);
                if (DP == 256) __builtin_amdgcn_sched_barrier(0);
            }
    }
    __device__ static constexpr int cell(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }
    __device__ __forceinline__ static f32x4 four(const float *v, int, int h, int t) {
        return *reinterpret_cast<const f32x4 *>(v + 8 * t + 4 * h);
    }
    __device__ __forceinline__ static void per_cell(const float *v, int b, int h, float (&out)[16]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f32x4 x = four(v, b, h, t);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[4 * t + j] = x[j];
        }
    }
};

// x = hi + mid + lo exactly (up to bits below 2^-133), each a bfloat16 number in the upper half of the word.
__device__ __forceinline__ void split3(float x, unsigned &hi, unsigned &mid, unsigned &lo) {
    hi = __builtin_bit_cast(unsigned, x);
    const float r = x - __builtin_bit_cast(float, hi & 0xffff0000u);
    mid = __builtin_bit_cast(unsigned, r);
    lo = __builtin_bit_cast(unsigned, r - __builtin_bit_cast(float, mid & 0xffff0000u));
}
// Upper halves of two words.
__device__ __forceinline__ unsigned uppers(unsigned first, unsigned second) { return __builtin_amdgcn_perm(second, first, 0x07060302u); }

// PLANES: of the streamed side, 3 (maps) or 1 (codes).
template <int DP, int PLANES>
struct SplitMath {
    typedef Math<BF16, DP> Narrow;
    static constexpr int kRows = 64;
    static constexpr int kCells = 8;
    static constexpr int kBytes = 2;
    static constexpr int kPlanes = PLANES;
    static constexpr bool kWide = true;
    static constexpr int kColumns = 32;
    static constexpr int kTile = DP * kRowBytes;
    struct Owned {
        bf16x8 f[3][DP / 16];
    };
    typedef typename Narrow::Addr Addr;
    __device__ __forceinline__ static Addr addr(int lane) { return Narrow::addr(lane); }
    __device__ __forceinline__ static void load_owned(Owned &o, const float *map, int col, int64_t ld, int d, bool ok, int h) {
        const unsigned lane = (unsigned)(8 * h * (int)ld + col) * sizeof(*map);
        map = scalar(map);
        each<DP / 16>([&](auto step) {
            constexpr int s = decltype(step)::value;
            float e[8];
            const bool whole = 16 * s + 16 <= d;
            eight_rows(map, lane, ld, whole, 16 * s + 8 * h, d, e);
            u32x4 w[3];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned a[3], b[3];
                split3(ok ? e[2 * j] : 0.f, a[0], a[1], a[2]);
                split3(ok ? e[2 * j + 1] : 0.f, b[0], b[1], b[2]);
#pragma unroll
                for (int x = 0; x < 3; ++x) w[x][j] = uppers(a[x], b[x]);
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                o.f[x][s] = __builtin_bit_cast(bf16x8, w[x]);
                if constexpr (DP >= 128) o.f[x][s] = accumulator_side(o.f[x][s]);
            }
            if (DP == 256 && s % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        });
    }
    __device__ __forceinline__ static void negate(Owned &o) {
        each<DP / 16>([&](auto step) {
            constexpr int s = decltype(step)::value;
#pragma unroll
            for (int x = 0; x < 3; ++x)
                o.f[x][s] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, o.f[x][s]) ^ 0x80008000u);
        });
    }
    // Planes x of one side and y of the other are multiplied where x + y < 3.  Planes are cut, not rounded: what is left out, mid lo
    // and lo mid in the main, has the product's sign and is 2^-21 of it at worst (7.8 half steps of float32), 2^-24.5 on
    // average.  Sums come out as near to 64 bits as those of float32 MFMAs (64x64x128: 2.8e-7, a float32 matrix product 1.3e-6).
    template <int N, bool AHEAD = true>
    __device__ __forceinline__ static void first(const char *tile, const Addr &a, int b0, const Owned &o, f32x16 (&acc)[N],
                                                 const f32x16 &from = f32x16{}) {
        typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
        constexpr int kSteps = DP / 16;
        auto frag = [&](int x, int n, int s) {
            union {
                s16x4 q[2];
                bf16x8 v;
            } u;
#pragma unroll
            for (int y = 0; y < 2; ++y)
                u.q[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_ptr)(tile + x * kTile + (a.tr[y] ^ ((b0 + n) << 6)) + s * 16 * kRowBytes));
            return u.v;
        };
        constexpr int kBuf = AHEAD && DP <= 128 ? 2 : 1;       // fragments read a step ahead, where registers are left
        bf16x8 f[kBuf][PLANES][N];
        auto read = [&](int s) {
#pragma unroll
            for (int x = 0; x < PLANES; ++x)
#pragma unroll
                for (int n = 0; n < N; ++n) f[s % kBuf][x][n] = frag(x, n, s);
        };
        read(0);
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] = from;
        each<kSteps>([&](auto step) {
            constexpr int s = decltype(step)::value;
            if constexpr (kBuf == 1 && s > 0) read(s);
            if constexpr (kBuf == 2 && s + 1 < kSteps) read(s + 1);
#pragma unroll
            for (int x = PLANES - 1; x >= 0; --x)
#pragma unroll
                for (int y = 2 - x; y >= 0; --y)
#pragma unroll
                    for (int n = 0; n < N; ++n)
                        acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[s % kBuf][x][n], o.f[y][s], acc[n], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    struct Weights {
        bf16x8 f[3][2];
    };
    __device__ __forceinline__ static Weights weights(const float (&p)[16]) {
        Weights w;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 v[3];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned a[3], b[3];
                split3(p[8 * s + 2 * j], a[0], a[1], a[2]);
                split3(p[8 * s + 2 * j + 1], b[0], b[1], b[2]);
#pragma unroll
                for (int x = 0; x < 3; ++x) v[x][j] = uppers(a[x], b[x]);
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) w.f[x][s] = __builtin_bit_cast(bf16x8, v[x]);
        }
        return w;
    }
    template <int N>
    __device__ __forceinline__ static void second(const char *tile, const Addr &a, int b, const Weights &w, f32x16 (&out)[N]) {
        each<2 * N>([&](auto step) {
            constexpr int s = decltype(step)::value & 1, c = decltype(step)::value >> 1;
            const char *at = tile + (a.nat ^ ((4 * b + 2 * s) << 4)) + c * 32 * kRowBytes;
#pragma unroll
            for (int x = PLANES - 1; x >= 0; --x) {
                const bf16x8 v = *reinterpret_cast<const bf16x8 *>(at + x * kTile);
#pragma unroll
                for (int y = 2 - x; y >= 0; --y)
                    out[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, w.f[y][s], out[c], 0, 0, 0);
            }
            if (s == 1 && c % 2 == 1) __builtin_amdgcn_sched_barrier(0);       // bounds the reads in flight
        });
    }
    __device__ static constexpr int cell(int i, int h) { return Narrow::cell(i, h); }
    __device__ __forceinline__ static f32x4 four(const float *v, int b, int h, int t) { return Narrow::four(v, b, h, t); }
    __device__ __forceinline__ static void per_cell(const float *v, int b, int h, float (&out)[16]) { Narrow::per_cell(v, b, h, out); }
};
template <int DP>
struct Math<F32S, DP> : SplitMath<DP, 3> {};
template <int DP>
struct Math<F32C, DP> : SplitMath<DP, 1> {};

// Up to 8 float32 queries against codes: the three planes of a query are three of a wave's columns, 8 apart, instead of
// three products (a third of the MFMAs and of the registers).  Sums over planes are sums over columns (fold).
template <int DP>
struct Math<F32Q, DP> : Math<BF16, DP> {
    typedef Math<BF16, DP> Narrow;
    typedef typename Narrow::Owned Owned;
    typedef typename Narrow::Weights Weights;
    static constexpr bool kWide = true;
    static constexpr int kColumns = 8;
    // The plane that this lane's column stands for; the fourth 8 columns hold zeros.
    struct Plane {
        unsigned m1, m2, keep;
        __device__ __forceinline__ Plane() {
            unsigned k = threadIdx.x;
            asm volatile("" : "+v"(k));                        // formed where it is used: registers
            k = (k >> 3) & 3;
            m1 = k >= 1 ? 0xffff0000u : 0u;
            m2 = k >= 2 ? 0xffff0000u : 0u;
            keep = k == 3 ? 0u : ~0u;
        }
        __device__ __forceinline__ unsigned operator()(float x) const {          // in the upper half of the word
            x -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & m1);
            x -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & m2);
            return __builtin_bit_cast(unsigned, x);
        }
        __device__ __forceinline__ unsigned operator()(float x, float y) const { return uppers((*this)(x), (*this)(y)) & keep; }
    };
    __device__ __forceinline__ static void load_owned(Owned &o, const float *map, int col, int64_t ld, int d, bool ok, int h) {
        const unsigned lane = (unsigned)(8 * h * (int)ld + col) * sizeof(*map);
        const Plane plane;
        map = scalar(map);
        each<DP / 16>([&](auto step) {
            constexpr int s = decltype(step)::value;
            float e[8];
            const bool whole = 16 * s + 16 <= d;
            eight_rows(map, lane, ld, whole, 16 * s + 8 * h, d, e);
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = ok ? plane(e[2 * j], e[2 * j + 1]) : 0u;
            o.f[s] = __builtin_bit_cast(bf16x8, w);
            if constexpr (DP == 256) o.f[s] = accumulator_side(o.f[s]);
            if (s % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        });
    }
    __device__ __forceinline__ static Weights weights(const float (&p)[16]) {
        const Plane plane;
        Weights w;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = plane(p[8 * s + 2 * j], p[8 * s + 2 * j + 1]);
            w.f[s] = __builtin_bit_cast(bf16x8, v);
        }
        return w;
    }
    // every column of a query gets the sum of all three: its row of 16 lanes turned by 8, then the other row's
    __device__ __forceinline__ static void fold(f32x16 &v) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = v[i];
            const float a = x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false));
            const auto b = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, a), false, false);
            const unsigned even = b[0], odd = b[1];
            v[i] = __builtin_bit_cast(float, even) + __builtin_bit_cast(float, odd);
        }
    }
};

// Channel of output accumulator register i of a 32-channel block.
__device__ __forceinline__ int out_channel(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// Stores 32-channel blocks of accumulators: channels c0 .. c0 + NC - 1 of column q of a map (d, n).
template <int NC, typename E>
__device__ __forceinline__ void store_columns(E *map, int64_t n, int q, int h, int c0, int d, const f32x16 (&o)[NC / 32]) {
    const unsigned lane = (unsigned)(4 * h * (int)n + q) * sizeof(E);
    E *row = scalar(map + c0 * n);
    each<NC / 32>([&](auto block) {
        constexpr int c = decltype(block)::value;
        if (c0 + 32 * c + 32 <= d) {                           // uniform
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                store_float(at_column(row, lane), o[c][i]);
                row += i % 4 < 3 ? n : 5 * n;
                next_row(row);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (c0 + 32 * c + out_channel(i, h) < d) store_float(at_column(row, lane), o[c][i]);
                row += i % 4 < 3 ? n : 5 * n;
                next_row(row);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    });
}

// Loader of one tile of codes: NT threads, thread t takes segment t & 7 of channel rows t / 8, t / 8 + NT / 8, ... and
// turns them into bfloat16, which holds an 8-bit code exactly; scales are applied to scores and weights.
// kAhead: the whole share of a thread fits a few registers, so that the loads of the next tile are issued (load) before
// the products of the present one and written to LDS (store) after them; else store does both, a few rows at a time.
// live: bit j = cell j of the tile takes part.  Cells past the map's end, masked cells and channels past d are staged as
// zeros: whatever a masked cell holds (a NaN code) meets a weight of zero in the second product and must not turn it
// into NaN.
template <typename M, typename SRC, int DP, int NT>
struct Loader {
    static constexpr int kN = M::kCells;
    static constexpr int kPer = DP * 8 / NT;
    typedef typename SRC::elem elem;
    typedef u32x2 raw;
    typedef u32x2 Unaligned __attribute__((aligned(1)));
    static constexpr bool kAhead = kPer * (int)sizeof(raw) <= (DP == 256 ? 32 : 128);
    static constexpr int kBatch = kAhead ? kPer : DP == 256 ? 1 : kPer < 8 ? kPer : 8;
    static constexpr int kLoop = kAhead ? kPer / kBatch : 1;
    static_assert(NT == 64 || NT % 128 == 0, "");
    raw r[kBatch];
    const elem *map;           // of the wave
    unsigned from;             // this thread's first segment in it
    int ok;                    // cells of the segment that the map has
    int back;                  // a segment that the row's end cuts is read this many cells before its place, up to that end

    __device__ __forceinline__ void rows(int i0, int64_t ld, int d) {
        const int row0 = threadIdx.x >> 3;
        const elem *row = map + (int64_t)i0 * (NT / 8) * ld;
        if (ld >= kN && (i0 + kBatch) * (NT / 8) <= d && __all(ok > 0)) {      // every lane loads: no branch between
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                r[i] = *(Global<const Unaligned> *)at_column(row, from);
                row += (int64_t)(NT / 8) * ld;
                next_row(row);
            }
            return;
        }
        stay_branch();
        asm volatile("" : "+s"(d));                            // the rows' masks anew for each tile: kept, they fill the registers
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            raw v = {};
            if (ok > 0 && row0 + (i0 + i) * (NT / 8) < d) {
                if (ld >= kN) {
                    v = *(Global<const Unaligned> *)at_column(row, from);
                } else {                                       // rows of fewer cells: byte by byte
                    stay_branch();
#pragma unroll 1
                    for (int j = 0; j < (int)ld; ++j) {
                        const uint64_t x = (uint64_t)(unsigned char)at_column(row, from)[j] << (8 * j);
                        v |= __builtin_bit_cast(raw, x);
                    }
                }
            }
            r[i] = v;
            row += (int64_t)(NT / 8) * ld;
            next_row(row);
        }
    }
    __device__ __forceinline__ void load(const elem *base, int64_t ld, int d, int64_t cell0, int64_t n) {
        const int64_t at = cell0 + (threadIdx.x & 7) * kN;
        const int64_t left = n - at;
        ok = left >= kN ? kN : left > 0 ? (int)left : 0;
        back = ok > 0 && ld >= kN ? kN - ok : 0;
        map = scalar(base);
        from = (unsigned)((int)(threadIdx.x >> 3) * (int)ld + (int)at - back);
        if constexpr (kAhead) rows(0, ld, d);
    }
    __device__ __forceinline__ void store(char *tile, int64_t ld, int d, uint64_t live) {
        const int seg = threadIdx.x & 7, row0 = threadIdx.x >> 3;
        const unsigned bits = (unsigned)(live >> (seg * kN)) & ((1u << kN) - 1u);
        u32x4 keep;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            keep[j] = ((bits >> (2 * j)) & 1u ? 0xffffu : 0u) | ((bits >> (2 * j + 1)) & 1u ? 0xffff0000u : 0u);
        const int at0 = row0 * kRowBytes + ((seg ^ swz(row0)) << 4);
#pragma unroll kLoop
        for (int i0 = 0; i0 < kPer; i0 += kBatch) {
            if constexpr (!kAhead) rows(i0, ld, d);
            if (__any(back > 0)) {
                stay_branch();
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    r[i] = __builtin_bit_cast(raw, __builtin_bit_cast(uint64_t, r[i]) >> (8 * back));
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                float x[4], y[4];
                decode4<SRC>(r[i][0], x);
                decode4<SRC>(r[i][1], y);
                u32x4 v;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    v[j] = uppers(__builtin_bit_cast(unsigned, x[2 * j]), __builtin_bit_cast(unsigned, x[2 * j + 1]));
                    v[2 + j] = uppers(__builtin_bit_cast(unsigned, y[2 * j]), __builtin_bit_cast(unsigned, y[2 * j + 1]));
                }
                if (live != ~0ull) v &= keep;
                // swz repeats every 16 rows; 8 rows further (one wave) it differs by 2
                const int at = at0 ^ (NT == 64 ? ((i0 + i) & 1) << 5 : 0);
                *reinterpret_cast<u32x4 *>(tile + at + (i0 + i) * (NT / 8) * kRowBytes) = v;
            }
        }
    }
};

// A map as Direct streams it: `d` rows (a multiple of 8) of `ld` cells per item, head and plane.
struct Stream {
    const void *map;
    int64_t ld;
    int d;
};

// Copies tiles of a map from memory into LDS without a register in between (global_load_lds, 16 bytes a lane), so that the
// next tile is under way during the products of the present one.  Wave w of WQ moves channel rows 8 (w kShare + e) .. + 7
// with instruction e; lane l lands on row l / 8, segment l % 8, and fetches the segment that swz keeps there.
// The map: rows of `ld` cells that start on 16-byte borders (ld a multiple of kCells), `d` rows, a multiple of 8; what
// does not come like that is copied into such a form first.
template <typename M, int DP, int WQ>
struct Direct {
    static constexpr int kSize = M::kBytes;
    static constexpr int kTile = DP * kRowBytes;
    static constexpr int kShare = DP / 8 / WQ;
    static constexpr int kUnroll = kShare > 4 ? 4 : kShare;    // scalar registers
    static_assert(kShare == 1 || kShare % 2 == 0, "a wave moves 8 rows or pairs of 8");
    unsigned off[2];           // byte offset of this lane's segment in rows 8 e .. 8 e + 7 for even, odd 8-row groups
    unsigned row;              // byte offset of its row
    unsigned ld8;              // bytes of 8 rows
    uint64_t from;             // first row this wave moves
    int first, groups;         // its 8-row group; the groups that the map has from there on
    // item: which of the maps (batch item and head)
    __device__ __forceinline__ void init(const Stream &s, int64_t item) {
        const int lane = threadIdx.x & 63;
        row = (unsigned)((lane >> 3) * s.ld * kSize);
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) off[odd] = row + (((lane & 7) ^ swz((lane >> 3) + 8 * odd)) << 4);
        ld8 = (unsigned)(8 * s.ld * kSize);
        first = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * kShare;
        groups = (s.d >> 3) - first;
        const uint64_t at = (uint64_t)s.map + (uint64_t)item * M::kPlanes * (uint64_t)(s.d >> 3) * ld8 + (uint64_t)first * ld8;
        from = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(uint32_t)at) |
               (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)) << 32;
    }
    // Rows past the map's are zero in LDS throughout.
    __device__ __forceinline__ void clear_rest(char *tile) const {
        for (int x = 0; x < M::kPlanes; ++x)
            for (int i = (first + groups) * 8 * kRowBytes + (int)threadIdx.x * 16; i < kTile; i += 64 * WQ * 16)
                *reinterpret_cast<u32x4 *>(tile + x * kTile + i) = u32x4{};
    }
    // Tile from `cell0` on, of a map with `cells` cells (a multiple of kCells) a row; asynchronous, wait() ends it.
    __device__ __forceinline__ void issue(int cell0, int cells, const char *tile) const {
        unsigned at[2] = {off[0], off[1]};
        if (cells - cell0 < M::kRows) {                        // segments past the end: the row's first of this tile instead
            stay_branch();
#pragma unroll
            for (int odd = 0; odd < 2; ++odd)
                if ((int)((at[odd] - row) / kSize) >= cells - cell0) at[odd] = row;
        }
        uint64_t base = from + (uint64_t)(unsigned)(cell0 * kSize);
        unsigned to = (unsigned)__builtin_amdgcn_readfirstlane(
            (int)((unsigned)(uintptr_t)(__attribute__((address_space(3))) const char *)tile + first * 1024));
#pragma unroll 1
        for (int x = 0; x < M::kPlanes; ++x) {
            uint64_t src = base;
            unsigned dst = to;
            if constexpr (kShare == 1) {
                if (groups > 0) copy(first & 1 ? at[1] : at[0], src, dst);
            } else if (groups >= kShare) {
#pragma unroll kUnroll
                for (int e = 0; e < kShare; ++e) {
                    copy(at[e & 1], src, dst);
                    src += ld8;
                    dst += 1024;
                }
            } else {
#pragma unroll 1
                for (int e = 0; e < groups; ++e) {
                    copy(e & 1 ? at[1] : at[0], src, dst);
                    src += ld8;
                    dst += 1024;
                }
            }
            base += (uint64_t)(first + groups) * ld8;
            to += kTile;
        }
    }
    __device__ __forceinline__ static void copy(unsigned voff, uint64_t sbase, unsigned dst) {
        // uniform by construction; said so, whatever the optimiser concludes about the control flow around
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(sbase >> 32));
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)sbase);
        const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)dst);
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2"
                     :
                     : "v"(voff), "s"(m0), "s"((uint64_t)hi << 32 | lo)
                     : "memory", "m0");
    }
    __device__ __forceinline__ static void wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
    // After wait(): zeros for the cells that take no part (see Loader), in the segments this lane itself has copied.
    __device__ __forceinline__ void mask(char *tile, uint64_t live) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const int seg = (lane & 7) ^ swz((lane >> 3) + 8 * odd);
            const unsigned bits = (unsigned)(live >> (seg * M::kCells)) & ((1u << M::kCells) - 1u);
            if (bits == (1u << M::kCells) - 1u) continue;
            u32x4 keep;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (kSize == 2)
                    keep[j] = ((bits >> (2 * j)) & 1u ? 0xffffu : 0u) | ((bits >> (2 * j + 1)) & 1u ? 0xffff0000u : 0u);
                else
                    keep[j] = (bits >> j) & 1u ? 0xffffffffu : 0u;
            }
            if (kShare == 1 && (first & 1) != odd) continue;
#pragma unroll
            for (int x = 0; x < M::kPlanes; ++x)
#pragma unroll kUnroll
                for (int e = kShare == 1 ? 0 : odd; e < kShare; e += 2) {
                    if (e < groups) {
                        u32x4 *p = reinterpret_cast<u32x4 *>(tile + x * kTile + (first + e) * 1024 + lane * 16);
                        *p = *p & keep;
                    }
                }
        }
    }
};

// Workgroups are dealt to the 8 dies in turn; this numbering gives each die a run of successive workgroups, so that those
// that stream the same maps share one L2.
__device__ __forceinline__ int die_major(int id, int n) {
    const int die = id & 7, per = n >> 3, more = n & 7;
    return die * per + (die < more ? die : more) + (id >> 3);
}

// ------------------------------------------------------------------------------------------------
// What a call computes; device pointers as the C ABI hands them over.
struct Params {
    const void *q, *k, *v;                 // (B,heads D,nq), (B,heads D,cells), (B,heads Dv,cells); codes for a store
    const float *kscale;                   // store: (n_view,cells)
    const int32_t *views;                  // store: (B,V)
    const uint8_t *mask;                   // (B,cells), store: (n_view,cells); NULL = all cells
    const float *falloff;                  // (heads) or NULL
    const float *query_xy;                 // (B,nq,2) or NULL: query i is cell (i % W, i / W)
    const int32_t *count;                  // (B) live queries or NULL
    void *out;
    float *out32, *lse;
    float *part_o, *part_ml;               // workspace of split calls
    // backward
    const void *d_out;
    const float *delta;                    // (B,heads,nq)
    void *dq, *dk, *dv;
    float *part_a, *part_b;
    int64_t nq, cells;
    int B, heads, D, Dv, W, V, n_view;
    int tiles_per_view, tiles, splits, blocks;       // streamed tiles of one item, split over `splits` workgroups
    Stream sk, sv, sq, so;                 // r, v, q, d_out for streaming: the maps themselves or their copies
    int shared;                            // the value map is the reference map
    int parts;                             // gradients go to part_a (and part_b), to be summed by soft_sum_kernel
    int c0;                                // first channel of the gradients this launch forms
    float scale, cap;
};

// The kernel's arguments read again: what only the end of a kernel wants need not wait in scalar registers through its loop
// (the asm keeps the loads from being moved up).
typedef const __attribute__((address_space(4))) Params LateParams;
__device__ __forceinline__ LateParams &late_params() {
    LateParams *p = (LateParams *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}

// What a kernel is built for: each sort of score has its own straight code, general ones branch at run time.
enum Mode {
    kPlain = 0,       // no cap, no falloff
    kCapped = 1,      // bfloat16, a cap of at most kFixedCap, no falloff
    kRows = 2,        // no cap, falloff on a grid whose rows the streamed groups of cells do not leave
    kGeneral = 3
};
constexpr float kFixedCap = 32.f;     // the cap stands for the maximum: weights are 2^(-2 cap log2 e) > 2^-93 at least
constexpr float kPlainCap = 64.f;     // see Score

// The scores of one item and head, in units of log2: z = bent - falloff d^2 with bent = in acc, or top tanh(in acc).
template <typename T>
struct Score {
    // tanh(y) = 1 - 2 r, r = 1 / (exp(2 y) + 1), has an absolute error of 2e-7, the cap's share of which is far below what the inputs of
    // the bfloat16 kernels leave in a score as long as the cap is small: 1.3e-5 for kPlainCap.  float32, and bfloat16 above that
    // (`exact`: 8 pairs of 64x64x128 forward 140 us for 109, with gradients 622 for 484), keep the relative error near
    // 1e-7 too: below 0.6 the odd polynomial y + y^3 c(y^2), c fitted to (tanh(y) / y - 1) / y^2 on [0, 0.36] by weighted least
    // squares.
    static constexpr bool kExact = !std::is_same_v<T, BF16>;
    float in, top, fall, in2, per;
    bool cap, exact;
    __device__ __forceinline__ Score(const Params &p, int head) {
        cap = p.cap > 0.f;
        exact = kExact || p.cap > kPlainCap;
        in = cap ? p.scale / p.cap : p.scale * kLog2e;
        in2 = in * (2.f * kLog2e);
        top = p.cap * kLog2e;
        per = -0.5f / top;
        fall = p.falloff ? p.falloff[head] * kLog2e : 0.f;
    }
    __device__ __forceinline__ float r(float acc) const { return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(acc * in2) + 1.f); }
    // -2 top r: what tanh leaves of the cap.  The factor rides in the sum under the reciprocal.
    __device__ __forceinline__ float below_cap(float acc) const {
        return __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(acc * in2), per, per));
    }
    // 2 r and the slope 1 - tanh^2 = e (2 r)^2 with e = exp(2 y): of factors, so that nothing cancels far in the cap, where
    // 1 - tanh^2 from a rounded tanh, and r - r^2 from an r near 1, lose all their bits.  e is kept finite (beside 2^126 the slope
    // is below 2^-124).
    __device__ __forceinline__ float two_r(float acc, float &slope) const {
        const float e = __builtin_amdgcn_exp2f(fminf(acc * in2, 126.f)), x = __builtin_amdgcn_rcpf(fmaf(e, 0.5f, 0.5f));
        slope = x * (e * x);
        return x;
    }
    __device__ __forceinline__ float bend(float acc) const {
        if constexpr (kExact) return bend_exact(acc);
        return fmaf(-2.f, r(acc), 1.f);
    }
    __device__ __forceinline__ float bend_exact(float acc) const { return near_zero(in * acc, fmaf(-2.f, r(acc), 1.f)); }
    // 16 products to tanh, by what the cap asks for.  TIGHT: a few at a time, where registers are short
    template <bool TIGHT>
    __device__ __forceinline__ void bend(f32x16 &acc) const {
        if (!kExact && exact) {                                // uniform
            stay_branch();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                acc[i] = bend_exact(acc[i]);
                if (TIGHT && i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                acc[i] = bend(acc[i]);
                if (TIGHT && i % 8 == 7) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    // tanh(y), and its slope
    __device__ __forceinline__ float bend(float acc, float &slope) const {
        const float y = in * acc, th = near_zero(y, 1.f - two_r(acc, slope));
        slope = fabsf(y) < 0.6f ? fmaf(-th, th, 1.f) : slope;
        return th;
    }
    // tanh(y) where |y| < 0.6, else `far`
    __device__ __forceinline__ static float near_zero(float y, float far) {
        const float u = y * y;
        float c = fmaf(u, -0.00589394523f, 0.020794617f);
        c = fmaf(u, c, -0.0537832938f);
        c = fmaf(u, c, 0.133319154f);
        c = fmaf(u, c, -0.333332986f);
        return fabsf(y) < 0.6f ? fmaf(y * u, c, y) : far;
    }
};

// offset - falloff d^2 of one owned cell at (x, y) to the 16 streamed cells of a lane.
// kRows: streamed cells lie on the grid in groups of kCells successive ones, whose rows' width is a multiple of that: a
// group stays in one row.  bfloat16: d^2 grows along it by a quadratic, whose own part, -falloff j^2, is the same in every
// group and lies in the accumulators' start (`from`), so that one operation a cell is left (FROM: where 16 registers are
// left for it).  Its parts cancel near the query, which leaves falloff 64 2^-23 of error in a score: 8e-6 for kGentle.  float32,
// and bfloat16 above that (`steep`), take the distances as they are.
// kGeneral: places read from LDS (`cell`: 64 x, 64 y).
template <typename M, int MODE, bool FROM = true>
struct Penalty {
    static constexpr bool kQuadratic = !M::kWide;
    static constexpr float kGentle = 1.f;
    bool on, steep;
    float fall, x, y, width, per_width;
    __device__ __forceinline__ Penalty(const Params &p, float fall_, float x_, float y_) {
        on = MODE == kRows || (MODE == kGeneral && p.falloff != nullptr);
        fall = fall_;
        steep = !kQuadratic || fabsf(fall) > kGentle * kLog2e;
        x = x_;
        y = y_;
        width = (float)p.W;
        per_width = 1.f / width;
    }
    __device__ __forceinline__ bool wants_places() const { return MODE == kGeneral && on; }
    __device__ __forceinline__ f32x16 from(float in) const {
        f32x16 v = {};
        if constexpr (MODE == kRows && FROM && kQuadratic) {
            const float f = steep ? 0.f : -fall / in;
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = f * (float)((i % M::kCells) * (i % M::kCells));
        }
        return v;
    }
    __device__ __forceinline__ void operator()(const float *cell, int cell0, int k, int h, float offset, float (&z)[16]) const {
        if constexpr (MODE == kRows) {
#pragma unroll
            for (int g = 0; g < 16; g += M::kCells) {
                // cells are fewer than 2^22: c + 0.5 is exact and the quotient's error cannot reach the next integer
                const float c = (float)(cell0 + 32 * k + M::cell(g, h));
                const float cy = floorf((c + 0.5f) * per_width);
                const float cx = fmaf(-width, cy, c), dx = cx - x, dy = cy - y;
                if (steep) {                                   // uniform
                    const float yy = dy * dy;
#pragma unroll
                    for (int j = 0; j < M::kCells; ++j) {
                        const float d = (cx + (float)j) - x;
                        z[g + j] = fmaf(-fall, fmaf(d, d, yy), offset);
                    }
                    continue;
                }
                const float base = fmaf(-fall, fmaf(dx, dx, dy * dy), offset), step = -2.f * fall * dx;
#pragma unroll
                for (int j = 0; j < M::kCells; ++j)
                    z[g + j] = fmaf((float)j, step, FROM ? base : fmaf((float)(-j * j), fall, base));
            }
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f32x4 cx = M::four(cell, k, h, t), cy = M::four(cell + 64, k, h, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float dx = cx[j] - x, dy = cy[j] - y;
                    z[4 * t + j] = fmaf(-fall, fmaf(dx, dx, dy * dy), offset);
                }
            }
        }
    }
};

// Two waves that share a SIMD and run the same loop tend to fall into step: both want the matrix pipe, then both the vector
// ALU, and neither hides the other.  Unequal priorities, by the parity of the hardware's wave slot, let one run ahead.
__device__ __forceinline__ void out_of_step() {
    constexpr int kHwId = 4, kWaveBits = 4;
    if (__builtin_amdgcn_s_getreg(kHwId | ((kWaveBits - 1) << 11)) & 1) __builtin_amdgcn_s_setprio(1);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int64_t live_queries(const Params &p, int b) {
    if (p.count == nullptr) return p.nq;
    const int64_t c = p.count[b];
    return c < 0 ? 0 : c < p.nq ? c : p.nq;
}

}  // namespace ispa_soft
