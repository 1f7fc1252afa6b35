// rf_block.h -- what the residual-block kernels share: loads and stores of
// eight elements, the 8-bit checkpoint code, wave sums.
//
// Every kernel gives a lane eight consecutive columns (a chunk): 16 bytes of
// a 16-bit tensor, 8 bytes of codes, a quarter of a checkpoint block.  Rows
// start at any element: gfx950 loads and stores vectors at any address that
// is aligned to the element, so odd widths and row strides take the same path
// as round ones; only the last chunk of a row goes element by element.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>

#include "rfadam8.h"

namespace rf {
// Records the calling thread's error message (rf_host.hip); never throws.
rf_status report(rf_status code, const char* msg) noexcept;
rf_status report_hip(hipError_t e, const char* what) noexcept;
// Compute units of the current device.
rf_status device_cus(int* out) noexcept;
}  // namespace rf

namespace rfb {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_at __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_at __attribute__((aligned(2)));
typedef uint32_t u32x4_at __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));

// Allows a kernel more than 64 KB of LDS, once on each device (rf_wgrad.hip).
[[nodiscard]] rf_status allow_lds(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) noexcept;

constexpr int CHUNK = 8;   // columns of a lane
constexpr int BLOCK = 32;  // columns that share a step: a quad of lanes
constexpr int WAVE = 64;

__host__ __device__ inline int64_t pitch_of(int64_t cols) { return (cols + BLOCK - 1) / BLOCK * BLOCK; }

template <typename T> struct Raw { u32x4 a; };  // eight 16-bit elements as loaded
template <> struct Raw<float> { u32x4 a, b; };

// Loads go in two halves so that a row's loads, and the next row's, are in
// flight together.  fetch8: eight columns from c of a row of at least eight, as
// one unconditional load; a chunk that the row ends in, or before, is loaded
// from the row's last eight columns instead.  (With a condition around it the
// compiler could not count the loads in flight, and would wait for all.)
// settle8: moves such a chunk's own columns to its front and clears the others;
// only waves that hold one branch there.
template <typename T> __device__ __forceinline__ Raw<T> fetch8(const T* row, int64_t c, int64_t cols)
{
    Raw<T> r;
    const T* const p = row + min(c, cols - CHUNK);
    r.a = *(const u32x4_at*)p;
    if constexpr (sizeof(T) == 4) r.b = *(const u32x4_at*)(p + 4);
    return r;
}

// TAIL: rows may end inside a chunk (cols % 8); without, the lane masks for it
// take no registers.
template <bool TAIL = true, typename T> __device__ __forceinline__ void settle8(Raw<T>& r, int64_t c, int64_t cols)
{
    const int64_t left = cols - c;
    if (!TAIL) {
        if (left <= 0) r = Raw<T>{};
        return;
    }
    if (left >= CHUNK || cols < CHUNK) return;  // (narrow rows: load8 put them in place)
    if (left <= 0) {
        r = Raw<T>{};
        return;
    }
    const int by = CHUNK - (int)left;  // 1 .. 7
    uint32_t w[CHUNK];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        w[k] = r.a[k];
        if constexpr (sizeof(T) == 4) w[k + 4] = r.b[k];
        else w[k + 4] = 0;
    }
    // whole words, by the bits of their number
    const int words = sizeof(T) == 4 ? by : by >> 1;
#pragma unroll
    for (int bit = 1; bit < CHUNK; bit *= 2) {
#pragma unroll
        for (int k = 0; k < CHUNK; ++k) {
            const uint32_t v = k + bit < CHUNK ? w[k + bit] : 0u;
            w[k] = words & bit ? v : w[k];
        }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            r.a[k] = w[k];
            r.b[k] = w[k + 4];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) r.a[k] = by & 1 ? (w[k] >> 16) | (w[k + 1] << 16) : w[k];
    }
}

// Both at once, in rows of any width.
template <typename T> __device__ __forceinline__ Raw<T> load8(const T* row, int64_t c, int64_t cols)
{
    Raw<T> r{};
    if (cols >= CHUNK) {
        r = fetch8(row, c, cols);
        settle8(r, c, cols);
        return r;
    }
#pragma unroll
    for (int k = 0; k < CHUNK - 1; ++k) {
        if (c + k < cols) {
            if constexpr (sizeof(T) == 4) {
                const uint32_t w = ((const uint32_t*)row)[c + k];
                if (k < 4) r.a[k & 3] = w;
                else r.b[k & 3] = w;
            } else {
                r.a[k >> 1] |= (uint32_t)((const uint16_t*)row)[c + k] << (16 * (k & 1));
            }
        }
    }
    return r;
}

// As fetch8, in rows of any width.
template <typename T> __device__ __forceinline__ Raw<T> fetch8_any(const T* row, int64_t c, int64_t cols)
{
    return cols >= CHUNK ? fetch8(row, c, cols) : load8(row, c, cols);
}

template <typename T> __device__ __forceinline__ void widen8(const Raw<T>& r, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = __uint_as_float(r.a[k]);
            v[k + 4] = __uint_as_float(r.b[k]);
        }
    } else if constexpr (__is_same(T, bf16)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = __uint_as_float(r.a[k] << 16);
            v[2 * k + 1] = __uint_as_float(r.a[k] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w = r.a[k];
            f16x2 h;
            __builtin_memcpy(&h, &w, 4);
            v[2 * k] = (float)h[0];
            v[2 * k + 1] = (float)h[1];
        }
    }
}

// To T, round to nearest even (f32: as is): the one rounding of an output.
template <typename T> __device__ __forceinline__ Raw<T> narrow8(const float (&v)[8])
{
    Raw<T> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            r.a[k] = __float_as_uint(v[k]);
            r.b[k] = __float_as_uint(v[k + 4]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f32x2 p = {v[2 * k], v[2 * k + 1]};
            uint32_t w;
            if constexpr (__is_same(T, bf16)) {
                bf16x2 h = __builtin_convertvector(p, bf16x2);
                __builtin_memcpy(&w, &h, 4);
            } else {
                f16x2 h = __builtin_convertvector(p, f16x2);
                __builtin_memcpy(&w, &h, 4);
            }
            r.a[k] = w;
        }
    }
    return r;
}

// Stores the first `left` of eight elements.  STREAM: past the caches.
template <bool TAIL = true, bool STREAM = false, typename T>
__device__ __forceinline__ void put8(T* p, const Raw<T>& r, int64_t left)
{
    if (STREAM && left >= CHUNK) {
        __builtin_nontemporal_store(r.a, (u32x4_at*)p);
        if constexpr (sizeof(T) == 4) __builtin_nontemporal_store(r.b, (u32x4_at*)(p + 4));
    } else if (TAIL ? left >= CHUNK : left > 0) {
        *(u32x4_at*)p = r.a;
        if constexpr (sizeof(T) == 4) *(u32x4_at*)(p + 4) = r.b;
    } else if (TAIL && left > 0) {
        const int n = (int)left;
        if constexpr (sizeof(T) == 4) {
            u32x4 v = r.a;
            if (n & 4) {
                *(u32x4_at*)p = v;
                v = r.b;
                p += 4;
            }
            if (n & 2) {
                *(u32x2_at*)p = u32x2{v[0], v[1]};
                v[0] = v[2];
                p += 2;
            }
            if (n & 1) *(uint32_t*)p = v[0];
        } else {
            u32x4 v = r.a;
            if (n & 4) {
                *(u32x2_at*)p = u32x2{v[0], v[1]};
                v[0] = v[2];
                v[1] = v[3];
                p += 4;
            }
            if (n & 2) {
                *(u32_at*)p = v[0];
                v[0] = v[1];
                p += 2;
            }
            if (n & 1) *(uint16_t*)p = (uint16_t)v[0];
        }
    }
}

// Columns of a parameter vector whose type is known at run time (RF_F32 /
// RF_BF16 / RF_F16), or `fill` for one that is not there; zero past the end.
// Loads of several vectors are sent before the first is looked at: `elsewhere`
// is any eight 16-bit elements that may be read instead of an absent vector's.
struct Vector8 {
    u32x4 a, b;

    __device__ __forceinline__ void fetch(const void* p, int dtype, int64_t c, int64_t cols, const void* elsewhere)
    {
        const int size = p && dtype == RF_F32 ? 4 : 2;
        const char* const q = p ? (const char*)p + min(c, cols - CHUNK) * size : (const char*)elsewhere;
        a = *(const u32x4_at*)q;
        b = *(const u32x4_at*)(q + (size == 4 ? 16 : 0));
    }
    template <bool TAIL>
    __device__ __forceinline__ void get(const void* p, int dtype, int64_t c, int64_t cols, float fill, float (&v)[8])
    {
        if (!p) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = c + (TAIL ? k : 0) < cols ? fill : 0.0f;
        } else if (dtype == RF_F32) {
            Raw<float> r{a, b};
            settle8<TAIL>(r, c, cols);
            widen8(r, v);
        } else {
            Raw<bf16> r{a};
            settle8<TAIL>(r, c, cols);
            if (dtype == RF_BF16) widen8(r, v);
            else widen8(Raw<f16>{r.a}, v);
        }
    }
};

// The same at once, in rows of any width; zero past the end.
__device__ __forceinline__ void vector8(const void* p, int dtype, int64_t c, int64_t cols, float fill, float (&v)[8])
{
    if (!p) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fill;
    } else if (dtype == RF_F32) {
        widen8(load8((const float*)p, c, cols), v);
    } else if (dtype == RF_BF16) {
        widen8(load8((const bf16*)p, c, cols), v);
    } else {
        widen8(load8((const f16*)p, c, cols), v);
    }
}

__device__ __forceinline__ float scalar_at(const void* p, int dtype, int64_t at)
{
    if (dtype == RF_F32) return ((const float*)p)[at];
    if (dtype == RF_BF16) return (float)((const bf16*)p)[at];
    return (float)((const f16*)p)[at];
}

__device__ __forceinline__ void put_scalar(void* p, int dtype, int64_t at, float v)
{
    if (dtype == RF_F32) ((float*)p)[at] = v;
    else if (dtype == RF_BF16) ((bf16*)p)[at] = (bf16)v;
    else ((f16*)p)[at] = (f16)v;
}

// ------------------------------------------------------- the 8-bit code ----
// A block's step is 2^(e - 127), e = max(E - 6, 1), E the biased exponent of
// its largest magnitude; a block with an Inf or NaN has e = 255 and reads
// back as NaN.  Codes are the values over the step, rounded to nearest even,
// within +-127 (a magnitude that rounds to 128 saturates).  With a power of
// two for the step the division is exact, and code * step has at most seven
// significant bits and a sign, so it is exact in bf16 too: products over a
// checkpoint need no rounding of their own.
struct Codes {
    u32x2 c;     // eight int8 codes
    uint32_t e;  // the block's exponent byte
};

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true);
}

// Called by whole quads of lanes that hold a block's 32 values in order
// (zeros past the end of the row).
__device__ __forceinline__ Codes encode8(const float (&v)[8])
{
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
    top = max(top, dpp<0xB1>(top));  // quad_perm [1, 0, 3, 2]
    top = max(top, dpp<0x4E>(top));  // quad_perm [2, 3, 0, 1]
    const uint32_t E = top >> 23;
    Codes r;
    r.e = E == 255 ? 255u : max(E, 7u) - 6u;
    const float inverse = __uint_as_float(E == 255 ? 0u : (254u - r.e) << 23);
    uint32_t b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        // 1.5 * 2^23: the sum's low byte is the rounded value in two's complement
        const float t = __builtin_amdgcn_fmed3f(v[k] * inverse, -127.0f, 127.0f);
        b[k] = __float_as_uint(t + 12582912.0f);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0C0C0400u);
        const uint32_t hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x04000C0Cu);
        r.c[h] = E == 255 ? 0u : lo | hi;
    }
    return r;
}

__device__ __forceinline__ void decode8(const Codes& r, float (&v)[8])
{
    const float step = __uint_as_float(r.e << 23);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)(int8_t)(r.c[k >> 2] >> (8 * (k & 3))) * step;
}

// A row's codes start at row * pitch, its exponents at row * pitch / 32; c is
// the chunk.  Only chunks below pitch / 8 exist.
__device__ __forceinline__ void put_codes(int8_t* codes, uint8_t* exps, int64_t row, int64_t pitch, int64_t c,
                                          const Codes& r)
{
    *(u32x2*)(codes + row * pitch + c * CHUNK) = r.c;
    if ((c & 3) == 0) exps[row * (pitch / BLOCK) + (c >> 2)] = (uint8_t)r.e;
}

__device__ __forceinline__ Codes get_codes(const int8_t* codes, const uint8_t* exps, int64_t row, int64_t pitch,
                                           int64_t c)
{
    Codes r;
    r.c = *(const u32x2*)(codes + row * pitch + c * CHUNK);
    r.e = exps[row * (pitch / BLOCK) + (c >> 2)];
    return r;
}

// Sum over the wave's 64 lanes, in a fixed order, in every lane.
__device__ __forceinline__ float wave_sum(float x)
{
    auto add = [](float s, int moved) { return s + __int_as_float(moved); };
    x = add(x, __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x111, 0xF, 0xF, true));  // row_shr:1
    x = add(x, __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x112, 0xF, 0xF, true));  // row_shr:2
    x = add(x, __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x114, 0xF, 0xF, true));  // row_shr:4
    x = add(x, __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x118, 0xF, 0xF, true));  // row_shr:8
    x = add(x, __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x142, 0xA, 0xF, false));  // row_bcast:15
    x = add(x, __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x143, 0xC, 0xF, false));  // row_bcast:31
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

}  // namespace rfb
