// rf_wgrad.hip -- a linear layer's weight gradient from its input's 8-bit
// checkpoint: out[n, k] = sum_t dy[t, n] code[t, k] 2^(e[t, k / 32] - 127).
//
// A code times its power-of-two step is exact in bf16, and dy is the sum of
// bf16 pieces (bf16: itself; f16, 11 bits: two; f32, 24 bits: three of 8 bits
// each, cut off, not rounded), so every product that the matrix cores form is
// exact and only the f32 sums round.  (Bits of an f32 gradient below 2^-133, bf16's
// least, are dropped: gradients under 2^-109, about 1.5e-33, lose their last ones.)
//
// Both operands have the summed index t along the rows, while the matrix
// instructions want each lane to hold eight t of one column.  The transpose is
// done on the way into LDS: a lane loads eight rows of four neighbouring
// columns and writes four 16-byte vectors, each the eight t of a column.  The
// codes pass through registers for their conversion anyway, so it costs them
// nothing, and dy half an instruction per element.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "rf_block.h"

using namespace rfb;
using rf::report;

namespace {

constexpr int STEP = 32;             // rows t of a step: four octets
constexpr int COL_BYTES = STEP * 2;  // LDS bytes of a column's step

typedef __attribute__((ext_vector_type(8))) bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

// LDS place of octet o of column c: four columns share 256 bytes, sixteen slots
// of 16 bytes, all banks once.  With ci, oi the bits of c and o the slot is the
// xor of the numbers
//   o0 1, o1 2, c0 4, c1 8, c2 3, c3 2, c4 4, c5 8.
// Lanes write columns 4 l + i and read columns 16 j + l % 16 of octet l / 16.
// 16-byte writes go by eight neighbouring lanes, 16-byte reads by the lanes 0-3,
// 12-15, 20-23, 24-27 (4-11, 16-19, 28-31; the same from 32 on), as counted
// conflicts of pairs of lanes show; either set touches different slots.  What a
// lane's own bits give is computed once, and four addresses with immediate
// offsets reach everything.
struct Places {
    int at[4];
};

__device__ __forceinline__ Places places(int base, int slot)
{
    Places p;
#pragma unroll
    for (int k = 0; k < 4; ++k) p.at[k] = base + ((slot ^ (k * 4)) * 16);
    return p;
}

template <typename T> struct Pieces { static constexpr int n = 1; };
template <> struct Pieces<f16> { static constexpr int n = 2; };
template <> struct Pieces<float> { static constexpr int n = 3; };

// Four neighbouring elements of a row.
template <typename T> struct Quad { u32x2 w; };
template <> struct Quad<float> { u32x4 w; };

typedef uint32_t u32x2_h __attribute__((ext_vector_type(2), aligned(2)));

template <typename T> __device__ __forceinline__ Quad<T> load_quad(const T* p)
{
    Quad<T> q;
    if constexpr (sizeof(T) == 4) q.w = *(const u32x4_at*)p;
    else q.w = *(const u32x2_h*)p;
    return q;
}

// The first `n` (0 .. 4) of four elements; the others are zero.
template <typename T> __device__ __forceinline__ Quad<T> load_some(const T* p, int n)
{
    Quad<T> q{};
    if constexpr (sizeof(T) == 4) {
        const uint32_t* s = (const uint32_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) q.w[i] = s[i];
    } else {
        const uint16_t* s = (const uint16_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) q.w[i >> 1] |= (uint32_t)s[i] << (16 * (i & 1));
    }
    return q;
}

// Drops the first `by` (0 .. 3) of four elements.
template <typename T> __device__ __forceinline__ Quad<T> drop(Quad<T> q, int by)
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v = q.w[i];
#pragma unroll
            for (int j = 1; j < 4; ++j)
                if (i + j < 4) v = by == j ? q.w[i + j] : v;
            q.w[i] = v;
        }
    } else {
        const uint64_t v = (((uint64_t)q.w[1] << 32) | q.w[0]) >> (16 * by);
        q.w[0] = (uint32_t)v;
        q.w[1] = (uint32_t)(v >> 32);
    }
    return q;
}

// High halves of two f32 bit patterns: a pair of bf16.
__device__ __forceinline__ uint32_t high_halves(uint32_t first, uint32_t second)
{
    return __builtin_amdgcn_perm(second, first, 0x07060302u);
}

// What is left of x (f32 bits) behind its high half, its leading eight
// significant bits: exact; zero behind an infinity (behind a NaN, a NaN).
__device__ __forceinline__ uint32_t rest(uint32_t x)
{
    const float r = __uint_as_float(x) - __uint_as_float(x & 0xFFFF0000u);
    return __builtin_isinf(__uint_as_float(x)) ? 0u : __float_as_uint(r);
}

// Steps 0 .. n - 1 in turn.  LAST: the steps that have no two behind them are
// told so (copies of the loop's body, which f32's kernel has registers for).
template <bool LAST, typename Even, typename Odd> __device__ __forceinline__ void in_pairs(int64_t n, Even even, Odd odd)
{
    int64_t q = 0;
    if constexpr (!LAST) {
        for (; q < n; q += 2) {
            even(q, std::true_type{});
            if (q + 1 < n) odd(q + 1, std::true_type{});
        }
    } else {
        for (; q + 3 < n; q += 2) {
            even(q, std::true_type{});
            odd(q + 1, std::true_type{});
        }
        if (q + 2 < n) {
            even(q, std::true_type{});
            odd(q + 1, std::false_type{});
            even(q + 2, std::false_type{});
        } else {
            even(q, std::false_type{});
            if (q + 1 < n) odd(q + 1, std::false_type{});
        }
    }
}

// Writes a wave's accumulators, columns from k and outputs from n on: a lane
// holds four neighbouring columns of an output's row.  `partial`: this split's
// sums, or null for the result.  f32 sums and plain bf16 results go as one vector;
// accumulation into 16 bits and f16 results element by element, which costs short
// sums: 512 x 11008 x 4096 into bf16 213 us, into f32 105.
template <int FK, int FN>
__device__ __forceinline__ void store_tile(const rf_weight_grad& a, float* __restrict__ partial, const f32x4 (&acc)[FK][FN],
                                           int64_t k_from, int64_t n_from)
{
    const int lane = threadIdx.x % WAVE;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int64_t n = n_from + 16 * j + lane % 16;
        if (n >= a.outs) continue;
#pragma unroll
        for (int i = 0; i < FK; ++i) {
            const int64_t k = k_from + 16 * i + lane / 16 * 4, left = a.cols - k, at = n * a.cols + k;
            if (partial) {
                float* const o = partial + at;
                if (left >= 4) {
                    *(u32x4_at*)o = __builtin_bit_cast(u32x4, acc[i][j]);
                } else {
                    for (int r = 0; r < 4; ++r)
                        if (r < left) o[r] = acc[i][j][r];
                }
                continue;
            }
            if (a.out_dtype == RF_F32 && left >= 4) {
                float* const o = (float*)a.out + at;
                f32x4 v = acc[i][j];
                if (a.accumulate) v += __builtin_bit_cast(f32x4, (u32x4) * (const u32x4_at*)o);
                *(u32x4_at*)o = __builtin_bit_cast(u32x4, v);
            } else if (a.out_dtype == RF_BF16 && left >= 4 && !a.accumulate) {
                const f32x4 v = acc[i][j];
                const bf16x2 lo = __builtin_convertvector((f32x2{v[0], v[1]}), bf16x2);
                const bf16x2 hi = __builtin_convertvector((f32x2{v[2], v[3]}), bf16x2);
                *(u32x2_h*)((bf16*)a.out + at) = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
            } else {
                for (int r = 0; r < 4; ++r)
                    if (r < left)
                        put_scalar(a.out, a.out_dtype, at + r,
                                   a.accumulate ? scalar_at(a.out, a.out_dtype, at + r) + acc[i][j][r] : acc[i][j][r]);
            }
        }
    }
}

// A side's data of one step: eight rows of this lane's four columns.
template <typename T> struct StagedD { Quad<T> q[8]; };
struct StagedX { uint32_t c[8], e[2]; };  // codes of the rows, exponents of rows lane % 4 and 4 + lane % 4

// A tile of TILE columns x TILE outputs per workgroup, WAVES_K x WAVES_N waves;
// the first half of the waves stages the codes, the second half dy.  A wave of
// each half runs on every SIMD.
//
// Step q multiplies LDS buffer q % 3.  In the same step the registers loaded for
// step q + 2 go into buffer (q + 2) % 3, the loads of step q + 4 are sent, and
// the first fragments of step q + 1 are read, whose buffer the barrier at the
// end of step q - 1 completed: nothing in a step waits for what was begun in it.
// The rows past the last whole step are step 0 of the last split, so that the
// loop's loads need no guard.
// EDGE: dy's rows are no multiple of four elements.
//
// Bound by the matrix cores' instruction slots, which the staging shares: f16 (two
// pieces) 8192 x 4096 x 4096 657 us (419 TFLOP/s, 837 of products), f32 1231 us (223,
// 670); short sums by the way through one step: 1001 x 517 x 301 f32 13.9 us.
template <typename T, int TILE, int WAVES_K, int WAVES_N, bool EDGE>
__global__ __launch_bounds__(WAVES_K* WAVES_N* WAVE, Pieces<T>::n < 3 ? 2 : 1) void k_wgrad(const rf_weight_grad a,
                                                                                           float* __restrict__ partial,
                                                                                           uint32_t tiles_k, uint32_t tiles,
                                                                                           uint32_t splits)
{
    constexpr int NP = Pieces<T>::n, HALF = WAVES_K * WAVES_N * WAVE / 2;
    constexpr int WK = TILE / WAVES_K, WN = TILE / WAVES_N, FK = WK / 16, FN = WN / 16;
    constexpr int PLANE = TILE * COL_BYTES, BUFFER = (1 + NP) * PLANE;
    static_assert(TILE == HALF, "a lane stages one octet of four columns of its side");
    static_assert(WK % 64 == 0 && WN % 64 == 0, "bits c4 and c5 are the fragment's number");
    extern __shared__ char lds[];
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    // Workgroups go to the eight XCDs in turn: an XCD takes neighbouring tiles,
    // which share rows of dy in its L2.
    const uint32_t all = tiles * splits, xcd = blockIdx.x % 8, each = all / 8;
    const uint32_t id = blockIdx.x < each * 8 ? xcd * each + blockIdx.x / 8 : blockIdx.x;
    const uint32_t tile = id % tiles, split = id / tiles;
    const int64_t k0 = (int64_t)(tile % tiles_k) * TILE, n0 = (int64_t)(tile / tiles_k) * TILE;
    const int64_t pitch = pitch_of(a.cols), blocks = pitch / BLOCK;
    const int64_t whole_steps = a.rows / STEP;
    const int64_t f0 = whole_steps * split / splits, f1 = whole_steps * (split + 1) / splits;
    const int tail = split + 1 == splits && a.rows % STEP ? 1 : 0;
    const int64_t steps = f1 - f0 + tail;

    // ---- staging: this lane's octet and its four columns.  Columns past the
    // end are loaded from valid places and never stored; the last four of dy's
    // row stand in for a group of columns that the row ends in, moved into place.
    const int oct = tid % HALF / (TILE / 4), col = tid % (TILE / 4) * 4;
    const int64_t xc = min(k0 + col, pitch - 4), dc = max(min(n0 + col, a.outs - 4), (int64_t)0);
    const bool narrow = EDGE && a.outs < 4;
    const int by = (int)min(n0 + col - dc, (int64_t)3);
    const int64_t d_pitch = a.dy_stride * (int64_t)sizeof(T);
    // bytes of this lane's first row from the step's first row (32 bits: see check())
    uint32_t x_off = (uint32_t)(oct * 8 * pitch + xc);
    uint32_t e_off = (uint32_t)((oct * 8 + lane % 4) * blocks + xc / BLOCK);  // (one block for the four lanes)
    uint32_t d_off = (uint32_t)(oct * 8 * d_pitch + dc * (int64_t)sizeof(T));
    // row i of a step: a scalar base and a 32-bit lane offset (hide() keeps the
    // compiler from extending it outside the loop and adding in 64 bits)
    auto hide = [&] { asm volatile("" : "+v"(x_off), "+v"(e_off), "+v"(d_off)); };
    auto load_x = [&](int64_t step, StagedX& r, int i) {
        const char* const x = (const char*)a.codes + step * STEP * pitch;
        const char* const e = (const char*)a.exponents + step * STEP * blocks;
        r.c[i] = *(const uint32_t*)(x + i * pitch + x_off);
        if (i % 4 == 0) r.e[i / 4] = *(const uint8_t*)(e + i * blocks + e_off);
    };
    auto load_d = [&](int64_t step, StagedD<T>& r, int i) {
        const char* const d = (const char*)a.dy + step * STEP * d_pitch;
        if (EDGE && narrow) r.q[i] = load_some((const T*)(d + i * d_pitch + d_off), (int)a.outs);
        else r.q[i] = load_quad((const T*)(d + i * d_pitch + d_off));
    };
    // the rows behind the last whole step; zeros behind them
    auto load_tail_x = [&](StagedX& r) {
        const int64_t t = whole_steps * STEP + oct * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            r.c[i] = 0;
            if (t + i < a.rows) r.c[i] = *(const uint32_t*)(a.codes + (t + i) * pitch + xc);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            r.e[i] = 0;
            if (t + 4 * i + lane % 4 < a.rows) r.e[i] = a.exponents[(t + 4 * i + lane % 4) * blocks + xc / BLOCK];
        }
    };
    auto load_tail_d = [&](StagedD<T>& r) {
        const int64_t t = whole_steps * STEP + oct * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            r.q[i] = Quad<T>{};
            if (t + i < a.rows) {
                const T* const p = (const T*)a.dy + (t + i) * a.dy_stride + dc;
                r.q[i] = a.outs < 4 ? load_some(p, (int)a.outs) : load_quad(p);
            }
        }
    };
    // col is a multiple of four: bits c2 .. c5 are the lane's
    const Places put = places(col / 4 * 256, oct ^ ((col >> 2) & 1) * 3 ^ ((col >> 3) & 1) * 2 ^ ((col >> 4) & 3) * 4);
    // column c of the four
    auto stage_x = [&](char* buf, const StagedX& r, int c) {
        const uint32_t e[8] = {dpp<0x00>(r.e[0]), dpp<0x55>(r.e[0]), dpp<0xAA>(r.e[0]), dpp<0xFF>(r.e[0]),
                               dpp<0x00>(r.e[1]), dpp<0x55>(r.e[1]), dpp<0xAA>(r.e[1]), dpp<0xFF>(r.e[1])};
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = (float)(int8_t)(r.c[2 * i] >> (8 * c)) * __uint_as_float(e[2 * i] << 23);
            const float hi = (float)(int8_t)(r.c[2 * i + 1] >> (8 * c)) * __uint_as_float(e[2 * i + 1] << 23);
            v[i] = high_halves(__float_as_uint(lo), __float_as_uint(hi));
        }
        *(u32x4*)(buf + put.at[c]) = v;
    };
    auto stage_d = [&](char* buf, StagedD<T>& r, int c) {
        if (EDGE && c == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) r.q[i] = drop(r.q[i], by);
        }
        u32x4 v[NP];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (NP == 1) {
                v[0][i] = __builtin_amdgcn_perm(r.q[2 * i + 1].w[c / 2], r.q[2 * i].w[c / 2],
                                                c & 1 ? 0x07060302u : 0x05040100u);
            } else {
                uint32_t x[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (NP == 3) {
                        x[j] = r.q[2 * i + j].w[c];
                    } else {
                        const uint16_t h = (uint16_t)(r.q[2 * i + j].w[c / 2] >> (16 * (c & 1)));
                        f16 f;
                        __builtin_memcpy(&f, &h, 2);
                        x[j] = __float_as_uint((float)f);
                    }
                }
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    v[p][i] = high_halves(x[0], x[1]);
                    if (p + 1 < NP) {
                        x[0] = rest(x[0]);
                        x[1] = rest(x[1]);
                    }
                }
            }
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) *(u32x4*)(buf + (1 + p) * PLANE + put.at[c]) = v[p];
    };

    // ---- the product: lane l holds column l % 16 of a fragment, octet l / 16
    const int wk = wave / WAVES_N * WK, wn = wave % WAVES_N * WN;
    const int slot = (lane >> 4) ^ (lane & 3) * 4 ^ ((lane >> 2) & 1) * 3 ^ ((lane >> 3) & 1) * 2;
    const Places get_x = places(wk / 4 * 256 + (lane & 15) / 4 * 256, slot);
    const Places get_d = places(PLANE + wn / 4 * 256 + (lane & 15) / 4 * 256, slot);
    auto read_x = [&](const char* buf, int i) { return *(const bf16x8*)(buf + get_x.at[i & 3] + i * 1024); };
    auto read_d = [&](const char* buf, int p, int j) { return *(const bf16x8*)(buf + get_d.at[j & 3] + p * PLANE + j * 1024); };
    f32x4 acc[FK][FN];
#pragma unroll
    for (int i = 0; i < FK; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // One side's run through the steps.
    struct Fragments {
        bf16x8 y[NP][FN], x[2];  // all of a step's on dy's side, the first two on the codes'
    };
    auto run = [&](auto load, auto load_tail, auto stage, auto& even, auto& odd) {
        // step p of this split, clamped: what lies past its end is staged and never read
        auto clamped = [&](int64_t p) { return max(min(f0 + p - tail, f1 - 1), (int64_t)0); };
        auto fetch = [&](int64_t p, auto& r) {
#pragma unroll
            for (int i = 0; i < 8; ++i) load(clamped(p), r, i);
        };
        auto stage_all = [&](char* buf, auto& r) {
#pragma unroll
            for (int c = 0; c < 4; ++c) stage(buf, r, c);
        };
        char *now = lds, *next = lds + BUFFER, *after = lds + 2 * BUFFER;
        if (tail) load_tail(even);
        else fetch(0, even);
        if (whole_steps) fetch(1, odd);
        stage_all(now, even);
        if (whole_steps) {
            fetch(2, even);
            stage_all(next, odd);
            fetch(3, odd);
        }
        __syncthreads();
        Fragments f, g;
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int j = 0; j < FN; ++j) f.y[p][j] = read_d(now, p, j);
        f.x[0] = read_x(now, 0);
        f.x[1] = read_x(now, 1);
        // The matrix instructions of fragment row i, then a piece of the other
        // work of the step that the matrix cores run beside.
        // Without MORE there is no step q + 2 to stage.
        auto step = [&](int64_t q, auto& regs, Fragments& f, Fragments& g, auto more) {
            constexpr bool MORE = decltype(more)::value;
            const int64_t ahead = clamped(q + 4);
            hide();
#pragma unroll
            for (int i = 0; i < FK; ++i) {
                const bf16x8 xi = f.x[i & 1];
                if (i + 2 < FK) f.x[i & 1] = read_x(now, i + 2);
                else g.x[i & 1] = read_x(next, i + 2 - FK);
                if (i + 2 >= FK) {
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int j = (i + 2 - FK) * FN / 2; j < (i + 3 - FK) * FN / 2; ++j) g.y[p][j] = read_d(next, p, j);
                }
#pragma unroll
                for (int p = 0; p < NP; ++p)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xi, f.y[p][j], acc[i][j], 0, 0, 0);
                // FK is 8 or 4: four columns in the first half, or a quarter each; then the loads
                if (MORE && i < 4) stage(after, regs, i);
                if (MORE && FK == 8 && i >= 4) {
                    load(ahead, regs, 2 * (i - 4));
                    load(ahead, regs, 2 * (i - 4) + 1);
                }
                if (MORE && FK == 4 && i == 3) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) load(ahead, regs, k);
                }
#pragma unroll
                for (int k = 0; k < NP * FN; ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction,
                    __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // up to six vector ones beside it
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            char* const t = now;
            now = next;
            next = after;
            after = t;
            __syncthreads();
        };
        if (whole_steps) {
            in_pairs<NP == 3>(steps, [&](int64_t q, auto more) { step(q, even, f, g, more); },
                     [&](int64_t q, auto more) { step(q, odd, g, f, more); });
        } else {  // fewer rows than a step
#pragma unroll
            for (int i = 0; i < FK; ++i)
#pragma unroll
                for (int p = 0; p < NP; ++p)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(i < 2 ? f.x[i & 1] : read_x(now, i), f.y[p][j],
                                                                           acc[i][j], 0, 0, 0);
        }
    };
    if (steps > 0) {
        if (wave < WAVES_K * WAVES_N / 2) {
            StagedX even, odd;
            run(load_x, load_tail_x, stage_x, even, odd);
        } else {
            StagedD<T> even, odd;
            run(load_d, load_tail_d, stage_d, even, odd);
        }
    }

    store_tile(a, splits == 1 ? nullptr : partial + (int64_t)split * a.outs * a.cols, acc, k0 + wk, n0 + wn);
}

// The same for bf16 gradients whose rows are whole 16-byte units, tiles of
// 256 x 256: every load goes straight to LDS (1 KB a wave instruction, no
// registers), several steps ahead.
//
// dy's rows stay as they are, [32 t][256 n], and are transposed as they are
// read: ds_read_b64_tr_b16 gives a lane four t of one column.  The codes and
// exponents land in rings of their own and go from there through registers to
// the same layout as above: a lane converts four rows of four columns.
//   step q:  loads of dy of step q + 3 and of the codes of step q + 5 sent;
//            codes of step q + 2 converted; products of step q; first fragments
//            of step q + 1 read; at its end the wave waits for its loads of dy
//            of step q + 2 and of the codes of step q + 3 (all but its last six),
//            and the barrier makes them everybody's.
// 32-byte units of dy's rows are xored by (t0, t1, t3) so that the sixteen rows
// of a transposed read lie in different banks.
//
// Measured beside k_wgrad (us): 16384 x 11008 x 4096 1389 / 1495, 8192 x 2304 x 768
// (eight splits) 41 / 42.  At 1379 us, 1.07 PFLOP/s, the matrix cores are busy 45 %
// of the cycles; 688 tiles on 256 CUs leave the last of three rounds two thirds full.
//
// The compiler must not count or order these loads (it would wait for all of
// them before each LDS read): they are written in assembly, have no results,
// and the waits for them are explicit.  (m0, which they set, is otherwise unused
// here.)
constexpr int DIRECT = 256, DIRECT_WAVES = 8;
constexpr int D_SLOT = STEP * DIRECT * 2, X_SLOT = STEP * DIRECT, E_SLOT = DIRECT_WAVES * WAVE * 4;
constexpr int D_RING = 4, X_RING = 4;
constexpr int AT_D = 0, AT_X = AT_D + D_RING * D_SLOT, AT_E = AT_X + X_RING * X_SLOT, AT_B = AT_E + X_RING * E_SLOT;
constexpr int DIRECT_LDS = AT_B + 3 * DIRECT * COL_BYTES;
static_assert(DIRECT_LDS <= 160 * 1024, "one workgroup a CU");

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((ext_vector_type(4))) short s16x4;

__device__ __forceinline__ void load_16_to_lds(uint32_t to, uint32_t off, const char* base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
}

__device__ __forceinline__ void load_byte_to_lds(uint32_t to, uint32_t off, const char* base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
}

__global__ __launch_bounds__(DIRECT_WAVES* WAVE) void k_wgrad_direct(const rf_weight_grad a, float* __restrict__ partial,
                                                                    uint32_t tiles_k, uint32_t tiles, uint32_t splits)
{
    constexpr int WK = 128, WN = 64, FK = WK / 16, FN = WN / 16;
    extern __shared__ char lds[];
    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const uint32_t all = tiles * splits, xcd = blockIdx.x % 8, each = all / 8;  // as in k_wgrad
    const uint32_t id = blockIdx.x < each * 8 ? xcd * each + blockIdx.x / 8 : blockIdx.x;
    const uint32_t tile = id % tiles, split = id / tiles;
    const int64_t k0 = (int64_t)(tile % tiles_k) * DIRECT, n0 = (int64_t)(tile / tiles_k) * DIRECT;
    const int64_t pitch = pitch_of(a.cols), blocks = pitch / BLOCK, d_pitch = a.dy_stride * 2;
    const int64_t whole_steps = a.rows / STEP;
    const int64_t f0 = whole_steps * split / splits, f1 = whole_steps * (split + 1) / splits;
    const int tail = split + 1 == splits && a.rows % STEP ? 1 : 0;
    const int64_t steps = f1 - f0 + tail;

    // ---- loads: this wave's rows 4 w .. 4 w + 3 of a step.  Columns past the
    // end come from valid places and are never stored.
    const int row0 = 4 * wave;
    auto unit = [](int t) { return (t & 3) | ((t >> 3) & 1) << 2; };  // xored onto a row's 32-byte units
    auto d_from = [&](int t) {  // byte of dy's row that this lane's 16 bytes of row t come from
        return min((int64_t)n0 * 2 + ((lane % 32) ^ (2 * unit(t))) * 16, a.outs * 2 - 16);
    };
    const uint32_t d_off0 = (uint32_t)((row0 + lane / 32) * d_pitch + d_from(row0 + lane / 32));
    const uint32_t d_off1 = (uint32_t)((row0 + 2 + lane / 32) * d_pitch + d_from(row0 + 2 + lane / 32));
    const int64_t x_from = min(k0 + lane % 16 * 16, pitch - 16), e_from = min(k0 + 4 * lane, pitch - 4) / BLOCK;
    const uint32_t x_off = (uint32_t)((row0 + lane / 16) * pitch + x_from);
    const uint32_t e_off = (uint32_t)((row0 + lane % 4) * blocks + e_from);
    const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char*)lds);
    // step p of this split, clamped: what lies past its end is loaded and never read
    auto clamped = [&](int64_t p) { return max(min(f0 + p - tail, f1 - 1), (int64_t)0); };
    auto load_d = [&](int64_t p, int half) {
        const char* const d = (const char*)a.dy + clamped(p) * STEP * d_pitch;
        const uint32_t to = base + AT_D + (uint32_t)(p % D_RING) * D_SLOT + row0 * (DIRECT * 2);
        load_16_to_lds(to + half * 2 * DIRECT * 2, half ? d_off1 : d_off0, d);
    };
    auto load_codes = [&](int64_t p) {
        load_16_to_lds(base + AT_X + (uint32_t)(p % X_RING) * X_SLOT + row0 * DIRECT, x_off,
                       (const char*)a.codes + clamped(p) * STEP * pitch);
    };
    auto load_exponents = [&](int64_t p) {
        load_byte_to_lds(base + AT_E + (uint32_t)(p % X_RING) * E_SLOT + wave * WAVE * 4, e_off,
                         (const char*)a.exponents + clamped(p) * STEP * blocks);
    };
    auto load_x = [&](int64_t p) {
        load_codes(p);
        load_exponents(p);
    };
    // the rows behind the last whole step, as step 0; zeros behind them
    auto load_tail = [&] {
        const int64_t t0 = whole_steps * STEP;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int t = row0 + 2 * j + lane / 32;
            u32x4 v{};
            if (t0 + t < a.rows) v = *(const u32x4*)((const char*)a.dy + (t0 + t) * d_pitch + d_from(t));
            *(u32x4*)(lds + AT_D + t * (DIRECT * 2) + lane % 32 * 16) = v;
        }
        const int t = row0 + lane / 16, te = row0 + lane % 4;
        u32x4 v{};
        if (t0 + t < a.rows) v = *(const u32x4*)(a.codes + (t0 + t) * pitch + x_from);
        *(u32x4*)(lds + AT_X + t * DIRECT + lane % 16 * 16) = v;
        *(uint32_t*)(lds + AT_E + (wave * WAVE + lane) * 4) = t0 + te < a.rows ? a.exponents[(t0 + te) * blocks + e_from] : 0u;
    };

    // ---- conversion: rows 4 w .. 4 w + 3 of columns 4 l .. 4 l + 3, half of octet w / 2
    const int col = 4 * lane;
    const Places put = places(AT_B + col / 4 * 256 + (wave & 1) * 8, (wave >> 1) ^ ((col >> 2) & 1) * 3 ^ ((col >> 3) & 1) * 2 ^
                                                                          ((col >> 4) & 3) * 4);
    const int raw_x = AT_X + row0 * DIRECT + col, raw_e = AT_E + (wave * WAVE + lane) * 4;
    struct Raw4 { uint32_t c[4], e; };
    auto read_raw = [&](int slot, Raw4& r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.c[i] = *(const uint32_t*)(lds + raw_x + slot * X_SLOT + i * DIRECT);
        r.e = *(const uint32_t*)(lds + raw_e + slot * E_SLOT);
    };
    auto convert = [&](int buf, const Raw4& r, int c) {
        const uint32_t e[4] = {dpp<0x00>(r.e), dpp<0x55>(r.e), dpp<0xAA>(r.e), dpp<0xFF>(r.e)};
        u32x2 v;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float lo = (float)(int8_t)(r.c[2 * i] >> (8 * c)) * __uint_as_float(e[2 * i] << 23);
            const float hi = (float)(int8_t)(r.c[2 * i + 1] >> (8 * c)) * __uint_as_float(e[2 * i + 1] << 23);
            v[i] = high_halves(__float_as_uint(lo), __float_as_uint(hi));
        }
        *(u32x2*)(lds + buf * (DIRECT * COL_BYTES) + put.at[c]) = v;
    };

    // ---- the product: lane l holds column l % 16 of a fragment, octet l / 16
    const int wk = wave / 4 * WK, wn = wave % 4 * WN;
    const Places get_x = places(AT_B + wk / 4 * 256 + (lane & 15) / 4 * 256,
                                (lane >> 4) ^ (lane & 3) * 4 ^ ((lane >> 2) & 1) * 3 ^ ((lane >> 3) & 1) * 2);
    int get_d[FN];  // four t of column wn + 16 j + l % 16, as the transposed read wants them addressed
    {
        const int t = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
        for (int j = 0; j < FN; ++j) get_d[j] = AT_D + t * (DIRECT * 2) + ((wn / 16 + j) ^ unit(t)) * 32 + (lane & 3) * 8;
    }
    auto read_x = [&](int buf, int i) {
        return *(const bf16x8*)(lds + buf * (DIRECT * COL_BYTES) + get_x.at[i & 3] + i * 1024);
    };
    auto read_d = [&](int slot, int j) {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        union { s16x4 h[2]; bf16x8 v; } u;
#pragma unroll
        for (int half = 0; half < 2; ++half)  // rows t + 4 half: the same xor
            u.h[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(lds_char*)(lds + slot * D_SLOT + get_d[j] + half * 4 * DIRECT * 2));
        return u.v;
    };
    f32x4 acc[FK][FN];
#pragma unroll
    for (int i = 0; i < FK; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    if (steps > 0) {
        if (tail) {
            load_tail();
        } else {
            load_d(0, 0);
            load_d(0, 1);
            load_x(0);
        }
        for (int p = 1; p < 3; ++p) {
            load_d(p, 0);
            load_d(p, 1);
        }
        load_x(1);
        load_x(2);
        load_x(3);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        Raw4 raw;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            read_raw(p, raw);
#pragma unroll
            for (int c = 0; c < 4; ++c) convert(p, raw, c);
        }
        __syncthreads();
        load_x(4);
        struct Fragments {
            bf16x8 y[FN], x[2];
        };
        Fragments f, g;
#pragma unroll
        for (int j = 0; j < FN; ++j) f.y[j] = read_d(0, j);
        f.x[0] = read_x(0, 0);
        f.x[1] = read_x(0, 1);
        int b = 0;  // q % 3
        auto step = [&](int64_t q, Fragments& f, Fragments& g) {
            const int b1 = b == 2 ? 0 : b + 1, b2 = b1 == 2 ? 0 : b1 + 1;
            read_raw((int)((q + 2) % X_RING), raw);
#pragma unroll
            for (int i = 0; i < FK; ++i) {
                const bf16x8 xi = f.x[i & 1];
                if (i + 2 < FK) f.x[i & 1] = read_x(b, i + 2);
                else g.x[i & 1] = read_x(b1, i + 2 - FK);
                if (i + 2 >= FK) {
#pragma unroll
                    for (int j = (i + 2 - FK) * FN / 2; j < (i + 3 - FK) * FN / 2; ++j)
                        g.y[j] = read_d((int)((q + 1) % D_RING), j);
                }
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xi, f.y[j], acc[i][j], 0, 0, 0);
                if (i >= 1 && i < 5) convert(b2, raw, i - 1);
                // one load at a time: a wave that sends them together waits until the others' are taken
                if (i == 0) load_d(q + 3, 0);
                if (i == 2) load_d(q + 3, 1);
                if (i == 4) load_codes(q + 5);
                if (i == 6) load_exponents(q + 5);
#pragma unroll
                for (int k = 0; k < FN; ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction,
                    __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // up to six vector ones beside it
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
            __syncthreads();
            b = b1;
        };
        for (int64_t q = 0; q < steps; q += 2) {
            step(q, f, g);
            if (q + 1 < steps) step(q + 1, g, f);
        }
        // nothing may land in LDS that is another workgroup's by then
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    store_tile(a, splits == 1 ? nullptr : partial + (int64_t)split * a.outs * a.cols, acc, k0 + wk, n0 + wn);
}

// Adds the splits' partial sums in their order.  Bound by memory: eight of 2304 x 768
// 10.1 us (5.6 TB/s read).
__global__ __launch_bounds__(256) void k_wgrad_join(const rf_weight_grad a, const float* __restrict__ partial,
                                                    uint32_t splits)
{
    const int64_t n = a.outs * a.cols, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    const int left = (int)min((int64_t)4, n - at);
    float s[4] = {};
    for (uint32_t p = 0; p < splits; p += 8) {  // eight loads in flight
        f32x4 v[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            v[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (p + k < splits) {
                const float* const q = partial + (int64_t)(p + k) * n + at;
                if (left == 4) {
                    v[k] = __builtin_bit_cast(f32x4, (u32x4) * (const u32x4_at*)q);
                } else {
                    for (int i = 0; i < 3; ++i)
                        if (i < left) v[k][i] = q[i];
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
            for (int i = 0; i < 4; ++i) s[i] += v[k][i];
    }
    for (int i = 0; i < left; ++i)
        put_scalar(a.out, a.out_dtype, at + i, a.accumulate ? scalar_at(a.out, a.out_dtype, at + i) + s[i] : s[i]);
}

// Tile and split of a call.
struct Plan {
    bool big, direct;
    uint32_t tiles_k, tiles, splits;
    int64_t workspace;
};

// The cheapest of the tiles and splits by what they take (us, measured on one
// GPU): 7 for a round of workgroups, `step` for 32 rows, and, split, 3 and the
// partial sums at 4 TB/s.  Workgroups at a time: one a CU with 256 x 256 tiles
// and with three pieces (LDS), else two.
Plan plan_of(const rf_weight_grad& a, int cus)
{
    Plan best{};
    double least = 1e30;
    const int64_t steps = (a.rows + STEP - 1) / STEP;
    for (int big = 0; big < (a.dy_dtype == RF_BF16 ? 2 : 1); ++big) {
        Plan p{};
        const int64_t tile = big ? 256 : 128;
        p.big = big != 0;
        p.tiles_k = (uint32_t)((a.cols + tile - 1) / tile);
        p.tiles = p.tiles_k * (uint32_t)((a.outs + tile - 1) / tile);
        const int64_t room = (int64_t)cus * (big || a.dy_dtype == RF_F32 ? 1 : 2);
        p.direct = big && a.rows >= STEP && a.outs % 8 == 0 && a.dy_stride % 8 == 0 && ((uintptr_t)a.dy & 15) == 0;
        const double step = big ? 1.0 : a.dy_dtype == RF_F32 ? 2.4 : a.dy_dtype == RF_F16 ? 1.4 : 0.9;
        for (int64_t n = 1; n <= std::min<int64_t>(std::max<int64_t>(1, steps), 64); ++n) {
            const double rounds = (double)((p.tiles * n + room - 1) / room);
            const double us = rounds * (7 + step * (double)((steps + n - 1) / n)) +
                              (n > 1 ? 3 + (double)n * (double)a.outs * (double)a.cols * 8 / 4e6 : 0);
            if (us < least) {
                least = us;
                best = p;
                best.splits = (uint32_t)n;
            }
        }
    }
    best.workspace = best.splits > 1 ? (int64_t)best.splits * a.outs * a.cols * 4 : 0;
    return best;
}

template <typename T, int TILE, int WK, int WN, bool EDGE>
rf_status launch(const rf_weight_grad& a, const Plan& p, float* partial, hipStream_t st)
{
    constexpr size_t LDS = 3 * (size_t)(1 + Pieces<T>::n) * TILE * COL_BYTES;
    static std::atomic<uint64_t> done;
    const auto f = k_wgrad<T, TILE, WK, WN, EDGE>;
    if (const rf_status s = allow_lds((const void*)f, LDS, done); s != RF_OK) return s;
    f<<<p.tiles * p.splits, WK * WN * WAVE, LDS, st>>>(a, partial, p.tiles_k, p.tiles, p.splits);
    return RF_OK;
}

rf_status launch_direct(const rf_weight_grad& a, const Plan& p, float* partial, hipStream_t st)
{
    static std::atomic<uint64_t> done;
    if (const rf_status s = allow_lds((const void*)k_wgrad_direct, DIRECT_LDS, done); s != RF_OK) return s;
    k_wgrad_direct<<<p.tiles * p.splits, DIRECT_WAVES * WAVE, DIRECT_LDS, st>>>(a, partial, p.tiles_k, p.tiles, p.splits);
    return RF_OK;
}

template <typename T, int TILE, int WK, int WN>
rf_status launch(const rf_weight_grad& a, const Plan& p, float* partial, hipStream_t st)
{
    return a.outs % 4 ? launch<T, TILE, WK, WN, true>(a, p, partial, st) : launch<T, TILE, WK, WN, false>(a, p, partial, st);
}

bool known(int32_t dtype) { return dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16; }

rf_status check(const rf_weight_grad* a)
{
    if (!a) return report(RF_ERR_INVALID, "null arguments");
    if (a->rows < 0 || a->rows >= (1ll << 31) || a->outs < 1 || a->outs >= (1ll << 24) || a->cols < 1 ||
        a->cols >= (1ll << 24))
        return report(RF_ERR_INVALID, "rows, outs or cols out of range");
    if (!known(a->dy_dtype) || !known(a->out_dtype)) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
    if (((uintptr_t)a->codes & 15) != 0) return report(RF_ERR_INVALID, "checkpoint codes must be 16-byte aligned");
    // a step's rows are addressed by 32 bits
    if (a->dy_stride < 0 || a->dy_stride >= (1ll << 24)) return report(RF_ERR_UNSUPPORTED, "dy's row stride out of range");
    if (((a->outs + 127) / 128) * ((a->cols + 127) / 128) > (1ll << 22))
        return report(RF_ERR_UNSUPPORTED, "too many outputs for one launch");
    return RF_OK;
}

}  // namespace

rf_status rfb::allow_lds(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) noexcept
{
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return rf::report_hip(e, "hipGetDevice");
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bytes <= 64 * 1024 || (done.load(std::memory_order_relaxed) & bit)) return RF_OK;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return rf::report_hip(e, "hipFuncSetAttribute");
    done.fetch_or(bit, std::memory_order_relaxed);
    return RF_OK;
}

extern "C" {

rf_status rf_linear_weight_grad_workspace(const rf_weight_grad* args, int64_t* bytes)
{
    if (!bytes) return report(RF_ERR_INVALID, "null output");
    if (const rf_status s = check(args); s != RF_OK) return s;
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    *bytes = plan_of(*args, cus).workspace;
    return RF_OK;
}

rf_status rf_linear_weight_grad(const rf_weight_grad* args, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (const rf_status s = check(args); s != RF_OK) return s;
    const rf_weight_grad& a = *args;
    if (!a.out || (a.rows && (!a.dy || !a.codes || !a.exponents))) return report(RF_ERR_INVALID, "null buffer");
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    const Plan p = plan_of(a, cus);
    if (p.workspace > workspace_bytes || (p.workspace && !workspace))
        return report(RF_ERR_INVALID, "workspace too small");
    hipStream_t st = (hipStream_t)stream;
    float* const partial = (float*)workspace;
    rf_status s;
    if (a.dy_dtype == RF_F32) s = launch<float, 128, 2, 2>(a, p, partial, st);
    else if (a.dy_dtype == RF_F16) s = launch<f16, 128, 2, 2>(a, p, partial, st);
    else if (p.direct) s = launch_direct(a, p, partial, st);
    else if (p.big) s = launch<bf16, 256, 2, 4>(a, p, partial, st);
    else s = launch<bf16, 128, 2, 2>(a, p, partial, st);
    if (s != RF_OK) return s;
    if (p.splits > 1) {
        const int64_t grid = (a.outs * a.cols + 1023) / 1024;
        k_wgrad_join<<<(unsigned)grid, 256, 0, st>>>(a, partial, p.splits);
    }
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return rf::report_hip(e, "rf_linear_weight_grad");
    return RF_OK;
}

}  // extern "C"
