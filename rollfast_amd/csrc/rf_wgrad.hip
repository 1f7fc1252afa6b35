// rf_wgrad.hip -- a linear layer's weight gradient from its input's 8-bit
// checkpoint: out[n, k] = sum_t dy[t, n] code[t, k] 2^(e[t, k / 32] - 127).
//
// A code times its power-of-two step is exact in bf16, and dy is the sum of
// bf16 pieces (bf16: itself; f16, 11 bits: two; f32, 24 bits: three of 8 bits
// each, cut off, not rounded), so every product that the matrix cores form is
// exact and only the f32 sums round.
//
// Both operands have the summed index t along the rows, while the matrix
// instructions want each lane to hold eight t of one column.  The transpose is
// done on the way into LDS: a lane loads eight rows of four neighbouring
// columns and writes four 16-byte vectors, each the eight t of a column.  The
// codes pass through registers for their conversion anyway, so it costs them
// nothing, and dy half an instruction per element.
#include <algorithm>

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
template <typename T, int TILE, int WAVES_K, int WAVES_N, bool EDGE>
__global__ __launch_bounds__(WAVES_K* WAVES_N* WAVE) void k_wgrad(const rf_weight_grad a, float* __restrict__ partial,
                                                                 uint32_t tiles_k, uint32_t tiles, uint32_t splits)
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
        auto step = [&](int64_t q, auto& regs, Fragments& f, Fragments& g) {
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
                if (i < 4) stage(after, regs, i);
                if (FK == 8 && i >= 4) {
                    load(ahead, regs, 2 * (i - 4));
                    load(ahead, regs, 2 * (i - 4) + 1);
                }
                if (FK == 4 && i == 3) {
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
            for (int64_t q = 0; q < steps; q += 2) {
                step(q, even, f, g);
                if (q + 1 < steps) step(q + 1, odd, g, f);
            }
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

    // ---- a lane holds four neighbouring columns of an output's row
    const bool whole = splits == 1;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int64_t n = n0 + wn + 16 * j + lane % 16;
        if (n >= a.outs) continue;
#pragma unroll
        for (int i = 0; i < FK; ++i) {
            const int64_t k = k0 + wk + 16 * i + lane / 16 * 4, left = a.cols - k, at = n * a.cols + k;
            if (!whole) {
                float* const o = partial + (int64_t)split * a.outs * a.cols + at;
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

// Adds the splits' partial sums in their order.
__global__ __launch_bounds__(256) void k_wgrad_join(const rf_weight_grad a, const float* __restrict__ partial,
                                                    uint32_t splits)
{
    const int64_t n = a.outs * a.cols, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    const int left = (int)min((int64_t)4, n - at);
    float s[4] = {};
    for (uint32_t p = 0; p < splits; ++p) {
        const float* const q = partial + (int64_t)p * n + at;
        if (left == 4) {
            const f32x4 v = __builtin_bit_cast(f32x4, (u32x4) * (const u32x4_at*)q);
            for (int i = 0; i < 4; ++i) s[i] += v[i];
        } else {
            for (int i = 0; i < left; ++i) s[i] += q[i];
        }
    }
    for (int i = 0; i < left; ++i)
        put_scalar(a.out, a.out_dtype, at + i, a.accumulate ? scalar_at(a.out, a.out_dtype, at + i) + s[i] : s[i]);
}

// Tile and split of a call.
struct Plan {
    bool big;
    uint32_t tiles_k, tiles, splits;
    int64_t workspace;
};

// The cheapest of the tiles and splits by what they take (us, measured on one
// GPU): 5 for a round of workgroups, `step` for 32 rows, and, split, 3 and the
// partial sums at 4 TB/s.  Workgroups at a time: one a CU with 256 x 256 tiles
// and with two or three pieces, else two.
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
        const int64_t room = (int64_t)cus * (big || a.dy_dtype != RF_BF16 ? 1 : 2);
        const double step = big ? 1.05 : a.dy_dtype == RF_F32 ? 1.2 : 0.9;
        for (int64_t n = 1; n <= std::min<int64_t>(std::max<int64_t>(1, steps), 64); ++n) {
            const double rounds = (double)((p.tiles * n + room - 1) / room);
            const double us = rounds * (5 + step * (double)((steps + n - 1) / n)) +
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
    const auto f = k_wgrad<T, TILE, WK, WN, EDGE>;
    if (LDS > 64 * 1024) {
        static const hipError_t e = hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS);
        if (e != hipSuccess) return rf::report_hip(e, "hipFuncSetAttribute");
    }
    f<<<p.tiles * p.splits, WK * WN * WAVE, LDS, st>>>(a, partial, p.tiles_k, p.tiles, p.splits);
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
