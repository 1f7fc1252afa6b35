// rf_loss.hip -- softmax cross entropy of logits = hidden weight^T over a large
// vocabulary, with the gradients of hidden and weight, without the logits of all
// tokens.
//
// With z[t, v] a token's logits, lse_t = log sum_v exp z[t, v] and y_t its target,
//   loss_t = lse_t - z[t, y_t] + z_loss lse_t^2,
//   dz[t, v] = dloss_t ((1 + 2 z_loss lse_t) exp(z[t, v] - lse_t) - [v = y_t]),
//   dhidden = dz weight,  dweight = dz^T hidden.
// Tokens that are ignored, or whose target is no row of weight (their loss is
// NaN), are told apart first; the rows that count are packed, so that the others
// cost nothing, and what lies in them, NaN included, reaches no sum.
//
//   k_select   the rows that count, in order, behind them the others
//   k_pack     their hidden vectors, k padded with zeros to whole steps
//   k_logits   a product's tile of logits becomes, for each token and each block
//              of the vocabulary (a wave's part of the tile: 64 or 128 entries), a
//              maximum m and a sum s of exp(z - m); for gradients exp(z - m) itself
//              too, in f16 (f32 tensors: in f32)
//   k_rows     lse and loss from m and s, factors of the gradient
//   k_dlogits  exp(z - m) to dz, in place (f32: to two f16 planes)
//   k_product  dhidden and dweight, two products of the same size
// Loss alone ends with k_rows and writes no logits.  With gradients a piece of
// tokens at a time holds at most PIECE bytes of exponentials; the pieces'
// weight gradients are added in f32.  Three products, none computed twice.
//
// exp(z - m) is in [0, 1]: f16 rounds it by at most 2^-12 of its value (below
// 2^-14 by 2^-25), a sixteenth of what bf16's rounding of dz adds.  At the target
// dz comes from the f32 logit through expm1, since 1 - p cancels there.
//
// f32 tensors go to the matrix cores as two f16 planes each, high and low parts of
// x 2^e (22 bits; e such that the tensor's largest finite magnitude is below
// 2^15), in three products: high high, high low, low high.
#include <algorithm>
#include <type_traits>

#include "rf_product.h"

using namespace rfb;
using namespace rfp;
using rf::report;

namespace {

constexpr int64_t PIECE = 2ll << 30;        // bytes of exponentials held at once
constexpr int64_t STATS = 256ll << 20;      // bytes of m and s held at once

// Written by the kernels, read by later ones.
struct Scalars {
    int32_t count, pad[3];
    uint32_t hidden_top, weight_top;  // f32: bits of the largest finite magnitudes
    uint32_t pad2[2];
    uint32_t dz_top[1];               // of each piece: bits of the largest row factor
};

// The power of two that brings magnitudes up to `top` below 2^15 (1: nothing finite, or zero).
__device__ __forceinline__ float scale_of(uint32_t top)
{
    if (top == 0) return 1.0f;
    const int e = min(max((int)(top >> 23) - 127, -100), 100);
    return __uint_as_float((uint32_t)(14 - e + 127) << 23);
}

__device__ __forceinline__ float inverse(float power_of_two) { return __uint_as_float((254u << 23) - __float_as_uint(power_of_two)); }

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// Raises *top to at least x.  Read first: it seldom has to be raised, and thousands
// of atomics on one address would take 12 ns each.  (The order does not matter to a
// maximum.)
__device__ __forceinline__ void raise(uint32_t* top, uint32_t x)
{
    if (x > __hip_atomic_load(top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(top, x);
}

constexpr int SELECT = 1024, RUN = 8;  // threads, tokens of a thread at a time

// order[0 .. count): the tokens that count, in order; the others, whose loss is
// set, from the end on backwards.  target[i]: of token order[i], -1 where it is no
// row of weight.  One workgroup: 16384 tokens take 8 us.
template <typename I>
__global__ __launch_bounds__(SELECT) void k_select(const I* __restrict__ targets, int64_t tokens, int64_t ignore, int64_t vocab,
                                                  float* __restrict__ loss, int32_t* __restrict__ order,
                                                  int32_t* __restrict__ target, Scalars* sc, int pieces)
{
    __shared__ int32_t part[2][SELECT / WAVE];
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    int32_t before = 0;  // tokens that count in the runs before
    for (int64_t at = 0, turn = 0; at < tokens; at += SELECT * RUN, turn ^= 1) {
        const int64_t t0 = at + tid * RUN;
        int64_t y[RUN];
        int32_t mine = 0;
#pragma unroll
        for (int k = 0; k < RUN; ++k) y[k] = t0 + k < tokens ? (int64_t)targets[t0 + k] : ignore;
#pragma unroll
        for (int k = 0; k < RUN; ++k) mine += y[k] != ignore;
        int32_t upto = mine;  // inclusive sum over the wave, then the waves before
        for (int d = 1; d < WAVE; d *= 2) {
            const int32_t v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == WAVE - 1) part[turn][wave] = upto;
        __syncthreads();  // (the other half of part may still be read)
        int32_t all = 0, ahead = 0;
        for (int w = 0; w < SELECT / WAVE; ++w) {
            const int32_t n = part[turn][w];
            if (w < wave) ahead += n;
            all += n;
        }
        int32_t on = before + ahead + upto - mine;  // tokens that count before this run
        int64_t off = tokens - 1 - (t0 - on);       // the next place of the others
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            const int64_t t = t0 + k;
            if (t >= tokens) break;
            if (y[k] != ignore) {
                order[on] = (int32_t)t;
                target[on++] = y[k] >= 0 && y[k] < vocab ? (int32_t)y[k] : -1;
            } else {
                order[off--] = (int32_t)t;
                loss[t] = 0.0f;
            }
        }
        before += all;
    }
    if (tid == 0) {
        sc->count = before;
        sc->hidden_top = sc->weight_top = 0;
    }
    for (int i = tid; i < pieces; i += SELECT) sc->dz_top[i] = 0;
}

// Largest finite magnitude of rows (of those that count, where order is given).
__global__ __launch_bounds__(256) void k_top(const float* __restrict__ x, int64_t rows, int64_t cols, int64_t stride,
                                            const int32_t* __restrict__ order, const Scalars* sc, uint32_t* top)
{
    if (order) rows = sc->count;
    uint32_t best = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float* const row = x + (order ? order[r] : r) * stride;
        for (int64_t c = threadIdx.x; c < cols; c += 256) {
            const uint32_t v = __float_as_uint(row[c]) & 0x7FFFFFFFu;
            best = max(best, v < 0x7F800000u ? v : 0u);
        }
    }
    for (int d = 1; d < WAVE; d *= 2) best = max(best, (uint32_t)__shfl_xor((int)best, d));
    if (threadIdx.x % WAVE == 0) raise(top, best);
}

// A high and a low part in f16 of scaled values.
__device__ __forceinline__ void split8(const float (&v)[8], float scale, Raw<f16>& hi, Raw<f16>& lo)
{
    float h[8], l[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = v[k] * scale;
    hi = narrow8<f16>(h);
    float back[8];
    widen8(hi, back);
#pragma unroll
    for (int k = 0; k < 8; ++k) l[k] = h[k] - back[k];
    lo = narrow8<f16>(l);
}

// Rows into the product's layout: 16 bits, columns padded with zeros to `pitch`.
// With `order`: the rows that count, zeros up to a whole step behind them, and
// zeros in the rows of `clear` that do not count.
template <typename T>
__global__ __launch_bounds__(256) void k_pack(const T* __restrict__ x, int64_t cols, int64_t stride, int64_t pitch,
                                             const int32_t* __restrict__ order, const Scalars* sc, const uint32_t* top,
                                             uint16_t* __restrict__ hi, uint16_t* __restrict__ lo, T* __restrict__ clear,
                                             int64_t rows)
{
    const int64_t r = blockIdx.x;
    int64_t from = r;
    bool zero = false;
    if (order) {
        const int64_t count = sc->count;
        zero = r >= count;
        if (r < rows) from = order[r];
        if (zero && r < rows && clear)
            for (int64_t c = (int64_t)threadIdx.x * 8; c < cols; c += 2048) put8(clear + from * cols + c, Raw<T>{}, cols - c);
        if (r >= (count + STEP - 1) / STEP * STEP) return;
    }
    const T* const row = x + from * stride;
    float scale = 1.0f;
    if constexpr (sizeof(T) == 4) scale = scale_of(*top);
    for (int64_t c = (int64_t)threadIdx.x * 8; c < pitch; c += 2048) {
        Raw<T> v{};
        if (!zero && c < cols) v = load8(row, c, cols);
        if constexpr (sizeof(T) == 4) {
            float w[8];
            widen8(v, w);
            Raw<f16> h, l;
            split8(w, scale, h, l);
            *(u32x4*)(hi + r * pitch + c) = h.a;
            *(u32x4*)(lo + r * pitch + c) = l.a;
        } else {
            *(u32x4*)(hi + r * pitch + c) = v.a;
        }
    }
}

// ------------------------------------------------------------- the logits ---
struct Logits {
    Side weight, hidden;           // p: vocabulary, q: packed tokens
    int64_t vocab, pitch;          // pitch of the exponentials, in elements: vocab to a whole step
    int64_t first, rows;           // packed tokens of this piece
    int64_t steps;
    int32_t pairs, blocks;         // blocks of the vocabulary
    const Scalars* sc;
    const int32_t* target;
    float2* stats;                 // [rows, blocks] m, s
    float* picked;                 // [rows] the target's logit
    void* e;                       // [rows, pitch] exp(z - m)
    uint32_t tiles_p, tiles_q;
};

// E: what is kept of the exponentials: nothing, f16 or f32.
template <typename H, typename E, int TILE, int WP, int WQ>
__global__ __launch_bounds__(WP* WQ* WAVE, 2) void k_logits(const Logits a)
{
    typedef Product<H, KALONG, KALONG, TILE, TILE, WP, WQ> G;
    extern __shared__ char lds[];
    const TileAt tile = tile_at(xcd_order(blockIdx.x, a.tiles_p * a.tiles_q), a.tiles_p, a.tiles_q);
    const int64_t count = min((int64_t)a.sc->count - a.first, a.rows);
    const int64_t p0 = (int64_t)tile.p * TILE, q0 = (int64_t)tile.q * TILE;
    if (q0 >= count) return;
    typename G::Sums acc;
    G::run(lds, a.weight, a.hidden, p0, q0, 0, a.steps, a.pairs, acc);
    const int lane = threadIdx.x % WAVE;
    float unscale = 1.0f;
    if (a.pairs > 1) unscale = inverse(scale_of(a.sc->hidden_top)) * inverse(scale_of(a.sc->weight_top));
    const int64_t v0 = p0 + G::wp() + lane / 16 * 4;
    if (a.pairs > 1) {
#pragma unroll
        for (int j = 0; j < G::FQ; ++j)
#pragma unroll
            for (int i = 0; i < G::FP; ++i) acc[i][j] *= unscale;
    }
    if (p0 + G::wp() + TILE / WP > a.vocab) {
#pragma unroll
        for (int j = 0; j < G::FQ; ++j)
#pragma unroll
            for (int i = 0; i < G::FP; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (v0 + 16 * i + r >= a.vocab) acc[i][j][r] = -__builtin_inff();
    }
    constexpr float LOG2E = 1.44269504088896341f;
#pragma unroll
    for (int j = 0; j < G::FQ; ++j) {
        const int64_t q = q0 + G::wq() + 16 * j + lane % 16;
        const bool mine = q < count;
        const int64_t y = mine ? a.target[a.first + q] - v0 : -1;
        if (__any(y >= 0 && y < TILE / WP)) {  // few waves hold a target
#pragma unroll
            for (int i = 0; i < G::FP; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (y == 16 * i + r) a.picked[q] = acc[i][j][r];
        }
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < G::FP; ++i)
            m = fmaxf(fmaxf(fmaxf(m, acc[i][j][0]), acc[i][j][1]), fmaxf(acc[i][j][2], acc[i][j][3]));
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        // exp(z - m) = 2^(z log2(e) - m log2(e)), the product in one rounding with the
        // difference; where nothing is here, exponentials of -inf are 0
        const float base = m == -__builtin_inff() ? 0.0f : m * -LOG2E;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < G::FP; ++i) {
            f32x4 e;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], LOG2E, base));
                s += e[r];
            }
            const int64_t v = v0 + 16 * i;
            if constexpr (!__is_same(E, void)) {
                if (mine && v < a.pitch) {
                    E* const o = (E*)a.e + q * a.pitch + v;
                    if constexpr (sizeof(E) == 4) {
                        *(f32x4*)o = e;
                    } else {
                        const f16x2 lo = __builtin_convertvector((f32x2{e[0], e[1]}), f16x2);
                        const f16x2 hi = __builtin_convertvector((f32x2{e[2], e[3]}), f16x2);
                        *(u32x2*)o = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
                    }
                }
            }
        }
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (mine) {
            const int64_t block = (p0 + G::wp()) / (TILE / WP);
            if (lane < 16 && block < a.blocks) a.stats[q * a.blocks + block] = make_float2(m, s);
        }
    }
}

struct Rows {
    int64_t first, rows, pitch;
    int32_t blocks, shift;  // entries of a block: 1 << shift
    int32_t piece, reduction;
    float z_loss;
    const Scalars* sc;
    uint32_t* dz_top;
    const int32_t *order, *target;
    const float2* stats;
    const float *picked, *dloss;
    float *loss, *top, *factor, *at_target;  // [rows] each but loss
    const void* e;
    void* dz;
    uint16_t* dz_low;
};

// A wave a token.
__global__ __launch_bounds__(256) void k_rows(const Rows a)
{
    const int64_t q = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
    if (q >= min((int64_t)a.sc->count - a.first, a.rows)) return;
    const int lane = threadIdx.x % WAVE;
    const float2* const stats = a.stats + q * a.blocks;
    float m = -__builtin_inff();
    for (int b = lane; b < a.blocks; b += WAVE) m = fmaxf(m, stats[b].x);
    for (int d = 1; d < WAVE; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    float s = 0.0f;
    for (int b = lane; b < a.blocks; b += WAVE) {
        const float2 x = stats[b];
        s += x.y * exp_of(x.x - m);
    }
    s = wave_sum(s);
    if (lane) return;
    const int32_t t = a.order[a.first + q];
    const bool known = a.target[a.first + q] >= 0;
    const float logs = logf(s), lse = m + logs, nan = __builtin_nanf("");
    const float below = known ? a.picked[q] - m - logs : nan;  // the target's log probability
    a.loss[t] = a.z_loss * lse * lse - below;
    if (!a.factor) return;
    float dl = a.dloss ? a.dloss[t] : a.reduction == RF_REDUCE_MEAN ? 1.0f / (float)a.sc->count : 1.0f;
    if (!known) dl = nan;
    const float spread = 1.0f + 2.0f * a.z_loss * lse;
    a.top[q] = m;
    a.factor[q] = dl * spread / s;
    a.at_target[q] = dl * (expm1f(below) + (spread - 1.0f) * expf(below));
    const uint32_t most = __float_as_uint(fmaxf(fabsf(dl * spread), fabsf(dl)));
    if (most < 0x7F800000u) raise(a.dz_top + a.piece, most);
}

// The sum or the mean of the losses that count: one workgroup, in a fixed order, in f64.
__global__ __launch_bounds__(SELECT) void k_total(const float* __restrict__ loss, const int32_t* __restrict__ order,
                                                 const Scalars* sc, int reduction, float* __restrict__ total)
{
    __shared__ double part[SELECT];
    const int tid = threadIdx.x, count = sc->count;
    double s = 0;
    for (int i = tid; i < count; i += SELECT) s += (double)loss[order[i]];
    part[tid] = s;
    __syncthreads();
    for (int d = SELECT / 2; d; d /= 2) {
        if (tid < d) part[tid] += part[tid + d];
        __syncthreads();
    }
    if (tid == 0) *total = (float)(reduction == RF_REDUCE_MEAN ? part[0] / (double)count : part[0]);
}

// dz is held as a fraction of the largest row factor (f16: of 2^14): a mean's
// dloss is the same for all tokens, and most of their targets' dz are then just
// below one, where bf16's rounding is least.
__device__ __forceinline__ float dz_scale(uint32_t top, bool wide)
{
    const float t = __uint_as_float(top);
    return t < 1e-30f ? 1.0f : (wide ? 1.0f : 16384.0f) / t;
}

// dz of a token from its exponentials; zeros up to a whole step of
// tokens.  A workgroup a token.  P: dz's type; E: the exponentials'.
template <typename P, typename E> __global__ __launch_bounds__(256) void k_dlogits(const Rows a)
{
    extern __shared__ float of_block[];
    const int64_t q = blockIdx.x, count = min((int64_t)a.sc->count - a.first, a.rows);
    if (q >= (count + STEP - 1) / STEP * STEP) return;
    P* const out = (P*)a.dz + q * a.pitch;
    if (q >= count) {
        for (int64_t v = (int64_t)threadIdx.x * 8; v < a.pitch; v += 2048) {
            *(u32x4*)(out + v) = u32x4{};
            if (sizeof(E) == 4) *(u32x4*)(a.dz_low + q * a.pitch + v) = u32x4{};
        }
        return;
    }
    const float scale = dz_scale(a.dz_top[a.piece], __is_same(P, bf16));
    const float m = a.top[q], f = a.factor[q] * scale;
    for (int b = threadIdx.x; b < a.blocks; b += 256) {
        const float top = a.stats[q * a.blocks + b].x;
        of_block[b] = top == -__builtin_inff() ? 0.0f * f : exp_of(top - m) * f;
    }
    __syncthreads();
    const int64_t y = a.target[a.first + q];
    const float at = a.at_target[q] * scale;
    const E* const in = (const E*)a.e + q * a.pitch;
    for (int64_t v = (int64_t)threadIdx.x * 8; v < a.pitch; v += 2048) {
        Raw<E> raw;
        raw.a = *(const u32x4*)(in + v);
        if constexpr (sizeof(E) == 4) raw.b = *(const u32x4*)(in + v + 4);
        float x[8];
        widen8(raw, x);
        const int64_t b = min(v >> a.shift, (int64_t)a.blocks - 1);
        const float w = of_block[b];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            x[k] *= w;
            if (v + k == y) x[k] = at;
        }
        if constexpr (sizeof(E) == 4) {
            Raw<f16> h, l;
            split8(x, 1.0f, h, l);
            *(u32x4*)(out + v) = h.a;
            *(u32x4*)(a.dz_low + q * a.pitch + v) = l.a;
        } else {
            *(u32x4*)(out + v) = narrow8<P>(x).a;
        }
    }
}

// ---------------------------------------------------------- the gradients ---
struct Grad {
    Side p, q;
    int64_t cols, rows;            // of the output: p below cols, q below rows
    int64_t first, piece_rows;     // packed tokens of this piece
    int64_t steps;                 // of the sum; 0: the tokens that count
    int32_t pairs, dtype, splits, piece;
    const Scalars* sc;
    const uint32_t* dz_top;
    const int32_t* order;          // dhidden: the output's row of packed token q; NULL: dweight
    void* out;
    float* sums;                   // dweight, several pieces: f32 sums so far (may be out)
    int32_t begin, end;            // the first piece, the last one
    float* partial;                // splits > 1: [splits, rows, cols]
    uint32_t tiles_p, tiles_q;
};

__device__ __forceinline__ float unscale_of(const Grad& a)
{
    float u = 1.0f / dz_scale(a.dz_top[a.piece], a.dtype == RF_BF16);
    if (a.pairs > 1) u *= inverse(scale_of(a.order ? a.sc->weight_top : a.sc->hidden_top));
    return u;
}

// Four neighbouring values of an output's row, unscaled sums.
__device__ __forceinline__ void finish(const Grad& a, int64_t q, int64_t p, f32x4 v, float unscale)
{
    const int64_t left = a.cols - p;
    v *= unscale;
    int64_t row = q;
    if (a.order) row = a.order[a.first + q];
    const int64_t at = row * a.cols + p;
    float* sums = nullptr;
    if (!a.order && !(a.begin && a.end)) sums = a.sums + at;
    if (sums && !a.begin) {
        if (left >= 4) v += __builtin_bit_cast(f32x4, *(const u32x4_at*)sums);
        else
            for (int r = 0; r < 3; ++r)
                if (r < left) v[r] += sums[r];
    }
    const int dtype = sums && !a.end ? (int)RF_F32 : a.dtype;
    void* const out = sums && !a.end ? (void*)a.sums : a.out;
    if (left < 4) {
        for (int r = 0; r < 3; ++r)
            if (r < left) put_scalar(out, dtype, at + r, v[r]);
    } else if (dtype == RF_F32) {
        *(u32x4_at*)((float*)out + at) = __builtin_bit_cast(u32x4, v);
    } else {
        uint32_t lo, hi;
        if (dtype == RF_BF16) {
            lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), bf16x2));
            hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), bf16x2));
        } else {
            lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), f16x2));
            hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), f16x2));
        }
        *(u32x2_at*)((uint16_t*)out + at) = u32x2{lo, hi};
    }
}

// dhidden: p the hidden columns of weight (summed down its rows), q the tokens of dz.
// dweight: p the hidden columns of the packed rows, q the vocabulary, both summed over tokens.
template <typename H, Layout LQ, int TILE, int WP, int WQ>
__global__ __launch_bounds__(WP* WQ* WAVE, 2) void k_product(const Grad a)
{
    typedef Product<H, KDOWN, LQ, TILE, TILE, WP, WQ> G;
    extern __shared__ char lds[];
    const uint32_t tiles = a.tiles_p * a.tiles_q, id = xcd_order(blockIdx.x, tiles * a.splits);
    const uint32_t split = id / tiles;
    const TileAt tile = tile_at(id % tiles, a.tiles_p, a.tiles_q);
    const int64_t count = max(min((int64_t)a.sc->count - a.first, a.piece_rows), (int64_t)0);
    const int64_t rows = LQ == KALONG ? count : a.rows;
    const int64_t p0 = (int64_t)tile.p * TILE, q0 = (int64_t)tile.q * TILE;
    if (q0 >= rows) return;
    const int64_t steps = LQ == KALONG ? a.steps : (count + STEP - 1) / STEP;
    if (LQ == KDOWN && !steps && !a.begin && !a.end) return;  // nothing to add
    typename G::Sums acc;
    G::run(lds, a.p, a.q, p0, q0, steps * split / a.splits, steps * (split + 1) / a.splits, a.pairs, acc);
    const int lane = threadIdx.x % WAVE;
    const float unscale = unscale_of(a);
#pragma unroll
    for (int j = 0; j < G::FQ; ++j) {
        const int64_t q = q0 + G::wq() + 16 * j + lane % 16;
        if (q >= rows) continue;
#pragma unroll
        for (int i = 0; i < G::FP; ++i) {
            const int64_t p = p0 + G::wp() + 16 * i + lane / 16 * 4;
            if (p >= a.cols) continue;
            if (a.splits > 1) {
                float* const o = a.partial + (split * a.rows + q) * a.cols + p;
                if (a.cols - p >= 4) *(u32x4_at*)o = __builtin_bit_cast(u32x4, acc[i][j]);
                else
                    for (int r = 0; r < 3; ++r)
                        if (r < a.cols - p) o[r] = acc[i][j][r];
            } else {
                finish(a, q, p, acc[i][j], unscale);
            }
        }
    }
}

// Adds the splits' sums in their order.
__global__ __launch_bounds__(256) void k_join(const Grad a)
{
    const int64_t quads = (a.cols + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t q = i / quads, p = i % quads * 4;
    const int64_t count = max(min((int64_t)a.sc->count - a.first, a.piece_rows), (int64_t)0);
    if (q >= (a.order ? count : a.rows)) return;
    if (!a.order && !count && !a.begin && !a.end) return;
    const float* o = a.partial + q * a.cols + p;
    f32x4 v{};
    for (int s = 0; s < a.splits; ++s, o += a.rows * a.cols) {
        if (a.cols - p >= 4) v += __builtin_bit_cast(f32x4, *(const u32x4_at*)o);
        else
            for (int r = 0; r < 3; ++r)
                if (r < a.cols - p) v[r] += o[r];
    }
    finish(a, q, p, v, unscale_of(a));
}

// ------------------------------------------------------------------- host ---
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Tile of a product, and splits of its sum: the cheapest by what they take
// (us, measured): 6 for a round of workgroups and `step` for 64 k; split, 5 and
// the partial sums at 4 TB/s.  A CU holds one workgroup with tiles of 256, two of 128.
struct Shape {
    bool big;
    uint32_t tiles_p, tiles_q, splits;
    double us;
};

Shape shape_of(int64_t cols, int64_t rows, int64_t steps, bool split, int cus)
{
    Shape best{};
    best.us = 1e30;
    for (int big = 0; big < 2; ++big) {
        const int64_t tile = big ? 256 : 128, tp = (cols + tile - 1) / tile, tq = (rows + tile - 1) / tile;
        const int64_t room = (int64_t)cus * (big ? 1 : 2);
        const double step = big ? 1.65 : 1.15;
        for (int64_t n = 1; n <= (split ? std::min<int64_t>(std::max<int64_t>(1, steps / 2), 64) : 1); ++n) {
            const double rounds = (double)((tp * tq * n + room - 1) / room);
            const double us = rounds * (6 + step * (double)((steps + n - 1) / n)) +
                              (n > 1 ? 5 + (double)n * (double)rows * (double)cols * 8 / 4e6 : 0);
            if (us < best.us) best = Shape{big != 0, (uint32_t)tp, (uint32_t)tq, (uint32_t)n, us};
        }
    }
    return best;
}

struct Plan {
    int64_t pad, vpad, rows, pieces;  // hidden and vocab padded, tokens of a piece, pieces
    bool own_weight, f32, grad;
    int32_t blocks, shift, pairs;
    Shape logits, dhidden, dweight;
    // offsets in the workspace
    int64_t scalars, order, target, stats, picked, top, factor, at_target, hidden, weight, e, dz, sums, partial, bytes;
};

bool known(int32_t dtype) { return dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16; }

Plan plan_of(const rf_cross_entropy& a, int cus)
{
    Plan p{};
    p.f32 = a.dtype == RF_F32;
    p.grad = a.dweight != nullptr;
    p.pairs = p.f32 ? 3 : 1;
    p.pad = up(a.hidden, STEP);
    p.vpad = up(a.vocab, STEP);
    // weight as it is: whole steps of k, 16-byte rows
    p.own_weight = p.f32 || a.hidden % STEP || a.weight_stride % 8 || ((uintptr_t)a.weight & 15) || a.weight_stride * 2 >= (1 << 24);
    const int64_t planes = p.f32 ? 2 : 1, steps = p.pad / STEP;
    p.logits = shape_of(a.vocab, a.tokens, steps * p.pairs, false, cus);
    p.shift = p.logits.big ? 7 : 6;
    p.blocks = (int32_t)((a.vocab + (1 << p.shift) - 1) >> p.shift);
    const int64_t each = p.grad ? p.vpad * (p.f32 ? 8 : 2) : p.blocks * 8, most = p.grad ? PIECE : STATS;
    // pieces of equal numbers of whole tiles
    const int64_t fit = std::max<int64_t>(64, most / each / 256 * 256);
    p.pieces = std::max<int64_t>(1, (a.tokens + fit - 1) / fit);
    p.rows = p.pieces == 1 ? std::max<int64_t>(1, a.tokens) : std::min(fit, up((a.tokens + p.pieces - 1) / p.pieces, 256));
    p.pieces = std::max<int64_t>(1, (a.tokens + p.rows - 1) / p.rows);
    p.logits = shape_of(a.vocab, p.rows, steps * p.pairs, false, cus);
    p.shift = p.logits.big ? 7 : 6;
    p.blocks = (int32_t)((a.vocab + (1 << p.shift) - 1) >> p.shift);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t from = at;
        at += up(bytes, 256);
        return from;
    };
    const int64_t held = up(p.rows, STEP);
    p.scalars = take(sizeof(Scalars) + p.pieces * 4);
    p.order = take(a.tokens * 4);
    p.target = take(a.tokens * 4);
    p.stats = take(p.rows * p.blocks * 8);
    p.picked = take(p.rows * 4);
    p.hidden = take(up(a.tokens, STEP) * p.pad * 2 * planes);
    if (p.own_weight) p.weight = take(a.vocab * p.pad * 2 * planes);
    if (p.grad) {
        p.top = take(p.rows * 4);
        p.factor = take(p.rows * 4);
        p.at_target = take(p.rows * 4);
        p.e = take(held * p.vpad * (p.f32 ? 4 : 2));
        p.dz = p.f32 ? take(held * p.vpad * 4) : p.e;
        if (p.pieces > 1 && !p.f32) p.sums = take(a.vocab * a.hidden * 4);
        p.dhidden = shape_of(a.hidden, p.rows, p.vpad / STEP * p.pairs, true, cus);
        p.dweight = shape_of(a.hidden, a.vocab, held / STEP * p.pairs, true, cus);
        const int64_t h = p.dhidden.splits > 1 ? p.dhidden.splits * p.rows * a.hidden * 4 : 0;
        const int64_t w = p.dweight.splits > 1 ? p.dweight.splits * a.vocab * a.hidden * 4 : 0;
        p.partial = take(std::max(h, w));
    }
    p.bytes = at;
    return p;
}

rf_status check(const rf_cross_entropy* a)
{
    if (!a) return report(RF_ERR_INVALID, "null arguments");
    if (a->tokens < 0 || a->tokens >= (1ll << 31) - 4096 || a->vocab < 1 || a->vocab > (1ll << 20) || a->hidden < 1 ||
        a->hidden > (1ll << 20))
        return report(RF_ERR_INVALID, "tokens, vocab or hidden out of range");
    if (!known(a->dtype)) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
    if (a->target_bits != 32 && a->target_bits != 64) return report(RF_ERR_UNSUPPORTED, "targets must be int32 or int64");
    if (a->reduction < RF_REDUCE_NONE || a->reduction > RF_REDUCE_MEAN) return report(RF_ERR_INVALID, "unknown reduction");
    if (!(a->z_loss >= 0.0f) || a->z_loss > 3e38f) return report(RF_ERR_INVALID, "z_loss must be finite and not negative");
    if (a->hidden_stride < 0 || a->weight_stride < 0) return report(RF_ERR_INVALID, "negative stride");
    return RF_OK;
}

template <auto K, typename... A> rf_status launch(int64_t grid, int threads, size_t lds, hipStream_t st, const A&... a)
{
    static std::atomic<uint64_t> done;
    if (grid <= 0) return RF_OK;
    if (grid > 0x7FFFFFFF) return report(RF_ERR_UNSUPPORTED, "too many workgroups for one launch");
    if (const rf_status s = allow_lds((const void*)K, lds, done); s != RF_OK) return s;
    K<<<(uint32_t)grid, threads, lds, st>>>(a...);
    return RF_OK;
}

template <typename H, typename E> rf_status logits(const Plan& p, const Logits& a, hipStream_t st)
{
    typedef Product<H, KALONG, KALONG, 256, 256, 2, 4> Big;
    typedef Product<H, KALONG, KALONG, 128, 128, 2, 2> Small;
    const int64_t tiles = (int64_t)a.tiles_p * a.tiles_q;
    return p.logits.big ? launch<k_logits<H, E, 256, 2, 4>>(tiles, Big::THREADS, Big::LDS, st, a)
                        : launch<k_logits<H, E, 128, 2, 2>>(tiles, Small::THREADS, Small::LDS, st, a);
}

template <typename H, Layout LQ> rf_status product(const Shape& shape, Grad& a, hipStream_t st)
{
    typedef Product<H, KDOWN, LQ, 256, 256, 2, 4> Big;
    typedef Product<H, KDOWN, LQ, 128, 128, 2, 2> Small;
    a.tiles_p = shape.tiles_p;
    a.tiles_q = shape.tiles_q;
    a.splits = (int32_t)shape.splits;
    const int64_t grid = (int64_t)a.tiles_p * a.tiles_q * a.splits;
    const rf_status s = shape.big ? launch<k_product<H, LQ, 256, 2, 4>>(grid, Big::THREADS, Big::LDS, st, a)
                                  : launch<k_product<H, LQ, 128, 2, 2>>(grid, Small::THREADS, Small::LDS, st, a);
    if (s != RF_OK || a.splits == 1) return s;
    return launch<k_join>((a.rows * ((a.cols + 3) / 4) + 255) / 256, 256, 0, st, a);
}

template <typename T, typename H> rf_status run(const rf_cross_entropy& a, const Plan& p, char* ws, hipStream_t st)
{
    const int planes = p.f32 ? 2 : 1;
    Scalars* const sc = (Scalars*)(ws + p.scalars);
    int32_t* const order = (int32_t*)(ws + p.order);
    int32_t* const target = (int32_t*)(ws + p.target);
    uint16_t* const hidden = (uint16_t*)(ws + p.hidden);
    const int64_t all = up(a.tokens, STEP), plane = all * p.pad;
    rf_status s = a.target_bits == 64
        ? launch<k_select<int64_t>>(1, SELECT, 0, st, (const int64_t*)a.targets, a.tokens, a.ignore_index, a.vocab, a.loss, order,
                                    target, sc, (int)p.pieces)
        : launch<k_select<int32_t>>(1, SELECT, 0, st, (const int32_t*)a.targets, a.tokens, a.ignore_index, a.vocab, a.loss, order,
                                    target, sc, (int)p.pieces);
    if (s != RF_OK) return s;
    const int32_t* const none = nullptr;
    if constexpr (sizeof(T) == 4) {
        s = launch<k_top>(std::min<int64_t>(a.tokens, 2048), 256, 0, st, (const float*)a.hidden_rows, a.tokens, a.hidden, a.hidden_stride,
                          (const int32_t*)order, (const Scalars*)sc, &sc->hidden_top);
        if (s != RF_OK) return s;
        s = launch<k_top>(std::min<int64_t>(a.vocab, 4096), 256, 0, st, (const float*)a.weight, a.vocab, a.hidden, a.weight_stride, none,
                          (const Scalars*)sc, &sc->weight_top);
        if (s != RF_OK) return s;
    }
    s = launch<k_pack<T>>(all, 256, 0, st, (const T*)a.hidden_rows, a.hidden, a.hidden_stride, p.pad, (const int32_t*)order,
                          (const Scalars*)sc, (const uint32_t*)&sc->hidden_top, hidden, hidden + plane, (T*)a.dhidden, a.tokens);
    if (s != RF_OK) return s;
    Side w{{a.weight, a.weight}, a.weight_stride * 2, a.vocab, a.vocab};
    if (p.own_weight) {
        uint16_t* const own = (uint16_t*)(ws + p.weight);
        s = launch<k_pack<T>>(a.vocab, 256, 0, st, (const T*)a.weight, a.hidden, a.weight_stride, p.pad, none, (const Scalars*)sc,
                              (const uint32_t*)&sc->weight_top, own, own + a.vocab * p.pad, (T*)nullptr, a.vocab);
        if (s != RF_OK) return s;
        w.base[0] = own;
        w.base[1] = own + (planes - 1) * a.vocab * p.pad;
        w.pitch = p.pad * 2;
    }
    for (int64_t piece = 0; piece < p.pieces; ++piece) {
        const int64_t first = piece * p.rows, rows = std::max<int64_t>(0, std::min(p.rows, a.tokens - first));
        const int64_t held = up(rows, STEP);
        uint16_t* const h = hidden + first * p.pad;
        Side x{{h, h + (planes - 1) * plane}, p.pad * 2, all - first, all - first};
        Logits l{};
        l.weight = w;
        l.hidden = x;
        l.vocab = a.vocab;
        l.pitch = p.vpad;
        l.first = first;
        l.rows = rows;
        l.steps = p.pad / STEP;
        l.pairs = p.pairs;
        l.blocks = p.blocks;
        l.sc = sc;
        l.target = target;
        l.stats = (float2*)(ws + p.stats);
        l.picked = (float*)(ws + p.picked);
        l.e = ws + p.e;
        l.tiles_p = p.logits.tiles_p;
        l.tiles_q = (uint32_t)((rows + (p.logits.big ? 255 : 127)) / (p.logits.big ? 256 : 128));
        if (!p.grad) s = logits<H, void>(p, l, st);
        else if (p.f32) s = logits<H, float>(p, l, st);
        else s = logits<H, f16>(p, l, st);
        if (s != RF_OK) return s;
        Rows r{};
        r.first = first;
        r.rows = rows;
        r.pitch = p.vpad;
        r.blocks = p.blocks;
        r.shift = p.shift;
        r.piece = (int32_t)piece;
        r.z_loss = a.z_loss;
        r.sc = sc;
        r.dz_top = sc->dz_top;
        r.order = order;
        r.target = target;
        r.stats = l.stats;
        r.picked = l.picked;
        r.dloss = a.dloss;
        r.loss = a.loss;
        r.reduction = a.reduction;
        if (p.grad) {
            r.top = (float*)(ws + p.top);
            r.factor = (float*)(ws + p.factor);
            r.at_target = (float*)(ws + p.at_target);
        }
        r.e = l.e;
        r.dz = ws + p.dz;
        r.dz_low = (uint16_t*)(ws + p.dz) + up(p.rows, STEP) * p.vpad;
        s = launch<k_rows>((rows + 3) / 4, 256, 0, st, r);
        if (s != RF_OK) return s;
        if (!p.grad) continue;
        s = launch<k_dlogits<H, std::conditional_t<sizeof(T) == 4, float, f16>>>(held, 256, (size_t)p.blocks * 4, st, r);
        if (s != RF_OK) return s;
        Grad g{};
        Side dz{{r.dz, p.f32 ? (const void*)r.dz_low : r.dz}, p.vpad * 2, held, held};
        g.sc = sc;
        g.dz_top = sc->dz_top;
        g.piece = (int32_t)piece;
        g.first = first;
        g.piece_rows = rows;
        g.pairs = p.pairs;
        g.dtype = a.dtype;
        g.cols = a.hidden;
        g.partial = (float*)(ws + p.partial);
        g.p = w;
        g.p.extent = p.pad;  // (its columns; as it is, hidden is a multiple of whole steps)
        g.q = dz;
        g.rows = rows;
        g.steps = p.vpad / STEP;
        g.order = order;
        g.out = a.dhidden;
        if (rows) {
            Shape shape = p.dhidden;
            shape.tiles_q = (uint32_t)((rows + (shape.big ? 255 : 127)) / (shape.big ? 256 : 128));
            s = product<H, KALONG>(shape, g, st);
            if (s != RF_OK) return s;
        }
        g.p = x;
        g.p.extent = p.pad;
        g.q.extent = p.vpad;
        g.rows = a.vocab;
        g.order = nullptr;
        g.out = a.dweight;
        g.sums = p.f32 ? (float*)a.dweight : (float*)(ws + p.sums);
        g.begin = piece == 0;
        g.end = piece + 1 == p.pieces;
        s = product<H, KDOWN>(p.dweight, g, st);
        if (s != RF_OK) return s;
    }
    if (a.reduction != RF_REDUCE_NONE)
        return launch<k_total>(1, SELECT, 0, st, (const float*)a.loss, (const int32_t*)order, (const Scalars*)sc, (int)a.reduction, a.total);
    return RF_OK;
}

}  // namespace

extern "C" {

rf_status rf_linear_cross_entropy_workspace(const rf_cross_entropy* args, int64_t* bytes)
{
    if (!bytes) return report(RF_ERR_INVALID, "null output");
    if (const rf_status s = check(args); s != RF_OK) return s;
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    *bytes = plan_of(*args, cus).bytes;
    return RF_OK;
}

rf_status rf_linear_cross_entropy(const rf_cross_entropy* args, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (const rf_status s = check(args); s != RF_OK) return s;
    const rf_cross_entropy& a = *args;
    if (!a.weight || (a.tokens && (!a.hidden_rows || !a.targets || !a.loss))) return report(RF_ERR_INVALID, "null buffer");
    if (a.reduction != RF_REDUCE_NONE && !a.total) return report(RF_ERR_INVALID, "a reduction needs total");
    if (a.reduction != RF_REDUCE_NONE && a.dloss) return report(RF_ERR_INVALID, "dloss and a reduction exclude each other");
    if (a.dloss || a.dhidden || a.dweight) {
        if (!a.dweight || (a.tokens && (!a.dhidden || (!a.dloss && a.reduction == RF_REDUCE_NONE))))
            return report(RF_ERR_INVALID, "gradients need dhidden, dweight and dloss or a reduction");
    }
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    const Plan p = plan_of(a, cus);
    if (p.bytes > workspace_bytes || !workspace) return report(RF_ERR_INVALID, "workspace too small");
    if ((uintptr_t)workspace & 255) return report(RF_ERR_INVALID, "workspace must be 256-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    rf_status s;
    if (a.dtype == RF_F32) s = run<float, f16>(a, p, (char*)workspace, st);
    else if (a.dtype == RF_F16) s = run<f16, f16>(a, p, (char*)workspace, st);
    else s = run<bf16, bf16>(a, p, (char*)workspace, st);
    if (s != RF_OK) return s;
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return rf::report_hip(e, "rf_linear_cross_entropy");
    return RF_OK;
}

}  // extern "C"
