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
//   LogitsJob  a product's tile of logits becomes, for each token and each block
//              of the vocabulary (a wave's part of the tile: 64 or 128 entries), a
//              maximum m and a sum s of exp(z - m); for gradients exp(z - m) itself
//              too, in f16 (f32 tensors: in f32)
//   k_rows     lse and loss from m and s, factors of the gradient
//   k_dlogits  exp(z - m) to dz, in place (f32: to two f16 planes; where few tokens
//              count to two planes of the tensors' type)
//   GradJob    dhidden and dweight, two products of the same size
//   k_level    between them, for tokens that weigh little beside others: hidden's rows
// Loss alone ends with k_rows and writes no logits.  With gradients a piece of
// tokens at a time holds at most PIECE bytes of exponentials; the pieces'
// weight gradients are added in f32.  Three products, none computed twice.
//
// exp(z - m) is in [0, 1]: f16 rounds it by at most 2^-11 of its value (below
// 2^-14 by 2^-25, so that what is below 2^-25 of the largest of its block is lost), an
// eighth of what bf16's rounding of dz adds, and as much as f16's.  At the target
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
// Where so few 16-bit tokens count, dz goes to its products in two parts, high and low:
// with few terms its rounding does not average out (bf16, 1 x 896 x 225: gradients off by
// up to 2.8e-3 of their norm, so 1.7e-3, the rounding of the result; 16 tokens: 2.1e-3).
// f16, 16 x 4000 x 96: off by 2.0e-4 where one part leaves 2.5e-4; beside the targets, where
// the exponential is rounded to f16 as well, 1.4 and 1.7 of the result's rounding.  For all of 67 f16 tokens with 32000 x 4096 it would take 327 us in place of 261.
constexpr int64_t FEW = 16;
static_assert(FEW <= STEP, "the low parts are one step of tokens");

// Written by the kernels, read by later ones.
struct Scalars {
    int32_t count, pad[3];
    uint32_t hidden_top, weight_top;  // f32: bits of the largest finite magnitudes
    uint32_t pad2[2];
};

// Of each piece of tokens: its products' shares, which depend on how many tokens count,
// and bits of the largest row factor.  (Lifted: k_dlogits.)
struct Piece {
    Share logits, dhidden, dweight;
    uint32_t dz_top;
    int32_t pairs;   // plane pairs of the gradients' products
    uint32_t uneven; // some token's dz was lifted
    uint32_t hidden_top, pad;  // f16, then: bits of the largest finite magnitude of the piece's rows of hidden
};

// The products of a piece, for k_select.  The last three: no tile is split, and nothing is
// launched that would settle one.
struct Products {
    int64_t rows, vocab, hidden, logits_steps, dhidden_steps;
    int32_t pieces, pairs, grad, few, cus;  // few: dz may go in two parts
    int32_t logits_tile, dhidden_tile, dweight_tile;
    int32_t logits_whole, dhidden_whole, dweight_whole;
};

// What dhidden's way through weight is counted as, whose rows it reads in pieces as wide as
// its tiles: 128 bytes at a time come at three quarters of the rate (34 tokens, 32000 x
// 4096: tiles of 64 97 us, of 128 74).
__host__ __device__ inline int64_t way_down(int64_t bytes, int tile) { return tile > 64 ? bytes : bytes / 3 * 4; }

// By a whole wave.
__device__ __forceinline__ Piece piece_of(const Products& p, int64_t count, int64_t piece)
{
    const int64_t rows = max(min(count - piece * p.rows, p.rows), (int64_t)0), steps = (rows + STEP - 1) / STEP;
    auto tiles = [](int64_t x, int64_t y, int tile) { return (uint32_t)(((x + tile - 1) / tile) * ((y + tile - 1) / tile)); };
    // each product reads weight, or writes a gradient as large
    const int64_t bytes = p.vocab * p.hidden * (p.pairs > 1 ? 4 : 2);
    auto share = [&](int64_t x, int64_t y, int64_t n, int tile, int pairs, int64_t bytes, bool whole) {
        if (whole) return Share{tiles(x, y, tile), 0, 1};
        return share_by_wave(tiles(x, y, tile), n, room_of(tile, p.cus), cost_of(tile, pairs, 0, bytes));
    };
    Piece out{};
    out.logits = share(p.vocab, rows, p.logits_steps, p.logits_tile, p.pairs, bytes, p.logits_whole);
    if (!p.grad) return out;
    out.pairs = p.few && count <= FEW ? 2 : p.pairs;
    out.dhidden = share(p.hidden, rows, p.dhidden_steps, p.dhidden_tile, out.pairs, way_down(bytes, p.dhidden_tile), p.dhidden_whole);
    // without tokens there is nothing to add, but what the pieces have summed is to be
    // written by the first and rounded by the last
    if (steps) out.dweight = share(p.hidden, p.vocab, steps, p.dweight_tile, out.pairs, bytes, p.dweight_whole);
    else if (piece == 0 || piece + 1 == p.pieces) out.dweight = {tiles(p.hidden, p.vocab, p.dweight_tile), 0, 1};
    return out;
}

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
// row of weight.  One workgroup: one token takes 5 us, 16384 take 23.
template <typename I>
__global__ __launch_bounds__(SELECT) void k_select(const I* __restrict__ targets, int64_t tokens, int64_t ignore, int64_t vocab,
                                                  float* __restrict__ loss, int32_t* __restrict__ order,
                                                  int32_t* __restrict__ target, Scalars* sc, Piece* pieces, Products products)
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
    for (int i = wave; i < products.pieces; i += SELECT / WAVE) {
        const Piece piece = piece_of(products, before, i);
        if (lane == 0) pieces[i] = piece;
    }
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
    __shared__ uint32_t tops[4];
    if (threadIdx.x % WAVE == 0) tops[threadIdx.x / WAVE] = best;
    __syncthreads();
    if (threadIdx.x == 0) raise(top, max(max(tops[0], tops[1]), max(tops[2], tops[3])));
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
// zeros in the rows of `clear` that do not count.  `tops` (f16): bits of the largest
// finite magnitude that each of a row's four waves has seen.
template <typename T>
__global__ __launch_bounds__(256) void k_pack(const T* __restrict__ x, int64_t cols, int64_t stride, int64_t pitch,
                                             const int32_t* __restrict__ order, const Scalars* sc, const uint32_t* top,
                                             uint16_t* __restrict__ hi, uint16_t* __restrict__ lo, void* __restrict__ clear,
                                             int wide, uint32_t* __restrict__ tops, int64_t rows)
{
    const int64_t r = blockIdx.x;
    int64_t from = r;
    bool zero = false;
    if (order) {
        const int64_t count = sc->count;
        zero = r >= count;
        if (r < rows) from = order[r];
        if (zero && r < rows && clear)
            for (int64_t c = (int64_t)threadIdx.x * 8; c < cols; c += 2048) {
                if (wide) put8((float*)clear + from * cols + c, Raw<float>{}, cols - c);
                else put8((T*)clear + from * cols + c, Raw<T>{}, cols - c);
            }
        if (r >= (count + STEP - 1) / STEP * STEP) return;
    }
    const T* const row = x + from * stride;
    float scale = 1.0f;
    if constexpr (sizeof(T) == 4) scale = scale_of(*top);
    uint32_t best = 0;
    for (int64_t c = (int64_t)threadIdx.x * 8; c < pitch; c += 2048) {
        Raw<T> v{};
        if (!zero && c < cols) v = load8(row, c, cols);
        if (sizeof(T) == 2 && tops) {
            float w[8];
            widen8(v, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t x = __float_as_uint(w[k]) & 0x7FFFFFFFu;
                best = max(best, x < 0x7F800000u ? x : 0u);
            }
        }
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
    if (sizeof(T) == 4 || !tops) return;
    for (int d = 1; d < WAVE; d *= 2) best = max(best, (uint32_t)__shfl_xor((int)best, d));
    if (threadIdx.x % WAVE == 0) tops[r * 4 + threadIdx.x / WAVE] = best;
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
    uint32_t tiles_p, room;
    float* partial;
    const Piece* piece;
};

// Tiles of equal steps in bands (tile_at), of which a packed piece of tokens has as
// many as there are tokens that count.
struct Even {
    int64_t p0, q0, steps;
};

// Measured: 8192 x 50257 x 768 without exponentials 570 to 620 us (1.0 to 1.1 PFLOP/s),
// with them 780 to 820, 824 MB written where the next tile's products could run; 16384 x 32000 x 4096
// 3170 us, 1.22 PFLOP/s.  A token alone is bound by weight's way from memory: 1 x 32000 x
// 4096 41 us, where part of it lies in the last-level cache, else 90 for 33 tokens (2.9
// TB/s: two steps of weight in flight a workgroup).
template <typename H, typename E, int TILE, int WP, int WQ> struct LogitsJob {
    typedef Logits Args;
    typedef Even Tile;
    typedef Product<H, KALONG, KALONG, TILE, TILE, WP, WQ> G;
    static constexpr int LDS = G::LDS;
    // The argument in registers: read where it lies it takes scalar ones past their end
    // here (8192 x 50257 x 768 with exponentials 741 us, so 857), while the gradients'
    // kernels need it there.
    static constexpr bool FEW_SCALARS = true;

    static __device__ int64_t count(const Logits& a) { return max(min((int64_t)a.sc->count - a.first, a.rows), (int64_t)0); }
    static __device__ uint32_t tiles_q(const Logits& a) { return (uint32_t)((count(a) + TILE - 1) / TILE); }
    static __device__ Share share(const Logits& a) { return a.piece->logits; }
    static __device__ Even tile(const Logits& a, uint32_t id)
    {
        const TileAt t = tile_at(id, a.tiles_p, tiles_q(a));
        return {(int64_t)t.p * TILE, (int64_t)t.q * TILE, a.steps};
    }
    static __device__ __forceinline__ void run(const Logits& a, const Even& t, char* lds, int64_t s0, int64_t s1, typename G::Sums& acc)
    {
        G::run(lds, a.weight, a.hidden, t.p0, t.q0, s0, s1, a.pairs, acc);
    }
    static __device__ __forceinline__ void finish(const Logits& a, const Even& t, typename G::Sums& acc, int wave, char*);
};

// E: what is kept of the exponentials: nothing, f16 or f32.
template <typename H, typename E, int TILE, int WP, int WQ>
__device__ __forceinline__ void LogitsJob<H, E, TILE, WP, WQ>::finish(const Logits& a, const Even& t, typename G::Sums& acc, int wave, char*)
{
    const int64_t count = LogitsJob::count(a), p0 = t.p0, q0 = t.q0;
    const int wp = G::wp(wave), wq = G::wq(wave);
    const int lane = own_lane();
    float unscale = 1.0f;
    if (a.pairs > 1) unscale = inverse(scale_of(a.sc->hidden_top)) * inverse(scale_of(a.sc->weight_top));
    const int64_t v0 = p0 + wp + lane / 16 * 4;
    if (a.pairs > 1) {
#pragma unroll
        for (int j = 0; j < G::FQ; ++j)
#pragma unroll
            for (int i = 0; i < G::FP; ++i) acc[i][j] *= unscale;
    }
    if (p0 + wp + TILE / WP > a.vocab) {
#pragma unroll
        for (int j = 0; j < G::FQ; ++j) {
            int left = (int)max(min(a.vocab - v0, (int64_t)TILE), (int64_t)0);
            asm volatile("" : "+v"(left));  // (no masks of 32 comparisons to be kept from one j to the next)
#pragma unroll
            for (int i = 0; i < G::FP; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * i + r >= left) acc[i][j][r] = -__builtin_inff();
        }
    }
    constexpr float LOG2E = 1.44269504088896341f;
    int32_t target[G::FQ];  // loaded together
#pragma unroll
    for (int j = 0; j < G::FQ; ++j) target[j] = a.target[a.first + min(q0 + wq + 16 * j + lane % 16, count - 1)];
#pragma unroll
    for (int j = 0; j < G::FQ; ++j) {
        const int64_t q = q0 + wq + 16 * j + lane % 16;
        const bool mine = q < count;
        const int64_t y = mine ? target[j] - v0 : -1;
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
        // the difference first: it is exact where it matters, and zero at the maximum, so that
        // s is at least one and no loss below zero (2^(z log2(e) - m log2(e)) in one FMA carries
        // the rounding of m log2(e), 2e-5 in the loss at logits of 400).  Where nothing is here,
        // exponentials of -inf are 0
        const float top = m == -__builtin_inff() ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < G::FP; i += 2) {
            f32x4 e[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    e[k][r] = __builtin_amdgcn_exp2f((acc[i + k][j][r] - top) * LOG2E);
                    s += e[k][r];
                }
            if constexpr (__is_same(E, f16)) {
                const u32x4 c = chunk(narrow4<f16>(e[0]), narrow4<f16>(e[1]));
                const int64_t v = p0 + wp + 16 * i + chunk_of(lane);
                if (mine && v < a.pitch) *(u32x4*)((f16*)a.e + q * a.pitch + v) = c;
            } else if constexpr (__is_same(E, float)) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (mine && v0 + 16 * (i + k) < a.pitch) *(f32x4*)((float*)a.e + q * a.pitch + v0 + 16 * (i + k)) = e[k];
            }
        }
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (mine) {
            const int64_t block = (p0 + wp) / (TILE / WP);
            if (lane < 16 && block < a.blocks) a.stats[q * a.blocks + block] = make_float2(m, s);
        }
    }
}

template <typename J> __global__ __launch_bounds__(J::G::THREADS, 2) void k_multiply(const typename J::Args a)
{
    extern __shared__ char lds[];
    if constexpr (J::FEW_SCALARS) multiply_tiles<J>(a, lds);
    else multiply_tiles<J>(argument<typename J::Args>(), lds);
}

template <typename J> __global__ __launch_bounds__(WAVE, 2) void k_settle(const typename J::Args a)
{
    if constexpr (J::FEW_SCALARS) settle_tiles<J>(a, nullptr);
    else settle_tiles<J>(argument<typename J::Args>(), nullptr);
}

struct Rows {
    int64_t first, rows, pitch;
    int32_t blocks, shift;  // entries of a block: 1 << shift
    int32_t reduction;
    float z_loss;
    const Scalars* sc;
    Piece* piece;
    const int32_t *order, *target;
    const float2* stats;
    const float *picked, *dloss;
    float *loss, *top, *factor, *at_target;  // [rows] each but loss
    float* reach;        // [rows] row factors' magnitudes; NULL: bf16, which has the range
    int32_t* lifts;      // [rows] powers of two that dz was lifted by
    const void* e;
    void* dz;
    uint16_t* dz_low;
};

// A wave a token at a time.  A workgroup's waves raise the largest factor once, so
// that few atomics meet.
__global__ __launch_bounds__(256) void k_rows(const Rows a)
{
    const int64_t count = min((int64_t)a.sc->count - a.first, a.rows);
    const int lane = threadIdx.x % WAVE;
    uint32_t most = 0;
    for (int64_t q = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE; q < count; q += (int64_t)gridDim.x * 4) {
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
        if (lane) continue;
        const int32_t t = a.order[a.first + q];
        const bool known = a.target[a.first + q] >= 0;
        const float logs = logf(s), lse = m + logs, nan = __builtin_nanf("");
        const float below = known ? a.picked[q] - m - logs : nan;  // the target's log probability
        a.loss[t] = a.z_loss * lse * lse - below;
        if (!a.factor) continue;
        float dl = a.dloss ? a.dloss[t] : a.reduction == RF_REDUCE_MEAN ? 1.0f / (float)a.sc->count : 1.0f;
        if (!known) dl = nan;
        const float spread = 1.0f + 2.0f * a.z_loss * lse;
        a.top[q] = m;
        a.factor[q] = dl * spread / s;
        a.at_target[q] = dl * (expm1f(below) + (spread - 1.0f) * expf(below));
        const float reach = fmaxf(fabsf(dl * spread), fabsf(dl));
        if (a.reach) a.reach[q] = reach;
        const uint32_t mine = __float_as_uint(reach);
        if (mine < 0x7F800000u) most = max(most, mine);
    }
    if (!a.factor) return;
    __shared__ uint32_t tops[4];
    if (lane == 0) tops[threadIdx.x / WAVE] = most;
    __syncthreads();
    if (threadIdx.x == 0) raise(&a.piece->dz_top, max(max(tops[0], tops[1]), max(tops[2], tops[3])));
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
    return t < 0x1p-110f ? 1.0f : (wide ? 1.0f : 16384.0f) / t;
}

// In f16, which keeps 2^-38 of the largest, a token whose own factor has an exponent of 5
// or more below its is lifted by a power of two to where the largest are: its dhidden keeps
// the bits of any other's (dloss 1e-8 of another's: off by 1.5e-2 of its norm without it),
// whose product takes the power away again; dweight's sums find it in the token's row of
// hidden (k_level).  Five, so that the factors of a z-loss alone move nothing.  As far as
// the scale is finite.
__device__ __forceinline__ int lift_of(uint32_t top, float reach)
{
    const int d = min((int)(top >> 23) - (int)(__float_as_uint(reach) >> 23), (int)(top >> 23) - 17);
    return d > 4 ? d : 0;
}

// dz of a token from its exponentials; zeros up to a whole step of
// tokens.  A workgroup a token.  P: dz's type; E: the exponentials'.  Bound by memory:
// 8192 x 50257 read and written in place, past the caches, which keep weight instead, 321
// us, 5.1 TB/s.
template <typename P, typename E> __global__ __launch_bounds__(256) void k_dlogits(const Rows a)
{
    extern __shared__ float of_block[];
    const int64_t q = blockIdx.x, count = min((int64_t)a.sc->count - a.first, a.rows);
    if (q >= (count + STEP - 1) / STEP * STEP) return;
    P* const out = (P*)a.dz + q * a.pitch;
    uint16_t* const low = a.piece->pairs > 1 ? a.dz_low : nullptr;
    if (q >= count) {
        for (int64_t v = (int64_t)threadIdx.x * 8; v < a.pitch; v += 2048) {
            *(u32x4*)(out + v) = u32x4{};
            if (low) *(u32x4*)(low + q * a.pitch + v) = u32x4{};
        }
        return;
    }
    float scale = dz_scale(a.piece->dz_top, __is_same(P, bf16));
    if (a.reach) {
        const int lift = lift_of(a.piece->dz_top, a.reach[q]);
        scale = ldexpf(scale, lift);
        if (threadIdx.x == 0) {
            a.lifts[q] = lift;
            if (lift) raise(&a.piece->uneven, 1);
        }
    }
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
        raw.a = __builtin_nontemporal_load((const u32x4*)(in + v));
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
            *(u32x4*)(low + q * a.pitch + v) = l.a;
        } else {
            const Raw<P> h = narrow8<P>(x);
            __builtin_nontemporal_store(h.a, (u32x4*)(out + v));
            if (low) {
                float back[8];
                widen8(h, back);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] -= back[k];
                *(u32x4*)(low + q * a.pitch + v) = narrow8<P>(x).a;
            }
        }
    }
}

// Where a token of the piece was lifted: hidden's packed rows once more, for dweight, each
// divided by what its dz was multiplied by.  f16 rows are brought up to the top of the
// range first, that less falls below it.
template <typename T>
__global__ __launch_bounds__(256) void k_level(const T* __restrict__ x, int64_t cols, int64_t stride, int64_t pitch,
                                              const int32_t* __restrict__ order, int64_t first, int64_t most, const Scalars* sc,
                                              Piece* piece, const int32_t* __restrict__ lifts, const uint32_t* __restrict__ tops,
                                              uint16_t* __restrict__ hi, uint16_t* __restrict__ lo)
{
    if (!piece->uneven) return;
    const int64_t rows = min((int64_t)sc->count - first, most);
    uint32_t top = sc->hidden_top;
    if (sizeof(T) == 2) {  // every workgroup for itself: k_pack's waves have 12 ns each for an atomic
        __shared__ uint32_t of_wave[4];
        top = 0;
        for (int64_t i = first * 4 + threadIdx.x; i < (first + rows) * 4; i += 256) top = max(top, tops[i]);
        for (int d = 1; d < WAVE; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        if (threadIdx.x % WAVE == 0) of_wave[threadIdx.x / WAVE] = top;
        __syncthreads();
        top = max(max(of_wave[0], of_wave[1]), max(of_wave[2], of_wave[3]));
        if (blockIdx.x == 0 && threadIdx.x == 0) piece->hidden_top = top;
    }
    const float scale = scale_of(top);
    for (int64_t q = blockIdx.x; q < rows; q += gridDim.x) {
        const T* const row = x + order[first + q] * stride;
        const int lift = lifts[q];
        for (int64_t c = (int64_t)threadIdx.x * 8; c < cols; c += 2048) {  // (zeros stay behind them)
            float v[8];
            widen8(load8(row, c, cols), v);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k] * scale, -lift);
            Raw<f16> h, l;
            split8(v, 1.0f, h, l);
            *(u32x4*)(hi + q * pitch + c) = h.a;
            if (sizeof(T) == 4) *(u32x4*)(lo + q * pitch + c) = l.a;
        }
    }
}

// ---------------------------------------------------------- the gradients ---
struct Grad {
    Side p, q;
    int64_t cols, rows;            // of the output: p below cols, q below rows
    int64_t first, piece_rows;     // packed tokens of this piece
    int64_t steps;                 // of the sum; 0: the tokens that count
    int32_t pairs, dtype;          // pairs: as hidden and weight have them; dtype: of the output
    const Scalars* sc;
    const Piece* piece;
    const int32_t* order;          // dhidden: the output's row of packed token q; NULL: dweight
    const int32_t* lifts;          // of the piece's tokens; NULL: none is lifted
    void* out;
    float* sums;                   // dweight, several pieces: f32 sums so far (may be out)
    int32_t begin, end;            // the first piece, the last one
    uint32_t tiles_p, room;
    float* partial;
};

__device__ __forceinline__ float unscale_of(const Grad& a, bool wide)
{
    float u = 1.0f / dz_scale(a.piece->dz_top, wide);
    if (a.pairs > 1) u *= inverse(scale_of(a.order ? a.sc->weight_top : a.sc->hidden_top));
    else if (!a.order && a.lifts && a.piece->uneven) u *= inverse(scale_of(a.piece->hidden_top));
    return u;
}

// What becomes of neighbouring sums of an output's row: unscaled, added to the
// pieces' before, and rounded, or kept for the pieces behind.
struct Finish {
    void* out;
    float* sums;       // NULL: nothing before and nothing behind
    const int32_t *order, *lifts;
    int64_t cols;
    float unscale;
    bool add, keep;
    int32_t dtype;

    __device__ __forceinline__ Finish(const Grad& a, bool wide)
        : out(a.out), sums(!a.order && !(a.begin && a.end) ? a.sums : nullptr), order(a.order ? a.order + a.first : nullptr),
          lifts(a.order && a.lifts && a.piece->uneven ? a.lifts : nullptr), cols(a.cols), unscale(unscale_of(a, wide)), add(sums && !a.begin), keep(sums && !a.end), dtype(a.dtype)
    {
    }
    // four of row q from p on, in f32 or element by element
    __device__ __forceinline__ void put4(int64_t q, int64_t p, f32x4 v) const
    {
        v *= unscale;
        if (lifts)
            for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], -lifts[q]);
        const int64_t left = cols - p, here = q * cols + p, at = (order ? order[q] : q) * cols + p;
        if (add) {
            if (left >= 4) v += __builtin_bit_cast(f32x4, *(const u32x4_at*)(sums + here));
            else
                for (int r = 0; r < 3; ++r)
                    if (r < left) v[r] += sums[here + r];
        }
        if (left >= 4 && (keep || dtype == RF_F32)) *(u32x4_at*)((float*)(keep ? sums : out) + at) = __builtin_bit_cast(u32x4, v);
        else
            for (int r = 0; r < 4; ++r)
                if (r < left) put_scalar(keep ? sums : out, keep ? (int)RF_F32 : dtype, at + r, v[r]);
    }
    // the usual case: 16 bits, nothing before and nothing behind
    __device__ __forceinline__ bool plain() const { return !sums && dtype != RF_F32; }
};

// dhidden: p the hidden columns of weight (summed down its rows), q the tokens of dz.
// dweight: p the hidden columns of the packed rows, q the vocabulary, both summed over tokens.
// Measured: 14746 x 32000 x 4096 2.99 and 3.10 ms (1.29 and 1.25 PFLOP/s), 6001 x 131101 x
// 2048 2.48 and 2.64 (1.30, 1.22), 8192 x 50257 x 768 571 and 543 us (1.11, 1.16), and 39 and
// 22 us to settle split tiles.
template <typename H, Layout LQ, int TILE, int WP, int WQ> struct GradJob {
    typedef Grad Args;
    typedef Even Tile;
    typedef Product<H, KDOWN, LQ, TILE, TILE, WP, WQ, LQ == KALONG> G;
    static constexpr int LDS = G::LDS;
    static constexpr bool FEW_SCALARS = false;

    static __device__ int64_t count(const Grad& a) { return max(min((int64_t)a.sc->count - a.first, a.piece_rows), (int64_t)0); }
    static __device__ int64_t rows(const Grad& a) { return LQ == KALONG ? count(a) : a.rows; }
    static __device__ int64_t steps(const Grad& a) { return LQ == KALONG ? a.steps : (count(a) + STEP - 1) / STEP; }
    static __device__ uint32_t tiles_q(const Grad& a) { return (uint32_t)((rows(a) + TILE - 1) / TILE); }
    static __device__ Share share(const Grad& a) { return LQ == KALONG ? a.piece->dhidden : a.piece->dweight; }
    static __device__ Even tile(const Grad& a, uint32_t id)
    {
        const TileAt t = tile_at(id, a.tiles_p, tiles_q(a));
        return {(int64_t)t.p * TILE, (int64_t)t.q * TILE, steps(a)};
    }
    static __device__ __forceinline__ void run(const Grad& a, const Even& t, char* lds, int64_t s0, int64_t s1, typename G::Sums& acc)
    {
        G::run(lds, a.p, a.q, t.p0, t.q0, s0, s1, a.piece->pairs, acc);
    }
    static __device__ __forceinline__ void finish(const Grad& a, const Even& t, typename G::Sums& acc, int wave, char*)
    {
        const int64_t rows = GradJob::rows(a);
        const Finish f(a, __is_same(H, bf16));
        const int lane = own_lane();
        const int64_t p0 = t.p0 + G::wp(wave);
#pragma unroll
        for (int j = 0; j < G::FQ; ++j) {
            const int64_t q = t.q0 + G::wq(wave) + 16 * j + lane % 16;
            if (f.plain()) {
                uint16_t* const row = (uint16_t*)f.out + (f.order ? f.order[min(q, rows - 1)] : q) * f.cols;
                const float unscale = f.lifts ? ldexpf(f.unscale, -f.lifts[min(q, rows - 1)]) : f.unscale;
#pragma unroll
                for (int i = 0; i < G::FP; i += 2) {
                    const f32x4 x = acc[i][j] * unscale, y = acc[i + 1][j] * unscale;
                    const u32x4 c = __is_same(H, bf16) ? chunk(narrow4<bf16>(x), narrow4<bf16>(y)) : chunk(narrow4<f16>(x), narrow4<f16>(y));
                    const int64_t from = p0 + 16 * i + chunk_of(lane);
                    if (q < rows && from < f.cols) put8<true, LQ == KDOWN>(row + from, Raw<uint16_t>{c}, f.cols - from);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < G::FP; ++i) {
                    const int64_t p = p0 + 16 * i + lane / 16 * 4;
                    if (q < rows && p < f.cols) f.put4(q, p, acc[i][j]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
};

// ------------------------------------------------------------------- host ---
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Tile of a product: the one that takes least by the measured costs in rf_product.h.
// Logits of 1 x 32000 x 4096: tiles of 64 40 us, of 128 53; both gradients of 6001 x
// 131101 x 2048: tiles of 256, dhidden's 192 in four parts, 2.5 ms, tiles of 128 3.4.
struct Shape {
    int tile;
    uint32_t tiles_p, room;
};

Shape shape_of(int64_t cols, int64_t rows, int64_t steps, int pairs, int64_t bytes, int cus, bool down = false)
{
    int tile = 0;
    double least = 0;
    for (const int of : {64, 128, 256}) {
        const int64_t tiles = ((cols + of - 1) / of) * ((rows + of - 1) / of);
        const uint32_t room = room_of(of, cus);
        const Cost c = cost_of(of, pairs, 0, down ? way_down(bytes, of) : bytes);
        const double ns = ns_of(share_of((uint32_t)std::min<int64_t>(tiles, 1u << 30), steps, room, c), steps, room, c);
        if (!tile || ns < least) {
            tile = of;
            least = ns;
        }
    }
    return {tile, (uint32_t)((cols + tile - 1) / tile), room_of(tile, cus)};
}

// Bytes of the parts of split tiles: of `tiles` at most, with sums of `steps`.
int64_t parts_of(const Shape& s, int64_t tiles, int64_t steps)
{
    const int64_t most = std::min<int64_t>({(int64_t)s.room * PARTS_ROOM, tiles * MOST_PARTS, tiles * std::max<int64_t>(1, steps / 2)});
    return most * s.tile * s.tile * 4;
}

struct Plan {
    int64_t pad, vpad, rows, pieces;  // hidden and vocab padded, tokens of a piece, pieces
    bool own_weight, f32, grad, few, wide;  // wide: gradients in f32
    bool lifts;  // tokens' dz may be lifted
    int32_t blocks, shift, pairs, cus;
    Shape logits, dhidden, dweight;
    bool logits_whole, dhidden_whole, dweight_whole;  // never split: k_select is told, and nothing launched that settles
    // offsets in the workspace
    int64_t scalars, piece, order, target, stats, picked, top, factor, at_target, reach, lift, tops, hidden, weight, e, dz, low, sums, partial, bytes;
};

bool known(int32_t dtype) { return dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16; }

int32_t reduction_of(const rf_cross_entropy& a) { return a.reduction & ~RF_GRADS_F32; }

// Whether no number of tokens that count splits a tile, where that is soon found: a
// launch with nothing to settle takes 4.5 us.
bool never_splits(const Shape& shape, const Plan& p, int64_t bytes, bool few, int64_t tiles_q, int64_t steps)
{
    if (steps < 4) return true;  // (no part of fewer than two)
    if (tiles_q > 4) return false;
    for (int pairs = p.pairs; pairs <= (few ? 2 : p.pairs); ++pairs) {
        const Cost c = cost_of(shape.tile, pairs, 0, bytes);
        for (int64_t q = 1; q <= (pairs > p.pairs ? 1 : tiles_q); ++q)  // (two pairs: of at most FEW tokens)
            if (share_of((uint32_t)(shape.tiles_p * q), steps, shape.room, c).rest) return false;
    }
    return true;
}

Plan plan_of(const rf_cross_entropy& a, int cus)
{
    Plan p{};
    p.cus = cus;
    p.f32 = a.dtype == RF_F32;
    p.grad = a.dweight != nullptr;
    p.wide = p.f32 || (a.reduction & RF_GRADS_F32);
    p.pairs = p.f32 ? 3 : 1;
    // row factors of a reduction without a z-loss are all alike
    p.lifts = p.grad && a.dtype != RF_BF16 && (reduction_of(a) == RF_REDUCE_NONE || a.z_loss > 0.0f);
    p.few = p.grad && !p.f32;
    p.pad = up(a.hidden, STEP);
    p.vpad = up(a.vocab, STEP);
    // weight as it is: whole steps of k, 16-byte rows
    p.own_weight = p.f32 || a.hidden % STEP || a.weight_stride % 8 || ((uintptr_t)a.weight & 15) || a.weight_stride * 2 >= (1 << 24);
    const int64_t planes = p.f32 ? 2 : 1, steps = p.pad / STEP;
    const int64_t bytes = a.vocab * a.hidden * (p.f32 ? 4 : 2);
    p.logits = shape_of(a.vocab, a.tokens, steps, p.pairs, bytes, cus);
    p.shift = p.logits.tile > 128 ? 7 : 6;
    p.blocks = (int32_t)((a.vocab + (1 << p.shift) - 1) >> p.shift);
    const int64_t each = p.grad ? p.vpad * (p.f32 ? 8 : 2) : p.blocks * 8, most = p.grad ? PIECE : STATS;
    // pieces of equal numbers of whole tiles
    const int64_t fit = std::max<int64_t>(64, most / each / 256 * 256);
    p.pieces = std::max<int64_t>(1, (a.tokens + fit - 1) / fit);
    p.rows = p.pieces == 1 ? std::max<int64_t>(1, a.tokens) : std::min(fit, up((a.tokens + p.pieces - 1) / p.pieces, 256));
    p.pieces = std::max<int64_t>(1, (a.tokens + p.rows - 1) / p.rows);
    p.logits = shape_of(a.vocab, p.rows, steps, p.pairs, bytes, cus);
    p.shift = p.logits.tile > 128 ? 7 : 6;
    p.blocks = (int32_t)((a.vocab + (1 << p.shift) - 1) >> p.shift);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t from = at;
        at += up(bytes, 256);
        return from;
    };
    const int64_t held = up(p.rows, STEP);
    p.scalars = take(sizeof(Scalars));
    p.piece = take(sizeof(Piece) * p.pieces);
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
        p.reach = take(p.rows * 4);
        p.lift = take(p.rows * 4);
        if (p.lifts && !p.f32) p.tops = take(up(a.tokens, STEP) * 16);
        // Low parts of few tokens: one step of rows.  A tile of dhidden reads as many rows of
        // them as of the high ones, up to `held`, for tokens that do not exist: those behind the
        // step are the first of e, which lies next to it (both are multiples of 256 bytes).
        if (p.few) p.low = take(STEP * p.vpad * 2);
        p.e = take(held * p.vpad * (p.f32 ? 4 : 2));
        p.dz = p.f32 ? take(held * p.vpad * 4) : p.e;
        if (p.pieces > 1 && !p.wide) p.sums = take(a.vocab * a.hidden * 4);
        p.dhidden = shape_of(a.hidden, p.rows, p.vpad / STEP, p.pairs, bytes, cus, true);
        p.dweight = shape_of(a.hidden, a.vocab, held / STEP, p.pairs, bytes, cus);
    }
    auto down = [&](const Shape& s) { return (p.rows + s.tile - 1) / s.tile; };
    p.logits_whole = never_splits(p.logits, p, bytes, false, down(p.logits), steps);
    if (p.grad) {  // dhidden: the sums' steps are known, of dweight the tiles
        p.dhidden_whole = never_splits(p.dhidden, p, way_down(bytes, p.dhidden.tile), p.few, down(p.dhidden), p.vpad / STEP);
        p.dweight_whole = held / STEP < 4;
    }
    auto tiles = [](const Shape& s, int64_t rows) { return (int64_t)s.tiles_p * ((rows + s.tile - 1) / s.tile); };
    int64_t parts = parts_of(p.logits, tiles(p.logits, p.rows), steps);
    if (p.grad)
        parts = std::max({parts, parts_of(p.dhidden, tiles(p.dhidden, p.rows), p.vpad / STEP), parts_of(p.dweight, tiles(p.dweight, a.vocab), held / STEP)});
    p.partial = take(parts);
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
    if (reduction_of(*a) < RF_REDUCE_NONE || reduction_of(*a) > RF_REDUCE_MEAN) return report(RF_ERR_INVALID, "unknown reduction");
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

// A product's launch, and the one that settles split tiles (which of them are is known on
// the device alone).
template <typename J> rf_status multiply(const Shape& shape, int64_t tiles, const typename J::Args& a, hipStream_t st, bool never_split = false)
{
    const rf_status s = launch<k_multiply<J>>(tiles + (never_split ? 0 : PARTS_ROOM * shape.room), J::G::THREADS, J::LDS, st, a);
    if (s != RF_OK || never_split) return s;
    return launch<k_settle<J>>((int64_t)std::min<int64_t>(tiles, shape.room) * J::G::WAVES, WAVE, 0, st, a);
}

int64_t tiles_of(const Shape& shape, int64_t rows) { return (int64_t)shape.tiles_p * ((rows + shape.tile - 1) / shape.tile); }

template <typename H, typename E> rf_status logits(const Plan& p, const Logits& a, hipStream_t st)
{
    const int64_t tiles = tiles_of(p.logits, a.rows);
    const bool whole = p.logits_whole;
    return p.logits.tile > 128  ? multiply<LogitsJob<H, E, 256, 2, 4>>(p.logits, tiles, a, st, whole)
           : p.logits.tile > 64 ? multiply<LogitsJob<H, E, 128, 2, 2>>(p.logits, tiles, a, st, whole)
                                : multiply<LogitsJob<H, E, 64, 1, 4>>(p.logits, tiles, a, st, whole);
}

template <typename H, Layout LQ> rf_status product(const Plan& p, const Shape& shape, float* partial, Grad& a, hipStream_t st)
{
    a.tiles_p = shape.tiles_p;
    a.room = shape.room;
    a.partial = partial;
    const int64_t tiles = tiles_of(shape, a.rows);
    const bool whole = LQ == KALONG ? p.dhidden_whole : p.dweight_whole;
    return shape.tile > 128  ? multiply<GradJob<H, LQ, 256, 2, 4>>(shape, tiles, a, st, whole)
           : shape.tile > 64 ? multiply<GradJob<H, LQ, 128, 2, 2>>(shape, tiles, a, st, whole)
                             : multiply<GradJob<H, LQ, 64, 2, 2>>(shape, tiles, a, st, whole);
}

template <typename T, typename H> rf_status run(const rf_cross_entropy& a, const Plan& p, char* ws, hipStream_t st)
{
    const int planes = p.f32 ? 2 : 1;
    Scalars* const sc = (Scalars*)(ws + p.scalars);
    int32_t* const order = (int32_t*)(ws + p.order);
    int32_t* const target = (int32_t*)(ws + p.target);
    uint16_t* const hidden = (uint16_t*)(ws + p.hidden);
    const int64_t all = up(a.tokens, STEP), plane = all * p.pad;
    const Products products{p.rows, a.vocab, a.hidden, p.pad / STEP, p.vpad / STEP, (int32_t)p.pieces, p.pairs, p.grad, p.few, p.cus,
                            p.logits.tile, p.dhidden.tile, p.dweight.tile, p.logits_whole, p.dhidden_whole, p.dweight_whole};
    rf_status s = a.target_bits == 64
        ? launch<k_select<int64_t>>(1, SELECT, 0, st, (const int64_t*)a.targets, a.tokens, a.ignore_index, a.vocab, a.loss, order,
                                    target, sc, (Piece*)(ws + p.piece), products)
        : launch<k_select<int32_t>>(1, SELECT, 0, st, (const int32_t*)a.targets, a.tokens, a.ignore_index, a.vocab, a.loss, order,
                                    target, sc, (Piece*)(ws + p.piece), products);
    if (s != RF_OK) return s;
    const int32_t* const none = nullptr;
    if constexpr (sizeof(T) == 4) {
        s = launch<k_top>(std::min<int64_t>(a.tokens, 1024), 256, 0, st, (const float*)a.hidden_rows, a.tokens, a.hidden, a.hidden_stride,
                          (const int32_t*)order, (const Scalars*)sc, &sc->hidden_top);
        if (s != RF_OK) return s;
        s = launch<k_top>(std::min<int64_t>(a.vocab, 1024), 256, 0, st, (const float*)a.weight, a.vocab, a.hidden, a.weight_stride, none,
                          (const Scalars*)sc, &sc->weight_top);
        if (s != RF_OK) return s;
    }
    s = launch<k_pack<T>>(all, 256, 0, st, (const T*)a.hidden_rows, a.hidden, a.hidden_stride, p.pad, (const int32_t*)order,
                          (const Scalars*)sc, (const uint32_t*)&sc->hidden_top, hidden, hidden + plane, a.dhidden, (int)p.wide,
                          p.lifts && !p.f32 ? (uint32_t*)(ws + p.tops) : (uint32_t*)nullptr, a.tokens);
    if (s != RF_OK) return s;
    Side w{{a.weight, a.weight}, a.weight_stride * 2, a.vocab, a.vocab};
    if (p.own_weight) {
        uint16_t* const own = (uint16_t*)(ws + p.weight);
        s = launch<k_pack<T>>(a.vocab, 256, 0, st, (const T*)a.weight, a.hidden, a.weight_stride, p.pad, none, (const Scalars*)sc,
                              (const uint32_t*)&sc->weight_top, own, own + a.vocab * p.pad, (void*)nullptr, 0, (uint32_t*)nullptr, a.vocab);
        if (s != RF_OK) return s;
        w.base[0] = own;
        w.base[1] = own + (planes - 1) * a.vocab * p.pad;
        w.pitch = p.pad * 2;
    }
    for (int64_t piece = 0; piece < p.pieces; ++piece) {
        const int64_t first = piece * p.rows, rows = std::max<int64_t>(0, std::min(p.rows, a.tokens - first));
        const int64_t held = up(rows, STEP);
        uint16_t* const h = hidden + first * p.pad;
        Piece* const piece_info = (Piece*)(ws + p.piece) + piece;
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
        l.room = p.logits.room;
        l.partial = (float*)(ws + p.partial);
        l.piece = piece_info;
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
        r.piece = piece_info;
        r.z_loss = a.z_loss;
        r.sc = sc;
        r.order = order;
        r.target = target;
        r.stats = l.stats;
        r.picked = l.picked;
        r.dloss = a.dloss;
        r.loss = a.loss;
        r.reduction = reduction_of(a);
        if (p.grad) {
            r.top = (float*)(ws + p.top);
            r.factor = (float*)(ws + p.factor);
            r.at_target = (float*)(ws + p.at_target);
            if (p.lifts) {
                r.reach = (float*)(ws + p.reach);
                r.lifts = (int32_t*)(ws + p.lift);
            }
        }
        r.e = l.e;
        r.dz = ws + p.dz;
        if (p.f32) r.dz_low = (uint16_t*)(ws + p.dz) + up(p.rows, STEP) * p.vpad;
        else if (p.few) r.dz_low = (uint16_t*)(ws + p.low);
        s = launch<k_rows>(std::min<int64_t>((rows + 3) / 4, 2048), 256, 0, st, r);
        if (s != RF_OK) return s;
        if (!p.grad) continue;
        s = launch<k_dlogits<H, std::conditional_t<sizeof(T) == 4, float, f16>>>(held, 256, (size_t)p.blocks * 4, st, r);
        if (s != RF_OK) return s;
        Grad g{};
        Side dz{{r.dz, r.dz_low ? (const void*)r.dz_low : r.dz}, p.vpad * 2, held, held};
        g.sc = sc;
        g.piece = piece_info;
        g.first = first;
        g.piece_rows = rows;
        g.pairs = p.pairs;
        g.dtype = p.wide ? RF_F32 : a.dtype;
        g.cols = a.hidden;
        g.p = w;
        g.p.extent = p.pad;  // (its columns; as it is, hidden is a multiple of whole steps)
        g.q = dz;
        g.rows = rows;
        g.steps = p.vpad / STEP;
        g.order = order;
        g.lifts = r.lifts;
        g.out = a.dhidden;
        if (rows) {
            s = product<H, KALONG>(p, p.dhidden, (float*)(ws + p.partial), g, st);
            if (s != RF_OK) return s;
        }
        if constexpr (!__is_same(T, bf16)) {
            if (p.lifts) {
                s = launch<k_level<T>>(std::min<int64_t>(rows, 1024), 256, 0, st, (const T*)a.hidden_rows, a.hidden, a.hidden_stride,
                                       p.pad, (const int32_t*)order, first, rows, (const Scalars*)sc, piece_info,
                                       (const int32_t*)r.lifts, (const uint32_t*)(ws + p.tops), h, h + (planes - 1) * plane);
                if (s != RF_OK) return s;
            }
        }
        g.p = x;
        g.p.extent = p.pad;
        g.q.extent = p.vpad;
        g.rows = a.vocab;
        g.order = nullptr;
        g.out = a.dweight;
        g.sums = p.wide ? (float*)a.dweight : (float*)(ws + p.sums);
        g.begin = piece == 0;
        g.end = piece + 1 == p.pieces;
        s = product<H, KDOWN>(p, p.dweight, (float*)(ws + p.partial), g, st);
        if (s != RF_OK) return s;
    }
    if (reduction_of(a) != RF_REDUCE_NONE)
        return launch<k_total>(1, SELECT, 0, st, (const float*)a.loss, (const int32_t*)order, (const Scalars*)sc, (int)reduction_of(a), a.total);
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
    if (reduction_of(a) != RF_REDUCE_NONE && !a.total) return report(RF_ERR_INVALID, "a reduction needs total");
    if (reduction_of(a) != RF_REDUCE_NONE && a.dloss) return report(RF_ERR_INVALID, "dloss and a reduction exclude each other");
    if (a.dloss || a.dhidden || a.dweight) {
        if (!a.dweight || (a.tokens && (!a.dhidden || (!a.dloss && reduction_of(a) == RF_REDUCE_NONE))))
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
