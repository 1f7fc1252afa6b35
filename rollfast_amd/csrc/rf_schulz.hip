// rf_schulz.hip -- matrices with their singular values brought near one:
//   X = G / (|G| + eps),  then for each step's a, b, c
//   A = X X^T,  B = b A + c A^2,  X = a X + B X
// with |G| the Frobenius norm.  With n <= m the sides of the matrix (a tall one is
// worked on transposed) a step is three products, n^2 m, n^3 and 2 n^2 m operations:
// A and B are symmetric, and only the tiles on and below the diagonal are computed.
//
// A list of matrices goes through the same launches, up to MAX at a time: the tiles
// of all of them fill the GPU where those of one would not.
//
// Types.  The products are f16 with f32 sums.  X has singular values below R (the
// bound that the coefficients allow, worked out on the host), so that no entry of X,
// A or B is larger than R, R^2 and the largest |b s^2 + c s^4|: fixed powers of two
// bring them near f16's largest, and entries 2^-29 of the bound are still exact to
// their last bits.  What f16 rounds away from X would be lost to small singular
// values, which grow by a factor of a in every step: X is kept in two parts, high
// and low, the low one a byte, 19 bits together, and the term (a + B_ii) X takes both;
// only the product with the rest of B takes the high part alone, B's diagonal being
// kept in f32 apart.  In 64-bit simulation that leaves an error of 3e-4 to 9e-4 of the
// result's norm for matrices of 256 x 256 to 768 x 2304, Gaussian or close to low rank
// (without low parts and diagonal: 1.5e-2 for the latter), and up to 1.2e-3 near rank
// one (low parts of 22 bits 1.1e-3, none 1.5e-1), beside bf16's rounding of the result,
// 1.7e-3.  Results in f32 or f16 take both parts of X, A and B everywhere, in
// three products: high high, high low, low high.
#include "rf_schulz.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "rf_product.h"

using namespace rfb;
using namespace rfp;
using rf::report;

namespace rfs {
namespace {

constexpr int64_t HELD = 8ll << 30;  // bytes of workspace of matrices worked on together

struct Item {
    const void* in;
    void* out;
    const void* add;
    double* sums;
    uint16_t* buffers;
    int64_t in_stride, out_stride, add_stride;
    int32_t n, m;      // padded to whole steps
    int32_t rows, cols;
    float scale, add_scale;
    uint32_t first;    // its first tile
    uint8_t tall, in_dtype, out_dtype, add_dtype;

    // X and the next X: [n, m] high parts, then low parts (a byte each, or f16 where they
    // are operands: split).  A and B: [n, n] high parts; split: then low parts.  B's
    // diagonal [n].
    __host__ __device__ int64_t plane() const { return (int64_t)n * m; }
    __host__ __device__ int64_t square(bool split) const { return (int64_t)n * n * (split ? 2 : 1); }
    __device__ uint16_t* x(int turn) const { return buffers + (turn ? 2 * plane() : 0); }
    __device__ uint16_t* a() const { return buffers + 4 * plane(); }
    __device__ uint16_t* b(bool split) const { return a() + square(split); }
    __device__ float* d(bool split) const { return (float*)(b(split) + square(split)); }
    __host__ int64_t bytes(bool split) const { return 8 * plane() + 4 * square(split) + 4 * (int64_t)n; }
};

struct Batch {
    int32_t count, turn;  // turn: x and y change places
    int32_t last;         // the last step: X's low parts are read no more
    float a, b, c;        // the step's coefficients
    float eps, x_scale, a_scale, b_scale;
    uint32_t tiles;
    Share share;          // what becomes of the tiles (rf_product.h)
    uint32_t room;
    float* partial;
    Item item[MAX];
};
static_assert(sizeof(Batch) <= 4096, "kernel arguments");

__device__ __forceinline__ int find(const Batch& t, uint32_t id)
{
    int i = 0;
    while (i + 1 < t.count && id >= t.item[i + 1].first) ++i;
    return i;
}

// What f16 rounded away of a value, in a byte: the difference of the two as f32 have
// it in their last bits, 13 of them, to 8 (so 19 bits of X's 24 are kept).  Where hi
// is below f16's normal numbers it may not fit, and is off by less than 2^-25.
__device__ __forceinline__ uint32_t low_byte(float v, float hi)
{
    const int d = (int)__float_as_uint(v) - (int)__float_as_uint(hi);
    return (uint32_t)min(max((d + 16) >> 5, -128), 127) & 255u;
}

__device__ __forceinline__ uint32_t low_bytes(f32x4 v, f32x4 hi)
{
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) w |= low_byte(v[k], hi[k]) << (8 * k);
    return w;
}

__device__ __forceinline__ f32x4 with_low_bytes(f32x4 hi, uint32_t low)
{
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int d = (int)(low << (24 - 8 * k)) >> 24;
        hi[k] = __uint_as_float(__float_as_uint(hi[k]) + (uint32_t)(d * 32));
    }
    return hi;
}

// Partial sums of squares, in f64 (a square of an f32 may have no f32): part s of a
// matrix takes every PARTS-th group of rows, as many as its lanes cover with eight
// columns each.
template <typename T> __device__ __forceinline__ double squares(const Item& it, int part)
{
    const int64_t chunks = (it.cols + 7) / 8;
    int lanes = 256;
    while (lanes > 1 && lanes / 2 >= chunks) lanes /= 2;
    const int rows = 256 / lanes;
    double sum = 0;
    for (int64_t r = (int64_t)part * rows + threadIdx.x / lanes; r < it.rows; r += (int64_t)PARTS * rows) {
        const T* const row = (const T*)it.in + r * it.in_stride;
        for (int64_t c = threadIdx.x % lanes; c < chunks; c += lanes) {
            float v[8];
            widen8(load8(row, c * 8, it.cols), v);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += (double)v[k] * (double)v[k];
        }
    }
    return sum;
}

__global__ __launch_bounds__(256) void k_squares(const Batch t)
{
    __shared__ double part[4];
    const Item& it = t.item[blockIdx.x / PARTS];
    const int s = blockIdx.x % PARTS, tid = threadIdx.x;
    double sum = it.in_dtype == RF_F32 ? squares<float>(it, s) : it.in_dtype == RF_BF16 ? squares<bf16>(it, s) : squares<f16>(it, s);
    for (int d = 1; d < WAVE; d *= 2) sum += __shfl_xor(sum, d);
    if (tid % WAVE == 0) part[tid / WAVE] = sum;
    __syncthreads();
    if (tid == 0) it.sums[s] = part[0] + part[1] + part[2] + part[3];
}

// G into X's layout, a tile of 64 x 64 of X a workgroup.
template <bool SPLIT> __global__ __launch_bounds__(256) void k_load(const Batch t)
{
    __shared__ float tile[64][65];
    const Item& it = t.item[find(t, blockIdx.x)];
    const uint32_t id = blockIdx.x - it.first, across = it.m / 64;
    const int64_t p0 = id % across * 64, q0 = id / across * 64;
    const int tid = threadIdx.x, lane = tid % WAVE;
    double norm = 0;
    for (int i = lane; i < PARTS; i += WAVE) norm += it.sums[i];
    for (int d = 1; d < WAVE; d *= 2) norm += __shfl_xor(norm, d);
    const double s = (double)t.x_scale / (sqrt(norm) + (double)t.eps);
    const int64_t r0 = it.tall ? p0 : q0, c0 = it.tall ? q0 : p0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = i * 32 + tid / 8, c = tid % 8 * 8;
        float v[8] = {};
        if (r0 + r < it.rows) {
            const int64_t at = (r0 + r) * it.in_stride;
            if (it.in_dtype == RF_F32) widen8(load8((const float*)it.in + at, c0 + c, it.cols), v);
            else if (it.in_dtype == RF_BF16) widen8(load8((const bf16*)it.in + at, c0 + c, it.cols), v);
            else widen8(load8((const f16*)it.in + at, c0 + c, it.cols), v);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float w = (float)((double)v[k] * s);
            if (it.tall) tile[c + k][r] = w;
            else tile[r][c + k] = w;
        }
    }
    __syncthreads();
    const int64_t plane = (int64_t)it.n * it.m;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int q = i * 32 + tid / 8, p = tid % 8 * 8;
        float v[8], back[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = tile[q][p + k];
        const Raw<f16> hi = narrow8<f16>(v);
        widen8(hi, back);
        const int64_t at = (q0 + q) * it.m + p0 + p;
        *(u32x4*)(it.x(0) + at) = hi.a;
        if constexpr (SPLIT) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] -= back[k];
            *(u32x4*)(it.x(0) + plane + at) = narrow8<f16>(v).a;
        } else {
            const u32x2 low = {low_bytes(f32x4{v[0], v[1], v[2], v[3]}, f32x4{back[0], back[1], back[2], back[3]}),
                               low_bytes(f32x4{v[4], v[5], v[6], v[7]}, f32x4{back[4], back[5], back[6], back[7]})};
            *(u32x2*)((uint8_t*)(it.x(0) + plane) + at) = low;
        }
    }
}

// Tile number `id` of the lower triangle, row by row.
__device__ __forceinline__ TileAt lower(uint32_t id)
{
    uint32_t q = (uint32_t)((sqrtf(8.0f * (float)id + 1.0f) - 1.0f) * 0.5f);
    while (q * (q + 1) / 2 > id) --q;
    while ((q + 1) * (q + 2) / 2 <= id) ++q;
    return {id - q * (q + 1) / 2, q};
}

// A wave's tile of a symmetric matrix, in f16: its rows, and where the tile is not
// on the diagonal its columns as rows, transposed through LDS (`room`: the wave's
// own, rows of PITCH bytes, so that neither writes nor reads of a column meet in a
// bank).  With `low` the low parts go to `o + low`.
template <typename G, int PITCH, bool LOW>
__device__ __forceinline__ void put_symmetric(uint16_t* o, int64_t low, int64_t n, int64_t q0, int64_t p0,
                                              const typename G::Sums& v, bool mirror, char* room)
{
    const int lane = own_lane();
#pragma unroll
    for (int part = 0; part < (LOW ? 2 : 1); ++part) {
#pragma unroll
        for (int j = 0; j < G::FQ; ++j) {
            const int64_t q = q0 + 16 * j + lane % 16;
#pragma unroll
            for (int i = 0; i < G::FP; i += 2) {
                u32x2 w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const f32x4 x = v[i + k][j];
                    w[k] = narrow4<f16>(x);
                    if (part) w[k] = narrow4<f16>(x - widen4<f16>(w[k]));
                }
                const u32x4 c = chunk(w[0], w[1]);
                const int64_t p = p0 + 16 * i + chunk_of(lane);
                if (q < n && p < n) *(u32x4*)(o + part * low + q * n + p) = c;
                if (mirror) *(u32x4*)(room + (16 * j + lane % 16) * PITCH + (16 * i + chunk_of(lane)) * 2) = c;
            }
        }
        if (!mirror) continue;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        // lane l: column l % 16 of a fragment, rows 8 (l / 16) .. + 7 of 32
#pragma unroll
        for (int h = 0; h < G::FQ / 2; ++h)
#pragma unroll
            for (int i = 0; i < G::FP; ++i) {
                union { s16x4 half[2]; u32x4 v; } u;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    u.half[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(lds_char*)(room + (32 * h + 8 * (lane >> 4) + ((lane & 15) >> 2) + 4 * k) * PITCH + i * 32 + (lane & 3) * 8));
                const int64_t p = p0 + 16 * i + lane % 16, q = q0 + 32 * h + lane / 16 * 8;
                if (p < n && q < n) *(u32x4*)(o + part * low + p * n + q) = u.v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// A tile of one of the batch's matrices; they differ in their number of steps.
struct Place {
    int item;
    int64_t p0, q0, steps;
};

// What the jobs of a batch share.  J: steps(item), place(item, tile) of TILE.
template <typename J> struct Batched {
    typedef Batch Args;
    typedef Place Tile;

    static __device__ Share share(const Batch& t) { return t.share; }
    static __device__ Place tile(const Batch& t, uint32_t id)
    {
        const int i = find(t, id);
        const TileAt at = J::place(t.item[i], id - t.item[i].first);
        return {i, (int64_t)at.p * J::TILE, (int64_t)at.q * J::TILE, J::steps(t.item[i])};
    }
};

// SQUARE: B from A; else A from X.  Bound by the matrix cores: for the seven matrices of a
// layer (four of 4096 x 4096, three of 11008 x 4096) the tiles on and below the diagonal
// are 0.88 TFLOP of A, 786 us (1.12 PFLOP/s), and 0.51 TFLOP of A^2, 455 us.
template <bool SQUARE, bool SPLIT, int TILE_, int WP, int WQ> struct Symmetric : Batched<Symmetric<SQUARE, SPLIT, TILE_, WP, WQ>> {
    static constexpr int TILE = TILE_;
    typedef Product<f16, KALONG, KALONG, TILE, TILE, WP, WQ> G;
    static constexpr int PITCH = TILE / WP * 2 + 16, ROOM = TILE / WQ * PITCH;
    static constexpr int LDS = std::max(G::LDS, G::WAVES * ROOM), SETTLE_LDS = ROOM, ENDS = TILE > 128 ? 8000 : TILE > 64 ? 5000 : 3000;

    static __host__ __device__ int64_t steps(const Item& it) { return (SQUARE ? it.n : it.m) / STEP; }
    static __host__ int64_t tiles(const Item& it)
    {
        const int64_t n = (it.n + TILE - 1) / TILE;
        return n * (n + 1) / 2;
    }
    static __device__ TileAt place(const Item&, uint32_t id) { return lower(id); }

    static __device__ __forceinline__ void run(const Batch& t, const Place& at, char* lds, int64_t s0, int64_t s1, typename G::Sums& acc)
    {
        const Item& it = t.item[at.item];
        const uint16_t* const from = SQUARE ? it.a() : it.x(t.turn);
        const int64_t depth = SQUARE ? it.n : it.m;
        const Side s{{from, from + (SPLIT ? it.n * depth : 0)}, depth * 2, it.n, it.n};
        G::run(lds, s, s, at.p0, at.q0, s0, s1, SPLIT ? 3 : 1, acc);
    }
    static __device__ __forceinline__ void finish(const Batch& t, const Place& at, typename G::Sums& acc, int wave, char* lds)
    {
        const Item& it = t.item[at.item];
        const int64_t n = it.n, plane = n * n;
        const int lane = own_lane();
        const bool mirror = at.p0 != at.q0;
        const int64_t wp = at.p0 + G::wp(wave), wq = at.q0 + G::wq(wave);
        // stored A = a_scale A, X = x_scale X
        const float of_a = t.a_scale / (t.x_scale * t.x_scale);
        const float b_of = t.b * t.b_scale / t.a_scale, c_of = t.c * t.b_scale / (t.a_scale * t.a_scale);
#pragma unroll
        for (int j = 0; j < G::FQ; ++j) {
            const int64_t q = wq + 16 * j + lane % 16;
            if constexpr (!SQUARE) {
#pragma unroll
                for (int i = 0; i < G::FP; ++i) acc[i][j] *= of_a;
            } else {
                u32x4 old[SPLIT ? 1 : G::FP / 2];  // A here; of one part all loads in flight together
                auto load = [&](int part, int i) {
                    return *(const u32x4*)(it.a() + part * plane + min(q, n - 1) * n + min(wp + 16 * i + chunk_of(lane), n - 8));
                };
                if (!SPLIT) {
#pragma unroll
                    for (int i = 0; i < G::FP; i += 2) old[SPLIT ? 0 : i / 2] = load(0, i);
                }
#pragma unroll
                for (int i = 0; i < G::FP; i += 2) {
                    f32x4 a[2] = {};
#pragma unroll
                    for (int part = 0; part < (SPLIT ? 2 : 1); ++part) {
                        u32x2 x, y;
                        quads(SPLIT ? load(part, i) : old[SPLIT ? 0 : i / 2], x, y);
                        a[0] += widen4<f16>(x);
                        a[1] += widen4<f16>(y);
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        f32x4 v = b_of * a[k] + c_of * acc[i + k][j];
                        const int64_t p = wp + 16 * (i + k) + lane / 16 * 4;
                        if (!mirror && q < n) {
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (p + r == q) {
                                    it.d(SPLIT)[q] = v[r] / t.b_scale;
                                    v[r] = 0.0f;
                                }
                        }
                        acc[i + k][j] = v;
                    }
                }
            }
        }
        // a wave's own room in LDS: its part of the workgroup's, or all of a settling wave's
        char* const room = lds + (blockDim.x > WAVE ? wave * ROOM : 0);
        put_symmetric<G, PITCH, SPLIT>(SQUARE ? it.b(SPLIT) : it.a(), plane, n, wq, wp, acc, mirror, room);
    }
};

// scale times eight neighbours of an output's row, and add_scale times what is to be
// added, from column c on.
__device__ __forceinline__ void put_out8(const Item& it, int64_t r, int64_t c, float (&v)[8])
{
    const int64_t left = it.cols - c;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= it.scale;
    if (it.add) {
        float w[8];
        if (it.add_dtype == RF_F32) widen8(load8((const float*)it.add + r * it.add_stride, c, it.cols), w);
        else if (it.add_dtype == RF_BF16) widen8(load8((const bf16*)it.add + r * it.add_stride, c, it.cols), w);
        else widen8(load8((const f16*)it.add + r * it.add_stride, c, it.cols), w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += it.add_scale * w[k];
    }
    const int64_t at = r * it.out_stride + c;
    if (it.out_dtype == RF_F32) put8((float*)it.out + at, narrow8<float>(v), left);
    else if (it.out_dtype == RF_BF16) put8((bf16*)it.out + at, narrow8<bf16>(v), left);
    else put8((f16*)it.out + at, narrow8<f16>(v), left);
}

// X = (a + B_ii) X + (the rest of B) X.  For the same matrices 1.66 TFLOP in 1.49 ms, 1.11
// PFLOP/s, of which reading and writing X, 6 bytes an element, would take 0.25 ms alone: a
// workgroup's products do not run beside its own epilogue, and tiles of 256 leave room for no
// other.  (Low parts of 16 bits, 8 bytes: 1.58 ms.)
template <bool SPLIT, int TILE_, int WP, int WQ> struct Apply : Batched<Apply<SPLIT, TILE_, WP, WQ>> {
    static constexpr int TILE = TILE_;
    typedef Product<f16, KDOWN, KALONG, TILE, TILE, WP, WQ> G;
    static constexpr int LDS = G::LDS, SETTLE_LDS = 0, ENDS = TILE > 128 ? 24000 : TILE > 64 ? 8500 : 5000;  // (X read and written)

    static __host__ __device__ int64_t steps(const Item& it) { return it.n / STEP; }
    static __host__ int64_t tiles(const Item& it) { return (int64_t)((it.n + TILE - 1) / TILE) * ((it.m + TILE - 1) / TILE); }
    static __device__ TileAt place(const Item& it, uint32_t id)
    {
        return tile_at(id, (uint32_t)((it.m + TILE - 1) / TILE), (uint32_t)((it.n + TILE - 1) / TILE));
    }
    static __device__ __forceinline__ void run(const Batch& t, const Place& at, char* lds, int64_t s0, int64_t s1, typename G::Sums& acc)
    {
        const Item& it = t.item[at.item];
        const int64_t n = it.n, m = it.m;
        const uint16_t *const x = it.x(t.turn), *const b = it.b(SPLIT);
        const Side sx{{x, x + (SPLIT ? it.plane() : 0)}, m * 2, m, n};
        const Side sb{{b, b + (SPLIT ? n * n : 0)}, n * 2, n, n};
        G::run(lds, sx, sb, at.p0, at.q0, s0, s1, SPLIT ? 3 : 1, acc);
    }
    static __device__ __forceinline__ void finish(const Batch& t, const Place& at, typename G::Sums& acc, int wave, char*);
};

template <bool SPLIT, int TILE, int WP, int WQ>
__device__ __forceinline__ void Apply<SPLIT, TILE, WP, WQ>::finish(const Batch& t, const Place& at, typename G::Sums& acc, int wave, char*)
{
    const Item& it = t.item[at.item];
    const int64_t n = it.n, m = it.m, plane = n * m;
    const uint16_t* const x = it.x(t.turn);
    uint16_t* const y = it.x(!t.turn);
    const int lane = own_lane();
    const float of_product = 1.0f / t.b_scale;
    const int64_t wp = at.p0 + G::wp(wave), wq = at.q0 + G::wq(wave);
    // X here, a row of fragments ahead: all of its loads in flight together
    typedef std::conditional_t<SPLIT, u32x4, u32x2> Low;
    struct Row { u32x4 hi[G::FP / 2]; Low lo[G::FP / 2]; float d; } row[2];
    auto fetch = [&](int j, Row& r) {
        const int64_t q = min(wq + 16 * j + lane % 16, n - 1);
        r.d = it.d(SPLIT)[q];
#pragma unroll
        for (int i = 0; i < G::FP; i += 2) {
            const int64_t from = q * m + min(wp + 16 * i + chunk_of(lane), m - 8);
            r.hi[i / 2] = *(const u32x4*)(x + from);
            if constexpr (SPLIT) r.lo[i / 2] = *(const u32x4*)(x + plane + from);
            else r.lo[i / 2] = *(const u32x2*)((const uint8_t*)(x + plane) + from);
        }
    };
    fetch(0, row[0]);
#pragma unroll
    for (int j = 0; j < G::FQ; ++j) {
        if (j + 1 < G::FQ) fetch(j + 1, row[(j + 1) & 1]);
        const Row& old = row[j & 1];
        const int64_t q = wq + 16 * j + lane % 16;
        const float diagonal = t.a + old.d;
#pragma unroll
        for (int i = 0; i < G::FP; i += 2) {
            f32x4 v[2];
            u32x2 h[2], l[2];
            uint32_t bytes[2];
            quads(old.hi[i / 2], h[0], h[1]);
            if constexpr (SPLIT) {
                quads(old.lo[i / 2], l[0], l[1]);
            } else {
                const auto b = __builtin_amdgcn_permlane16_swap(old.lo[i / 2][0], old.lo[i / 2][1], false, false);
                bytes[0] = b[0];
                bytes[1] = b[1];
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f32x4 was = SPLIT ? widen4<f16>(h[k]) + widen4<f16>(l[k]) : with_low_bytes(widen4<f16>(h[k]), bytes[k]);
                v[k] = diagonal * was + of_product * acc[i + k][j];
                h[k] = narrow4<f16>(v[k]);
                if (SPLIT) l[k] = narrow4<f16>(v[k] - widen4<f16>(h[k]));
                else bytes[k] = low_bytes(v[k], widen4<f16>(h[k]));
            }
            const int64_t p = wp + 16 * i + chunk_of(lane), to = q * m + p;
            const u32x4 hi = chunk(h[0], h[1]);
            if constexpr (SPLIT) {
                const u32x4 lo = chunk(l[0], l[1]);
                if (q < n && p < m) {
                    *(u32x4*)(y + to) = hi;
                    *(u32x4*)(y + plane + to) = lo;
                }
            } else {
                const auto lo = __builtin_amdgcn_permlane16_swap(bytes[0], bytes[1], false, false);
                if (q < n && p < m) {
                    *(u32x4*)(y + to) = hi;
                    if (!t.last) *(u32x2*)((uint8_t*)(y + plane) + to) = u32x2{lo[0], lo[1]};
                }
            }
        }
    }
}

template <typename J> __global__ __launch_bounds__(J::G::THREADS, 2) void k_multiply(const Batch)
{
    extern __shared__ char lds[];
    multiply_tiles<J>(argument<Batch>(), lds);
}

template <typename J> __global__ __launch_bounds__(WAVE, 2) void k_settle(const Batch)
{
    extern __shared__ char lds[];
    settle_tiles<J>(argument<Batch>(), lds);
}

// Outputs from X, a tile of 64 x 64 a workgroup; tall matrices' are transposed.  (In the
// last product's epilogue they would need registers that its sums take: with tiles of 256
// it spilled 340 and took 942 us where this and the product take 560.)  bf16 results are
// rounded from X's high part, whose 11 bits add an eighth to their worst half step.
template <bool SPLIT> __global__ __launch_bounds__(256) void k_store(const Batch t)
{
    __shared__ float tile[64][65];
    const Item& it = t.item[find(t, blockIdx.x)];
    const uint32_t id = blockIdx.x - it.first, across = it.m / 64;
    const int64_t p0 = id % across * 64, q0 = id / across * 64, plane = it.plane();
    const int tid = threadIdx.x;
    const float last = 1.0f / t.x_scale;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int q = i * 32 + tid / 8, p = tid % 8 * 8;
        const uint16_t* const o = it.x(t.turn) + (q0 + q) * it.m + p0 + p;
        float w[8], w2[8] = {};
        widen8(Raw<f16>{*(const u32x4*)o}, w);
        if (SPLIT) widen8(Raw<f16>{*(const u32x4*)(o + plane)}, w2);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float v = (w[k] + w2[k]) * last;
            if (it.tall) tile[p + k][q] = v;
            else tile[q][p + k] = v;
        }
    }
    __syncthreads();
    const int64_t r0 = it.tall ? p0 : q0, c0 = it.tall ? q0 : p0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = i * 32 + tid / 8, c = tid % 8 * 8;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = tile[r][c + k];
        if (r0 + r < it.rows && c0 + c < it.cols) put_out8(it, r0 + r, c0 + c, v);
    }
}

// ------------------------------------------------------------------- host ---
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

template <auto K> rf_status launch(int64_t grid, int threads, size_t lds, hipStream_t st, const Batch& t)
{
    static std::atomic<uint64_t> done;
    if (grid <= 0) return RF_OK;
    if (grid > 0x7FFFFFFF) return report(RF_ERR_UNSUPPORTED, "too many workgroups for one launch");
    if (const rf_status s = allow_lds((const void*)K, lds, done); s != RF_OK) return s;
    K<<<(uint32_t)grid, threads, lds, st>>>(t);
    return RF_OK;
}

// Numbers the batch's tiles and gives their number.
template <typename F> uint32_t number(Batch& t, F tiles)
{
    uint32_t all = 0;
    for (int i = 0; i < t.count; ++i) {
        t.item[i].first = all;
        all += (uint32_t)tiles(t.item[i]);
    }
    return t.tiles = all;
}

// A product of all matrices of the batch: numbers its tiles, those with the longest
// sums first as the list is (see run), and shares them out.  ns: what it takes.
template <typename J> double lay_out(Batch& t, int cus, int pairs)
{
    t.room = room_of(J::TILE, cus);
    t.tiles = 0;
    int64_t units = 0, longest = 0, shortest = 1ll << 40;
    for (int i = 0; i < t.count; ++i) {
        const int64_t tiles = J::tiles(t.item[i]), steps = J::steps(t.item[i]);
        t.item[i].first = t.tiles;
        t.tiles += (uint32_t)tiles;
        units += tiles * steps;
        longest = std::max(longest, steps);
        shortest = std::min(shortest, steps);
    }
    // sums of unlike length are split, all alike, only where there is less than a round of
    // them: a last round is of the shortest
    const Cost c = cost_of(J::TILE, pairs, J::ENDS);
    t.share = {t.tiles, 0, 1};
    if (longest == shortest || t.tiles < t.room) t.share = share_of(t.tiles, longest, t.room, c);
    if (longest == shortest || t.share.rest) return ns_of(t.share, longest, t.room, c);
    return std::max((double)longest, (double)units / std::min(t.room, t.tiles) + (double)shortest / 2) * c.step +
           (double)((t.tiles + t.room - 1) / t.room) * c.ends;
}

template <typename J> rf_status multiply(Batch& t, hipStream_t st)
{
    const rf_status s = launch<k_multiply<J>>((int64_t)t.share.whole + (int64_t)t.share.rest * t.share.parts, J::G::THREADS, J::LDS, st, t);
    return s != RF_OK ? s : launch<k_settle<J>>((int64_t)t.share.rest * J::G::WAVES, WAVE, J::SETTLE_LDS, st, t);
}

// With the tiles that take least.
template <typename Big, typename Middle, typename Small> rf_status product(Batch& t, int cus, int pairs, hipStream_t st)
{
    const double big = lay_out<Big>(t, cus, pairs), middle = lay_out<Middle>(t, cus, pairs);
    if (lay_out<Small>(t, cus, pairs) <= std::min(big, middle)) return multiply<Small>(t, st);
    if (middle <= big) {
        lay_out<Middle>(t, cus, pairs);
        return multiply<Middle>(t, st);
    }
    lay_out<Big>(t, cus, pairs);
    return multiply<Big>(t, st);
}

template <bool SPLIT> rf_status step(Batch& t, int cus, hipStream_t st)
{
    constexpr int PAIRS = SPLIT ? 3 : 1;
    rf_status s = product<Symmetric<false, SPLIT, 256, 2, 4>, Symmetric<false, SPLIT, 128, 2, 2>, Symmetric<false, SPLIT, 64, 2, 2>>(t, cus, PAIRS, st);
    if (s == RF_OK) s = product<Symmetric<true, SPLIT, 256, 2, 4>, Symmetric<true, SPLIT, 128, 2, 2>, Symmetric<true, SPLIT, 64, 2, 2>>(t, cus, PAIRS, st);
    if (s != RF_OK) return s;
    return product<Apply<SPLIT, 256, 2, 4>, Apply<SPLIT, 128, 2, 2>, Apply<SPLIT, 64, 2, 2>>(t, cus, PAIRS, st);
}

// The largest singular value, and the largest |b s^2 + c s^4|, that the steps can
// reach from 0 .. 1: each step's extremes lie where its derivative a + 3 b s^2 +
// 5 c s^4 is zero, or at the ends.
struct Bounds { double x, b; };

Bounds bounds_of(const Method& how)
{
    double top = 1, most = 1, b_most = 0;
    for (int s = 0; s < how.steps; ++s) {
        const double a = how.coefficients[3 * s], b = how.coefficients[3 * s + 1], c = how.coefficients[3 * s + 2];
        auto f = [&](double v) { return std::fabs(v * (a + v * v * (b + c * v * v))); };
        auto g = [&](double v) { return std::fabs(v * v * (b + c * v * v)); };
        double next = f(top), g_next = g(top);
        const double root = 9 * b * b - 20 * a * c;
        for (int sign = -1; sign <= 1; sign += 2) {
            const double s2 = c != 0 && root >= 0 ? (-3 * b + sign * std::sqrt(root)) / (10 * c) : c == 0 && b != 0 ? -a / (3 * b) : -1;
            if (s2 > 0 && s2 < top * top) next = std::max(next, f(std::sqrt(s2)));
        }
        if (c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < top * top) g_next = std::max(g_next, g(std::sqrt(-b / (2 * c))));
        top = next;
        most = std::max(most, top);
        b_most = std::max(b_most, g_next);
        if (!(top < 1e6) || !(b_most < 1e9)) return {1e9, 1e9};
    }
    return {most, b_most};
}

bool split_of(const Matrix& m) { return m.out_dtype != RF_BF16; }

bool known(int32_t dtype) { return dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16; }

// A matrix' item, without its buffers.
Item item_of(const Matrix& m)
{
    Item it{};
    it.in = m.in;
    it.out = m.out;
    it.add = m.add;
    it.in_stride = m.in_stride;
    it.out_stride = m.out_stride;
    it.add_stride = m.add_stride;
    it.rows = (int32_t)m.rows;
    it.cols = (int32_t)m.cols;
    it.tall = m.rows > m.cols;
    it.n = (int32_t)up(std::min(m.rows, m.cols), STEP);
    it.m = (int32_t)up(std::max(m.rows, m.cols), STEP);
    it.scale = m.scale;
    it.add_scale = m.add_scale;
    it.in_dtype = (uint8_t)m.in_dtype;
    it.out_dtype = (uint8_t)m.out_dtype;
    it.add_dtype = (uint8_t)m.add_dtype;
    return it;
}

int64_t bytes_of(const Matrix& m) { return up(item_of(m).bytes(split_of(m)), 256); }

// The matrices from `at` on that are worked on together, and what they need: sums of
// squares, the parts of split tiles, their buffers.
struct Needs {
    int64_t end, sums, parts, buffers;
    int64_t all() const { return sums + parts + buffers; }
};

Needs needs_of(const Matrix* list, int64_t count, int64_t at, int cus)
{
    Needs need{at, 0, 0, 0};
    constexpr int64_t TILES[3] = {64, 128, 256};
    int64_t tiles[3] = {};  // of the product with the most
    for (; need.end < count && need.end - at < MAX; ++need.end) {
        const Matrix& m = list[need.end];
        const bool some = m.rows && m.cols;
        const int64_t more = some ? bytes_of(m) : 0;
        if (need.end > at && (need.buffers + more > HELD || split_of(m) != split_of(list[at]))) break;
        need.buffers += more;
        if (!some) continue;
        const Item it = item_of(m);
        for (int k = 0; k < 3; ++k) tiles[k] += ((it.n + TILES[k] - 1) / TILES[k]) * ((it.m + TILES[k] - 1) / TILES[k]);
    }
    for (int k = 0; k < 3; ++k)
        need.parts = std::max(need.parts, std::min<int64_t>((int64_t)room_of((int)TILES[k], cus) * PARTS_ROOM, tiles[k] * MOST_PARTS) * TILES[k] * TILES[k] * 4);
    need.sums = (need.end - at) * PARTS * 8;
    return need;
}

}  // namespace

rf_status check(const Matrix* list, int64_t count, const Method& how) noexcept
{
    if (count < 0 || (count && !list)) return report(RF_ERR_INVALID, "null list");
    if (how.steps < 0 || how.steps > 100 || (how.steps && !how.coefficients)) return report(RF_ERR_INVALID, "steps out of range");
    for (int i = 0; i < 3 * how.steps; ++i)
        if (!std::isfinite(how.coefficients[i])) return report(RF_ERR_INVALID, "coefficients must be finite");
    if (!(how.eps >= 0.0f) || !std::isfinite(how.eps)) return report(RF_ERR_INVALID, "eps must be finite and not negative");
    const Bounds most = bounds_of(how);
    if (most.x > 64 || most.b > 30000) return report(RF_ERR_INVALID, "coefficients let singular values grow past 64");
    for (int64_t i = 0; i < count; ++i) {
        const Matrix& m = list[i];
        if (m.rows < 0 || m.cols < 0 || m.rows > (1 << 20) || m.cols > (1 << 20) || std::min(m.rows, m.cols) > (1 << 16))
            return report(RF_ERR_INVALID, "matrix size out of range");
        if (!known(m.in_dtype) || !known(m.out_dtype) || (m.add && !known(m.add_dtype)))
            return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
        if (m.in_stride < 0 || m.out_stride < 0 || m.add_stride < 0) return report(RF_ERR_INVALID, "negative stride");
        if (m.rows && m.cols && (!m.in || !m.out)) return report(RF_ERR_INVALID, "null buffer");
    }
    return RF_OK;
}

rf_status workspace(const Matrix* list, int64_t count, int64_t* bytes) noexcept
{
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    *bytes = 0;
    for (int64_t at = 0; at < count;) {
        const Needs need = needs_of(list, count, at, cus);
        at = need.end;
        *bytes = std::max(*bytes, need.all());
    }
    return RF_OK;
}

rf_status run(const Matrix* list, int64_t count, const Method& how, char* ws, hipStream_t st, Source source, void* context) noexcept
{
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    const Bounds most = bounds_of(how);
    auto scale = [](double bound) { return (float)std::exp2(std::min(15.0, std::floor(std::log2(60000.0 / std::max(bound, 1e-3))))); };
    for (int64_t at = 0; at < count;) {
        const Needs need = needs_of(list, count, at, cus);
        const int64_t end = need.end;
        const bool split = split_of(list[at]);
        Batch t{};
        t.eps = how.eps;
        t.x_scale = scale(most.x);
        t.a_scale = scale(most.x * most.x);
        t.b_scale = scale(most.b);
        t.partial = (float*)(ws + need.sums);
        int64_t used = need.sums + need.parts;
        int64_t which[MAX];
        float* u[MAX];
        double* sums[MAX];
        for (int64_t i = at; i < end; ++i) {
            const Matrix& m = list[i];
            if (!m.rows || !m.cols) continue;
            Item& it = t.item[t.count];
            it = item_of(m);
            it.sums = sums[t.count] = (double*)ws + (int64_t)t.count * PARTS;
            it.buffers = (uint16_t*)(ws + used);
            used += up(it.bytes(split), 256);
            which[t.count] = i;
            u[t.count] = (float*)(it.buffers + 2 * it.plane());  // where the next X will lie
            if (source) {
                it.in = u[t.count];
                it.in_dtype = RF_F32;
                it.in_stride = m.cols;
            }
            ++t.count;
        }
        at = end;
        if (!t.count) continue;
        // those with the longest sums first: what is left at a launch's end is short
        std::stable_sort(t.item, t.item + t.count, [](const Item& x, const Item& y) { return x.m > y.m; });
        rf_status s = RF_OK;
        s = source ? source(context, which, t.count, u, sums, st) : launch<k_squares>((int64_t)t.count * PARTS, 256, 0, st, t);
        if (s != RF_OK) return s;
        const uint32_t squares = number(t, [](const Item& it) { return (int64_t)it.n / 64 * (it.m / 64); });
        s = split ? launch<k_load<true>>(squares, 256, 0, st, t) : launch<k_load<false>>(squares, 256, 0, st, t);
        if (s != RF_OK) return s;
        for (int i = 0; i < how.steps && s == RF_OK; ++i) {
            t.a = how.coefficients[3 * i];
            t.b = how.coefficients[3 * i + 1];
            t.c = how.coefficients[3 * i + 2];
            t.turn = i & 1;
            t.last = i + 1 == how.steps;
            s = split ? step<true>(t, cus, st) : step<false>(t, cus, st);
        }
        t.turn = how.steps & 1;
        number(t, [](const Item& it) { return (int64_t)it.n / 64 * (it.m / 64); });
        if (s == RF_OK) s = split ? launch<k_store<true>>(squares, 256, 0, st, t) : launch<k_store<false>>(squares, 256, 0, st, t);
        if (s != RF_OK) return s;
    }
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return rf::report_hip(e, "orthogonalisation");
    return RF_OK;
}

}  // namespace rfs

namespace {

// The C entry's table as the library's.
void convert(const rf_orthogonal_matrix* list, int64_t count, rfs::Matrix* out)
{
    for (int64_t i = 0; i < count; ++i) {
        const rf_orthogonal_matrix& m = list[i];
        out[i] = {m.in, m.out, nullptr, m.rows, m.cols, m.in_stride, m.out_stride, 0, m.dtype, m.dtype, m.dtype, m.scale, 0.0f};
    }
}

}  // namespace

extern "C" {

rf_status rf_orthogonalize_workspace(const rf_orthogonal_matrix* matrices, int32_t count, int64_t* bytes)
{
    if (!bytes) return report(RF_ERR_INVALID, "null output");
    if (count < 0 || count > 256 || (count && !matrices)) return report(RF_ERR_INVALID, "at most 256 matrices in a call");
    rfs::Matrix list[256];
    convert(matrices, count, list);
    if (const rf_status s = rfs::check(list, count, {0, nullptr, 0.0f}); s != RF_OK) return s;
    return rfs::workspace(list, count, bytes);
}

rf_status rf_orthogonalize(const rf_orthogonal_matrix* matrices, int32_t count, int32_t steps, const float* coefficients, float eps,
                           void* workspace, int64_t workspace_bytes, void* stream)
{
    if (count < 0 || count > 256 || (count && !matrices)) return report(RF_ERR_INVALID, "at most 256 matrices in a call");
    rfs::Matrix list[256];
    convert(matrices, count, list);
    const rfs::Method how{steps, coefficients, eps};
    if (const rf_status s = rfs::check(list, count, how); s != RF_OK) return s;
    int64_t need = 0;
    if (const rf_status s = rfs::workspace(list, count, &need); s != RF_OK) return s;
    if (need && (!workspace || need > workspace_bytes)) return report(RF_ERR_INVALID, "workspace too small");
    if ((uintptr_t)workspace & 255) return report(RF_ERR_INVALID, "workspace must be 256-byte aligned");
    return rfs::run(list, count, how, (char*)workspace, (hipStream_t)stream);
}

}  // extern "C"
