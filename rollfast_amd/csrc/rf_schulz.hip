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
// and low, 22 bits, and the term (a + B_ii) X takes both; only the product with the
// rest of B takes the high part alone, B's diagonal being kept in f32 apart.  In
// 64-bit simulation that leaves an error of 3e-4 to 9e-4 of the result's norm for
// matrices of 256 x 256 to 768 x 2304, Gaussian or close to low rank (both parts left
// out: 1.5e-2 for the latter, 1.2e-1 near rank one), beside bf16's rounding of the
// result, 1.7e-3.  Results in f32 or f16 take both parts of X, A and B everywhere, in
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
    const double* sums;
    uint16_t* buffers;
    int64_t in_stride, out_stride, add_stride;
    int32_t n, m;      // padded to whole steps
    int32_t rows, cols;
    float scale, add_scale;
    uint32_t first;    // its first tile
    uint8_t tall, in_dtype, out_dtype, add_dtype;

    // X and the next X: [n, m] high parts, then low parts.  A and B: [n, n] high
    // parts; split: then low parts.  B's diagonal [n].
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
    float a, b, c;        // the step's coefficients
    float eps, x_scale, a_scale, b_scale;
    uint32_t tiles;
    double* sums;         // [count, PARTS]
    Item item[MAX];
};
static_assert(sizeof(Batch) <= 4096, "kernel arguments");

__device__ __forceinline__ int find(const Batch& t, uint32_t id)
{
    int i = 0;
    while (i + 1 < t.count && id >= t.item[i + 1].first) ++i;
    return i;
}

__device__ __forceinline__ u32x2 narrow4(f32x4 v)
{
    const f16x2 lo = __builtin_convertvector((f32x2{v[0], v[1]}), f16x2);
    const f16x2 hi = __builtin_convertvector((f32x2{v[2], v[3]}), f16x2);
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

__device__ __forceinline__ f32x4 widen4(u32x2 w)
{
    const uint32_t first = w[0], second = w[1];  // (a vector's element has no address of its own for the cast)
    const f16x2 lo = __builtin_bit_cast(f16x2, first), hi = __builtin_bit_cast(f16x2, second);
    return f32x4{(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]};
}

// Partial sums of squares: part s of a matrix takes every PARTS-th group of rows.
__global__ __launch_bounds__(256) void k_squares(const Batch t)
{
    __shared__ double part[4];
    const Item& it = t.item[blockIdx.x / PARTS];
    const int s = blockIdx.x % PARTS, tid = threadIdx.x;
    // a workgroup's threads along a row, or several rows if they are short
    const int across = min(256, max(8, (it.cols + 7) / 8 * 8));
    const int lanes = across >= 256 ? 256 : across >= 128 ? 128 : across >= 64 ? 64 : across >= 32 ? 32 : across >= 16 ? 16 : 8;
    const int rows = 256 / lanes;
    double sum = 0;
    for (int64_t r = s * rows + tid / lanes; r < it.rows; r += PARTS * rows)
        for (int64_t c = tid % lanes; c < it.cols; c += lanes) {
            const double v = scalar_at(it.in, it.in_dtype, r * it.in_stride + c);
            sum += v * v;
        }
    for (int d = 1; d < WAVE; d *= 2) sum += __shfl_xor(sum, d);
    if (tid % WAVE == 0) part[tid / WAVE] = sum;
    __syncthreads();
    if (tid == 0) t.sums[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// G into X's layout, a tile of 64 x 64 of X a workgroup.
__global__ __launch_bounds__(256) void k_load(const Batch t)
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
    // G's rows along the wave: X's columns, or its rows if G is tall
    const int64_t r0 = it.tall ? p0 : q0, c0 = it.tall ? q0 : p0;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
        const int64_t r = r0 + tid / WAVE * 16 + i, c = c0 + lane;
        float v = 0.0f;
        if (r < it.rows && c < it.cols) v = (float)((double)scalar_at(it.in, it.in_dtype, r * it.in_stride + c) * s);
        if (it.tall) tile[lane][tid / WAVE * 16 + i] = v;
        else tile[tid / WAVE * 16 + i][lane] = v;
    }
    __syncthreads();
    const int64_t plane = (int64_t)it.n * it.m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int q = i * 16 + tid / 16, p = tid % 16 * 4;
        const f32x4 v = {tile[q][p], tile[q][p + 1], tile[q][p + 2], tile[q][p + 3]};
        const u32x2 hi = narrow4(v);
        uint16_t* const o = it.x(0) + (q0 + q) * it.m + p0 + p;
        *(u32x2*)o = hi;
        *(u32x2*)(o + plane) = narrow4(v - widen4(hi));
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

// Four neighbouring values of a row of a symmetric matrix, and where the tile is
// not on the diagonal the same values down a column.
template <bool SPLIT>
__device__ __forceinline__ void put_symmetric(uint16_t* o, int64_t n, int64_t q, int64_t p, f32x4 v, bool mirror)
{
    const u32x2 hi = narrow4(v), lo = narrow4(v - widen4(hi));
    *(u32x2*)(o + q * n + p) = hi;
    if (SPLIT) *(u32x2*)(o + n * n + q * n + p) = lo;
    if (mirror) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            o[(p + r) * n + q] = (uint16_t)(hi[r / 2] >> (16 * (r & 1)));
            if (SPLIT) o[n * n + (p + r) * n + q] = (uint16_t)(lo[r / 2] >> (16 * (r & 1)));
        }
    }
}

// SQUARE: B from A; else A from X.
template <bool SQUARE, bool SPLIT, int TILE, int WP, int WQ>
__global__ __launch_bounds__(WP* WQ* WAVE, 2) void k_symmetric(const Batch t)
{
    typedef Product<f16, KALONG, KALONG, TILE, TILE, WP, WQ> G;
    extern __shared__ char lds[];
    const uint32_t id = xcd_order(blockIdx.x, t.tiles);
    const Item& it = t.item[find(t, id)];
    const TileAt tile = lower(id - it.first);
    const int64_t n = it.n, p0 = (int64_t)tile.p * TILE, q0 = (int64_t)tile.q * TILE;
    const uint16_t* const from = SQUARE ? it.a() : it.x(t.turn);
    const int64_t depth = SQUARE ? n : it.m, plane = n * depth;
    const Side s{{from, from + (SPLIT ? plane : 0)}, depth * 2, n, n};
    typename G::Sums acc;
    G::run(lds, s, s, p0, q0, 0, depth / STEP, SPLIT ? 3 : 1, acc);
    const int lane = threadIdx.x % WAVE;
    const bool mirror = tile.p != tile.q;
    // stored A = a_scale A, X = x_scale X
    const float of_a = t.a_scale / (t.x_scale * t.x_scale);
    const float b_of = t.b * t.b_scale / t.a_scale, c_of = t.c * t.b_scale / (t.a_scale * t.a_scale);
#pragma unroll
    for (int j = 0; j < G::FQ; ++j) {
        const int64_t q = q0 + G::wq() + 16 * j + lane % 16;
        if (q >= n) continue;
#pragma unroll
        for (int i = 0; i < G::FP; ++i) {
            const int64_t p = p0 + G::wp() + 16 * i + lane / 16 * 4;
            if (p >= n) continue;
            f32x4 v = acc[i][j];
            if constexpr (SQUARE) {
                f32x4 a = widen4(*(const u32x2*)(it.a() + q * n + p));
                if (SPLIT) a += widen4(*(const u32x2*)(it.a() + n * n + q * n + p));
                v = b_of * a + c_of * v;
                if (!mirror) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (p + r == q) {
                            it.d(SPLIT)[q] = v[r] / t.b_scale;
                            v[r] = 0.0f;
                        }
                }
                put_symmetric<SPLIT>(it.b(SPLIT), n, q, p, v, mirror);
            } else {
                put_symmetric<SPLIT>(it.a(), n, q, p, v * of_a, mirror);
            }
        }
    }
}

__device__ __forceinline__ void put_out(const Item& it, int64_t r, int64_t c, float v)
{
    v *= it.scale;
    if (it.add) v += it.add_scale * scalar_at(it.add, it.add_dtype, r * it.add_stride + c);
    put_scalar(it.out, it.out_dtype, r * it.out_stride + c, v);
}

// X = (a + B_ii) X + (the rest of B) X.  LAST: to the output.
template <bool LAST, bool SPLIT, int TILE, int WP, int WQ>
__global__ __launch_bounds__(WP* WQ* WAVE, 2) void k_apply(const Batch t)
{
    typedef Product<f16, KDOWN, KALONG, TILE, TILE, WP, WQ> G;
    extern __shared__ char lds[];
    const uint32_t id = xcd_order(blockIdx.x, t.tiles);
    const Item& it = t.item[find(t, id)];
    const int64_t n = it.n, m = it.m, plane = n * m;
    const TileAt tile = tile_at(id - it.first, (uint32_t)((m + TILE - 1) / TILE), (uint32_t)((n + TILE - 1) / TILE));
    const int64_t p0 = (int64_t)tile.p * TILE, q0 = (int64_t)tile.q * TILE;
    const uint16_t* const x = it.x(t.turn);
    uint16_t* const y = it.x(!t.turn);
    const Side sx{{x, x + (SPLIT ? plane : 0)}, m * 2, m, n};
    const uint16_t* const b = it.b(SPLIT);
    const Side sb{{b, b + (SPLIT ? n * n : 0)}, n * 2, n, n};
    typename G::Sums acc;
    G::run(lds, sx, sb, p0, q0, 0, n / STEP, SPLIT ? 3 : 1, acc);
    const int lane = threadIdx.x % WAVE;
    const float of_product = 1.0f / t.b_scale, last = 1.0f / t.x_scale;
#pragma unroll
    for (int j = 0; j < G::FQ; ++j) {
        const int64_t q = q0 + G::wq() + 16 * j + lane % 16;
        if (q >= n) continue;
        const float diagonal = t.a + it.d(SPLIT)[q];
#pragma unroll
        for (int i = 0; i < G::FP; ++i) {
            const int64_t p = p0 + G::wp() + 16 * i + lane / 16 * 4;
            if (p >= m) continue;
            const int64_t at = q * m + p;
            const f32x4 old = widen4(*(const u32x2*)(x + at)) + widen4(*(const u32x2*)(x + plane + at));
            const f32x4 v = diagonal * old + of_product * acc[i][j];
            if constexpr (LAST) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t row = it.tall ? p + r : q, col = it.tall ? q : p + r;
                    if (row < it.rows && col < it.cols) put_out(it, row, col, v[r] * last);
                }
            } else {
                const u32x2 hi = narrow4(v);
                *(u32x2*)(y + at) = hi;
                *(u32x2*)(y + plane + at) = narrow4(v - widen4(hi));
            }
        }
    }
}

// Without steps: X itself.
__global__ __launch_bounds__(256) void k_copy(const Batch t)
{
    const Item& it = t.item[find(t, blockIdx.x)];
    const uint32_t id = blockIdx.x - it.first, across = it.m / 64;
    const int64_t plane = (int64_t)it.n * it.m;
    for (int i = 0; i < 16; ++i) {
        const int64_t q = id / across * 64 + threadIdx.x / 64 * 16 + i, p = id % across * 64 + threadIdx.x % 64, at = q * it.m + p;
        const int64_t row = it.tall ? p : q, col = it.tall ? q : p;
        const f16 hi = __builtin_bit_cast(f16, it.x(0)[at]), lo = __builtin_bit_cast(f16, it.x(0)[plane + at]);
        if (row < it.rows && col < it.cols) put_out(it, row, col, ((float)hi + (float)lo) / t.x_scale);
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

int64_t triangle(int64_t n, int tile) { const int64_t t = (n + tile - 1) / tile; return t * (t + 1) / 2; }

// Whether tiles of 256 (a workgroup a CU, 1.65 us for 64 k) or of 128 (two, 1.15 us)
// take less, 6 us for a round of workgroups.
template <typename F> bool large(const Batch& t, int cus, bool split, F work)
{
    double us[2];
    for (int big = 0; big < 2; ++big) {
        const int64_t room = cus * (big ? 1 : 2);
        int64_t tiles = 0, steps = 0, longest = 0;
        for (int i = 0; i < t.count; ++i) {
            const auto [n, k] = work(t.item[i], big ? 256 : 128);
            tiles += n;
            steps += n * k;
            longest = std::max<int64_t>(longest, k);
        }
        const double rounds = (double)((tiles + room - 1) / room), each = (big ? 1.65 : 1.15) * (split ? 3 : 1);
        us[big] = rounds * 6 + each * std::max((double)longest, (double)steps / (double)std::max<int64_t>(tiles, 1) * rounds);
    }
    return us[1] < us[0];
}

template <bool SQUARE, bool SPLIT> rf_status symmetric(Batch& t, int cus, hipStream_t st)
{
    typedef Product<f16, KALONG, KALONG, 256, 256, 2, 4> Big;
    typedef Product<f16, KALONG, KALONG, 128, 128, 2, 2> Small;
    struct Work { int64_t tiles, steps; };
    const bool big = large(t, cus, SPLIT, [](const Item& it, int tile) { return Work{triangle(it.n, tile), (SQUARE ? it.n : it.m) / STEP}; });
    const uint32_t grid = number(t, [&](const Item& it) { return triangle(it.n, big ? 256 : 128); });
    return big ? launch<k_symmetric<SQUARE, SPLIT, 256, 2, 4>>(grid, Big::THREADS, Big::LDS, st, t)
               : launch<k_symmetric<SQUARE, SPLIT, 128, 2, 2>>(grid, Small::THREADS, Small::LDS, st, t);
}

template <bool LAST, bool SPLIT> rf_status apply(Batch& t, int cus, hipStream_t st)
{
    typedef Product<f16, KDOWN, KALONG, 256, 256, 2, 4> Big;
    typedef Product<f16, KDOWN, KALONG, 128, 128, 2, 2> Small;
    struct Work { int64_t tiles, steps; };
    auto tiles = [](const Item& it, int tile) { return (int64_t)((it.n + tile - 1) / tile) * ((it.m + tile - 1) / tile); };
    const bool big = large(t, cus, SPLIT, [&](const Item& it, int tile) { return Work{tiles(it, tile), it.n / STEP}; });
    const uint32_t grid = number(t, [&](const Item& it) { return tiles(it, big ? 256 : 128); });
    return big ? launch<k_apply<LAST, SPLIT, 256, 2, 4>>(grid, Big::THREADS, Big::LDS, st, t)
               : launch<k_apply<LAST, SPLIT, 128, 2, 2>>(grid, Small::THREADS, Small::LDS, st, t);
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

int64_t bytes_of(const Matrix& m) { return up(item_of(m).bytes(split_of(m)), 256) + PARTS * 8; }

// The matrices from `at` on that are worked on together.
int64_t batch_end(const Matrix* list, int64_t count, int64_t at, int64_t& bytes)
{
    int64_t end = at;
    bytes = 0;
    for (; end < count && end - at < MAX; ++end) {
        const int64_t more = list[end].rows && list[end].cols ? bytes_of(list[end]) : PARTS * 8;
        if (end > at && (bytes + more > HELD || split_of(list[end]) != split_of(list[at]))) break;
        bytes += more;
    }
    return end;
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

int64_t workspace(const Matrix* list, int64_t count) noexcept
{
    int64_t most = 0;
    for (int64_t at = 0; at < count;) {
        int64_t bytes;
        at = batch_end(list, count, at, bytes);
        most = std::max(most, bytes);
    }
    return most;
}

rf_status run(const Matrix* list, int64_t count, const Method& how, char* ws, hipStream_t st, Source source, void* context) noexcept
{
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    const Bounds most = bounds_of(how);
    auto scale = [](double bound) { return (float)std::exp2(std::min(15.0, std::floor(std::log2(60000.0 / std::max(bound, 1e-3))))); };
    for (int64_t at = 0; at < count;) {
        int64_t bytes;
        const int64_t end = batch_end(list, count, at, bytes);
        const bool split = split_of(list[at]);
        Batch t{};
        t.eps = how.eps;
        t.x_scale = scale(most.x);
        t.a_scale = scale(most.x * most.x);
        t.b_scale = scale(most.b);
        t.sums = (double*)ws;
        int64_t used = (end - at) * PARTS * 8;
        int64_t which[MAX];
        float* u[MAX];
        double* sums[MAX];
        for (int64_t i = at; i < end; ++i) {
            const Matrix& m = list[i];
            if (!m.rows || !m.cols) continue;
            Item& it = t.item[t.count];
            it = item_of(m);
            it.sums = sums[t.count] = t.sums + (int64_t)t.count * PARTS;
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
        rf_status s = RF_OK;
        s = source ? source(context, which, t.count, u, sums, st) : launch<k_squares>((int64_t)t.count * PARTS, 256, 0, st, t);
        if (s != RF_OK) return s;
        const uint32_t squares = number(t, [](const Item& it) { return (int64_t)it.n / 64 * (it.m / 64); });
        s = launch<k_load>(squares, 256, 0, st, t);
        if (s != RF_OK) return s;
        if (!how.steps) s = launch<k_copy>(squares, 256, 0, st, t);
        for (int i = 0; i < how.steps && s == RF_OK; ++i) {
            t.a = how.coefficients[3 * i];
            t.b = how.coefficients[3 * i + 1];
            t.c = how.coefficients[3 * i + 2];
            t.turn = i & 1;
            const bool last = i + 1 == how.steps;
            s = split ? symmetric<false, true>(t, cus, st) : symmetric<false, false>(t, cus, st);
            if (s == RF_OK) s = split ? symmetric<true, true>(t, cus, st) : symmetric<true, false>(t, cus, st);
            if (s != RF_OK) break;
            if (split) s = last ? apply<true, true>(t, cus, st) : apply<false, true>(t, cus, st);
            else s = last ? apply<true, false>(t, cus, st) : apply<false, false>(t, cus, st);
        }
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
    *bytes = rfs::workspace(list, count);
    return RF_OK;
}

rf_status rf_orthogonalize(const rf_orthogonal_matrix* matrices, int32_t count, int32_t steps, const float* coefficients, float eps,
                           void* workspace, int64_t workspace_bytes, void* stream)
{
    if (count < 0 || count > 256 || (count && !matrices)) return report(RF_ERR_INVALID, "at most 256 matrices in a call");
    rfs::Matrix list[256];
    convert(matrices, count, list);
    const rfs::Method how{steps, coefficients, eps};
    if (const rf_status s = rfs::check(list, count, how); s != RF_OK) return s;
    const int64_t need = rfs::workspace(list, count);
    if (need && (!workspace || need > workspace_bytes)) return report(RF_ERR_INVALID, "workspace too small");
    if ((uintptr_t)workspace & 255) return report(RF_ERR_INVALID, "workspace must be 256-byte aligned");
    return rfs::run(list, count, how, (char*)workspace, (hipStream_t)stream);
}

}  // extern "C"
