// rf_product.h -- the matrix product that the vocabulary loss and the
// orthogonalisation are made of: a workgroup's tile of
//   out[q, p] = sum over k of P[p, k] Q[q, k],
// 16-bit operands, f32 sums.  What becomes of a tile is its caller's: each of
// them keeps on from the accumulators.
//
// An operand lies in memory with k along its rows (KALONG: element (x, k) at
// x * pitch + k) or with k down its columns (KDOWN: at k * pitch + x).  Both are
// loaded to LDS as they are, 16 bytes a lane without passing through registers,
// 64 k at a time.  KALONG fragments are 16-byte reads there, KDOWN ones are
// transposed by ds_read_b64_tr_b16.
//
// Two slots of 64 k suffice without a wait for what was just begun.  A step has
// two halves, `a` and `b`, of 32 k:
//   a: products of k 0 .. 31; the fragments of b are read, each into the
//      registers that its product has just left;
//   b: after two rows of products the workgroup meets.  By then every wave has
//      read all it needs of this slot, and its loads of the next step, sent a
//      whole step before, have landed.  The loads of the step after that are
//      sent into this slot, and the fragments of the next step's a are read.
#pragma once

#include <type_traits>

#include "rf_block.h"

namespace rfp {

using namespace rfb;

constexpr int STEP = 64;             // k of a step
constexpr int ROW = STEP * 2;        // LDS bytes of a KALONG row's step

typedef __attribute__((ext_vector_type(8))) bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) f16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

enum Layout { KALONG, KDOWN };

// One operand.  Two planes of the same shape, the high and the low part of a split
// tensor, or one (twice).
struct Side {
    const void* base[2];
    int64_t pitch;   // bytes, a multiple of 16 below 2^24
    int64_t extent;  // x that may be read: KDOWN at least 8 and a multiple of 8
    int64_t depth;   // KDOWN, where a product ends in half a step: rows k that may be read, at least 1
};

template <typename H> struct Eight;
template <> struct Eight<bf16> { typedef bf16x8 type; };
template <> struct Eight<f16> { typedef f16x8 type; };

__device__ __forceinline__ f32x4 multiply(bf16x8 x, bf16x8 y, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(f16x8 x, f16x8 y, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
}

// A value that all lanes hold, to scalar registers (divisions leave it in vector ones).
__device__ __forceinline__ int64_t uniform(int64_t v)
{
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// Loads straight to LDS are written in assembly, so that the compiler neither
// counts nor orders them (it would wait for all of them before each LDS read);
// the waits for them are explicit.  m0, which they set, is otherwise unused.
__device__ __forceinline__ void load_to_lds(uint32_t to, uint32_t off, const char* base)
{
    const uint32_t at = __builtin_amdgcn_readfirstlane(to);
    const char* const from = (const char*)uniform((int64_t)base);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(from) : "memory");
}

// A kernel's only argument where it lies.  Through the parameter, of which parts are
// picked at run time, the compiler would copy all of it to scratch memory and read it
// back into vector registers.
template <typename A> __device__ __forceinline__ const A& argument() { return *(const A*)__builtin_amdgcn_kernarg_segment_ptr(); }

// This lane's number, of which the compiler does not know that it never changes: it
// would work out all that follows from it ahead of a loop over tiles, and keep it in
// registers that the sums need.
__device__ __forceinline__ int own_lane()
{
    int lane = threadIdx.x % WAVE;
    asm volatile("" : "+v"(lane));
    return lane;
}

// KDOWN: 32-byte units of a row are xored by this, so that the rows of a
// transposed read lie in different banks.  (Tiles of 64: two rows fill the banks, four
// units a row.)
template <int T> __device__ __forceinline__ int unit(int k)
{
    static_assert(T >= 64, "");
    return T > 64 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
}

// A side of a tile: T of its x, staged by W waves, read by waves that hold F
// fragments of 16 x each, the first of them at x `mine`.
// RAGGED: the last step may have fewer rows k than 64 (KDOWN); its last one stands for those behind
// it, which meet zeros of the other side.
template <typename H, Layout L, int T, int W, int F, bool RAGGED> struct Staged {
    typedef typename Eight<H>::type h8;
    static constexpr int BYTES = T * ROW, N = BYTES / 1024 / W;  // loads of a wave
    static_assert(N * W * 1024 == BYTES, "whole wave loads");

    uint32_t off[N];   // this lane's 16 bytes of each load, from the step's base
    uint32_t at[2];    // LDS: this lane's part of fragment 0 of either half
    const char* base;  // the step to be loaded next
    int64_t pitch;
    int k0;            // KDOWN: row of this lane in the wave's first load
    int left;          // RAGGED: rows from the step on, or 64

    __device__ __forceinline__ void set(const Side& s, int64_t x0, int wave, int mine, int lane)
    {
        pitch = s.pitch;
        if constexpr (L == KALONG) {
#pragma unroll
            for (int j = 0; j < N; ++j) {  // eight rows of 128 bytes; their 16-byte units xored by the row
                const int64_t row = min(x0 + (wave * N + j) * 8 + lane / 8, s.extent - 1) - x0;
                off[j] = (uint32_t)(row * s.pitch) + ((lane % 8) ^ (lane / 8)) * 16;
            }
            at[0] = (mine + lane % 16) * ROW + ((lane / 16) ^ (lane & 7)) * 16;
            at[1] = at[0] ^ 64;
        } else {
            constexpr int ROWS = 512 / T, LANES = WAVE / ROWS;  // rows of a load, lanes of a row
            k0 = wave * N * ROWS + lane / LANES;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int k = k0 + j * ROWS;
                const int64_t from = min(x0 * 2 + ((lane % LANES) ^ (2 * unit<T>(k))) * 16, s.extent * 2 - 16);
                off[j] = (uint32_t)(k * s.pitch + from);
            }
            const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
            at[0] = k * (T * 2) + ((mine / 16) ^ unit<T>(k)) * 32 + (lane & 3) * 8;
            at[1] = at[0] + 32 * (T * 2);
        }
    }
    // the operand's plane from step `step` on
    __device__ __forceinline__ void seek(const Side& s, int plane, int64_t x0, int64_t step)
    {
        const char* const b = (const char*)s.base[plane];
        base = L == KALONG ? b + x0 * s.pitch + step * ROW : b + step * STEP * s.pitch;
        if (RAGGED) rows(s, step);
    }
    __device__ __forceinline__ void next(const Side& s, int64_t step)
    {
        base += L == KALONG ? (int64_t)ROW : STEP * pitch;
        if (RAGGED) rows(s, step);
    }
    __device__ __forceinline__ void rows(const Side& s, int64_t step)
    {
        left = __builtin_amdgcn_readfirstlane((int)min(s.depth - step * STEP, (int64_t)STEP));
    }
    // load j of the step at `base`
    __device__ __forceinline__ void load(uint32_t slot, int wave, int j) const
    {
        const uint32_t to = slot + (wave * N + j) * 1024;
        if constexpr (RAGGED) {
            if (left < STEP) {  // rows behind the last: that one again
                const int k = k0 + j * (512 / T), over = max(k - left + 1, 0);
                load_to_lds(to, off[j] - (uint32_t)(over * pitch), base);
                return;
            }
        }
        load_to_lds(to, off[j], base);
    }
    // fragment i of half h
    __device__ __forceinline__ h8 read(const char* slot, int h, int i) const
    {
        if constexpr (L == KALONG) {
            return *(const h8*)(slot + at[h] + i * 16 * ROW);
        } else {
            // (mine / 16 + i) ^ unit: mine / 16 is a multiple of F, i below it
            const char* const p = slot + (at[h] ^ (uint32_t)(i * 32));
            union { s16x4 half[2]; h8 v; } u;
#pragma unroll
            for (int k = 0; k < 2; ++k)  // rows k + 4: the same unit
                u.half[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_char*)(p + k * 4 * (T * 2)));
            return u.v;
        }
    }
};

// A tile of TP x TQ by WP x WQ waves.
template <typename H, Layout LP, Layout LQ, int TP, int TQ, int WP, int WQ, bool RAGGED = false> struct Product {
    static constexpr int WAVES = WP * WQ, THREADS = WAVES * WAVE;
    static constexpr int FP = TP / WP / 16, FQ = TQ / WQ / 16;  // fragments of a wave
    typedef Staged<H, LP, TP, WAVES, FP, RAGGED && LP == KDOWN> P;  // (Q's rows are whole steps)
    typedef Staged<H, LQ, TQ, WAVES, FQ, false> Q;
    typedef typename Eight<H>::type h8;
    static constexpr int SLOT = P::BYTES + Q::BYTES, LDS = 2 * SLOT;
    static_assert(LDS <= 160 * 1024, "");
    // Small tiles: the last fragment of P is read where its half begins and Q's as
    // soon as they may be, so that nothing read late in a half is waited for at the
    // next one's start, and the last two steps are copies of the loop's body without
    // loads (4096 cubed, tiles of 128: 146 -> 139 us with both operands KALONG, 172 ->
    // 139 with both KDOWN).  Large tiles have no registers for it (4 % slower).
    static constexpr int LATE = FP <= 4 ? 1 : 0;
    typedef f32x4 Sums[FP][FQ];

    // A wave's place in the tile:
    // acc[i][j][r] = out[q0 + wq + 16 j + lane % 16, p0 + wp + 16 i + lane / 16 * 4 + r]
    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE); }
    static __device__ __forceinline__ int wp(int w) { return w / WQ * (TP / WP); }
    static __device__ __forceinline__ int wq(int w) { return w % WQ * (TQ / WQ); }

    // The sums over steps s0 .. s1 - 1 of each of the plane pairs (3: high times low, low
    // times high, high times high: the small ones first, that fewer sums are rounded at
    // full size).  Ends with no load in flight.
    static __device__ __forceinline__ void run(char* lds, const Side& sp, const Side& sq, int64_t p0, int64_t q0,
                                               int64_t s0, int64_t s1, int pairs, Sums& acc)
    {
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        p0 = uniform(p0);
        q0 = uniform(q0);
        const int from = __builtin_amdgcn_readfirstlane((int)s0), to = __builtin_amdgcn_readfirstlane((int)s1);
        const int steps = (to - from) * __builtin_amdgcn_readfirstlane(pairs);
        if (steps <= 0) return;
        const int lane = own_lane(), w = wave();
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char*)lds);
        P p;
        Q q;
        p.set(sp, p0, w, wp(w), lane);
        q.set(sq, q0, w, wq(w), lane);
        int pair = 0, ahead = from;  // of the step to be loaded next
        auto seek = [&] {
            p.seek(sp, pair == 1, p0, ahead);
            q.seek(sq, pairs > 1 && pair == 0, q0, ahead);
        };
        auto next = [&] {
            ++ahead;
            if (ahead == to) {
                ahead = from;
                ++pair;
                if (pair < pairs) seek();
            } else {
                p.next(sp, ahead);
                q.next(sq, ahead);
            }
        };
        auto load = [&](uint32_t slot, int j) {
            if (j < P::N) p.load(lds0 + slot, w, j);
            else q.load(lds0 + slot + P::BYTES, w, j - P::N);
        };
        constexpr int LOADS = P::N + Q::N;
        seek();
#pragma unroll
        for (int j = 0; j < LOADS; ++j) load(0, j);
        next();
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // (also: a tile before this one may be read no more)
        if (steps > 1) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) load(SLOT, j);
            next();
        }
        h8 x[FP], y[2][FQ];
#pragma unroll
        for (int j = 0; j < FQ; ++j) y[0][j] = q.read(lds + P::BYTES, 0, j);
#pragma unroll
        for (int i = 0; i < FP - LATE; ++i) x[i] = p.read(lds, 0, i);
        constexpr int MEET = FP > 4 ? 2 : 1;  // rows of products of b before the workgroup meets
        uint32_t now = 0;
        // one of Q's fragments for each of the first rows, or two as soon as they may be read
        auto fill = [&](const char* slot, int half, int row, int rows) {
            const int from = LATE ? min(2 * row, FQ) : row * FQ / rows, to = LATE ? min(2 * row + 2, FQ) : (row + 1) * FQ / rows;
#pragma unroll
            for (int j = 0; j < FQ; ++j)
                if (j >= from && j < to) y[half][j] = q.read(slot + P::BYTES, half, j);
        };
        auto step = [&](auto more) {
            const char* const here = lds + now;
            const char* const there = lds + (now ^ SLOT);
            if (LATE) x[FP - 1] = p.read(here, 0, FP - 1);
#pragma unroll
            for (int i = 0; i < FP; ++i) {  // a
                fill(here, 1, i, FP);
#pragma unroll
                for (int j = 0; j < FQ; ++j) acc[i][j] = multiply(x[i], y[0][j], acc[i][j]);
                if (i < FP - LATE) x[i] = p.read(here, 1, i);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (LATE) x[FP - 1] = p.read(here, 1, FP - 1);
#pragma unroll
            for (int i = 0; i < FP; ++i) {  // b
                if (i == MEET) {
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < MEET; ++j) x[j] = p.read(there, 0, j);
                }
                if (i >= MEET) fill(there, 0, i - MEET, FP - MEET);
#pragma unroll
                for (int j = 0; j < FQ; ++j) acc[i][j] = multiply(x[i], y[1][j], acc[i][j]);
                if (i >= MEET) {
                    constexpr int ROWS = FP - MEET;
                    if (i < FP - LATE) x[i] = p.read(there, 0, i);
                    if (more) {
#pragma unroll
                        for (int j = (i - MEET) * LOADS / ROWS; j < (i - MEET + 1) * LOADS / ROWS; ++j) load(now, j);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (more) next();
            now ^= SLOT;
        };
        if constexpr (LATE) {
            for (int s = 2; s < steps; ++s) step(std::true_type{});
            if (steps > 1) step(std::false_type{});
            step(std::false_type{});
        } else {
            for (int s = 0; s < steps; ++s) step(s + 2 < steps);
        }
        static_assert((SLOT & (SLOT - 1)) == 0, "the slots' offsets are 0 and SLOT");
    }
};

// Of a tile's sums a lane holds four neighbours of a row (acc[i][j]), and its row's
// other three quads of those 16 lie 16, 32 and 48 lanes on.  In 16 bits two
// fragments' quads become eight neighbours of one of them: lanes of an even sixteen
// take fragment i's, those of an odd one fragment i + 1's, so that the four lanes of
// a row hold 64 bytes in order.  chunk_of() is the place of the first of them
// behind fragment i's first column; quads() takes them apart again.
__device__ __forceinline__ int chunk_of(int lane) { return (lane >> 4 & 1) * 16 + (lane >> 5) * 8; }

__device__ __forceinline__ u32x4 chunk(u32x2 first, u32x2 second)
{
    const auto a = __builtin_amdgcn_permlane16_swap(first[0], second[0], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(first[1], second[1], false, false);
    return u32x4{a[0], b[0], a[1], b[1]};
}

__device__ __forceinline__ void quads(u32x4 chunk, u32x2& first, u32x2& second)
{
    const auto a = __builtin_amdgcn_permlane16_swap(chunk[0], chunk[2], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(chunk[1], chunk[3], false, false);
    first = u32x2{a[0], b[0]};
    second = u32x2{a[1], b[1]};
}

template <typename T> __device__ __forceinline__ u32x2 narrow4(f32x4 v)
{
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 lo = __builtin_convertvector((f32x2{v[0], v[1]}), t2), hi = __builtin_convertvector((f32x2{v[2], v[3]}), t2);
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

template <typename T> __device__ __forceinline__ f32x4 widen4(u32x2 w)
{
    const uint32_t a = w[0], b = w[1];  // (a vector's element has no address of its own for the casts)
    if constexpr (__is_same(T, bf16)) {
        return f32x4{__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xFFFF0000u)};
    } else {
        const f16x2 lo = __builtin_bit_cast(f16x2, a), hi = __builtin_bit_cast(f16x2, b);
        return f32x4{(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]};
    }
}

// Workgroups go to the eight XCDs in turn.  Of every `room` of them, as many as the
// GPU holds at a time, an XCD takes neighbouring ids, which go through bands of eight
// q-tiles, q first: its workgroups share rows of both operands in its L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t block, uint32_t all, uint32_t room)
{
    const uint32_t from = block / room * room, in = block - from, here = min(room, all - from), each = here / 8;
    return from + (in < each * 8 ? in % 8 * each + in / 8 : in);
}

struct TileAt { uint32_t p, q; };

__device__ __forceinline__ TileAt tile_at(uint32_t id, uint32_t tiles_p, uint32_t tiles_q)
{
    constexpr uint32_t BAND = 8;
    const uint32_t band = id / (BAND * tiles_p), high = min(BAND, tiles_q - band * BAND);
    const uint32_t in = id - band * BAND * tiles_p;
    return {in / high, band * BAND + in % high};
}

// How a launch deals with its tiles.  Each has a workgroup; but where the last round
// of them would leave much of the GPU idle, or there is less than a round, the sums of
// its tiles are split into parts along k.  Parts go to memory, and a second launch
// (settle) adds those of a tile in their order and does what the first does with a
// whole tile's sums.  Parts are in the order of k: those that run at a time read the
// same k of both operands.
struct Share {
    uint32_t whole, rest, parts;  // tiles with a workgroup of their own, the others, parts of each of these
};

// Parts of a launch, in rooms of workgroups (with two in place of four a product of 192
// tiles of 256 stayed whole, or took tiles of 128: 3.4 ms, so 2.5); parts of a tile.
constexpr uint32_t PARTS_ROOM = 4, MOST_PARTS = 64;

// What a launch takes, in ns, measured: `step` a step of as many tiles as the GPU holds
// at a time (256 wide: one a CU, 128 wide: two, 64 wide: four), `alone` of at most one a
// CU, `ends` a tile's start and end, a part's way through memory and back, the second
// launch, and `least` what all of its operands' way from memory takes.  (With 900 and
// 10000 for the tiles of 64 and 10000 for the second launch of those of 128 lists of
// small matrices took 9 to 21 % longer, with 650 for 780 some 5 % less, others 2 % more.)
struct Cost {
    int32_t step, alone, ends, part, again;
    uint32_t alone_in;  // `alone` holds up to this part of the room
    int64_t least;
};

__host__ __device__ inline uint32_t room_of(int tile, int cus) { return (uint32_t)cus * (tile > 128 ? 1 : tile > 64 ? 2 : 4); }

__host__ __device__ inline Cost cost_of(int tile, int pairs, int ends = 0, int64_t bytes = 0)
{
    const int64_t least = bytes / 4900;  // at 4.9 TB/s
    if (tile > 128) return {1600 * pairs, 1600 * pairs, ends ? ends : 6000, 110, 10000, 2, least};
    if (tile > 64) return {1050 * pairs, 630 * pairs, ends ? ends : 4000, 28, 14000, 2, least};
    return {780 * pairs, 400 * pairs, ends ? ends : 3000, 7, 6000, 4, least};
}

// The last, incomplete round of `rest` tiles in n parts each; -1 where that is not done.
__host__ __device__ inline int64_t ns_of_rest(uint32_t rest, int64_t steps, uint32_t room, uint32_t n, const Cost& c)
{
    if (n > 1 && (n * rest > PARTS_ROOM * room || 2 * n > steps)) return -1;
    const uint32_t all = n * rest;
    const int64_t ns = (all + room - 1) / room * ((steps + n - 1) / n * (all <= room / c.alone_in ? c.alone : c.step) + c.ends);
    return (ns > c.least ? ns : c.least) + (n > 1 ? c.again + (int64_t)c.part * all : 0);
}

inline Share share_of(uint32_t tiles, int64_t steps, uint32_t room, const Cost& c)
{
    const uint32_t rest = tiles % room;
    uint32_t best = 1;
    int64_t least = ns_of_rest(rest, steps, room, 1, c);
    for (uint32_t n = 2; rest && n <= MOST_PARTS; ++n)
        if (const int64_t ns = ns_of_rest(rest, steps, room, n, c); ns >= 0 && ns < least) {
            least = ns;
            best = n;
        }
    return best == 1 ? Share{tiles, 0, 1} : Share{tiles - rest, rest, best};
}

// The same by a whole wave, a number of parts to each lane.
__device__ __forceinline__ Share share_by_wave(uint32_t tiles, int64_t steps, uint32_t room, const Cost& c)
{
    static_assert(MOST_PARTS == WAVE, "");
    const uint32_t rest = tiles % room, n = threadIdx.x % WAVE + 1;
    int64_t least = rest ? ns_of_rest(rest, steps, room, n, c) : -1;
    if (least < 0) least = 1ll << 62;
    uint32_t best = n;
    for (int d = 1; d < WAVE; d *= 2) {
        const int64_t ns = __shfl_xor(least, d);
        const uint32_t other = (uint32_t)__shfl_xor((int)best, d);
        if (ns < least || (ns == least && other < best)) {
            least = ns;
            best = other;
        }
    }
    return rest == 0 || best == 1 ? Share{tiles, 0, 1} : Share{tiles - rest, rest, best};
}

inline double ns_of(const Share& s, int64_t steps, uint32_t room, const Cost& c)
{
    return (double)((s.whole + room - 1) / room) * (double)(steps * c.step + c.ends) +
           (s.rest ? (double)ns_of_rest(s.rest, steps, room, s.parts, c) : 0.0);
}

// A job J has
//   G                  its Product
//   Args               the launch's arguments, with `room` and `partial`
//   Tile               where a tile lies, with its `steps`
//   share, tile        a batch's Share of tiles; tile number i
//   run                the tile's sums over some of its steps
//   finish             what becomes of a wave's sums
template <typename J> __device__ __forceinline__ float* part_of(const typename J::Args& a, uint32_t part)
{
    typedef typename J::G G;
    return a.partial + (int64_t)part * (G::THREADS * G::FP * G::FQ * 4);
}

template <typename J> __device__ __forceinline__ void multiply_tiles(const typename J::Args& a, char* lds)
{
    typedef typename J::G G;
    const Share sh = J::share(a);
    typename G::Sums acc;
    if (blockIdx.x < sh.whole) {
        const typename J::Tile t = J::tile(a, xcd_order(blockIdx.x, sh.whole, a.room));
        J::run(a, t, lds, 0, t.steps, acc);
        J::finish(a, t, acc, G::wave(), lds);
        return;
    }
    const uint32_t block = blockIdx.x - sh.whole, all = sh.rest * sh.parts;
    if (block >= all) return;
    const uint32_t part = xcd_order(block, all, a.room), number = part / sh.rest;
    const typename J::Tile t = J::tile(a, sh.whole + part % sh.rest);
    J::run(a, t, lds, t.steps * number / sh.parts, t.steps * (number + 1) / sh.parts, acc);
    float* const o = part_of<J>(a, part);
#pragma unroll
    for (int i = 0; i < G::FP; ++i)
#pragma unroll
        for (int j = 0; j < G::FQ; ++j) *(f32x4*)(o + ((i * G::FQ + j) * G::THREADS + threadIdx.x) * 4) = acc[i][j];
}

// A wave of a split tile to each workgroup.
template <typename J> __device__ __forceinline__ void settle_tiles(const typename J::Args& a, char* lds)
{
    typedef typename J::G G;
    const Share sh = J::share(a);
    const uint32_t which = blockIdx.x / G::WAVES;
    const int wave = blockIdx.x % G::WAVES;
    if (which >= sh.rest) return;
    const typename J::Tile t = J::tile(a, sh.whole + which);
    typename G::Sums acc;
#pragma unroll
    for (int i = 0; i < G::FP; ++i)
#pragma unroll
        for (int j = 0; j < G::FQ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // small tiles: two parts on their way at a time
#pragma unroll(G::FP <= 4 ? 2 : 1)
    for (uint32_t n = 0; n < sh.parts; ++n) {
        const float* const o = part_of<J>(a, n * sh.rest + which);
#pragma unroll
        for (int i = 0; i < G::FP; ++i)
#pragma unroll
            for (int j = 0; j < G::FQ; ++j) acc[i][j] += *(const f32x4*)(o + ((i * G::FQ + j) * G::THREADS + wave * WAVE + threadIdx.x) * 4);
    }
    J::finish(a, t, acc, wave, lds);
}

}  // namespace rfp
