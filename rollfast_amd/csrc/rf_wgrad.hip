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

constexpr int STEP = 64;              // rows t of a step: eight octets
constexpr int COL_BYTES = STEP * 2;   // LDS bytes of a column's step

typedef __attribute__((ext_vector_type(8))) bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

// LDS place of octet o of column c: two columns share 256 bytes, sixteen slots
// of 16 bytes, all banks once; column c's octet o is in slot
//   (8 c0 + o) ^ (c2 + 2 c3 + 4 (c1 ^ c4) + 8 c5)     (ci: bit i of c).
// Lanes write columns 4 l + i and read columns 16 j + l, and either way sixteen
// neighbouring lanes touch the sixteen different slots.  What a lane's own bits
// give is computed once; i, j and the half of the octets xor 4 and 8 onto it,
// so four addresses and immediate offsets reach everything.
struct Places {
    int at[4];  // by the two bits xored onto the slot, 4 and 8
};

__device__ __forceinline__ Places places(int base, int slot)
{
    Places p;
#pragma unroll
    for (int k = 0; k < 4; ++k) p.at[k] = base + ((slot ^ (4 * k)) * 16);
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

// f32 bits cut to their leading eight significant bits (Inf and NaN stay what they are).
__device__ __forceinline__ uint32_t head(uint32_t x)
{
    const uint32_t quiet = (x & 0x7FFFFFFFu) > 0x7F800000u ? 0x00400000u : 0u;
    return (x | quiet) & 0xFFFF0000u;
}

// What the head leaves: exact; nothing behind an Inf or NaN.
__device__ __forceinline__ uint32_t rest(uint32_t x, uint32_t h)
{
    const float r = __uint_as_float(x) - __uint_as_float(h);
    return (h & 0x7F800000u) == 0x7F800000u ? 0u : __float_as_uint(r);
}

// A tile of TK columns x TN outputs per workgroup, WAVES_K x WAVES_N waves.
// Steps go through two LDS buffers: while one is multiplied, the next step's
// registers are converted into the other and the loads of the step after that
// are sent.  The two waves of a SIMD do the two things in opposite order, so
// that one's conversion runs beside the other's matrix instructions.
template <typename T, int TK, int TN, int WAVES_K, int WAVES_N>
__global__ __launch_bounds__(WAVES_K* WAVES_N* WAVE) void k_wgrad(const rf_weight_grad a, float* __restrict__ partial,
                                                                 uint32_t tiles_k, uint32_t tiles, uint32_t splits)
{
    constexpr int NP = Pieces<T>::n, THREADS = WAVES_K * WAVES_N * WAVE;
    constexpr int WK = TK / WAVES_K, WN = TN / WAVES_N, FK = WK / 16, FN = WN / 16;
    constexpr int X_BYTES = TK * COL_BYTES, D_BYTES = TN * COL_BYTES, BUFFER = X_BYTES + NP * D_BYTES;
    static_assert(TK / 4 * 8 == THREADS && TN / 4 * 8 == THREADS, "a lane stages one octet of four columns of each side");
    extern __shared__ char lds[];
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const uint32_t tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
    const int64_t k0 = (int64_t)(tile % tiles_k) * TK, n0 = (int64_t)(tile / tiles_k) * TN;
    const int64_t pitch = pitch_of(a.cols), blocks = pitch / BLOCK;
    const int64_t all = (a.rows + STEP - 1) / STEP;
    const int64_t s0 = all * split / splits, s1 = all * (split + 1) / splits;

    // ---- staging: this lane's octet and its four columns on either side.
    // Columns past the end are loaded from valid places and never stored; the
    // last four of dy's row stand in for a group of columns that the row ends
    // in, shifted into place.
    const int oct = tid / (TK / 4), col = tid % (TK / 4) * 4;
    const int64_t xc = min(k0 + col, pitch - 4), dc = max(min(n0 + col, a.outs - 4), (int64_t)0);
    const bool narrow = a.outs < 4, edge = n0 + TN > a.outs && (a.outs & 3) != 0;
    const int by = (int)min(n0 + col - dc, (int64_t)3);
    const int have = (int)max(min(a.outs - (n0 + col), (int64_t)4), (int64_t)0);
    const int64_t d_pitch = a.dy_stride * (int64_t)sizeof(T);
    // bytes of this lane's first row from the step's first row (32 bits: see check())
    const uint32_t x_off = (uint32_t)(oct * 8 * pitch + xc), e_off = (uint32_t)(oct * 8 * blocks + xc / BLOCK);
    const uint32_t d_off = (uint32_t)(oct * 8 * d_pitch + dc * (int64_t)sizeof(T));
    uint32_t xr[8], er[8];
    Quad<T> dr[8];
    auto load = [&](int64_t step) {
        const char* const x = (const char*)a.codes + step * STEP * pitch;
        const char* const e = (const char*)a.exponents + step * STEP * blocks;
        const char* const d = (const char*)a.dy + step * STEP * d_pitch;
        if (step * STEP + STEP <= a.rows && !narrow) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                xr[i] = *(const uint32_t*)(x + i * pitch + x_off);
                er[i] = *(const uint8_t*)(e + i * blocks + e_off);
                dr[i] = load_quad((const T*)(d + i * d_pitch + d_off));
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 8; ++i) dr[i] = drop(dr[i], by);
            }
        } else {  // the last rows, or a row of fewer than four outputs
            const int64_t t = step * STEP + oct * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                xr[i] = er[i] = 0;
                dr[i] = Quad<T>{};
                if (t + i < a.rows) {
                    xr[i] = *(const uint32_t*)(x + i * pitch + x_off);
                    er[i] = *(const uint8_t*)(e + i * blocks + e_off);
                    dr[i] = load_some((const T*)a.dy + (t + i) * a.dy_stride + (have ? n0 + col : 0), have);
                }
            }
        }
    };
    // col is a multiple of four: bits c2 .. c5 are the lane's
    const Places put = places(col / 2 * 256, oct ^ (((col >> 2) & 3) | ((col >> 4) & 1) << 2 | ((col >> 5) & 1) << 3));
    auto stage = [&](char* buf) {
        float step[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) step[i] = __uint_as_float(er[i] << 23);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float lo = (float)(int8_t)(xr[2 * i] >> (8 * c)) * step[2 * i];
                const float hi = (float)(int8_t)(xr[2 * i + 1] >> (8 * c)) * step[2 * i + 1];
                v[i] = high_halves(__float_as_uint(lo), __float_as_uint(hi));
            }
            *(u32x4*)(buf + put.at[(c >> 1) | (c & 1) << 1] + (c >> 1) * 256) = v;
        }
        char* const d = buf + X_BYTES;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u32x4 v[NP];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (NP == 1) {
                    v[0][i] = __builtin_amdgcn_perm(dr[2 * i + 1].w[c / 2], dr[2 * i].w[c / 2],
                                                    c & 1 ? 0x07060302u : 0x05040100u);
                } else {
                    uint32_t x[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if constexpr (NP == 3) {
                            x[j] = dr[2 * i + j].w[c];
                        } else {
                            const uint16_t h = (uint16_t)(dr[2 * i + j].w[c / 2] >> (16 * (c & 1)));
                            f16 f;
                            __builtin_memcpy(&f, &h, 2);
                            x[j] = __float_as_uint((float)f);
                        }
                    }
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        const uint32_t h0 = head(x[0]), h1 = head(x[1]);
                        v[p][i] = high_halves(h0, h1);
                        if (p + 1 < NP) {
                            x[0] = rest(x[0], h0);
                            x[1] = rest(x[1], h1);
                        }
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) *(u32x4*)(d + p * D_BYTES + put.at[(c >> 1) | (c & 1) << 1] + (c >> 1) * 256) = v[p];
        }
    };

    // ---- the product: lane l holds column l % 16 of a fragment, octet l / 16
    const int wk = wave / WAVES_N * WK, wn = wave % WAVES_N * WN;
    static_assert(WK % 64 == 0 && WN % 64 == 0, "bits c4 and c5 are the fragment's number");
    const int slot = (((lane & 1) << 3) | (lane >> 4)) ^ (((lane >> 2) & 3) | ((lane >> 1) & 1) << 2);
    const Places get_x = places(wk / 2 * 256 + (lane & 15) / 2 * 256, slot);
    const Places get_d = places(X_BYTES + wn / 2 * 256 + (lane & 15) / 2 * 256, slot);
    f32x4 acc[FK][FN];
#pragma unroll
    for (int i = 0; i < FK; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](const char* buf) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            bf16x8 x[FK];
#pragma unroll
            for (int i = 0; i < FK; ++i)
                x[i] = *(const bf16x8*)(buf + get_x.at[(half ^ (i & 1)) | ((i >> 1) & 1) << 1] + i * 2048);
#pragma unroll
            for (int p = 0; p < NP; ++p) {
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    const bf16x8 y = *(const bf16x8*)(buf + get_d.at[(half ^ (j & 1)) | ((j >> 1) & 1) << 1] +
                                                      p * D_BYTES + j * 2048);
#pragma unroll
                    for (int i = 0; i < FK; ++i)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], y, acc[i][j], 0, 0, 0);
                }
            }
        }
    };

    if (s0 < s1) {
        load(s0);
        stage(lds);
        if (s0 + 1 < s1) load(s0 + 1);
        __syncthreads();
        for (int64_t s = s0; s < s1; ++s) {
            char* const now = lds + ((s - s0) & 1) * BUFFER;
            char* const next = lds + ((s - s0 + 1) & 1) * BUFFER;
            if (wave < WAVES_K * WAVES_N / 2) {
                if (s + 1 < s1) stage(next);
                if (s + 2 < s1) load(s + 2);
                multiply(now);
            } else {
                multiply(now);
                if (s + 1 < s1) stage(next);
                if (s + 2 < s1) load(s + 2);
            }
            __syncthreads();
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

Plan plan_of(const rf_weight_grad& a, int cus)
{
    Plan p{};
    auto count = [&](int64_t tk, int64_t tn) {
        p.tiles_k = (uint32_t)((a.cols + tk - 1) / tk);
        p.tiles = p.tiles_k * (uint32_t)((a.outs + tn - 1) / tn);
    };
    count(256, 256);
    p.big = a.dy_dtype == RF_BF16 && (int64_t)p.tiles * 4 >= (int64_t)cus * 3;
    if (!p.big) count(128, 128);
    // few tiles: the rows are split so that the chip is filled, four steps a split at least
    const int64_t steps = (a.rows + STEP - 1) / STEP, room = (int64_t)cus * (p.big || a.dy_dtype != RF_BF16 ? 1 : 2);
    p.splits = (uint32_t)std::max<int64_t>(1, std::min<int64_t>(steps / 4, room / p.tiles));
    p.workspace = p.splits > 1 ? (int64_t)p.splits * a.outs * a.cols * 4 : 0;
    return p;
}

template <typename T, int TK, int TN, int WK, int WN>
rf_status launch(const rf_weight_grad& a, const Plan& p, float* partial, hipStream_t st)
{
    constexpr size_t LDS = 2 * (size_t)(TK + Pieces<T>::n * TN) * COL_BYTES;
    const auto f = k_wgrad<T, TK, TN, WK, WN>;
    if (LDS > 64 * 1024) {
        static const hipError_t e = hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS);
        if (e != hipSuccess) return rf::report_hip(e, "hipFuncSetAttribute");
    }
    f<<<p.tiles * p.splits, WK * WN * WAVE, LDS, st>>>(a, partial, p.tiles_k, p.tiles, p.splits);
    return RF_OK;
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
    if (a.dy_dtype == RF_F32) s = launch<float, 128, 128, 2, 2>(a, p, partial, st);
    else if (a.dy_dtype == RF_F16) s = launch<f16, 128, 128, 2, 2>(a, p, partial, st);
    else if (p.big) s = launch<bf16, 256, 256, 2, 4>(a, p, partial, st);
    else s = launch<bf16, 128, 128, 2, 2>(a, p, partial, st);
    if (s != RF_OK) return s;
    if (p.splits > 1) {
        const int64_t grid = (a.outs * a.cols + 1023) / 1024;
        k_wgrad_join<<<(unsigned)grid, 256, 0, st>>>(a, partial, p.splits);
    }
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return rf::report_hip(e, "rf_linear_weight_grad");
    return RF_OK;
}

}  // extern "C"
