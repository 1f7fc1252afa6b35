// rf_norm.h -- the norms around a block: forward and backward kernels.
//
// Rows of up to 16384 columns are loaded once and kept, as loaded, in registers
// (two chunks of eight columns per lane at most, 64 to 1024 lanes a row); wider
// rows are walked again by the lanes that loaded them (k_*_wide).  What is computed
// from a row stays in registers too, except where both norms meet and a lane has
// two chunks.  There the compiler spills, registers a lane:
//   k_norm_backward        RMS/RMS   16-bit 0 to 51, f32 14 to 69
//                          LayerNorm 16-bit 36 to 120, f32 56 to 188
//   k_norm_backward_broad  RMS/RMS   16-bit 10 to 16, f32 15 to 73
//                          LayerNorm 16-bit 46 to 84, f32 53 to 179
//   k_norm_forward of 1024 lanes, LayerNorm 16-bit 37 to 85, f32 97 to 129
// The parameter vectors' gradients are sums over rows: a workgroup adds its
// own rows in registers and writes one partial row, k_norm_finish adds the
// partial rows in their order.  No atomics: the same inputs give the same bits.
//
// The gradients of the gate, the weight and the bias of the post part come
// from two column sums of a group of rows with a common gate,
//   P = sum uhat t,  Q = sum t:
//   dgate = s (w P + b Q),  dweight = s sum_groups gate P,  dbias = s sum_groups gate Q.
//
// The backward pass needs the row means of g2 xhat and of gn uhat, gn = h t
// with h = s gate w and t = e - k0 - k1 xhat, e = dhidden + rstd2 g2,
// k1 = rstd2 mean(g2 xhat), k0 = rstd2 mean(g2).  The second mean depends on
// the first through t; written out,
//   sum gn uhat = sum h e uhat - k0 sum h uhat - k1 sum h xhat uhat
//   sum gn      = sum h e      - k0 sum h      - k1 sum h xhat
// every sum is known after one walk of the row, so a row costs one exchange
// between its waves instead of two.
#pragma once

#include "rf_block.h"

namespace rfb {

constexpr int MAX_WAVES = 16;  // waves of a row

// n things dealt to `of` takers in runs; the first `more` get one more than `each`.
// (Kernels divide nothing: a 64-bit division is 140 instructions.)
struct Share {
    uint32_t each, more;
};

__host__ __device__ inline Share share_of(int64_t n, int64_t of)
{
    return {(uint32_t)(n / of), (uint32_t)(n % of)};
}

__device__ __forceinline__ int64_t first_of(const Share& s, uint32_t i) { return (int64_t)s.each * i + min(i, s.more); }

// How the rows of a pass are dealt out.
struct NormPlan {
    int32_t pieces;    // pieces of a group, each a workgroup (0: workgroups take whole groups)
    int32_t workers;   // workgroups = partial rows
    int32_t vectors;   // partial rows' vectors
    int32_t i_p, i_q, i_w2, i_b2;  // their indices, -1 absent
    int64_t group_rows;            // rows that share a gate
    int64_t groups;
    Share rows;                    // forward: a workgroup's rows; backward: a piece's rows, or a workgroup's groups
};

// Sums of NS values over the tpr lanes of a row.  `red` has two halves used
// in turn, so one barrier a call is enough: a half is written again only
// after the barrier of the call between.
template <int NS> __device__ __forceinline__ void row_sums(float (&s)[NS], float (*red)[MAX_WAVES][8], int& half)
{
#pragma unroll
    for (int k = 0; k < NS; ++k) s[k] = wave_sum(s[k]);
    const int waves = blockDim.x / WAVE;
    if (waves > 1) {
        const int w = threadIdx.x / WAVE;
        if ((threadIdx.x & (WAVE - 1)) == 0) {
#pragma unroll
            for (int k = 0; k < NS; ++k) red[half][w][k] = s[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            float t = 0.0f;
            for (int i = 0; i < waves; ++i) t += red[half][i][k];
            s[k] = t;
        }
        half ^= 1;
    }
}

__device__ __forceinline__ const void* gate_row(const rf_norm& a, int64_t g)
{
    return a.gate ? (const char*)a.gate + g * a.cols * (a.gate_dtype == RF_F32 ? 4 : 2) : nullptr;
}

// ------------------------------------------------------------- forward -----
// blockDim (tpr, ny): tpr lanes a row; ny > 1 only where a wave holds a row.
// FULL: LayerNorm or a bias somewhere.  TAIL: rows that end inside a chunk.  The
// next row's loads are sent before this row's sums.  Past the end of a row the
// elements and the vectors are zero, and so is what they give.
// Variances are taken around the mean in a second walk of the registers: a sum of
// squares alone loses the digits that a large mean shares.
// Bound by memory where there are rows enough: 16384 x 4096 bf16, post and next
// RMSNorm with both checkpoints, 132 us (5.1 TB/s).  Else by the way of one row
// through load, sums and barriers: 8192 x 768 11.5 us, 4 x 4096 with one norm 2.8,
// with both 4.8.
// LANES: 1024 for rows of more than 8192 columns.  8192 x 16384 bf16 without
// checkpoints, the next norm alone 105 us, both 212 (k_norm_forward_wide 182, 367);
// with them 132 and 253.
template <typename T, typename U, bool EXIT, bool NEXT, bool FULL, bool TAIL, int NV, int LANES>
__global__ __launch_bounds__(LANES) void k_norm_forward(const rf_norm a, const Share share, const uint32_t group_rows)
{
    __shared__ float red[2][MAX_WAVES][8];
    int half = 0;
    const int tid = threadIdx.x, tpr = blockDim.x, ty = __builtin_amdgcn_readfirstlane(threadIdx.y), ny = blockDim.y;
    const int64_t cols = a.cols, pitch = pitch_of(cols), nch = pitch / CHUNK;
    const float inv_cols = 1.0f / (float)cols;
    const int64_t r0 = first_of(share, blockIdx.x) + ty, r1 = first_of(share, blockIdx.x + 1);
    if (r0 >= r1) return;  // a wave of its own (ny > 1): no other waits for it
    int at = tid;
    struct Row {
        Raw<T> r[NV];
        Raw<U> u[EXIT ? NV : 1];
    };
    auto load = [&](int64_t r) {
        Row x;
        const T* rp = EXIT ? (const T*)a.residual + r * a.residual_stride : (const T*)a.hidden + r * a.hidden_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (int64_t)(at + j * tpr) * CHUNK;
            x.r[j] = fetch8(rp, c, cols);
            if constexpr (EXIT) x.u[j] = fetch8((const U*)a.branch + r * a.branch_stride, c, cols);
        }
        return x;
    };
    Row now = load(r0);
    const void* const some = EXIT ? a.residual : a.hidden;
    float w2[NEXT ? NV : 1][8], b2[NEXT && FULL ? NV : 1][8];
    if constexpr (NEXT) {
        Vector8 w[NV], b[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (int64_t)(at + j * tpr) * CHUNK;
            w[j].fetch(a.next_weight, a.next_weight_dtype, c, cols, some);
            if constexpr (FULL) b[j].fetch(a.next_bias, a.next_bias_dtype, c, cols, some);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (int64_t)(at + j * tpr) * CHUNK;
            w[j].template get<TAIL>(a.next_weight, a.next_weight_dtype, c, cols, 1.0f, w2[j]);
            if constexpr (FULL) b[j].template get<TAIL>(a.next_bias, a.next_bias_dtype, c, cols, 0.0f, b2[j]);
        }
    }
    // mean and 1 / sqrt(variance + eps) of a row; columns past the end are zero
    auto stats = [&](const auto& x, bool layer, float eps, float& mean, float& rstd) {
        mean = 0.0f;
        if (layer) {
            float s[1] = {0.0f};
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float v[8];
                widen8(x[j], v);
#pragma unroll
                for (int k = 0; k < 8; ++k) s[0] += v[k];
            }
            row_sums(s, red, half);
            mean = s[0] * inv_cols;
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t left = cols - (int64_t)(at + j * tpr) * CHUNK;
            float v[8], t = 0.0f;
            widen8(x[j], v);
            if (FULL && TAIL) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = k < left ? v[k] : mean;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float d = FULL ? v[k] - mean : v[k];
                t = fmaf(d, d, t);
            }
            s[0] += FULL && left <= 0 ? 0.0f : t;
        }
        row_sums(s, red, half);
        rstd = 1.0f / sqrtf(s[0] * inv_cols + eps);
    };
    for (int64_t r = r0; r < r1;) {
        // the rows of one gate
        const int64_t g = group_rows ? (uint32_t)r / group_rows : 0, end = group_rows ? min(r1, (g + 1) * group_rows) : r1;
        float A[EXIT ? NV : 1][8], B[EXIT && FULL ? NV : 1][8];
        if constexpr (EXIT) {
            Vector8 w[NV], b[NV], gt[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = (int64_t)(at + j * tpr) * CHUNK;
                w[j].fetch(a.weight, a.weight_dtype, c, cols, some);
                gt[j].fetch(gate_row(a, g), a.gate_dtype, c, cols, some);
                if constexpr (FULL) b[j].fetch(a.bias, a.bias_dtype, c, cols, some);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = (int64_t)(at + j * tpr) * CHUNK;
                float v[8];
                w[j].template get<TAIL>(a.weight, a.weight_dtype, c, cols, 1.0f, A[j]);
                gt[j].template get<TAIL>(gate_row(a, g), a.gate_dtype, c, cols, 1.0f, v);
                if constexpr (FULL) b[j].template get<TAIL>(a.bias, a.bias_dtype, c, cols, 0.0f, B[j]);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    v[k] *= a.branch_scale;
                    A[j][k] *= v[k];
                    if constexpr (FULL) B[j][k] *= v[k];
                }
            }
        }
        for (; r < end; r += ny) {
            if constexpr (LANES > 512) asm volatile("" : "+v"(at));  // 128 registers: no addresses kept from row to row
            const Row ahead = load(r + ny < r1 ? r + ny : r);  // the last row again: still cached
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = (int64_t)(at + j * tpr) * CHUNK;
                settle8<TAIL>(now.r[j], c, cols);
                if constexpr (EXIT) settle8<TAIL>(now.u[j], c, cols);
            }
            if constexpr (EXIT) {
                float mean = 0.0f, rstd = 1.0f;
                if (a.post != RF_NORM_NONE) {
                    stats(now.u, FULL && a.post == RF_NORM_LAYER, a.post_eps, mean, rstd);
                    if (tid == 0) {
                        if (a.post_rstd) a.post_rstd[r] = rstd;
                        if (a.post_mean) a.post_mean[r] = mean;
                    }
                }
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int64_t ch = at + j * tpr, c = ch * CHUNK;
                    if (ch < nch) {
                        float u[8], x[8], o[8];
                        widen8(now.u[j], u);
                        widen8(now.r[j], x);
                        if (a.branch_codes) put_codes(a.branch_codes, a.branch_exponents, r, pitch, ch, encode8(u));
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float n = FULL ? fmaf((u[k] - mean) * rstd, A[j][k], B[FULL ? j : 0][k]) : u[k] * rstd * A[j][k];
                            o[k] = fmaf(a.residual_scale, x[k], n);
                        }
                        now.r[j] = narrow8<T>(o);
                        put8<TAIL>((T*)a.hidden + r * cols + c, now.r[j], cols - c);
                    }
                }
            }
            if constexpr (NEXT) {
                float mean, rstd;
                stats(now.r, FULL && a.next == RF_NORM_LAYER, a.next_eps, mean, rstd);
                if (tid == 0) {
                    if (a.next_rstd) a.next_rstd[r] = rstd;
                    if (a.next_mean) a.next_mean[r] = mean;
                }
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int64_t ch = at + j * tpr, c = ch * CHUNK;
                    if (ch < nch) {
                        float v[8], y[8];
                        widen8(now.r[j], v);
                        if (a.hidden_codes) put_codes(a.hidden_codes, a.hidden_exponents, r, pitch, ch, encode8(v));
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            y[k] = FULL ? fmaf((v[k] - mean) * rstd, w2[j][k], b2[FULL ? j : 0][k]) : v[k] * rstd * w2[j][k];
                        }
                        const Raw<U> yr = narrow8<U>(y);
                        put8<TAIL>((U*)a.y + r * cols + c, yr, cols - c);
                        if (a.y_codes) {
                            widen8(yr, y);
                            put_codes(a.y_codes, a.y_exponents, r, pitch, ch, encode8(y));
                        }
                    }
                }
            }
            now = ahead;
        }
    }
}

// Rows wider than the register kernels take: the lanes walk their columns
// again instead of keeping them.  A lane reads back only what it wrote itself.
template <typename T, typename U, bool EXIT, bool NEXT>
__global__ __launch_bounds__(512) void k_norm_forward_wide(const rf_norm a)
{
    __shared__ float red[2][MAX_WAVES][8];
    int half = 0;
    const int tid = threadIdx.x, tpr = blockDim.x;
    const int64_t cols = a.cols, pitch = pitch_of(cols), nch = pitch / CHUNK;
    const float inv_cols = 1.0f / (float)cols;
    // mean and 1 / sqrt(variance + eps) of the row at p
    auto stats = [&](auto* p, int kind, float eps, float& mean, float& rstd) {
        mean = 0.0f;
        if (kind == RF_NORM_LAYER) {
            float s[1] = {0.0f};
            for (int64_t ch = tid; ch < nch; ch += tpr) {
                float v[8];
                widen8(load8(p, ch * CHUNK, cols), v);
#pragma unroll
                for (int k = 0; k < 8; ++k) s[0] += v[k];
            }
            row_sums(s, red, half);
            mean = s[0] * inv_cols;
        }
        float s[1] = {0.0f};
        for (int64_t ch = tid; ch < nch; ch += tpr) {
            const int64_t left = cols - ch * CHUNK;
            float v[8];
            widen8(load8(p, ch * CHUNK, cols), v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float d = k < left ? v[k] - mean : 0.0f;
                s[0] = fmaf(d, d, s[0]);
            }
        }
        row_sums(s, red, half);
        rstd = 1.0f / sqrtf(s[0] * inv_cols + eps);
    };
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int64_t g = a.gates > 1 ? r / (a.rows / a.gates) : 0;
        T* hp = (T*)a.hidden + r * (EXIT ? cols : a.hidden_stride);
        if constexpr (EXIT) {
            const U* up = (const U*)a.branch + r * a.branch_stride;
            const T* rp = (const T*)a.residual + r * a.residual_stride;
            float mean = 0.0f, rstd = 1.0f;
            if (a.post != RF_NORM_NONE) {
                stats(up, a.post, a.post_eps, mean, rstd);
                if (tid == 0) {
                    if (a.post_rstd) a.post_rstd[r] = rstd;
                    if (a.post_mean) a.post_mean[r] = mean;
                }
            }
            for (int64_t ch = tid; ch < nch; ch += tpr) {
                const int64_t c = ch * CHUNK, left = cols - c;
                float u[8], x[8], w[8], b[8], gt[8], o[8];
                widen8(load8(up, c, cols), u);
                widen8(load8(rp, c, cols), x);
                vector8(a.weight, a.weight_dtype, c, cols, 1.0f, w);
                vector8(a.bias, a.bias_dtype, c, cols, 0.0f, b);
                vector8(gate_row(a, g), a.gate_dtype, c, cols, 1.0f, gt);
                if (a.branch_codes) put_codes(a.branch_codes, a.branch_exponents, r, pitch, ch, encode8(u));
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float s = a.branch_scale * gt[k];
                    o[k] = fmaf(a.residual_scale, x[k], fmaf((u[k] - mean) * rstd, w[k] * s, b[k] * s));
                }
                put8(hp + c, narrow8<T>(o), left);
            }
        }
        if constexpr (NEXT) {
            float mean, rstd;
            stats(hp, a.next, a.next_eps, mean, rstd);
            if (tid == 0) {
                if (a.next_rstd) a.next_rstd[r] = rstd;
                if (a.next_mean) a.next_mean[r] = mean;
            }
            for (int64_t ch = tid; ch < nch; ch += tpr) {
                const int64_t c = ch * CHUNK, left = cols - c;
                float v[8], w[8], b[8], y[8];
                widen8(load8((const T*)hp, c, cols), v);
                vector8(a.next_weight, a.next_weight_dtype, c, cols, 1.0f, w);
                vector8(a.next_bias, a.next_bias_dtype, c, cols, 0.0f, b);
                if (a.hidden_codes) put_codes(a.hidden_codes, a.hidden_exponents, r, pitch, ch, encode8(v));
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = k < left ? fmaf((v[k] - mean) * rstd, w[k], b[k]) : 0.0f;
                const Raw<U> yr = narrow8<U>(y);
                put8((U*)a.y + r * cols + c, yr, left);
                if (a.y_codes) {
                    widen8(yr, y);
                    put_codes(a.y_codes, a.y_exponents, r, pitch, ch, encode8(y));
                }
            }
        }
    }
}

// ------------------------------------------------------------ backward -----
// A chunk of a saved row: of a checkpoint, or of the tensor itself.  WIDE: rows
// of at least eight columns.
template <typename T, bool SRC8, bool WIDE, bool TAIL = true> struct Saved {
    Raw<T> t;
    __device__ __forceinline__ void fetch(const T* p, int64_t stride, const int8_t*, const uint8_t*, int64_t r, int64_t,
                                          int64_t ch, int64_t, int64_t cols)
    {
        t = WIDE ? fetch8(p + r * stride, ch * CHUNK, cols) : fetch8_any(p + r * stride, ch * CHUNK, cols);
    }
    __device__ __forceinline__ void settle(int64_t ch, int64_t cols) { settle8<TAIL>(t, ch * CHUNK, cols); }
    __device__ __forceinline__ void values(float (&v)[8]) const { widen8(t, v); }
    __device__ __forceinline__ void get(float (&v)[8], int64_t ch, int64_t cols)
    {
        settle(ch, cols);
        values(v);
    }
};
template <typename T, bool WIDE, bool TAIL> struct Saved<T, true, WIDE, TAIL> {
    Codes t;
    __device__ __forceinline__ void fetch(const T*, int64_t, const int8_t* codes, const uint8_t* exps, int64_t r,
                                          int64_t pitch, int64_t ch, int64_t nch, int64_t)
    {
        t = get_codes(codes, exps, r, pitch, min(ch, nch - 1));
        if (ch >= nch) t.e = 0;  // reads as zero
    }
    __device__ __forceinline__ void settle(int64_t, int64_t) {}
    __device__ __forceinline__ void values(float (&v)[8]) const { decode8(t, v); }
    __device__ __forceinline__ void get(float (&v)[8], int64_t, int64_t) const { values(v); }
};

// Past the end of a row dy, dhidden and h are zero, so xhat and uhat may be
// anything finite there.
// FULL: LayerNorm or a bias somewhere (the sums of g, t and their columns).
// Bound by memory: 16384 x 4096 bf16, both norms, from 8 bits 158 us (4.3 TB/s; the
// chip's mix of reads and writes); small calls by the few rows that a lane has to
// hide its loads behind: 8192 x 768 15.4 us, 2317 x 1283 f32 LayerNorm 23.6.
// LayerNorms on both sides, which spill most, take 231 us for 8192 x 8192 bf16
// (RMSNorms 156) and 90 for 2048 x 5120 f32 (46).
template <typename T, typename U, bool EXIT, bool NEXT, bool FULL, bool SRC8, bool TAIL, int NV>
__global__ __launch_bounds__(512) void k_norm_backward(const rf_norm a, const NormPlan plan, float* __restrict__ partial)
{
    __shared__ float red[2][MAX_WAVES][8];
    extern __shared__ float cols_lds[];
    int half = 0;
    const int tid = threadIdx.x, tpr = blockDim.x, ty = __builtin_amdgcn_readfirstlane(threadIdx.y), ny = blockDim.y;
    const int64_t cols = a.cols, pitch = pitch_of(cols), nch = pitch / CHUNK;
    const float inv_cols = 1.0f / (float)cols;
    const bool post_layer = FULL && EXIT && a.post == RF_NORM_LAYER, next_layer = FULL && NEXT && a.next == RF_NORM_LAYER;
    const bool post_norm = EXIT && a.post != RF_NORM_NONE;
    const bool whole_groups = EXIT && plan.pieces == 0;
    float P[EXIT ? NV : 1][8] = {}, Q[EXIT && FULL ? NV : 1][8] = {};
    float W2[NEXT ? NV : 1][8] = {}, B2[NEXT && FULL ? NV : 1][8] = {};
    float h[EXIT ? NV : 1][8], w2[NEXT ? NV : 1][8];
    // This wave's (or workgroup's) rows: whole groups in a run, or every ny-th
    // row of a piece of one group.
    int64_t r0, r1, g;
    const int64_t step = whole_groups ? 1 : ny;
    if (whole_groups) {
        const int64_t ga = first_of(plan.rows, blockIdx.x), n = first_of(plan.rows, blockIdx.x + 1) - ga;
        g = ga + (ny == 4 ? n * ty / 4 : 0);
        r0 = g * plan.group_rows;
        r1 = (ga + (ny == 4 ? n * (ty + 1) / 4 : n)) * plan.group_rows;
    } else {
        const uint32_t piece = blockIdx.x % (uint32_t)plan.pieces;
        g = blockIdx.x / (uint32_t)plan.pieces;
        r0 = g * plan.group_rows + first_of(plan.rows, piece) + ty;
        r1 = g * plan.group_rows + first_of(plan.rows, piece + 1);
    }
    struct Row {
        Raw<T> dh[NV];
        Raw<U> dy[NEXT ? NV : 1];
        Saved<U, SRC8, true, TAIL> u[EXIT ? NV : 1];
        Saved<T, SRC8, true, TAIL> h[NEXT ? NV : 1];
        float rstd1, mean1, rstd2, mean2;
    };
    auto load = [&](int64_t r) {
        Row x;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t ch = tid + j * tpr, c = ch * CHUNK;
            // without one: any rows that may be read, cleared below
            x.dh[j] = fetch8(a.dhidden ? (const T*)a.dhidden + r * a.dhidden_stride : (const T*)a.dresidual + r * cols, c, cols);
            if constexpr (NEXT) {
                x.dy[j] = fetch8((const U*)a.dy + r * a.dy_stride, c, cols);
                x.h[j].fetch((const T*)a.hidden, a.hidden_stride, a.hidden_codes, a.hidden_exponents, r, pitch, ch, nch, cols);
            }
            if constexpr (EXIT)
                x.u[j].fetch((const U*)a.branch, a.branch_stride, a.branch_codes, a.branch_exponents, r, pitch, ch, nch, cols);
        }
        x.rstd1 = post_norm ? a.post_rstd[r] : 1.0f;
        x.mean1 = post_layer ? a.post_mean[r] : 0.0f;
        x.rstd2 = NEXT ? a.next_rstd[r] : 0.0f;
        x.mean2 = next_layer ? a.next_mean[r] : 0.0f;
        return x;
    };
    Row now;
    if (r0 < r1) now = load(r0);  // (a wave without rows has sums of zero)
    if constexpr (NEXT) {
        Vector8 w[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) w[j].fetch(a.next_weight, a.next_weight_dtype, (int64_t)(tid + j * tpr) * CHUNK, cols, a.dy);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            w[j].template get<TAIL>(a.next_weight, a.next_weight_dtype, (int64_t)(tid + j * tpr) * CHUNK, cols, 1.0f, w2[j]);
    }
    // whole groups: the sums over groups, of this wave's or workgroup's columns
    float* const sums_p = cols_lds + (int64_t)ty * (FULL ? 2 : 1) * pitch;
    float* const sums_q = sums_p + pitch;
    if (whole_groups) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t ch = tid + j * tpr;
            if (ch < nch) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    sums_p[ch * CHUNK + k] = 0.0f;
                    if (FULL) sums_q[ch * CHUNK + k] = 0.0f;
                }
            }
        }
    }
    for (int64_t r = r0; r < r1; ++g) {
        const int64_t end = whole_groups ? r + plan.group_rows : r1;
        if constexpr (EXIT) {
            Vector8 w[NV], gt[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = (int64_t)(tid + j * tpr) * CHUNK;
                w[j].fetch(a.weight, a.weight_dtype, c, cols, a.dbranch);
                gt[j].fetch(gate_row(a, g), a.gate_dtype, c, cols, a.dbranch);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = (int64_t)(tid + j * tpr) * CHUNK;
                float v[8];
                w[j].template get<TAIL>(a.weight, a.weight_dtype, c, cols, 1.0f, h[j]);
                gt[j].template get<TAIL>(gate_row(a, g), a.gate_dtype, c, cols, 1.0f, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) h[j][k] *= a.branch_scale * v[k];
            }
        }
        for (; r < end; r += step) {
            const Row ahead = load(r + step < r1 ? r + step : r);
            const float rstd1 = now.rstd1, mean1 = now.mean1, rstd2 = now.rstd2, mean2 = now.mean2;
            float e[NV][8], x[NEXT ? NV : 1][8], u[EXIT ? NV : 1][8];
            // g2 xhat, h e uhat, h xhat uhat; FULL: g2, h uhat, h e, h, h xhat
            float s[FULL ? 8 : 3] = {};
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t ch = tid + j * tpr;
                settle8<TAIL>(now.dh[j], ch * CHUNK, cols);
                widen8(now.dh[j], e[j]);
                if (!a.dhidden) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) e[j][k] = 0.0f;
                }
                if constexpr (NEXT) {
                    float dy[8];
                    settle8<TAIL>(now.dy[j], ch * CHUNK, cols);
                    widen8(now.dy[j], dy);
                    now.h[j].get(x[j], ch, cols);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        x[j][k] = FULL ? (x[j][k] - mean2) * rstd2 : x[j][k] * rstd2;
                        const float g2 = dy[k] * w2[j][k];
                        W2[j][k] = fmaf(dy[k], x[j][k], W2[j][k]);
                        if constexpr (FULL) {
                            B2[j][k] += dy[k];
                            s[3] += g2;
                        }
                        s[0] = fmaf(g2, x[j][k], s[0]);
                        e[j][k] = fmaf(rstd2, g2, e[j][k]);
                    }
                }
                if constexpr (EXIT) {
                    now.u[j].get(u[j], ch, cols);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        u[j][k] = FULL ? (u[j][k] - mean1) * rstd1 : u[j][k] * rstd1;
                        const float hu = h[j][k] * u[j][k];
                        s[1] = fmaf(e[j][k], hu, s[1]);
                        if constexpr (NEXT) s[2] = fmaf(x[j][k], hu, s[2]);
                        if constexpr (FULL) {
                            s[4] += hu;
                            s[5] = fmaf(h[j][k], e[j][k], s[5]);
                            s[6] += h[j][k];
                            if constexpr (NEXT) s[7] = fmaf(h[j][k], x[j][k], s[7]);
                        }
                    }
                }
            }
            row_sums(s, red, half);
            const float k1 = NEXT ? rstd2 * (s[0] * inv_cols) : 0.0f;
            float k0 = 0.0f, m1 = s[1] - k1 * s[2], m0 = 0.0f;
            if constexpr (FULL) {
                k0 = next_layer ? rstd2 * (s[3] * inv_cols) : 0.0f;
                m1 -= k0 * s[4];
                m0 = post_layer ? (s[5] - k0 * s[6] - k1 * s[7]) * inv_cols : 0.0f;
            }
            m1 = post_norm ? m1 * inv_cols : 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t ch = tid + j * tpr, c = ch * CHUNK;
                if (ch < nch) {
                    float o[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if constexpr (NEXT) e[j][k] -= fmaf(k1, x[j][k], k0);
                        o[k] = EXIT ? a.residual_scale * e[j][k] : e[j][k];
                    }
                    put8<TAIL>((T*)a.dresidual + r * cols + c, narrow8<T>(o), cols - c);
                    if constexpr (EXIT) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            P[j][k] = fmaf(u[j][k], e[j][k], P[j][k]);
                            if constexpr (FULL) Q[j][k] += e[j][k];
                            const float um = post_norm ? u[j][k] * m1 : 0.0f;  // (m1 is zero without one, u perhaps infinite)
                            o[k] = rstd1 * (FULL ? fmaf(h[j][k], e[j][k], -m0) - um : fmaf(h[j][k], e[j][k], -um));
                        }
                        put8<TAIL>((U*)a.dbranch + r * cols + c, narrow8<U>(o), cols - c);
                    }
                }
            }
            now = ahead;
        }
        if constexpr (EXIT) {
            if (whole_groups) {  // this group is complete: its gate's gradient, and its share of the sums
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int64_t ch = tid + j * tpr, c = ch * CHUNK;
                    if (ch < nch) {
                        float w[8], b[8], gt[8];
                        vector8(a.weight, a.weight_dtype, c, cols, 1.0f, w);
                        vector8(a.bias, a.bias_dtype, c, cols, 0.0f, b);
                        vector8(gate_row(a, g), a.gate_dtype, c, cols, 1.0f, gt);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float q = FULL ? Q[FULL ? j : 0][k] : 0.0f;
                            if (a.dgate && c + k < cols)
                                put_scalar(a.dgate, a.gate_dtype, g * cols + c + k,
                                           a.branch_scale * fmaf(w[k], P[j][k], b[k] * q));
                            sums_p[c + k] = fmaf(gt[k], P[j][k], sums_p[c + k]);
                            P[j][k] = 0.0f;
                            if constexpr (FULL) {
                                sums_q[c + k] = fmaf(gt[k], q, sums_q[c + k]);
                                Q[j][k] = 0.0f;
                            }
                        }
                    }
                }
            }
        }
    }
    if constexpr (EXIT) {
        if (whole_groups) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t ch = tid + j * tpr;
                if (ch < nch) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        P[j][k] = sums_p[ch * CHUNK + k];
                        if constexpr (FULL) Q[j][k] = sums_q[ch * CHUNK + k];
                    }
                }
            }
        }
    }
    // one partial row a workgroup: its waves' sums are added in their order
    float* const out = partial + (int64_t)blockIdx.x * plan.vectors * cols;
    auto finish = [&](auto& acc, int index) {
        if (index < 0) return;
        if (ny > 1) {
            for (int k = 0; k < ny; ++k) {
                __syncthreads();
                if (ty == k) {
#pragma unroll
                    for (int j = 0; j < NV; ++j) {
                        const int64_t ch = tid + j * tpr;
                        if (ch < nch) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                float* at = cols_lds + ch * CHUNK + i;
                                acc[j][i] = k ? *at + acc[j][i] : acc[j][i];
                                *at = acc[j][i];
                            }
                        }
                    }
                }
            }
        }
        if (ty == ny - 1) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t ch = tid + j * tpr, c = ch * CHUNK;
                if (ch < nch) {
                    Raw<float> v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v.a[i] = __float_as_uint(acc[j][i]);
                        v.b[i] = __float_as_uint(acc[j][i + 4]);
                    }
                    put8<TAIL>(out + index * cols + c, v, cols - c);
                }
            }
        }
    };
    if constexpr (EXIT) {
        finish(P, plan.i_p);
        if constexpr (FULL) finish(Q, plan.i_q);
    }
    if constexpr (NEXT) {
        finish(W2, plan.i_w2);
        if constexpr (FULL) finish(B2, plan.i_b2);
    }
}

// Keeps the compiler from seeing that a value is the one from before, and so from
// keeping in registers what was computed from it.
__device__ __forceinline__ void forget(Raw<float>& r) { asm volatile("" : "+v"(r.a), "+v"(r.b)); }
template <typename T> __device__ __forceinline__ void forget(Raw<T>& r) { asm volatile("" : "+v"(r.a)); }
__device__ __forceinline__ void forget(Codes& r) { asm volatile("" : "+v"(r.c), "+v"(r.e)); }

// Rows of more than 8192 columns and at most 16384, pieces of one group: two
// chunks a lane, up to 1024 lanes, so 128 registers.  They hold the row as loaded
// and the column sums; what the row's values give is computed before and after the
// row's sums, the vectors are read again for each row (they stay in the caches),
// and the next row is loaded when this one is done: a row is 100 KB and more, few
// trips to memory for what it takes to stream it.  With both norms two of the
// column sums lie in LDS: in registers they were spilled, by all CUs together more
// than the L2 caches hold.
// Bound by memory for one norm: 8192 x 16384 bf16 from 8 bits 204 us (next norm) and
// 233 (post norm; 4.1 TB/s; 775 with k_norm_backward_wide); with both norms by the
// second reading of the values too: 399 (1452 with the wide kernel, 865 with all sums
// in registers; LDS atomics instead of loads and stores 1476).  LayerNorms on both
// sides: 8192 x 12288 643 us, RMSNorms 332.
template <typename T, typename U, bool EXIT, bool NEXT, bool FULL, bool SRC8, bool TAIL>
__global__ __launch_bounds__(1024) void k_norm_backward_broad(const rf_norm a, const NormPlan plan,
                                                              float* __restrict__ partial)
{
    constexpr int NV = 2;
    constexpr bool IN_LDS = EXIT && NEXT;
    __shared__ float red[2][MAX_WAVES][8];
    extern __shared__ float cols_lds[];  // IN_LDS: P and W2, [2][NV][8][1024]
    int half = 0;
    const int tid = threadIdx.x, tpr = blockDim.x;
    const int64_t cols = a.cols, pitch = pitch_of(cols), nch = pitch / CHUNK;
    const float inv_cols = 1.0f / (float)cols;
    const bool post_layer = FULL && EXIT && a.post == RF_NORM_LAYER, next_layer = FULL && NEXT && a.next == RF_NORM_LAYER;
    const bool post_norm = EXIT && a.post != RF_NORM_NONE;
    float P[EXIT && !IN_LDS ? NV : 1][8] = {}, Q[EXIT && FULL ? NV : 1][8] = {};
    float W2[NEXT && !IN_LDS ? NV : 1][8] = {}, B2[NEXT && FULL ? NV : 1][8] = {};
    // this lane's place of vector v (0: P, 1: W2), chunk j, column k
    auto place = [&](int v, int j, int k) { return cols_lds + ((v * NV + j) * 8 + k) * 1024 + tid; };
    auto add = [&](int v, int j, int k, float x) {
        *place(v, j, k) += x;
    };
    if constexpr (IN_LDS) {
#pragma unroll
        for (int i = 0; i < 2 * NV * 8; ++i) cols_lds[i * 1024 + tid] = 0.0f;
    }
    const uint32_t piece = blockIdx.x % (uint32_t)plan.pieces;
    const int64_t g = blockIdx.x / (uint32_t)plan.pieces;
    const int64_t r0 = g * plan.group_rows + first_of(plan.rows, piece), r1 = g * plan.group_rows + first_of(plan.rows, piece + 1);
    struct Row {
        Raw<T> dh[NV];
        Raw<U> dy[NEXT ? NV : 1];
        Saved<U, SRC8, true, TAIL> u[EXIT ? NV : 1];
        Saved<T, SRC8, true, TAIL> h[NEXT ? NV : 1];
    };
    for (int64_t r = r0; r < r1; ++r) {
        // (what is computed from it is not kept from row to row)
        int at = tid;
        asm volatile("" : "+v"(at));
        Row now;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t ch = at + j * tpr, c = ch * CHUNK;
            // without one: any rows that may be read, cleared below
            now.dh[j] = fetch8(a.dhidden ? (const T*)a.dhidden + r * a.dhidden_stride : (const T*)a.dresidual + r * cols, c, cols);
            if constexpr (NEXT) {
                now.dy[j] = fetch8((const U*)a.dy + r * a.dy_stride, c, cols);
                now.h[j].fetch((const T*)a.hidden, a.hidden_stride, a.hidden_codes, a.hidden_exponents, r, pitch, ch, nch, cols);
            }
            if constexpr (EXIT)
                now.u[j].fetch((const U*)a.branch, a.branch_stride, a.branch_codes, a.branch_exponents, r, pitch, ch, nch, cols);
        }
        const float rstd1 = post_norm ? a.post_rstd[r] : 1.0f, mean1 = post_layer ? a.post_mean[r] : 0.0f;
        const float rstd2 = NEXT ? a.next_rstd[r] : 0.0f, mean2 = next_layer ? a.next_mean[r] : 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t ch = at + j * tpr;
            settle8<TAIL>(now.dh[j], ch * CHUNK, cols);
            if (!a.dhidden) now.dh[j] = Raw<T>{};
            if constexpr (NEXT) {
                settle8<TAIL>(now.dy[j], ch * CHUNK, cols);
                now.h[j].settle(ch, cols);
            }
            if constexpr (EXIT) now.u[j].settle(ch, cols);
        }
        // e = dhidden + rstd2 g2, xhat, uhat, h, dy and g2 of a chunk, one after the
        // other: the registers are full
        auto expand = [&](int j, float (&e)[8], float (&x)[8], float (&u)[8], float (&h)[8], float (&dy)[8], float (&g2)[8]) {
            const int64_t c = (int64_t)(at + j * tpr) * CHUNK;
            if constexpr (EXIT) {
                Vector8 w, gt;
                float v[8];
                w.fetch(a.weight, a.weight_dtype, c, cols, a.dbranch);
                gt.fetch(gate_row(a, g), a.gate_dtype, c, cols, a.dbranch);
                w.template get<TAIL>(a.weight, a.weight_dtype, c, cols, a.branch_scale, h);
                if (a.weight) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) h[k] *= a.branch_scale;
                }
                gt.template get<TAIL>(gate_row(a, g), a.gate_dtype, c, cols, 1.0f, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) h[k] *= v[k];
                __builtin_amdgcn_sched_barrier(0);
            }
            widen8(now.dh[j], e);
            if constexpr (NEXT) {
                Vector8 w2;
                w2.fetch(a.next_weight, a.next_weight_dtype, c, cols, a.dy);
                w2.template get<TAIL>(a.next_weight, a.next_weight_dtype, c, cols, 1.0f, g2);
                now.h[j].values(x);
                widen8(now.dy[j], dy);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[k] = FULL ? (x[k] - mean2) * rstd2 : x[k] * rstd2;
                    g2[k] *= dy[k];
                    e[k] = fmaf(rstd2, g2[k], e[k]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (EXIT) {
                now.u[j].values(u);
#pragma unroll
                for (int k = 0; k < 8; ++k) u[k] = FULL ? (u[k] - mean1) * rstd1 : u[k] * rstd1;
            }
        };
        float s[FULL ? 8 : 3] = {};  // as in k_norm_backward
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float e[8], x[8], u[8], h[8], dy[8], g2[8];
            expand(j, e, x, u, h, dy, g2);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (NEXT) {
                    s[0] = fmaf(g2[k], x[k], s[0]);
                    if constexpr (FULL) s[3] += g2[k];
                }
                if constexpr (EXIT) {
                    const float hu = h[k] * u[k];
                    s[1] = fmaf(e[k], hu, s[1]);
                    if constexpr (NEXT) s[2] = fmaf(x[k], hu, s[2]);
                    if constexpr (FULL) {
                        s[4] += hu;
                        s[5] = fmaf(h[k], e[k], s[5]);
                        s[6] += h[k];
                        if constexpr (NEXT) s[7] = fmaf(h[k], x[k], s[7]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        row_sums(s, red, half);
        const float k1 = NEXT ? rstd2 * (s[0] * inv_cols) : 0.0f;
        float k0 = 0.0f, m1 = s[1] - k1 * s[2], m0 = 0.0f;
        if constexpr (FULL) {
            k0 = next_layer ? rstd2 * (s[3] * inv_cols) : 0.0f;
            m1 -= k0 * s[4];
            m0 = post_layer ? (s[5] - k0 * s[6] - k1 * s[7]) * inv_cols : 0.0f;
        }
        m1 = post_norm ? m1 * inv_cols : 0.0f;
        asm volatile("" : "+v"(at));
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            forget(now.dh[j]);
            if constexpr (NEXT) {
                forget(now.dy[j]);
                forget(now.h[j].t);
            }
            if constexpr (EXIT) forget(now.u[j].t);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t ch = at + j * tpr, c = ch * CHUNK;
            float e[8], x[8], u[8], h[8], dy[8], g2[8], o[8];
            expand(j, e, x, u, h, dy, g2);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (NEXT) {
                    if constexpr (IN_LDS) add(1, j, k, dy[k] * x[k]);
                    else W2[j][k] = fmaf(dy[k], x[k], W2[j][k]);
                    if constexpr (FULL) B2[j][k] += dy[k];
                    e[k] -= fmaf(k1, x[k], k0);
                }
                o[k] = EXIT ? a.residual_scale * e[k] : e[k];
            }
            if (ch < nch) put8<TAIL>((T*)a.dresidual + r * cols + c, narrow8<T>(o), cols - c);
            if constexpr (EXIT) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if constexpr (IN_LDS) add(0, j, k, u[k] * e[k]);
                    else P[j][k] = fmaf(u[k], e[k], P[j][k]);
                    if constexpr (FULL) Q[j][k] += e[k];
                    const float um = post_norm ? u[k] * m1 : 0.0f;
                    o[k] = rstd1 * (FULL ? fmaf(h[k], e[k], -m0) - um : fmaf(h[k], e[k], -um));
                }
                if (ch < nch) put8<TAIL>((U*)a.dbranch + r * cols + c, narrow8<U>(o), cols - c);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    float* const out = partial + (int64_t)blockIdx.x * plan.vectors * cols;
    auto finish = [&](auto& acc, int index) {
        if (index < 0) return;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (int64_t)(tid + j * tpr) * CHUNK;
            put8<TAIL>(out + index * cols + c, narrow8<float>(acc[j]), cols - c);
        }
    };
    auto finish_lds = [&](int v, int index) {
        float acc[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[j][k] = *place(v, j, k);
        finish(acc, index);
    };
    if constexpr (EXIT) {
        if constexpr (IN_LDS) finish_lds(0, plan.i_p);
        else finish(P, plan.i_p);
        if constexpr (FULL) finish(Q, plan.i_q);
    }
    if constexpr (NEXT) {
        if constexpr (IN_LDS) finish_lds(1, plan.i_w2);
        else finish(W2, plan.i_w2);
        if constexpr (FULL) finish(B2, plan.i_b2);
    }
}

// Rows wider than the register kernels take.  A workgroup's column sums are
// its own partial row in memory, each column added to by one lane.
template <typename T, typename U, bool EXIT, bool NEXT, bool SRC8>
__global__ __launch_bounds__(512) void k_norm_backward_wide(const rf_norm a, const NormPlan plan,
                                                            float* __restrict__ partial)
{
    __shared__ float red[2][MAX_WAVES][8];
    int half = 0;
    const int tid = threadIdx.x, tpr = blockDim.x;
    const int64_t cols = a.cols, pitch = pitch_of(cols), nch = pitch / CHUNK;
    const float inv_cols = 1.0f / (float)cols;
    const bool post_layer = EXIT && a.post == RF_NORM_LAYER, next_layer = NEXT && a.next == RF_NORM_LAYER;
    const bool post_norm = EXIT && a.post != RF_NORM_NONE;
    const bool whole_groups = EXIT && plan.pieces == 0;
    float* const mine = partial + (int64_t)blockIdx.x * plan.vectors * cols;
    // whole groups: the sums of the current group, behind the partial rows
    float* const group_sums = partial + ((int64_t)plan.workers * plan.vectors + 2 * (int64_t)blockIdx.x) * cols;
    for (int64_t ch = tid; ch < nch; ch += tpr)
        for (int64_t c = ch * CHUNK; c < min(cols, (ch + 1) * CHUNK); ++c) {
            for (int v = 0; v < plan.vectors; ++v) mine[v * cols + c] = 0.0f;
            if (whole_groups) group_sums[c] = group_sums[cols + c] = 0.0f;
        }
    const int64_t g0 = whole_groups ? first_of(plan.rows, blockIdx.x) : blockIdx.x / max(plan.pieces, 1);
    const int64_t g1 = whole_groups ? first_of(plan.rows, blockIdx.x + 1) : g0 + 1;
    float* const sum_p = whole_groups ? group_sums : mine + (int64_t)max(plan.i_p, 0) * cols;
    float* const sum_q = whole_groups ? group_sums + cols : mine + (int64_t)max(plan.i_q, 0) * cols;
    const bool want_q = whole_groups || plan.i_q >= 0;
    for (int64_t g = g0; g < g1; ++g) {
        int64_t r0 = g * plan.group_rows, r1 = r0 + plan.group_rows;
        if (!whole_groups) {
            const uint32_t piece = blockIdx.x % max(plan.pieces, 1);
            r1 = r0 + first_of(plan.rows, piece + 1);
            r0 += first_of(plan.rows, piece);
        }
        for (int64_t r = r0; r < r1; ++r) {
            const float rstd1 = post_norm ? a.post_rstd[r] : 1.0f, mean1 = post_layer ? a.post_mean[r] : 0.0f;
            const float rstd2 = NEXT ? a.next_rstd[r] : 0.0f, mean2 = next_layer ? a.next_mean[r] : 0.0f;
            // e = dhidden + rstd2 g2, xhat, uhat and h of a chunk
            auto chunk = [&](int64_t ch, float (&e)[8], float (&x)[8], float (&u)[8], float (&h)[8], float (&dy)[8],
                             float (&g2)[8]) {
                const int64_t c = ch * CHUNK, left = cols - c;
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] = x[k] = u[k] = h[k] = dy[k] = g2[k] = 0.0f;
                if (a.dhidden) widen8(load8((const T*)a.dhidden + r * a.dhidden_stride, c, cols), e);
                if constexpr (NEXT) {
                    float w[8];
                    Saved<T, SRC8, false> hs;
                    hs.fetch((const T*)a.hidden, a.hidden_stride, a.hidden_codes, a.hidden_exponents, r, pitch, ch, nch, cols);
                    hs.get(x, ch, cols);
                    widen8(load8((const U*)a.dy + r * a.dy_stride, c, cols), dy);
                    vector8(a.next_weight, a.next_weight_dtype, c, cols, 1.0f, w);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        x[k] = k < left ? (x[k] - mean2) * rstd2 : 0.0f;
                        g2[k] = dy[k] * w[k];
                        e[k] = fmaf(rstd2, g2[k], e[k]);
                    }
                }
                if constexpr (EXIT) {
                    float gt[8];
                    Saved<U, SRC8, false> us;
                    us.fetch((const U*)a.branch, a.branch_stride, a.branch_codes, a.branch_exponents, r, pitch, ch, nch, cols);
                    us.get(u, ch, cols);
                    vector8(a.weight, a.weight_dtype, c, cols, 1.0f, h);
                    vector8(gate_row(a, g), a.gate_dtype, c, cols, 1.0f, gt);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        u[k] = k < left ? (u[k] - mean1) * rstd1 : 0.0f;
                        h[k] = k < left ? h[k] * a.branch_scale * gt[k] : 0.0f;
                    }
                }
            };
            float s[8] = {};
            for (int64_t ch = tid; ch < nch; ch += tpr) {
                float e[8], x[8], u[8], h[8], dy[8], g2[8];
                chunk(ch, e, x, u, h, dy, g2);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float hu = h[k] * u[k];
                    s[0] = fmaf(g2[k], x[k], s[0]);
                    s[1] = fmaf(e[k], hu, s[1]);
                    s[2] = fmaf(x[k], hu, s[2]);
                    s[3] += ch * CHUNK + k < cols ? g2[k] : 0.0f;
                    s[4] += hu;
                    s[5] = fmaf(h[k], e[k], s[5]);
                    s[6] += h[k];
                    s[7] = fmaf(h[k], x[k], s[7]);
                }
            }
            row_sums(s, red, half);
            const float k1 = rstd2 * (s[0] * inv_cols), k0 = next_layer ? rstd2 * (s[3] * inv_cols) : 0.0f;
            const float m1 = post_norm ? (s[1] - k1 * s[2] - k0 * s[4]) * inv_cols : 0.0f;
            const float m0 = post_layer ? (s[5] - k0 * s[6] - k1 * s[7]) * inv_cols : 0.0f;
            for (int64_t ch = tid; ch < nch; ch += tpr) {
                const int64_t c = ch * CHUNK;
                float e[8], x[8], u[8], h[8], dy[8], g2[8], o[8];
                chunk(ch, e, x, u, h, dy, g2);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if constexpr (NEXT) e[k] -= fmaf(k1, x[k], k0);
                    o[k] = EXIT ? a.residual_scale * e[k] : e[k];
                }
                put8((T*)a.dresidual + r * cols + c, narrow8<T>(o), cols - c);
                for (int k = 0; k < 8 && c + k < cols; ++k) {
                    if constexpr (NEXT) {
                        if (plan.i_w2 >= 0) mine[plan.i_w2 * cols + c + k] += dy[k] * x[k];
                        if (plan.i_b2 >= 0) mine[plan.i_b2 * cols + c + k] += dy[k];
                    }
                    if constexpr (EXIT) {
                        if (plan.i_p >= 0) sum_p[c + k] += u[k] * e[k];
                        if (want_q && plan.i_p >= 0) sum_q[c + k] += e[k];
                    }
                }
                if constexpr (EXIT) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) o[k] = rstd1 * (fmaf(h[k], e[k], -m0) - (post_norm ? u[k] * m1 : 0.0f));
                    put8((U*)a.dbranch + r * cols + c, narrow8<U>(o), cols - c);
                }
            }
        }
        if constexpr (EXIT) {
            if (whole_groups && plan.i_p >= 0) {
                for (int64_t ch = tid; ch < nch; ch += tpr)
                    for (int64_t c = ch * CHUNK; c < min(cols, (ch + 1) * CHUNK); ++c) {
                        const float w = a.weight ? scalar_at(a.weight, a.weight_dtype, c) : 1.0f;
                        const float b = a.bias ? scalar_at(a.bias, a.bias_dtype, c) : 0.0f;
                        const float gt = scalar_at(a.gate, a.gate_dtype, g * cols + c);
                        const float p = sum_p[c], q = sum_q[c];
                        if (a.dgate) put_scalar(a.dgate, a.gate_dtype, g * cols + c, a.branch_scale * fmaf(w, p, b * q));
                        mine[plan.i_p * cols + c] += gt * p;
                        if (plan.i_q >= 0) mine[plan.i_q * cols + c] += gt * q;
                        sum_p[c] = sum_q[c] = 0.0f;
                    }
            }
        }
    }
}

}  // namespace rfb
