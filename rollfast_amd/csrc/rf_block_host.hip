// rf_block_host.hip -- C entries of the residual-block operators: argument
// checks and launch shapes of the norms, the checkpoint and the gated
// activation kernels.
#include <algorithm>
#include <cmath>

#include "rf_norm_launch.h"

using namespace rfb;
using rf::report;

namespace {

#define BLK_TRY(call)                                          \
    do {                                                       \
        const hipError_t e_ = (call);                          \
        if (e_ != hipSuccess) return rf::report_hip(e_, #call); \
    } while (0)

bool known(int32_t dtype) { return dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Sizes whose index arithmetic stays within 62 bits.
bool sane(int64_t rows, int64_t cols) { return rows >= 0 && cols >= 1 && rows < (1ll << 31) && cols < (1ll << 28); }

rf_status bad(const char* msg) { return report(RF_ERR_INVALID, msg); }

rf_status check_kept(const int8_t* codes, const uint8_t* exps)
{
    if (!codes != !exps) return bad("codes and exponents go together");
    if (!aligned16(codes)) return bad("checkpoint codes must be 16-byte aligned");
    return RF_OK;
}

// ------------------------------------- checkpoints and gated activation ----
// Lanes lie along a row's chunks, bx of them, and over 256 / bx rows.  A lane
// takes four rows, so that several loads are in flight, where that still gives
// every CU eight workgroups, else one (1501 x 1363 f16, forward and backward of
// the gated activation: 23.4 us with four, 17.1 with one).
struct Tiles {
    int bx, by;
    bool four;
    uint32_t across;  // tiles along a row
    int64_t grid;
};

// The widest bx whose last tile wastes at most 6 % of the lanes; else the one
// that wastes least.
Tiles tiles_of(int64_t rows, int64_t nch, int cus)
{
    Tiles t{};
    double best = 1e9;
    for (int bx = 256; bx >= 4; bx /= 2) {
        const double waste = (double)((nch + bx - 1) / bx * bx) / (double)nch;
        if (waste < best - 1e-12) {
            best = waste;
            t.bx = bx;
        }
        if (waste <= 1.06) break;
    }
    t.by = 256 / t.bx;
    t.across = (uint32_t)((nch + t.bx - 1) / t.bx);
    auto grid = [&](int64_t each) { return (int64_t)t.across * ((rows + t.by * each - 1) / (t.by * each)); };
    t.four = grid(4) >= 8 * (int64_t)cus;
    t.grid = grid(t.four ? 4 : 1);
    return t;
}

struct Place {
    int64_t ch, row;
};

template <int ROWS> __device__ __forceinline__ Place place(uint32_t across)
{
    const uint32_t tile = blockIdx.x / across;
    return {(int64_t)(blockIdx.x - tile * across) * blockDim.x + threadIdx.x,
            (int64_t)tile * (blockDim.y * ROWS) + threadIdx.y};
}

// One walk: a quad of lanes has a block of 32, whose largest magnitude takes two
// exchanges in the quad.  Bound by memory: 16384 x 11008 bf16 96 us (5.7 TB/s of
// reads and writes), 3001 x 769 f32 6.2, most of it latency.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void k_checkpoint_store(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                          int64_t stride, int8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ exps, uint32_t across)
{
    const Place p = place<ROWS>(across);
    const int64_t pitch = pitch_of(cols);
    if (p.ch >= pitch / CHUNK) return;  // whole quads
    Raw<T> v[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        v[i] = fetch8_any(x + min(p.row + i * (int64_t)blockDim.y, rows - 1) * stride, p.ch * CHUNK, cols);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        float f[8];
        settle8(v[i], p.ch * CHUNK, cols);
        widen8(v[i], f);
        const Codes c = encode8(f);
        if (r < rows) put_codes(codes, exps, r, pitch, p.ch, c);
    }
}

// Bound by memory: 16384 x 11008 bf16 123 us (4.4 TB/s) where other work lies between
// store and load, as in a training step; 89 us right after the store, the codes in
// part from the last-level cache.
// STREAM: an output that the last-level cache cannot hold beside the codes is
// stored past it, so that its lines need not be written back in front of what
// comes next.  Store and load in turn, us with and without: 16384 x 11008 bf16
// 184 / 205, 16384 x 8192 122 / 149, 16384 x 11008 f32 376 / 393; smaller ones are
// left in the cache for their reader.
template <typename T, int ROWS, bool STREAM>
__global__ __launch_bounds__(256) void k_checkpoint_load(const int8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ exps, int64_t rows, int64_t cols,
                                                         T* __restrict__ out, uint32_t across)
{
    const Place p = place<ROWS>(across);
    const int64_t pitch = pitch_of(cols);
    if (p.ch >= pitch / CHUNK) return;
    Codes v[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) v[i] = get_codes(codes, exps, min(p.row + i * (int64_t)blockDim.y, rows - 1), pitch, p.ch);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        float f[8];
        decode8(v[i], f);
        if (r < rows) put8<true, STREAM>(out + r * cols + p.ch * CHUNK, narrow8<T>(f), cols - p.ch * CHUNK);
    }
}

// exp and 1 / (1 + exp(-x)).  FULL (f32 tensors): within an ulp.  Else the native
// exponential of the rounded product x log2(e), off by |x| 2^-24 of its value, and
// the native reciprocal: far below the rounding of a 16-bit result.
template <bool FULL> __device__ __forceinline__ float exponential(float x) { return FULL ? expf(x) : __expf(x); }

template <bool FULL> __device__ __forceinline__ float sigmoid(float x)
{
    const float d = 1.0f + exponential<FULL>(-x);
    return FULL ? 1.0f / d : __builtin_amdgcn_rcpf(d);
}

// a(x) and a'(x).  The tanh form is x sigmoid(2 z), z = sqrt(2 / pi) (x + 0.044715 x^3).
template <int ACT, bool FULL> __device__ __forceinline__ void activation(float x, float& a, float& slope)
{
    if constexpr (ACT == RF_ACT_SILU) {
        const float s = sigmoid<FULL>(x);
        a = x * s;
        slope = s * fmaf(x, 1.0f - s, 1.0f);
    } else if constexpr (ACT == RF_ACT_GELU) {
        const float phi = fmaf(0.5f, erff(x * 0.70710678118654752f), 0.5f);
        a = x * phi;
        slope = fmaf(x * 0.39894228040143268f, exponential<FULL>(-0.5f * x * x), phi);
    } else {
        const float x2 = x * x;
        const float s = sigmoid<FULL>(1.59576912160573071f * x * fmaf(0.044715f, x2, 1.0f));
        a = x * s;
        // from |x| = 100 on s (1 - s) is zero, beside a square that must not be infinite
        slope = fmaf(x * s * (1.0f - s), 1.59576912160573071f * fmaf(0.134145f, fminf(x2, 1e4f), 1.0f), s);
    }
}

// h = a(gate) up; the checkpoints of gate, up and (rounded) h are written in the
// same pass.  Bound by memory: 16384 x 11008 bf16 with those of gate and up 265 us
// (5.5 TB/s).
template <typename T, int ACT, int ROWS>
__global__ __launch_bounds__(256) void k_gated_forward(const rf_gated a, uint32_t across)
{
    const Place p = place<ROWS>(across);
    const int64_t pitch = pitch_of(a.cols);
    if (p.ch >= pitch / CHUNK) return;
    const int64_t c = p.ch * CHUNK, left = a.cols - c;
    Raw<T> g[ROWS], u[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = min(p.row + i * (int64_t)blockDim.y, a.rows - 1);
        g[i] = fetch8_any((const T*)a.gate + r * a.gate_stride, c, a.cols);
        u[i] = fetch8_any((const T*)a.up + r * a.up_stride, c, a.cols);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        if (r >= a.rows) break;  // the same for the whole quad
        float x[8], y[8], h[8];
        settle8(g[i], c, a.cols);
        settle8(u[i], c, a.cols);
        widen8(g[i], x);
        widen8(u[i], y);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float s;
            activation<ACT, sizeof(T) == 4>(x[k], h[k], s);
            h[k] *= y[k];
        }
        const Raw<T> hr = narrow8<T>(h);
        put8((T*)a.h + r * a.cols + c, hr, left);
        if (a.gate_codes) {
            put_codes(a.gate_codes, a.gate_exponents, r, pitch, p.ch, encode8(x));
            put_codes(a.up_codes, a.up_exponents, r, pitch, p.ch, encode8(y));
        }
        if (a.h_codes) {
            widen8(hr, h);
            if (left < CHUNK) {  // a(0) * 0 behind the last column
#pragma unroll
                for (int k = 0; k < 8; ++k) h[k] = k < left ? h[k] : 0.0f;
            }
            put_codes(a.h_codes, a.h_exponents, r, pitch, p.ch, encode8(h));
        }
    }
}

// dgate = dh up a'(gate), dup = dh a(gate), a and a' computed again from what was
// kept.  Bound by memory: 16384 x 11008 bf16 from 8 bits 260 us (5.6 TB/s).
template <typename T, int ACT, bool SRC8, int ROWS>
__global__ __launch_bounds__(256) void k_gated_backward(const rf_gated a, uint32_t across)
{
    const Place p = place<ROWS>(across);
    const int64_t pitch = pitch_of(a.cols), nch = pitch / CHUNK;
    const int64_t c = p.ch * CHUNK, left = a.cols - c;
    if (left <= 0) return;
    Raw<T> d[ROWS];
    Saved<T, SRC8, false> g[ROWS], u[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = min(p.row + i * (int64_t)blockDim.y, a.rows - 1);
        d[i] = fetch8_any((const T*)a.dh + r * a.dh_stride, c, a.cols);
        g[i].fetch((const T*)a.gate, a.gate_stride, a.gate_codes, a.gate_exponents, r, pitch, p.ch, nch, a.cols);
        u[i].fetch((const T*)a.up, a.up_stride, a.up_codes, a.up_exponents, r, pitch, p.ch, nch, a.cols);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        if (r >= a.rows) break;
        float x[8], y[8], dh[8];
        g[i].get(x, p.ch, a.cols);
        u[i].get(y, p.ch, a.cols);
        settle8(d[i], c, a.cols);
        widen8(d[i], dh);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float v, s;
            activation<ACT, sizeof(T) == 4>(x[k], v, s);
            x[k] = dh[k] * y[k] * s;
            y[k] = dh[k] * v;
        }
        put8((T*)a.dgate + r * a.dgate_stride + c, narrow8<T>(x), left);
        put8((T*)a.dup + r * a.dup_stride + c, narrow8<T>(y), left);
    }
}

template <typename T, int ACT, int ROWS> void launch_gated(const rf_gated& a, bool back, const Tiles& t, hipStream_t st)
{
    const dim3 grid((unsigned)t.grid), block(t.bx, t.by);
    if (!back) k_gated_forward<T, ACT, ROWS><<<grid, block, 0, st>>>(a, t.across);
    else if (a.gate_codes) k_gated_backward<T, ACT, true, ROWS><<<grid, block, 0, st>>>(a, t.across);
    else k_gated_backward<T, ACT, false, ROWS><<<grid, block, 0, st>>>(a, t.across);
}

template <typename T, int ACT> void launch_gated(const rf_gated& a, bool back, const Tiles& t, hipStream_t st)
{
    if (t.four) launch_gated<T, ACT, 4>(a, back, t, st);
    else launch_gated<T, ACT, 1>(a, back, t, st);
}

template <typename T> void launch_gated(const rf_gated& a, bool back, const Tiles& t, hipStream_t st)
{
    if (a.activation == RF_ACT_SILU) launch_gated<T, RF_ACT_SILU>(a, back, t, st);
    else if (a.activation == RF_ACT_GELU) launch_gated<T, RF_ACT_GELU>(a, back, t, st);
    else launch_gated<T, RF_ACT_GELU_TANH>(a, back, t, st);
}

template <typename T>
void store(const T* x, int64_t rows, int64_t cols, int64_t stride, int8_t* codes, uint8_t* exps, const Tiles& t, hipStream_t st)
{
    const dim3 grid((unsigned)t.grid), block(t.bx, t.by);
    if (t.four) k_checkpoint_store<T, 4><<<grid, block, 0, st>>>(x, rows, cols, stride, codes, exps, t.across);
    else k_checkpoint_store<T, 1><<<grid, block, 0, st>>>(x, rows, cols, stride, codes, exps, t.across);
}

template <typename T>
void load(const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, T* out, const Tiles& t, hipStream_t st)
{
    const dim3 grid((unsigned)t.grid), block(t.bx, t.by);
    constexpr int64_t CACHE = 256 << 20;  // the last-level cache
    if (t.four && rows * (cols * (int64_t)sizeof(T) + pitch_of(cols)) > CACHE)
        k_checkpoint_load<T, 4, true><<<grid, block, 0, st>>>(codes, exps, rows, cols, out, t.across);
    else if (t.four) k_checkpoint_load<T, 4, false><<<grid, block, 0, st>>>(codes, exps, rows, cols, out, t.across);
    else k_checkpoint_load<T, 1, false><<<grid, block, 0, st>>>(codes, exps, rows, cols, out, t.across);
}

rf_status check_checkpoint(const void* tensor, int32_t dtype, int64_t rows, int64_t cols, const int8_t* codes,
                           const uint8_t* exps, Tiles* t)
{
    if (!sane(rows, cols)) return bad("rows or cols out of range");
    if (!known(dtype)) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
    if (rows == 0) return RF_OK;
    if (!tensor || !codes || !exps) return bad("null buffer");
    if (const rf_status s = check_kept(codes, exps); s != RF_OK) return s;
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    *t = tiles_of(rows, pitch_of(cols) / CHUNK, cus);
    return t->grid > 0x7FFFFFFF ? report(RF_ERR_UNSUPPORTED, "too many elements for one launch") : RF_OK;
}

rf_status gated(const rf_gated* a, bool back, void* stream)
{
    if (!a) return bad("null arguments");
    if (!sane(a->rows, a->cols)) return bad("rows or cols out of range");
    if (!known(a->dtype)) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
    if (a->activation < RF_ACT_SILU || a->activation > RF_ACT_GELU_TANH) return bad("unknown activation");
    if (!a->gate_codes != !a->up_codes) return bad("gate and up are kept together");
    for (rf_status s : {check_kept(a->gate_codes, a->gate_exponents), check_kept(a->up_codes, a->up_exponents),
                        check_kept(a->h_codes, a->h_exponents)})
        if (s != RF_OK) return s;
    if (a->rows == 0) return RF_OK;
    if (back ? !a->dh || !a->dgate || !a->dup || (!a->gate_codes && (!a->gate || !a->up))
             : !a->gate || !a->up || !a->h)
        return bad("null buffer");
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    const Tiles t = tiles_of(a->rows, pitch_of(a->cols) / CHUNK, cus);
    if (t.grid > 0x7FFFFFFF) return report(RF_ERR_UNSUPPORTED, "too many elements for one launch");
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == RF_F32) launch_gated<float>(*a, back, t, st);
    else if (a->dtype == RF_BF16) launch_gated<bf16>(*a, back, t, st);
    else launch_gated<f16>(*a, back, t, st);
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

// ----------------------------------------------------------------- norms ---
constexpr int64_t MAX_REGISTER_COLS = 16384;  // 1024 lanes, two chunks each
constexpr size_t MAX_LDS = 64 * 1024;

// Lanes and chunks of a row, measured on one GPU (us):
// - one chunk a lane, or two: forward 16384 x 4096 bf16 122 / 128, 8192 x 768
//   14.3 / 13.9 (two chunks in one wave need no barrier); backward in 16 bits,
//   16384 x 4096 LayerNorm 298 / 194, 20000 x 1280 76 / 68; backward in f32,
//   2317 x 1283 LayerNorm 25 / 39 (two chunks spill).  Rows of more than 4096
//   columns have more than 512 chunks and so two a lane in every type, f32's
//   backward with its spills among them (figures in rf_norm.h).
// - threads a CU: forward 16384 x 4096 157 / 122 / 126 with 512 / 1024 / 2048;
//   backward 158 / 173 with 512 / 768 (more partial rows to write and add);
//   forward 2317 x 1283 f32 18.3 with 1365 workgroups of 192, which do not fit
//   at once, 16.6 with 1280, five on every CU.
NormShape shape_of(const rf_norm& a, int cus, bool back)
{
    NormShape s{};
    const int64_t nch = pitch_of(a.cols) / CHUNK;
    const bool two = nch > 512 || (nch > 64 && (back ? a.dtype != RF_F32 : nch <= 128));
    const int64_t lanes = two ? (nch + 1) / 2 : nch;
    s.tpr = (int)std::min<int64_t>(1024, (lanes + 63) / 64 * 64);
    s.nv = a.cols > MAX_REGISTER_COLS || a.cols < CHUNK ? 0 : two ? 2 : 1;
    if (s.nv == 0) s.tpr = 512;
    s.ny = s.tpr == 64 && s.nv ? 4 : 1;
    s.full = a.post == RF_NORM_LAYER || a.next == RF_NORM_LAYER ||
             (back ? a.dbias || a.dnext_bias || (a.bias && a.dgate) : a.bias || a.next_bias);
    s.src8 = a.post == RF_NORM_ABSENT ? a.hidden_codes != nullptr : a.branch_codes != nullptr;
    s.workers = std::max<int64_t>(1, std::min<int64_t>((a.rows + s.ny - 1) / s.ny, (int64_t)cus * (1024 / (s.tpr * s.ny))));
    if (s.nv == 0) s.workers = std::max<int64_t>(1, std::min<int64_t>(a.rows, (int64_t)cus * 4));
    return s;
}

// Rows are cut into pieces of a group, about 512 threads a CU, and two rows a wave
// or workgroup at least, where that gives every CU a piece, else one (196 x 15296
// f16 28.7 us with one, 31.0 with two, 38.8 with four; 300 x 768 LayerNorms 18.2, 21.0,
// 23.8; 2048 x 1024 RMSNorms 18.4, 17.0, 19.1); with more groups than pieces a workgroup takes whole groups.
// Workgroups come in whole rounds of the CUs where there are more than one:
// 2317 x 1283 LayerNorm in f32 took 25 us with 512 of them and 36 with 574.
void plan_of(const rf_norm& a, int cus, NormShape& s, NormPlan& p)
{
    p = NormPlan{};
    const bool exit = a.post != RF_NORM_ABSENT;
    const int64_t target = (int64_t)cus * std::max(1, 512 / (s.tpr * s.ny));
    p.groups = exit ? std::max<int64_t>(1, a.gates) : 1;
    p.group_rows = a.rows / p.groups;
    if (p.groups > target) {
        p.pieces = 0;
        p.workers = (int32_t)target;
    } else {
        int64_t all = std::min<int64_t>(std::max<int64_t>(1, a.rows / s.ny), std::max<int64_t>(cus, a.rows / (2 * s.ny)));
        all = std::min(target, all);
        if (all > cus) all = all / cus * cus;
        p.pieces = (int32_t)std::max<int64_t>(1, all / p.groups);
        p.workers = (int32_t)(p.pieces * p.groups);
    }
    p.rows = p.pieces ? share_of(p.group_rows, p.pieces) : share_of(p.groups, p.workers);
    int n = 0;
    p.i_p = exit && (a.dweight || a.dbias || a.dgate) ? n++ : -1;
    p.i_q = exit && (a.dbias || (a.dgate && a.bias)) ? n++ : -1;
    p.i_w2 = a.next != RF_NORM_ABSENT && a.dnext_weight ? n++ : -1;
    p.i_b2 = a.next != RF_NORM_ABSENT && a.dnext_bias ? n++ : -1;
    p.vectors = n;
    const int64_t pitch = pitch_of(a.cols);
    s.lds = s.ny > 1 ? pitch * sizeof(float) : 0;
    if (p.pieces == 0) s.lds = (size_t)s.ny * (s.full ? 2 : 1) * pitch * sizeof(float);
    // (the broad kernel takes pieces of one group only)
    if (s.lds > MAX_LDS - 2048 || (p.pieces == 0 && s.tpr > 512)) s.nv = 0, s.ny = 1, s.tpr = 512, s.lds = 0;
}

int64_t workspace_of(const rf_norm& a, const NormShape& s, const NormPlan& p)
{
    int64_t n = (int64_t)p.workers * p.vectors * a.cols;
    if (s.nv == 0 && p.pieces == 0) n += (int64_t)p.workers * 2 * a.cols;
    return n * (int64_t)sizeof(float);
}

// Adds the partial rows: 32 columns a workgroup (a cache line of a row), 32 lanes
// a column.  The lanes are dealt to the groups of rows (all of them to one group,
// or one to each of 32 groups at a time), and within a group to its pieces.
// blockIdx.y: 0 the next norm's vectors, 1 the post norm's and the gate (not
// launched without).
// Bound by what a CU has on the way to memory, since few take part: 512 partial
// rows of 4096 columns and two vectors 7.3 us (2.3 TB/s), of 768 columns and one
// 4.4.  16 columns and 64 lanes, twice the workgroups with half a line each: 14.1 us
// and 5.0.
constexpr int FIN_COLS = 32, FIN_LANES = 32;

// Sums of partial rows w0 + i * step below w1, of vectors p and, not null, q;
// sixteen rows' loads in flight (512 rows are one round).
struct Pair {
    float p, q;
};

__device__ __forceinline__ Pair add_rows(const float* p, const float* q, int64_t w0, int64_t w1, int64_t step, int64_t pitch)
{
    constexpr int N = 16;
    Pair s = {0.0f, 0.0f};
    for (int64_t w = w0; w < w1; w += N * step) {
        float v[N], u[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t at = min(w + i * step, w1 - 1) * pitch;  // (loads without a condition do not wait for another)
            v[i] = p ? p[at] : 0.0f;
            u[i] = q ? q[at] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s.p += w + i * step < w1 ? v[i] : 0.0f;
            s.q += w + i * step < w1 ? u[i] : 0.0f;
        }
    }
    return s;
}

__global__ __launch_bounds__(FIN_COLS* FIN_LANES) void k_norm_finish(const rf_norm a, const NormPlan p,
                                                                    const float* __restrict__ partial)
{
    __shared__ float lds[4][FIN_LANES][FIN_COLS];
    const int tx = threadIdx.x, ty = threadIdx.y;
    const int64_t cols = a.cols, c = (int64_t)blockIdx.x * FIN_COLS + tx, at = min(c, cols - 1), pitch = p.vectors * cols;
    const bool in = c < cols;
    const bool has_q = p.i_q >= 0;
    // whole groups: the gate is in the sums already, and its gradient is written
    const bool gated = p.pieces > 0 && a.gate;
    const int64_t groups = p.pieces > 0 ? p.groups : 1, pieces = p.pieces > 0 ? p.pieces : p.workers;
    const int lanes = (int)max((int64_t)1, FIN_LANES / groups), slots = FIN_LANES / lanes;
    const int slot = ty / lanes, sub = ty % lanes;
    if (blockIdx.y == 0) {  // the next norm's vectors
        const Pair v = add_rows(p.i_w2 >= 0 ? partial + p.i_w2 * cols + at : nullptr,
                                p.i_b2 >= 0 ? partial + p.i_b2 * cols + at : nullptr, ty, p.workers, FIN_LANES, pitch);
        lds[0][ty][tx] = v.p;
        lds[1][ty][tx] = v.q;
        __syncthreads();
        void* const out = ty == 0 ? a.dnext_weight : a.dnext_bias;
        if (ty < 2 && in && out) {
            float s = 0.0f;
            for (int i = 0; i < FIN_LANES; ++i) s += lds[ty][i][tx];
            put_scalar(out, ty == 0 ? a.next_weight_dtype : a.next_bias_dtype, c, s);
        }
        return;
    }
    const float w = a.weight ? scalar_at(a.weight, a.weight_dtype, at) : 1.0f;
    const float b = a.bias ? scalar_at(a.bias, a.bias_dtype, at) : 0.0f;
    float dw = 0.0f, db = 0.0f;
    // a group's sums are there: its gate's gradient, and its part of the vectors'
    auto add_group = [&](int64_t g, float gt, float P, float Q) {
        if (gated && a.dgate && in) put_scalar(a.dgate, a.gate_dtype, g * cols + c, a.branch_scale * fmaf(w, P, b * Q));
        dw = fmaf(gt, P, dw);
        db = fmaf(gt, Q, db);
    };
    // More groups than half the lanes: a lane takes every FIN_LANES-th of them, their
    // pieces in one run, eight on their way at a time.  382 groups of 99 columns 10.0 us,
    // 66 of 391 5.4 (36.3 and 9.8 by the loop below, with a trip to memory and two
    // barriers for each FIN_LANES groups).
    const int64_t run = lanes > 1 ? 0 : (groups + FIN_LANES - 1) / FIN_LANES * pieces;
    const int64_t last = max(p.workers - 1, 0);
    float P = 0.0f, Q = 0.0f;
    for (int64_t e0 = 0, k = 0, piece = 0; e0 < run; e0 += 8) {
        float v[8], u[8];
        uint16_t lo[8], hi[8];  // the gates', as they are stored
        int64_t kk = k, pp = piece;
        const int halves = gated && a.gate_dtype == RF_F32 ? 2 : 1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t g = min(ty + kk * FIN_LANES, groups - 1), row = min(g * pieces + pp, last) * pitch;
            v[i] = partial[row + p.i_p * cols + at];
            u[i] = has_q ? partial[row + p.i_q * cols + at] : 0.0f;
            const uint16_t* const gp = gated ? (const uint16_t*)a.gate + (g * cols + at) * halves : (const uint16_t*)partial;
            lo[i] = gp[0];
            hi[i] = gp[halves - 1];
            if (++pp == pieces) pp = 0, ++kk;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t g = ty + k * FIN_LANES;
            P += p.workers ? v[i] : 0.0f;  // (no rows: nothing has been written)
            Q += p.workers ? u[i] : 0.0f;
            if (++piece == pieces) {
                const float gt = !gated ? 1.0f
                                 : a.gate_dtype == RF_F16
                                     ? (float)__builtin_bit_cast(f16, hi[i])
                                     : __uint_as_float((uint32_t)hi[i] << 16 | (halves == 2 ? lo[i] : 0u));
                if (g < groups && e0 + i < run) add_group(g, gt, P, Q);
                P = Q = 0.0f;
                piece = 0;
                ++k;
            }
        }
    }
    for (int64_t first = 0; first < groups && lanes > 1; first += slots) {
        const int64_t g = first + slot, w0 = g * pieces;
        const bool mine = slot < slots && g < groups;
        const int64_t w1 = mine ? min(w0 + pieces, (int64_t)p.workers) : 0;
        const Pair v = add_rows(partial + p.i_p * cols + at, has_q ? partial + p.i_q * cols + at : nullptr, w0 + sub, w1, lanes,
                                pitch);
        lds[2][ty][tx] = v.p;
        lds[3][ty][tx] = v.q;
        __syncthreads();
        if (mine && sub == 0) {
            P = Q = 0.0f;
            for (int i = 0; i < lanes; ++i) {
                P += lds[2][ty + i][tx];
                Q += lds[3][ty + i][tx];
            }
            add_group(g, gated ? scalar_at(a.gate, a.gate_dtype, g * cols + at) : 1.0f, P, Q);
        }
        __syncthreads();
    }
    lds[2][ty][tx] = dw;
    lds[3][ty][tx] = db;
    __syncthreads();
    void* const out = ty == 0 ? a.dweight : a.dbias;
    if (ty >= 2 || !in || !out) return;
    float s = 0.0f;
    for (int i = 0; i < FIN_LANES; ++i) s += lds[2 + ty][i][tx];
    put_scalar(out, ty == 0 ? a.weight_dtype : a.bias_dtype, c, a.branch_scale * s);
}

bool has_pair(const rf_norm& a)
{
    return known(a.dtype) && known(a.branch_dtype) && (a.dtype == a.branch_dtype || a.dtype == RF_F32);
}

rf_status check_norm(const rf_norm* a)
{
    if (!a) return bad("null arguments");
    if (!sane(a->rows, a->cols)) return bad("rows or cols out of range");
    if (a->post < RF_NORM_ABSENT || a->post > RF_NORM_LAYER) return bad("unknown post norm");
    if (a->next != RF_NORM_ABSENT && a->next != RF_NORM_RMS && a->next != RF_NORM_LAYER) return bad("unknown next norm");
    if ((a->post >= RF_NORM_RMS && !(a->post_eps >= 0.0f)) || (a->next >= RF_NORM_RMS && !(a->next_eps >= 0.0f)))
        return bad("eps must not be negative");
    if (a->post == RF_NORM_ABSENT && a->next == RF_NORM_ABSENT) return bad("neither a post norm nor a next norm");
    if (!has_pair(*a))
        return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16, and the branch's the same or 16-bit beside f32");
    const struct { const void* p; int32_t dtype; } vectors[] = {
        {a->weight, a->weight_dtype}, {a->bias, a->bias_dtype}, {a->gate, a->gate_dtype},
        {a->next_weight, a->next_weight_dtype}, {a->next_bias, a->next_bias_dtype}};
    for (const auto& v : vectors)
        if (v.p && !known(v.dtype)) return report(RF_ERR_UNSUPPORTED, "a vector's dtype must be f32, bf16 or f16");
    if (a->gates < 0 || (a->gates > 0 && (a->rows % a->gates || !a->gate)) || (a->gates == 0 && a->gate))
        return bad("gates must divide the rows and come with a gate");
    if (a->post == RF_NORM_ABSENT && (a->gates || a->weight || a->bias)) return bad("a gate or weight without a post norm");
    if (a->post == RF_NORM_NONE && (a->weight || a->bias)) return bad("a weight or bias without a norm");
    for (rf_status s : {check_kept(a->branch_codes, a->branch_exponents), check_kept(a->hidden_codes, a->hidden_exponents),
                        check_kept(a->y_codes, a->y_exponents)})
        if (s != RF_OK) return s;
    return RF_OK;
}

rf_status check_backward(const rf_norm* a)
{
    if (const rf_status s = check_norm(a); s != RF_OK) return s;
    const bool exit = a->post != RF_NORM_ABSENT, next = a->next != RF_NORM_ABSENT;
    if (exit && next && !a->branch_codes != !a->hidden_codes) return bad("both rows are kept in 8 bits, or neither");
    if ((a->dweight && !a->weight) || (a->dbias && !a->bias) || (a->dgate && !a->gate) ||
        (a->dnext_weight && !a->next_weight) || (a->dnext_bias && !a->next_bias))
        return bad("a gradient of an absent vector");
    return RF_OK;
}

using forward_t = void (*)(const rf_norm&, const NormShape&, hipStream_t);
using backward_t = rf_status (*)(const rf_norm&, const NormShape&, const NormPlan&, float*, hipStream_t);

forward_t forward_of(const rf_norm& a)
{
    if (a.dtype == RF_BF16) return norm_forward_1_1;
    if (a.dtype == RF_F16) return norm_forward_2_2;
    return a.branch_dtype == RF_F32 ? norm_forward_0_0 : a.branch_dtype == RF_BF16 ? norm_forward_0_1 : norm_forward_0_2;
}

backward_t backward_of(const rf_norm& a)
{
    if (a.dtype == RF_BF16) return norm_backward_1_1;
    if (a.dtype == RF_F16) return norm_backward_2_2;
    return a.branch_dtype == RF_F32 ? norm_backward_0_0 : a.branch_dtype == RF_BF16 ? norm_backward_0_1 : norm_backward_0_2;
}

}  // namespace

extern "C" {

rf_status rf_checkpoint_store(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride,
                              int8_t* codes, uint8_t* exponents, void* stream)
{
    Tiles t;
    if (const rf_status s = check_checkpoint(x, dtype, rows, cols, codes, exponents, &t); s != RF_OK || rows == 0) return s;
    if (dtype == RF_F32) store((const float*)x, rows, cols, row_stride, codes, exponents, t, (hipStream_t)stream);
    else if (dtype == RF_BF16) store((const bf16*)x, rows, cols, row_stride, codes, exponents, t, (hipStream_t)stream);
    else store((const f16*)x, rows, cols, row_stride, codes, exponents, t, (hipStream_t)stream);
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

rf_status rf_checkpoint_load(const int8_t* codes, const uint8_t* exponents, int64_t rows, int64_t cols, int32_t dtype,
                             void* out, void* stream)
{
    Tiles t;
    if (const rf_status s = check_checkpoint(out, dtype, rows, cols, codes, exponents, &t); s != RF_OK || rows == 0) return s;
    if (dtype == RF_F32) load(codes, exponents, rows, cols, (float*)out, t, (hipStream_t)stream);
    else if (dtype == RF_BF16) load(codes, exponents, rows, cols, (bf16*)out, t, (hipStream_t)stream);
    else load(codes, exponents, rows, cols, (f16*)out, t, (hipStream_t)stream);
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

rf_status rf_gated_forward(const rf_gated* args, void* stream) { return gated(args, false, stream); }

rf_status rf_gated_backward(const rf_gated* args, void* stream) { return gated(args, true, stream); }

rf_status rf_norm_forward(const rf_norm* args, void* stream)
{
    if (const rf_status s = check_norm(args); s != RF_OK) return s;
    const rf_norm& a = *args;
    const bool exit = a.post != RF_NORM_ABSENT, next = a.next != RF_NORM_ABSENT;
    if (a.rows == 0) return RF_OK;
    if (!a.hidden || (exit && (!a.residual || !a.branch)) || (next && !a.y)) return bad("null buffer");
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    forward_of(a)(a, shape_of(a, cus, false), (hipStream_t)stream);
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

rf_status rf_norm_backward_workspace(const rf_norm* args, int64_t* bytes)
{
    if (!bytes) return bad("null output");
    if (const rf_status s = check_backward(args); s != RF_OK) return s;
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    NormShape s = shape_of(*args, cus, true);
    NormPlan p;
    plan_of(*args, cus, s, p);
    *bytes = workspace_of(*args, s, p);
    return RF_OK;
}

rf_status rf_norm_backward(const rf_norm* args, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (const rf_status s = check_backward(args); s != RF_OK) return s;
    const rf_norm& a = *args;
    const bool exit = a.post != RF_NORM_ABSENT, next = a.next != RF_NORM_ABSENT;
    if (a.rows && (!a.dresidual || (exit && (!a.dbranch || (!a.branch && !a.branch_codes))) ||
                   (next && (!a.dy || !a.next_rstd || (!a.hidden && !a.hidden_codes)))))
        return bad("null buffer");
    if (a.rows && ((a.post >= RF_NORM_RMS && !a.post_rstd) || (a.post == RF_NORM_LAYER && !a.post_mean) ||
                   (a.next == RF_NORM_LAYER && !a.next_mean)))
        return bad("null statistics");
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    NormShape s = shape_of(a, cus, true);
    NormPlan p;
    plan_of(a, cus, s, p);
    if (workspace_bytes < workspace_of(a, s, p) || (workspace_of(a, s, p) && !workspace)) return bad("workspace too small");
    hipStream_t st = (hipStream_t)stream;
    if (a.rows) {
        if (const rf_status e = backward_of(a)(a, s, p, (float*)workspace, st); e != RF_OK) return e;
    } else {  // sums over no rows: there are no partial rows
        p.workers = 0;
        p.pieces = 1;
    }
    if (p.vectors) {
        const unsigned tiles = (unsigned)((a.cols + FIN_COLS - 1) / FIN_COLS);
        // y = 0: the next norm's vectors, y = 1: the post norm's and the gate
        k_norm_finish<<<dim3(tiles, p.i_p >= 0 ? 2 : 1), dim3(FIN_COLS, FIN_LANES), 0, st>>>(a, p, (const float*)workspace);
    }
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

}  // extern "C"
