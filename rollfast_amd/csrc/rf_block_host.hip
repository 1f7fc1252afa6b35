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
// Lanes lie along a row's chunks, bx of them, and over 256 / bx rows; a lane
// takes ROWS rows so that several loads are in flight.
constexpr int ROWS = 4;

struct Tiles {
    int bx, by;
    uint32_t across;  // tiles along a row
    int64_t grid;
};

// The widest bx whose last tile wastes at most 6 % of the lanes; else the one
// that wastes least.
Tiles tiles_of(int64_t rows, int64_t nch)
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
    t.grid = (int64_t)t.across * ((rows + t.by * ROWS - 1) / (t.by * ROWS));
    return t;
}

struct Place {
    int64_t ch, row;
};

__device__ __forceinline__ Place place(uint32_t across)
{
    const uint32_t tile = blockIdx.x / across;
    return {(int64_t)(blockIdx.x - tile * across) * blockDim.x + threadIdx.x,
            (int64_t)tile * (blockDim.y * ROWS) + threadIdx.y};
}

template <typename T>
__global__ __launch_bounds__(256) void k_checkpoint_store(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                          int64_t stride, int8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ exps, uint32_t across)
{
    const Place p = place(across);
    const int64_t pitch = pitch_of(cols);
    if (p.ch >= pitch / CHUNK) return;  // whole quads
    Raw<T> v[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        v[i] = zero8<T>();
        if (r < rows) v[i] = load8(x + r * stride + p.ch * CHUNK, cols - p.ch * CHUNK);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        float f[8];
        widen8(v[i], f);
        const Codes c = encode8(f);
        if (r < rows) put_codes(codes, exps, r, pitch, p.ch, c);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_checkpoint_load(const int8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ exps, int64_t rows, int64_t cols,
                                                         T* __restrict__ out, uint32_t across)
{
    const Place p = place(across);
    const int64_t pitch = pitch_of(cols);
    if (p.ch >= pitch / CHUNK) return;
    Codes v[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        v[i] = Codes{};
        if (r < rows) v[i] = get_codes(codes, exps, r, pitch, p.ch);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        float f[8];
        decode8(v[i], f);
        if (r < rows) put8(out + r * cols + p.ch * CHUNK, narrow8<T>(f), cols - p.ch * CHUNK);
    }
}

__device__ __forceinline__ float sigmoid(float x)
{
    return __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}

// a(x) and a'(x).  The tanh form is x sigmoid(2 z), z = sqrt(2 / pi) (x + 0.044715 x^3).
template <int ACT> __device__ __forceinline__ void activation(float x, float& a, float& slope)
{
    if constexpr (ACT == RF_ACT_SILU) {
        const float s = sigmoid(x);
        a = x * s;
        slope = s * fmaf(x, 1.0f - s, 1.0f);
    } else if constexpr (ACT == RF_ACT_GELU) {
        const float phi = fmaf(0.5f, erff(x * 0.70710678118654752f), 0.5f);
        a = x * phi;
        slope = fmaf(x * 0.39894228040143268f, __expf(-0.5f * x * x), phi);
    } else {
        const float x2 = x * x;
        const float s = sigmoid(1.59576912160573071f * x * fmaf(0.044715f, x2, 1.0f));
        a = x * s;
        slope = fmaf(x * s * (1.0f - s), 1.59576912160573071f * fmaf(0.134145f, x2, 1.0f), s);
    }
}

template <typename T, int ACT> __global__ __launch_bounds__(256) void k_gated_forward(const rf_gated a, uint32_t across)
{
    const Place p = place(across);
    const int64_t pitch = pitch_of(a.cols);
    if (p.ch >= pitch / CHUNK) return;
    const int64_t c = p.ch * CHUNK, left = a.cols - c;
    Raw<T> g[ROWS], u[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        g[i] = u[i] = zero8<T>();
        if (r < a.rows) {
            g[i] = load8((const T*)a.gate + r * a.gate_stride + c, left);
            u[i] = load8((const T*)a.up + r * a.up_stride + c, left);
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        if (r >= a.rows) break;  // the same for the whole quad
        float x[8], y[8], h[8];
        widen8(g[i], x);
        widen8(u[i], y);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float s;
            activation<ACT>(x[k], h[k], s);
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

template <typename T, int ACT, bool SRC8>
__global__ __launch_bounds__(256) void k_gated_backward(const rf_gated a, uint32_t across)
{
    const Place p = place(across);
    const int64_t pitch = pitch_of(a.cols), nch = pitch / CHUNK;
    const int64_t c = p.ch * CHUNK, left = a.cols - c;
    if (left <= 0) return;
    Raw<T> d[ROWS];
    Saved<T, SRC8> g[ROWS], u[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = min(p.row + i * blockDim.y, a.rows - 1);
        d[i] = load8((const T*)a.dh + r * a.dh_stride + c, left);
        g[i].load((const T*)a.gate, a.gate_stride, a.gate_codes, a.gate_exponents, r, pitch, p.ch, nch, a.cols);
        u[i].load((const T*)a.up, a.up_stride, a.up_codes, a.up_exponents, r, pitch, p.ch, nch, a.cols);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = p.row + i * blockDim.y;
        if (r >= a.rows) break;
        float x[8], y[8], dh[8];
        g[i].get(x);
        u[i].get(y);
        widen8(d[i], dh);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float v, s;
            activation<ACT>(x[k], v, s);
            x[k] = dh[k] * y[k] * s;
            y[k] = dh[k] * v;
        }
        put8((T*)a.dgate + r * a.dgate_stride + c, narrow8<T>(x), left);
        put8((T*)a.dup + r * a.dup_stride + c, narrow8<T>(y), left);
    }
}

template <typename T, int ACT> void launch_gated(const rf_gated& a, bool back, const Tiles& t, hipStream_t st)
{
    const dim3 grid((unsigned)t.grid), block(t.bx, t.by);
    if (!back) k_gated_forward<T, ACT><<<grid, block, 0, st>>>(a, t.across);
    else if (a.gate_codes) k_gated_backward<T, ACT, true><<<grid, block, 0, st>>>(a, t.across);
    else k_gated_backward<T, ACT, false><<<grid, block, 0, st>>>(a, t.across);
}

template <typename T> void launch_gated(const rf_gated& a, bool back, const Tiles& t, hipStream_t st)
{
    if (a.activation == RF_ACT_SILU) launch_gated<T, RF_ACT_SILU>(a, back, t, st);
    else if (a.activation == RF_ACT_GELU) launch_gated<T, RF_ACT_GELU>(a, back, t, st);
    else launch_gated<T, RF_ACT_GELU_TANH>(a, back, t, st);
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
    const Tiles t = tiles_of(a->rows, pitch_of(a->cols) / CHUNK);
    if (t.grid > 0x7FFFFFFF) return report(RF_ERR_UNSUPPORTED, "too many elements for one launch");
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == RF_F32) launch_gated<float>(*a, back, t, st);
    else if (a->dtype == RF_BF16) launch_gated<bf16>(*a, back, t, st);
    else launch_gated<f16>(*a, back, t, st);
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

// ----------------------------------------------------------------- norms ---
constexpr int64_t MAX_REGISTER_COLS = 8192;  // 512 lanes, two chunks each
constexpr size_t MAX_LDS = 64 * 1024;

NormShape shape_of(const rf_norm& a, int cus)
{
    NormShape s{};
    const int64_t nch = pitch_of(a.cols) / CHUNK;
    s.tpr = nch <= 128 ? 64 : nch <= 256 ? 128 : nch <= 512 ? 256 : 512;
    s.nv = a.cols > MAX_REGISTER_COLS ? 0 : nch <= s.tpr ? 1 : 2;
    s.ny = s.tpr == 64 ? 4 : 1;
    s.full = a.post == RF_NORM_LAYER || a.next == RF_NORM_LAYER || a.dbias || a.dnext_bias || (a.bias && a.dgate);
    s.src8 = a.post == RF_NORM_ABSENT ? a.hidden_codes != nullptr : a.branch_codes != nullptr;
    s.workers = std::max<int64_t>(1, std::min<int64_t>((a.rows + s.ny - 1) / s.ny, (int64_t)cus * 2048 / (s.tpr * s.ny) * 2));
    if (s.nv == 0) s.workers = std::max<int64_t>(1, std::min<int64_t>(a.rows, (int64_t)cus * 4));
    return s;
}

// Rows are cut into pieces of a group, about two workgroups a CU; with more
// groups than that a workgroup takes whole groups.
void plan_of(const rf_norm& a, int cus, NormShape& s, NormPlan& p)
{
    p = NormPlan{};
    const bool exit = a.post != RF_NORM_ABSENT;
    const int64_t target = (int64_t)cus * 2;
    p.groups = exit ? std::max<int64_t>(1, a.gates) : 1;
    p.group_rows = a.rows / p.groups;
    if (p.groups > target) {
        p.pieces = 0;
        p.workers = (int32_t)target;
    } else {
        const int64_t per = std::max<int64_t>(1, (p.group_rows + s.ny - 1) / s.ny);
        p.pieces = (int32_t)std::min<int64_t>(per, std::max<int64_t>(1, target / p.groups));
        p.workers = (int32_t)(p.pieces * p.groups);
    }
    int n = 0;
    p.i_p = exit && (a.dweight || a.dbias || a.dgate) ? n++ : -1;
    p.i_q = exit && (a.dbias || (a.dgate && a.bias)) ? n++ : -1;
    p.i_w2 = a.next != RF_NORM_ABSENT && a.dnext_weight ? n++ : -1;
    p.i_b2 = a.next != RF_NORM_ABSENT && a.dnext_bias ? n++ : -1;
    p.vectors = n;
    const int64_t pitch = pitch_of(a.cols);
    s.lds = s.ny > 1 ? pitch * sizeof(float) : 0;
    if (p.pieces == 0) s.lds = (size_t)s.ny * (s.full ? 2 : 1) * pitch * sizeof(float);
    if (s.lds > MAX_LDS - 1024) s.nv = 0, s.ny = 1, s.tpr = 512, s.lds = 0;
}

int64_t workspace_of(const rf_norm& a, const NormShape& s, const NormPlan& p)
{
    int64_t n = (int64_t)p.workers * p.vectors * a.cols;
    if (s.nv == 0 && p.pieces == 0) n += (int64_t)p.workers * 2 * a.cols;
    return n * (int64_t)sizeof(float);
}

// Adds the partial rows.  A column's rows are dealt to 16 lanes: those of one
// group, or, with many groups of few pieces, the groups themselves.
constexpr int FIN_COLS = 64, FIN_LANES = 16;

__global__ __launch_bounds__(FIN_COLS* FIN_LANES) void k_norm_finish(const rf_norm a, const NormPlan p,
                                                                    const float* __restrict__ partial)
{
    __shared__ float lds[FIN_LANES][FIN_COLS];
    const int64_t c = (int64_t)blockIdx.x * FIN_COLS + threadIdx.x, cols = a.cols;
    const int ty = threadIdx.y;
    const bool in = c < cols;
    auto sum = [&](float v) {  // over the lanes of a column, in their order
        __syncthreads();
        lds[ty][threadIdx.x] = v;
        __syncthreads();
        float s = 0.0f;
        for (int i = 0; i < FIN_LANES; ++i) s += lds[i][threadIdx.x];
        return s;
    };
    auto rows = [&](int index, int64_t w0, int64_t w1, int64_t from, int64_t step) {
        float s = 0.0f;
        if (in && index >= 0)
            for (int64_t w = w0 + from; w < min(w1, (int64_t)p.workers); w += step) s += partial[(w * p.vectors + index) * cols + c];
        return s;
    };
    if (p.i_w2 >= 0) {
        const float v = sum(rows(p.i_w2, 0, p.workers, ty, FIN_LANES));
        if (in && ty == 0) put_scalar(a.dnext_weight, a.next_weight_dtype, c, v);
    }
    if (p.i_b2 >= 0) {
        const float v = sum(rows(p.i_b2, 0, p.workers, ty, FIN_LANES));
        if (in && ty == 0) put_scalar(a.dnext_bias, a.next_bias_dtype, c, v);
    }
    if (p.i_p < 0) return;
    const float w = in && a.weight ? scalar_at(a.weight, a.weight_dtype, c) : 1.0f;
    const float b = in && a.bias ? scalar_at(a.bias, a.bias_dtype, c) : 0.0f;
    auto gate = [&](int64_t g) { return in && a.gate ? scalar_at(a.gate, a.gate_dtype, g * cols + c) : 1.0f; };
    auto put_gate = [&](int64_t g, float P, float Q) {
        if (in && a.dgate) put_scalar(a.dgate, a.gate_dtype, g * cols + c, a.branch_scale * fmaf(w, P, b * Q));
    };
    float dw, db;
    if (p.pieces == 0) {  // the gate is in the sums already
        dw = sum(rows(p.i_p, 0, p.workers, ty, FIN_LANES));
        db = sum(rows(p.i_q, 0, p.workers, ty, FIN_LANES));
    } else if (p.pieces >= FIN_LANES || p.groups == 1) {
        dw = db = 0.0f;
        for (int64_t g = 0; g < p.groups; ++g) {
            const float P = sum(rows(p.i_p, g * p.pieces, (g + 1) * p.pieces, ty, FIN_LANES));
            const float Q = p.i_q >= 0 ? sum(rows(p.i_q, g * p.pieces, (g + 1) * p.pieces, ty, FIN_LANES)) : 0.0f;
            if (ty == 0) put_gate(g, P, Q);
            dw = fmaf(gate(g), P, dw);
            db = fmaf(gate(g), Q, db);
        }
    } else {
        float sw = 0.0f, sb = 0.0f;
        for (int64_t g = ty; g < p.groups; g += FIN_LANES) {
            const float P = rows(p.i_p, g * p.pieces, (g + 1) * p.pieces, 0, 1);
            const float Q = rows(p.i_q, g * p.pieces, (g + 1) * p.pieces, 0, 1);
            put_gate(g, P, Q);
            sw = fmaf(gate(g), P, sw);
            sb = fmaf(gate(g), Q, sb);
        }
        dw = sum(sw);
        db = sum(sb);
    }
    if (in && ty == 0) {
        if (a.dweight) put_scalar(a.dweight, a.weight_dtype, c, a.branch_scale * dw);
        if (a.dbias) put_scalar(a.dbias, a.bias_dtype, c, a.branch_scale * db);
    }
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
using backward_t = void (*)(const rf_norm&, const NormShape&, const NormPlan&, float*, hipStream_t);

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
    if (!sane(rows, cols)) return bad("rows or cols out of range");
    if (!known(dtype)) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
    if (rows == 0) return RF_OK;
    if (!x || !codes || !exponents) return bad("null buffer");
    if (const rf_status s = check_kept(codes, exponents); s != RF_OK) return s;
    const Tiles t = tiles_of(rows, pitch_of(cols) / CHUNK);
    if (t.grid > 0x7FFFFFFF) return report(RF_ERR_UNSUPPORTED, "too many elements for one launch");
    const dim3 grid((unsigned)t.grid), block(t.bx, t.by);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RF_F32)
        k_checkpoint_store<float><<<grid, block, 0, st>>>((const float*)x, rows, cols, row_stride, codes, exponents, t.across);
    else if (dtype == RF_BF16)
        k_checkpoint_store<bf16><<<grid, block, 0, st>>>((const bf16*)x, rows, cols, row_stride, codes, exponents, t.across);
    else
        k_checkpoint_store<f16><<<grid, block, 0, st>>>((const f16*)x, rows, cols, row_stride, codes, exponents, t.across);
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

rf_status rf_checkpoint_load(const int8_t* codes, const uint8_t* exponents, int64_t rows, int64_t cols, int32_t dtype,
                             void* out, void* stream)
{
    if (!sane(rows, cols)) return bad("rows or cols out of range");
    if (!known(dtype)) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
    if (rows == 0) return RF_OK;
    if (!out || !codes || !exponents) return bad("null buffer");
    if (const rf_status s = check_kept(codes, exponents); s != RF_OK) return s;
    const Tiles t = tiles_of(rows, pitch_of(cols) / CHUNK);
    if (t.grid > 0x7FFFFFFF) return report(RF_ERR_UNSUPPORTED, "too many elements for one launch");
    const dim3 grid((unsigned)t.grid), block(t.bx, t.by);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RF_F32) k_checkpoint_load<float><<<grid, block, 0, st>>>(codes, exponents, rows, cols, (float*)out, t.across);
    else if (dtype == RF_BF16) k_checkpoint_load<bf16><<<grid, block, 0, st>>>(codes, exponents, rows, cols, (bf16*)out, t.across);
    else k_checkpoint_load<f16><<<grid, block, 0, st>>>(codes, exponents, rows, cols, (f16*)out, t.across);
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
    forward_of(a)(a, shape_of(a, cus), (hipStream_t)stream);
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

rf_status rf_norm_backward_workspace(const rf_norm* args, int64_t* bytes)
{
    if (!bytes) return bad("null output");
    if (const rf_status s = check_backward(args); s != RF_OK) return s;
    int cus = 0;
    if (const rf_status s = rf::device_cus(&cus); s != RF_OK) return s;
    NormShape s = shape_of(*args, cus);
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
    NormShape s = shape_of(a, cus);
    NormPlan p;
    plan_of(a, cus, s, p);
    if (workspace_bytes < workspace_of(a, s, p) || (workspace_of(a, s, p) && !workspace)) return bad("workspace too small");
    hipStream_t st = (hipStream_t)stream;
    if (a.rows) {
        backward_of(a)(a, s, p, (float*)workspace, st);
    } else {  // sums over no rows: there are no partial rows
        p.workers = 0;
        p.pieces = 1;
    }
    if (p.vectors) {
        const unsigned tiles = (unsigned)((a.cols + FIN_COLS - 1) / FIN_COLS);
        k_norm_finish<<<dim3(tiles), dim3(FIN_COLS, FIN_LANES), 0, st>>>(a, p, (const float*)workspace);
    }
    BLK_TRY(hipGetLastError());
    return RF_OK;
}

}  // extern "C"
