// rf_wgrad.hip -- a linear layer's weight gradient from its input's 8-bit
// checkpoint: out[n, k] = sum_t dy[t, n] code[t, k] 2^(e[t, k / 32] - 127).
#include <algorithm>

#include "rf_block.h"

using namespace rfb;
using rf::report;

namespace {

constexpr int TILE = 64, STEP = 16;

// One 64 x 64 tile of out per workgroup, 16 rows at a time through LDS, 4 x 4
// outputs a lane in f32.
template <typename T, typename O>
__global__ __launch_bounds__(256) void k_wgrad(const rf_weight_grad a)
{
    __shared__ float ds[STEP][TILE], xs[STEP][TILE];
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int64_t n0 = (int64_t)blockIdx.y * TILE, k0 = (int64_t)blockIdx.x * TILE, pitch = pitch_of(a.cols);
    float acc[4][4] = {};
    for (int64_t t0 = 0; t0 < a.rows; t0 += STEP) {
        __syncthreads();
        for (int i = tid; i < STEP * TILE / CHUNK; i += 256) {
            const int r = i / (TILE / CHUNK), c = i % (TILE / CHUNK) * CHUNK;
            const int64_t t = t0 + r;
            float v[8], x[8];
            Raw<T> d = zero8<T>();
            Codes q{};
            if (t < a.rows) {
                d = load8((const T*)a.dy + t * a.dy_stride + n0 + c, a.outs - n0 - c);
                if (k0 + c < pitch) q = get_codes(a.codes, a.exponents, t, pitch, (k0 + c) / CHUNK);
            }
            widen8(d, v);
            decode8(q, x);
            for (int k = 0; k < 8; ++k) {
                ds[r][c + k] = v[k];
                xs[r][c + k] = x[k];
            }
        }
        __syncthreads();
        for (int r = 0; r < STEP; ++r)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ds[r][ty * 4 + i], xs[r][tx * 4 + j], acc[i][j]);
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + ty * 4 + i, k = k0 + tx * 4 + j;
            if (n < a.outs && k < a.cols) {
                O* at = (O*)a.out + n * a.cols + k;
                *at = (O)(a.accumulate ? (float)*at + acc[i][j] : acc[i][j]);
            }
        }
}

template <typename T> void launch(const rf_weight_grad& a, hipStream_t st)
{
    const dim3 grid((unsigned)((a.cols + TILE - 1) / TILE), (unsigned)((a.outs + TILE - 1) / TILE));
    if (a.out_dtype == RF_F32) k_wgrad<T, float><<<grid, 256, 0, st>>>(a);
    else if (a.out_dtype == RF_BF16) k_wgrad<T, bf16><<<grid, 256, 0, st>>>(a);
    else k_wgrad<T, f16><<<grid, 256, 0, st>>>(a);
}

bool known(int32_t dtype) { return dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16; }

rf_status check(const rf_weight_grad* a)
{
    if (!a) return report(RF_ERR_INVALID, "null arguments");
    if (a->rows < 0 || a->rows >= (1ll << 31) || a->outs < 1 || a->outs >= (1ll << 22) || a->cols < 1 ||
        a->cols >= (1ll << 28))
        return report(RF_ERR_INVALID, "rows, outs or cols out of range");
    if (!known(a->dy_dtype) || !known(a->out_dtype)) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
    if (((uintptr_t)a->codes & 15) != 0) return report(RF_ERR_INVALID, "checkpoint codes must be 16-byte aligned");
    return RF_OK;
}

}  // namespace

extern "C" {

rf_status rf_linear_weight_grad_workspace(const rf_weight_grad* args, int64_t* bytes)
{
    if (!bytes) return report(RF_ERR_INVALID, "null output");
    if (const rf_status s = check(args); s != RF_OK) return s;
    *bytes = 0;
    return RF_OK;
}

rf_status rf_linear_weight_grad(const rf_weight_grad* args, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (const rf_status s = check(args); s != RF_OK) return s;
    const rf_weight_grad& a = *args;
    if (!a.out || (a.rows && (!a.dy || !a.codes || !a.exponents))) return report(RF_ERR_INVALID, "null buffer");
    hipStream_t st = (hipStream_t)stream;
    if (a.dy_dtype == RF_F32) launch<float>(a, st);
    else if (a.dy_dtype == RF_BF16) launch<bf16>(a, st);
    else launch<f16>(a, st);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return rf::report_hip(e, "rf_linear_weight_grad");
    return RF_OK;
}

}  // extern "C"
