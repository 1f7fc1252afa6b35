// rf_muon.hip -- an optimizer step's updates from momentum in 8-bit blocks and
// orthogonalised matrices:
//   m = beta m + (1 - beta) g           (stored as codes and a scale per block)
//   u = beta m + (1 - beta) g, or m     (with m as computed, before it is stored)
//   update = scale orthogonalised(u) + decay p
// k_momentum reads the gradient and the codes once and writes the new codes and
// scales, u in f32 to the place where the orthogonalisation's next X will lie (of
// the same size, and free until then), and the sums of its squares; the
// orthogonalisation (rf_schulz.hip) takes both up.
//
// A gradient that is not finite makes its matrix' update NaN, but does not get into the
// momentum: a block of codes that it would (of an f32 momentum an element) stays as it
// was.  A NaN's code would stand for about one, where its neighbours are a thousandth,
// and every update would follow it for a hundred steps.
#include <algorithm>

#include "rf_device.h"
#include "rf_schulz.h"

using namespace rf;

namespace rf {
// This device's lookup tables (rf_host.hip).
rf_status lookup_tables_of(const uint4** out) noexcept;
}  // namespace rf

namespace {

constexpr int MAX = rfs::MAX;

struct Moment {
    const void* grad;
    uint8_t* codes;   // NULL: f32 momentum
    float* scales;
    float* momentum;
    float* u;
    double* sums;
    int64_t size;
    int32_t block_size, grad_dtype;
};

struct Moments {
    int32_t count, nesterov;
    float beta, rest;
    Moment item[MAX];
};

// Eight elements from e on, or as many as there are; zeros behind them.
__device__ __forceinline__ void load_grad(const Moment& a, int64_t e, int64_t left, float (&g)[8])
{
    if (left >= 8) {
        if (a.grad_dtype == RF_F32) {
            rfb::widen8(rfb::fetch8((const float*)a.grad + e, 0, 8), g);
        } else if (a.grad_dtype == RF_BF16) {
            rfb::widen8(rfb::fetch8((const rfb::bf16*)a.grad + e, 0, 8), g);
        } else {
            rfb::widen8(rfb::fetch8((const rfb::f16*)a.grad + e, 0, 8), g);
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) g[k] = k < left ? load1(a.grad, a.grad_dtype, e + k) : 0.0f;
}

__device__ __forceinline__ void put_u(const Moment& a, int64_t e, int64_t left, const float (&u)[8])
{
    rfb::Raw<float> r = rfb::narrow8<float>(u);
    rfb::put8(a.u + e, r, left);
}

// A workgroup takes every PARTS-th block of a matrix; eight elements a lane, whole
// blocks of up to 2048 in registers between the block's largest magnitude and its
// codes, longer ones read twice.  Of blocks of 8, 16 .. 512 a wave takes as many as it has
// lanes for.  Bound by memory: 202 million elements with bf16 gradients 363 us, 8 bytes an
// element at 4.5 TB/s, with seven workgroups a CU (four registers more, and six: 395).
// (Fewer workgroups, which would stage fewer tables of 22 KB: 7 us less, but 24 matrices of
// 2304 x 768 and 768 x 768 then take 4 more.)
// CODES: of the matrices whose momentum is codes, else of those with an f32 one.  (In one
// kernel, with what is done where values are not finite: 432 us.)
template <bool CODES> __global__ __launch_bounds__(WG, 7) void k_momentum(const Moments t, const uint4* __restrict__ tables)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[CODES ? TABLE_BYTES : 16];
    __shared__ uint32_t tops[WAVES_PER_WG];
    __shared__ double parts[WAVES_PER_WG];
    const Moment& a = t.item[blockIdx.x / rfs::PARTS];
    if ((a.codes != nullptr) != CODES) return;
    const int part = blockIdx.x % rfs::PARTS, tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const float* const book = (const float*)(lds + L_CBS);
    const int64_t bs = CODES ? a.block_size : 2048, blocks = (a.size + bs - 1) / bs;
    const bool small = CODES && bs >= 8 && bs <= WAVE * 8 && (bs & (bs - 1)) == 0;
    // what the workgroup takes at a time: a block, or as many small ones as it has lanes for
    const int64_t each = small ? WG * 8 / bs : 1, turns = (blocks + each - 1) / each;
    if (CODES && part < turns) stage_tables(lds, tables);
    double sum = 0;
    for (int64_t turn = part; turn < turns; turn += rfs::PARTS) {
        const int64_t b = small ? min(turn * each + tid * 8 / bs, blocks - 1) : turn;
        const bool mine = !small || turn * each + tid * 8 / bs < blocks;
        const int64_t from = b * bs;
        const float old = CODES ? a.scales[b] : 1.0f;
        float m[8];
        uint32_t top = 0;
        // momentum of the eight elements at c of the block
        auto moment = [&](int64_t c, float (&g)[8]) {
            const int64_t left = min(bs - c, a.size - from - c);
            load_grad(a, from + c, left, g);
            if constexpr (CODES) {
                uint32_t w[2] = {};
                const uint8_t* const p = a.codes + from + c;
                if (bs - c >= 8) {
                    const rfb::u32x2 v = *(const rfb::u32x2_at*)p;
                    w[0] = v[0];
                    w[1] = v[1];
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k < bs - c) w[k / 4] |= (uint32_t)p[k] << (8 * (k & 3));
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) m[k] = k < left ? book[(w[k / 4] >> (8 * (k & 3))) & 255u] * old : 0.0f;
            } else {
                float g2[8];
                Moment f = a;
                f.grad = a.momentum;
                f.grad_dtype = RF_F32;
                load_grad(f, from + c, left, g2);
#pragma unroll
                for (int k = 0; k < 8; ++k) m[k] = g2[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) m[k] = t.beta * m[k] + t.rest * g[k];
            return left;
        };
        const int64_t first = small ? (int64_t)(tid * 8) & (bs - 1) : (int64_t)tid * 8;
        for (int64_t c = mine ? first : bs; c < bs; c += WG * 8) {
            float g[8], u[8];
            const int64_t left = moment(c, g);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                top = max(top, __float_as_uint(m[k]) & 0x7FFFFFFFu);
                u[k] = t.nesterov ? t.beta * m[k] + t.rest * g[k] : m[k];
                if (k < left) sum += (double)u[k] * (double)u[k];
            }
            if (left > 0) {
                put_u(a, from + c, left, u);
                if (!CODES && top < 0x7F800000u) {
                    rfb::put8(a.momentum + from + c, rfb::narrow8<float>(m), left);
                } else if (!CODES) {
                    for (int k = 0; k < 8 && k < left; ++k)
                        if (__builtin_isfinite(m[k])) a.momentum[from + c + k] = m[k];
                }
            }
        }
        if (!CODES) continue;
        if (small) {
            for (int d = 1; d < bs / 8; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        } else {
            top = wave_max_u32(top);
            __syncthreads();  // the block before has been coded
            if (lane == 0) tops[wave] = top;
            __syncthreads();
            for (int w = 0; w < WAVES_PER_WG; ++w) top = max(top, tops[w]);
        }
        const bool kept = mine && top < 0x7F800000u;
        const float scale = scale_from_absmax_bits(top), rs = 1.0f / scale;
        const bool fast = block_is_fast(top, scale);
        for (int64_t c = mine ? first : bs; c < bs; c += WG * 8) {
            if (bs > WG * 8) {
                float g[8];
                moment(c, g);
            }
            uint32_t w[2] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t code = fast ? code_signed_fast(lds, m[k], scale, rs) : code_literal(book, m[k], scale, false, 0u);
                w[k / 4] |= code << (8 * (k & 3));
            }
            uint8_t* const p = a.codes + from + c;
            if (!kept) {
            } else if (bs - c >= 8) {
                *(rfb::u32x2_at*)p = rfb::u32x2{w[0], w[1]};
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < bs - c) p[k] = (uint8_t)(w[k / 4] >> (8 * (k & 3)));
            }
        }
        // (read at the block's start: before the barriers, or by this wave itself)
        if (kept && (small ? first == 0 : tid == 0)) a.scales[b] = scale;
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) parts[wave] = sum;
    __syncthreads();
    if (tid == 0) a.sums[part] = (parts[0] + parts[1]) + (parts[2] + parts[3]);
}

struct Call {
    const rf_muon8_leaf* leaves;
    float beta, rest;
    bool nesterov;
    const uint4* tables;
};

// The directions of the matrices `which` [count], at u with their sums.
rf_status directions(void* context, const int64_t* which, int count, float* const* u, double* const* sums, hipStream_t st)
{
    const Call& call = *(const Call*)context;
    Moments t{};
    t.count = count;
    t.nesterov = call.nesterov;
    t.beta = call.beta;
    t.rest = call.rest;
    for (int i = 0; i < count; ++i) {
        const rf_muon8_leaf& l = call.leaves[which[i]];
        t.item[i] = {l.grad, l.codes, l.scales, l.momentum, u[i], sums[i], l.rows * l.cols, l.block_size, l.dtype};
    }
    const auto coded = [](const Moment& m) { return m.codes != nullptr; };
    if (std::any_of(t.item, t.item + count, coded)) k_momentum<true><<<count * rfs::PARTS, WG, 0, st>>>(t, call.tables);
    if (!std::all_of(t.item, t.item + count, coded)) k_momentum<false><<<count * rfs::PARTS, WG, 0, st>>>(t, call.tables);
    return RF_OK;
}

bool known(int32_t dtype) { return dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16; }

rf_status check(const rf_muon8_leaf* leaves, int32_t count)
{
    if (count < 0 || count > 256 || (count && !leaves)) return report(RF_ERR_INVALID, "at most 256 leaves in a call");
    for (int32_t i = 0; i < count; ++i) {
        const rf_muon8_leaf& l = leaves[i];
        if (l.rows < 0 || l.cols < 0 || l.rows > (1 << 20) || l.cols > (1 << 20)) return report(RF_ERR_INVALID, "matrix size out of range");
        if (!known(l.dtype) || (l.param && !known(l.param_dtype))) return report(RF_ERR_UNSUPPORTED, "dtype must be f32, bf16 or f16");
        if (l.codes && (l.block_size < 1 || !l.scales)) return report(RF_ERR_INVALID, "codes need scales and a block size");
        if (l.rows && l.cols && (!l.grad || !l.update || (!l.codes && !l.momentum))) return report(RF_ERR_INVALID, "null buffer");
    }
    return RF_OK;
}

void convert(const rf_muon8_leaf* leaves, int32_t count, rfs::Matrix* out)
{
    for (int32_t i = 0; i < count; ++i) {
        const rf_muon8_leaf& l = leaves[i];
        out[i] = {l.grad, l.update, l.param, l.rows, l.cols, l.cols, l.cols, l.cols, RF_F32, l.dtype, l.param ? l.param_dtype : RF_F32,
                  l.scale, l.decay};
    }
}

}  // namespace

extern "C" {

rf_status rf_muon8_update_workspace(const rf_muon8_leaf* leaves, int32_t count, int64_t* bytes)
{
    if (!bytes) return report(RF_ERR_INVALID, "null output");
    if (const rf_status s = check(leaves, count); s != RF_OK) return s;
    rfs::Matrix list[256];
    convert(leaves, count, list);
    if (const rf_status s = rfs::check(list, count, {0, nullptr, 0.0f}); s != RF_OK) return s;
    return rfs::workspace(list, count, bytes);
}

rf_status rf_muon8_update(const rf_muon8_leaf* leaves, int32_t count, float momentum, float rest, int32_t nesterov, int32_t steps,
                          const float* coefficients, float eps, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (const rf_status s = check(leaves, count); s != RF_OK) return s;
    rfs::Matrix list[256];
    convert(leaves, count, list);
    const rfs::Method how{steps, coefficients, eps};
    if (const rf_status s = rfs::check(list, count, how); s != RF_OK) return s;
    int64_t need = 0;
    if (const rf_status s = rfs::workspace(list, count, &need); s != RF_OK) return s;
    if (need && (!workspace || need > workspace_bytes)) return report(RF_ERR_INVALID, "workspace too small");
    if ((uintptr_t)workspace & 255) return report(RF_ERR_INVALID, "workspace must be 256-byte aligned");
    Call call{leaves, momentum, rest, nesterov != 0, nullptr};
    if (const rf_status s = lookup_tables_of(&call.tables); s != RF_OK) return s;
    return rfs::run(list, count, how, (char*)workspace, (hipStream_t)stream, directions, &call);
}

}  // extern "C"
