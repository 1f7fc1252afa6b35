// rf_norm_inst.hip -- the norm kernels of one (residual type, branch type)
// pair, RFI_T and RFI_U (RF_F32 / RF_BF16 / RF_F16); one object each.
#include "rf_norm.h"
#include "rf_norm_launch.h"

namespace rfb {

template <int DT> struct Elem;
template <> struct Elem<RF_F32> { using type = float; };
template <> struct Elem<RF_BF16> { using type = bf16; };
template <> struct Elem<RF_F16> { using type = f16; };
using T = Elem<RFI_T>::type;
using U = Elem<RFI_U>::type;

template <bool EXIT, bool NEXT, bool FULL, bool TAIL>
static void forward(const rf_norm& a, const NormShape& s, hipStream_t st)
{
    const dim3 grid((unsigned)s.workers), block(s.tpr, s.ny);
    const Share rows = share_of(a.rows, s.workers);
    const uint32_t per_gate = a.gates > 1 ? (uint32_t)(a.rows / a.gates) : 0;
    if (s.nv == 1) k_norm_forward<T, U, EXIT, NEXT, FULL, TAIL, 1, 512><<<grid, block, 0, st>>>(a, rows, per_gate);
    else if (s.tpr <= 512) k_norm_forward<T, U, EXIT, NEXT, FULL, TAIL, 2, 512><<<grid, block, 0, st>>>(a, rows, per_gate);
    else k_norm_forward<T, U, EXIT, NEXT, FULL, TAIL, 2, 1024><<<grid, block, 0, st>>>(a, rows, per_gate);
}

template <bool EXIT, bool NEXT> static void forward(const rf_norm& a, const NormShape& s, hipStream_t st)
{
    if (s.nv == 0) {
        k_norm_forward_wide<T, U, EXIT, NEXT><<<dim3((unsigned)s.workers), dim3(s.tpr), 0, st>>>(a);
    } else if (a.cols % CHUNK) {
        if (s.full) forward<EXIT, NEXT, true, true>(a, s, st);
        else forward<EXIT, NEXT, false, true>(a, s, st);
    } else {
        if (s.full) forward<EXIT, NEXT, true, false>(a, s, st);
        else forward<EXIT, NEXT, false, false>(a, s, st);
    }
}

template <bool EXIT, bool NEXT, bool FULL, bool SRC8, bool TAIL>
static rf_status backward(const rf_norm& a, const NormShape& s, const NormPlan& p, float* partial, hipStream_t st)
{
    const dim3 grid((unsigned)p.workers), block(s.tpr, s.ny);
    if (s.nv == 1) k_norm_backward<T, U, EXIT, NEXT, FULL, SRC8, TAIL, 1><<<grid, block, s.lds, st>>>(a, p, partial);
    else if (s.tpr <= 512) k_norm_backward<T, U, EXIT, NEXT, FULL, SRC8, TAIL, 2><<<grid, block, s.lds, st>>>(a, p, partial);
    else {
        static std::atomic<uint64_t> done;
        const auto f = k_norm_backward_broad<T, U, EXIT, NEXT, FULL, SRC8, TAIL>;
        constexpr size_t lds = EXIT && NEXT ? 1024 * 2 * 2 * 8 * sizeof(float) : 0;
        if (const rf_status e = allow_lds((const void*)f, lds, done); e != RF_OK) return e;
        f<<<grid, block, lds, st>>>(a, p, partial);
    }
    return RF_OK;
}

template <bool EXIT, bool NEXT, bool SRC8>
static rf_status backward(const rf_norm& a, const NormShape& s, const NormPlan& p, float* partial, hipStream_t st)
{
    if (s.nv == 0) {
        k_norm_backward_wide<T, U, EXIT, NEXT, SRC8><<<dim3((unsigned)p.workers), dim3(s.tpr), 0, st>>>(a, p, partial);
        return RF_OK;
    }
    if (a.cols % CHUNK) {
        return s.full ? backward<EXIT, NEXT, true, SRC8, true>(a, s, p, partial, st)
                      : backward<EXIT, NEXT, false, SRC8, true>(a, s, p, partial, st);
    }
    return s.full ? backward<EXIT, NEXT, true, SRC8, false>(a, s, p, partial, st)
                  : backward<EXIT, NEXT, false, SRC8, false>(a, s, p, partial, st);
}

template <bool EXIT, bool NEXT>
static rf_status backward(const rf_norm& a, const NormShape& s, const NormPlan& p, float* partial, hipStream_t st)
{
    return s.src8 ? backward<EXIT, NEXT, true>(a, s, p, partial, st) : backward<EXIT, NEXT, false>(a, s, p, partial, st);
}

#define RFI_CAT2(a, b, c) a##b##_##c
#define RFI_CAT(a, b, c) RFI_CAT2(a, b, c)

void RFI_CAT(norm_forward_, RFI_T, RFI_U)(const rf_norm& a, const NormShape& s, hipStream_t st)
{
    if (a.post == RF_NORM_ABSENT) forward<false, true>(a, s, st);
    else if (a.next == RF_NORM_ABSENT) forward<true, false>(a, s, st);
    else forward<true, true>(a, s, st);
}

rf_status RFI_CAT(norm_backward_, RFI_T, RFI_U)(const rf_norm& a, const NormShape& s, const NormPlan& p, float* partial,
                                                hipStream_t st)
{
    if (a.post == RF_NORM_ABSENT) return backward<false, true>(a, s, p, partial, st);
    if (a.next == RF_NORM_ABSENT) return backward<true, false>(a, s, p, partial, st);
    return backward<true, true>(a, s, p, partial, st);
}

}  // namespace rfb
