// rf_norm_launch.h -- the launch shape of a norm call, and its launchers (one
// object per pair of element types).
#pragma once

#include "rf_norm.h"

namespace rfb {

struct NormShape {
    int tpr, ny, nv;  // lanes a row, rows a workgroup at a time, chunks a lane (0: the wide kernels)
    int64_t workers;  // forward: workgroups
    bool full, src8;
    size_t lds;
};

void norm_forward_0_0(const rf_norm&, const NormShape&, hipStream_t);
void norm_forward_1_1(const rf_norm&, const NormShape&, hipStream_t);
void norm_forward_2_2(const rf_norm&, const NormShape&, hipStream_t);
void norm_forward_0_1(const rf_norm&, const NormShape&, hipStream_t);
void norm_forward_0_2(const rf_norm&, const NormShape&, hipStream_t);
// A status other than RF_OK: nothing was launched.
[[nodiscard]] rf_status norm_backward_0_0(const rf_norm&, const NormShape&, const NormPlan&, float*, hipStream_t);
[[nodiscard]] rf_status norm_backward_1_1(const rf_norm&, const NormShape&, const NormPlan&, float*, hipStream_t);
[[nodiscard]] rf_status norm_backward_2_2(const rf_norm&, const NormShape&, const NormPlan&, float*, hipStream_t);
[[nodiscard]] rf_status norm_backward_0_1(const rf_norm&, const NormShape&, const NormPlan&, float*, hipStream_t);
[[nodiscard]] rf_status norm_backward_0_2(const rf_norm&, const NormShape&, const NormPlan&, float*, hipStream_t);

}  // namespace rfb
