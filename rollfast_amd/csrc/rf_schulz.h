// rf_schulz.h -- orthogonalisation of a list of matrices by Newton-Schulz
// products, as its callers inside the library use it (rf_schulz.hip).
#pragma once

#include "rf_block.h"

namespace rfs {

constexpr int PARTS = 128;  // partial sums of squares of a matrix

// One matrix.  sums: its partial sums of squares [PARTS], written by the caller; NULL: by the call.
struct Matrix {
    const void* in;
    void* out;
    const void* add;     // out = scale * orthogonalised + add_scale * add; NULL: none
    int64_t rows, cols, in_stride, out_stride, add_stride;
    int32_t in_dtype, out_dtype, add_dtype;
    float scale, add_scale;
    const double* sums;
};

struct Method {
    int32_t steps;
    const float* coefficients;  // [steps, 3]
    float eps;
};

// Checks sizes, types and coefficients.
rf_status check(const Matrix* list, int64_t count, const Method& how) noexcept;
int64_t workspace(const Matrix* list, int64_t count) noexcept;
rf_status run(const Matrix* list, int64_t count, const Method& how, char* workspace, hipStream_t stream) noexcept;

}  // namespace rfs
