// rf_schulz.h -- orthogonalisation of a list of matrices by Newton-Schulz
// products, as its callers inside the library use it (rf_schulz.hip).
#pragma once

#include "rf_block.h"

namespace rfs {

constexpr int PARTS = 512;  // partial sums of squares of a matrix
constexpr int MAX = 32;     // matrices of a launch

struct Matrix {
    const void* in;
    void* out;
    const void* add;     // out = scale * orthogonalised + add_scale * add; NULL: none
    int64_t rows, cols, in_stride, out_stride, add_stride;
    int32_t in_dtype, out_dtype, add_dtype;
    float scale, add_scale;
};

struct Method {
    int32_t steps;
    const float* coefficients;  // [steps, 3]
    float eps;
};

// Checks sizes, types and coefficients.
rf_status check(const Matrix* list, int64_t count, const Method& how) noexcept;
rf_status workspace(const Matrix* list, int64_t count, int64_t* bytes) noexcept;

// Enqueues what writes the matrices list[which[i]], i < count <= MAX, dense in f32 to
// u[i], and to sums[i] [PARTS] partial sums of their squares.
typedef rf_status (*Source)(void* context, const int64_t* which, int count, float* const* u, double* const* sums, hipStream_t stream);

// source: writes the matrices themselves (`in`, its stride and type are not read).
rf_status run(const Matrix* list, int64_t count, const Method& how, char* workspace, hipStream_t stream, Source source = nullptr,
              void* context = nullptr) noexcept;

}  // namespace rfs
