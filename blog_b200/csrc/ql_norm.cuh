// The residual's addition with the RMS norm and its Q8_1 rows (ql_norm.cu): launch arguments.
#pragma once
#include "ql_common.cuh"

namespace ql {

constexpr int kNormMaxHidden = 32768;  // a row stands in the registers of one CTA

struct AddNormArgs {
    const void *x, *residual;  // residual null: none
    void *sum, *y;             // either may be null
    const float *gamma;        // null: 1
    uint8_t *xq;               // null: none
    int64_t x_stride, residual_stride, sum_stride, y_stride;  // elements
    float eps;
    int rows, hidden;
    bool mmq, raw_sum;
};

cudaError_t add_norm_launch(const AddNormArgs &a, bool bf16, int sms, cudaStream_t s);

}  // namespace ql
