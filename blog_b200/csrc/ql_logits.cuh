// Rules on logits before the next token is taken (ql_logits.cu): launch arguments.
#pragma once
#include "ql_common.cuh"

namespace ql {

constexpr uint32_t kLogitsMaxHistory = (1u << 20) - 1;  // ids per row

struct LogitsArgs {
    const float *logits;
    float *out;  // null: the token only
    int64_t logits_stride, out_stride;
    int rows, vocab;
    const int *history, *history_len, *prompt_len;
    int64_t history_stride;
    const float *repetition, *frequency, *presence;
    const int *bias_ids, *bias_start;
    const float *bias_values;
    const uint32_t *mask;
    int64_t mask_stride;
    int mask_rows;
    const int *mask_row;
    int *token;
    unsigned long long *keys;  // [rows] best key, zero between calls
    unsigned *done;            // [rows] CTAs that have finished, zero between calls
    int *err;
};

cudaError_t logits_launch(const LogitsArgs &a, int sms, cudaStream_t s);

}  // namespace ql
