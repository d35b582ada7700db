// Low-rank adapters beside a shared projection (ql_lora.cu): launch arguments.
#pragma once
#include "ql_common.cuh"

namespace ql {

constexpr int kLoraMaxRank = 256, kLoraMaxProj = 3;
constexpr int kLoraChunk = 512;  // rows among which those of one adapter are brought together

struct LoraArgs {
    const void *a[kLoraMaxProj], *b[kLoraMaxProj];  // null: this projection has no adapters
    int out[kLoraMaxProj], col[kLoraMaxProj];       // outputs, first column of y
    int n_proj, in_dim, n_adapters, max_rank;
    const int *rank;     // [n_adapters] or null: max_rank
    const float *scale;  // [n_adapters] or null: 1
    const float *x, *base;  // base null: 0
    float *y;
    int64_t x_stride, base_stride, y_stride;
    const int *adapter, *q_start;  // [n_seqs]; [n_seqs + 1] or null: a row per sequence
    int n_seqs, rows;
    bool x_vec;       // rows of x start on 16 bytes
    int cluster;      // CTAs that share a tile of rows
    int chunk_tiles;  // tiles of a chunk, at most
    int *err;
};

// Rows of a tile, by the rows of the call.
int lora_tile_rows(int rows, int n_seqs);
cudaError_t lora_launch(const LoraArgs &a, int type, int tile_rows, cudaStream_t s);

}  // namespace ql
