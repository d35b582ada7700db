// 8-bit KV cache: cache view and launch arguments of the append, gather and attention kernels
// (ql_kv8.cu, ql_kv8_attn.cu).
#pragma once
#include <cuda_bf16.h>

#include "ql_common.cuh"

namespace ql {

constexpr int kKvBlock = 32;        // tokens per block (= page); one scale per block and KV head
constexpr int kKvMaxHeadDim = 256;  // head_dim: multiples of 32 up to this

// The caller's cache (ql_kv8_cache in include/qlinear_b200.h) as the kernels see it.
struct Kv8View {
    uint8_t *k_codes, *v_codes;  // [n_pages][kv_heads][32][head_dim], code + 128
    float *k_scale, *v_scale;    // [n_pages][kv_heads]
    float *k_open, *v_open;      // [n_slots][2][kv_heads][32][head_dim]
    const int *page_table;       // [n_seqs][max_pages]
    const int *slots;            // [n_seqs] or null
    int n_pages, n_slots, n_seqs, max_pages, kv_heads, head_dim;
    int *err;                    // device error word
};

// Which sequence a row belongs to: q_start[n_seqs + 1] (null: row s is sequence s's one token).
struct Kv8Rows {
    const int *kv_len;   // [n_seqs] tokens in the cache, this call's among them
    const int *q_start;  // [n_seqs + 1] or null
    int rows;
};

struct Kv8AppendArgs {
    Kv8View c;
    Kv8Rows r;
    const void *q, *k, *v;
    void *q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;  // elements between rows
    int n_heads;
    const float *q_gamma, *k_gamma;  // [head_dim] or null
    float eps;
    const float *rope;  // [max_positions][rotary_dim]: cosines, then sines
    int rotary_dim, max_positions;
};

struct Kv8AttnArgs {
    Kv8View c;
    Kv8Rows r;
    const void *q, *gate;
    void *out;
    int64_t q_stride, gate_stride, out_stride;
    int n_heads;
    float scale_log2;  // softmax scale x log2(e)
    bool vec;          // q and out: every row starts on 16 bytes
    int splits;        // CTAs over the keys of one (sequence, KV head, row group): clusters of `cluster`
    int cluster;       // 1, 2, 4 or 8 (prompts: 1 to 8, all of the splits)
    bool longest_first;  // CTAs start by their sequences' lengths, at most kKvAttnSorted sequences
    int row_groups;    // groups of 8 (query token, head of the KV head's group) rows per sequence (prompts: kv8_prompt_rows)
    int tile0;         // prompts: the launch's first tile of rows, from the sequence's end
    unsigned *arrivals;  // [n_seqs x kv_heads x row_groups][8] zero between calls (several clusters)
    float *part;         // [...][clusters][8][head_dim + 4]
};

// Slot of a sequence's open rows, or -1 (recorded in the error word).
__device__ __forceinline__ int kv8_slot(const Kv8View &c, int seq) {
    const int s = c.slots != nullptr ? c.slots[seq] : seq;
    if (s < 0 || s >= c.n_slots) {
        atomicExch(c.err, kErrKvSlot);
        return -1;
    }
    return s;
}
// Page of a sequence's block, or -1 (recorded in the error word).
__device__ __forceinline__ int kv8_page(const Kv8View &c, int seq, int block) {
    const int p = block < c.max_pages ? c.page_table[(int64_t)seq * c.max_pages + block] : -1;
    if (p < 0 || p >= c.n_pages) {
        atomicExch(c.err, kErrKvPage);
        return -1;
    }
    return p;
}
__device__ __forceinline__ int64_t kv8_open_at(const Kv8View &c, int slot, int block, int kh) {
    return (((int64_t)slot * 2 + (block & 1)) * c.kv_heads + kh) * kKvBlock * c.head_dim;
}
__device__ __forceinline__ int64_t kv8_codes_at(const Kv8View &c, int page, int kh) {
    return ((int64_t)page * c.kv_heads + kh) * kKvBlock * c.head_dim;
}

// Rows of a sequence in the call (never outside the call's rows).
__device__ __forceinline__ void kv8_rows_of(const Kv8Rows &r, int seq, int &row0, int &n) {
    row0 = seq;
    n = 1;
    if (r.q_start != nullptr) {
        row0 = min(max(r.q_start[seq], 0), r.rows);
        n = max(min(r.q_start[seq + 1], r.rows) - row0, 0);
    }
}

// Sequence of a row: the last s with q_start[s] <= row (32 candidates per step, one load round for up
// to 32 sequences).  The whole warp calls it with the same row.
__device__ __forceinline__ int kv8_seq_of_row(const int *q_start, int n_seqs, int row, int lane) {
    int lo = 0, n = n_seqs;  // the answer lies in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const bool le = lane * step < n && q_start[at] <= row;
        const unsigned b = __ballot_sync(0xffffffffu, le);
        const int hit = b == 0 ? 0 : 31 - __clz(b);
        n = min(step, n - hit * step);
        lo += hit * step;
    }
    return lo;
}

cudaError_t kv8_append_launch(const Kv8AppendArgs &a, bool bf16, cudaStream_t s);
cudaError_t kv8_gather_launch(const Kv8View &c, const int *kv_len, const int *start, int count, void *k_out, void *v_out,
                              bool bf16, cudaStream_t s);
cudaError_t kv8_attn_launch(const Kv8AttnArgs &a, bool bf16, cudaStream_t s);
// The tensor-core form for prompts (ql_kv8_prompt.cu).
constexpr int kKvMaxTiles = 65535;            // tiles of rows of one launch (the grid's z)
int kv8_prompt_rows(int head_dim, bool f32);  // rows per CTA, 0: not taken
cudaError_t kv8_prompt_launch(const Kv8AttnArgs &a, bool bf16, cudaStream_t s);

// CTAs of the attention's split kernel that one SM holds (the host sizes the split count by it).
int kv8_attn_ctas_per_sm(int head_dim);
constexpr int kKvAttnMaxCtasPerSm = 4;    // of any head_dim
constexpr int kKvAttnWarps = 4;           // warps per CTA, each with key blocks of its own
constexpr int kKvAttnRows = 8;            // rows per CTA: query tokens x heads of one KV head's group
constexpr int kKvAttnMaxClusters = 16;
constexpr int kKvAttnSorted = 32 * kKvAttnWarps;  // sequences that a CTA ranks, one per thread

}  // namespace ql
