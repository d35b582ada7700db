// Low-rank adapters beside a shared projection (ql_lora.cu): launch arguments.
#pragma once
#include "ql_common.cuh"

namespace ql {

constexpr int kLoraMaxRank = 256, kLoraMaxProj = 3;
constexpr int kLoraChunk = 512;  // rows among which those of one adapter are brought together
constexpr int kLoraTile = 128;   // rows of a tile on tcgen05, where an adapter has at least
constexpr int kLoraTileFrom = 48;  // so many on average

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
    // tiles on tcgen05 only:
    bool y_vec;       // base, y and every projection's columns start on 16 bytes, whole groups of 4
    bool split;       // a projection per blockIdx.y, not all in one
    int ring, ring_bytes;  // stages of widened weights
    int *err;
};

enum { kW32, kW16, kWB16 };  // types of the weights

// v = hi + lo + less than 2^-22 |v|, both tf32.  (hi is cut off, so that it cannot overflow; the rest is exact.)
__device__ __forceinline__ void limbs(float v, uint32_t &hi, uint32_t &lo) {
    hi = __float_as_uint(v) & 0xFFFFE000u;
    lo = (__float_as_uint(v - __uint_as_float(hi)) + 0x1000u) & 0xFFFFE000u;
}

template <int WT>
struct Weight {
    static constexpr int bytes = WT == kW32 ? 4 : 2;
};
// N consecutive weights as fp32 values (N = 2, 4, 8; the address a multiple of N elements).
template <int WT, int N>
__device__ __forceinline__ void load_weights(const void *p, int64_t at, uint32_t (&raw)[8]) {
    const char *q = static_cast<const char *>(p) + at * Weight<WT>::bytes;
    constexpr int words = N * Weight<WT>::bytes / 4;
    if constexpr (words == 8) {
        const uint4 u = reinterpret_cast<const uint4 *>(q)[0], v = reinterpret_cast<const uint4 *>(q)[1];
        raw[0] = u.x, raw[1] = u.y, raw[2] = u.z, raw[3] = u.w, raw[4] = v.x, raw[5] = v.y, raw[6] = v.z, raw[7] = v.w;
    } else if constexpr (words == 4) {
        const uint4 u = *reinterpret_cast<const uint4 *>(q);
        raw[0] = u.x, raw[1] = u.y, raw[2] = u.z, raw[3] = u.w;
    } else if constexpr (words == 2) {
        const uint2 u = *reinterpret_cast<const uint2 *>(q);
        raw[0] = u.x, raw[1] = u.y;
    } else {
        raw[0] = *reinterpret_cast<const uint32_t *>(q);
    }
}
// Weight i of them.
template <int WT>
__device__ __forceinline__ float weight(const uint32_t (&raw)[8], int i) {
    if (WT == kW32) return __uint_as_float(raw[i]);
    const uint32_t w = raw[i / 2];
    if (WT == kWB16) return __uint_as_float(i % 2 ? w & 0xFFFF0000u : w << 16);
    return half_bits_to_float(i % 2 ? w >> 16 : w);
}

// The tile that a cluster works on.
struct LoraTile {
    int id, first, n;  // adapter (< 0: none), place of its first row among the adapter's, rows
};

// Finds tile t of the rows r0 .. r0 + n: rows of equal adapters in order, tm at a time, tiles in the order of their
// first rows.  list receives the rows; every thread returns the same tile (n = 0: there are fewer).
template <int THREADS>
__device__ LoraTile find_tile(const LoraArgs &a, int t, int r0, int n, int tm, int *ids, int *list, int *box) {
    const int tid = threadIdx.x;
    constexpr int kNone = -1, kOutside = -2;  // of no adapter; of no sequence: left as it is
    constexpr int kPer = kLoraChunk / THREADS;
    int id[kPer], place[kPer];
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int i = h * THREADS + tid;
        id[h] = kOutside;
        if (i < n) {
            int s = r0 + i;
            if (a.q_start != nullptr) {  // the last sequence that starts at or before the row
                int lo = 0, hi = a.n_seqs + 1;
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (a.q_start[mid] <= r0 + i)
                        lo = mid + 1;
                    else
                        hi = mid;
                }
                s = lo - 1;
            }
            if (s >= 0 && s < a.n_seqs) {
                id[h] = a.adapter[s];
                if (id[h] >= a.n_adapters) {
                    atomicExch(a.err, kErrAdapter);
                    id[h] = kNone;
                }
                id[h] = max(id[h], kNone);
            }
        }
        ids[i] = id[h];
    }
    if (tid < tm) list[tid] = -1;
    if (tid == 0) box[0] = 0, box[1] = 0, box[2] = 0;  // rows, adapter, place
    __syncthreads();
    __shared__ int leaders[kPer * (THREADS / 32)];
    unsigned before[kPer];
    bool leads[kPer];
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int i = h * THREADS + tid;
        place[h] = 0;
        if (id[h] > kOutside) {
            for (int j = 0; j + 4 <= i; j += 4) {
                const int4 v = *reinterpret_cast<const int4 *>(ids + j);
                place[h] += (v.x == id[h]) + (v.y == id[h]) + (v.z == id[h]) + (v.w == id[h]);
            }
            for (int j = i & ~3; j < i; ++j) place[h] += ids[j] == id[h];
        }
        leads[h] = id[h] > kOutside && place[h] % tm == 0;
        const unsigned m = __ballot_sync(0xffffffffu, leads[h]);
        before[h] = __popc(m & ((1u << (tid % 32)) - 1));
        if (tid % 32 == 0) leaders[h * (THREADS / 32) + tid / 32] = __popc(m);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        int k = before[h];
        for (int w = 0; w < h * (THREADS / 32) + tid / 32; ++w) k += leaders[w];
        if (leads[h] && k == t) box[0] = 1, box[1] = id[h], box[2] = place[h];
    }
    __syncthreads();
    const LoraTile found{box[1], box[2], box[0]};
    __syncthreads();
    if (found.n == 0) return found;
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int k = place[h] - found.first;
        if (id[h] == found.id && k >= 0 && k < tm) {
            list[k] = r0 + h * THREADS + tid;
            atomicMax(box, k + 1);
        }
    }
    __syncthreads();
    return LoraTile{found.id, found.first, box[0]};
}

// Rows of a tile, by the rows of the call.
int lora_tile_rows(int rows, int n_seqs);
cudaError_t lora_launch(const LoraArgs &a, int type, int tile_rows, cudaStream_t s);
// Tiles of 128 rows: fills in what the launch needs; false: not for these sizes or this alignment.
bool lora_tiles_plan(LoraArgs &a, int type, int distinct, int sms);
cudaError_t lora_tiles_launch(const LoraArgs &a, int type, cudaStream_t s);

}  // namespace ql
