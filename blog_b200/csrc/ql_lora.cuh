// Low-rank adapters beside a shared projection (ql_lora.cu): launch arguments.
#pragma once
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "ql_common.cuh"

namespace ql {

constexpr int kLoraMaxRank = 256, kLoraMaxProj = 3;
constexpr int kLoraChunk = 512;  // rows among which those of one adapter are brought together
constexpr int kPairs = 128;      // rows of a chunk that are compared with one another
constexpr int kLoraTile = 128;   // rows of a tile on tcgen05, for calls of at least so many rows, and kLoraTileFrom of each
constexpr int kLoraTileFrom = 32;  // adapter on average

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
    int ring, ring_bytes;      // stages of A in the products' layout
    int raw_bytes, raw_total;  // a stage of weights on their way, and all of them
    int *err;
};

// x, base and y as rows of f32, in boxes of 32 columns and a tile's rows (base: y's where there is none); bf16 A as rows of
// ranks, in boxes of 64 columns and 16 or 64 ranks.
struct LoraMaps {
    CUtensorMap x, base, y, a16[kLoraMaxProj], a64[kLoraMaxProj];
};

enum { kW32, kW16, kWB16 };  // types of the weights

// v = hi + lo + less than 2^-22 |v|, both tf32.  (hi is cut off, so that it cannot overflow; the rest is exact.)  Of a v that
// is not finite lo is NaN: the rest is 0x7FFFFFFF then, and the half added to round it would carry into the sign; as signed
// numbers that is the one sum which is not the larger.
__device__ __forceinline__ void limbs(float v, uint32_t &hi, uint32_t &lo) {
    hi = __float_as_uint(v) & 0xFFFFE000u;
    const uint32_t rest = __float_as_uint(v - __uint_as_float(hi));
    lo = (uint32_t)max((int)(rest + 0x1000u), (int)rest) & 0xFFFFE000u;
}

// Two values in three bf16 limbs, cut off one after another (8 bits each: nothing is left), packed.
__device__ __forceinline__ void limbs_b16(float x, float y, uint32_t &a, uint32_t &b, uint32_t &c) {
    constexpr uint32_t m = 0xFFFF0000u;
    a = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    const float x1 = x - __uint_as_float(__float_as_uint(x) & m), y1 = y - __uint_as_float(__float_as_uint(y) & m);
    b = __byte_perm(__float_as_uint(x1), __float_as_uint(y1), 0x7632);
    const float x2 = x1 - __uint_as_float(__float_as_uint(x1) & m), y2 = y1 - __uint_as_float(__float_as_uint(y1) & m);
    c = __byte_perm(__float_as_uint(x2), __float_as_uint(y2), 0x7632);
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

// What find_tile needs of shared memory.
struct LoraFind {
    int starts[kLoraChunk + 1], adapters[kLoraChunk];  // of the sequences, where there are no more
    alignas(16) int2 kinds[24 * 32];                               // per warp (24 at most): adapters and how many of its rows have them
    int n_kinds[24], leaders[24];
    int found[3];
};

// Finds tile t of the rows r0 .. r0 + n: rows of equal adapters in order, tm at a time, tiles in the order of their
// first rows.  list receives the rows; every thread returns the same tile (n = 0: there are fewer).
template <int THREADS>
__device__ LoraTile find_tile(const LoraArgs &a, int t, int r0, int n, int tm, LoraFind &f, int *list) {
    const int tid = threadIdx.x, lane = tid % 32;
    constexpr int kNone = -1, kOutside = -2;  // of no adapter; of no sequence: left as it is
    constexpr int kPer = (kLoraChunk + THREADS - 1) / THREADS, kWarps = THREADS / 32;
    if (a.q_start == nullptr && n <= 32) {  // a few single tokens: every warp finds the tile by itself
        int id = kOutside;
        if (lane < n) {
            id = a.adapter[r0 + lane];
            if (id >= a.n_adapters) {
                atomicExch(a.err, kErrAdapter);
                id = kNone;
            }
            id = max(id, kNone);
        }
        const unsigned same = __match_any_sync(0xffffffffu, id);
        const int place = __popc(same & ((1u << lane) - 1));
        unsigned leaders = __ballot_sync(0xffffffffu, id != kOutside && place % tm == 0);
        for (int k = 0; k < t && leaders != 0; ++k) leaders &= leaders - 1;
        if (leaders == 0) return LoraTile{0, 0, 0};
        const int at = __ffs(leaders) - 1;
        const LoraTile found{__shfl_sync(0xffffffffu, id, at), __shfl_sync(0xffffffffu, place, at),
                             min(tm, __popc(__shfl_sync(0xffffffffu, same, at)) - __shfl_sync(0xffffffffu, place, at))};
        if (tid < 32 && id == found.id && place >= found.first && place < found.first + tm) list[place - found.first] = r0 + lane;
        __syncthreads();
        return found;
    }
    const bool staged = a.q_start != nullptr && a.n_seqs <= kLoraChunk;
    if (staged)
#pragma unroll 1
        for (int i = tid; i <= a.n_seqs; i += THREADS) {
            f.starts[i] = a.q_start[i];
            if (i < a.n_seqs) f.adapters[i] = a.adapter[i];
        }
#pragma unroll 1
    for (int i = tid; i < tm; i += THREADS) list[i] = -1;
    if (tid < 3) f.found[tid] = 0;
    __syncthreads();
    int id[kPer], place[kPer];
    bool leads[kPer];
    unsigned same[kPer];
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int i = h * THREADS + tid;
        id[h] = kOutside;
        if (i < n) {
            int s = r0 + i;
            if (a.q_start != nullptr) {  // the last sequence that starts at or before the row
                int lo = 0, hi = a.n_seqs + 1;
#pragma unroll 1
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if ((staged ? f.starts[mid] : a.q_start[mid]) <= r0 + i)
                        lo = mid + 1;
                    else
                        hi = mid;
                }
                s = lo - 1;
            }
            if (s >= 0 && s < a.n_seqs) {
                id[h] = staged ? f.adapters[s] : a.adapter[s];
                if (id[h] >= a.n_adapters) {
                    atomicExch(a.err, kErrAdapter);
                    id[h] = kNone;
                }
                id[h] = max(id[h], kNone);
            }
        }
    }
    if (n <= kPairs) {  // few rows: a thread looks at all of them
        int *ids = reinterpret_cast<int *>(f.kinds);
        if (tid < kPairs) ids[tid] = id[0];  // (from n on: outside)
        __syncthreads();
        int before = 0, all = 0;
        bool lead = false;
        if (tid < kPairs) {
#pragma unroll 4
            for (int j = 0; j < n; j += 4) {
                const int4 v = *reinterpret_cast<const int4 *>(ids + j);
                const int e0 = v.x == id[0], e1 = v.y == id[0], e2 = v.z == id[0], e3 = v.w == id[0];
                all += e0 + e1 + e2 + e3;
                before += (e0 && j < tid) + (e1 && j + 1 < tid) + (e2 && j + 2 < tid) + (e3 && j + 3 < tid);
            }
            lead = id[0] != kOutside && before % tm == 0;
            const unsigned m = __ballot_sync(0xffffffffu, lead);
            if (lane == 0) f.leaders[tid / 32] = __popc(m);
            same[0] = __popc(m & ((1u << lane) - 1));
        }
        __syncthreads();
        if (lead) {
            int k = (int)same[0];
#pragma unroll
            for (int w = 0; w < kPairs / 32 - 1; ++w) k += w < tid / 32 ? f.leaders[w] : 0;
            if (k == t) f.found[0] = min(tm, all - before), f.found[1] = id[0], f.found[2] = before;
        }
        __syncthreads();
        const LoraTile found{f.found[1], f.found[2], f.found[0]};
        if (tid < kPairs && id[0] == found.id && before >= found.first && before < found.first + found.n)
            list[before - found.first] = r0 + tid;
        __syncthreads();
        return found;
    }
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int w = h * kWarps + tid / 32;
        // the warp's adapters, each with its rows: their lowest lanes write them down
        same[h] = __match_any_sync(0xffffffffu, id[h]);
        const unsigned firsts = __ballot_sync(0xffffffffu, __ffs(same[h]) - 1 == lane);
        place[h] = __popc(same[h] & ((1u << lane) - 1));
        if (__ffs(same[h]) - 1 == lane) f.kinds[w * 32 + __popc(firsts & ((1u << lane) - 1))] = make_int2(id[h], __popc(same[h]));
        if (lane == 0) f.n_kinds[w] = __popc(firsts);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int w = h * kWarps + tid / 32, first = __ffs(same[h]) - 1;
        int before = 0;  // rows of this adapter in the warps before
        const unsigned firsts = __ballot_sync(0xffffffffu, first == lane && id[h] != kOutside);
        if (__popc(firsts) <= 4) {  // few kinds: a lane looks through a warp's
#pragma unroll 1
            for (unsigned left = firsts; left != 0; left &= left - 1) {
                const int kind = __shfl_sync(0xffffffffu, id[h], __ffs(left) - 1);
                int n_before = 0;
                if (lane < w)
#pragma unroll 1
                    for (int k = 0; k < f.n_kinds[lane]; ++k) {
                        const int2 v = f.kinds[lane * 32 + k];
                        if (v.x == kind) n_before = v.y;
                    }
                n_before = __reduce_add_sync(0xffffffffu, n_before);
                if (id[h] == kind) before = n_before;
            }
        } else {  // the lowest lane of each looks through all
            if (first == lane && id[h] != kOutside)
#pragma unroll 1
                for (int v = 0; v < w; ++v)
#pragma unroll 1
                    for (int k = 0; k < f.n_kinds[v]; ++k) {
                        const int2 kind = f.kinds[v * 32 + k];
                        if (kind.x == id[h]) before += kind.y;
                    }
            before = __shfl_sync(0xffffffffu, before, first);
        }
        place[h] += before;
        leads[h] = id[h] != kOutside && place[h] % tm == 0;
        const unsigned m = __ballot_sync(0xffffffffu, leads[h]);
        same[h] = __popc(m & ((1u << lane) - 1));  // (from here: leaders before this one in its warp)
        if (lane == 0) f.leaders[w] = __popc(m);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int w = h * kWarps + tid / 32;
        const int k = (int)same[h] + __reduce_add_sync(0xffffffffu, lane < w ? f.leaders[lane] : 0);
        if (leads[h] && k == t) f.found[0] = 1, f.found[1] = id[h], f.found[2] = place[h];
    }
    __syncthreads();
    const LoraTile found{f.found[1], f.found[2], f.found[0]};
    __syncthreads();
    if (found.n == 0) return found;
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
        const int k = place[h] - found.first;
        if (id[h] == found.id && k >= 0 && k < tm) {
            list[k] = r0 + h * THREADS + tid;
            atomicMax(f.found, k + 1);
        }
    }
    __syncthreads();
    return LoraTile{found.id, found.first, f.found[0]};
}

// Adapters among n neighbouring rows, about: those of the sequences that touch them.
inline double lora_kinds(const LoraArgs &a, int n) {
    return std::min<double>(std::max(1, std::min(a.n_adapters, a.n_seqs)), (double)n * a.n_seqs / a.rows + (a.q_start != nullptr ? 1 : 0));
}
// About how many tiles of tm rows of a call of several chunks have rows: at least one for each adapter of a chunk, and half a tile
// more for each but one.
inline double lora_filled(const LoraArgs &a, int tm) {
    const int chunks = (a.rows - 1) / kLoraChunk + 1;
    const double kinds = lora_kinds(a, kLoraChunk);
    return std::max(chunks * kinds, (double)a.rows / tm + 0.5 * chunks * (kinds - 1));
}
// What a search takes beyond 2 us where a chunk's warps have more than four adapters each: a lane looks through those of all.
inline double lora_search_us(const LoraArgs &a) {
    const double kinds = lora_kinds(a, 32);
    return a.rows > kLoraChunk && kinds > 4 ? 0.0156 * (kLoraChunk / 32) * kinds : 0;
}
// A launch has tiles for every adapter of the call in every chunk of rows (which chunk has which is known on the device alone).
// What those without rows take in all: each occupies its CTAs until its search ends, 2 us where the sequences' starts stand in
// shared memory, 2.6 us beyond (65536 rows of 1024 prompts, 896 -> 896 + 128 + 128 at rank 16, with 1 and 1024 adapters: tiles of
// 128 rows 213 and 1340 us, of 32 rows 634 and 3940 us).  at_once: tiles that run at once; what does not fill a round of its own
// passes beside the others.
inline double lora_empty_us(const LoraArgs &a, double launched, double filled, int at_once) {
    return std::max(0.0, std::floor(launched / at_once) - std::ceil(filled / at_once)) * (a.n_seqs <= kLoraChunk ? 2.0 : 2.6);
}

// Fills in what the launch needs and about how long it takes; returns the rows of a tile.
int lora_plan(LoraArgs &a, int type, int distinct, int sms, double &us);
cudaError_t lora_launch(const LoraArgs &a, int type, int tile_rows, cudaStream_t s);
// Tiles of 128 rows: fills in the same; false: not for these sizes or this alignment.
bool lora_tiles_plan(LoraArgs &a, int type, int distinct, int sms, double &us);
cudaError_t lora_tiles_launch(const LoraArgs &a, const LoraMaps &maps, int type, cudaStream_t s);

}  // namespace ql
