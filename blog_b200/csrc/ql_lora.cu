// Low-rank adapters of many requests beside a shared projection,
//   h = scale_i x A_i^T,   y = base + h B_i^T,   i the adapter of the row's sequence,
// up to three projections of one x side by side, one launch.
//
// A tile is up to 8 NT rows of one adapter, gathered from kLoraChunk rows (single tokens of many sequences share an
// adapter's weights), and belongs to a cluster of CTAs: each takes its share of x's columns for h, the shares are added
// through distributed shared memory in rank order, and each takes its share of the outputs.  So nothing but y is
// written to memory, and the result does not depend on the order in which CTAs run.
//
// Both products run on the tensor cores as mma.sync m16n8k8 with the weights as the 16 rows (tf32 holds f16 and bf16
// weights exactly) and the tile's rows as the 8 columns, x and h as two tf32 limbs (22 bits), weights of 32 bits as two.
// A warp reads x and A from memory straight into the registers of its fragments: it has columns of its own, so nothing
// is shared before the warps' sums.  The tensor cores cut what they add up off towards zero, so their sums are added to
// others with rounding every 64 columns or 32 ranks.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "ql_lora.cuh"

namespace ql {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPass = 64;  // ranks that a warp sums at once

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A fragment of 16 rows x 8: elements 2 j and 2 j + 1 of the rows g and g + 8, and their second limbs.
template <int WT>
__device__ __forceinline__ void fragment(const uint32_t (&r0)[8], const uint32_t (&r1)[8], int j, uint32_t (&hi)[4],
                                         uint32_t (&lo)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float v = weight<WT>(q % 2 ? r1 : r0, 2 * j + q / 2);
        if (WT == kW32) {
            limbs(v, hi[q], lo[q]);
        } else {
            hi[q] = __float_as_uint(v);
        }
    }
}

// KU: ranks per step of the second product (8, 16 or 32): a lane has KU / 4 consecutive ranks.
template <int WT, int NT, int KU>
__device__ __forceinline__ void expand(const LoraArgs &a, const LoraTile &tile, int proj, int rank, int part, int parts,
                                       const int *list, const float *hi, const float *lo, int pitch) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int n_out = a.out[proj];
    const int64_t w0 = (int64_t)max(tile.id, 0) * n_out * a.max_rank;
    for (int o0 = (part * kWarps + warp) * 16; o0 < n_out; o0 += parts * kWarps * 16) {
        float base[NT][4], acc[NT][4], total[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int tok = nt * 8 + 2 * t + q % 2, o = o0 + g + 8 * (q / 2);
                acc[nt][q] = total[nt][q] = 0.f;
                base[nt][q] = a.base != nullptr && tok < tile.n && o < n_out
                                  ? a.base[(int64_t)list[tok] * a.base_stride + a.col[proj] + o]
                                  : 0.f;
            }
        for (int k0 = 0; k0 < rank; k0 += KU) {
            uint32_t raw[2][8];
            const int k = k0 + t * (KU / 4);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[r][i] = 0;
                const int o = o0 + g + 8 * r;
                if (o < n_out && k < rank) {
                    load_weights<WT, KU / 4>(a.b[proj], w0 + (int64_t)o * a.max_rank + k, raw[r]);
                    if (k + KU / 4 > rank) {  // what stands behind the last rank is of no meaning
#pragma unroll
                        for (int i = 0; i < KU / 4; ++i)
                            if (k + i >= rank) {
                                if (WT == kW32)
                                    raw[r][i] = 0;
                                else
                                    raw[r][i / 2] &= i % 2 ? 0x0000FFFFu : 0xFFFF0000u;
                            }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < KU / 8; ++j) {
                uint32_t wh[4], wl[4];
                fragment<WT>(raw[0], raw[1], j, wh, wl);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float2 h = *reinterpret_cast<const float2 *>(hi + (nt * 8 + g) * pitch + k + 2 * j);
                    const float2 l = *reinterpret_cast<const float2 *>(lo + (nt * 8 + g) * pitch + k + 2 * j);
                    mma_tf32(acc[nt], wh, __float_as_uint(l.x), __float_as_uint(l.y));
                    if (WT == kW32) mma_tf32(acc[nt], wl, __float_as_uint(h.x), __float_as_uint(h.y));
                    mma_tf32(acc[nt], wh, __float_as_uint(h.x), __float_as_uint(h.y));
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    total[nt][q] += acc[nt][q];
                    acc[nt][q] = 0.f;
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int tok = nt * 8 + 2 * t + q % 2, o = o0 + g + 8 * (q / 2);
                if (tok < tile.n && o < n_out)
                    a.y[(int64_t)list[tok] * a.y_stride + a.col[proj] + o] = base[nt][q] + total[nt][q];
            }
    }
}

template <int WT, int NT>
__global__ void __launch_bounds__(kThreads) lora_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int TM = 8 * NT, MT = kPass / 16;
    extern __shared__ __align__(16) float smem[];
    __shared__ LoraFind find;
    __shared__ int list[TM];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
    const int parts = a.cluster, part = blockIdx.x % parts, proj = blockIdx.y;
    const int tile_no = blockIdx.x / parts, r0 = tile_no / a.chunk_tiles * kLoraChunk;
    const LoraTile tile = find_tile<kThreads>(a, tile_no % a.chunk_tiles, r0, min(kLoraChunk, a.rows - r0), TM, find, list);
    if (tile.n == 0) return;  // (every CTA of the cluster)
    int rank = 0;
    if (tile.id >= 0 && a.a[proj] != nullptr) {
        rank = a.rank != nullptr ? a.rank[tile.id] : a.max_rank;
        if (rank < 0 || rank > a.max_rank) {
            if (tid == 0) atomicExch(a.err, kErrAdapter);
            rank = 0;
        }
    }
    if (rank == 0 && a.y == a.base) return;
    const int padded = (a.max_rank + 31) / 32 * 32, pitch = padded + 4;
    float *h = smem;                    // [padded][TM], this CTA's share; read by its cluster
    float *hi = smem + padded * TM;     // [TM][pitch] twice: h in two limbs; before that the warps' sums
    float *lo = hi + TM * pitch;
    float *sums = hi;                   // [kWarps][kPass][TM]
    cg::cluster_group cl = cg::this_cluster();
    if (rank > 0) {
        const int units = a.in_dim / 32;
        const float *xr[NT];
        bool there[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            there[nt] = nt * 8 + g < tile.n;
            xr[nt] = a.x + (int64_t)(there[nt] ? list[nt * 8 + g] : 0) * a.x_stride + 8 * t;
        }
        for (int p0 = 0; p0 < rank; p0 += kPass) {
            const int mts = min(MT, (rank - p0 + 15) / 16);
            const int64_t w0 = ((int64_t)tile.id * a.max_rank + p0) * a.in_dim + 8 * t;
            float total[MT][NT][4], acc[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < 4; ++q) total[mt][nt][q] = acc[mt][nt][q] = 0.f;
            auto settle = [&] {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            total[mt][nt][q] += acc[mt][nt][q];
                            acc[mt][nt][q] = 0.f;
                        }
            };
            int since = 0;
#pragma unroll 2
            for (int u = part * kWarps + warp; u < units; u += parts * kWarps) {
                uint32_t raw[MT][2][8];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int row = mt * 16 + g + 8 * r;
                        if (p0 + row < rank) {
                            load_weights<WT, 8>(a.a[proj], w0 + (int64_t)row * a.in_dim + u * 32, raw[mt][r]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) raw[mt][r][i] = 0;
                        }
                    }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float v[8];
                    const float *p = xr[nt] + u * 32;
                    if (!there[nt]) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = 0.f;
                    } else if (a.x_vec) {
                        const float4 c = reinterpret_cast<const float4 *>(p)[0], d = reinterpret_cast<const float4 *>(p)[1];
                        v[0] = c.x, v[1] = c.y, v[2] = c.z, v[3] = c.w, v[4] = d.x, v[5] = d.y, v[6] = d.z, v[7] = d.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = p[i];
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t h0, h1, l0, l1;
                        limbs(v[2 * j], h0, l0);
                        limbs(v[2 * j + 1], h1, l1);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            if (mt >= mts) break;
                            uint32_t wh[4], wl[4];
                            fragment<WT>(raw[mt][0], raw[mt][1], j, wh, wl);
                            mma_tf32(acc[mt][nt], wh, l0, l1);
                            if (WT == kW32) mma_tf32(acc[mt][nt], wl, h0, h1);
                            mma_tf32(acc[mt][nt], wh, h0, h1);
                        }
                    }
                }
                if (++since == 2) {
                    settle();
                    since = 0;
                }
            }
            settle();
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        *reinterpret_cast<float2 *>(sums + (warp * kPass + mt * 16 + g + 8 * r) * TM + nt * 8 + 2 * t) =
                            make_float2(total[mt][nt][2 * r], total[mt][nt][2 * r + 1]);
            __syncthreads();
            for (int e = tid; e < mts * 16 * TM; e += kThreads) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) s += sums[w * kPass * TM + e];
                h[p0 * TM + e] = s;
            }
            __syncthreads();
        }
        if (parts > 1) cl.sync();
        const float scale = a.scale != nullptr ? a.scale[tile.id] : 1.f;
        const int upto = rank <= 8 ? 8 : rank <= 16 ? 16 : (rank + 31) / 32 * 32;
        for (int e = tid; e < upto * TM; e += kThreads) {
            const int r = e / TM, tok = e % TM;
            float s = 0.f;
            if (r < rank) {
                if (parts > 1)
                    for (int c = 0; c < parts; ++c) s += *cl.map_shared_rank(h + e, c);
                else
                    s = h[e];
            }
            uint32_t v0, v1;
            limbs(s * scale, v0, v1);
            hi[tok * pitch + r] = __uint_as_float(v0);
            lo[tok * pitch + r] = __uint_as_float(v1);
        }
        __syncthreads();
        if (parts > 1) cl.barrier_arrive();  // (its share is read until all have arrived)
    }
    if (rank <= 8)
        expand<WT, NT, 8>(a, tile, proj, rank, part, parts, list, hi, lo, pitch);
    else if (rank <= 16)
        expand<WT, NT, 16>(a, tile, proj, rank, part, parts, list, hi, lo, pitch);
    else
        expand<WT, NT, 32>(a, tile, proj, rank, part, parts, list, hi, lo, pitch);
    if (rank > 0 && parts > 1) cl.barrier_wait();
}

template <int WT, int NT>
cudaError_t launch(const LoraArgs &a, cudaStream_t s) {
    constexpr int TM = 8 * NT;
    const int padded = (a.max_rank + 31) / 32 * 32;
    const size_t smem = sizeof(float) * (padded * TM + std::max(2 * TM * (padded + 4), kWarps * kPass * TM));
    cudaError_t e = cudaFuncSetAttribute(lora_kernel<WT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    const int chunks = (a.rows + kLoraChunk - 1) / kLoraChunk;
    cfg.gridDim = dim3((unsigned)(chunks * a.chunk_tiles * a.cluster), (unsigned)a.n_proj, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)a.cluster, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, lora_kernel<WT, NT>, a);
}
template <int WT>
cudaError_t launch(const LoraArgs &a, int tile_rows, cudaStream_t s) {
    return tile_rows <= 8 ? launch<WT, 1>(a, s) : tile_rows <= 16 ? launch<WT, 2>(a, s) : launch<WT, 4>(a, s);
}
}  // namespace

int lora_tile_rows(int rows, int n_seqs) {
    const int each = rows / std::max(1, n_seqs);
    return each <= 8 ? 8 : each <= 16 ? 16 : 32;
}

cudaError_t lora_launch(const LoraArgs &a, int type, int tile_rows, cudaStream_t s) {
    return type == 0 ? launch<kW32>(a, tile_rows, s) : type == 1 ? launch<kW16>(a, tile_rows, s) : launch<kWB16>(a, tile_rows, s);
}

}  // namespace ql
