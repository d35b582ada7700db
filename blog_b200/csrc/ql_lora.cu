// Low-rank adapters of many requests beside a shared projection,
//   h = scale_i x A_i^T,   y = base + h B_i^T,   i the adapter of the row's sequence,
// up to three projections of one x side by side, one launch.
//
// A tile is up to 8 NT rows of one adapter, gathered from kLoraChunk rows (single tokens of many sequences share an
// adapter's weights), and belongs to a cluster of CTAs: each takes its share of x's columns for h, the shares are added
// through distributed shared memory in rank order, and each takes its share of the outputs.  So nothing but y is
// written to memory, and the result does not depend on the order in which CTAs run.
//
// Both products run on the tensor cores (mma.sync) with the weights as the 16 rows and the tile's rows as the 8 columns, so
// that weights go from memory straight into fragments, which hold them exactly; the fp32 operand is taken apart:
//   bf16 weights  m16n8k16 bf16, x and h in three bf16 limbs (all of their bits)
//   f16 weights   x: m16n8k8 tf32, two limbs (22 bits); h: m16n8k16 f16, two limbs of h times a power of two per row (22 bits
//                 of the row's largest)
//   f32 weights   m16n8k8 tf32, two limbs on both sides
// A warp has columns of its own, so nothing is shared before the warps' sums.  The tensor cores cut what they add up off
// towards zero, so their sums are added to others with rounding every 64 columns or 32 ranks.
//
// Bound: latency.  One token over 3584 -> 3584 + 512 + 512 at rank 16 takes 6.5 us: the launch, finding the tile, loads of A,
// the cluster's sum, loads of B, each after the other.  64 tokens of 16 adapters of ranks up to 64 over 3584 -> 2 x 18944
// take 32 us where the bytes take 8: every group of outputs waits once for its weights, and the CTAs of the highest ranks
// end last.  Slower there: weights of all outputs asked into L2 before h (38 us: A waits behind them), a ring of weights
// filled ahead in shared memory by cp.async (38 us: more instructions per output), two tiles of outputs at a time (37 us),
// three CTAs an SM (40 us).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

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
template <bool BF16>
__device__ __forceinline__ void mma_16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// KU: ranks per step of the second product (16 or 32): a lane has KU / 4 consecutive ranks.  OT: tiles of 16 outputs
// whose loads are under way together (2 or 4).  A lane's outputs lie side by side, so that its rows of base and y are read
// and written 16 bytes at a time: row g + 8 r of tile u is output 32 (u / 2) + 4 g + 2 (u % 2) + r.  o_begin .. o_end: this
// CTA's groups of 32 outputs.
template <int WT, int NT, int KU, int OT>
__device__ __forceinline__ void expand(const LoraArgs &a, const LoraTile &tile, int proj, int rank, int o_begin, int o_end,
                                       const int *list, const float *limb, int pitch, const float *unit) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int n_out = a.out[proj];
    const int64_t w0 = (int64_t)max(tile.id, 0) * n_out * a.max_rank;
    int row[NT][2];  // of the two rows that a lane has results of: the outputs of a row lie together
    bool there[NT][2];
    float scale[NT][2];  // (f16 limbs: of h's row)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            there[nt][q] = nt * 8 + 2 * t + q < tile.n;
            row[nt][q] = there[nt][q] ? list[nt * 8 + 2 * t + q] : 0;
            scale[nt][q] = WT == kW16 && rank > 0 ? unit[nt * 8 + 2 * t + q] : 0.f;
        }
#pragma unroll 1
    for (int group = o_begin + warp * (OT / 2); group < o_end; group += kWarps * (OT / 2)) {
        const int o_end1 = min(n_out, o_end * 32);
        auto out_of = [&](int u, int r) { return (group + u / 2) * 32 + 4 * g + 2 * (u % 2) + r; };
        // base and result: [pair of tiles][token][4 outputs]
        float total[OT][NT][4];
        float4 base[OT / 2][NT][2];
#pragma unroll
        for (int v = 0; v < OT / 2; ++v)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int o = out_of(2 * v, 0);
                    base[v][nt][q] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (a.base == nullptr || !there[nt][q]) continue;
                    const float *p = a.base + (int64_t)row[nt][q] * a.base_stride + a.col[proj] + o;
                    if (a.y_vec && o + 3 < o_end1) {
                        base[v][nt][q] = *reinterpret_cast<const float4 *>(p);
                    } else {
                        if (o < o_end1) base[v][nt][q].x = p[0];
                        if (o + 1 < o_end1) base[v][nt][q].y = p[1];
                        if (o + 2 < o_end1) base[v][nt][q].z = p[2];
                        if (o + 3 < o_end1) base[v][nt][q].w = p[3];
                    }
                }
#pragma unroll
        for (int u = 0; u < OT; ++u)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 4; ++q) total[u][nt][q] = 0.f;
#pragma unroll 1
        for (int k0 = 0; k0 < rank; k0 += KU) {
            uint32_t raw[OT][2][8];
            const int k = k0 + t * (KU / 4);
#pragma unroll
            for (int u = 0; u < OT; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) raw[u][r][i] = 0;
                    const int o = out_of(u, r);
                    if (o < o_end1 && k < rank)
                        load_weights<WT, KU / 4>(a.b[proj], w0 + (int64_t)o * a.max_rank + k, raw[u][r]);
                }
            if (k + KU / 4 > rank) {  // what stands behind the last rank is of no meaning
#pragma unroll
                for (int u = 0; u < OT; ++u)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int i = 0; i < KU / 4; ++i)
                            if (k + i >= rank) {
                                if (WT == kW32)
                                    raw[u][r][i] = 0;
                                else
                                    raw[u][r][i / 2] &= i % 2 ? 0x0000FFFFu : 0xFFFF0000u;
                            }
            }
            float acc[OT][NT][4];
#pragma unroll
            for (int u = 0; u < OT; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[u][nt][q] = 0.f;
            if constexpr (WT != kW32) {  // 16-bit limbs: those of a lane's ranks lie together
                constexpr int L = WT == kWB16 ? 3 : 2;
                const uint16_t *l16 = reinterpret_cast<const uint16_t *>(limb);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int l = L - 1; l >= 0; --l) {
                        uint32_t h[4] = {0, 0, 0, 0};
                        const uint16_t *p = l16 + (l * 8 * NT + nt * 8 + g) * pitch + k;
                        if (KU == 32) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(p);
                            h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2 *>(p);
                            h[0] = v.x, h[1] = v.y;
                        }
#pragma unroll
                        for (int j = 0; j < KU / 16; ++j)
#pragma unroll
                            for (int u = 0; u < OT; ++u)
                                mma_16<WT == kWB16>(acc[u][nt], raw[u][0][2 * j], raw[u][1][2 * j], raw[u][0][2 * j + 1],
                                                    raw[u][1][2 * j + 1], h[2 * j], h[2 * j + 1]);
                    }
            } else {
                const float *hi = limb, *lo = limb + 8 * NT * pitch;
#pragma unroll
                for (int j = 0; j < KU / 8; ++j) {
                    float2 h[NT], l[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        h[nt] = *reinterpret_cast<const float2 *>(hi + (nt * 8 + g) * pitch + k + 2 * j);
                        l[nt] = *reinterpret_cast<const float2 *>(lo + (nt * 8 + g) * pitch + k + 2 * j);
                    }
#pragma unroll
                    for (int u = 0; u < OT; ++u) {
                        uint32_t wh[4], wl[4];
                        fragment<WT>(raw[u][0], raw[u][1], j, wh, wl);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_tf32(acc[u][nt], wh, __float_as_uint(l[nt].x), __float_as_uint(l[nt].y));
                            mma_tf32(acc[u][nt], wl, __float_as_uint(h[nt].x), __float_as_uint(h[nt].y));
                            mma_tf32(acc[u][nt], wh, __float_as_uint(h[nt].x), __float_as_uint(h[nt].y));
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < OT; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < 4; ++q) total[u][nt][q] += acc[u][nt][q];
        }
#pragma unroll
        for (int v = 0; v < OT / 2; ++v)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int o = out_of(2 * v, 0);
                    auto sum = [&](float b, int u, int r) {
                        const float d = total[u][nt][2 * r + q];
                        return WT == kW16 ? __fmaf_rn(d, scale[nt][q], b) : b + d;
                    };
                    const float4 z = base[v][nt][q];
                    const float4 w = make_float4(sum(z.x, 2 * v, 0), sum(z.y, 2 * v, 1), sum(z.z, 2 * v + 1, 0), sum(z.w, 2 * v + 1, 1));
                    if (!there[nt][q]) continue;
                    float *p = a.y + (int64_t)row[nt][q] * a.y_stride + a.col[proj] + o;
                    if (a.y_vec && o + 3 < o_end1) {
                        *reinterpret_cast<float4 *>(p) = w;
                    } else {
                        if (o < o_end1) p[0] = w.x;
                        if (o + 1 < o_end1) p[1] = w.y;
                        if (o + 2 < o_end1) p[2] = w.z;
                        if (o + 3 < o_end1) p[3] = w.w;
                    }
                }
    }
}

template <int WT, int NT>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) lora_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int TM = 8 * NT;
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
    const int n32 = (a.out[proj] + 31) / 32;  // this CTA's outputs
    const int o_begin = (int)((uint32_t)n32 * part / parts), o_end = (int)((uint32_t)n32 * (part + 1) / parts);
    const int padded = (a.max_rank + 31) / 32 * 32, pitch = padded + (WT == kW32 ? 4 : 8);
    float *h = smem;                    // [padded][TM], this CTA's share; read by its cluster
    float *limb = smem + padded * TM;   // [limbs][TM][pitch] of h, 16 bits each or 32; before that the warps' sums
    float *sums = limb;                 // [kWarps][kPass][TM]
    __shared__ float unit[TM];          // f16 limbs: what a row of them stands for
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
        // MT tiles of 16 ranks at a time, the loads of UN units of 32 columns under way together
        auto pass = [&](auto mt_, auto un_, int p0) {
            constexpr int MT = decltype(mt_)::value, UN = decltype(un_)::value;
            const int mts = min(MT, (rank - p0 + 15) / 16);
            const int64_t w0 = ((int64_t)tile.id * a.max_rank + p0) * a.in_dim + 8 * t;
            float total[MT][NT][4], acc[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < 4; ++q) total[mt][nt][q] = acc[mt][nt][q] = 0.f;
            int since = 0;
            const int step = parts * kWarps;
#pragma unroll 1
            for (int u0 = part * kWarps + warp; u0 < units; u0 += UN * step) {
                uint32_t raw[UN][MT][2][8];
                float4 x[UN][NT][2];
#pragma unroll
                for (int n = 0; n < UN; ++n) {
                    const int u = u0 + n * step;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int row = mt * 16 + g + 8 * r;
#pragma unroll
                            for (int i = 0; i < 8; ++i) raw[n][mt][r][i] = 0;
                            if (u < units && p0 + row < rank)
                                load_weights<WT, 8>(a.a[proj], w0 + (int64_t)row * a.in_dim + u * 32, raw[n][mt][r]);
                        }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float *p = xr[nt] + u * 32;
                        x[n][nt][0] = x[n][nt][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (u >= units || !there[nt]) continue;
                        if (a.x_vec) {
                            x[n][nt][0] = reinterpret_cast<const float4 *>(p)[0], x[n][nt][1] = reinterpret_cast<const float4 *>(p)[1];
                        } else {
                            x[n][nt][0] = make_float4(p[0], p[1], p[2], p[3]), x[n][nt][1] = make_float4(p[4], p[5], p[6], p[7]);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < UN; ++n) {
                    if (u0 + n * step >= units) break;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float4 c = x[n][nt][0], d = x[n][nt][1];
                        const float v[8] = {c.x, c.y, c.z, c.w, d.x, d.y, d.z, d.w};
                        if constexpr (WT == kWB16) {
                            uint32_t l[3][4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) limbs_b16(v[2 * i], v[2 * i + 1], l[0][i], l[1][i], l[2][i]);
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                if (mt >= mts) break;
#pragma unroll
                                for (int m = 2; m >= 0; --m)
#pragma unroll
                                    for (int j = 0; j < 2; ++j)
                                        mma_16<true>(acc[mt][nt], raw[n][mt][0][2 * j], raw[n][mt][1][2 * j], raw[n][mt][0][2 * j + 1],
                                                     raw[n][mt][1][2 * j + 1], l[m][2 * j], l[m][2 * j + 1]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t h0, h1, l0, l1;
                                limbs(v[2 * j], h0, l0);
                                limbs(v[2 * j + 1], h1, l1);
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    if (mt >= mts) break;
                                    uint32_t wh[4], wl[4];
                                    fragment<WT>(raw[n][mt][0], raw[n][mt][1], j, wh, wl);
                                    mma_tf32(acc[mt][nt], wh, l0, l1);
                                    if (WT == kW32) mma_tf32(acc[mt][nt], wl, h0, h1);
                                    mma_tf32(acc[mt][nt], wh, h0, h1);
                                }
                            }
                        }
                    }
                    if (++since == 2 || n == UN - 1) {
                        since = 0;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    total[mt][nt][q] += acc[mt][nt][q];
                                    acc[mt][nt][q] = 0.f;
                                }
                    }
                }
                since = 0;
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < 4; ++q) total[mt][nt][q] += acc[mt][nt][q];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        *reinterpret_cast<float2 *>(sums + (warp * kPass + mt * 16 + g + 8 * r) * TM + nt * 8 + 2 * t) =
                            make_float2(total[mt][nt][2 * r], total[mt][nt][2 * r + 1]);
            __syncthreads();
#pragma unroll 1
            for (int e = tid; e < mts * 16 * TM; e += kThreads) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) s += sums[w * kPass * TM + e];
                h[p0 * TM + e] = s;
            }
            __syncthreads();
        };
        using std::integral_constant;
        if (rank <= 16)
            pass(integral_constant<int, 1>(), integral_constant<int, NT == 1 ? 4 : NT == 2 ? 2 : 1>(), 0);
        else
#pragma unroll 1
            for (int p0 = 0; p0 < rank; p0 += kPass)
                pass(integral_constant<int, kPass / 16>(), integral_constant<int, NT == 1 && WT != kW32 ? 2 : 1>(), p0);
        if (parts > 1) cl.sync();
        const float scale = a.scale != nullptr ? a.scale[tile.id] : 1.f;
        const int upto = rank <= 16 ? 16 : (rank + 31) / 32 * 32;
        uint16_t *l16 = reinterpret_cast<uint16_t *>(limb);
#pragma unroll 1
        for (int e = tid; e < upto * TM; e += kThreads) {
            const int r = e / TM, tok = e % TM;
            float s = 0.f;
            if (r < rank) {
                if (parts > 1)
                    for (int c = 0; c < parts; ++c) s += *cl.map_shared_rank(h + e, c);
                else
                    s = h[e];
            }
            s *= scale;
            if constexpr (WT == kWB16) {
                uint32_t l[3];
                limbs_b16(s, 0.f, l[0], l[1], l[2]);
#pragma unroll
                for (int i = 0; i < 3; ++i) l16[(i * TM + tok) * pitch + r] = (uint16_t)l[i];
            } else if constexpr (WT == kW16) {
                limb[tok * pitch + r] = s;  // (taken apart below, when the row's largest is known)
            } else {
                uint32_t v0, v1;
                limbs(s, v0, v1);
                limb[tok * pitch + r] = __uint_as_float(v0);
                limb[(TM + tok) * pitch + r] = __uint_as_float(v1);
            }
        }
        if constexpr (WT == kW16) {
            __syncthreads();
            uint16_t *to = reinterpret_cast<uint16_t *>(limb + TM * pitch);
            for (int tok = warp; tok < TM; tok += kWarps) {
                uint32_t top = 0;  // (magnitudes order like their bits)
                for (int r = lane; r < rank; r += 32) top = max(top, __float_as_uint(limb[tok * pitch + r]) & 0x7FFFFFFFu);
                top = __reduce_max_sync(0xffffffffu, top);
                // 2^f with the largest in [2^10, 2^11), within the normal range
                const int f = min(max(264 - (int)(top >> 23), 1), 253);
                const float up = __uint_as_float((uint32_t)f << 23);
                if (lane == 0) unit[tok] = __uint_as_float((uint32_t)(254 - f) << 23);
                for (int r = lane; r < upto; r += 32) {
                    const float v = limb[tok * pitch + r] * up;
                    const __half a0 = __float2half_rn(v);
                    to[tok * pitch + r] = __half_as_ushort(a0);
                    to[(TM + tok) * pitch + r] = __half_as_ushort(__float2half_rn(v - __half2float(a0)));
                }
            }
        }
        __syncthreads();
        if (parts > 1) cl.barrier_arrive();  // (its share is read until all have arrived)
    }
    // (several tiles of outputs at a time where every warp has as many)
    constexpr int OT = NT == 1 && WT != kW32 ? 4 : 2;
    const bool many = OT > 2 && o_end - o_begin >= kWarps * (OT / 2);
    const float *from = limb + (WT == kW16 ? TM * pitch : 0);
    auto go = [&](auto ku) {
        constexpr int KU = decltype(ku)::value;
        if (many)
            expand<WT, NT, KU, OT>(a, tile, proj, rank, o_begin, o_end, list, from, pitch, unit);
        else
            expand<WT, NT, KU, 2>(a, tile, proj, rank, o_begin, o_end, list, from, pitch, unit);
    };
    if (rank <= 16)
        go(std::integral_constant<int, 16>());
    else
        go(std::integral_constant<int, 32>());
    if (rank > 0 && parts > 1) cl.barrier_wait();
}

// h, and the larger of its limbs (f16: with h once more before them) and the warps' sums
size_t smem_bytes(int max_rank, int TM) {
    const int padded = (max_rank + 31) / 32 * 32;
    return sizeof(float) * (padded * TM + std::max(2 * TM * (padded + 8), kWarps * kPass * TM));
}

// The kernel may have what the largest rank takes: the same for every call, so that calls of several threads do not undo it.
template <int WT, int NT>
cudaError_t allow_smem() {
    return cudaFuncSetAttribute(lora_kernel<WT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(kLoraMaxRank, 8 * NT));
}

template <int WT, int NT>
cudaError_t launch(const LoraArgs &a, cudaStream_t s) {
    const size_t smem = smem_bytes(a.max_rank, 8 * NT);
    cudaError_t e = allow_smem<WT, NT>();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    const int chunks = (a.rows - 1) / kLoraChunk + 1;
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

namespace {
// How many clusters of c CTAs run at once, by the rows of a tile (8, 16, 32: two CTAs of an SM, two, one).
int clusters_at_once(int nt, int c, int sms) {
    static std::atomic<int> known[64][3][9];
    const int k = nt == 1 ? 0 : nt == 2 ? 1 : 2;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return std::max(1, sms / c);
    int n = known[dev][k][c].load();
    if (n == 0) {
        const void *f = k == 0   ? (const void *)lora_kernel<kWB16, 1>
                        : k == 1 ? (const void *)lora_kernel<kWB16, 2>
                                 : (const void *)lora_kernel<kWB16, 4>;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(c), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem_bytes(64, 8 * nt);
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {(unsigned)c, 1, 1};
        cfg.attrs = at, cfg.numAttrs = 1;
        const cudaError_t e = k == 0 ? allow_smem<kWB16, 1>() : k == 1 ? allow_smem<kWB16, 2>() : allow_smem<kWB16, 4>();
        if (e != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, f, &cfg) != cudaSuccess || n <= 0) {
            (void)cudaGetLastError();
            n = std::max(1, sms / c);
        }
        known[dev][k][c].store(n);
    }
    return n;
}
}  // namespace

int lora_plan(LoraArgs &a, int type, int distinct, int sms, double &us) {
    const int each = a.rows / distinct, tm = each <= 8 ? 8 : each <= 16 ? 16 : 32;
    const int chunk = std::min(a.rows, kLoraChunk);
    // n rows of d adapters make at most (n + d (tm - 1)) / tm tiles, and about half of those that are not full
    a.chunk_tiles = (int)std::min<int64_t>(chunk, (chunk + (int64_t)distinct * (tm - 1)) / tm);
    const int kinds = std::max(1, std::min(a.n_seqs, a.n_adapters));
    const double tiles = (a.rows > kLoraChunk ? lora_filled(a, tm)
                                              : std::max<double>(std::min(kinds, a.rows), (double)a.rows / tm + kinds / 2)) * a.n_proj;
    const double launched = (double)((a.rows - 1) / kLoraChunk + 1) * a.chunk_tiles * a.n_proj;
    double widest = 0, mean = 0;
    for (int p = 0; p < a.n_proj; ++p) widest = std::max<double>(widest, a.out[p]), mean += (double)a.out[p] / a.n_proj;
    // CTAs per tile: what the rounds of the GPU take in all.
    us = 0;
    for (int c = 1; c <= 8; c += tm < 32 ? c : 1) {
        const int at_once = clusters_at_once(tm / 8, c, sms);
        const double rounds = tiles / at_once;
        double time;
        if (tm < 32) {
            // parts of rounds count, tiles of low rank end early; beside its share a CTA takes as long as 2400 columns (64
            // rows of one adapter of rank 16, 4096 -> 4096 x 3: 41, 25, 17, 12 us with 1, 2, 4, 8)
            time = std::max(1.0, rounds) * ((a.in_dim + 2.0 * widest) / c + 2400.0) * 0.0035;
        } else {
            // us of a CTA, from measured times of 128 rows: a column costs as much up to 16 ranks, and again up to 64
            const double per_in = a.max_rank <= 16 ? 0.0033 : (type == 0 ? 0.0134 : 0.0105) * ((a.max_rank + kPass - 1) / kPass);
            const double per_out = 0.008 + (type == 0 ? 0.0002 : 0.00011) * a.max_rank;
            time = rounds <= 1 ? 1 : kinds == 1 ? std::ceil(rounds) : (rounds + std::ceil(rounds)) / 2;
            time *= 7.5 + lora_search_us(a) + 0.05 * a.max_rank + (per_in * a.in_dim + per_out * (rounds <= 1 ? widest : mean)) / c;
        }
        time += lora_empty_us(a, launched, tiles, at_once);
        if (us == 0 || time < us) us = time, a.cluster = c;
    }
    return tm;
}

cudaError_t lora_launch(const LoraArgs &a, int type, int tile_rows, cudaStream_t s) {
    return type == 0 ? launch<kW32>(a, tile_rows, s) : type == 1 ? launch<kW16>(a, tile_rows, s) : launch<kWB16>(a, tile_rows, s);
}

}  // namespace ql
