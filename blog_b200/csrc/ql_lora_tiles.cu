// Low-rank adapters beside a shared projection for prompts: h = scale x A^T, y = base + h B^T over tiles of 128 rows of
// one adapter on tcgen05 (kind::tf32), one launch.
//
// A cluster of CTAs has a tile: each CTA takes its share of x's columns, all projections' ranks side by side (N of one
// product), adds the shares through distributed shared memory and takes its share of the outputs, 64 at a time.  x, the
// base and y go through memory once.
//
//   h:  x arrives by cp.async in blocks of 32 columns, a warp its own 32 rows; a thread takes its row's 32 values apart
//       into two tf32 limbs and writes them to tensor memory, the A operand.  A (f16, bf16: exact in tf32; f32: two
//       limbs) is the B operand in shared memory.
//   y:  h's limbs are the A operand in tensor memory, B's rows the B operand; a warp adds the product to the base, which
//       arrives by cp.async as x did, and writes its rows' 128 bytes together.
//
// The tensor cores cut off what they add up, so a sum over thousands of columns would lose bits in one direction: h's
// accumulators start again every kGroup blocks, in two buffers, and are added up in registers with rounding; y's second
// limbs have accumulators of their own.
//
// Bound: memory, x once in and y once through.  Roles: 8 warps for rows (two per quarter of the tile, one for even and
// one for odd blocks, then one for each half of 64 outputs), 4 that widen weights, one that issues the products.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "ql_lora.cuh"

namespace ql {
namespace {

constexpr int kThreads = 512, kRowWarps = 8;
constexpr int kTile = kLoraTile, kDepth = 4;   // rows; blocks of a warp in flight and in use
constexpr int kSlice = 64;                     // outputs of one product
constexpr int kSlot = 32 * 128;                // bytes of a warp's block: 32 rows of 32 values
constexpr int kMaxRing = 4, kRaw = 4;          // stages of widened weights, and of weights on their way
constexpr uint32_t kLimbs = 384;               // TMEM columns: h's two accumulators of up to 192, then x's limbs twice
// Registers per thread of the roles; 16 warps launch with 128 each.
constexpr int kRowRegs = 184, kOtherRegs = 72;
static_assert(2 * kRowRegs + 2 * kOtherRegs == 4 * 128, "the block's registers at launch");

struct Bars {
    uint64_t land[kRowWarps][kDepth];          // a warp's blocks from memory
    uint64_t x_full[2], x_empty[2];            // x's limbs, by parity of the block
    uint64_t w_full[kMaxRing], w_empty[kMaxRing];
    uint64_t sum_full[2], sum_empty[2];        // h's accumulators
    uint64_t h_full;                           // h's limbs
    uint64_t y_full[2], y_empty[2];            // the products of 64 outputs
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// D (+)= A B: A in tensor memory, B in shared memory (K-major rows of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes).
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(hi)
        : "memory");
}
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }
// f32 accumulator, tf32 operands, both K-major, M 128.
__device__ __forceinline__ uint32_t idesc_of(int n) {
    return (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// 32 lanes x 16 columns; the registers are valid after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e != 0;
}
template <int N>
__device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const void *map, int c0, int c1, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void stores_read() {  // all but the last N have read their shared memory
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 remote(uint32_t addr, uint32_t rank) {  // of another CTA's shared memory
    uint32_t r;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(r) : "memory");
    return v;
}

// Where outputs stand: slice j of the tile's projections p0 .. p0 + np, 64 columns of one projection.
struct Slice {
    int p, o0;
};
__device__ __forceinline__ Slice slice_of(const LoraArgs &a, int p0, int np, int j) {
    int p = p0;
#pragma unroll
    for (int q = 0; q < kLoraMaxProj - 1; ++q) {
        const int n = (a.out[p] + kSlice - 1) / kSlice;
        if (p < p0 + np - 1 && j >= n) j -= n, ++p;
    }
    return {p, j * kSlice};
}

template <int WT>
__global__ void __launch_bounds__(kThreads, 1) lora_tiles_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LoraMaps maps) {
    constexpr int LW = WT == kW32 ? 2 : 1;  // limbs of a weight
    constexpr int kGroup = 4 / LW;          // blocks of 32 columns between two sums in registers
    extern __shared__ uint8_t sm_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = sm;                                              // [kDepth][kRowWarps][kSlot]
    uint8_t *weights = sm + kRowWarps * kDepth * kSlot;              // [a.ring][a.ring_bytes]
    float *shares = reinterpret_cast<float *>(sm);                   // [kTile][ranks], between the two products
    __shared__ Bars b;
    __shared__ int list[kTile];
    auto uni = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
    const int warp = uni(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int parts = a.cluster, part = blockIdx.x % parts;
    // the chunks' first tiles come first: empty ones stand at the end
    const int chunks = (a.rows + kLoraChunk - 1) / kLoraChunk, tile_no = blockIdx.x / parts;
    const int r0 = tile_no % chunks * kLoraChunk;
    const LoraTile tile = find_tile<kThreads>(a, tile_no / chunks, r0, min(kLoraChunk, a.rows - r0), kTile,
                                              *reinterpret_cast<LoraFind *>(sm), list);
    if (tile.n == 0) return;  // (every CTA of the cluster)
    int rank = 0;
    if (tile.id >= 0) {
        rank = a.rank != nullptr ? a.rank[tile.id] : a.max_rank;
        if (rank < 0 || rank > a.max_rank) {
            if (threadIdx.x == 0) atomicExch(a.err, kErrAdapter);
            rank = 0;
        }
    }
    if (rank == 0 && a.y == a.base) return;
    const int p0 = a.split ? blockIdx.y : 0, np = a.split ? 1 : a.n_proj;
    const int r16 = (rank + 15) / 16 * 16;
    int first[kLoraMaxProj], R = 0, slices = 0;  // first rank of each projection, all ranks
#pragma unroll
    for (int p = 0; p < kLoraMaxProj; ++p) {
        first[p] = -1;
        if (p < p0 || p >= p0 + np) continue;
        slices += (a.out[p] + kSlice - 1) / kSlice;
        if (rank > 0 && a.a[p] != nullptr) first[p] = R, R += r16;
    }
    const int blocks = a.in_dim / 32, i0 = (int)((int64_t)blocks * part / parts);
    const int n_blocks = R > 0 ? (int)((int64_t)blocks * (part + 1) / parts) - i0 : 0;
    const int j0 = (int)((int64_t)slices * part / parts), j1 = (int)((int64_t)slices * (part + 1) / parts);
    const int groups = (n_blocks + kGroup - 1) / kGroup;
    // the outputs' accumulators, of first and of second limbs: two pairs where h's limbs leave room, behind them
    const int bufs = 2 * R + 4 * kSlice <= 512 ? 2 : 1;
    auto out_at = [](int buf) { return 512u - 2 * kSlice * (buf + 1); };

    // a row warp's rows: how many there are, and whether they lie together
    const int q32 = (warp & 3) * 32, live = warp < kRowWarps ? max(0, min(32, tile.n - q32)) : 0;
    const int row0 = live > 0 ? uni(list[q32]) : 0;
    const bool together = live > 0 && uni(list[q32 + live - 1]) - row0 == live - 1;
    if (live > 0 && lane < kDepth) mbar_init(&b.land[warp][lane], together ? 1 : 32);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b.x_full[i], 4), mbar_init(&b.x_empty[i], 1);
            mbar_init(&b.sum_full[i], 1), mbar_init(&b.sum_empty[i], kRowWarps);
            mbar_init(&b.y_full[i], 1), mbar_init(&b.y_empty[i], kRowWarps);
        }
        for (int i = 0; i < kMaxRing; ++i) mbar_init(&b.w_full[i], 4), mbar_init(&b.w_empty[i], 1);
        mbar_init(&b.h_full, kRowWarps);
        b.abort = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == 12) tmem_alloc(&b.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uni(b.tmem);
    volatile int *abort_flag = &b.abort;
    // Bounded wait (about 2 s): false, and everybody told, when it ran out or another role gave up.
    auto wait = [&](uint64_t *bar, int phase) {
        if (mbar_try_wait(bar, (uint32_t)phase & 1u)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, (uint32_t)phase & 1u)) {
            if (*abort_flag) return false;
            if (clock64() - t0 > 4000000000ll) {
                atomicExch(a.err, kErrWaitFull);
                *abort_flag = 1;
                return false;
            }
        }
        return true;
    };

    if (warp < kRowWarps) {
        // ------------------------------------ rows: a thread per row and parity ------------------------------------
        reg_inc<kRowRegs>();
        const int q = warp & 3, wg = warp >> 2;
        uint8_t *mine = ring + warp * kSlot;  // (its slots kRowWarps * kSlot apart)
        const uint32_t lanes = (uint32_t)(32 * q) << 16;
        auto place = [&](int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) * 16)); };
        auto slot_of = [&](int m) { return mine + (m % kDepth) * (kRowWarps * kSlot); };
        int issued = 0, used = 0;  // blocks asked for, and taken
        // 32 columns of this warp's rows into the next slot: one tiled copy where the rows lie together (in rows that are
        // another sequence's, too), 16 bytes per lane elsewhere
        auto fetch = [&](const CUtensorMap &map, const float *from, int64_t stride, int col, int width) {
            if (live > 0) {
                uint64_t *bar = &b.land[warp][issued % kDepth];
                const uint32_t dst = smem_u32(slot_of(issued));
                if (together) {
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar, kSlot);
                        tma_box2d(slot_of(issued), &map, col, row0, bar);
                    }
                } else {
                    const int c = (lane & 7) * 4;
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int r = 4 * it + lane / 8;
                        if (r < live && c < width) copy16(dst + place(r, lane & 7), from + list[32 * q + r] * stride + col + c);
                    }
                    cp_async_mbar_arrive(bar);
                }
            }
            ++issued;
        };
        auto landed = [&](int m) {
            return live == 0 || __all_sync(0xffffffffu, wait(&b.land[warp][m % kDepth], m / kDepth));
        };
        bool ok = true;
        // the first of 64 outputs, this warp's 32 of them, and whether there are any
        auto outputs = [&](int j, Slice &s, int &col, int &width) {
            s = slice_of(a, p0, np, j);
            width = min(32, a.out[s.p] - s.o0 - 32 * wg);
            col = a.col[s.p] + s.o0 + 32 * wg;
            return width > 0;
        };
        int asked = j0;  // outputs whose base has been asked for
        int taken = 0;   // slots that the shares of h stand in, until they are read by all (the cluster's second barrier)
        auto free_slots = [&] {
            if (taken == 0) return;
            taken = 0;
            cluster_wait();
            fence_proxy_async_smem();
        };
        auto fetch_base = [&] {
            Slice s;
            int col, width;
            if (asked < j1 && outputs(asked, s, col, width)) {
                if (issued % kDepth < taken) free_slots();
                if (a.base != nullptr)
                    fetch(maps.base, a.base, a.base_stride, col, width);
                else
                    ++issued;
            }
            ++asked;
        };
        if (R > 0) {
            float sum[6][16];
#pragma unroll
            for (int c = 0; c < 6; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[c][e] = 0.f;
            auto fetch_x = [&](int k) {  // block wg + 2 k
                if (wg + 2 * k < n_blocks) fetch(maps.x, a.x, a.x_stride, (i0 + wg + 2 * k) * 32, 32);
            };
            int settled = 0;
            auto settle = [&] {  // one more group of blocks
                const int buf = settled & 1;
                if (!__all_sync(0xffffffffu, wait(&b.sum_full[buf], settled >> 1))) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 6; c += 2) {
                    uint32_t v[2][16];
                    const uint32_t at = tmem + lanes + buf * (kLimbs / 2) + (2 * c + wg) * 16;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if ((2 * (c + i) + wg) * 16 < R) tmem_ld16(at + 32 * i, v[i]);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if ((2 * (c + i) + wg) * 16 < R) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) sum[c + i][e] += __uint_as_float(v[i][e]);
                        }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.sum_empty[buf]);
                ++settled;
                return true;
            };
            for (int k = 0; k < kDepth - 1; ++k) fetch_x(k);
            const uint32_t limbs_at = tmem + lanes + kLimbs + wg * 64;
            for (int k = 0; wg + 2 * k < n_blocks && ok; ++k) {
                ok = landed(k) && (k == 0 || __all_sync(0xffffffffu, wait(&b.x_empty[wg], k - 1)));
                if (!ok) break;
                tc_fence_after();
                const uint8_t *slot = slot_of(k);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float4 v = *reinterpret_cast<const float4 *>(slot + place(lane, 4 * h + c));
                        limbs(v.x, hi[4 * c], lo[4 * c]);
                        limbs(v.y, hi[4 * c + 1], lo[4 * c + 1]);
                        limbs(v.z, hi[4 * c + 2], lo[4 * c + 2]);
                        limbs(v.w, hi[4 * c + 3], lo[4 * c + 3]);
                    }
                    tmem_st16(limbs_at + 16 * h, hi);
                    tmem_st16(limbs_at + 32 + 16 * h, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();  // (every lane has read its row: the slot before this one's may be filled)
                if (lane == 0) mbar_arrive(&b.x_full[wg]);
                ++used;
                fetch_x(k + kDepth - 1);
                // the groups before this block's
                while (ok && settled < (wg + 2 * k) / kGroup) ok = settle();
            }
            while (ok && settled < groups) ok = settle();
            // the CTA's share of h, by rows (4 ranks at a place that neighbours do not have a bank in common with); the
            // slots of x are all read by now
            const int spread = R % 32 == 0 ? 7 : 3;
            auto share_at = [&](int col) { return (32 * q + lane) * R + ((col / 4) ^ (lane & spread)) * 4; };
            asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
            for (int c = 0; c < 6; ++c) {
                const int col = (2 * c + wg) * 16;
                if (col < R) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4 *>(shares + share_at(col + e)) =
                            make_float4(sum[c][e], sum[c][e + 1], sum[c][e + 2], sum[c][e + 3]);
                }
            }
            // meanwhile the base into slots that the shares leave free
            taken = (R * kTile * 4 + kRowWarps * kSlot - 1) / (kRowWarps * kSlot);
            if (ok)
                for (int k = 0; k < kDepth - 1 && issued % kDepth >= taken; ++k) fetch_base();
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            // h's limbs of the projections that this CTA's outputs need, 16 ranks at a time
            const float scale = a.scale != nullptr ? a.scale[tile.id] : 1.f;
            const int pa = j0 < j1 ? slice_of(a, p0, np, j0).p : 0, pb = j0 < j1 ? slice_of(a, p0, np, j1 - 1).p : -1;
            for (int c = wg; c * 16 < R; c += 2) {
                bool need = false;
#pragma unroll
                for (int p = 0; p < kLoraMaxProj; ++p)
                    need |= first[p] >= 0 && p >= pa && p <= pb && c * 16 >= first[p] && c * 16 < first[p] + r16;
                if (!need) continue;
                uint32_t hi[16], lo[16];
                float s[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 0.f;
                for (int y = 0; y < parts; y += 4) {  // (four CTAs' loads in flight)
                    float4 v[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v[i][e] = y + i < parts ? remote(smem_u32(shares + share_at(16 * c + 4 * e)), y + i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[4 * e] += v[i][e].x, s[4 * e + 1] += v[i][e].y, s[4 * e + 2] += v[i][e].z, s[4 * e + 3] += v[i][e].w;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) limbs(s[e] * scale, hi[e], lo[e]);
                tmem_st16(tmem + lanes + c * 16, hi);
                tmem_st16(tmem + lanes + R + c * 16, lo);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.h_full);
            __syncwarp();
            cluster_arrive();  // the shares are read
        }
        // outputs: 64 at a time, this warp's 32 rows and half of the columns
        if (ok)
            while (asked < j0 + kDepth - 1) fetch_base();
        int done = 0;  // products so far
        for (int j = j0; j < j1 && ok; ++j) {
            Slice s;
            int col, width;
            const bool any = outputs(j, s, col, width);
            bool has = false;
#pragma unroll
            for (int p = 0; p < kLoraMaxProj; ++p) has |= p == s.p && first[p] >= 0;
            uint8_t *slot = slot_of(used);
            float4 w[8];
            if (any && a.base != nullptr) {
                ok = landed(used);
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < 8; ++c) w[c] = *reinterpret_cast<const float4 *>(slot + place(lane, c));
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) w[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (has) {
                const int buf = done % bufs;
                ok = __all_sync(0xffffffffu, wait(&b.y_full[buf], done / bufs));
                if (!ok) break;
                tc_fence_after();
                uint32_t v[32], z[32];
                const uint32_t at = tmem + lanes + out_at(buf) + 32 * wg;
                tmem_ld16(at, v);
                tmem_ld16(at + 16, v + 16);
                tmem_ld16(at + kSlice, z);
                tmem_ld16(at + kSlice + 16, z + 16);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.y_empty[buf]);
                ++done;
                auto sum = [&](int e) { return __uint_as_float(v[e]) + __uint_as_float(z[e]); };
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    w[c].x += sum(4 * c), w[c].y += sum(4 * c + 1), w[c].z += sum(4 * c + 2), w[c].w += sum(4 * c + 3);
            }
            if (any) {
                if (has || a.base == nullptr) {  // (else the slot holds the result)
#pragma unroll
                    for (int c = 0; c < 8; ++c) *reinterpret_cast<float4 *>(slot + place(lane, c)) = w[c];
                }
                if (together && live == 32 && width == 32) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tma_store_2d(&maps.y, col, row0, smem_u32(slot));
                } else {
                    __syncwarp();
                    const int c = (lane & 7) * 4;
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int r = 4 * it + lane / 8;
                        if (r < live && c < width)
                            *reinterpret_cast<float4 *>(a.y + list[32 * q + r] * a.y_stride + col + c) =
                                *reinterpret_cast<const float4 *>(slot + place(r, lane & 7));
                    }
                }
                ++used;
            }
            if (lane == 0) stores_read<1>();
            __syncwarp();  // (the slot before this one's is free)
            fetch_base();
        }
        free_slots();
        // never leave with copies in flight
        if (live > 0 && (a.base != nullptr || used < issued))
            for (int m = used; m < issued; ++m) mbar_wait(&b.land[warp][m % kDepth], (uint32_t)(m / kDepth) & 1u, nullptr, 0);
        if (lane == 0) stores_read<0>();
        __syncwarp();
        reg_dec<128>();
    } else if (warp < 12) {
        // ------------------------------------ weights: widened to tf32 ------------------------------------
        reg_dec<kOtherRegs>();
        if (R > 0) {
            const int wt = threadIdx.x - 32 * kRowWarps;
            const int limb_bytes = a.ring_bytes / LW;
            // Stages: this CTA's blocks of A, then 64 rows of B and 32 ranks at a time.  A thread copies its chunks of 8
            // weights kRaw stages ahead and widens them itself: chunk c = wt + 128 m is a quarter of row c / 4.
            const int steps = (rank + 31) / 32, n_chunks = R * 4;
            int n_stages = n_blocks;
            for (int j = j0; j < j1; ++j) n_stages += a.a[slice_of(a, p0, np, j).p] != nullptr ? steps : 0;
            constexpr int kMax = 6 / LW;
            const char *from[kMax];  // null: a row of zeros
#pragma unroll
            for (int m = 0; m < kMax; ++m) {
                from[m] = nullptr;
#pragma unroll
                for (int p = 0; p < kLoraMaxProj; ++p) {
                    const int r = ((wt + 128 * m) >> 2) - first[p];
                    if (first[p] >= 0 && r >= 0 && r < rank)
                        from[m] = static_cast<const char *>(a.a[p]) +
                                  (((int64_t)tile.id * a.max_rank + r) * a.in_dim + i0 * 32 + (wt & 3) * 8) * Weight<WT>::bytes;
                }
            }
            uint8_t *raw = weights + a.ring * a.ring_bytes + wt * 16 * LW;
            auto raw_at = [&](int e, int m) { return raw + (e % kRaw) * a.raw_bytes + m * (128 * 16 * LW); };
            auto copy = [&](uint8_t *dst, const char *src) {
#pragma unroll
                for (int h = 0; h < LW; ++h) copy16(smem_u32(dst) + 16 * h, src + 16 * h);
            };
            // the slice and step of the next stage of B, for the copies and for the widening
            struct At {
                int j, k;
            };
            auto next = [&](At &at) {
                if (++at.k == steps) {
                    at.k = 0;
                    do ++at.j;
                    while (at.j < j1 && a.a[slice_of(a, p0, np, at.j).p] == nullptr);
                }
            };
            At ahead{j0 - 1, steps - 1}, here{j0 - 1, steps - 1};
            next(ahead), next(here);
            auto fetch = [&](int e) {
                if (e < n_blocks) {
#pragma unroll
                    for (int m = 0; m < kMax; ++m)
                        if (from[m] != nullptr) copy(raw_at(e, m), from[m] + (int64_t)e * 32 * Weight<WT>::bytes);
                } else if (e < n_stages) {
                    const Slice s = slice_of(a, p0, np, ahead.j);
                    const int r = 32 * ahead.k + (wt & 3) * 8;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const int o = s.o0 + (wt >> 2) + 32 * m;
                        if (o < a.out[s.p] && r < rank)
                            copy(raw_at(e, m), static_cast<const char *>(a.b[s.p]) +
                                                   (((int64_t)tile.id * a.out[s.p] + o) * a.max_rank + r) * Weight<WT>::bytes);
                    }
                    next(ahead);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            // a chunk of 8 weights, those from `valid` on zero, into two 16-byte places of its row of 128 bytes
            auto put = [&](uint8_t *stage, int m, const uint8_t *src, int valid) {
                uint32_t w[8];
                load_weights<WT, 8>(src, 0, w);
                const int row = (wt >> 2) + 32 * m, ch = wt & 3;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = 4 * h + e < valid ? weight<WT>(w, 4 * h + e) : 0.f;
                        if (WT == kW32)
                            limbs(v, hi[e], lo[e]);
                        else
                            hi[e] = __float_as_uint(v);
                    }
                    uint8_t *at = stage + row * 128 + (((2 * ch + h) ^ (row & 7)) * 16);
                    *reinterpret_cast<uint4 *>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (WT == kW32) *reinterpret_cast<uint4 *>(at + limb_bytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            };
            for (int e = 0; e < kRaw - 1; ++e) fetch(e);
            bool ok = true, passed = false;  // the cluster's barrier between the two products
            auto pass = [&] {
                if (!passed) {
                    __syncwarp();
                    cluster_arrive();
                    cluster_wait();
                    cluster_arrive();
                }
                passed = true;
            };
            for (int e = 0; e < n_stages && ok; ++e) {
                if (e == n_blocks) pass();
                const int st = e % a.ring;
                if (e >= a.ring) ok = __all_sync(0xffffffffu, wait(&b.w_empty[st], e / a.ring - 1));
                if (!ok) break;
                asm volatile("cp.async.wait_group %0;" ::"n"(kRaw - 2) : "memory");
                uint8_t *stage = weights + st * a.ring_bytes;
                if (e < n_blocks) {
#pragma unroll
                    for (int m = 0; m < kMax; ++m)
                        if (wt + 128 * m < n_chunks) put(stage, m, raw_at(e, m), from[m] != nullptr ? 8 : 0);
                } else {
                    const Slice s = slice_of(a, p0, np, here.j);
                    const int valid = rank - 32 * here.k - (wt & 3) * 8;  // (what stands behind the last rank is of no meaning)
#pragma unroll
                    for (int m = 0; m < 2; ++m) put(stage, m, raw_at(e, m), s.o0 + (wt >> 2) + 32 * m < a.out[s.p] ? valid : 0);
                    next(here);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.w_full[st]);
                fetch(e + kRaw - 1);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            pass();
            __syncwarp();
            cluster_wait();
        }
    } else {
        // ------------------------------------ products ------------------------------------
        reg_dec<kOtherRegs>();
        if (R > 0) {
            const int limb = a.ring_bytes / LW / 16;
            int entry = 0;
            bool ok = true;
            if (warp == 12) {
                const uint32_t idesc = idesc_of(R);
                for (int i = 0; i < n_blocks && ok; ++i) {
                    const int wg = i & 1, g = i / kGroup, buf = g & 1, st = entry % a.ring;
                    if (i % kGroup == 0 && g >= 2) ok = wait(&b.sum_empty[buf], g / 2 - 1);
                    ok = ok && wait(&b.x_full[wg], i >> 1) && wait(&b.w_full[st], entry / a.ring);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t d = tmem + buf * (kLimbs / 2), x = tmem + kLimbs + wg * 64;
                        const uint32_t w = desc_lo(smem_u32(weights + st * a.ring_bytes));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            mma(d, x + 32 + 8 * k, w + 2 * k, idesc, i % kGroup != 0 || k != 0);
                            if (WT == kW32) mma(d, x + 8 * k, w + limb + 2 * k, idesc, 1);
                            mma(d, x + 8 * k, w + 2 * k, idesc, 1);
                        }
                        mma_commit(&b.x_empty[wg]);
                        mma_commit(&b.w_empty[st]);
                        if (i % kGroup == kGroup - 1 || i == n_blocks - 1) mma_commit(&b.sum_full[buf]);
                    }
                    __syncwarp();
                    ++entry;
                }
            }
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            cluster_arrive();
            if (warp == 12 && ok) {
                const uint32_t idesc = idesc_of(kSlice);
                const int steps = (rank + 31) / 32;
                int done = 0;
                ok = __all_sync(0xffffffffu, wait(&b.h_full, 0));
                for (int j = j0; j < j1 && ok; ++j) {
                    const Slice s = slice_of(a, p0, np, j);
                    int h0 = -1;
#pragma unroll
                    for (int p = 0; p < kLoraMaxProj; ++p)
                        if (p == s.p) h0 = first[p];
                    if (h0 < 0) continue;
                    const int buf = done % bufs;
                    if (done >= bufs) ok = __all_sync(0xffffffffu, wait(&b.y_empty[buf], done / bufs - 1));
                    for (int k = 0; k < steps && ok; ++k) {
                        const int st = entry % a.ring;
                        ok = __all_sync(0xffffffffu, wait(&b.w_full[st], entry / a.ring));
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t d = tmem + out_at(buf), h = tmem + h0 + 32 * k;
                            const uint32_t w = desc_lo(smem_u32(weights + st * a.ring_bytes));
#pragma unroll
                            for (int m = 0; m < 4; ++m) {
                                if (32 * k + 8 * m >= r16) break;
                                mma(d + kSlice, h + R + 8 * m, w + 2 * m, idesc, k + m != 0);
                                if (WT == kW32) mma(d + kSlice, h + 8 * m, w + limb + 2 * m, idesc, 1);
                                mma(d, h + 8 * m, w + 2 * m, idesc, k + m != 0);
                            }
                            mma_commit(&b.w_empty[st]);
                            if (k == steps - 1) mma_commit(&b.y_full[buf]);
                        }
                        __syncwarp();
                        ++entry;
                    }
                    ++done;
                }
            }
            __syncwarp();
            cluster_wait();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp >= kRowWarps) reg_inc<128>();  // (the rows' warps have given theirs back)
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int WT>
cudaError_t launch(const LoraArgs &a, const LoraMaps &maps, cudaStream_t s) {
    const int smem = 1024 + kRowWarps * kDepth * kSlot + a.ring * a.ring_bytes + kRaw * a.raw_bytes;
    cudaError_t e = cudaFuncSetAttribute(lora_tiles_kernel<WT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    const int chunks = (a.rows + kLoraChunk - 1) / kLoraChunk;
    cfg.gridDim = dim3((unsigned)(chunks * a.chunk_tiles * a.cluster), (unsigned)(a.split ? a.n_proj : 1), 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)a.cluster, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, lora_tiles_kernel<WT>, a, maps);
}
}  // namespace

bool lora_tiles_plan(LoraArgs &a, int type, int distinct, int sms) {
    const int limbs = type == 0 ? 2 : 1, most = 192 / limbs, r16 = (a.max_rank + 15) / 16 * 16;
    a.split = r16 * a.n_proj > most;
    const int ranks = a.split ? r16 : r16 * a.n_proj;
    if (ranks > most || !a.x_vec || !a.y_vec) return false;
    a.ring_bytes = limbs * std::max(ranks, kSlice) * 128;
    a.raw_bytes = std::max((ranks * 4 + 127) / 128, 2) * 128 * 16 * limbs;
    a.ring = std::min(kMaxRing, (224 * 1024 - kRowWarps * kDepth * kSlot - kRaw * a.raw_bytes) / a.ring_bytes);
    const int chunk = std::min(a.rows, kLoraChunk);
    a.chunk_tiles = (int)std::min<int64_t>(chunk, (chunk + (int64_t)distinct * (kTile - 1)) / kTile);
    // CTAs per tile: the fewest rounds of the SMs in all, counting what a CTA takes beside its share (as much as a
    // share of one eighth of 8192 inputs and as many outputs)
    const int64_t tiles = ((int64_t)a.rows + kTile - 1) / kTile * (a.split ? a.n_proj : 1);
    double best = 0;
    a.cluster = 1;
    for (int c = 1; c <= std::min(8, a.in_dim / 32); ++c) {
        int64_t width = a.in_dim;
        for (int p = 0; p < a.n_proj; ++p) width += 2 * a.out[p];
        const double time = (double)((tiles * c + sms - 1) / sms) * ((double)width / c + 3000.0);
        if (best == 0 || time < best) best = time, a.cluster = c;
    }
    return true;
}

cudaError_t lora_tiles_launch(const LoraArgs &a, const LoraMaps &maps, int type, cudaStream_t s) {
    return type == 0 ? launch<kW32>(a, maps, s) : type == 1 ? launch<kW16>(a, maps, s) : launch<kWB16>(a, maps, s);
}

}  // namespace ql
