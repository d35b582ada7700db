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
constexpr int kGroup = 2;                      // blocks of 32 columns between two sums in registers
constexpr int kSlice = 64;                     // outputs of one product
constexpr int kSlot = 32 * 128;                // bytes of a warp's block: 32 rows of 32 values
constexpr int kMaxRing = 4;                    // stages of widened weights
constexpr uint32_t kLimbs = 384;               // TMEM columns: h's two accumulators of up to 192, then x's limbs twice
// Registers per thread of the roles; 16 warps launch with 128 each.
constexpr int kRowRegs = 168, kOtherRegs = 88;
static_assert(2 * kRowRegs + 2 * kOtherRegs == 4 * 128, "the block's registers at launch");

struct Bars {
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
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float remote(uint32_t addr, uint32_t rank) {  // a word of another CTA's shared memory
    uint32_t r;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
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
__global__ void __launch_bounds__(kThreads, 1) lora_tiles_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int LW = WT == kW32 ? 2 : 1;  // limbs of a weight
    extern __shared__ uint8_t sm_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = sm;                                              // [kRowWarps][kDepth][kSlot]
    uint8_t *weights = sm + kRowWarps * kDepth * kSlot;              // [a.ring][a.ring_bytes]
    float *shares = reinterpret_cast<float *>(sm);                   // [ranks][kTile], between the two products
    __shared__ Bars b;
    __shared__ int list[kTile], box[3];
    auto uni = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
    const int warp = uni(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int parts = a.cluster, part = blockIdx.x % parts;
    // the chunks' first tiles come first: empty ones stand at the end
    const int chunks = (a.rows + kLoraChunk - 1) / kLoraChunk, tile_no = blockIdx.x / parts;
    const int r0 = tile_no % chunks * kLoraChunk;
    const LoraTile tile = find_tile<kThreads>(a, tile_no / chunks, r0, min(kLoraChunk, a.rows - r0), kTile,
                                              reinterpret_cast<int *>(sm), list, box);
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

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b.x_full[i], 4), mbar_init(&b.x_empty[i], 1);
            mbar_init(&b.sum_full[i], 1), mbar_init(&b.sum_empty[i], kRowWarps);
            mbar_init(&b.y_full[i], 1), mbar_init(&b.y_empty[i], kRowWarps);
        }
        for (int i = 0; i < kMaxRing; ++i) mbar_init(&b.w_full[i], 4), mbar_init(&b.w_empty[i], 1);
        mbar_init(&b.h_full, kRowWarps);
        b.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
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
        uint8_t *mine = ring + warp * kDepth * kSlot;
        const uint32_t mine32 = smem_u32(mine);
        const uint32_t lanes = (uint32_t)(32 * q) << 16;
        int row_of[8];  // the rows that this lane copies: 8 lanes a row of 128 bytes
#pragma unroll
        for (int it = 0; it < 8; ++it) row_of[it] = 32 * q + 4 * it + lane / 8 < tile.n ? list[32 * q + 4 * it + lane / 8] : -1;
        auto place = [&](int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) * 16)); };
        bool ok = true;
        if (R > 0) {
            float sum[6][16];
#pragma unroll
            for (int c = 0; c < 6; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[c][e] = 0.f;
            auto fetch = [&](int k) {  // block wg + 2 k into slot k
                if (wg + 2 * k < n_blocks) {
                    const uint32_t dst = mine32 + (k % kDepth) * kSlot;
                    const float *src = a.x + (int64_t)(i0 + wg + 2 * k) * 32 + (lane & 7) * 4;
#pragma unroll
                    for (int it = 0; it < 8; ++it)
                        if (row_of[it] >= 0) copy16(dst + place(4 * it + lane / 8, lane & 7), src + row_of[it] * a.x_stride);
                }
                copies_end();
            };
            int settled = 0;
            auto settle = [&] {  // one more group of blocks
                const int buf = settled & 1;
                if (!__all_sync(0xffffffffu, wait(&b.sum_full[buf], settled >> 1))) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 6; ++c) {
                    const int col = (2 * c + wg) * 16;
                    if (col < R) {
                        uint32_t v[16];
                        tmem_ld16(tmem + lanes + buf * (kLimbs / 2) + col, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) sum[c][e] += __uint_as_float(v[e]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.sum_empty[buf]);
                ++settled;
                return true;
            };
            for (int k = 0; k < kDepth - 1; ++k) fetch(k);
            const uint32_t limbs_at = tmem + lanes + kLimbs + wg * 64;
            for (int k = 0; wg + 2 * k < n_blocks && ok; ++k) {
                copies_wait<kDepth - 2>();
                __syncwarp();
                if (k > 0) ok = __all_sync(0xffffffffu, wait(&b.x_empty[wg], k - 1));
                if (!ok) break;
                tc_fence_after();
                const uint8_t *slot = mine + (k % kDepth) * kSlot;
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
                fetch(k + kDepth - 1);
                // the group before this block's
                const int g = (wg + 2 * k) / kGroup;
                while (ok && settled < g) ok = settle();
            }
            copies_wait<0>();
            while (ok && settled < groups) ok = settle();
            // the CTA's share of h, a rank's rows together; the slots of x are all read by now
            asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
            for (int c = 0; c < 6; ++c) {
                const int col = (2 * c + wg) * 16;
                if (col < R) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) shares[(col + e) * kTile + 32 * q + lane] = sum[c][e];
                }
            }
            if (parts > 1) {
                __syncwarp();
                cluster_arrive();
                cluster_wait();
            } else {
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
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
                const uint32_t at = smem_u32(shares + c * 16 * kTile + 32 * q + lane);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 0.f;
                for (int y = 0; y < parts; ++y) {
                    float v[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = remote(at + e * kTile * 4, y);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] += v[e];
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
            if (parts > 1) {  // the shares are read: what follows may take their place
                cluster_arrive();
                cluster_wait();
            } else {
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
        }
        // outputs: 64 at a time, this warp's 32 rows and half of the columns
        auto fetch = [&](int j) {
            if (j < j1 && a.base != nullptr) {
                const Slice s = slice_of(a, p0, np, j);
                const int o = s.o0 + 32 * wg + (lane & 7) * 4;
                if (o < a.out[s.p]) {
                    const uint32_t dst = mine32 + ((j - j0) % kDepth) * kSlot;
                    const float *src = a.base + a.col[s.p] + o;
#pragma unroll
                    for (int it = 0; it < 8; ++it)
                        if (row_of[it] >= 0) copy16(dst + place(4 * it + lane / 8, lane & 7), src + row_of[it] * a.base_stride);
                }
            }
            copies_end();
        };
        for (int k = 0; k < kDepth - 1; ++k) fetch(j0 + k);
        int done = 0;  // products so far
        for (int j = j0; j < j1 && ok; ++j) {
            copies_wait<kDepth - 2>();
            __syncwarp();
            const Slice s = slice_of(a, p0, np, j);
            bool has = false;
#pragma unroll
            for (int p = 0; p < kLoraMaxProj; ++p) has |= p == s.p && first[p] >= 0;
            uint8_t *slot = mine + ((j - j0) % kDepth) * kSlot;
            if (has) {
                const int buf = done % bufs;
                ok = __all_sync(0xffffffffu, wait(&b.y_full[buf], done / bufs));
                if (!ok) break;
                tc_fence_after();
                uint32_t v[32], w[32];
                const uint32_t at = tmem + lanes + out_at(buf) + 32 * wg;
                tmem_ld16(at, v);
                tmem_ld16(at + 16, v + 16);
                tmem_ld16(at + kSlice, w);
                tmem_ld16(at + kSlice + 16, w + 16);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(w[e]));
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.y_empty[buf]);
                ++done;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    float4 *at = reinterpret_cast<float4 *>(slot + place(lane, c));
                    float4 w = a.base != nullptr ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                    w.x += __uint_as_float(v[4 * c]), w.y += __uint_as_float(v[4 * c + 1]);
                    w.z += __uint_as_float(v[4 * c + 2]), w.w += __uint_as_float(v[4 * c + 3]);
                    *at = w;
                }
                __syncwarp();
            }
            const int o = s.o0 + 32 * wg + (lane & 7) * 4;
            if (o < a.out[s.p]) {
                float *dst = a.y + a.col[s.p] + o;
#pragma unroll
                for (int it = 0; it < 8; ++it) {
                    if (row_of[it] < 0) continue;
                    const float4 w = has || a.base != nullptr ? *reinterpret_cast<const float4 *>(slot + place(4 * it + lane / 8, lane & 7))
                                                              : make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4 *>(dst + row_of[it] * a.y_stride) = w;
                }
            }
            __syncwarp();  // (the slot is read)
            fetch(j + kDepth - 1);
        }
        copies_wait<0>();
        reg_dec<128>();
    } else if (warp < 12) {
        // ------------------------------------ weights: widened to tf32 ------------------------------------
        reg_dec<kOtherRegs>();
        const int wt = threadIdx.x - 32 * kRowWarps;
        const int limb_bytes = a.ring_bytes / LW;
        int entry = 0;
        bool ok = true;
        // chunks of 8 weights: chunk c of a row of 4 goes to two 16-byte places of its 128 bytes
        auto put = [&](uint8_t *stage, int c, const uint32_t (&raw)[8]) {
            const int row = c >> 2, ch = c & 3;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = weight<WT>(raw, 4 * h + e);
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
        auto take = [&] {  // the next stage, empty
            const int st = entry % a.ring;
            if (entry >= a.ring) ok = __all_sync(0xffffffffu, wait(&b.w_empty[st], entry / a.ring - 1));
            return weights + st * a.ring_bytes;
        };
        auto give = [&] {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.w_full[entry % a.ring]);
            ++entry;
        };
        if (R > 0) {
            constexpr int kMax = (WT == kW32 ? 96 : 192) / 32;  // chunks of a thread
            uint32_t raw[kMax][8];
            const int n_chunks = R * 4;
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
            auto fetch = [&](int i) {
#pragma unroll
                for (int m = 0; m < kMax; ++m) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) raw[m][e] = 0;
                    if (from[m] != nullptr && i < n_blocks) load_weights<WT, 8>(from[m], (int64_t)i * 32, raw[m]);
                }
            };
            fetch(0);
            for (int i = 0; i < n_blocks && ok; ++i) {
                uint8_t *stage = take();
                if (!ok) break;
#pragma unroll
                for (int m = 0; m < kMax; ++m)
                    if (wt + 128 * m < n_chunks) put(stage, wt + 128 * m, raw[m]);
                fetch(i + 1);  // (under way while the stages are used up)
                give();
            }
            if (parts > 1) {
                __syncwarp();
                cluster_arrive();
                cluster_wait();
                cluster_arrive();
            }
            // 64 rows of B, 32 ranks at a time
            const int steps = (rank + 31) / 32;
            for (int j = j0; j < j1 && ok; ++j) {
                const Slice s = slice_of(a, p0, np, j);
                if (a.a[s.p] == nullptr) continue;
                for (int k = 0; k < steps; ++k) {
                    uint32_t two[2][8];
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const int c = wt + 128 * m, o = s.o0 + (c >> 2), r = 32 * k + (c & 3) * 8;
#pragma unroll
                        for (int e = 0; e < 8; ++e) two[m][e] = 0;
                        if (o < a.out[s.p] && r < rank) {
                            load_weights<WT, 8>(a.b[s.p], ((int64_t)tile.id * a.out[s.p] + o) * a.max_rank + r, two[m]);
                            if (r + 8 > rank) {  // what stands behind the last rank is of no meaning
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    if (r + e >= rank) {
                                        if (WT == kW32)
                                            two[m][e] = 0;
                                        else
                                            two[m][e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
                                    }
                            }
                        }
                    }
                    uint8_t *stage = take();
                    if (!ok) break;
                    put(stage, wt, two[0]);
                    put(stage, wt + 128, two[1]);
                    give();
                }
            }
            if (parts > 1) {
                __syncwarp();
                cluster_wait();
            }
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
            if (parts > 1) {
                __syncwarp();
                cluster_arrive();
                cluster_wait();
                cluster_arrive();
            }
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
            if (parts > 1) {
                __syncwarp();
                cluster_wait();
            }
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
cudaError_t launch(const LoraArgs &a, cudaStream_t s) {
    const int smem = 1024 + kRowWarps * kDepth * kSlot + a.ring * a.ring_bytes;
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
    return cudaLaunchKernelEx(&cfg, lora_tiles_kernel<WT>, a);
}
}  // namespace

bool lora_tiles_plan(LoraArgs &a, int type, int distinct, int sms) {
    const int limbs = type == 0 ? 2 : 1, most = 192 / limbs, r16 = (a.max_rank + 15) / 16 * 16;
    a.split = r16 * a.n_proj > most;
    const int ranks = a.split ? r16 : r16 * a.n_proj;
    if (ranks > most || !a.x_vec || !a.y_vec) return false;
    a.ring_bytes = limbs * std::max(ranks, kSlice) * 128;
    a.ring = std::min(kMaxRing, (224 * 1024 - kRowWarps * kDepth * kSlot) / a.ring_bytes);
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

cudaError_t lora_tiles_launch(const LoraArgs &a, int type, cudaStream_t s) {
    return type == 0 ? launch<kW32>(a, s) : type == 1 ? launch<kW16>(a, s) : launch<kWB16>(a, s);
}

}  // namespace ql
