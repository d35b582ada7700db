// Low-rank adapters beside a shared projection for prompts: h = scale x A^T, y = base + h B^T over tiles of 128 rows of
// one adapter on tcgen05, one launch.
//
// A cluster of CTAs has a tile: each CTA takes its share of x's columns, all projections' ranks side by side (N of one
// product), adds the shares through distributed shared memory and takes its share of the outputs, 64 at a time.  x, the
// base and y go through memory once.
//
//   h:  a warp's 32 rows of x arrive in blocks of 32 columns; a thread takes its row's values apart into limbs and writes
//       them to tensor memory, the A operand; A's ranks are the B operand in shared memory.
//   y:  h's limbs are the A operand in tensor memory, B's rows the B operand; a warp adds the product to its rows of the
//       base, which arrive as x did, and they leave as a tiled copy.
// bf16 weights: kind::f16, x and h in three bf16 limbs (8 bits each, cut off: together every bit of the value); A goes from
// memory to the operand's place by tiled copies.  f16 and f32 weights: kind::tf32, two limbs (22 bits) of x and h; 4 warps
// widen the weights, f16 to one limb, f32 to two.
//
// The tensor cores cut off what they add up, so a sum over thousands of columns would lose bits in one direction: h's
// accumulators start again every kGroup blocks, in two buffers, and are added up in registers with rounding; beyond 64
// ranks y's lower limbs have accumulators of their own.
//
// Bound: memory, x once in and y once through; 4096 rows of one adapter over 8192 -> 8192 + 1024 + 1024 at rank 64 in bf16
// take 123 us (3.85 TB/s; the bytes alone 72 us): the outputs move 25 bytes a cycle and SM, near what a copy does, h's blocks
// of 32 columns half of that (limbs, products and sums in registers after one another), and some 30000 of 225000 cycles
// pass before the first, between the two and after the last.  Slower: 16 and 24 warps for rows, one CTA for half of a tile
// or two for a pair, limbs made before the wait for their place.
// Roles: 8 warps for rows (two per quarter of the tile, one for even and
// one for odd blocks, then one for each half of 64 outputs), 4 for weights, one that issues the products.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "ql_lora.cuh"
#include "ql_tcgen05.cuh"

namespace ql {
namespace {

constexpr int kThreads = 512, kRowWarps = 8;
constexpr int kTile = kLoraTile, kDepth = 4;   // rows; blocks of a warp in flight and in use
constexpr int kSlice = 64;                     // outputs of one product
constexpr int kSlot = 32 * 128;                // bytes of a warp's block: 32 rows of 32 values; four lie together
constexpr int kMaxRing = 4, kRaw = 4;          // stages of widened weights, and of weights on their way
constexpr int kMaxOut = 8, kAhead = 4;         // stages of 64 rows of B, and how far ahead they are asked for
static_assert(kAhead <= 4, "the waits for copies");
constexpr uint32_t kTries = 1u << 27;          // of a wait, each of 20 cycles or more
constexpr uint32_t kLimbs = 384;               // TMEM columns: h's two accumulators of up to 192, then x's limbs twice
// Registers per thread of the roles; 16 warps launch with 128 each.
constexpr int kRowRegs = 184, kOtherRegs = 72;
static_assert(2 * kRowRegs + 2 * kOtherRegs == 4 * 128, "the block's registers at launch");

struct Bars {
    uint64_t land[2][kDepth], free[2][kDepth];  // blocks of x, then of the base, by half of the row warps
    uint64_t x_full[2], x_empty[2];            // x's limbs, by parity of the block
    uint64_t w_full[kMaxRing], w_empty[kMaxRing];  // stages of A
    uint64_t v_free, v_full[kMaxOut], v_empty[kMaxOut];  // A's stages are all read: B's take their place
    uint64_t sum_full[2], sum_empty[2];        // h's accumulators
    uint64_t h_full;                           // h's limbs
    uint64_t y_full[2], y_empty[2];            // the products of 64 outputs
    uint32_t tmem;
    int abort;
};

// D (+)= A B: A in tensor memory, B in shared memory (K-major rows of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes).
template <bool B16>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    if constexpr (B16)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
            "mov.b64 db, {%2, %5};\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(hi)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
            "mov.b64 db, {%2, %5};\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(hi)
            : "memory");
}
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }
// f32 accumulator, bf16 (1) or tf32 (2) operands, both K-major, M 128.
template <bool B16>
__device__ __forceinline__ uint32_t idesc_of(int n) {
    constexpr uint32_t t = B16 ? 1 : 2;
    return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
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
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const void *map, int c0, int c1, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1), "r"(src)
                 : "memory");
}
template <int N>
__device__ __forceinline__ void stores_read() {  // all but the last N have read their shared memory
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t remote(uint32_t addr, uint32_t rank) {  // the same place in another CTA's shared memory
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 remote_load(uint32_t p) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store(uint32_t p, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// A place in a ring of n and the round that it is in.
struct Turn {
    int at = 0;
    uint32_t round = 0;
    __device__ __forceinline__ void next(int n) {
        if (++at == n) at = 0, ++round;
    }
};

// Where outputs stand: 64 columns from o0 of projection p.
struct Slice {
    int p, o0;
    // the one after j others, of projections p0 .. p0 + np
    __device__ __forceinline__ void seek(const LoraArgs &a, int p0, int np, int j) {
        p = p0;
#pragma unroll
        for (int q = 0; q < kLoraMaxProj - 1; ++q) {
            const int n = (a.out[p] + kSlice - 1) / kSlice;
            if (p < p0 + np - 1 && j >= n) j -= n, ++p;
        }
        o0 = j * kSlice;
    }
    __device__ __forceinline__ void step(const LoraArgs &a) {
        o0 += kSlice;
        if (o0 >= a.out[p]) o0 = 0, p = min(p + 1, kLoraMaxProj - 1);
    }
};
__device__ __forceinline__ int pick(const int (&v)[kLoraMaxProj], int p) { return p == 0 ? v[0] : p == 1 ? v[1] : v[2]; }

template <int WT>
__global__ void __launch_bounds__(kThreads, 1) lora_tiles_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LoraMaps maps) {
    constexpr bool B16 = WT == kWB16;
    constexpr int LW = WT == kW32 ? 2 : 1;  // limbs of a weight
    constexpr int kGroup = 4 / LW;          // blocks of 32 columns between two sums in registers
    constexpr int NC = 6 / LW;              // groups of 16 ranks that a row warp sums, at most
    constexpr int kPer = B16 ? 64 : 32;     // columns of a stage of A, ranks of a stage of B: rows of 128 bytes
    extern __shared__ uint8_t sm_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = sm;                                              // [kDepth][kRowWarps][kSlot]
    uint8_t *weights = sm + kRowWarps * kDepth * kSlot;              // [a.ring][a.ring_bytes]
    float *shares = reinterpret_cast<float *>(sm);                   // [ranks][kTile], between the two products
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
    // n k / parts, n k below 2^29 (a division would take its time several times over before the first load)
    const uint32_t inverse = 0xFFFFFFFFu / (uint32_t)parts + 1;  // (parts 1: 0, and the product itself)
    auto part_of = [&](int n, int k) { return (int)(parts == 1 ? (uint32_t)(n * k) : __umulhi((uint32_t)(n * k), inverse)); };
    int first[kLoraMaxProj], R = 0, slices = 0;  // first rank of each projection, all ranks
#pragma unroll
    for (int p = 0; p < kLoraMaxProj; ++p) {
        first[p] = -1;
        if (p < p0 || p >= p0 + np) continue;
        slices += (a.out[p] + kSlice - 1) / kSlice;
        if (rank > 0 && a.a[p] != nullptr) first[p] = R, R += r16;
    }
    const int blocks = a.in_dim / 32, i0 = part_of(blocks, part);
    const int n_blocks = R > 0 ? part_of(blocks, part + 1) - i0 : 0;
    const int j0 = part_of(slices, part), j1 = part_of(slices, part + 1);
    const int groups = (n_blocks + kGroup - 1) / kGroup;
    // the ranks of h that this CTA's outputs need, and their limbs' columns of tensor memory: all first limbs, all second
    Slice from, to;
    from.seek(a, p0, np, min(j0, slices - 1)), to.seek(a, p0, np, max(j1 - 1, 0));
    int need[kLoraMaxProj], n_need = 0;
#pragma unroll
    for (int p = 0; p < kLoraMaxProj; ++p) {
        need[p] = -1;
        if (j0 < j1 && p >= from.p && p <= to.p && first[p] >= 0) need[p] = n_need, n_need += r16;
    }
    const int limb_cols = B16 ? n_need / 2 : n_need, h_cols = (B16 ? 3 : 2) * limb_cols;
    // the outputs' accumulators at the end of tensor memory, two where h's limbs leave room
    const bool apart = rank > 64;
    const int out_cols = apart ? 2 * kSlice : kSlice, bufs = h_cols + 2 * out_cols <= 512 ? 2 : 1;
    auto out_at = [&](int buf) { return 512u - out_cols * (buf + 1); };

    // Whether the tile's rows lie together: then one warp asks for them in tiled copies of 128 rows (of another sequence's
    // among them where the tile has fewer), and sends y off; else the row warps copy theirs 16 bytes at a time.
    const int row0 = uni(list[0]);
    const bool joint = uni(list[tile.n - 1]) - row0 == tile.n - 1;
    if (warp == 13) {  // (by one thread they took 2000 cycles)
        if (lane < 2 * kDepth) {
            mbar_init(&b.land[0][0] + lane, joint ? 1 : (tile.n + 31) / 32 * 32);
            mbar_init(&b.free[0][0] + lane, 4);
        }
        if (lane < kMaxOut) mbar_init(&b.v_full[lane], 4), mbar_init(&b.v_empty[lane], 1);
        if (lane < kMaxRing) mbar_init(&b.w_full[lane], B16 ? 1 : 4), mbar_init(&b.w_empty[lane], 1);
        if (lane < 2) {
            mbar_init(&b.x_full[lane], 4), mbar_init(&b.x_empty[lane], 1);
            mbar_init(&b.sum_full[lane], 1), mbar_init(&b.sum_empty[lane], kRowWarps);
            mbar_init(&b.y_full[lane], 1), mbar_init(&b.y_empty[lane], kRowWarps);
        }
        if (lane == 0) mbar_init(&b.v_free, 1), mbar_init(&b.h_full, kRowWarps), b.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) tmem_alloc(&b.tmem, 512);
    fence_proxy_async_smem();  // (the search's tables stand where copies will)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uni(b.tmem);
    volatile int *abort_flag = &b.abort;
    // Bounded wait: false, and everybody told, when it ran out (seconds) or another role gave up.  (Few instructions: there
    // are many of these, and the roles' code has to stay in the instruction cache.)
    auto wait = [&](uint64_t *bar, uint32_t parity) {
#pragma unroll 1
        for (uint32_t n = 0; !mbar_try_wait(bar, parity & 1u); ++n)
            if (n >= kTries || *abort_flag) {
                atomicExch(a.err, kErrWaitFull);
                *abort_flag = 1;
                return false;
            }
        return true;
    };

    // a half's 32 of a slice's 64 outputs: the first column of y, and how many there are
    auto col_of = [&](const Slice &s, int half) { return a.col[s.p] + s.o0 + 32 * half; };
    auto width_of = [&](const Slice &s, int half) { return min(32, a.out[s.p] - s.o0 - 32 * half); };
    // slots of the ring that the shares of h take, until its limbs are written
    const int taken = (R * kTile * 4 + kRowWarps * kSlot - 1) / (kRowWarps * kSlot);

    if (warp < kRowWarps) {
        // ------------------------------------ rows: a thread per row and parity ------------------------------------
        reg_inc<kRowRegs>();
        const int q = warp & 3, wg = warp >> 2;
        const int live = max(0, min(32, tile.n - 32 * q));
        uint8_t *mine = ring + warp * kSlot;  // (its slots kRowWarps * kSlot apart)
        const uint32_t lanes = (uint32_t)(32 * q) << 16;
        auto place = [&](int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) * 16)); };
        auto slot_of = [&](int m) { return mine + (m % kDepth) * (kRowWarps * kSlot); };
        int issued = 0, used = 0;  // blocks asked for (by this warp), and taken
        // 32 columns of this warp's rows into the next slot, where the tile's rows do not lie together
        auto fetch = [&](const float *from, int64_t stride, int col, int width) {
            if (live > 0) {
                const uint32_t dst = smem_u32(slot_of(issued));
                const int c = (lane & 7) * 4;
#pragma unroll
                for (int it = 0; it < 8; ++it) {
                    const int r = 4 * it + lane / 8;
                    if (r < live && c < width) copy16(dst + place(r, lane & 7), from + list[32 * q + r] * stride + col + c);
                }
                cp_async_mbar_arrive(&b.land[wg][issued % kDepth]);
            }
            ++issued;
        };
        auto landed = [&] {
            return (!joint && live == 0) || __all_sync(0xffffffffu, wait(&b.land[wg][used % kDepth], used / kDepth));
        };
        auto give_back = [&] {  // the slot in use
            __syncwarp();
            if (joint && lane == 0) mbar_arrive(&b.free[wg][used % kDepth]);
            ++used;
        };
        bool ok = true;
        if (R > 0) {
            float sum[NC][16];
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[c][e] = 0.f;
            int settled = 0;
            auto settle = [&] {  // one more group of blocks
                const int buf = settled & 1;
                if (!__all_sync(0xffffffffu, wait(&b.sum_full[buf], settled >> 1))) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < NC; ++c) {
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
            int asked = wg;  // the next block to ask for
            auto fetch_x = [&] {
                if (!joint && asked < n_blocks) fetch(a.x, a.x_stride, (i0 + asked) * 32, 32);
                asked += 2;
            };
#pragma unroll 1
            for (int k = 0; k < kDepth; ++k) fetch_x();
            float4 v[8];  // this row's part of a block
            auto take = [&] {
                if (!landed()) return false;
                const uint8_t *slot = slot_of(used);
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = *reinterpret_cast<const float4 *>(slot + place(lane, c));
                give_back();
                fetch_x();
                return true;
            };
            if (wg < n_blocks) ok = take();
            const uint32_t limbs_at = tmem + lanes + kLimbs + wg * 64;
#pragma unroll 1
            for (int i = wg; i < n_blocks && ok; i += 2) {
                if (i >= 2) ok = __all_sync(0xffffffffu, wait(&b.x_empty[wg], (i >> 1) - 1));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (B16) {
                        uint32_t l[3][8];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float4 w = v[4 * h + c];
                            limbs_b16(w.x, w.y, l[0][2 * c], l[1][2 * c], l[2][2 * c]);
                            limbs_b16(w.z, w.w, l[0][2 * c + 1], l[1][2 * c + 1], l[2][2 * c + 1]);
                        }
#pragma unroll
                        for (int n = 0; n < 3; ++n) tmem_st8(limbs_at + 16 * n + 8 * h, l[n]);
                    } else {
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float4 w = v[4 * h + c];
                            limbs(w.x, hi[4 * c], lo[4 * c]);
                            limbs(w.y, hi[4 * c + 1], lo[4 * c + 1]);
                            limbs(w.z, hi[4 * c + 2], lo[4 * c + 2]);
                            limbs(w.w, hi[4 * c + 3], lo[4 * c + 3]);
                        }
                        tmem_st16(limbs_at + 16 * h, hi);
                        tmem_st16(limbs_at + 32 + 16 * h, lo);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.x_full[wg]);
                __syncwarp();
                if (i + 2 < n_blocks) ok = take();
                // the groups before this block's
#pragma unroll 1
                while (ok && settled < i / kGroup) ok = settle();
            }
#pragma unroll 1
            while (ok && settled < groups) ok = settle();
            // the CTA's share of h, a rank's rows together; the slots of x are all read by now
            asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int col = (2 * c + wg) * 16;
                if (col < R) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) shares[(col + e) * kTile + 32 * q + lane] = sum[c][e];
                }
            }
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            // Every CTA adds up its share of the ranks, in the order of the CTAs, and hands the sums to all (each reading from
            // all what it needs took longer: four prompts, 896 -> 896 + 128 + 128, 33.8 us against 32.3)
            if (parts > 1) {
                const int r1 = part_of(R, part + 1);
#pragma unroll 1
                for (int r = part_of(R, part) + warp; r < r1; r += 2 * kRowWarps) {  // a warp: two ranks of all rows
                    float4 *mine = reinterpret_cast<float4 *>(shares + r * kTile + 4 * lane);
                    const uint32_t at = smem_u32(mine), next = kRowWarps * kTile * 4;
                    const bool two = r + kRowWarps < r1;
                    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
                    float4 s[2] = {zero, zero};
#pragma unroll 1
                    for (int y = 0; y < parts; y += 4) {  // (four CTAs' loads in flight)
                        float4 v[4][2];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[i][0] = v[i][1] = zero;
                            if (y + i == part) {
                                v[i][0] = mine[0];
                                if (two) v[i][1] = mine[next / 16];
                            } else if (y + i < parts) {
                                const uint32_t p = remote(at, y + i);
                                v[i][0] = remote_load(p);
                                if (two) v[i][1] = remote_load(p + next);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                s[e].x += v[i][e].x, s[e].y += v[i][e].y, s[e].z += v[i][e].z, s[e].w += v[i][e].w;
                    }
                    mine[0] = s[0];
                    if (two) mine[next / 16] = s[1];
#pragma unroll 1
                    for (int y = 0; y < parts; ++y) {
                        if (y == part) continue;
                        const uint32_t p = remote(at, y);
                        remote_store(p, s[0]);
                        if (two) remote_store(p + next, s[1]);
                    }
                }
                __syncwarp();
            }
            cluster_arrive();
            cluster_wait();
            // h's limbs, 16 ranks at a time
            const float scale = a.scale != nullptr ? a.scale[tile.id] : 1.f;
#pragma unroll 1
            for (int c = wg; c * 16 < n_need; c += 2) {
                int col = 0, left = 0;  // where the 16 stand among all ranks, and how many of them are in use
#pragma unroll
                for (int p = 0; p < kLoraMaxProj; ++p)
                    if (need[p] >= 0 && c * 16 >= need[p] && c * 16 < need[p] + r16)
                        col = first[p] + c * 16 - need[p], left = rank - (c * 16 - need[p]);
                float s[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = shares[(col + e) * kTile + 32 * q + lane];
                // (what stands behind the last rank is of no meaning)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = e < left ? s[e] * scale : 0.f;
                uint32_t l[3][16];
                if constexpr (B16) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) limbs_b16(s[2 * e], s[2 * e + 1], l[0][e], l[1][e], l[2][e]);
#pragma unroll
                    for (int i = 0; i < 3; ++i) tmem_st8(tmem + lanes + i * limb_cols + c * 8, l[i]);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) limbs(s[e], l[0][e], l[1][e]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) tmem_st16(tmem + lanes + i * limb_cols + c * 16, l[i]);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.h_full);
            asm volatile("bar.sync 1, 256;" ::: "memory");  // the sums are read: their slots are free
        }
        // outputs: 64 at a time, this warp's 32 rows and half of the columns
        Slice next = from;
        int asked = j0;
        auto fetch_base = [&] {  // the next base to ask for
#pragma unroll 1
            for (; asked < j1 && !joint && a.base != nullptr; ++asked) {
                const int width = width_of(next, wg), col = col_of(next, wg);
                next.step(a);
                if (width > 0) {
                    fetch(a.base, a.base_stride, col, width);
                    ++asked;
                    return;
                }
            }
        };
        if (ok)
#pragma unroll 1
            for (int k = 0; k < kDepth; ++k) fetch_base();
        Turn out;  // of the accumulators
        Slice s = from;
#pragma unroll 1
        for (int j = j0; j < j1 && ok; ++j, s.step(a)) {
            const int col = col_of(s, wg), width = width_of(s, wg);
            const bool any = width > 0, has = pick(need, s.p) >= 0;
            uint8_t *slot = slot_of(used);
            float4 w[8];
            if (any && (joint || a.base != nullptr)) {
                ok = landed();
                if (!ok) break;
            }
            if (any && a.base != nullptr) {
#pragma unroll
                for (int c = 0; c < 8; ++c) w[c] = *reinterpret_cast<const float4 *>(slot + place(lane, c));
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) w[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (has) {
                const int buf = out.at;
                ok = __all_sync(0xffffffffu, wait(&b.y_full[buf], out.round));
                if (!ok) break;
                tc_fence_after();
                uint32_t v[32];
                const uint32_t at = tmem + lanes + out_at(buf) + 32 * wg;
                tmem_ld16(at, v);
                tmem_ld16(at + 16, v + 16);
                if (apart) {
                    uint32_t z[32];
                    tmem_ld16(at + kSlice, z);
                    tmem_ld16(at + kSlice + 16, z + 16);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(z[e]));
                } else {
                    tmem_wait_ld();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.y_empty[buf]);
                out.next(bufs);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    w[c].x += __uint_as_float(v[4 * c]), w[c].y += __uint_as_float(v[4 * c + 1]);
                    w[c].z += __uint_as_float(v[4 * c + 2]), w[c].w += __uint_as_float(v[4 * c + 3]);
                }
            }
            if (any) {
                if (has || a.base == nullptr) {  // (else the slot holds the result)
#pragma unroll
                    for (int c = 0; c < 8; ++c) *reinterpret_cast<float4 *>(slot + place(lane, c)) = w[c];
                }
                if (joint && tile.n == kTile && width == 32) {
                    fence_proxy_async_smem();  // (it is sent off when all four warps have written theirs)
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
                    if (joint) fence_proxy_async_smem();  // (the slot's next content is a copy's)
                }
                give_back();
                fetch_base();
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        reg_dec<128>();
    } else if (warp < 12) {
        // ------------------------------------ weights ------------------------------------
        reg_dec<kOtherRegs>();
        if (R > 0) {
            const int wt = threadIdx.x - 32 * kRowWarps;
            bool ok = true;
            // A chunk of 8 weights (those from `valid` on zero) widened into two 16-byte places of its row of 128 bytes.
            auto put = [&](uint8_t *at_row, int row, int ch, const uint32_t (&w)[8], int valid, int limb) {
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
                    uint8_t *at = at_row + row * 128 + (((2 * ch + h) ^ (row & 7)) * 16);
                    *reinterpret_cast<uint4 *>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (WT == kW32) *reinterpret_cast<uint4 *>(at + limb) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            };
            if constexpr (B16) {
                // A as it stands, 64 columns of 64 or 16 ranks in a copy (ranks not in use among them: their sums are left out)
                if (wt == 0) {
                    const int n = (n_blocks + 1) / 2;
                    int e = 0;
                    Turn w;
#pragma unroll 1
                    for (; e < n; ++e, w.next(a.ring)) {
                        const int st = w.at;
                        if (w.round > 0 && !wait(&b.w_empty[st], w.round - 1)) break;
                        mbar_arrive_expect_tx(&b.w_full[st], R * 128);
                        uint8_t *stage = weights + st * a.ring_bytes;
#pragma unroll
                        for (int p = 0; p < kLoraMaxProj; ++p)
                            if (first[p] >= 0)
#pragma unroll 1
                                for (int r = 0; r < r16;) {
                                    const bool many = r16 - r >= 64;
                                    tma_box2d(stage + (first[p] + r) * 128, many ? &maps.a64[p] : &maps.a16[p], (i0 + 2 * e) * 32,
                                              tile.id * a.max_rank + r, &b.w_full[st]);
                                    r += many ? 64 : 16;
                                }
                    }
                    // never leave with copies in flight
#pragma unroll 1
                    for (int m = max(0, e - a.ring); m < e; ++m)
                        mbar_wait(&b.w_full[m % a.ring], (uint32_t)(m / a.ring) & 1u, nullptr, 0);
                }
                __syncwarp();
            } else {
                // A thread copies its chunks of 8 weights kRaw stages ahead and widens them itself: chunk wt + 128 m is a
                // quarter of row (wt + 128 m) / 4.
                constexpr int kMax = 6 / LW;
                const char *src[kMax];  // null: a row of zeros
#pragma unroll
                for (int m = 0; m < kMax; ++m) {
                    src[m] = nullptr;
#pragma unroll
                    for (int p = 0; p < kLoraMaxProj; ++p) {
                        const int r = ((wt + 128 * m) >> 2) - first[p];
                        if (first[p] >= 0 && r >= 0 && r < rank)
                            src[m] = static_cast<const char *>(a.a[p]) +
                                     (((int64_t)tile.id * a.max_rank + r) * a.in_dim + i0 * 32 + (wt & 3) * 8) * Weight<WT>::bytes;
                    }
                }
                uint8_t *raw = weights + a.ring * a.ring_bytes + wt * 16 * LW;
                auto raw_at = [&](int e, int m) { return raw + (e % kRaw) * a.raw_bytes + m * (128 * 16 * LW); };
                auto fetch = [&](int e) {
                    if (e < n_blocks) {
#pragma unroll
                        for (int m = 0; m < kMax; ++m)
                            if (src[m] != nullptr)
#pragma unroll
                                for (int h = 0; h < LW; ++h)
                                    copy16(smem_u32(raw_at(e, m)) + 16 * h, src[m] + (int64_t)e * 32 * Weight<WT>::bytes + 16 * h);
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
#pragma unroll 1
                for (int e = 0; e < kRaw - 1; ++e) fetch(e);
                Turn t;
#pragma unroll 1
                for (int e = 0; e < n_blocks; ++e, t.next(a.ring)) {
                    const int st = t.at;
                    if (t.round > 0) ok = __all_sync(0xffffffffu, wait(&b.w_empty[st], t.round - 1));
                    if (!ok) break;
                    asm volatile("cp.async.wait_group %0;" ::"n"(kRaw - 2) : "memory");
                    uint8_t *stage = weights + st * a.ring_bytes;
                    uint32_t w[kMax][8];
#pragma unroll
                    for (int m = 0; m < kMax; ++m)
                        if (wt + 128 * m < 4 * R) load_weights<WT, 8>(raw_at(e, m), 0, w[m]);
#pragma unroll
                    for (int m = 0; m < kMax; ++m)
                        if (wt + 128 * m < 4 * R) put(stage, (wt >> 2) + 32 * m, wt & 3, w[m], src[m] != nullptr ? 8 : 0, a.ring_bytes / 2);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&b.w_full[st]);
                    fetch(e + kRaw - 1);
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            cluster_arrive();
            // B: 64 rows and kPer ranks at a time, kAhead stages ahead, in the place of A's stages
            ok = ok && __all_sync(0xffffffffu, wait(&b.v_free, 0));
            constexpr int kBytes = kSlice * 128 * LW, kChunks = B16 ? 4 : 2;  // of a stage; chunks of a thread
            const int n_out = min(kMaxOut, a.ring * a.ring_bytes / kBytes), steps = (rank + kPer - 1) / kPer;
            const int n_ahead = min(kAhead, n_out - 1);
            struct At {  // a stage: its outputs and its step of ranks
                Slice s;
                int j, k;
            };
            At ahead{from, j0, 0};
#pragma unroll 1
            while (ahead.j < j1 && pick(need, ahead.s.p) < 0) ahead.s.step(a), ++ahead.j;
            At here = ahead;
            auto step = [&](At &at) {
                if (++at.k < steps) return;
                at.k = 0;
                do at.s.step(a), ++at.j;
#pragma unroll 1
                while (at.j < j1 && pick(need, at.s.p) < 0);
            };
            // this thread's chunk m of 8 ranks: its row and first rank, null where there is none
            auto chunk = [&](const At &at, int m, int &row, int &ch, int &valid) {
                row = B16 ? (wt >> 3) + 16 * m : (wt >> 2) + 32 * m;
                ch = B16 ? wt & 7 : wt & 3;
                const int o = at.s.o0 + row, r = at.k * kPer + 8 * ch;
                valid = o < a.out[at.s.p] ? rank - r : 0;
                return static_cast<const char *>(a.b[at.s.p]) + (((int64_t)tile.id * a.out[at.s.p] + o) * a.max_rank + r) * Weight<WT>::bytes;
            };
            int asked = 0, e = 0;
            Turn to, in;  // of the stages asked for, and given
            uint8_t *raw = weights + a.ring * a.ring_bytes + wt * 16 * LW;
            auto fetch = [&] {
                if (ahead.j < j1) {
                    const int st = to.at;
                    if (to.round > 0) ok = __all_sync(0xffffffffu, wait(&b.v_empty[st], to.round - 1));
                    if (ok) {
#pragma unroll
                        for (int m = 0; m < kChunks; ++m) {
                            int row, ch, valid;
                            const char *p = chunk(ahead, m, row, ch, valid);
                            if (B16) {  // straight to its place
                                uint8_t *at = weights + st * kBytes + row * 128 + ((ch ^ (row & 7)) * 16);
                                if (valid >= 8) {
                                    copy16(smem_u32(at), p);
                                } else if (ahead.k * kPer + 8 * ch < r16) {  // (what stands behind the last rank is of no meaning)
                                    uint4 w = valid > 0 ? *reinterpret_cast<const uint4 *>(p) : make_uint4(0, 0, 0, 0);
                                    uint32_t *v = &w.x;
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        v[i] = 2 * i + 1 < valid ? v[i] : 2 * i < valid ? v[i] & 0xFFFFu : 0u;
                                    *reinterpret_cast<uint4 *>(at) = w;
                                }
                            } else if (valid > 0) {
#pragma unroll
                                for (int h = 0; h < LW; ++h)
                                    copy16(smem_u32(raw + (asked % (kAhead + 1)) * (kChunks * 128 * 16 * LW) + m * (128 * 16 * LW)) + 16 * h, p + 16 * h);
                            }
                        }
                    }
                    step(ahead), to.next(n_out);
                    ++asked;
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            if (ok)
#pragma unroll 1
                for (int i = 0; i < n_ahead; ++i) fetch();
#pragma unroll 1
            while (ok && here.j < j1) {
                const int st = in.at;
                switch (n_ahead) {  // the oldest of them
                case 4: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
                case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
                case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
                default: asm volatile("cp.async.wait_group 0;" ::: "memory");
                }
                if constexpr (!B16) {
                    uint32_t w[kChunks][8];
                    int row[kChunks], ch[kChunks], valid[kChunks];
#pragma unroll
                    for (int m = 0; m < kChunks; ++m) {
                        chunk(here, m, row[m], ch[m], valid[m]);
                        load_weights<WT, 8>(raw + (e % (kAhead + 1)) * (kChunks * 128 * 16 * LW) + m * (128 * 16 * LW), 0, w[m]);
                    }
#pragma unroll
                    for (int m = 0; m < kChunks; ++m) put(weights + st * kBytes, row[m], ch[m], w[m], valid[m], kBytes / 2);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.v_full[st]);
                ++e;
                step(here), in.next(n_out);
                fetch();
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            cluster_wait();
        }
    } else {
        // (all four warps of a group change their registers at one place)
        reg_dec<kOtherRegs>();
        if (warp == 13) {
            // ------------------------------------ rows that lie together, to and from memory ------------------------------------
            int issued[2] = {0, 0};
            bool ok = true;
            auto load = [&](int half, const CUtensorMap *map, int col) {  // null: the slot only
                const int m = issued[half], st = m % kDepth;
                if (m >= kDepth && !wait(&b.free[half][st], m / kDepth - 1)) return false;
                if (map != nullptr) {
                    mbar_arrive_expect_tx(&b.land[half][st], 4 * kSlot);
                    tma_box2d(ring + (st * kRowWarps + 4 * half) * kSlot, map, col, row0, &b.land[half][st]);
                } else {
                    mbar_arrive(&b.land[half][st]);
                }
                ++issued[half];
                return true;
            };
            Slice next[2] = {from, from};
            int asked[2] = {j0, j0};
            // the next base of a half, unless its slot is one of those below `from_slot`
            auto load_base = [&](int half, int from_slot) {
#pragma unroll 1
                while (asked[half] < j1 && width_of(next[half], half) <= 0) next[half].step(a), ++asked[half];
                if (asked[half] >= j1 || issued[half] % kDepth < from_slot) return false;
                ok = ok && load(half, a.base != nullptr ? &maps.base : nullptr, col_of(next[half], half));
                next[half].step(a), ++asked[half];
                return ok;
            };
            int ahead[2] = {0, 0};
            if (joint && lane == 0) {
#pragma unroll 1
                for (int i = 0; i < n_blocks && ok; ++i) {
                    if (i & 1)
                        ok = load(1, &maps.x, (i0 + i) * 32);
                    else
                        ok = load(0, &maps.x, (i0 + i) * 32);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll 1
                    while (ok && ahead[h] < kDepth && load_base(h, taken)) ++ahead[h];
            }
            __syncwarp();
            if (R > 0) {
                cluster_arrive();
                cluster_wait();
                cluster_arrive();
                cluster_wait();
                ok = __all_sync(0xffffffffu, wait(&b.h_full, 0)) && ok;  // (the sums are read: their slots are free)
                fence_proxy_async_smem();
            }
            if (joint && lane == 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll 1
                    while (ok && ahead[h] < kDepth && load_base(h, 0)) ++ahead[h];
                // A slot is filled again when its store has read it, three stores later.
                int used[2] = {(n_blocks + 1) / 2, n_blocks / 2}, stored = 0;
                unsigned order = 0;  // the halves of the last stores, the latest in bit 0
                Slice s = from;
#pragma unroll 1
                for (int j = j0; j < j1 && ok; ++j, s.step(a)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int width = width_of(s, h);
                        if (width <= 0 || !ok) continue;
                        const int st = used[h] % kDepth;
                        ok = wait(&b.free[h][st], used[h] / kDepth);
                        if (!ok) break;
                        ++used[h], ++stored, order = order << 1 | h;
                        if (tile.n == kTile && width == 32)
                            tma_store_2d(&maps.y, col_of(s, h), row0, smem_u32(ring + (st * kRowWarps + 4 * h) * kSlot));
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        if (stored > 3) {
                            stores_read<3>();
                            if (order >> 3 & 1)
                                load_base(1, 0);
                            else
                                load_base(0, 0);
                        }
                    }
                }
                // never leave with copies in flight
                stores_read<0>();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll 1
                    for (int m = max(0, issued[h] - kDepth); m < issued[h]; ++m)
                        mbar_wait(&b.land[h][m % kDepth], (uint32_t)(m / kDepth) & 1u, nullptr, 0);
            }
            __syncwarp();
        } else {
            // ------------------------------------ products ------------------------------------
            if (R > 0) {
                bool ok = true;
                if (warp == 12) {
                    const uint32_t idesc = idesc_of<B16>(R);
                    Turn w_at;
#pragma unroll 1
                    for (int i = 0; i < n_blocks && ok; ++i) {
                        const int wg = i & 1, g = i / kGroup, buf = g & 1, st = w_at.at;
                        if (i % kGroup == 0 && g >= 2) ok = wait(&b.sum_empty[buf], g / 2 - 1);
                        ok = ok && wait(&b.x_full[wg], i >> 1) && wait(&b.w_full[st], w_at.round);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t d = tmem + buf * (kLimbs / 2), x = tmem + kLimbs + wg * 64;
                            const uint32_t w = desc_lo(smem_u32(weights + st * a.ring_bytes));
                            if constexpr (B16) {
#pragma unroll
                                for (int k = 0; k < 2; ++k)
#pragma unroll
                                    for (int l = 2; l >= 0; --l)
                                        mma<true>(d, x + 16 * l + 8 * k, w + 4 * wg + 2 * k, idesc, i % kGroup != 0 || k != 0 || l != 2);
                            } else {
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    mma<false>(d, x + 32 + 8 * k, w + 2 * k, idesc, i % kGroup != 0 || k != 0);
                                    if (WT == kW32) mma<false>(d, x + 8 * k, w + a.ring_bytes / 32 + 2 * k, idesc, 1);
                                    mma<false>(d, x + 8 * k, w + 2 * k, idesc, 1);
                                }
                            }
                            mma_commit(&b.x_empty[wg]);
                            if (!B16 || wg == 1 || i == n_blocks - 1) mma_commit(&b.w_empty[st]);
                            if (i % kGroup == kGroup - 1 || i == n_blocks - 1) mma_commit(&b.sum_full[buf]);
                            if (i == n_blocks - 1) mma_commit(&b.v_free);
                        }
                        __syncwarp();
                        if (!B16 || wg == 1) w_at.next(a.ring);
                    }
                }
                __syncwarp();
                cluster_arrive();
                cluster_wait();
                cluster_arrive();
                if (warp == 12 && ok) {
                    constexpr int kBytes = kSlice * 128 * LW;
                    const uint32_t idesc = idesc_of<B16>(kSlice);
                    const int n_out = min(kMaxOut, a.ring * a.ring_bytes / kBytes), steps = (rank + kPer - 1) / kPer;
                    const uint32_t second = apart ? kSlice : 0;  // the lower limbs' accumulators
                    Turn in, out;  // the stages of B, and the accumulators
                    Slice s = from;
                    ok = __all_sync(0xffffffffu, wait(&b.h_full, 0));
#pragma unroll 1
                    for (int j = j0; j < j1 && ok; ++j, s.step(a)) {
                        const int h0 = pick(need, s.p);
                        if (h0 < 0) continue;
                        const int buf = out.at;
                        if (out.round > 0) ok = __all_sync(0xffffffffu, wait(&b.y_empty[buf], out.round - 1));
#pragma unroll 1
                        for (int k = 0; k < steps && ok; ++k) {
                            const int st = in.at;
                            ok = __all_sync(0xffffffffu, wait(&b.v_full[st], in.round));
                            if (!ok) break;
                            tc_fence_after();
                            if (elect_one()) {
                                const uint32_t d = tmem + out_at(buf);
                                const uint32_t w = desc_lo(smem_u32(weights + st * kBytes));
                                if constexpr (B16) {
                                    const uint32_t h = tmem + (h0 + 64 * k) / 2;
#pragma unroll
                                    for (int m = 0; m < 4; ++m) {
                                        if (64 * k + 16 * m >= r16) break;
#pragma unroll
                                        for (int l = 2; l >= 0; --l)
                                            mma<true>(d + (l > 0 ? second : 0), h + l * limb_cols + 8 * m, w + 2 * m, idesc,
                                                      k != 0 || m != 0 || (l != 2 && (l != 0 || !apart)));
                                    }
                                } else {
                                    const uint32_t h = tmem + h0 + 32 * k;
#pragma unroll
                                    for (int m = 0; m < 4; ++m) {
                                        if (32 * k + 8 * m >= r16) break;
                                        mma<false>(d + second, h + limb_cols + 8 * m, w + 2 * m, idesc, k + m != 0);
                                        if (WT == kW32) mma<false>(d + second, h + 8 * m, w + kBytes / 32 + 2 * m, idesc, 1);
                                        mma<false>(d, h + 8 * m, w + 2 * m, idesc, k + m != 0 || !apart);
                                    }
                                }
                                mma_commit(&b.v_empty[st]);
                                if (k == steps - 1) mma_commit(&b.y_full[buf]);
                            }
                            __syncwarp();
                            in.next(n_out);
                        }
                        out.next(bufs);
                    }
                }
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

constexpr int kSmem = 224 * 1024;  // of the rings together, at most

// The same for every call, so that calls of several threads do not undo it.
template <int WT>
cudaError_t allow_smem() {
    return cudaFuncSetAttribute(lora_tiles_kernel<WT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 1024 + kSmem);
}

template <int WT>
cudaError_t launch(const LoraArgs &a, const LoraMaps &maps, cudaStream_t s) {
    const int smem = 1024 + kRowWarps * kDepth * kSlot + a.ring * a.ring_bytes + a.raw_total;
    cudaError_t e = allow_smem<WT>();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    const int chunks = (a.rows + kLoraChunk - 1) / kLoraChunk;
    cfg.gridDim = dim3((unsigned)chunks * a.chunk_tiles * a.cluster, (unsigned)(a.split ? a.n_proj : 1), 1);
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

namespace {
// How many clusters of c CTAs the device runs at once (one CTA takes an SM's shared memory; an odd GPC holds fewer).
int clusters_at_once(int c, int sms) {
    static std::atomic<int> known[64][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return std::max(1, sms / c);
    int n = known[dev][c].load();
    if (n == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(c), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = kSmem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {(unsigned)c, 1, 1};
        cfg.attrs = at, cfg.numAttrs = 1;
        if (allow_smem<kWB16>() != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, lora_tiles_kernel<kWB16>, &cfg) != cudaSuccess || n <= 0) {
            (void)cudaGetLastError();
            n = std::max(1, sms / c);
        }
        known[dev][c].store(n);
    }
    return n;
}
}  // namespace

bool lora_tiles_plan(LoraArgs &a, int type, int distinct, int sms, double &us) {
    const int limbs = type == 0 ? 2 : 1, most = 192 / limbs, r16 = (a.max_rank + 15) / 16 * 16;
    a.split = r16 * a.n_proj > most;
    const int ranks = a.split ? r16 : r16 * a.n_proj;
    if (ranks > most || !a.x_vec || !a.y_vec) return false;
    a.ring_bytes = limbs * std::max(ranks, kSlice) * 128;
    a.raw_bytes = (ranks * 4 + 127) / 128 * 128 * 16 * limbs;
    // (bf16: none on the way; others: four stages of A, five of B)
    a.raw_total = type == 2 ? 0 : std::max(kRaw * a.raw_bytes, (kAhead + 1) * 2 * 128 * 16 * limbs);
    a.ring = std::min(kMaxRing, (kSmem - kRowWarps * kDepth * kSlot - a.raw_total) / a.ring_bytes);
    if (a.ring < 2) return false;
    const int chunk = std::min(a.rows, kLoraChunk);
    a.chunk_tiles = (int)std::min<int64_t>(chunk, (chunk + (int64_t)distinct * (kTile - 1)) / kTile);
    // CTAs per tile: what the rounds of the GPU take in all.  us of a CTA, from measured times of 512 rows: what passes before,
    // between and after the products (more with the ranks, whose sums go from CTA to CTA), its columns and its outputs.
    const int grid_y = a.split ? a.n_proj : 1;
    const double tiles = (a.rows > kLoraChunk ? lora_filled(a, kTile) : (a.rows + kTile - 1) / kTile + distinct - 1) * grid_y;
    const int64_t launched = ((int64_t)a.rows + kLoraChunk - 1) / kLoraChunk * a.chunk_tiles;
    double out = 0;
    for (int p = 0; p < a.n_proj; ++p) out += (double)a.out[p] / grid_y;
    const double per_in = type == 0 ? 0.0165 : type == 1 ? 0.022 : 0.0145, per_out = type == 0 ? 0.026 : type == 1 ? 0.027 : 0.024;
    us = 0;
    a.cluster = 1;
    for (int c = 1; c <= std::min(8, a.in_dim / 32); ++c) {
        const int at_once = clusters_at_once(c, sms);
        if (launched * c > INT32_MAX) break;
        const double time = std::ceil(tiles / at_once) *
                                (9.5 + lora_search_us(a) + (type == 0 ? 0.11 : 0.065) * ranks + (per_in * a.in_dim + per_out * out) / c) +
                            lora_empty_us(a, (double)launched * grid_y, tiles, at_once);
        if (us == 0 || time < us) us = time, a.cluster = c;
    }
    return us > 0;
}

cudaError_t lora_tiles_launch(const LoraArgs &a, const LoraMaps &maps, int type, cudaStream_t s) {
    return type == 0 ? launch<kW32>(a, maps, s) : type == 1 ? launch<kW16>(a, maps, s) : launch<kWB16>(a, maps, s);
}

}  // namespace ql
