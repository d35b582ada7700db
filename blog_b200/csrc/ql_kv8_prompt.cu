// Attention over the 8-bit KV cache for prompts: the same function as ql_kv8_attn.cu's, on the 5th-generation
// tensor cores.
//
// A CTA takes 256 rows (query token, head of one KV head's group; the group's heads share every key) as two tiles
// of 128, or one tile at head_dim 256, and walks over the keys 64 at a time with a running maximum and total per row:
//   S = Q K^T       tcgen05.mma, Q and K in shared memory, S (fp32) in TMEM
//   P = 2^(S f - m) one thread per row; f: the block's scale of K x the row's scale; P (f16) over S in TMEM
//   O += P V        tcgen05.mma, P from TMEM, V in shared memory, O (fp32) in TMEM
// S has two buffers, so that a row tile's next scores are computed while it exponentiates these: 2 x (2 x 64 + 128)
// columns are all of TMEM.
// Codes are exact in f16.  bf16 rows: q scaled by a power of two is exact in f16 too, P is rounded to f16's 11
// bits (its result is rounded to 8).  f32 rows: q and P in two f16 limbs, twice the products, fp32 results.
// The scale of V's block is multiplied into P relative to the row's largest such product, as in the split
// kernel, and O is rescaled only when one passes that by 2^7.
//
// Roles, 16 warps: 0-3 and 4-7 a thread per row of tile 0 and 1 (S from TMEM, P to TMEM, the result); 13 copies
// the pages' codes into shared memory (one bulk copy per block and operand), 8-11 turn them into f16 in the layout
// the MMA reads (128-byte swizzle; K with the head dimension contiguous and V too, as the transposed operand), a
// tile ahead; 12 issues the MMAs.
// The rows of the block that is not full make a last tile of 64 keys: their upper f16 limbs, then their lower.
//
// Where the tiles of rows alone would leave SMs idle, the keys are split over the CTAs of a cluster, and their
// sums are joined through distributed shared memory, each CTA finishing its share of the rows.
//
// Bound: the latency of the softmax threads (reading S, one exponential per row and key at 16 per clock and SM, weighing,
// writing P): 3000 clocks per 64 keys of two tiles in bf16 and 5300 in f32, where the products take 1024 and 2048 of the
// tensor cores.  Two softmax warps per scheduler do not hide their own chain: at 2048 tokens 47 to 49 % of the issue slots
// are used, the tensor pipe 31 % (f32) and 23 % (bf16), the exponential unit 18 and 30 %.  28/4/128 heads, 8192 tokens in
// bf16 640 us (751 TFLOP/s of 4 head_dim flops per row and key, 0.45 of a library matrix product's), 2048 tokens in f32
// 99 us (304 TFLOP/s, twice that with both limbs).  Two row tiles, so that one's products run under the other's softmax;
// tiles of 64 keys, so that S has two buffers (tiles of 128 with one: 714 and 110 us).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ql_kv8_limbs.cuh"

namespace cg = cooperative_groups;

namespace ql {
namespace {

constexpr int kThreads = 512;
constexpr int kKeys = 64;    // keys per tile: 2 blocks
constexpr int kTileBlocks = kKeys / kKvBlock;
// Tiles of 128 rows per CTA: two, or one where O takes 256 columns of TMEM.
constexpr int row_tiles(int hd) { return hd <= 128 ? 2 : 1; }

// Registers per thread of the roles; 16 warps launch with 128 each.
constexpr int kSoftmaxRegs = 200, kConvertRegs = 64, kIssueRegs = 48;
static_assert(2 * kSoftmaxRegs + kConvertRegs + kIssueRegs == 4 * 128, "the block's registers at launch");

template <int HD, int LIMBS>
struct Layout {
    static constexpr int A = HD / 64;                        // 128-byte columns of a row
    static constexpr int MT = row_tiles(HD), ROWS = 128 * MT;
    static constexpr int ST = HD <= 128 ? 2 : 1;             // K and V stages, and of their codes
    static constexpr int QT = A * 128 * 128;                 // one limb of one tile of Q
    static constexpr int KV = A * kKeys * 128;               // one stage of K or of V
    static constexpr int RAW = kKeys * HD;                   // a tile's codes of K or of V
    static constexpr int q = 0, k = q + MT * LIMBS * QT, v = k + ST * KV, raw = v + ST * KV, end = raw + 2 * ST * RAW;
    static constexpr int bytes = 1024 + end + 512;
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
// Upper words of the operand descriptors: 128-byte swizzle, the next 8 rows (K-major) or keys (MN-major) 1024
// bytes on.  The lower words: address / 16, and in the upper half the leading byte offset / 16.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// D (+)= A B, A and B in shared memory.
template <bool ADD>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "n"(ADD ? 1 : 0), "r"(kDescHi)
        : "memory");
}
// The same with A in tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// 32 lanes x 32 columns; the registers are valid after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
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
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
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
// One contiguous copy, global to shared memory, its bytes counted on bar (addresses and size multiples of 16).
__device__ __forceinline__ void bulk_copy(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// One lane of a converged warp.
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
// Lower descriptor words.  K-major: 8-row atoms of 1024 B, the leading byte offset unused (1).  MN-major (V, the
// head dimension contiguous): 64 x 8 atoms of 1024 B, the next 64 dimensions `lead` bytes on.
__device__ __forceinline__ uint32_t desc_k(uint32_t a) { return ((a >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t a, uint32_t lead) { return ((a >> 4) & 0x3FFFu) | ((lead >> 4) << 16); }
// Instruction descriptor: f32 accumulator, f16 operands, M 128; bit 16: B is MN-major.
constexpr uint32_t idesc(int n, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ float2 ffma2_of(float2 a, float2 b, float2 c) {
    ffma2(c, a, b);
    return c;
}
template <typename T>
__device__ __forceinline__ void load8(float *x, const T *p, bool vec) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            const uint4 z = *reinterpret_cast<const uint4 *>(p);
            const uint32_t w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4)
                x[i] = p[i];
            else
                x[i] = __bfloat162float(p[i]);
        }
    }
}

// V (2 or 4) elements of one lane's part of a row, as loaded.
template <int V, typename T>
struct Few {
    using P = typename std::conditional<V * sizeof(T) == 16, uint4,
                                        typename std::conditional<V * sizeof(T) == 8, uint2, uint32_t>::type>::type;
    P raw;
    __device__ __forceinline__ void load(const T *p, bool vec, bool there) {
        T e[V];
        if (!there) {
            memset(&raw, 0, sizeof(raw));
        } else if (vec) {
            raw = *reinterpret_cast<const P *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = p[i];
            memcpy(&raw, e, sizeof(raw));
        }
    }
    __device__ __forceinline__ void get(float (&x)[V]) const {
        T e[V];
        memcpy(e, &raw, sizeof(raw));
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (float)e[i];
    }
};

// Hand-overs.  No waiter may fall two phases behind its barrier: what is handed from tile to tile by roles that
// run ahead of one another has a ring.
struct Bars {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t raw_full[2][2], raw_empty[2][2];  // [operand][stage]
    uint64_t s_full[2][2], p_full[2][2];       // [tile of rows][S buffer]
    uint64_t o_full[2];                        // a tile's product with V has been added
    uint64_t scales[4], open_max, done;
    uint32_t tmem;
    int abort;
    // A tile's scales (K's < 0: no such block).  When they are written the scores two tiles before are done, which
    // their rows may be about to read, and no earlier ones: four are in use at most.
    float ks[4][kTileBlocks], vs[4][kTileBlocks], lv[4][kTileBlocks];  // lv: log2 of vs
    int plain[4];   // every block of the tile is there, its scales positive and finite
    unsigned bad;   // tokens of the open block that hold NaN or infinity
};
static_assert(sizeof(Bars) <= 512, "Bars at the end of shared memory");

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ Kv8AttnArgs a) {
    constexpr int LIMBS = sizeof(T) == 4 ? 2 : 1;
    using L = Layout<HD, LIMBS>;
    constexpr int A = L::A, ST = L::ST, MT = L::MT, ROWS = L::ROWS;
    constexpr uint32_t kS = 0, kO = 2 * kKeys, kTile = 256;  // TMEM columns of a tile of rows: S (then P) twice, O
    constexpr int kPitch = HD + 4;                       // floats of a row's sums in shared memory at the end
    static_assert(ROWS * kPitch * 4 <= L::end, "the sums take the operands' place");
    extern __shared__ uint8_t sm_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
    Bars &b = *reinterpret_cast<Bars *>(sm + L::end);

    // (values of the whole warp pass a shuffle, which tells the compiler so: the MMA's operands are uniform registers)
    auto uni = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
    const int warp = uni(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int G = a.n_heads / a.c.kv_heads;
    // grid: the tiles of rows slowest, those that see the most keys first
    const int split = blockIdx.x % a.cluster, kh = blockIdx.x / a.cluster, seq = blockIdx.y;
    const int r_base = (a.row_groups - 1 - (int)blockIdx.z - a.tile0) * ROWS;
    int row0, q_len;
    kv8_rows_of(a.r, seq, row0, q_len);
    const int n_rows = q_len * G;
    if (r_base >= n_rows) return;
    int kv_len = a.r.kv_len[seq];
    if ((unsigned)kv_len > (unsigned)(a.c.max_pages * kKvBlock)) {  // (negative too; the host bounds max_pages)
        if (threadIdx.x == 0) atomicExch(a.c.err, kErrKvPage);
        kv_len = 0;
    }
    // tiles of keys that each tile of rows needs; the open block's, where it is needed, is tile n_closed
    const int blocks = kv_len / kKvBlock, open0 = blocks * kKvBlock, n_closed = (blocks + kTileBlocks - 1) / kTileBlocks;
    int n_tiles[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r1 = min(r_base + 128 * (i + 1), n_rows) - 1;  // the tile's last row
        const int keys = i < MT && r_base + 128 * i < n_rows ? max(0, min(kv_len, kv_len - q_len + r1 / G + 1)) : 0;
        const int bl = min((keys + kKvBlock - 1) / kKvBlock, blocks);
        n_tiles[i] = (bl + kTileBlocks - 1) / kTileBlocks + (keys > open0 ? 1 : 0);
    }
    // this CTA's of them: tiles j0 + jj, jj < n_tiles[i]
    const int n_total = max(n_tiles[0], n_tiles[1]), per = (n_total + a.cluster - 1) / a.cluster, j0 = split * per;
#pragma unroll
    for (int i = 0; i < 2; ++i) n_tiles[i] = max(0, min(n_tiles[i], j0 + per) - j0);
    const int n_all = max(n_tiles[0], n_tiles[1]);
    const int n_c = max(0, min(n_all, n_closed - j0));  // closed tiles among them

    if (threadIdx.x == 0) {
        mbar_init(&b.q_full, ROWS);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b.k_full[i], 4), mbar_init(&b.k_empty[i], 1), mbar_init(&b.v_full[i], 4), mbar_init(&b.v_empty[i], 1);
            for (int k = 0; k < 2; ++k) {
                mbar_init(&b.s_full[i][k], 1), mbar_init(&b.p_full[i][k], 4);
                mbar_init(&b.raw_full[i][k], 1), mbar_init(&b.raw_empty[i][k], 4);
            }
            mbar_init(&b.o_full[i], 1);
        }
        for (int k = 0; k < 4; ++k) mbar_init(&b.scales[k], 1);
        mbar_init(&b.open_max, 4);
        mbar_init(&b.done, 1);
        b.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) tmem_alloc(&b.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uni(b.tmem);
    volatile int *abort_flag = &b.abort;
    // Bounded wait (about 2 s): false, and everybody told, when it ran out or another role gave up.  The limit is by
    // the SM's own clock: a read of the global timer at every hand-over would cost more than the hand-over.
    auto wait = [&](uint64_t *bar, int phase) {
        if (mbar_try_wait(bar, (uint32_t)phase & 1u)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, (uint32_t)phase & 1u)) {
            if (*abort_flag) return false;
            if (clock64() - t0 > 4000000000ll) {
                atomicExch(a.c.err, kErrWaitFull);
                *abort_flag = 1;
                return false;
            }
        }
        return true;
    };

    if (warp < 8) {
        // ------------------------------------ a thread per row ------------------------------------
        reg_inc<kSoftmaxRegs>();
        if (warp < 4 * MT) {
        const int i = warp >> 2, r = threadIdx.x & 127, gr = r_base + 128 * i + r;
        const bool live = gr < n_rows;
        const int tok = live ? gr / G : 0, head = kh * G + (live ? gr % G : 0);
        // the last key that the row sees (past the rows' end: a row of zeros, kept on the others' paths)
        const int pos = live ? kv_len - q_len + tok : kv_len - 1;
        float row_scale = 0.f;
        {
            // Q: the warp's 32 rows one after another, a row over the lanes, 16 rows' loads in flight
            constexpr int V = HD / 32, B = 16;
            const int64_t mine = (int64_t)(row0 + tok) * a.q_stride + (int64_t)head * HD;
#pragma unroll 1
            for (int k0 = 0; k0 < 32; k0 += B) {
                Few<V, T> raw[B];
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    const T *q = static_cast<const T *>(a.q) + __shfl_sync(0xffffffffu, mine, k0 + k) + lane * V;
                    raw[k].load(q, a.vec, r_base + 128 * i + 32 * (warp & 3) + k0 + k < n_rows);
                }
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    float x[V], inv;
                    raw[k].get(x);
                    uint32_t bits = 0;  // (magnitudes order like their bits; NaN above all)
#pragma unroll
                    for (int e = 0; e < V; ++e) bits = max(bits, __float_as_uint(fabsf(x[e])));
                    const float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, bits));
                    // (a negative softmax scale: its sign goes to q, so that scores and products order alike)
                    const float f = copysignf(limb_scale(amax, inv), a.scale_log2);
                    if (lane == k0 + k) row_scale = fabsf(a.scale_log2) * (amax > 0.f ? inv : 1.f);
                    const int rr = 32 * (warp & 3) + k0 + k, d = lane * V;
                    uint8_t *p = sm + L::q + i * L::QT + d / 64 * (128 * 128) + rr * 128 + ((d / 8 & 7) ^ (rr & 7)) * 16 + d % 8 * 2;
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        uint32_t hi, lo;
                        split_f16(x[2 * e] * f, x[2 * e + 1] * f, hi, lo);
                        reinterpret_cast<uint32_t *>(p)[e] = hi;
                        if (LIMBS == 2) reinterpret_cast<uint32_t *>(p + MT * L::QT)[e] = lo;
                    }
                }
            }
        }
        fence_proxy_async_smem();
        mbar_arrive(&b.q_full);

        const uint32_t tS0 = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + i * kTile + kS, tO = tS0 - kS + kO;
        float m = -INFINITY, l = 0.f, h = -INFINITY, wf = 0.f;  // (as in the split kernel; wf: its w)
        const int n = n_tiles[i];
        bool ok = true;
        float acc[LIMBS == 2 ? HD : 1];  // f32 rows: the sum over tiles, see below
        if constexpr (LIMBS == 2) {
#pragma unroll
            for (int e = 0; e < HD; ++e) acc[e] = 0.f;
        }
        // The tensor cores truncate when they accumulate, so a sum over thousands of keys in TMEM would lose
        // bits in one direction.  For f32 rows a tile's product starts from zero and is added here, rounded.
        auto add_tile = [&](float z) {  // z: the unit of the rows' weights has changed since
            if constexpr (LIMBS == 2) {
                const float2 z2 = make_float2(z, z);
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(tO + 32 * c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 x = ffma2_of(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), z2,
                                                  make_float2(acc[32 * c + e], acc[32 * c + e + 1]));
                        acc[32 * c + e] = x.x, acc[32 * c + e + 1] = x.y;
                    }
                }
            }
        };
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const uint32_t tS = tS0 + (j & 1) * kKeys;
            ok = __all_sync(0xffffffffu, wait(&b.scales[j & 3], j >> 2) && wait(&b.s_full[i][j & 1], j >> 1));
            if (!ok) break;
            tc_fence_after();
            const bool open = j0 + j == n_closed;
            // the last key of the tile that the row sees (a closed tile ends with the closed blocks)
            const int see = open ? pos - open0 : min(pos, open0 - 1) - (j0 + j) * kKeys;
            const float *ks = b.ks[j & 3], *vs = b.vs[j & 3], *lv = b.lv[j & 3];
            // (per warp) ordinary: all of the tile's scales are positive and finite
            const bool masked = __any_sync(0xffffffffu, see < kKeys - 1);
            bool plain = b.plain[j & 3] && a.scale_log2 != 0.f;
            if (plain && masked) {  // hidden scores have to end far below the others
                const float least = fminf(ks[0], ks[1]) * row_scale;
                plain = __all_sync(0xffffffffu, least > 1e-30f);
            }

            // Largest score of each block.
            float t[kTileBlocks] = {-INFINITY, -INFINITY};
            // GR products from column GR u, as they came; the open block's: the two limbs' sums
            constexpr int GR = LIMBS == 2 ? 16 : 32;
            auto raw = [&](int u, uint32_t *s) {
                auto ld = [](uint32_t at, uint32_t *v) {
                    if constexpr (GR == 16)
                        tmem_ld16(at, v);
                    else
                        tmem_ld32(at, v);
                };
                ld(tS + GR * u, s);
                if (open) {
                    uint32_t s1[GR];
                    ld(tS + 32 + GR * u, s1);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < GR; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) + __uint_as_float(s1[e]));
                } else {
                    tmem_wait_ld();
                }
            };
            auto hide = [&](int first, int count, uint32_t *s) {  // keys not seen: the lowest finite (x f below: plain)
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (e < count && first + e > see) s[e] = 0xFF7FFFFFu;
            };
            auto top32 = [](const uint32_t *s) {
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e & 3] = fmaxf(x[e & 3], __uint_as_float(s[e]));
                return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            };
            const int grains = (open ? kKvBlock : kKeys) / GR;
            const unsigned bad = open ? b.bad : 0;
            // Whether a score, or a score and log2 of its value's scale, has passed what the weights stand in relation to
            // by more than the headroom, in some row of the warp; and if so, the new relation and z, the factor of the
            // sums so far.
            float z = 1.f;
            auto exceeds = [&]() {
                return __any_sync(0xffffffffu, fmaxf(t[0], t[1]) > m + kHeadroom ||
                                                   fmaxf(t[0] + lv[0], t[1] + lv[1]) - m > h + kHeadroom);
            };
            auto settle = [&]() {
                const float top = fmaxf(t[0], t[1]);
                if (top > m) {
                    const float x = ceilf(top);
                    l *= ex2(m - x);
                    h -= x - m;
                    m = x;
                }
                const float u = ceilf(fmaxf(t[0] - m + lv[0], t[1] - m + lv[1]));  // of the heaviest weight x scale
                if (u > h) {
                    z = ex2(h - u);
                    h = u;
                }
                wf = weight_unit(h);
                if (!__any_sync(0xffffffffu, z != 1.f)) return true;
                if constexpr (LIMBS == 2) {
#pragma unroll
                    for (int e = 0; e < HD; ++e) acc[e] *= z;
                } else if (j > 0) {  // (the product before is the last so far: this tile's waits for its weights)
                    if (!__all_sync(0xffffffffu, wait(&b.o_full[i], j - 1))) return false;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tO + 32 * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * z);
                        tmem_st32(tO + 32 * c, o);
                    }
                }
                return true;
            };
            auto is_deep = [&]() { return __any_sync(0xffffffffu, (h < kDeep || m > kHuge || m < -kHuge) && h != -INFINITY); };
            bool weighed = false;
            if constexpr (LIMBS == 1) {
                if (plain && !is_deep()) {
                    // bf16 rows: all 64 scores in registers, their weights computed in the relation that stands, their
                    // maxima beside; seldom, when these exceed it, once more.
                    uint32_t s[kKeys];
#pragma unroll
                    for (int c = 0; c < kTileBlocks; ++c) tmem_ld32(tS + 32 * c, s + 32 * c);
                    tmem_wait_ld();
                    if (masked) {
                        hide(0, 32, s);
                        hide(32, 32, s + 32);
                    }
#pragma unroll 1
                    for (int again = 0; again < 2; ++again) {
                        uint32_t w[kKeys / 2];
                        float2 sum = make_float2(0.f, 0.f);
                        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
                        for (int c = 0; c < kTileBlocks; ++c) {
                            const float f = ks[c] * row_scale, g = vs[c] * wf;
                            const float2 f2 = make_float2(f, f), b2 = make_float2(-base, -base), g2 = make_float2(g, g);
                            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                const float2 v = make_float2(__uint_as_float(s[32 * c + e]), __uint_as_float(s[32 * c + e + 1]));
                                const float2 d = ffma2_of(v, f2, b2), p = make_float2(ex2(d.x), ex2(d.y));
                                top[0] = fmaxf(top[0], v.x), top[1] = fmaxf(top[1], v.y);
                                sum = fadd2(sum, p);
                                const float2 x = fmul2(p, g2);
                                w[16 * c + e / 2] = pack_f16(x.x, x.y);
                            }
                            t[c] = 32 * c > see ? -INFINITY : fmaxf(top[0], top[1]) * f;
                        }
                        if (!exceeds()) {
                            tmem_st32(tS, w);
                            l += sum.x + sum.y;
                            weighed = true;
                            break;
                        }
                        if (!(ok = settle()) || is_deep()) break;
                    }
                }
                if (!ok) break;
            }
            if (!weighed) {
            if (LIMBS == 2 && plain) {
#pragma unroll
                for (int c = 0; c < kTileBlocks; ++c) {
                    uint32_t s[32];
                    tmem_ld32(tS + 32 * c, s);
                    tmem_wait_ld();
                    if (masked) hide(32 * c, 32, s);
                    t[c] = 32 * c > see ? -INFINITY : top32(s) * (ks[c] * row_scale);
                }
            } else {
                t[0] = t[1] = -INFINITY;
#pragma unroll 1
                for (int u = 0; u < grains; ++u) {
                    uint32_t s[GR];
                    raw(u, s);
                    const int c = u * GR / 32;
                    const float f = ks[c] * row_scale;
                    float x = -INFINITY;
#pragma unroll
                    for (int e = 0; e < GR; ++e)
                        if (GR * u + e <= see && !(bad >> (GR * u + e & 31) & 1)) x = fmaxf(x, __uint_as_float(s[e]));
                    x = x == -INFINITY || f < 0.f ? -INFINITY : x * f;
#pragma unroll
                    for (int k = 0; k < kTileBlocks; ++k)
                        if (k == c) t[k] = fmaxf(t[k], x);
                }
            }
            if (exceeds() && !(ok = settle())) break;
            const float base = m == -INFINITY ? 0.f : m;
            const bool deep = is_deep();
            float2 sum = make_float2(0.f, 0.f);
            // Weights take the place of scores: one limb, 16 columns per 32 keys from column 16 c; two limbs, 8 of the
            // upper and 8 of the lower per 16 keys from column 16 u.
            auto put = [&](int u, const uint32_t *w) {
                tmem_st16(tS + 16 * u, w);
                if (open) tmem_st16(tS + (GR == 16 ? 32 : 16) + 16 * u, w);  // the values' lower limbs: the same weights
            };
            if (LIMBS == 2 && plain && !deep) {
#pragma unroll 1
                for (int c = 0; c < kTileBlocks; ++c) {
                    uint32_t s[32];
                    tmem_ld32(tS + 32 * c, s);
                    const float f = ks[c] * row_scale, g = vs[c] * wf, f_lo = fmaf(ks[c], row_scale, -f);
                    const float2 f2 = make_float2(f, f), fl2 = make_float2(f_lo, f_lo), b2 = make_float2(-base, -base);
                    const float2 g2 = make_float2(g, g);
                    tmem_wait_ld();
                    if (masked) hide(32 * c, 32, s);
#pragma unroll
                    for (int u = 0; u < 32; u += 16) {
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 v = make_float2(__uint_as_float(s[u + e]), __uint_as_float(s[u + e + 1]));
                            // (the scale's own rounding is added back)
                            const float2 d = ffma2_of(v, fl2, ffma2_of(v, f2, b2)), p = make_float2(ex2(d.x), ex2(d.y));
                            sum = fadd2(sum, p);
                            const float2 x = fmul2(p, g2);
                            split_f16(x.x, x.y, w[e / 2], w[8 + e / 2]);
                        }
                        tmem_st16(tS + 32 * c + u, w);
                    }
                }
            } else {
                // (the open block, scales of zero or NaN, pages that are not there, rows whose heaviest keys have no value)
#pragma unroll 1
                for (int u = 0; u < grains; ++u) {
                    uint32_t s[GR], w[16];
                    raw(u, s);
                    const int c = u * GR / 32;
                    const float f = ks[c] * row_scale, f_lo = LIMBS == 2 ? fmaf(ks[c], row_scale, -f) : 0.f;
                    const float g = vs[c] * wf, nan = __int_as_float(0x7FC00000);
                    const int last = f < 0.f ? -1 : see - GR * u;
                    const bool huge = fabsf(base) > kHuge;
#pragma unroll
                    for (int e = 0; e < GR; ++e) {
                        const float v = __uint_as_float(s[e]);
                        float d = huge ? __fsub_rn(__fmul_rn(v, f), base) : fmaf(v, f, -base);
                        if (LIMBS == 2 && !huge) d = fmaf(v, f_lo, d);
                        if (bad >> (GR * u + e & 31) & 1) d = nan;
                        s[e] = __float_as_uint(e <= last ? d : -INFINITY);
                    }
                    if (!deep) {
#pragma unroll
                        for (int e = 0; e < GR; ++e) {
                            const float p = ex2(__uint_as_float(s[e]));
                            sum.x += p;
                            s[e] = __float_as_uint(e <= last ? p * g : 0.f);  // (nor may a NaN scale reach others)
                        }
                    } else {
                        const bool lift = h != -INFINITY;
                        const float gl = lift ? vs[c] * ex2(kWBits) : g, up = lift ? h : 0.f;
                        // (huge scores: h says nothing of the values' scale any more, so their product is kept in f16 by
                        // itself; NaN stays)
                        const float most = fminf(126.f, kHeadroom + 0.9f - lv[c]);
#pragma unroll
                        for (int e = 0; e < GR; ++e) {
                            const float d = __uint_as_float(s[e]);
                            sum.x += ex2(d);
                            s[e] = __float_as_uint(e <= last ? ex2(fminf(d - up, most)) * gl : 0.f);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < GR; e += 2) {
                        if (LIMBS == 2)
                            split_f16(__uint_as_float(s[e]), __uint_as_float(s[e + 1]), w[e / 2], w[8 + e / 2]);
                        else
                            w[e / 2] = pack_f16(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                    }
                    put(u, w);
                }
            }
            l += sum.x + sum.y;
            }
            if (LIMBS == 2 && j > 0) {  // the tile before's product, ere this one's takes its place
                ok = __all_sync(0xffffffffu, wait(&b.o_full[i], j - 1));
                if (!ok) break;
                tc_fence_after();
                add_tile(z);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.p_full[i][j & 1]);
        }
        if (n > 0) {
            ok = __all_sync(0xffffffffu, ok && wait(&b.o_full[i], n - 1));
            tc_fence_after();
            add_tile(1.f);
        }
        // Every product of the CTA has been computed: Q, K and V make way for the rows' sums, x 2^(h - kWBits) (the
        // power in two steps where it leaves the range), their maxima and totals.
        ok = __all_sync(0xffffffffu, wait(&b.done, 0) && ok);
        const float e0 = h - kWBits, u0 = h == -INFINITY ? 0.f : ex2(fmaxf(e0, -120.f));
        const float u1 = h == -INFINITY ? 1.f : ex2(fminf(e0 + 120.f, 0.f));
        float *row = reinterpret_cast<float *>(sm) + (128 * i + r) * kPitch;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            if constexpr (LIMBS == 2) {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(acc[32 * c + e]);
            } else if (n > 0) {
                tmem_ld32(tO + 32 * c, o);
                tmem_wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = n > 0 ? __uint_as_float(o[e + k]) * u0 * u1 : 0.f;
                *reinterpret_cast<float4 *>(row + 32 * c + e) = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
        row[HD] = m;
        row[HD + 1] = l;
        }
        reg_dec<128>();  // as launched: the others take theirs back when all rows' warps have come here
    } else if (warp < 12) {
        // ------------------------------------ codes to f16 ------------------------------------
        reg_dec<kConvertRegs>();
        const int w = warp - 8;
        // Pieces of 16 codes, 32 to a warp access.  A phase's 8 lanes hold four pieces of two rows: of different
        // halves of the rows where these are 128 bytes, so that the reads meet distinct banks, and the rows'
        // swizzles differ, so that the writes do.
        constexpr int RPI = 8 / A;            // rows per warp access
        constexpr int U = kKeys / (4 * RPI);  // accesses per warp, operand and tile
        const int pc = lane & 3, rb = (lane >> 2) & 1, at = (lane >> 3) % A ^ (A >= 2 ? rb : 0), rl = rb + 2 * ((lane >> 3) / A);
        auto row_of = [&](int u) { return (u * 4 + w) * RPI + rl; };
        bool ok = true;
        auto full = [&](uint64_t *bar) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto empty = [&](uint64_t *bar, int j) {  // the stage's former tile has been read
            return j < ST || __all_sync(0xffffffffu, wait(bar, j / ST - 1));
        };
        auto convert = [&](int op, int j, uint64_t *stage_empty, uint8_t *tile) {
            if (!__all_sync(0xffffffffu, wait(&b.raw_full[op][j % ST], j / ST))) return false;
            const uint8_t *src = sm + L::raw + (op * ST + j % ST) * L::RAW + (at * 4 + pc) * 16;
            uint8_t *p = tile + at * (kKeys * 128);
            if (!empty(stage_empty, j)) return false;
            constexpr int H = U < 4 ? U : 4;
#pragma unroll
            for (int u0 = 0; u0 < U; u0 += H) {
                uint4 raw[H];
#pragma unroll
                for (int u = 0; u < H; ++u) raw[u] = *reinterpret_cast<const uint4 *>(src + row_of(u0 + u) * HD);
#pragma unroll
                for (int u = 0; u < H; ++u) {
                    const uint32_t z[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                    uint32_t h[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[2 * e] = codes2(z[e], 0x4140);
                        h[2 * e + 1] = codes2(z[e], 0x4342);
                    }
                    const int row = row_of(u0 + u);
                    *reinterpret_cast<uint4 *>(p + row * 128 + ((2 * pc) ^ (row & 7)) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(p + row * 128 + ((2 * pc + 1) ^ (row & 7)) * 16) = make_uint4(h[4], h[5], h[6], h[7]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.raw_empty[op][j % ST]);
            return true;
        };
        // scales of a tile's blocks (lanes 0 .. 3 of the first warp)
        float next_ks = -1.f, next_vs = 0.f;
        auto scales = [&](int j) {
            if (w != 0 || lane >= kTileBlocks) return;
            const int block = (j0 + j) * kTileBlocks + lane;
            if (block >= blocks) {  // past the closed blocks: all of its keys are hidden by their position
                next_ks = next_vs = 1.f;
                return;
            }
            const int c = kv8_page(a.c, seq, block);
            const int64_t z = (int64_t)c * a.c.kv_heads + kh;
            // (no such page: its keys are hidden by the sign)
            next_ks = c >= 0 ? a.c.k_scale[z] : -1.f;
            next_vs = c >= 0 ? a.c.v_scale[z] : 0.f;
        };
        // K two tiles ahead of V, as the MMAs take them: the scores of tile j + 2 follow the values of tile j.
        auto convert_k = [&](int j) {
            const int st = j % ST;
            if (j >= n_c) return true;
            if (!convert(0, j, &b.k_empty[st], sm + L::k + st * L::KV)) return false;
            full(&b.k_full[st]);
            if (w == 0) {
                const bool good = next_ks > 0.f && next_ks < INFINITY && next_vs > 0.f && next_vs < INFINITY;
                const unsigned all = __ballot_sync(0xffffffffu, good || lane >= kTileBlocks);
                if (lane < kTileBlocks) {
                    b.ks[j & 3][lane] = next_ks;
                    b.vs[j & 3][lane] = next_vs;
                    b.lv[j & 3][lane] = log2f(next_vs);
                }
                if (lane == 0) b.plain[j & 3] = all == 0xffffffffu;
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.scales[j & 3]);
                if (j + 1 < n_c) scales(j + 1);
            }
            return true;
        };
        if (n_c > 0) scales(0);
        ok = convert_k(0) && convert_k(1);
#pragma unroll 1
        for (int j = 0; j < n_c && ok; ++j) {
            const int st = j % ST;
            if (!(ok = convert_k(j + 2) && convert(1, j, &b.v_empty[st], sm + L::v + st * L::KV))) break;
            full(&b.v_full[st]);
        }
        if (ok && n_all > n_c) {  // the open block: upper limbs in rows 0..31, lower in 32..63
            const int j = n_c, st = j % ST, there = kv_len - open0, slot = kv8_slot(a.c, seq);
            __shared__ float s_max[2][4];
            __shared__ unsigned s_bad[4];
            // a thread per 8 values of a row
            constexpr int PPR = HD / 8, RP = 128 / PPR;  // pieces per row, rows per step
            const int tid = threadIdx.x - 256, piece = tid % PPR;
            unsigned bad = 0;
            float amax[2] = {0.f, 0.f};
            auto piece_of = [&](int op, int t, float (&x)[8]) {
                const float *p = (op ? a.c.v_open : a.c.k_open) + kv8_open_at(a.c, max(slot, 0), open0 / kKvBlock, kh) +
                                 t * HD + piece * 8;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 z = slot >= 0 && t < there ? *reinterpret_cast<const float4 *>(p + e) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[e] = z.x, x[e + 1] = z.y, x[e + 2] = z.z, x[e + 3] = z.w;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(fabsf(x[e]) < INFINITY)) {
                        bad |= 1u << t;
                        x[e] = 0.f;
                    }
            };
            for (int op = 0; op < 2; ++op)
#pragma unroll 1
                for (int t = tid / PPR; t < kKvBlock; t += RP) {
                    float x[8];
                    piece_of(op, t, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) amax[op] = fmaxf(amax[op], fabsf(x[e]));
                }
            bad = __reduce_or_sync(0xffffffffu, bad);
#pragma unroll
            for (int op = 0; op < 2; ++op) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) amax[op] = fmaxf(amax[op], __shfl_xor_sync(0xffffffffu, amax[op], o));
                if (lane == 0) s_max[op][w] = amax[op];
            }
            if (lane == 0) s_bad[w] = bad;
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.open_max);
            ok = __all_sync(0xffffffffu, wait(&b.open_max, 0));
            float scale[2], inv[2];
#pragma unroll
            for (int op = 0; op < 2; ++op)
                scale[op] = limb_scale(fmaxf(fmaxf(s_max[op][0], s_max[op][1]), fmaxf(s_max[op][2], s_max[op][3])), inv[op]);
            ok = ok && empty(&b.k_empty[st], j);
            if (ok && tid == 0) {
                b.bad = slot >= 0 ? s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3] : 0;
                b.ks[j & 3][0] = slot >= 0 ? inv[0] : 0.f;
                b.vs[j & 3][0] = slot >= 0 ? inv[1] : 0.f;
                b.lv[j & 3][0] = log2f(b.vs[j & 3][0]);
                b.ks[j & 3][1] = b.vs[j & 3][1] = 0.f;
                b.lv[j & 3][1] = -INFINITY;
                b.plain[j & 3] = 0;
                mbar_arrive(&b.scales[j & 3]);
            }
            for (int op = 0; op < 2 && ok; ++op) {
                if (op == 1 && !(ok = empty(&b.v_empty[st], j))) break;
                uint8_t *tile = sm + (op ? L::v : L::k) + st * L::KV;
#pragma unroll 1
                for (int t = tid / PPR; t < kKvBlock; t += RP) {
                    float x[8];
                    piece_of(op, t, x);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) split_f16(x[2 * e] * scale[op], x[2 * e + 1] * scale[op], hi[e], lo[e]);
                    uint8_t *p = tile + piece / 8 * (kKeys * 128);
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const uint32_t(&h)[4] = z ? lo : hi;
                        const int row = t + 32 * z;
                        *reinterpret_cast<uint4 *>(p + row * 128 + ((piece & 7) ^ (row & 7)) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
                full(op ? &b.v_full[st] : &b.k_full[st]);
            }
        }
    } else {
        // ------------------------------------ MMA issue ------------------------------------
        reg_dec<kIssueRegs>();
        if (warp == 12) {
            // The whole warp goes along, one elected lane issues: 24 or 48 MMAs a tile, descriptors sums of constants.
            const uint32_t sq = smem_u32(sm + L::q), sk = smem_u32(sm + L::k), sv = smem_u32(sm + L::v);
            const uint32_t dq = desc_k(sq), dk = desc_k(sk), dv = desc_mn(sv, kKeys * 128);
            const int nt0 = uni(n_tiles[0]), nt1 = uni(n_tiles[1]), nt = max(nt0, nt1), closed = uni(n_closed - j0);
            const int last_blocks = uni(blocks - (n_closed - 1) * kTileBlocks);  // of the last closed tile
            auto all_wait = [&](uint64_t *bar, int phase) { return __all_sync(0xffffffffu, wait(bar, phase)); };
            auto scores = [&](int i, int j) {
                const uint32_t qb = dq + (i * L::QT >> 4), kb = dk + (j % ST * L::KV >> 4);
                const uint32_t d = tmem + i * kTile + kS + (j & 1) * kKeys;
#pragma unroll
                for (int z = LIMBS - 1; z >= 0; --z)  // (lower limbs first: fewer additions to a full-sized sum)
#pragma unroll
                    for (int at = 0; at < A; ++at)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t qa = qb + ((MT * z * L::QT + at * (128 * 128) + 32 * k) >> 4);
                            const uint32_t ka = kb + ((at * (kKeys * 128) + 32 * k) >> 4);
                            if (z == LIMBS - 1 && at == 0 && k == 0)
                                mma_ss<false>(d, qa, ka, idesc(kKeys, false));
                            else
                                mma_ss<true>(d, qa, ka, idesc(kKeys, false));
                        }
                mma_commit(&b.s_full[i][j & 1]);
            };
            auto values = [&](int i, int j) {
                const uint32_t vb = dv + (j % ST * L::KV >> 4);
                const uint32_t d = tmem + i * kTile + kO, p = tmem + i * kTile + kS + (j & 1) * kKeys;
                const uint32_t first = LIMBS == 2 ? 0u : (uint32_t)(j > 0);  // f32 rows: each tile's product by itself
                // 16 keys are 8 columns of P; two limbs: 8 of the upper, then 8 of the lower
                auto step = [&](int z, int k, uint32_t add) {
                    mma_ts(d, p + (LIMBS == 2 ? 16 * k + 8 * z : 8 * k), vb + (k * 2048 >> 4), idesc(HD, true), add);
                };
                const bool half = j == closed - 1 && last_blocks == 1;  // one block in the tile
#pragma unroll
                for (int z = LIMBS - 1; z >= 0; --z)
#pragma unroll
                    for (int k = 0; k < 2 * kTileBlocks; ++k)
                        if (k < 2 || !half) step(z, k, z == LIMBS - 1 && k == 0 ? first : 1u);
                mma_commit(&b.o_full[i]);
            };
            bool ok = all_wait(&b.q_full, 0);  // (a CTA without keys too: the rows' sums take Q's place after `done`)
            for (int j = 0; j < 2 && j < nt && ok; ++j) {
                if (!(ok = all_wait(&b.k_full[j % ST], j / ST))) break;
                tc_fence_after();
                if (elect_one()) {
                    if (j < nt0) scores(0, j);
                    if (j < nt1) scores(1, j);
                    mma_commit(&b.k_empty[j % ST]);
                }
                __syncwarp();
            }
#pragma unroll 1
            for (int j = 0; j < nt && ok; ++j) {
                if (!(ok = all_wait(&b.v_full[j % ST], j / ST))) break;
                const bool more = j + 2 < nt;
                bool k = false;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int n_i = i ? nt1 : nt0;
                    if (j >= n_i || !ok) continue;
                    if (!(ok = all_wait(&b.p_full[i][j & 1], j >> 1))) continue;
                    tc_fence_after();
                    if (elect_one()) {
                        values(i, j);
                        if (MT == 1) mma_commit(&b.v_empty[j % ST]);  // (the next values may precede the next K)
                    }
                    __syncwarp();
                    if (j + 2 >= n_i) continue;
                    // (only now: with one stage the converters need these values done before they come to K)
                    if (!(ok = k || all_wait(&b.k_full[(j + 2) % ST], (j + 2) / ST))) continue;
                    k = true;
                    tc_fence_after();
                    if (elect_one()) scores(i, j + 2);  // into the buffer of the weights just multiplied, after them
                    __syncwarp();
                }
                if (ok && elect_one()) {
                    if (MT == 2) mma_commit(&b.v_empty[j % ST]);
                    if (more) mma_commit(&b.k_empty[(j + 2) % ST]);
                }
                __syncwarp();
            }
            // every MMA has completed before TMEM is freed
            if (elect_one()) mma_commit(&b.done);
            __syncwarp();
            wait(&b.done, 0);
        } else if (warp == 13 && lane == 0) {
            // ------------------------------------ pages to shared memory ------------------------------------
            constexpr uint32_t kBytes = kKvBlock * HD;
            int issued[2] = {0, 0};
            auto load = [&](int op, int j) {
                if (j >= n_c) return true;
                const int st = j % ST;
                int page[kTileBlocks], count = 0;
#pragma unroll
                for (int c = 0; c < kTileBlocks; ++c) {
                    const int block = (j0 + j) * kTileBlocks + c;
                    page[c] = block < blocks ? kv8_page(a.c, seq, block) : -1;
                    count += page[c] >= 0;
                }
                if (j >= ST && !wait(&b.raw_empty[op][st], j / ST - 1)) return false;
                // (where no page is, what stood there stays: its keys are hidden, its values not multiplied)
                mbar_arrive_expect_tx(&b.raw_full[op][st], count * kBytes);
#pragma unroll
                for (int c = 0; c < kTileBlocks; ++c)
                    if (page[c] >= 0)
                        bulk_copy(sm + L::raw + (op * ST + st) * L::RAW + c * kBytes,
                                  (op ? a.c.v_codes : a.c.k_codes) + kv8_codes_at(a.c, page[c], kh), kBytes, &b.raw_full[op][st]);
                issued[op] = j + 1;
                return true;
            };
            bool ok = load(0, 0) && load(0, 1);
            for (int j = 0; j < n_c && ok; ++j) ok = load(1, j) && load(0, j + 2);
            // never leave with copies in flight
#pragma unroll
            for (int op = 0; op < 2; ++op)
                for (int j = max(0, issued[op] - ST); j < issued[op]; ++j)
                    mbar_wait(&b.raw_full[op][j % ST], (uint32_t)(j / ST) & 1u, nullptr, 0);
        } else if (warp == 14 && lane == 0 && r_base == 0 && n_rows > a.row_groups * ROWS) {
            atomicExch(a.c.err, kErrKvLength);  // rows that no CTA takes (an idle warp's check: at the top it cost 7 %)
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp >= 8) reg_inc<128>();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    // This CTA's share of the rows from every CTA of the cluster, consecutive threads along a row.
    cg::cluster_group cl = cg::this_cluster();
    if (a.cluster > 1) cl.sync();
    const int share = (ROWS + a.cluster - 1) / a.cluster, r0 = split * share, r1 = min(min(r0 + share, ROWS), n_rows - r_base);
    if (*abort_flag == 0) {
        const float *sums = reinterpret_cast<const float *>(sm);
        for (int x = threadIdx.x; x < (r1 - r0) * (HD / 4); x += kThreads) {
            const int r = r0 + x / (HD / 4), c = x % (HD / 4), gr = r_base + r;
            float m = -INFINITY, l = 0.f;
            float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
            if (a.cluster == 1) {
                l = sums[r * kPitch + HD + 1];
                z = *reinterpret_cast<const float4 *>(sums + r * kPitch + 4 * c);
            } else {
                for (int y = 0; y < a.cluster; ++y) m = fmaxf(m, *cl.map_shared_rank(sums + r * kPitch + HD, y));
                for (int y = 0; y < a.cluster; ++y) {
                    const float *p = cl.map_shared_rank(sums + r * kPitch, y);
                    const float pm = p[HD], pl = p[HD + 1];
                    const float4 w = *reinterpret_cast<const float4 *>(p + 4 * c);
                    // 0 where the CTA saw no key, NaN where its total is one (its maximum then says nothing)
                    const float f = pl != pl ? pl : pm == -INFINITY ? 0.f : ex2(pm - m);
                    if (f == 0.f) continue;
                    z.x = fmaf(w.x, f, z.x), z.y = fmaf(w.y, f, z.y), z.z = fmaf(w.z, f, z.z), z.w = fmaf(w.w, f, z.w);
                    l = fmaf(pl, f, l);
                }
            }
            const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that sees no key: zeros
            float v[4] = {z.x * inv, z.y * inv, z.z * inv, z.w * inv};
            const int64_t row = row0 + gr / G;
            const int d = (kh * G + gr % G) * HD + 4 * c;
            if (a.gate != nullptr) {
                const T *g = static_cast<const T *>(a.gate) + row * a.gate_stride + d;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] *= 1.0f / (1.0f + expf(-(float)g[k]));
            }
            T *o = static_cast<T *>(a.out) + row * a.out_stride + d;
            if (a.vec) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    __nv_bfloat162 w[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
                    *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<uint2 *>(w);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (sizeof(T) == 4)
                        o[k] = v[k];
                    else
                        o[k] = __float2bfloat16_rn(v[k]);
                }
            }
        }
    }
    if (a.cluster > 1) cl.sync();  // (its shared memory is read until all have arrived)
}

template <typename T, int HD>
cudaError_t launch_hd(const Kv8AttnArgs &a, cudaStream_t s) {
    constexpr int smem = Layout<HD, sizeof(T) == 4 ? 2 : 1>::bytes;
    static_assert(smem <= 232448, "shared memory of one SM");
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        if ((e = cudaFuncSetAttribute(prompt_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess)
            return e;
        if (dev < 64) ready.fetch_or(1ull << dev);
    }
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)a.cluster, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    // The tiles of rows lie in the grid's z, one launch but for calls of millions of rows.  (All in x, by divisions, the
    // 2048 tokens in f32 take 101.2 us and four chunks of narrow heads 79.3, so 99.5 and 78.1.)
    Kv8AttnArgs b = a;
    for (b.tile0 = 0; b.tile0 < a.row_groups; b.tile0 += kKvMaxTiles) {
        cfg.gridDim = dim3(a.c.kv_heads * a.cluster, a.c.n_seqs, std::min(a.row_groups - b.tile0, kKvMaxTiles));
        if ((e = cudaLaunchKernelEx(&cfg, prompt_kernel<T, HD>, b)) != cudaSuccess) return e;
    }
    return cudaSuccess;
}
}  // namespace

// (f32 rows of 256 would need 256 registers for their sums)
int kv8_prompt_rows(int head_dim, bool f32) {
    return head_dim == 64 || head_dim == 128 || (head_dim == 256 && !f32) ? 128 * row_tiles(head_dim) : 0;
}

cudaError_t kv8_prompt_launch(const Kv8AttnArgs &a, bool bf16, cudaStream_t s) {
    if (a.c.head_dim == 256) return launch_hd<__nv_bfloat16, 256>(a, s);
    if (a.c.head_dim == 64)
        return bf16 ? launch_hd<__nv_bfloat16, 64>(a, s) : launch_hd<float, 64>(a, s);
    return bf16 ? launch_hd<__nv_bfloat16, 128>(a, s) : launch_hd<float, 128>(a, s);
}

}  // namespace ql
