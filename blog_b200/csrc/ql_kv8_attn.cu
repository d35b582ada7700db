// Attention over the 8-bit KV cache, split over the keys: the form for single tokens and few queries.
//
//   out_h = softmax_j(scale q_h . k_j) . v_j  (* sigmoid(gate_h)),   j = 0 .. the query's position,
//   k_j = (ck_j - 128) sk_b,  v_j = (cv_j - 128) sv_b,  b = j / 32 the token's block,
// and the exact f32 rows for the tokens of the block that is not full.
//
// Mathematics.  A code is an integer of 8 bits and so exact in f16: with q = 2^-e (qh + ql) in two f16 limbs
// (22 bits) the products q . c are exact and summed in fp32, and one multiplication by sk_b scale 2^-e gives
// the score.  What meets V's codes is p sv_b, p = 2^(s - m): it is taken relative to the row's largest such
// product so far (2^h, a running maximum of s - m + log2 sv_b beside that of s) and split into two f16 limbs in
// the same way, so the result is as exact as fp32 sums make it, however unlike the blocks' scales are.  The
// two limbs cost nothing: mma.m16n8k16 has 16 rows, the 8 rows' upper limbs and their lower
// ones, and the two halves of an accumulator fragment are added.  The MMA truncates as it accumulates (about
// 3e-8 of the sum, always downwards, per step of 16), so f32 results are summed per block there and added up
// with rounding outside.
//
// Layout.  A CTA has 4 warps and 8 rows (query token, head of one KV head's group); each warp walks over
// key blocks of its own (32 tokens x head_dim codes of K and of V, two contiguous pieces of a page) through
// a ring in shared memory filled by cp.async, with its own m, l and accumulators, so the loop has no barrier.
// The order of the head dimension within a product and of the tokens within a block is free as long as both
// operands agree, so the fragments are 16-byte pieces of the rows as they lie in the page: 16 codes of K
// serve four k-steps, and V pairs of tokens are gathered from two rows by one byte permute.
// The CTAs of one (sequence, KV head, row group) form clusters of up to 8; warps are merged in shared memory,
// a cluster's CTAs through distributed shared memory (each finishes its share of the rows), and clusters by
// the last to arrive, always in split order: the result does not depend on which that is.
//
// Bound: HBM for the codes (2 head_dim bytes per token and KV head) where the keys are many: 64 sequences of 4096 to
// 8192 tokens, 64/8/128 heads, bf16, 681 MB in 122 us, 5.6 TB/s (0.87 of a copy's).  Below that the chain of one
// CTA's loads, products and merges: one sequence of 28/4/128 heads, f32, 17.6 us at 32768 tokens (1.9 TB/s) and
// 7.6 us at 200.  Tiles of 8 rows and not of 16: a group of 7 or 8 heads fills them, and a single token has no more.
#include <cooperative_groups.h>

#include <atomic>
#include <climits>

#include "ql_kv8_limbs.cuh"

namespace cg = cooperative_groups;

namespace ql {
namespace {

constexpr int kThreads = 32 * kKvAttnWarps;

__device__ __forceinline__ void cp16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ float load_f32(const T *p);
template <>
__device__ __forceinline__ float load_f32<float>(const float *p) { return *p; }
template <>
__device__ __forceinline__ float load_f32<__nv_bfloat16>(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
// Four elements whose address is a multiple of theirs together.
template <typename T>
__device__ __forceinline__ void load4(float *x, const T *p) {
    if constexpr (sizeof(T) == 4) {
        const float4 z = *reinterpret_cast<const float4 *>(p);
        x[0] = z.x, x[1] = z.y, x[2] = z.z, x[3] = z.w;
    } else {
        const uint2 z = *reinterpret_cast<const uint2 *>(p);  // bf16: the upper half of an f32
        x[0] = __uint_as_float(z.x << 16), x[1] = __uint_as_float(z.x & 0xFFFF0000u);
        x[2] = __uint_as_float(z.y << 16), x[3] = __uint_as_float(z.y & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void store_f32(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// Ring stages per warp, and CTAs per SM, by head_dim: 64 head_dim bytes per stage, 4 warps, 227 KB per SM.
constexpr int stages(int hd) { return hd <= 64 ? 3 : hd <= 128 ? 2 : 3; }
constexpr int ctas_per_sm(int hd) { return hd <= 64 ? 4 : hd <= 128 ? 3 : 1; }
static_assert(ctas_per_sm(32) <= kKvAttnMaxCtasPerSm, "the workspace's counters");

// 16-byte chunk of a row at which chunk c of row t lies.  K: a load phase (8 lanes) reads 64 bytes of two
// rows, which share their banks where a row is a multiple of 128 bytes: the odd row's halves are swapped.
// V: a phase reads two chunks of four rows (the lanes' token pairs); the XOR spreads them over all banks.
template <int HD>
__device__ __forceinline__ int k_chunk(int c, int t) {
    return HD % 128 == 0 ? c ^ ((t & 1) << 2) : c;
}
template <int HD>
__device__ __forceinline__ int v_chunk(int c, int t) {
    const int p = (t >> 1) & 3;
    if (HD == 128) return c ^ (p << 1);
    if (HD == 256) return c ^ ((p & 1) | ((p & 2) << 1));
    if (HD == 64) return c ^ ((p & 1) << 1);
    return c;
}

// Factor of a partial (maximum pm, total pt) in the sum with maximum m: 0 where it saw no key, NaN where
// its total is one (its maximum then says nothing).
__device__ __forceinline__ float part_factor(float pm, float pt, float m) {
    return pt != pt ? pt : pm == -INFINITY ? 0.f : ex2(pm - m);
}

// What turns sums of w 2^(s - m) sv code into sums of 2^(s - m) sv code: x 2^(h - kWBits), in two steps where
// the power leaves the range.
__device__ __forceinline__ float weight_undo(float x, float h) {
    const float e = h - kWBits;
    return h == -INFINITY ? x * 0.f : x * ex2(fmaxf(e, -120.f)) * ex2(fminf(e + 120.f, 0.f));  // (NaN stays)
}

// Running state of one warp: row g8 = lane / 4 in the first two floats of a fragment (upper limbs) and the
// last two (lower limbs).
template <int HD, bool EXACT>
struct Acc {
    float o[HD / 8][4];
    float m, l;  // maximum of the scores, total of 2^(s - m)
    float h, w;  // maximum of s - m + log2 of V's scale; 2^(kWBits - h): o holds sums of w 2^(s - m) sv code

    // Block's products s[n][2] of row g8, columns 2 q4, 2 q4 + 1 of n-tile n (-inf: a masked key), to weights:
    // returns the two limbs' A fragments.  The score (a base-2 logarithm) is s k r, r >= 0 the row's scale and k the
    // block's; less m it is one rounding, and f32 rows add back that of k r.  vs: the scale of the block's values.
    static __device__ __forceinline__ float less_m(float s, float kr, float kr_lo, float m) {
        const float d = fmaf(s, kr, -m);
        return EXACT ? fmaf(s, kr_lo, d) : d;
    }
    template <int NT>
    __device__ __forceinline__ void weights(const float (&s)[NT][2], float k, float r_, float vs, uint32_t (&hi)[NT],
                                            uint32_t (&lo)[NT]) {
        const float kr = k * r_, kr_lo = EXACT ? fmaf(k, r_, -kr) : 0.f;
        float t = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n) t = fmaxf(t, fmaxf(s[n][0], s[n][1]));
        if (t != -INFINITY) t *= kr;
        const float lv = log2f(vs);  // (0: -inf, which never passes h; NaN neither)
        if (__any_sync(0xffffffffu, t > m + kHeadroom || t - m + lv > h + kHeadroom)) {
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));  // the row's four lanes agree
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            if (t > m) {
                const float z = ceilf(t);
                l *= ex2(m - z);  // m = -inf: 0
                h -= z - m;       // (o's unit 2^(m + h) stays)
                m = z;
            }
            float r = 1.0f;
            if (t - m + lv > h) {
                const float z = ceilf(t - m + lv);
                r = ex2(h - z);
                h = z;
            }
            w = weight_unit(h);
            if (__any_sync(0xffffffffu, r != 1.0f)) {
#pragma unroll
                for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][i] *= r;
            }
        }
        const float f = vs * w;
        const float base = m == -INFINITY ? 0.f : m;
        // (a masked key: a NaN scale must not reach its weight)
        if (__any_sync(0xffffffffu, h < kDeep || fabsf(base) > kHuge)) {
            const bool huge = fabsf(base) > kHuge;
            const float lift = h == -INFINITY ? 0.f : h, g = h == -INFINITY ? f : vs * ex2(kWBits);
            // (huge scores: h says nothing of the values' scale any more, so their product is kept in f16 by itself; NaN stays)
            const float most = fminf(126.f, kHeadroom + 0.9f - lv);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool seen = s[n][e] != -INFINITY;
                    const float d = huge ? __fsub_rn(__fmul_rn(s[n][e], kr), base) : less_m(s[n][e], kr, kr_lo, base);
                    l += seen ? ex2(d) : 0.f;
                    x[e] = seen ? ex2(fminf(d - lift, most)) * g : 0.f;
                }
                split_f16(x[0], x[1], hi[n], lo[n]);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bool s0 = s[n][0] != -INFINITY, s1 = s[n][1] != -INFINITY;
                const float p0 = s0 ? ex2(less_m(s[n][0], kr, kr_lo, base)) : 0.f;
                const float p1 = s1 ? ex2(less_m(s[n][1], kr, kr_lo, base)) : 0.f;
                l += p0 + p1;
                split_f16(s0 ? p0 * f : 0.f, s1 ? p1 * f : 0.f, hi[n], lo[n]);
            }
        }
    }
};

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(HD)) attn_kernel(const __grid_constant__ Kv8AttnArgs a) {
    extern __shared__ __align__(128) uint8_t sm[];
    constexpr int ST = stages(HD), BLK = kKvBlock * HD;  // codes of one operand's block
    constexpr int G64 = HD / 64, REM = HD % 64 / 32;     // K row: groups of 64 codes, and one of 32
    constexpr int KS = HD / 16;                          // k-steps of q . k
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, q4 = lane & 3;
    const int G = a.n_heads / a.c.kv_heads;
    const int split = blockIdx.x % a.splits, at = blockIdx.x / a.splits;
    const int kh = at % a.c.kv_heads, rg = at / a.c.kv_heads;
    int seq = blockIdx.y;
    if (a.longest_first) {  // the sequence of this rank by length, a thread per sequence (equals: in their order)
        __shared__ int4 s_len[kThreads / 4];
        __shared__ int s_seq;
        const int n = a.c.n_seqs, me = threadIdx.x, mine = me < n ? a.r.kv_len[me] : INT_MIN;
        reinterpret_cast<int *>(s_len)[me] = mine;
        __syncthreads();
        int rank = 0;
#pragma unroll 1
        for (int j = 0; j < n; j += 4) {
            const int4 x = s_len[j / 4];
            rank += x.x > mine || (x.x == mine && j < me);
            rank += x.y > mine || (x.y == mine && j + 1 < me);
            rank += x.z > mine || (x.z == mine && j + 2 < me);
            rank += x.w > mine || (x.w == mine && j + 3 < me);
        }
        if (me < n && rank == seq) s_seq = me;
        __syncthreads();
        seq = s_seq;
    }
    uint8_t *ring = sm + warp * (ST * 2 * BLK);
    uint4 *qf = reinterpret_cast<uint4 *>(sm + kKvAttnWarps * ST * 2 * BLK);  // [KS][32] A fragments of q
    __shared__ float s_m[kKvAttnWarps][kKvAttnRows], s_l[kKvAttnWarps][kKvAttnRows], s_q[kKvAttnRows];
    __shared__ float c_m[kKvAttnRows], c_l[kKvAttnRows];  // this CTA's maximum and total, read by its cluster
    __shared__ unsigned s_last;

    int row0, q_len;
    kv8_rows_of(a.r, seq, row0, q_len);
    int kv_len = a.r.kv_len[seq];
    if (threadIdx.x == 0 && rg == 0 && q_len * G > a.row_groups * kKvAttnRows) atomicExch(a.c.err, kErrKvLength);
    if (rg * kKvAttnRows >= q_len * G) return;  // (uniform: every split of the group leaves here)
    if ((unsigned)kv_len > (unsigned)(a.c.max_pages * kKvBlock)) {  // (negative too; the host bounds max_pages)
        if (threadIdx.x == 0) atomicExch(a.c.err, kErrKvPage);
        kv_len = 0;
    }
    // this lane's row: token t of the call, head h
    const int grow = rg * kKvAttnRows + g8;
    const bool live = grow < q_len * G;
    const int tok = live ? grow / G : 0, head = kh * G + (live ? grow % G : 0);
    const int pos = live ? kv_len - q_len + tok : -1;  // the last key that the row sees (-1: none)
    // keys that any row of this CTA sees, and keys that all of them see
    const int tok_hi = min(rg * kKvAttnRows + kKvAttnRows - 1, q_len * G - 1) / G, tok_lo = rg * kKvAttnRows / G;
    const int keys = max(0, min(kv_len, kv_len - q_len + tok_hi + 1)), keys_all = kv_len - q_len + tok_lo + 1;
    const int full_blocks = min((keys + kKvBlock - 1) / kKvBlock, kv_len / kKvBlock);
    const int open0 = kv_len / kKvBlock * kKvBlock;  // the first open token
    const int open_units = keys > open0 ? (keys - open0 + 7) / 8 : 0;

    // blocks of this warp: w, w + W, ...; page numbers and scales of 32 of them at a time, one per lane
    const int W = a.splits * kKvAttnWarps, w = split * kKvAttnWarps + warp;
    const int n_blocks = full_blocks > w ? (full_blocks - w + W - 1) / W : 0;
    int page = -1;
    float ks = 0.f, vs = 0.f;
    auto fetch_pages = [&](int i0) {  // blocks i0 .. i0 + 31 of the warp's list
        page = -1;
        if (i0 + lane < n_blocks) page = kv8_page(a.c, seq, w + (i0 + lane) * W);
        if (page >= 0) {
            ks = a.c.k_scale[(int64_t)page * a.c.kv_heads + kh];
            vs = a.c.v_scale[(int64_t)page * a.c.kv_heads + kh];
        }
    };
    // a lane's 16-byte pieces of a block: u * 512 + lane * 16; their places repeat every P pieces (8 rows)
    constexpr int NU = BLK / 512, P = NU < 4 ? NU : HD == 128 ? 2 : 4;
    static_assert(HD * 8 == P * 512 || P == NU || (HD != 64 && HD != 128 && HD != 256), "8 rows per P pieces");
    int k_off[P], v_off[P];
#pragma unroll
    for (int u = 0; u < P; ++u) {
        const int x = u * 32 + lane, t = x / (HD / 16), c = x % (HD / 16);
        k_off[u] = t * HD + k_chunk<HD>(c, t) * 16;
        v_off[u] = t * HD + v_chunk<HD>(c, t) * 16;
    }
    auto issue = [&](int i, int pg) {  // block i of the list into its stage (one group, empty past the end)
        if (i < n_blocks && pg >= 0) {
            uint8_t *dst = ring + i % ST * 2 * BLK;
            const int64_t at = kv8_codes_at(a.c, pg, kh) + lane * 16;
            const uint8_t *kp = a.c.k_codes + at, *vp = a.c.v_codes + at;
#pragma unroll
            for (int u = 0; u < NU; ++u) cp16(dst + u / P * (P * 512) + k_off[u % P], kp + u * 512);
#pragma unroll
            for (int u = 0; u < NU; ++u) cp16(dst + BLK + u / P * (P * 512) + v_off[u % P], vp + u * 512);
        }
        cp_commit();
    };
    fetch_pages(0);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) issue(i, __shfl_sync(0xffffffffu, page, i));

    // q: two limbs per row, scaled by a power of two, as A fragments (warp 0 writes, all read)
    if (warp == 0) {
        float x[KS][4], amax = 0.f;
        const T *q = static_cast<const T *>(a.q) + (int64_t)(row0 + tok) * a.q_stride + (int64_t)head * HD;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d = k < 4 * G64 ? k / 4 * 64 + 16 * q4 + k % 4 * 4 : 64 * G64 + 8 * q4 + (k - 4 * G64) * 4;
            if (live && a.vec) {
                load4<T>(x[k], q + d);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[k][i] = live ? load_f32<T>(q + d + i) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[k][i]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        float inv;
        // (a negative softmax scale: its sign goes to q, so that products order like scores)
        const float f = copysignf(limb_scale(amax, inv), a.scale_log2);
        if (q4 == 0) s_q[g8] = fabsf(a.scale_log2) * inv;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint4 u;
            split_f16(x[k][0] * f, x[k][1] * f, u.x, u.y);  // rows g8 (upper limb), g8 + 8 (lower)
            split_f16(x[k][2] * f, x[k][3] * f, u.z, u.w);
            qf[k * 32 + lane] = u;
        }
    }
    __syncthreads();
    const float row_scale = s_q[g8];

    constexpr bool EXACT = sizeof(T) == 4;
    Acc<HD, EXACT> acc;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.o[n][i] = 0.f;
    acc.m = -INFINITY;
    acc.l = 0.f;
    acc.h = -INFINITY;
    acc.w = 0.f;

    for (int i = 0; i < n_blocks; ++i) {
        const int pg = __shfl_sync(0xffffffffu, page, i & 31);
        const float bk = __shfl_sync(0xffffffffu, ks, i & 31), bv = __shfl_sync(0xffffffffu, vs, i & 31);
        {   // the block ST - 1 ahead; its page may be in the next batch, which is fetched when this one ends
            const int nx = i + ST - 1;
            int npg;
            if ((nx & ~31) == (i & ~31))
                npg = __shfl_sync(0xffffffffu, page, nx & 31);
            else
                npg = nx < n_blocks ? kv8_page(a.c, seq, w + nx * W) : -1;
            cp_wait<ST - 2>();
            __syncwarp();
            issue(nx, npg);
        }
        if ((i & 31) == 31) fetch_pages(i + 1);
        if (pg < 0) continue;
        const uint8_t *kt = ring + i % ST * 2 * BLK, *vt = kt + BLK;

        // scores of 32 tokens: n-tile n holds tokens 8 n .. 8 n + 7, this lane's column g8 of K
        float c[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) c[n][j] = 0.f;
#pragma unroll
        for (int g = 0; g < G64; ++g) {
            uint4 kw[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int t = 8 * n + g8;
                kw[n] = *reinterpret_cast<const uint4 *>(kt + t * HD + k_chunk<HD>(4 * g + q4, t) * 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 qa = qf[(4 * g + j) * 32 + lane];
                const uint32_t af[4] = {qa.x, qa.y, qa.z, qa.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t u = reinterpret_cast<const uint32_t *>(&kw[n])[j];
                    mma16816(c[n], af, codes2(u, 0x4140), codes2(u, 0x4342));
                }
            }
        }
        if constexpr (REM != 0) {
            uint2 kw[4];
#pragma unroll
            for (int n = 0; n < 4; ++n)
                kw[n] = *reinterpret_cast<const uint2 *>(kt + (8 * n + g8) * HD + 64 * G64 + q4 * 8);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint4 qa = qf[(4 * G64 + j) * 32 + lane];
                const uint32_t af[4] = {qa.x, qa.y, qa.z, qa.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t u = j ? kw[n].y : kw[n].x;
                    mma16816(c[n], af, codes2(u, 0x4140), codes2(u, 0x4342));
                }
            }
        }
        const int key0 = (w + i * W) * kKvBlock;
        float s[4][2];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[n][e] = c[n][e] + c[n][e + 2];
        if (key0 + kKvBlock > keys_all) {  // some row does not see the whole block
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (key0 + 8 * n + 2 * q4 + e > pos) s[n][e] = -INFINITY;
        }
        uint32_t hi[4], lo[4];
        acc.weights(s, bk, row_scale, bv, hi, lo);

        // values: n-tile n's column g8 is dimension g8 * HD / 8 + n; a k-step's tokens are those of two score
        // n-tiles, so the weights are already the A fragment.  The tensor cores truncate when they accumulate: f32
        // rows start each block's products from zero and add them here, rounded.
        constexpr int WD = HD / 32;  // 4-byte words per lane and row
        constexpr int WC = EXACT ? (WD % 2 == 0 ? 2 : 1) : WD % 4 == 0 ? 4 : WD % 2 == 0 ? 2 : 1;
        auto rows4 = [&](int kk, int x, uint32_t (&r)[4][WC]) {  // rows t0, t0 + 1, t0 + 8, t0 + 9 of the k-step
            const int t0 = 16 * kk + 2 * q4;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int t = t0 + (y & 1) + (y >> 1) * 8, byte = g8 * (HD / 8) + 4 * x;
                const uint8_t *p = vt + t * HD + v_chunk<HD>(byte / 16, t) * 16 + byte % 16;
                if constexpr (WC == 4) {
                    const uint4 z = *reinterpret_cast<const uint4 *>(p);
                    r[y][0] = z.x, r[y][1] = z.y, r[y][2] = z.z, r[y][3] = z.w;
                } else if constexpr (WC == 2) {
                    const uint2 z = *reinterpret_cast<const uint2 *>(p);
                    r[y][0] = z.x, r[y][1] = z.y;
                } else {
                    r[y][0] = *reinterpret_cast<const uint32_t *>(p);
                }
            }
        };
        auto product = [&](float (&d)[4][4], const uint32_t (&r)[4][WC], int z, int kk) {  // four n-tiles
            const uint32_t af[4] = {hi[2 * kk], lo[2 * kk], hi[2 * kk + 1], lo[2 * kk + 1]};
            const uint32_t a01 = __byte_perm(r[0][z], r[1][z], 0x5140), a23 = __byte_perm(r[0][z], r[1][z], 0x7362);
            const uint32_t b01 = __byte_perm(r[2][z], r[3][z], 0x5140), b23 = __byte_perm(r[2][z], r[3][z], 0x7362);
            mma16816(d[0], af, codes2(a01, 0x4140), codes2(b01, 0x4140));
            mma16816(d[1], af, codes2(a01, 0x4342), codes2(b01, 0x4342));
            mma16816(d[2], af, codes2(a23, 0x4140), codes2(b23, 0x4140));
            mma16816(d[3], af, codes2(a23, 0x4342), codes2(b23, 0x4342));
        };
        if constexpr (EXACT) {
#pragma unroll
            for (int x = 0; x < WD; x += WC) {
                uint32_t r0[4][WC], r1[4][WC];
                rows4(0, x, r0);
                rows4(1, x, r1);
#pragma unroll
                for (int z = 0; z < WC; ++z) {
                    float d[4][4] = {};
                    product(d, r0, z, 0);
                    product(d, r1, z, 1);
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc.o[4 * (x + z) + n][e] += d[n][e];
                }
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int x = 0; x < WD; x += WC) {
                    uint32_t r[4][WC];
                    rows4(kk, x, r);
#pragma unroll
                    for (int z = 0; z < WC; ++z)
                        product(*reinterpret_cast<float(*)[4][4]>(&acc.o[4 * (x + z)]), r, z, kk);
                }
        }
    }
    cp_wait<0>();

    // Open rows: units of 8 tokens, given to the warps with the fewest blocks; K and V split into two limbs
    // like q.  A token with a NaN or infinity gives NaN to the rows that see it and nothing to the others.
    for (int u = W - 1 - w; u < open_units; u += W) {
        const int slot = kv8_slot(a.c, seq);
        if (slot < 0) break;
        const int64_t rows_at = kv8_open_at(a.c, slot, open0 / kKvBlock, kh) + (int64_t)u * 8 * HD;
        const int key0 = open0 + 8 * u, there = min(8, kv_len - key0);
        unsigned bad = 0;
        // f32 rows: three sums, every other step's upper limbs and the lower limbs.  (The MMA truncates products of two
        // limbs of 11 bits as it aligns them to its sum: in one sum scores of head_dim 256 have an error of 7e-7, so 3e-7.)
        constexpr int C1 = EXACT ? 1 : 0, C2 = EXACT ? 2 : 0;
        float c[C2 + 1][4] = {};
        float kinv;
        {
            float x[KS][4], amax = 0.f;
            const float *k = a.c.k_open + rows_at + g8 * HD;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = s < 4 * G64 ? s / 4 * 64 + 16 * q4 + s % 4 * 4 : 64 * G64 + 8 * q4 + (s - 4 * G64) * 4;
                const float4 z = g8 < there ? *reinterpret_cast<const float4 *>(k + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[s][0] = z.x, x[s][1] = z.y, x[s][2] = z.z, x[s][3] = z.w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!(fabsf(x[s][i]) < INFINITY)) {
                        bad |= 1u << g8;
                        x[s][i] = 0.f;
                    }
                    amax = fmaxf(amax, fabsf(x[s][i]));
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float f = limb_scale(amax, kinv);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint4 qa = qf[s * 32 + lane];
                const uint32_t af[4] = {qa.x, qa.y, qa.z, qa.w};
                uint32_t h0, l0, h1, l1;
                split_f16(x[s][0] * f, x[s][1] * f, h0, l0);
                split_f16(x[s][2] * f, x[s][3] * f, h1, l1);
                mma16816(c[s & C1], af, h0, h1);
                mma16816(c[C2], af, l0, l1);
            }
        }
        float v[2][HD / 8], vmax = 0.f, vinv;
        const float *vp = a.c.v_open + rows_at + g8 * (HD / 8);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int t = 2 * q4 + y;
#pragma unroll
            for (int n = 0; n < HD / 8; n += 4) {
                const float4 z =
                    t < there ? *reinterpret_cast<const float4 *>(vp + t * HD + n) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[y][n] = z.x, v[y][n + 1] = z.y, v[y][n + 2] = z.z, v[y][n + 3] = z.w;
            }
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
                if (!(fabsf(v[y][n]) < INFINITY)) {
                    bad |= 1u << t;
                    v[y][n] = 0.f;
                }
                vmax = fmaxf(vmax, fabsf(v[y][n]));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
        const float vf = limb_scale(vmax, vinv);
        bad = __reduce_or_sync(0xffffffffu, bad);
        float s[1][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int t = 2 * q4 + e;
            s[0][e] = c[0][e] + c[0][e + 2];
            if (EXACT) s[0][e] = (c[0][e] + c[C1][e]) + ((c[0][e + 2] + c[C1][e + 2]) + (c[C2][e] + c[C2][e + 2]));
            if (bad >> t & 1) s[0][e] = __int_as_float(0x7FC00000);
            if (key0 + t > pos) s[0][e] = -INFINITY;
        }
        uint32_t hi[1], lo[1];
        acc.weights(s, kinv, row_scale, vinv, hi, lo);
        const uint32_t af[4] = {hi[0], lo[0], 0u, 0u};
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
            uint32_t h, l;
            split_f16(v[0][n] * vf, v[1][n] * vf, h, l);
            mma16816(acc.o[n], af, h, 0u);
            mma16816(acc.o[n], af, l, 0u);
        }
    }

    // Warps: [warp][row][HD] in the ring's memory, in chunks of 4 dimensions; the lanes of a store phase (two
    // rows, four q4) have the same chunk modulo 8 and are spread by an XOR.
    float l = acc.l + __shfl_xor_sync(0xffffffffu, acc.l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    __syncthreads();
    float *so = reinterpret_cast<float *>(sm);
    auto so_at = [&](int y, int r, int chunk) {
        // (the key must not change within 8 chunks: head_dim 64, 128, 256)
        constexpr bool pow2 = HD == 64 || HD == 128 || HD == 256;
        return so + (y * kKvAttnRows + r) * HD + (pow2 ? chunk ^ ((chunk / (HD / 16) * 2 + (r & 1)) & 7) : chunk) * 4;
    };
    {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < HD / 8; n += 4) {
                float4 z;
                z.x = weight_undo(acc.o[n][e] + acc.o[n][e + 2], acc.h);
                z.y = weight_undo(acc.o[n + 1][e] + acc.o[n + 1][e + 2], acc.h);
                z.z = weight_undo(acc.o[n + 2][e] + acc.o[n + 2][e + 2], acc.h);
                z.w = weight_undo(acc.o[n + 3][e] + acc.o[n + 3][e + 2], acc.h);
                *reinterpret_cast<float4 *>(so_at(warp, g8, (2 * q4 + e) * (HD / 32) + n / 4)) = z;
            }
        if (q4 == 0) {
            s_m[warp][g8] = acc.m;
            s_l[warp][g8] = l;
        }
    }
    __syncthreads();
    auto add4 = [](float4 &z, const float4 &w, float f) {
        if (f == 0.f) return;  // (saw no key: whatever stands there)
        z.x = fmaf(w.x, f, z.x), z.y = fmaf(w.y, f, z.y), z.z = fmaf(w.z, f, z.z), z.w = fmaf(w.w, f, z.w);
    };
    for (int x = threadIdx.x; x < kKvAttnRows * HD / 4; x += kThreads) {
        const int r = x / (HD / 4), c = x % (HD / 4);
        float m = -INFINITY, t = 0.f;
#pragma unroll
        for (int y = 0; y < kKvAttnWarps; ++y) m = fmaxf(m, s_m[y][r]);
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int y = 0; y < kKvAttnWarps; ++y) {
            const float f = part_factor(s_m[y][r], s_l[y][r], m);
            add4(z, *reinterpret_cast<const float4 *>(so_at(y, r, c)), f);
            if (f != 0.f) t = fmaf(s_l[y][r], f, t);
        }
        *reinterpret_cast<float4 *>(so_at(0, r, c)) = z;  // (read by this thread alone so far)
        if (c == 0) {
            c_m[r] = m;
            c_l[r] = t;
        }
    }
    auto finish = [&](int r, int c, const float4 &z, float total) {
        const int gr = rg * kKvAttnRows + r;
        if (gr >= q_len * G) return;
        const int64_t row = row0 + gr / G;
        const int d = (kh * G + gr % G) * HD + 4 * c;
        const float inv = total == 0.f ? 0.f : 1.0f / total;  // a row that sees no key: zeros
        float v[4] = {z.x * inv, z.y * inv, z.z * inv, z.w * inv};
        if (a.gate != nullptr) {
            const T *g = static_cast<const T *>(a.gate) + row * a.gate_stride + d;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] *= 1.0f / (1.0f + expf(-load_f32<T>(g + i)));
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
            for (int i = 0; i < 4; ++i) store_f32(o + i, v[i]);
        }
    };
    if (a.splits == 1) {
        __syncthreads();
        for (int x = threadIdx.x; x < kKvAttnRows * HD / 4; x += kThreads) {
            const int r = x / (HD / 4), c = x % (HD / 4);
            finish(r, c, *reinterpret_cast<const float4 *>(so_at(0, r, c)), c_l[r]);
        }
        return;
    }
    // cluster: rank k of n finishes rows k 8 / n .. from every CTA's shared memory
    cg::cluster_group cl = cg::this_cluster();
    const int n_cta = a.cluster, rank = split % n_cta, rows = kKvAttnRows / n_cta, r0 = rank * rows;
    const int clusters = a.splits / n_cta, cluster = split / n_cta;
    cl.sync();
    const int64_t group = ((int64_t)seq * a.row_groups + rg) * a.c.kv_heads + kh;
    constexpr int PR = HD + 4;  // a partial's row: sums, maximum, total
    for (int x = threadIdx.x; x < rows * HD / 4; x += kThreads) {
        const int r = r0 + x / (HD / 4), c = x % (HD / 4);
        float pm[8], pl[8], m = -INFINITY, t = 0.f;
        float4 w[8];
#pragma unroll
        for (int y = 0; y < 8; ++y)
            if (y < n_cta) {
                pm[y] = *cl.map_shared_rank(&c_m[r], y);
                pl[y] = *cl.map_shared_rank(&c_l[r], y);
                w[y] = *reinterpret_cast<const float4 *>(cl.map_shared_rank(so_at(0, r, c), y));
                m = fmaxf(m, pm[y]);
            }
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int y = 0; y < 8; ++y)
            if (y < n_cta) {
                const float f = part_factor(pm[y], pl[y], m);
                add4(z, w[y], f);
                if (f != 0.f) t = fmaf(pl[y], f, t);
            }
        if (clusters == 1) {
            finish(r, c, z, t);
        } else {
            float *p = a.part + ((group * clusters + cluster) * kKvAttnRows + r) * PR;
            *reinterpret_cast<float4 *>(p + 4 * c) = z;
            if (c == 0) *reinterpret_cast<float2 *>(p + HD) = make_float2(m, t);
        }
    }
    __syncwarp();
    cl.barrier_arrive();  // (waited for at the end: a CTA's shared memory is read until all have arrived)
    if (clusters > 1) {
        __threadfence();
        __syncthreads();
        unsigned *arrived = a.arrivals + group * kKvAttnRows + rank;
        if (threadIdx.x == 0) s_last = atomicAdd(arrived, 1u) == (unsigned)clusters - 1;
        __syncthreads();
        if (s_last) {
            __threadfence();
            for (int x = threadIdx.x; x < rows * HD / 4; x += kThreads) {
                const int r = r0 + x / (HD / 4), c = x % (HD / 4);
                const float *p = a.part + (group * clusters * kKvAttnRows + r) * PR;
                float m = -INFINITY, t = 0.f;
                float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int y0 = 0; y0 < clusters; y0 += 8) {  // eight partials in flight
                    float2 ml[8];
                    float4 w[8];
                    float mb = m;
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        if (y0 + y < clusters) {
                            const float *g = p + (int64_t)(y0 + y) * kKvAttnRows * PR;
                            ml[y] = __ldcg(reinterpret_cast<const float2 *>(g + HD));
                            w[y] = __ldcg(reinterpret_cast<const float4 *>(g + 4 * c));
                            mb = fmaxf(mb, ml[y].x);
                        }
                    const float f0 = m == -INFINITY ? (t == t ? 0.f : t) : ex2(m - mb);
                    z.x *= f0, z.y *= f0, z.z *= f0, z.w *= f0, t *= f0;
                    m = mb;
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        if (y0 + y < clusters) {
                            const float f = part_factor(ml[y].x, ml[y].y, m);
                            add4(z, w[y], f);
                            if (f != 0.f) t = fmaf(ml[y].y, f, t);
                        }
                }
                finish(r, c, z, t);
            }
            if (threadIdx.x == 0) *arrived = 0;
        }
    }
    __syncwarp();
    cl.barrier_wait();
}

template <typename T, int HD>
cudaError_t launch_hd(const Kv8AttnArgs &a, cudaStream_t s) {
    const int smem = kKvAttnWarps * stages(HD) * 2 * kKvBlock * HD + HD / 16 * 32 * 16;
    // (the attribute is the device's: set once for each)
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        if ((e = cudaFuncSetAttribute(attn_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess)
            return e;
        if (dev < 64) ready.fetch_or(1ull << dev);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.splits * a.c.kv_heads * a.row_groups), a.c.n_seqs);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)a.cluster, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_kernel<T, HD>, a);
}
template <typename T>
cudaError_t launch_t(const Kv8AttnArgs &a, cudaStream_t s) {
    switch (a.c.head_dim) {
        case 32: return launch_hd<T, 32>(a, s);
        case 64: return launch_hd<T, 64>(a, s);
        case 96: return launch_hd<T, 96>(a, s);
        case 128: return launch_hd<T, 128>(a, s);
        case 160: return launch_hd<T, 160>(a, s);
        case 192: return launch_hd<T, 192>(a, s);
        case 224: return launch_hd<T, 224>(a, s);
        default: return launch_hd<T, 256>(a, s);
    }
}
}  // namespace

int kv8_attn_ctas_per_sm(int head_dim) { return ctas_per_sm(head_dim); }

cudaError_t kv8_attn_launch(const Kv8AttnArgs &a, bool bf16, cudaStream_t s) {
    return bf16 ? launch_t<__nv_bfloat16>(a, s) : launch_t<float>(a, s);
}

}  // namespace ql
