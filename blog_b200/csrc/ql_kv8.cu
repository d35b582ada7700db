// The 8-bit KV cache's writer and reader.
//
// Append, for each row (token) of a call: q_h and k_h of every head are normalised and rotated, v_h is
// taken as it is,
//   n = x / sqrt(mean(x^2) + eps) * gamma,   (a, b) -> (a cos - b sin, b cos + a sin)
// for the pairs (i, i + rotary_dim / 2) of the first rotary_dim elements, and k and v go to the cache:
//   a block of 32 tokens that is full is stored as scale = max|x| / 127 over its 32 x head_dim values of
//   one head and code = rint(x / scale) + 128 in a byte;
//   the rows of the last block and of the one before it are kept in f32 ("open" rows), so that a block
//   is quantised once, from exact values, when its last token arrives.
// The codes therefore do not depend on how a sequence was cut into calls, no code is ever re-scaled, and
// the last 32 tokens can be taken back.  A block that holds NaN or infinity gets a NaN scale.
//
// Every value is read once and written once, so the bound is HBM bandwidth for prompts and the launch for
// single tokens: one launch holds both kinds of work (CTAs of query heads, a warp per row and head, and
// CTAs of one block, KV head and operand, 4 rows per warp in registers until the block's maximum is known).
#include "ql_kv8.cuh"

namespace ql {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRowsPerWarp = kKvBlock / kWarps;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, as the widest accesses that N * sizeof(T) allows where VEC (the host has
// checked that every row starts on 16 bytes), else one by one.
template <int BYTES>
struct Piece;
template <>
struct Piece<16> { using type = uint4; };
template <>
struct Piece<8> { using type = uint2; };
template <>
struct Piece<4> { using type = uint32_t; };
template <>
struct Piece<2> { using type = uint16_t; };
template <>
struct Piece<1> { using type = uint8_t; };
constexpr int piece_bytes(int n) { return n % 16 == 0 ? 16 : n % 8 == 0 ? 8 : n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1; }

template <int N, bool VEC, typename T>
__device__ __forceinline__ void load_row(float *x, const T *p) {
    if constexpr (VEC) {
        constexpr int PB = piece_bytes(N * (int)sizeof(T)), NP = N * (int)sizeof(T) / PB, PE = PB / (int)sizeof(T);
        using P = typename Piece<PB>::type;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const P w = reinterpret_cast<const P *>(p)[i];
            const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int j = 0; j < PE; ++j) x[i * PE + j] = to_f32<T>(e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_f32<T>(p[i]);
    }
}
template <int N, bool VEC, typename T>
__device__ __forceinline__ void store_row(T *p, const float *x) {
    if constexpr (VEC) {
        constexpr int PB = piece_bytes(N * (int)sizeof(T)), NP = N * (int)sizeof(T) / PB, PE = PB / (int)sizeof(T);
        using P = typename Piece<PB>::type;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            P w;
            T *e = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int j = 0; j < PE; ++j) e[j] = from_f32<T>(x[i * PE + j]);
            reinterpret_cast<P *>(p)[i] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_f32<T>(x[i]);
    }
}

// Norm (gamma non-null) and rotation of one row spread over a warp, V consecutive elements per lane.
// cs: the position's cosines and sines, or null.  rotary_dim / 2 is a multiple of V, so an element and
// its partner have the same index in two lanes.
template <int V>
__device__ __forceinline__ void norm_rope(float *x, const float *gamma, float eps, const float *cs, int rotary_dim,
                                          int lane) {
    if (gamma != nullptr) {
        float g[V];
        load_row<V, false>(g, gamma + lane * V);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = 1.0f / sqrtf(ss * (1.0f / (32 * V)) + eps);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = x[i] * r * g[i];
    }
    if (cs != nullptr) {
        const int half = rotary_dim / 2, hl = half / V;  // lanes [0, hl): first halves; [hl, 2 hl): second
        const bool first = lane < hl, in = lane < 2 * hl;
        const int partner = in ? (first ? lane + hl : lane - hl) : lane;
        const int at = (first ? lane : lane - hl) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float o = __shfl_sync(0xffffffffu, x[i], partner);
            if (in) {
                const float c = cs[at + i], s = cs[half + at + i];
                x[i] = first ? x[i] * c - o * s : x[i] * c + o * s;
            }
        }
    }
}

// Cosines and sines of a position, or null when there is no rotation (or, recorded, no such position).
__device__ __forceinline__ const float *rope_row(const Kv8AppendArgs &a, int pos) {
    if (a.rotary_dim == 0) return nullptr;
    if (pos >= a.max_positions) {
        atomicExch(a.c.err, kErrKvPosition);
        return nullptr;
    }
    return a.rope + (int64_t)pos * a.rotary_dim;
}

// One block's rows of one KV head, K (norm, rotation) or V: rows [t0, t1) of the block come from this
// call, earlier ones from the open rows.  The whole CTA calls it.
template <typename T, int V, bool VEC>
__device__ void append_block(const Kv8AppendArgs &a, bool is_v, int seq, int slot, int kh, int block, int pos0, int row0,
                             int kv_len, bool keep, float *red) {
    constexpr int HD = 32 * V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int base = block * kKvBlock;
    const bool full = base + kKvBlock <= kv_len;
    const T *src = static_cast<const T *>(is_v ? a.v : a.k) + (int64_t)kh * HD + lane * V;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    float *open = (is_v ? a.c.v_open : a.c.k_open) + kv8_open_at(a.c, slot, block, kh) + lane * V;
    float x[kRowsPerWarp][V];
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u) {
        const int t = warp + u * kWarps, pos = base + t;
        if (pos >= pos0 && pos < kv_len) {
            load_row<V, VEC>(x[u], src + (int64_t)(row0 + pos - pos0) * stride);
        } else if (full) {  // an earlier token of a block that this call fills
            load_row<V, true>(x[u], open + t * HD);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x[u][i] = 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u) {
        const int t = warp + u * kWarps, pos = base + t;
        if (pos < pos0 || pos >= kv_len) continue;
        if (!is_v) norm_rope<V>(x[u], a.k_gamma, a.eps, rope_row(a, pos), a.rotary_dim, lane);
        if (keep) store_row<V, true>(open + t * HD, x[u]);
    }
    if (!full) return;
    float amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            amax = fmaxf(amax, fabsf(x[u][i]));
            bad |= !(fabsf(x[u][i]) < INFINITY);
        }
    if (bad) amax = INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) red[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) amax = fmaxf(amax, red[w]);
    const float scale = amax < INFINITY ? amax / 127.0f : __int_as_float(0x7FC00000);
    const int page = kv8_page(a.c, seq, block);
    if (page < 0) return;
    uint8_t *codes = (is_v ? a.c.v_codes : a.c.k_codes) + kv8_codes_at(a.c, page, kh) + lane * V;
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u) {
        const int t = warp + u * kWarps;
        constexpr int PB = piece_bytes(V);
        using P = typename Piece<PB>::type;
        uint8_t c[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float r = scale > 0.f ? fminf(fmaxf(rintf(x[u][i] / scale), -127.f), 127.f) : 0.f;
            c[i] = (uint8_t)((int)r + 128);
        }
#pragma unroll
        for (int i = 0; i < V / PB; ++i) {
            P w;
            uint8_t *e = reinterpret_cast<uint8_t *>(&w);
#pragma unroll
            for (int j = 0; j < PB; ++j) e[j] = c[i * PB + j];
            reinterpret_cast<P *>(codes + (int64_t)t * HD)[i] = w;
        }
    }
    if (threadIdx.x == 0) (is_v ? a.c.v_scale : a.c.k_scale)[(int64_t)page * a.c.kv_heads + kh] = scale;
}

// Grid: [0, q_ctas): query heads, a warp per (row, head); then a CTA per (tile, KV head, K or V).  With
// q_start, tile t belongs to the sequence s with start(s) <= t < start(s + 1), start(s) = q_start[s] / 32 +
// 2 s: a sequence of n rows touches at most floor(n / 32) + 2 blocks, and start(s + 1) - start(s) is at
// least that, so every block has a tile.
template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ Kv8AppendArgs a, int q_ctas) {
    constexpr int HD = 32 * V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if ((int)blockIdx.x < q_ctas) {
        const int64_t task = (int64_t)blockIdx.x * kWarps + warp;
        const int row = (int)(task / a.n_heads), h = (int)(task - (int64_t)row * a.n_heads);
        if (row >= a.r.rows) return;
        float x[V];
        load_row<V, VEC>(x, static_cast<const T *>(a.q) + (int64_t)row * a.q_stride + (int64_t)h * HD + lane * V);
        int seq = row, left = 1;  // rows of the sequence from this one on
        if (a.r.q_start != nullptr) {
            seq = kv8_seq_of_row(a.r.q_start, a.c.n_seqs, row, lane);
            left = a.r.q_start[seq + 1] - row;
        }
        const int pos = a.r.kv_len[seq] - left;
        if (pos < 0) return;  // an empty sequence (a length below its rows is recorded by the cache's CTAs)
        norm_rope<V>(x, a.q_gamma, a.eps, rope_row(a, pos), a.rotary_dim, lane);
        store_row<V, VEC>(static_cast<T *>(a.q_out) + (int64_t)row * a.q_out_stride + (int64_t)h * HD + lane * V, x);
        return;
    }
    __shared__ float red[kWarps];
    int t = blockIdx.x - q_ctas;
    const bool is_v = t & 1;
    t >>= 1;
    const int kh = t % a.c.kv_heads;
    t /= a.c.kv_heads;
    int seq = t, j = 0;
    if (a.r.q_start != nullptr) {
        // the last sequence whose first tile is at or before t
        int lo = 0, n = a.c.n_seqs;
        while (n > 1) {
            const int step = (n + 31) / 32, at = lo + lane * step;
            const bool le = lane * step < n && a.r.q_start[at] / kKvBlock + 2 * at <= t;
            const unsigned b = __ballot_sync(0xffffffffu, le);
            const int hit = b == 0 ? 0 : 31 - __clz(b);
            n = min(step, n - hit * step);
            lo += hit * step;
        }
        seq = lo;
        j = t - (a.r.q_start[seq] / kKvBlock + 2 * seq);
    }
    int row0, q_len;
    kv8_rows_of(a.r, seq, row0, q_len);
    const int kv_len = a.r.kv_len[seq];
    if (q_len <= 0 || kv_len <= 0) return;
    if (kv_len < q_len) {
        if (threadIdx.x == 0) atomicExch(a.c.err, kErrKvLength);
        return;
    }
    const int pos0 = kv_len - q_len, first = pos0 / kKvBlock, last = (kv_len - 1) / kKvBlock;
    const int block = first + j;
    if (block > last) return;
    if (last >= a.c.max_pages) {
        if (threadIdx.x == 0) atomicExch(a.c.err, kErrKvPage);
        return;
    }
    // The first block's earlier rows lie in the open rows of its parity, which one of the last two blocks
    // of the call overwrites: the first block's CTA does that one too, afterwards.
    const bool partial = pos0 % kKvBlock != 0;
    const int alias = ((last ^ first) & 1) == 0 ? last : last - 1;
    const bool deferred = partial && alias > first;
    if (deferred && block == alias) return;
    const int slot = kv8_slot(a.c, seq);
    if (slot < 0) return;
    append_block<T, V, VEC>(a, is_v, seq, slot, kh, block, pos0, row0, kv_len, block >= last - 1, red);
    if (deferred && block == first) {
        __syncthreads();
        append_block<T, V, VEC>(a, is_v, seq, slot, kh, alias, pos0, row0, kv_len, true, red);
    }
}

// Rows start .. start + count - 1 of every sequence, [n_seqs][count][kv_heads][head_dim]; positions outside
// the sequence give zeros.  A warp per (position, KV head, K or V).
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) gather_kernel(const __grid_constant__ Kv8View c, const int *kv_len,
                                                          const int *start, int count, T *k_out, T *v_out) {
    constexpr int HD = 32 * V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tasks = (int64_t)c.n_seqs * count * c.kv_heads * 2;
    const int64_t task = (int64_t)blockIdx.x * kWarps + warp;
    if (task >= tasks) return;
    const bool is_v = task >= tasks / 2;
    const int64_t row = is_v ? task - tasks / 2 : task;  // (seq, i, kh)
    T *out = is_v ? v_out : k_out;
    if (out == nullptr) return;
    const int kh = (int)(row % c.kv_heads);
    const int64_t si = row / c.kv_heads;
    const int seq = (int)(si / count);
    const int64_t pos64 = (int64_t)(start != nullptr ? start[seq] : 0) + si % count;
    const int len = kv_len[seq];
    float x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = 0.f;
    if (pos64 >= 0 && pos64 < len) {
        const int pos = (int)pos64, block = pos / kKvBlock, t = pos % kKvBlock;
        if ((block + 1) * kKvBlock > len) {
            const int slot = kv8_slot(c, seq);
            if (slot >= 0)
                load_row<V, true>(x, (is_v ? c.v_open : c.k_open) + kv8_open_at(c, slot, block, kh) + t * HD + lane * V);
        } else {
            const int page = kv8_page(c, seq, block);
            if (page >= 0) {
                const uint8_t *p = (is_v ? c.v_codes : c.k_codes) + kv8_codes_at(c, page, kh) + t * HD + lane * V;
                const float s = (is_v ? c.v_scale : c.k_scale)[(int64_t)page * c.kv_heads + kh];
                constexpr int PB = piece_bytes(V);
                using P = typename Piece<PB>::type;
#pragma unroll
                for (int i = 0; i < V / PB; ++i) {
                    const P w = reinterpret_cast<const P *>(p)[i];
                    const uint8_t *e = reinterpret_cast<const uint8_t *>(&w);
#pragma unroll
                    for (int j = 0; j < PB; ++j) x[i * PB + j] = (float)((int)e[j] - 128) * s;
                }
            }
        }
    }
    store_row<V, true>(out + row * HD + lane * V, x);
}

template <typename T, int V>
cudaError_t append_v(const Kv8AppendArgs &a, cudaStream_t s) {
    const int64_t q_ctas = a.q != nullptr ? ((int64_t)a.r.rows * a.n_heads + kWarps - 1) / kWarps : 0;
    const int64_t tiles = a.r.q_start != nullptr ? a.r.rows / kKvBlock + 2 * (int64_t)a.c.n_seqs : a.r.rows;
    const int64_t grid = q_ctas + tiles * a.c.kv_heads * 2;
    const size_t el = sizeof(T);
    auto ok = [&](const void *p, int64_t stride) {
        return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * el) % 16 == 0);
    };
    const bool vec = ok(a.q, a.q_stride) && ok(a.k, a.k_stride) && ok(a.v, a.v_stride) && ok(a.q_out, a.q_out_stride);
    if (vec)
        append_kernel<T, V, true><<<(unsigned)grid, kThreads, 0, s>>>(a, (int)q_ctas);
    else
        append_kernel<T, V, false><<<(unsigned)grid, kThreads, 0, s>>>(a, (int)q_ctas);
    return cudaGetLastError();
}
template <typename T>
cudaError_t append_t(const Kv8AppendArgs &a, cudaStream_t s) {
    switch (a.c.head_dim / 32) {
        case 1: return append_v<T, 1>(a, s);
        case 2: return append_v<T, 2>(a, s);
        case 3: return append_v<T, 3>(a, s);
        case 4: return append_v<T, 4>(a, s);
        case 5: return append_v<T, 5>(a, s);
        case 6: return append_v<T, 6>(a, s);
        case 7: return append_v<T, 7>(a, s);
        default: return append_v<T, 8>(a, s);
    }
}
template <typename T, int V>
cudaError_t gather_v(const Kv8View &c, const int *kv_len, const int *start, int count, void *k, void *v, cudaStream_t s) {
    const int64_t tasks = (int64_t)c.n_seqs * count * c.kv_heads * 2;
    gather_kernel<T, V><<<(unsigned)((tasks + kWarps - 1) / kWarps), kThreads, 0, s>>>(
        c, kv_len, start, count, static_cast<T *>(k), static_cast<T *>(v));
    return cudaGetLastError();
}
template <typename T>
cudaError_t gather_t(const Kv8View &c, const int *kv_len, const int *start, int count, void *k, void *v, cudaStream_t s) {
    switch (c.head_dim / 32) {
        case 1: return gather_v<T, 1>(c, kv_len, start, count, k, v, s);
        case 2: return gather_v<T, 2>(c, kv_len, start, count, k, v, s);
        case 3: return gather_v<T, 3>(c, kv_len, start, count, k, v, s);
        case 4: return gather_v<T, 4>(c, kv_len, start, count, k, v, s);
        case 5: return gather_v<T, 5>(c, kv_len, start, count, k, v, s);
        case 6: return gather_v<T, 6>(c, kv_len, start, count, k, v, s);
        case 7: return gather_v<T, 7>(c, kv_len, start, count, k, v, s);
        default: return gather_v<T, 8>(c, kv_len, start, count, k, v, s);
    }
}
}  // namespace

cudaError_t kv8_append_launch(const Kv8AppendArgs &a, bool bf16, cudaStream_t s) {
    return bf16 ? append_t<__nv_bfloat16>(a, s) : append_t<float>(a, s);
}
cudaError_t kv8_gather_launch(const Kv8View &c, const int *kv_len, const int *start, int count, void *k_out, void *v_out,
                              bool bf16, cudaStream_t s) {
    return bf16 ? gather_t<__nv_bfloat16>(c, kv_len, start, count, k_out, v_out, s)
                : gather_t<float>(c, kv_len, start, count, k_out, v_out, s);
}

}  // namespace ql
