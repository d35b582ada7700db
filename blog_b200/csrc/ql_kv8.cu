// The 8-bit KV cache's writer and reader.
//
// Append, for each row (token) of a call: q_h and k_h of every head are normalised and rotated, v_h is
// taken as it is,
//   n = x / sqrt(mean(x^2) + eps) * gamma,   (a, b) -> (a cos - b sin, b cos + a sin)
// for the pairs (i, i + rotary_dim / 2) of the first rotary_dim elements, and k and v go to the cache:
//   a block of 32 tokens that is full is stored as scale = max|x| / 127 over its 32 x head_dim values of
//   one head and code = rint(x / scale) + 128 in a byte (x / scale within +-127);
//   the rows of the last block and of the one before it are kept in f32 ("open" rows), so that a block
//   is quantised once, from exact values, when its last token arrives.
// The codes therefore do not depend on how a sequence was cut into calls, no code is ever re-scaled, and
// the last 32 tokens can be taken back.  A block that holds NaN or infinity gets a NaN scale.
//
// Every value is read once and written once, so the bound is HBM bandwidth for prompts and the launch for
// single tokens: one launch holds both kinds of work (CTAs of query heads, a warp per row and head, and
// CTAs of one block, KV head and operand, 4 rows per warp in registers until the block's maximum is known).
// With the read-back of the rows it touched: 4096 tokens of 28/4/128 heads in f32, 147 MB: 36 us, 4.1 TB/s (the append by
// itself 31 us).  8 chunks of up to 1500 tokens of 64/8/128 heads in bf16, 347 MB: 128 us, 2.7 TB/s (111 us): two thirds of
// the issue slots go to norm, rotation and conversion (half the bytes per value), the rest waits for loads and shuffles.
// One token: 4.4 us.
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
            if constexpr (sizeof(T) == 2 && PE % 2 == 0) {
                __nv_bfloat162 *e = reinterpret_cast<__nv_bfloat162 *>(&w);
#pragma unroll
                for (int j = 0; j < PE / 2; ++j) e[j] = __floats2bfloat162_rn(x[i * PE + 2 * j], x[i * PE + 2 * j + 1]);
            } else {
                T *e = reinterpret_cast<T *>(&w);
#pragma unroll
                for (int j = 0; j < PE; ++j) e[j] = from_f32<T>(x[i * PE + j]);
            }
            reinterpret_cast<P *>(p)[i] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_f32<T>(x[i]);
    }
}

// What a lane needs of a position's rotation: the cosines and sines of its V elements, the lane that holds
// their partners (the same index there: rotary_dim / 2 is a multiple of V) and the sign of the partner's term.
template <int V>
struct Rotation {
    float c[V], s[V];
    int partner;
    bool in;
    __device__ __forceinline__ void load(const float *cs, int rotary_dim, int lane) {
        const int hl = rotary_dim / (2 * V);  // lanes [0, hl): first halves; [hl, 2 hl): second
        const bool first = lane < hl;
        in = cs != nullptr && lane < 2 * hl;
        partner = in ? (first ? lane + hl : lane - hl) : lane;
        const int at = (first ? lane : lane - hl) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c[i] = in ? cs[at + i] : 1.f;
            const float z = in ? cs[rotary_dim / 2 + at + i] : 0.f;
            s[i] = first ? -z : z;
        }
    }
};

// Norm (gamma non-null: the lane's g) and rotation of one row spread over a warp, V consecutive elements per
// lane.
template <int V>
__device__ __forceinline__ void norm_rope(float *x, bool norm, const float *g, float eps, bool rotate, const Rotation<V> &r) {
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float f = rsqrtf(fmaf(ss, 1.0f / (32 * V), eps));
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = x[i] * f * g[i];
    }
    if (rotate) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float o = __shfl_sync(0xffffffffu, x[i], r.partner);
            if (r.in) x[i] = fmaf(o, r.s[i], x[i] * r.c[i]);
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
    float x[kRowsPerWarp][V], g[V];
    const bool norm = !is_v && a.k_gamma != nullptr, rotate = !is_v && a.rotary_dim > 0;
    if (norm) load_row<V, false>(g, a.k_gamma + lane * V);
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
        Rotation<V> rot;
        if (rotate) rot.load(rope_row(a, pos), a.rotary_dim, lane);
        norm_rope<V>(x[u], norm, g, a.eps, rotate, rot);
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
    // rint(x / scale): the quotient from the block's one reciprocal and a residual step, which rounds it
    // correctly (P. Markstein, 1990; ties of bf16 values are common and go by the last bit), then 1.5 x 2^23
    // added, which rounds to an integer, half to even, with the code in the low byte.  Scales near the ends of
    // the range are divided by, and the quotient kept within 127: a subnormal scale is too coarse to keep it there.
    const float inv = 1.0f / scale;
    const bool divide = !(scale > 1e-30f && scale < 1e30f);
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u) {
        const int t = warp + u * kWarps;
        constexpr int PB = piece_bytes(V);
        using P = typename Piece<PB>::type;
        uint32_t c[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float r = x[u][i] * inv;
            r = divide ? (scale > 0.f ? fminf(fmaxf(x[u][i] / scale, -127.f), 127.f) : 0.f)
                       : fmaf(fmaf(-r, scale, x[u][i]), inv, r);
            c[i] = __float_as_uint(r + 12582912.0f) ^ 0x80u;
        }
#pragma unroll
        for (int i = 0; i < V / PB; ++i) {
            P w;
            if constexpr (PB >= 4) {
                uint32_t *e = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
                for (int j = 0; j < PB / 4; ++j) {
                    const uint32_t *z = c + i * PB + 4 * j;
                    e[j] = __byte_perm(__byte_perm(z[0], z[1], 0x0040), __byte_perm(z[2], z[3], 0x0040), 0x5410);
                }
            } else {
                uint8_t *e = reinterpret_cast<uint8_t *>(&w);
#pragma unroll
                for (int j = 0; j < PB; ++j) e[j] = (uint8_t)c[i * PB + j];
            }
            reinterpret_cast<P *>(codes + (int64_t)t * HD)[i] = w;
        }
    }
    if (threadIdx.x == 0) (is_v ? a.c.v_scale : a.c.k_scale)[(int64_t)page * a.c.kv_heads + kh] = scale;
}

// Grid: [0, q_ctas): query heads, a warp per row and HPW heads of it; then a CTA per (tile, KV head, K or V).
// With q_start, tile t belongs to the sequence s with start(s) <= t < start(s + 1), start(s) = q_start[s] / 32 +
// 2 s: a sequence of n rows touches at most floor(n / 32) + 2 blocks, and start(s + 1) - start(s) is at
// least that, so every block has a tile.
template <typename T, int V, bool VEC, int HPW>
__global__ void __launch_bounds__(kThreads, V <= 4 ? 5 : 3) append_kernel(const __grid_constant__ Kv8AppendArgs a, int q_ctas) {
    constexpr int HD = 32 * V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if ((int)blockIdx.x < q_ctas) {
        const int per_row = (a.n_heads + HPW * kWarps - 1) / (HPW * kWarps);  // CTAs
        const int row = blockIdx.x / per_row, h0 = ((blockIdx.x - row * per_row) * kWarps + warp) * HPW;
        if (h0 >= a.n_heads) return;
        float x[HPW][V], g[V];
        const T *q = static_cast<const T *>(a.q) + (int64_t)row * a.q_stride + (int64_t)h0 * HD + lane * V;
#pragma unroll
        for (int u = 0; u < HPW; ++u)
            if (h0 + u < a.n_heads) load_row<V, VEC>(x[u], q + u * HD);
        const bool norm = a.q_gamma != nullptr;
        if (norm) load_row<V, false>(g, a.q_gamma + lane * V);
        int seq = row, left = 1;  // rows of the sequence from this one on
        if (a.r.q_start != nullptr) {
            seq = kv8_seq_of_row(a.r.q_start, a.c.n_seqs, row, lane);
            left = a.r.q_start[seq + 1] - row;
        }
        const int pos = a.r.kv_len[seq] - left;
        if (pos < 0) return;  // an empty sequence (a length below its rows is recorded by the cache's CTAs)
        Rotation<V> rot;
        if (a.rotary_dim > 0) rot.load(rope_row(a, pos), a.rotary_dim, lane);
        T *o = static_cast<T *>(a.q_out) + (int64_t)row * a.q_out_stride + (int64_t)h0 * HD + lane * V;
#pragma unroll
        for (int u = 0; u < HPW; ++u)
            if (h0 + u < a.n_heads) {
                norm_rope<V>(x[u], norm, g, a.eps, a.rotary_dim > 0, rot);
                store_row<V, VEC>(o + u * HD, x[u]);
            }
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
    if (q_len <= 0 || kv_len == 0) return;
    if (kv_len < q_len) {
        if (threadIdx.x == 0) atomicExch(a.c.err, kErrKvLength);
        return;
    }
    const int pos0 = kv_len - q_len, first = pos0 / kKvBlock, last = (kv_len - 1) / kKvBlock;
    const int block = first + j;
    if (j < 0 || block > last) return;  // (j < 0: rows before q_start[0] are nobody's)
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
// the sequence give zeros.  A thread per 16 values of K or of V.
template <typename T>
__global__ void __launch_bounds__(kThreads) gather_kernel(const __grid_constant__ Kv8View c, const int *kv_len,
                                                          const int *start, int count, T *k_out, T *v_out, int64_t pieces) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const bool is_v = blockIdx.y != 0;
    T *out = is_v ? v_out : k_out;
    if (i >= pieces || out == nullptr) return;
    const int per = c.head_dim / 16;
    const int64_t row = i / per;  // (seq, token, kh)
    const int at = (int)(i - row * per) * 16, kh = (int)(row % c.kv_heads);
    const int64_t si = row / c.kv_heads;
    const int seq = (int)(si / count);
    const int64_t pos64 = (int64_t)(start != nullptr ? start[seq] : 0) + (si - (int64_t)seq * count);
    const int len = kv_len[seq];
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.f;
    if (pos64 >= 0 && pos64 < len) {
        const int pos = (int)pos64, block = pos / kKvBlock, t = pos % kKvBlock;
        if ((block + 1) * kKvBlock > len) {
            const int slot = kv8_slot(c, seq);
            if (slot >= 0)
                load_row<16, true>(x, (is_v ? c.v_open : c.k_open) + kv8_open_at(c, slot, block, kh) + t * c.head_dim + at);
        } else {
            const int page = kv8_page(c, seq, block);
            if (page >= 0) {
                const uint4 w = *reinterpret_cast<const uint4 *>((is_v ? c.v_codes : c.k_codes) + kv8_codes_at(c, page, kh) +
                                                                 t * c.head_dim + at);
                const float s = (is_v ? c.v_scale : c.k_scale)[(int64_t)page * c.kv_heads + kh];
                const uint8_t *e = reinterpret_cast<const uint8_t *>(&w);
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = (float)((int)e[j] - 128) * s;
            }
        }
    }
    store_row<16, true>(out + i * 16, x);
}

template <typename T, int V, bool VEC>
cudaError_t append_hpw(const Kv8AppendArgs &a, cudaStream_t s) {
    const int64_t tiles = a.r.q_start != nullptr ? a.r.rows / kKvBlock + 2 * (int64_t)a.c.n_seqs : a.r.rows;
    const int64_t kv_ctas = tiles * a.c.kv_heads * 2;
    // Heads per warp: 1 for single tokens, where the launch is as long as one warp's chain of loads; for
    // prompts 4, whose loads are in flight together and share the row's cosines and sines.
    const bool many = (int64_t)a.r.rows * a.n_heads >= 8192;
    const int hpw = many ? 4 : 1;
    const int64_t q_ctas = a.q != nullptr ? (int64_t)a.r.rows * ((a.n_heads + hpw * kWarps - 1) / (hpw * kWarps)) : 0;
    if (many)
        append_kernel<T, V, VEC, 4><<<(unsigned)(q_ctas + kv_ctas), kThreads, 0, s>>>(a, (int)q_ctas);
    else
        append_kernel<T, V, VEC, 1><<<(unsigned)(q_ctas + kv_ctas), kThreads, 0, s>>>(a, (int)q_ctas);
    return cudaGetLastError();
}
template <typename T, int V>
cudaError_t append_v(const Kv8AppendArgs &a, cudaStream_t s) {
    auto ok = [](const void *p, int64_t stride) {
        return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0);
    };
    return ok(a.q, a.q_stride) && ok(a.k, a.k_stride) && ok(a.v, a.v_stride) && ok(a.q_out, a.q_out_stride)
               ? append_hpw<T, V, true>(a, s)
               : append_hpw<T, V, false>(a, s);
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
template <typename T>
cudaError_t gather_t(const Kv8View &c, const int *kv_len, const int *start, int count, void *k, void *v, cudaStream_t s) {
    const int64_t pieces = (int64_t)c.n_seqs * count * c.kv_heads * (c.head_dim / 16);
    gather_kernel<T><<<dim3((unsigned)((pieces + kThreads - 1) / kThreads), 2), kThreads, 0, s>>>(
        c, kv_len, start, count, static_cast<T *>(k), static_cast<T *>(v), pieces);
    return cudaGetLastError();
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
