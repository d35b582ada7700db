// Rules on logits before the next token is taken, one pass: for token t of a row, with n the times t was
// generated and "seen" whether it is in the prompt or was generated,
//   y = x,   seen: y = x > 0 ? x / repetition : x * repetition
//   y = y - frequency * n,   n > 0: y = y - presence
//   y = y + each bias listed for t, in list order
//   y = -inf where the row's mask has a zero bit
// and the row's greedy token: the largest y, the lowest index among equals, -1 where nothing is above -inf.
// Each step is one fp32 operation, rounded once, in this order.
//
// Bound: HBM, each logit read once and written once.  A CTA takes a chunk of a row: it issues the loads of
// its logits first, and while they are in flight counts the history's tokens that fall into the chunk in
// shared memory (integer counts: their order does not matter), so no table of the vocabulary goes through
// memory.  The history is read once per chunk, from L2.
#include "ql_logits.cuh"

namespace ql {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u, kBias = 0x40000000u, kCount = 0x3FFFFFFFu;

// NV: groups of 4 logits per thread; a chunk is kThreads * 4 * NV tokens.  VEC: rows start on 16 bytes and
// a group is one 16-byte access; otherwise a group's four tokens are kThreads apart.
template <int NV, bool VEC>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ LogitsArgs a) {
    constexpr int kChunk = kThreads * 4 * NV;
    __shared__ __align__(16) uint32_t tab[kChunk];
    __shared__ unsigned long long s_key[kThreads / 32];
    const int row = blockIdx.y, base = blockIdx.x * kChunk, n_tok = min(kChunk, a.vocab - base);
    const int tid = threadIdx.x;
    const float *x = a.logits + (int64_t)row * a.logits_stride + base;
    auto at = [&](int v, int e) { return VEC ? (v * kThreads + tid) * 4 + e : (v * 4 + e) * kThreads + tid; };
    float y[NV][4];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (VEC && at(v, 3) < n_tok) {
            const float4 w = *reinterpret_cast<const float4 *>(x + at(v, 0));
            y[v][0] = w.x, y[v][1] = w.y, y[v][2] = w.z, y[v][3] = w.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[v][e] = at(v, e) < n_tok ? x[at(v, e)] : -INFINITY;
        }
    }
    const int hist = a.history != nullptr ? (int)min((int64_t)a.history_len[row], a.history_stride) : 0;
    const int prompt = a.history != nullptr && a.prompt_len != nullptr ? a.prompt_len[row] : 0;
    const int b0 = a.bias_ids != nullptr ? a.bias_start[row] : 0, b1 = a.bias_ids != nullptr ? a.bias_start[row + 1] : 0;
    const bool table = hist > 0 || b1 > b0;
    if (table) {
#pragma unroll
        for (int v = 0; v < NV; ++v) reinterpret_cast<uint4 *>(tab)[v * kThreads + tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int *h = a.history + (int64_t)row * a.history_stride;
        for (int i = tid; i < hist; i += kThreads) {
            const int t = h[i] - base;
            if (t >= 0 && t < n_tok) {
                if (i < prompt)
                    atomicOr(&tab[t], kPrompt);
                else
                    atomicAdd(&tab[t], 1u);
            }
        }
        for (int i = b0 + tid; i < b1; i += kThreads) {
            const int t = a.bias_ids[i] - base;
            if (t >= 0 && t < n_tok) atomicOr(&tab[t], kBias);
        }
        __syncthreads();
        const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
        const float freq = a.frequency != nullptr ? a.frequency[row] : 0.f;
        const float pres = a.presence != nullptr ? a.presence[row] : 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t c = tab[at(v, e)];
                if (c == 0) continue;
                float z = y[v][e];
                const uint32_t n = c & kCount;
                if ((c & ~kBias) != 0 && a.repetition != nullptr) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
                if (n != 0) {
                    z = __fsub_rn(z, __fmul_rn(freq, (float)n));
                    z = __fsub_rn(z, pres);
                }
                if (c & kBias)
                    for (int i = b0; i < b1; ++i)
                        if (a.bias_ids[i] - base == at(v, e)) z = __fadd_rn(z, a.bias_values[i]);
                y[v][e] = z;
            }
        }
    }
    const int mr = a.mask == nullptr ? -1 : a.mask_row != nullptr ? a.mask_row[row] : row;
    if (mr >= 0) {
        const bool ok = mr < a.mask_rows;  // a row outside the masks allows nothing
        if (!ok && tid == 0) atomicExch(a.err, kErrMaskRow);
        const uint32_t *m = a.mask + (int64_t)mr * a.mask_stride + base / 32;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = at(v, e);
                if (t < n_tok && !(ok && (m[t / 32] >> (t % 32) & 1))) y[v][e] = -INFINITY;
            }
        }
    }
    if (a.out != nullptr) {
        float *o = a.out + (int64_t)row * a.out_stride + base;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (VEC && at(v, 3) < n_tok) {
                *reinterpret_cast<float4 *>(o + at(v, 0)) = make_float4(y[v][0], y[v][1], y[v][2], y[v][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at(v, e) < n_tok) o[at(v, e)] = y[v][e];
            }
        }
    }
    if (a.token == nullptr) return;
    unsigned long long key = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned long long k = at(v, e) < n_tok ? amax_key(y[v][e], (uint32_t)(base + at(v, e))) : 0ull;
            key = k > key ? k : key;
        }
    key = warp_max_u64(key);
    if (tid % 32 == 0) s_key[tid / 32] = key;
    __syncthreads();
    if (tid != 0) return;
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) key = s_key[w] > key ? s_key[w] : key;
    if (gridDim.x > 1) {
        atomicMax(a.keys + row, key);
        __threadfence();
        if (atomicAdd(a.done + row, 1u) != gridDim.x - 1) return;
        __threadfence();
        key = atomicExch(a.keys + row, 0ull);
        a.done[row] = 0;
    }
    a.token[row] = key != 0 ? amax_index(key) : -1;
}

template <int NV>
cudaError_t launch(const LogitsArgs &a, cudaStream_t s) {
    auto ok = [](const void *p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 4 == 0; };
    constexpr int chunk = kThreads * 4 * NV;
    const dim3 grid((a.vocab + chunk - 1) / chunk, a.rows);
    if (ok(a.logits, a.logits_stride) && ok(a.out, a.out_stride))
        logits_kernel<NV, true><<<grid, kThreads, 0, s>>>(a);
    else
        logits_kernel<NV, false><<<grid, kThreads, 0, s>>>(a);
    return cudaGetLastError();
}
}  // namespace

cudaError_t logits_launch(const LogitsArgs &a, int sms, cudaStream_t s) {
    (void)sms;
    return launch<4>(a, s);
}

}  // namespace ql
