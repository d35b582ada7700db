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
// memory.  The history is read once per chunk, from L2.  Only the tokens that the table marks go through the rules.
// 64 rows of 152064 with histories of up to 4096, 300 biases and half of them masked, 79 MB: 30.5 us, 2.6 TB/s, the
// chain of history, count and rules of each chunk at 4 CTAs per SM; one row of 32001: 5.1 us.  Chunks of 8192 tokens
// read the history 19 times a row, of 1024 150 times; those are for few rows (NV = 1).
#include "ql_logits.cuh"

namespace ql {
namespace {

constexpr int kThreads = 256;
// A token's word in the table: in the prompt, has a bias, has several, the list's slot of the first, and how
// often it was generated.
constexpr uint32_t kPrompt = 1u << 31, kBias = 1u << 30, kMore = 1u << 29, kCount = kLogitsMaxHistory;
constexpr int kSlotBit = 20;
static_assert(kCount + 1 == 1u << kSlotBit, "counts below the slot");

constexpr int kBiasList = 512;  // biases of one chunk kept in shared memory

// NV: groups of 4 logits per thread; a chunk is kThreads * 4 * NV tokens.  VEC: rows start on 16 bytes and
// a group is one 16-byte access; otherwise a group's four tokens are kThreads apart.
template <int NV, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) logits_kernel(const __grid_constant__ LogitsArgs a) {
    constexpr int kChunk = kThreads * 4 * NV;
    __shared__ __align__(16) uint32_t tab[kChunk];      // counts and flags, then the value under the rules
    __shared__ unsigned long long s_key[kThreads / 32];
    __shared__ int b_tok[kBiasList], b_no[kBiasList], n_bias;  // the chunk's biases in any order: token, number
    __shared__ float b_val[kBiasList], s_best[kThreads / 32];
    const int row = blockIdx.y, base = blockIdx.x * kChunk, n_tok = min(kChunk, a.vocab - base);
    const int tid = threadIdx.x;
    const float *x = a.logits + (int64_t)row * a.logits_stride + base;
    auto at = [&](int v, int e) { return VEC ? (v * kThreads + tid) * 4 + e : (v * 4 + e) * kThreads + tid; };
    // what the row needs from memory, all of it under way before the first wait
    const int mr = a.mask == nullptr ? -1 : a.mask_row != nullptr ? a.mask_row[row] : row;
    const int hist = a.history != nullptr ? (int)min((int64_t)a.history_len[row], a.history_stride) : 0;
    const int prompt = a.history != nullptr && a.prompt_len != nullptr ? a.prompt_len[row] : 0;
    const int b0 = a.bias_ids != nullptr ? a.bias_start[row] : 0, b1 = a.bias_ids != nullptr ? a.bias_start[row + 1] : 0;
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
    const bool mask_ok = mr < a.mask_rows;  // a row outside the masks allows nothing
    if (mr >= 0 && !mask_ok && tid == 0) atomicExch(a.err, kErrMaskRow);
    uint32_t allow = 0xFFFFFFFFu;  // bit 4 v + e: the token at(v, e)
    static_assert(NV <= 8, "one bit per token of the thread");
    if (mr >= 0) {
        allow = 0;
        const uint32_t *m = a.mask + (int64_t)mr * a.mask_stride + base / 32;
        if (mask_ok) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (VEC) {  // four tokens of one word
                    if (at(v, 0) < n_tok) allow |= (m[at(v, 0) / 32] >> (at(v, 0) % 32) & 15u) << (4 * v);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at(v, e) < n_tok) allow |= (m[at(v, e) / 32] >> (at(v, e) % 32) & 1u) << (4 * v + e);
                }
            }
        }
    }
    if (hist > 0 || b1 > b0) {
#pragma unroll
        for (int v = 0; v < NV; ++v) reinterpret_cast<uint4 *>(tab)[v * kThreads + tid] = make_uint4(0, 0, 0, 0);
        if (tid == 0) n_bias = 0;
        __syncthreads();
        // the first kThreads biases are loaded before the history is gone through
        const int my_id = b0 + tid < b1 ? a.bias_ids[b0 + tid] : 0;
        const float my_w = b0 + tid < b1 ? a.bias_values[b0 + tid] : 0.f;
        const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
        const float freq = a.frequency != nullptr ? a.frequency[row] : 0.f;
        const float pres = a.presence != nullptr ? a.presence[row] : 0.f;
        const int *h = a.history + (int64_t)row * a.history_stride;
        auto count = [&](int id, int i) {
            const uint32_t t = (uint32_t)(id - base);
            if (t >= (uint32_t)n_tok) return;
            if (i < prompt)
                atomicOr(&tab[t], kPrompt);
            else
                atomicAdd(&tab[t], 1u);
        };
        // eight ids per thread in flight; the few that fall into the chunk are counted one by one
        const bool vec = reinterpret_cast<uintptr_t>(h) % 16 == 0;
        for (int i0 = 0; i0 < hist; i0 += 8 * kThreads) {
            int id[8];
            if (vec && i0 + 8 * kThreads <= hist) {
                const int4 p = reinterpret_cast<const int4 *>(h + i0)[2 * tid], q = reinterpret_cast<const int4 *>(h + i0)[2 * tid + 1];
                id[0] = p.x, id[1] = p.y, id[2] = p.z, id[3] = p.w, id[4] = q.x, id[5] = q.y, id[6] = q.z, id[7] = q.w;
            } else {
                const int *g = h + i0 + 8 * tid;
                const int n = hist - i0 - 8 * tid;
#pragma unroll
                for (int u = 0; u < 8; ++u) id[u] = u < n ? g[u] : -1;
            }
            bool any = false;
#pragma unroll
            for (int u = 0; u < 8; ++u) any |= (uint32_t)(id[u] - base) < (uint32_t)n_tok;
            if (!any) continue;
#pragma unroll
            for (int u = 0; u < 8; ++u) count(id[u], i0 + 8 * tid + u);
        }
        for (int i = b0 + tid; i < b1; i += kThreads) {
            const bool mine = i == b0 + tid;
            const uint32_t t = (uint32_t)((mine ? my_id : a.bias_ids[i]) - base);
            if (t >= (uint32_t)n_tok) continue;
            const int to = atomicAdd(&n_bias, 1);
            if (to < kBiasList) {
                b_tok[to] = (int)t;
                b_no[to] = i;
                b_val[to] = mine ? my_w : a.bias_values[i];
            }
            const bool more = atomicOr(&tab[t], kBias) & kBias;
            atomicOr(&tab[t], more || to >= kBiasList ? kMore : (uint32_t)to << kSlotBit);
        }
        __syncthreads();
        const int nb = n_bias;
        // of the thread's tokens, those that some rule touches (few): one code path for all of them
        uint32_t hit = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (VEC) {
                const uint4 c = reinterpret_cast<const uint4 *>(tab)[v * kThreads + tid];
                hit |= ((c.x != 0) | (c.y != 0) << 1 | (c.z != 0) << 2 | (c.w != 0) << 3) << (4 * v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) hit |= (uint32_t)(tab[at(v, e)] != 0) << (4 * v + e);
            }
        }
        for (uint32_t left = hit; left != 0; left &= left - 1) {
            const int k = __ffs(left) - 1, t = at(k / 4, k % 4);
            const uint32_t c = tab[t], n = c & kCount;
            float z = x[t];
            if ((c & (kPrompt | kCount)) != 0 && a.repetition != nullptr) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
            if (n != 0) {
                z = __fsub_rn(z, __fmul_rn(freq, (float)n));
                z = __fsub_rn(z, pres);
            }
            if (c & kBias) {
                if (!(c & kMore)) {
                    z = __fadd_rn(z, b_val[(c & ~(kPrompt | kBias)) >> kSlotBit]);
                } else if (nb <= kBiasList) {  // the token's biases by their numbers
                    for (int last = -1;;) {
                        int next = INT32_MAX;
                        float w = 0.f;
                        for (int i = 0; i < nb; ++i)
                            if (b_tok[i] == t && b_no[i] > last && b_no[i] < next) {
                                next = b_no[i];
                                w = b_val[i];
                            }
                        if (next == INT32_MAX) break;
                        z = __fadd_rn(z, w);
                        last = next;
                    }
                } else {  // more of them than the list holds
                    for (int i = b0; i < b1; ++i)
                        if (a.bias_ids[i] - base == t) z = __fadd_rn(z, a.bias_values[i]);
                }
            }
            tab[t] = __float_as_uint(z);  // (the thread's own token)
        }
        if (hit != 0) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (hit >> (4 * v + e) & 1u) y[v][e] = __uint_as_float(tab[at(v, e)]);
        }
    }
    if (mr >= 0) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(allow >> (4 * v + e) & 1u)) y[v][e] = -INFINITY;
    }
    if (a.token != nullptr) {
        // the chunk's largest value first, then the lowest of its places: only the warps that hold it look
        float best = -INFINITY;  // (also past the row's end; NaN never wins)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e) best = fmaxf(best, y[v][e]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (tid % 32 == 0) s_best[tid / 32] = best;
        if (tid < kThreads / 32) s_key[tid] = 0;
        __syncthreads();
        float top = s_best[0];
#pragma unroll
        for (int w = 1; w < kThreads / 32; ++w) top = fmaxf(top, s_best[w]);
        unsigned long long key = 0;
        if (best == top) {
            int where = kChunk;
#pragma unroll
            for (int v = NV - 1; v >= 0; --v)
#pragma unroll
                for (int e = 3; e >= 0; --e)
                    if (y[v][e] == top) where = at(v, e);
            where = __reduce_min_sync(0xffffffffu, where);
            if (tid % 32 == 0) s_key[tid / 32] = amax_key(top, (uint32_t)(base + where));
        }
        __syncthreads();
        if (tid == 0) {  // (before the stores: the fence has nothing of theirs to wait for)
            bool last = true;
#pragma unroll
            for (int w = 0; w < kThreads / 32; ++w) key = s_key[w] > key ? s_key[w] : key;
            if (gridDim.x > 1) {
                atomicMax(a.keys + row, key);
                __threadfence();
                last = atomicAdd(a.done + row, 1u) == gridDim.x - 1;
                if (last) {
                    __threadfence();
                    key = atomicExch(a.keys + row, 0ull);
                    a.done[row] = 0;
                }
            }
            if (last) a.token[row] = key != 0 ? amax_index(key) : -1;
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
    return (int64_t)a.rows * ((a.vocab + 8191) / 8192) >= sms ? launch<8>(a, s) : launch<1>(a, s);
}

}  // namespace ql
