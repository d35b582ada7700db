// Choice of experts, a warp per token:
//   s_e = softmax over the experts' logits, or sigmoid of each;   c_e = s_e + bias_e
//   group g counts by the sum of its group_best largest c; the top_groups best groups stay
//   the k experts of largest c in them, the lowest id among equals, by descending c
//   w_e = s_e [/ sum of the chosen s] * scale
// Without a bias experts stand by their logits, which no rounding touches.  Otherwise the order is that of 64-bit scores:
// the kernel first goes by scores in fp32, each within kNear of its value, and where two that stand next to each other
// in the order, or at the border of the groups, are nearer than that (one token in a thousand of 256 experts), the
// token is done again in 64 bits.  So neighbours 1e-7 apart come out as the definition says at the cost of fp32.
//
// Bound: the launch and a warp's chain of loads, scores and k rounds of a maximum; a round is one warp reduction of an
// order-preserving 32-bit key and one ballot.  Lane l has the NPL consecutive experts from l * NPL.
#include "ql_route.cuh"

namespace ql {
namespace {

constexpr int kWarps = 4;
// How far an fp32 score is from its value, at most, in parts of the largest score ("unit") and of the sums that it goes
// into: expf 2 units of 2^-24, the rounded exponent 0.4, the quotient 2, a sum of 1024 exponentials 37, the sums with
// biases and in groups 1 each.  2^-18 holds 64.
constexpr float kNear = 3.8146973e-6f;
constexpr float kTiny = 1e-30f;  // chosen scores whose sum is below this are taken in 64 bits, too
constexpr unsigned kAll = 0xffffffffu;

// Larger key, larger value; 0 for what cannot be chosen (-inf, NaN).
__device__ __forceinline__ uint32_t order(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// The definition in 64 bits, one token by one warp.  c, s: n_experts values each in shared memory.
__device__ __noinline__ void route_exact(const RouteArgs &a, int token, double *s, double *c) {
    const int lane = threadIdx.x % 32, E = a.n_experts, per = E / a.n_groups;
    const float *x = a.logits + (int64_t)token * a.logits_stride;
    double mx = -INFINITY, total = 0.0;
    if (!a.sigmoid) {
        for (int e = lane; e < E; e += 32)
            if (isfinite(x[e])) mx = fmax(mx, (double)x[e]);
        for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(kAll, mx, o));
        for (int e = lane; e < E; e += 32)
            if (isfinite(x[e])) total += exp((double)x[e] - mx);
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
    }
    for (int e = lane; e < E; e += 32) {
        const bool ok = isfinite(x[e]);
        double v = 0.0;
        if (ok) v = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[e])) : exp((double)x[e] - mx) / total;
        double w = v;
        if (a.bias != nullptr) w += (double)a.bias[e];
        s[e] = v;
        c[e] = ok && w > -INFINITY ? w : -INFINITY;  // (a bias of NaN or -inf: never chosen)
    }
    __syncwarp();
    unsigned open = kAll;
    if (a.n_groups > 1) {
        double g = -INFINITY;  // lane g: its group's score
        if (lane < a.n_groups) {
            double b0 = -INFINITY, b1 = -INFINITY;
            for (int e = lane * per; e < (lane + 1) * per; ++e) {
                const double v = c[e];
                if (v > b0)
                    b1 = b0, b0 = v;
                else if (v > b1)
                    b1 = v;
            }
            g = b0;
            if (a.group_best > 1 && b1 > -INFINITY) g += b1;
        }
        int better = 0;
        for (int o = 0; o < a.n_groups; ++o) {
            const double v = __shfl_sync(kAll, g, o);
            better += v > g || (v == g && o < lane);
        }
        open = __ballot_sync(kAll, g > -INFINITY && better < a.top_groups);
    }
    double sum = 0.0, mine = 0.0;
    int mine_e = -1;
    for (int r = 0; r < a.k; ++r) {
        double best = -INFINITY;
        int at = E;
        // without a bias the logits decide (two scores may round to the same 64 bits)
        for (int e = lane; e < E; e += 32) {
            if (!(c[e] > -INFINITY) || (a.n_groups > 1 && !(open >> (e / per) & 1u))) continue;
            const double v = a.bias != nullptr ? c[e] : (double)x[e];
            if (at == E || v > best) best = v, at = e;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(kAll, best, o);
            const int e = __shfl_xor_sync(kAll, at, o);
            if (e < E && (at == E || v > best || (v == best && e < at))) best = v, at = e;
        }
        if (at < E) {
            const double p = s[at];
            sum += p;
            if (lane == r) mine = p, mine_e = at;
            __syncwarp();
            if (at % 32 == lane) c[at] = -INFINITY;
        }
        __syncwarp();
    }
    if (lane < a.k) {
        const double w = a.renorm ? (sum > 0.0 ? mine / sum : 0.0) : mine;
        a.top_idx[(int64_t)token * a.k + lane] = mine_e;
        a.top_w[(int64_t)token * a.k + lane] = (float)(w * (double)a.scale);
    }
    __syncwarp();
}

template <int NPL>
__global__ void __launch_bounds__(32 * kWarps) route_kernel(const __grid_constant__ RouteArgs a) {
    extern __shared__ double smem[];  // per warp 2 n_experts; the fp32 pass takes n_experts floats of it
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, E = a.n_experts;
    const int token = blockIdx.x * kWarps + warp;
    if (token >= a.tokens) return;
    const float *x = a.logits + (int64_t)token * a.logits_stride;
    const int e0 = lane * NPL;
    float l[NPL], s[NPL];
    const bool vec = NPL % 4 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
#pragma unroll
    for (int i = 0; i < NPL; i += NPL % 4 == 0 ? 4 : 1) {
        if (NPL % 4 == 0 && vec && e0 + i + 3 < E) {
            const float4 w = *reinterpret_cast<const float4 *>(x + e0 + i);
            l[i] = w.x, l[(i + 1) % NPL] = w.y, l[(i + 2) % NPL] = w.z, l[(i + 3) % NPL] = w.w;
        } else {
#pragma unroll
            for (int j = 0; j < (NPL % 4 == 0 ? 4 : 1); ++j) l[(i + j) % NPL] = e0 + i + j < E ? x[e0 + i + j] : -INFINITY;
        }
    }
    float mx = -INFINITY, unit = 1.f;  // unit: no score is above it
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        if (!(fabsf(l[i]) < INFINITY)) l[i] = -INFINITY;
        mx = fmaxf(mx, l[i]);
    }
    if (!a.sigmoid) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
        if (!(mx > -INFINITY)) mx = 0.f;
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            s[i] = expf(l[i] - mx);
            total += s[i];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
        const float inv = total > 0.f ? __fdiv_rn(1.f, total) : 0.f;
#pragma unroll
        for (int i = 0; i < NPL; ++i) s[i] *= inv;
        unit = inv;
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const float z = expf(-fabsf(l[i]));  // in (0, 1]: no overflow on either side
            s[i] = __fdividef(l[i] < 0.f ? z : 1.f, 1.f + z);
        }
    }
    bool near = false;  // two scores too near for fp32
    uint32_t key[NPL];
    if (a.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) key[i] = e0 + i < E && l[i] > -INFINITY ? order(s[i] + a.bias[e0 + i]) : 0u;
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) key[i] = order(l[i]);
    }
    double *sw = smem + (size_t)warp * 2 * E;
    if (a.n_groups > 1) {
        const int per = E / a.n_groups;
        float *c = reinterpret_cast<float *>(sw);
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (e0 + i < E) c[e0 + i] = key[i] == 0u ? -INFINITY : a.bias != nullptr ? value(key[i]) : s[i];
        __syncwarp();
        // 32 / n_groups lanes (a power of two) look through each group
        const int share = 1 << (31 - __clz(32 / a.n_groups));
        const int g = lane / share, j = lane % share;
        float b0 = -INFINITY, b1 = -INFINITY;
        if (g < a.n_groups)
            for (int e = j; e < per; e += share) {
                const float v = c[g * per + e];
                b1 = fmaxf(b1, fminf(b0, v));
                b0 = fmaxf(b0, v);
            }
        for (int o = share / 2; o > 0; o /= 2) {
            const float v0 = __shfl_xor_sync(kAll, b0, o), v1 = __shfl_xor_sync(kAll, b1, o);
            b1 = fmaxf(fmaxf(b1, v1), fminf(b0, v0));
            b0 = fmaxf(b0, v0);
        }
        const bool two = a.group_best > 1 && b1 > -INFINITY;
        const float score = two ? b0 + b1 : b0;  // (the same in every lane of a group)
        const float size = fabsf(b0) + (two ? fabsf(b1) : 0.f) + unit;
        int better = 0;
        unsigned close = 0;  // groups whose scores are too near to this one's, bit o * share
        for (int o = 0; o < a.n_groups; ++o) {
            const float v = __shfl_sync(kAll, score, o * share), z = __shfl_sync(kAll, size, o * share);
            better += v > score || (v == score && o < g);
            if (fabsf(v - score) <= kNear * (size + z)) close |= 1u << (o * share);
        }
        const bool stays = g < a.n_groups && j == 0 && score > -INFINITY && better < a.top_groups;
        const unsigned open = __ballot_sync(kAll, stays);  // bit g * share
        near = __any_sync(kAll, j == 0 && g < a.n_groups && score > -INFINITY && ((stays ? ~open : open) & close) != 0);
        int gi = e0 / per, rest = e0 - gi * per;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            if (e0 + i < E && !(open >> (gi * share) & 1u)) key[i] = 0u;
            if (++rest == per) rest = 0, ++gi;
        }
        __syncwarp();
    }
    // k rounds (one more where the border could be near): the warp's largest key, its lowest lane, that lane's first
    uint32_t top = 0;
    int where = 0;
    auto lane_best = [&] {
        top = key[0], where = 0;
#pragma unroll
        for (int i = 1; i < NPL; ++i)
            if (key[i] > top) top = key[i], where = i;
    };
    lane_best();
    const int rounds = a.bias != nullptr ? a.k + 1 : a.k;
    float mine = 0.f, sum = 0.f, last = 0.f;
    int mine_e = -1;
    for (int r = 0; r < rounds; ++r) {
        const uint32_t best = __reduce_max_sync(kAll, top);
        if (best == 0u) break;
        const int owner = __ffs(__ballot_sync(kAll, top == best)) - 1;
        const float c = value(best);
        if (a.bias != nullptr) {
            if (r > 0 && last - c <= kNear * (fabsf(c) + fabsf(last) + unit)) near = true;
            last = c;
            if (r == a.k) break;
        }
        float p = 0.f;
        if (lane == owner) {
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                if (i == where) {
                    p = s[i];
                    key[i] = 0u;
                }
        }
        const int e = __shfl_sync(kAll, e0 + where, owner);
        p = __shfl_sync(kAll, p, owner);
        sum += p;
        if (lane == r) mine = p, mine_e = e;
        if (lane == owner) lane_best();
    }
    near = near || (a.renorm && !(sum >= kTiny));
    if (near) {
        route_exact(a, token, sw, sw + E);
        return;
    }
    if (lane < a.k) {
        const float w = a.renorm ? __fdiv_rn(mine, sum) : mine;
        a.top_idx[(int64_t)token * a.k + lane] = mine_e;
        a.top_w[(int64_t)token * a.k + lane] = w * a.scale;
    }
}

template <int NPL>
cudaError_t launch(const RouteArgs &a, cudaStream_t s) {
    const size_t smem = sizeof(double) * 2 * kWarps * (size_t)a.n_experts;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(route_kernel<NPL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    route_kernel<NPL><<<(a.tokens + kWarps - 1) / kWarps, 32 * kWarps, smem, s>>>(a);
    return cudaGetLastError();
}
}  // namespace

cudaError_t route_launch(const RouteArgs &a, int sms, cudaStream_t s) {
    (void)sms;
    const int need = (a.n_experts + 31) / 32;
    return need <= 2    ? launch<2>(a, s)
           : need <= 4  ? launch<4>(a, s)
           : need <= 8  ? launch<8>(a, s)
           : need <= 12 ? launch<12>(a, s)
           : need <= 16 ? launch<16>(a, s)
                        : launch<32>(a, s);
}

}  // namespace ql
