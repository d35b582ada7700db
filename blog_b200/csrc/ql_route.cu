// Choice of experts, a warp per token:
//   s_e = softmax over the experts' logits, or sigmoid of each;   c_e = s_e + bias_e
//   group g counts by the sum of its group_best largest c; the top_groups best groups stay
//   the k experts of largest c in them, the lowest id among equals, by descending c
//   w_e = s_e [/ sum of the chosen s] * scale
// Without a bias experts stand by their logits, which no rounding touches.  Otherwise the order is that of 64-bit scores:
// the kernel goes by scores in fp32, whose errors have a bound, and picks on past the k-th until the next one is clearly
// less.  Where two that stand next to each other in that order are nearer than the bound, the picked ones, one per lane, are
// ranked by their scores in 64 bits; where the border of the groups is in doubt, the groups are counted again in 64 bits.
// So neighbours 1e-7 apart come out as the definition says.  (Everything in 64 bits for such a token: one in 200 held
// 8192 tokens up to 23 us.)
//
// Bound: one token or few, the launch and a warp's chain of loads, scores and k rounds of a maximum (2.3 us for one token of
// 64 experts, 5.3 us for 64 of 256 in groups); thousands, issue slots: 8191 tokens of 384 experts by softmax 11.7 us at some
// 900 instructions a warp, 8192 of 256 by sigmoid in 8 groups 18.7 us at 1500 (58 and 65 % of the slots; HBM 10 and 4 %).
// So: a warp per token, everything in registers; a round is one warp reduction of the values as they are and one ballot.
// Lane l has the NPL consecutive experts from l * NPL.
#include "ql_route.cuh"

namespace ql {
namespace {

constexpr int kWarps = 4;
constexpr float kTiny = 1e-30f;  // chosen scores whose sum is below this are taken in 64 bits, too
constexpr unsigned kAll = 0xffffffffu;

// What is compared: fp32 values as they are, 64-bit ones as order-preserving words (a warp's maximum takes 32 bits at a time);
// the lowest of each for what cannot be chosen (-inf, NaN).
template <typename T>
struct Key;
template <>
struct Key<float> {
    using type = float;
    static constexpr float none = -INFINITY;
};
template <>
struct Key<double> {
    using type = uint64_t;
    static constexpr uint64_t none = 0;
};
__device__ __forceinline__ float order(float v) { return v > -INFINITY ? v : -INFINITY; }
__device__ __forceinline__ uint64_t order(double v) {
    if (!(v > -INFINITY)) return 0ull;
    const uint64_t u = (uint64_t)__double_as_longlong(v == 0.0 ? 0.0 : v);
    return (u >> 63) ? ~u : (u | 1ull << 63);
}
__device__ __forceinline__ float value(float k) { return k; }
__device__ __forceinline__ double value(uint64_t k) { return __longlong_as_double((long long)(k >> 63 ? k ^ (1ull << 63) : ~k)); }
__device__ __forceinline__ float warp_max(float k) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(k));
    return r;
}
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(k >> 32));
    return (uint64_t)hi << 32 | __reduce_max_sync(kAll, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
}
// For x <= 0.  The fast one, for the order: 2 + 1.2 |x| units in the last place, at most 4 of exp(0)'s.
__device__ __forceinline__ float exp_fast(float x) { return __expf(x); }
__device__ __forceinline__ double exp_fast(double x) { return exp(x); }
__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float quotient(float a, float b) { return __fdividef(a, b); }
__device__ __forceinline__ double quotient(double a, double b) { return a / b; }

// The score of a logit that may be chosen; mx and inv: the softmax's largest logit and the inverse of its sum.
template <bool SIGMOID, bool FAST, typename T>
__device__ __forceinline__ T score_of(float l, float mx, T inv) {
    if (!SIGMOID) {
        const T d = (T)l - (T)mx;
        return (FAST ? exp_fast(d) : exp_of(d)) * inv;
    }
    const T d = -fabs((T)l), z = FAST ? exp_fast(d) : exp_of(d);  // (in (0, 1]: no overflow on either side)
    return quotient(l < 0.f ? z : (T)1, (T)1 + z);
}

// Lanes that look through a group (a power of two).
__device__ __forceinline__ int group_share(const RouteArgs &a) { return 1 << (31 - __clz(32 / a.n_groups)); }

// The groups that stay, bit g * group_share, by the values in c (-inf: not to be chosen); near: in fp32 the border is in doubt.
template <typename T>
__device__ __forceinline__ unsigned groups_open(const RouteArgs &a, const T *c, T score_err, T sum_err, T unit, bool &near) {
    constexpr bool fast = sizeof(T) == 4;
    const int lane = threadIdx.x % 32, per = a.n_experts / a.n_groups, share = group_share(a);
    const int g = lane / share, j = lane % share;
    T b0 = -INFINITY, b1 = -INFINITY;
    if (g < a.n_groups)
#pragma unroll 4
        for (int e = j; e < per; e += share) {
            const T v = c[g * per + e];
            b1 = fmax(b1, fmin(b0, v));
            b0 = fmax(b0, v);
        }
#pragma unroll 1
    for (int o = share / 2; o > 0; o /= 2) {
        const T v0 = __shfl_xor_sync(kAll, b0, o), v1 = __shfl_xor_sync(kAll, b1, o);
        b1 = fmax(fmax(b1, v1), fmin(b0, v0));
        b0 = fmax(b0, v0);
    }
    const bool two = a.group_best > 1 && b1 > -INFINITY;
    const T score = two ? b0 + b1 : b0;  // (the same in every lane of a group)
    const T size = sum_err * (fabs(b0) + (two ? fabs(b1) : (T)0)) + 2 * score_err * unit;
    // Groups with an expert to choose.  (Not by the sum of two, which passes fp32's range where biases are of its lowest value.)
    const unsigned some = __ballot_sync(kAll, g < a.n_groups && j == 0 && b0 > -INFINITY);
    int better = 0;
    unsigned close = 0;  // groups whose scores are too near to this one's, or both beyond the range, bit o * share
    const int turns = (a.n_groups + share - 1) / share;  // a group's lanes look at the others in turn
#pragma unroll 1
    for (int n = 0; n < turns; ++n) {
        const int o = n * share + j, from = min(o, a.n_groups - 1) * share;
        const T v = __shfl_sync(kAll, score, from), z = fast ? __shfl_sync(kAll, size, from) : (T)0;
        if (o >= a.n_groups || !(some >> (o * share) & 1u)) continue;
        better += v > score || (v == score && o < g);
        if (fast && !(fabs(v - score) > size + z)) close |= 1u << (o * share);
    }
#pragma unroll 1
    for (int o = share / 2; o > 0; o /= 2) {
        better += __shfl_xor_sync(kAll, better, o);
        if (fast) close |= __shfl_xor_sync(kAll, close, o);
    }
    const bool stays = (some >> lane & 1u) && better < a.top_groups;
    const unsigned open = __ballot_sync(kAll, stays);
    if (fast) near = __any_sync(kAll, (some >> lane & 1u) && ((stays ? ~open : open) & close) != 0);
    return open;
}

// 64 bits: the inverse of the softmax's sum, and the groups that stay.
template <bool SIGMOID>
__device__ __noinline__ double exact_inverse(const RouteArgs &a, int token, float mx) {
    if (SIGMOID) return 1.0;
    const float *x = a.logits + (int64_t)token * a.logits_stride;
    double total = 0.0;
#pragma unroll 2
    for (int e = threadIdx.x % 32; e < a.n_experts; e += 32)
        if (fabsf(x[e]) < INFINITY) total += exp((double)x[e] - (double)mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
    return total > 0.0 ? 1.0 / total : 0.0;
}
template <bool SIGMOID>
__device__ __noinline__ unsigned groups_exactly(const RouteArgs &a, int token, float mx, double *c) {
    const float *x = a.logits + (int64_t)token * a.logits_stride;
    const double inv = exact_inverse<SIGMOID>(a, token, mx);
    __syncwarp();
#pragma unroll 2
    for (int e = threadIdx.x % 32; e < a.n_experts; e += 32) {
        double v = -INFINITY;
        if (fabsf(x[e]) < INFINITY) v = score_of<SIGMOID, false>(x[e], mx, inv) + (a.bias != nullptr ? (double)a.bias[e] : 0.0);
        c[e] = v > -INFINITY ? v : -INFINITY;
    }
    __syncwarp();
    bool near;
    return groups_open(a, c, 0.0, 0.0, 0.0, near);
}
// Of m candidates, lane i's expert e, the rank of each by its score in 64 bits (equal ones by id).
template <bool SIGMOID>
__device__ __noinline__ int rank_exactly(const RouteArgs &a, int token, float mx, int e, int m) {
    const double inv = exact_inverse<SIGMOID>(a, token, mx);
    double v = -INFINITY;
    if (e >= 0) v = score_of<SIGMOID, false>(a.logits[(int64_t)token * a.logits_stride + e], mx, inv) + (double)a.bias[e];
    int rank = 0;
#pragma unroll 1
    for (int i = 0; i < m; ++i) {
        const double w = __shfl_sync(kAll, v, i);
        const int f = __shfl_sync(kAll, e, i);
        rank += w > v || (w == v && f < e);
    }
    return rank;
}

// One token by one warp, in fp32 or in 64 bits.  c: n_experts values in shared memory where there are groups.  false: not
// to be decided in fp32, nothing is written.
template <typename T, int NPL, bool SIGMOID>
__device__ __forceinline__ bool choose(const RouteArgs &a, int token, T *c) {
    using K = typename Key<T>::type;
    constexpr bool fast = sizeof(T) == 4;
    constexpr K none = Key<T>::none;
    const int lane = threadIdx.x % 32, E = a.n_experts, e0 = lane * NPL;
    const float *x = a.logits + (int64_t)token * a.logits_stride;
    K key[NPL];
    float mx = 0.f;
    T inv = 1, unit = 1;  // unit: no score is above it
    {
        float l[NPL], bias[NPL];
        if (a.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) bias[i] = e0 + i < E ? a.bias[e0 + i] : 0.f;
        }
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
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (!(fabsf(l[i]) < INFINITY)) l[i] = -INFINITY;
        const bool all = a.bias != nullptr || a.n_groups > 1;  // every expert's score is needed, not the chosen ones' alone
        if (!SIGMOID) {
            mx = l[0];
#pragma unroll
            for (int i = 1; i < NPL; ++i) mx = fmaxf(mx, l[i]);
            mx = warp_max(mx);
            if (!(mx > -INFINITY)) mx = 0.f;
            if (all || !a.renorm) {
                T total = 0;
#pragma unroll
                for (int i = 0; i < NPL; ++i) total += exp_fast((T)l[i] - (T)mx);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
                inv = total > 0 ? (T)1 / total : (T)0;
                unit = inv;
            }
        }
        if (all) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const bool there = e0 + i < E && l[i] > -INFINITY;
                const T s = score_of<SIGMOID, true>(l[i], mx, inv);
                const T v = a.bias != nullptr && there ? s + (T)bias[i] : s;
                key[i] = there ? a.bias != nullptr ? order(v) : order((T)l[i]) : none;
                if (a.n_groups > 1 && e0 + i < E) c[e0 + i] = key[i] != none ? v : (T)-INFINITY;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NPL; ++i) key[i] = order((T)l[i]);
        }
    }
    // How far an fp32 score is from its value, in units of 2^-24 of "unit": the exponential 4, its rounded argument 0.4,
    // 1 + z or the product 1, the quotient 4, and in a softmax the sum's NPL + 5 additions, its terms and inverse.  Sums of
    // scores are rounded once more, 2^-24 of themselves.
    const T score_err = (T)((SIGMOID ? 12 : NPL + 16) * 5.9604645e-8), sum_err = (T)1.2e-7;
    if (a.n_groups > 1) {
        const int per = E / a.n_groups, share = group_share(a);
        __syncwarp();
        bool near = false;
        unsigned open = groups_open(a, c, score_err, sum_err, unit, near);  // bit g * share
        if (fast && near) open = groups_exactly<SIGMOID>(a, token, mx, reinterpret_cast<double *>(c));
        int gi = e0 / per, rest = e0 - gi * per;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            if (e0 + i < E && !(open >> (gi * share) & 1u)) key[i] = none;
            if (++rest == per) rest = 0, ++gi;
        }
    }
    // k rounds (more where the border is in doubt): the warp's largest key, its lowest lane, that lane's first
    K top = none;
    int where = 0;
    auto lane_best = [&] {
        top = key[0], where = 0;
#pragma unroll
        for (int i = 1; i < NPL; ++i)
            if (key[i] > top) top = key[i], where = i;
    };
    lane_best();
    const bool check = fast && a.bias != nullptr;
    T last = 0;
    int mine_e = -1, n = 0;
    bool near = false;
#pragma unroll 1
    for (;; ++n) {
        if (!check && n == a.k) break;
        const K best = warp_max(top);
        if (best == none) break;
        if (check) {
            const T v = value(best);
            const bool close = n > 0 && last - v <= sum_err * (fabs(v) + fabs(last)) + 2 * score_err * unit;
            if (n >= a.k && !close) break;
            if (n == 32) return false;  // (more than a lane each)
            near |= close;
            last = v;
        }
        const int owner = __ffs(__ballot_sync(kAll, top == best)) - 1;
        const int e = __shfl_sync(kAll, e0 + where, owner);
        if (lane == n) mine_e = e;
        if (lane == owner) {
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                if (i == where) key[i] = none;
            lane_best();
        }
    }
    if (check && near) {  // lane i's candidate to the lane of its rank
        const int rank = rank_exactly<SIGMOID>(a, token, mx, mine_e, n);
        int e = -1;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int to = __shfl_sync(kAll, rank, i), f = __shfl_sync(kAll, mine_e, i);
            if (to == lane) e = f;
        }
        mine_e = e;
    }
    if (lane >= a.k) mine_e = -1;
    // lane r has the r-th
    const T mine = mine_e >= 0 ? score_of<SIGMOID, false>(x[mine_e], mx, inv) : (T)0;
    T w = mine;
    if (a.renorm) {
        T sum = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
        if (fast && !(sum >= (T)kTiny)) return false;
        w = sum > 0 ? mine / sum : (T)0;
    }
    if (lane < a.k) {
        a.top_idx[(int64_t)token * a.k + lane] = mine_e;
        a.top_w[(int64_t)token * a.k + lane] = (float)(w * (T)a.scale);
    }
    return true;
}

template <int NPL, bool SIGMOID>
__device__ __noinline__ void choose_exactly(const RouteArgs &a, int token, double *c) {
    choose<double, NPL, SIGMOID>(a, token, c);
}

// The registers of 12, 8 or 4 CTAs: 48, 32 or 16 warps an SM.  (8192 tokens are 55 warps an SM: 1.15 rounds of them with 8
// experts a lane, 1.7 with 12.  The seldom 64-bit form may spill.)
template <int NPL, bool SIGMOID>
__global__ void __launch_bounds__(32 * kWarps, NPL <= 8 ? 12 : NPL <= 16 ? 8 : 4) route_kernel(const __grid_constant__ RouteArgs a) {
    extern __shared__ double smem[];  // n_experts per warp where there are groups
    const int warp = threadIdx.x / 32, token = blockIdx.x * kWarps + warp;
    if (token >= a.tokens) return;
    double *c = smem + (size_t)warp * a.n_experts;
    if (!choose<float, NPL, SIGMOID>(a, token, reinterpret_cast<float *>(c))) choose_exactly<NPL, SIGMOID>(a, token, c);
}

template <int NPL>
cudaError_t launch(const RouteArgs &a, cudaStream_t s) {
    const size_t smem = a.n_groups > 1 ? sizeof(double) * kWarps * (size_t)a.n_experts : 0;
    const unsigned grid = (unsigned)((a.tokens - 1) / kWarps + 1);
    if (a.sigmoid)
        route_kernel<NPL, true><<<grid, 32 * kWarps, smem, s>>>(a);
    else
        route_kernel<NPL, false><<<grid, 32 * kWarps, smem, s>>>(a);
    return cudaGetLastError();
}
static_assert(sizeof(double) * kWarps * kRouteMaxExperts <= 48 * 1024, "shared memory without asking for more");
}  // namespace

cudaError_t route_launch(const RouteArgs &a, cudaStream_t s) {
    const int need = (a.n_experts + 31) / 32;
    return need <= 2    ? launch<2>(a, s)
           : need <= 4  ? launch<4>(a, s)
           : need <= 8  ? launch<8>(a, s)
           : need <= 12 ? launch<12>(a, s)
           : need <= 16 ? launch<16>(a, s)
                        : launch<32>(a, s);
}

}  // namespace ql
