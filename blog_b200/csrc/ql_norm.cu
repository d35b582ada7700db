// The residual's addition, the RMS norm and its 8-bit rows, one pass over a row:
//   v = x + residual   (one fp32 addition, rounded to the type: what is stored is what is normed)
//   y = v / sqrt(mean(v^2) + eps) * gamma
//   per 32 of y (before y is rounded to its type): d = max|y| / 127, code = rint(y / d), and the block's sum: the bytes
//   of the Q8_1 quantiser (ql_q81.cu) for that y, in either of its layouts, with the same arithmetic and the same
//   order of the raw sum.
//
// Bound: HBM in f32, every value read once and written once; a CTA holds its row in registers between the two uses.  A
// thread has groups of 4 consecutive values (16 bytes in f32), so the 8 threads of an 8-bit block are neighbours and
// its maximum and sums take three shuffles.  Squares are summed in fp32, a tree over the threads.
//
// Measured, residual and Q8_1 rows: 4096 rows of 8192 f32 with sum and y 91.7 us (6.26 TB/s, 0.96 of a plain copy); 777 rows
// of 2048, no y, 7.8 us; 64 rows of 8192 bf16 4.2 us and one row of 3584 2.8 us: a launch, a load and two reductions.  5000
// rows of 8192 bf16 93 us (0.61 of a copy): 81 % of the issue slots, since a value takes as many instructions as in f32.
#include <cuda_bf16.h>

#include "ql_norm.cuh"

namespace ql {
namespace {

template <bool BF16>
struct Io;
template <>
struct Io<false> {
    using T = float;
    static __device__ __forceinline__ float4 load(const float *p) { return *reinterpret_cast<const float4 *>(p); }
    static __device__ __forceinline__ float one(const float *p) { return *p; }
    static __device__ __forceinline__ float rounded(float v) { return v; }
    static __device__ __forceinline__ void store(float *p, const float (&v)[4]) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
    static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
};
template <>
struct Io<true> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float4 load(const T *p) {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xFFFF0000u));
    }
    static __device__ __forceinline__ float one(const T *p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ float rounded(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
    static __device__ __forceinline__ void store(T *p, const float (&v)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    static __device__ __forceinline__ void put(T *p, float v) { *p = __float2bfloat16_rn(v); }
};

// NV: groups of 4 values per thread, blockDim.x apart, MAXT threads at most.  VEC: every row of every operand starts on
// a group and holds whole groups.
template <bool BF16, int NV, int MAXT, bool VEC>
__global__ void __launch_bounds__(MAXT) add_norm_kernel(const __grid_constant__ AddNormArgs a) {
    using D = Io<BF16>;
    using T = typename D::T;
    const int row = blockIdx.x, tid = threadIdx.x, nt = blockDim.x, H = a.hidden;
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.x_stride;
    const T *res = a.residual ? static_cast<const T *>(a.residual) + (int64_t)row * a.residual_stride : nullptr;
    auto at = [&](int i) { return (i * nt + tid) * 4; };
    float v[NV][4], g[NV][4];
    auto fetch = [&](const T *p, int i, float (&o)[4]) {
        if (VEC) {
            const float4 w = at(i) < H ? D::load(p + at(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
            o[0] = w.x, o[1] = w.y, o[2] = w.z, o[3] = w.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = at(i) + e < H ? D::one(p + at(i) + e) : 0.f;
        }
    };
    auto scales = [&](int i) {
        if (VEC && a.gamma != nullptr) {
            const float4 w = at(i) < H ? *reinterpret_cast<const float4 *>(a.gamma + at(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
            g[i][0] = w.x, g[i][1] = w.y, g[i][2] = w.z, g[i][3] = w.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) g[i][e] = a.gamma != nullptr && at(i) + e < H ? a.gamma[at(i) + e] : 1.f;
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) fetch(x, i, v[i]);
    if (res != nullptr) {
        float r[NV][4];
#pragma unroll
        for (int i = 0; i < NV; ++i) fetch(res, i, r[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = D::rounded(__fadd_rn(v[i][e], r[i][e]));
    }
    if (NV <= 4) {  // under way while the squares are summed
#pragma unroll
        for (int i = 0; i < NV; ++i) scales(i);
    }
    auto write = [&](T *p, int i, const float (&o)[4]) {
        if (VEC) {
            if (at(i) < H) D::store(p + at(i), o);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at(i) + e < H) D::put(p + at(i) + e, o[e]);
        }
    };
    if (a.sum != nullptr) {
        T *sum = static_cast<T *>(a.sum) + (int64_t)row * a.sum_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) write(sum, i, v[i]);
    }
    if (a.y == nullptr && a.xq == nullptr) return;
    auto squares = [&] {  // the row's sum of squares
        __shared__ float part[32];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            ss += __fmaf_rn(v[i][0], v[i][0], __fmul_rn(v[i][1], v[i][1])) + __fmaf_rn(v[i][2], v[i][2], __fmul_rn(v[i][3], v[i][3]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (nt > 32) {
            if (tid % 32 == 0) part[tid / 32] = ss;
            __syncthreads();
            ss = tid % 32 < nt / 32 ? part[tid % 32] : 0.f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        return ss;
    };
    float ss = squares(), eps = a.eps;
    // squares outside fp32's range: the row once more times 2^-96 or 2^96 (beside an eps of 2^-66 or more the small ones
    // do not count); the norm takes the factor out again
    const bool large = ss == INFINITY, small = ss < 0x1p-100f && eps < 0x1p-66f;
    if (large || small) {
        const float f = large ? 0x1p-96f : 0x1p96f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] *= f;
        eps = eps * f * f;
        __syncthreads();
        ss = squares();
    }
    const float inv = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)H), eps));
    const int nb = (H + 31) / 32, written = a.mmq ? (nb + 3) / 4 * 4 : nb;  // (the packed layout has whole groups of four)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (NV > 4) scales(i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = __fmul_rn(__fmul_rn(v[i][e], inv), g[i][e]);
        if (a.y != nullptr) write(static_cast<T *>(a.y) + (int64_t)row * a.y_stride, i, v[i]);
        if (a.xq == nullptr) continue;
        const int b = at(i) / 32, lane8 = tid % 8;
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(v[i][e]));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float d = amax > 0.f ? __fdiv_rn(amax, 127.f) : 0.f;
        const float id = d > 0.f ? __fdiv_rn(1.f, d) : 0.f;
        uint32_t code = 0;
        int qs = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int q = max(-127, min(127, __float2int_rn(__fmul_rn(v[i][e], id))));
            qs += q;
            code |= (uint32_t)(q & 0xFF) << (8 * e);
        }
        float total;
        if (a.raw_sum) {  // values 16, 8, 4, 2 and 1 apart, in this order (the quantiser's tree)
            float t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = v[i][e];
#pragma unroll
            for (int o = 4; o > 0; o >>= 1)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = __fadd_rn(t[e], __shfl_xor_sync(0xffffffffu, t[e], o));
            total = __fadd_rn(__fadd_rn(t[0], t[2]), __fadd_rn(t[1], t[3]));
        } else {
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) qs += __shfl_xor_sync(0xffffffffu, qs, o);
            total = __fmul_rn(d, (float)qs);
        }
        if (b >= nb) total = 0.f;  // (behind the row: zeros beside a row of NaN too)
        if (b < written) {
            uint8_t *ds, *qd;
            if (a.mmq) {
                uint8_t *grp = a.xq + ((int64_t)(b / 4) * a.rows + row) * 144;
                ds = grp + 4 * (b % 4);
                qd = grp + 16 + 32 * (b % 4);
            } else {
                ds = a.xq + ((int64_t)row * nb + b) * 36;
                qd = ds + 4;
            }
            reinterpret_cast<uint32_t *>(qd)[lane8] = code;
            if (lane8 == 0)
                *reinterpret_cast<uint32_t *>(ds) = (uint32_t)__half_as_ushort(__float2half(d)) |
                                                    (uint32_t)__half_as_ushort(__float2half(total)) << 16;
        }
    }
}

template <bool BF16, int NV, int MAXT>
cudaError_t launch(const AddNormArgs &a, int threads, cudaStream_t s) {
    constexpr int el = BF16 ? 2 : 4;
    auto ok = [](const void *p, int64_t stride) {
        return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (4 * el) == 0 && stride % 4 == 0);
    };
    if (a.hidden % 4 == 0 && ok(a.x, a.x_stride) && ok(a.residual, a.residual_stride) && ok(a.sum, a.sum_stride) &&
        ok(a.y, a.y_stride) && reinterpret_cast<uintptr_t>(a.gamma) % 16 == 0)
        add_norm_kernel<BF16, NV, MAXT, true><<<a.rows, threads, 0, s>>>(a);
    else
        add_norm_kernel<BF16, NV, MAXT, false><<<a.rows, threads, 0, s>>>(a);
    return cudaGetLastError();
}
template <bool BF16>
cudaError_t pick(const AddNormArgs &a, int sms, cudaStream_t s) {
    const int groups = a.mmq ? (a.hidden + 127) / 128 * 32 : (a.hidden + 31) / 32 * 8;  // of 4 values, whole 8-bit blocks, or four
    auto threads = [&](int nv) { return ((groups + nv - 1) / nv + 31) / 32 * 32; };
    // One group per thread where rows are few (latency) or narrow; else two, so that loads in flight do not need many threads
    // (one, two, four of them: 5000 rows of 3584 f32 59, 49, 51 us, 300 rows of 896 2.6, 3.0, 4.0 us; eight are slower
    // everywhere), and more for rows that need them.
    const bool few = a.rows <= 2 * sms || (a.rows <= 8 * sms && threads(1) <= 256);
    if (few && threads(1) <= 1024) return launch<BF16, 1, 1024>(a, threads(1), s);
    if (threads(2) <= 1024) return launch<BF16, 2, 1024>(a, threads(2), s);
    if (threads(4) <= 1024) return launch<BF16, 4, 1024>(a, threads(4), s);
    return launch<BF16, 8, 1024>(a, threads(8), s);
}
}  // namespace

cudaError_t add_norm_launch(const AddNormArgs &a, bool bf16, int sms, cudaStream_t s) {
    return bf16 ? pick<true>(a, sms, s) : pick<false>(a, sms, s);
}

}  // namespace ql
