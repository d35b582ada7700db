// Attention over the 8-bit KV cache: what its two kernels (ql_kv8_attn.cu, ql_kv8_prompt.cu) share of the arithmetic of
// codes, f16 limbs and weights.
#pragma once
#include <cuda_fp16.h>

#include "ql_kv8.cuh"

namespace ql {

// m and h are whole numbers, at or above the maxima they stand for when they are set, and kept until a value
// passes them by kHeadroom (so the sums are seldom rescaled).  Weights are scaled by 2^kWBits: at most
// 2^(7 + 8) in f16, and limbs down to 2^-24 / 2^8 of the row's largest.
inline constexpr float kHeadroom = 7.0f, kWBits = 8.0f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two codes (bytes sel of w) as f16: 0x6400 | u is 1024 + u, minus 1152 is exact.
__device__ __forceinline__ uint32_t codes2(uint32_t w, uint32_t sel) {
    uint32_t r = __byte_perm(w, 0x64646464u, sel);
    const uint32_t bias = 0x64806480u;  // 1152, 1152
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(bias));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
// x = hi + lo in two f16 limbs, two values packed.
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    hi = pack_f16(x0, x1);
    const float2 h = unpack_f16(hi);
    lo = pack_f16(x0 - h.x, x1 - h.y);
}
// 2^k with amax * 2^k in [2^10, 2^11) (within the normal range), and 2^-k.
__device__ __forceinline__ float limb_scale(float amax, float &inv) {
    const int e = (int)(__float_as_uint(amax) >> 23) & 0xFF;
    const int f = min(max(264 - e, 1), 253);
    inv = __uint_as_float((uint32_t)(254 - f) << 23);
    return __uint_as_float((uint32_t)f << 23);
}

// 2^(kWBits - h), 0 while nothing but zeros has been met (h = -inf).
__device__ __forceinline__ float weight_unit(float h) { return h == -INFINITY ? 0.f : ex2(kWBits - h); }
// Below this h the weights' factor sv w leaves the range, and 2^(s - m) with it, where the weights themselves
// do not (the row's heaviest keys have values of zero): they are computed from s - m - h then.
inline constexpr float kDeep = -60.0f;
// Beyond this |m| a score is rounded before m is taken off it: m is a rounded score then, and what one rounding
// of the difference would keep is larger than the range of the weights.
inline constexpr float kHuge = 1e6f;

}  // namespace ql
