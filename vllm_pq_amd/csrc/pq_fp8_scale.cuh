// The scale of a group of values and their quotients by it, shared by everything that writes e4m3.
#pragma once
#include <hip/hip_runtime.h>

#include "pq_common.cuh"
#include "pq_kernels.h"

namespace pq {

constexpr uint32_t AMAX_MIN_BITS = (127 - 96) << 23;   // 2^-96

// What divides a group: its scale s, an approximate reciprocal of it, and what the quotient is corrected with.
struct GroupScale {
    float s, r, c;
};
__device__ __forceinline__ GroupScale scale_of(float amax) {      // no floor: amax far enough from 0 that amax / 448 is normal
    GroupScale g;
    g.s = amax / FP8_MAX;
    g.r = __builtin_amdgcn_rcpf(g.s);         // within one unit of the last place
    g.c = __builtin_isinf(g.s) ? 0.f : g.s;   // an infinite scale: v * r stands as it is (0, or NaN for the infinity itself)
    return g;
}
__device__ __forceinline__ GroupScale group_scale(uint32_t amax_bits) {
    return scale_of(__uint_as_float(amax_bits > AMAX_MIN_BITS ? amax_bits : AMAX_MIN_BITS));
}
// v / s in fp32: the product with the reciprocal is within 2^-22 of the quotient, and one Newton step on its exact residual
// takes that to 2^-44, so the rounded result is the correctly rounded quotient unless that lies within 2^-44 of half way
// between two numbers.  A third of a division's instructions, which is what bounds these kernels next to memory; the bare
// product would move values that lie on a tie between two e4m3 numbers, and with act-dtype inputs many do.
__device__ __forceinline__ float div_group(float v, const GroupScale &g) {
    const float q = v * g.r;
    return __builtin_fmaf(__builtin_fmaf(-q, g.c, v), g.r, q);
}
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// four values -> four e4m3 bytes
__device__ __forceinline__ uint32_t pack4(const float *v, const GroupScale &g) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(div_group(v[0], g), div_group(v[1], g), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(div_group(v[2], g), div_group(v[3], g), p, true);
}
}  // namespace pq
