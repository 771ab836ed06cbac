// The matrix instruction of the e4m3 products, shared by their kernels.
#pragma once
#include <hip/hip_runtime.h>

#include "pq_common.cuh"

namespace pq {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Inner sum over one block of 128 features for 16 weight rows x 16 tokens, e4m3 x e4m3, from zero and without scales.
// Lane l brings 32 features of weight row l % 16 and the same 32 of token l % 16, and gets rows 4 (l / 16) .. + 3 of token
// l % 16.  The sum has fp32 precision between groups of 8 products; inside a group each product is cut to a multiple of 2^-13
// of the power of two that the largest one's exponents give (test_gpu_matrix_instruction), on average about 2^-19 of
// the sum of magnitudes over a block -- two decimal digits below an act dtype's rounding, and four times the rate of the
// products in the act dtype.
__device__ __forceinline__ f32x4 mfma_block(const i32x8 &w, const i32x8 &x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8 join(const u32x4 &lo, const u32x4 &hi) {
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

}  // namespace pq
