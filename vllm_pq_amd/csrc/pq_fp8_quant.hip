// Activations in 8-bit floating point with one scale per token and group of 128 features, written by the step that
// produces them:
//   fp8_group_quant             v = x
//   silu_and_mul_fp8            v[t][j] = silu(x[t][j]) * x[t][I + j]
//   (fused_add_)rms_norm_fp8    z = x (+ residual, which becomes round(z)); v = z * rsqrt(mean(z^2) + eps) * w
// and for each of them, with b = j / 128,
//   s[t][b] = max(max over the group of |v|, 2^-96) / 448,     q[t][j] = e4m3(v[t][j] / s[t][b])       (nearest even).
// 448 is the largest finite e4m3 value, so nothing overflows; the floor keeps a group of zeros at q = 0 with a finite
// scale.  v stays in fp32 up to the one rounding to e4m3: the act-dtype roundings of the separate operators (silu, product,
// norm) would only add error that the 8-bit value does not need.  The maximum is taken over the absolute values' bits as
// unsigned integers: the same order for numbers, and an infinity or NaN in a group ends up in its scale, so that the product
// that reads it gives NaN and not a plausible number.
//
// All are bound by HBM (2 bytes in, 1 out per value) or, for a few tokens, by the launch.  One thread owns 8 consecutive
// values (one 16-byte load), 16 neighbouring lanes a group: its maximum is four lane exchanges, nothing passes through LDS.
#include <hip/hip_runtime.h>

#include "pq_common.cuh"
#include "pq_fp8_scale.cuh"
#include "pq_kernels.h"

namespace pq {

constexpr int QT = 256;                  // threads per block of the quantising kernels without a norm
constexpr int QV = FP8_GROUP / 8;        // threads per group

// maximum over the 16 lanes of a group
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
#pragma unroll
    for (int off = 1; off < QV; off <<= 1) m = umax(m, (uint32_t)__shfl_xor((int)m, off, 64));
    return m;
}

// silu(g) * u in fp32
__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

template <typename AT>
__device__ __forceinline__ void unpack8(const u32x4 &a, float *f) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[2 * w] = Act<AT>::to_f32((uint16_t)a[w]);
        f[2 * w + 1] = Act<AT>::to_f32((uint16_t)(a[w] >> 16));
    }
}

// ---- without a norm: groups are independent ------------------------------------------------------------
// 16-byte aligned rows, H a multiple of 8.  A block takes 2048 features of R consecutive rows.
template <typename AT, bool SILU, int R>
__global__ __launch_bounds__(QT) void quant_vec_kernel(QuantArgs a) {
    const int v = blockIdx.x * QT + threadIdx.x, H = a.H;
    const int64_t t0 = (int64_t)blockIdx.y * R;
    const bool in = v * 8 < H;
    const uint16_t *x = static_cast<const uint16_t *>(a.x) + (in ? v * 8 : 0);
    uint8_t *q = static_cast<uint8_t *>(a.q) + v * 8;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t t = t0 + i;
        if (t >= a.T) break;
        float f[8] = {};
        if (in) {
            const uint16_t *row = x + t * a.x_stride;
            unpack8<AT>(__builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row)), f);
            if constexpr (SILU) {
                float u[8];
                unpack8<AT>(__builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + H)), u);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = silu_mul(f[j], u[j]);
            }
        }
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = umax(m, abs_bits(f[j]));
        const GroupScale g = group_scale(group_max(m));
        if (in) {
            *reinterpret_cast<u32x2 *>(q + t * a.q_stride) = u32x2{pack4(f, g), pack4(f + 4, g)};
            if (threadIdx.x % QV == 0) a.scales[(int64_t)(v / QV) * a.scale_stride + t] = g.s;
        }
    }
}

// any H, any alignment: one wave per token and group, two values per lane
template <typename AT, bool SILU>
__global__ __launch_bounds__(QT) void quant_scalar_kernel(QuantArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, H = a.H;
    const int groups = (H + FP8_GROUP - 1) / FP8_GROUP;
    const int64_t total = (int64_t)a.T * groups;
    for (int64_t i = (int64_t)blockIdx.x * (QT / 64) + wave; i < total; i += (int64_t)gridDim.x * (QT / 64)) {
        const int64_t t = i / groups;
        const int b = (int)(i % groups);
        const uint16_t *row = static_cast<const uint16_t *>(a.x) + t * a.x_stride;
        float f[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = b * FP8_GROUP + h * 64 + lane;
            if (j < H) {
                f[h] = Act<AT>::to_f32(row[j]);
                if constexpr (SILU) f[h] = silu_mul(f[h], Act<AT>::to_f32(row[H + j]));
            }
        }
        uint32_t m = umax(abs_bits(f[0]), abs_bits(f[1]));
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) m = umax(m, (uint32_t)__shfl_xor((int)m, off, 64));
        const GroupScale g = group_scale(m);
        uint8_t *qr = static_cast<uint8_t *>(a.q) + t * a.q_stride;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = b * FP8_GROUP + h * 64 + lane;
            if (j < H) qr[j] = pack1(f[h], g);
        }
        if (lane == 0) a.scales[(int64_t)b * a.scale_stride + t] = g.s;
    }
}

// ---- with a norm -----------------------------------------------------------------------------------------
// One block of THREADS per token row; the row stays in registers between the sum of squares and the scaling, as in
// rms_norm_kernel.  ADD: z = x + residual, the residual becomes the rounded sum (the norm uses the unrounded one).
template <typename AT, int THREADS, int NV, bool ADD>
__global__ __launch_bounds__(THREADS) void norm_quant_kernel(QuantArgs a) {
    __shared__ float s_part[THREADS / 64];
    const int64_t t = blockIdx.x;
    const int nvec = a.H / 8;
    const uint16_t *xr = static_cast<const uint16_t *>(a.x) + t * a.x_stride;
    uint16_t *rr = ADD ? static_cast<uint16_t *>(a.residual) + t * a.res_stride : nullptr;
    float z[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = i * THREADS + threadIdx.x;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[i][j] = 0.f;
        if (v < nvec) {
            unpack8<AT>(__builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(xr + v * 8)), z[i]);
            if constexpr (ADD) {
                float r[8];
                unpack8<AT>(*reinterpret_cast<const u32x4 *>(rr + v * 8), r);
                u32x4 o;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    z[i][2 * w] += r[2 * w];
                    z[i][2 * w + 1] += r[2 * w + 1];
                    o[w] = Act<AT>::pack2(z[i][2 * w], z[i][2 * w + 1]);
                }
                *reinterpret_cast<u32x4 *>(rr + v * 8) = o;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(z[i][j], z[i][j], ss);
        }
    }
    const float rs = rsqrtf(block_sum<THREADS>(ss, s_part) / (float)a.H + a.eps);
    uint8_t *qr = static_cast<uint8_t *>(a.q) + t * a.q_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = i * THREADS + threadIdx.x;
        uint32_t m = 0;
        if (v < nvec) {
            float w[8];
            unpack8<AT>(*reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.weight) + v * 8), w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z[i][j] = z[i][j] * rs * w[j];
                m = umax(m, abs_bits(z[i][j]));
            }
        }
        const GroupScale g = group_scale(group_max(m));
        if (v < nvec) {
            *reinterpret_cast<u32x2 *>(qr + v * 8) = u32x2{pack4(z[i], g), pack4(z[i] + 4, g)};
            if (threadIdx.x % QV == 0) a.scales[(int64_t)(v / QV) * a.scale_stride + t] = g.s;
        }
    }
}

// any H, any alignment: the fp32 row in LDS, then one wave per group
template <typename AT, bool ADD>
__global__ __launch_bounds__(QT) void norm_quant_scalar_kernel(QuantArgs a) {
    __shared__ float s_part[QT / 64];
    extern __shared__ float s_row[];   // H floats
    const int64_t t = blockIdx.x;
    const int H = a.H, lane = threadIdx.x & 63;
    const uint16_t *xr = static_cast<const uint16_t *>(a.x) + t * a.x_stride;
    uint16_t *rr = ADD ? static_cast<uint16_t *>(a.residual) + t * a.res_stride : nullptr;
    const uint16_t *w = static_cast<const uint16_t *>(a.weight);
    float ss = 0.f;
    for (int j = threadIdx.x; j < H; j += QT) {
        float f = Act<AT>::to_f32(xr[j]);
        if constexpr (ADD) {
            f += Act<AT>::to_f32(rr[j]);
            rr[j] = Act<AT>::from_f32(f);
        }
        s_row[j] = f;
        ss = __builtin_fmaf(f, f, ss);
    }
    const float rs = rsqrtf(block_sum<QT>(ss, s_part) / (float)H + a.eps);   // (its barrier also orders s_row)
    uint8_t *qr = static_cast<uint8_t *>(a.q) + t * a.q_stride;
    const int groups = (H + FP8_GROUP - 1) / FP8_GROUP;
    for (int b = threadIdx.x >> 6; b < groups; b += QT / 64) {
        const int j0 = b * FP8_GROUP + lane, j1 = j0 + 64;
        const float f0 = j0 < H ? s_row[j0] * rs * Act<AT>::to_f32(w[j0]) : 0.f;
        const float f1 = j1 < H ? s_row[j1] * rs * Act<AT>::to_f32(w[j1]) : 0.f;
        uint32_t m = umax(abs_bits(f0), abs_bits(f1));
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) m = umax(m, (uint32_t)__shfl_xor((int)m, off, 64));
        const GroupScale g = group_scale(m);
        if (j0 < H) qr[j0] = pack1(f0, g);
        if (j1 < H) qr[j1] = pack1(f1, g);
        if (lane == 0) a.scales[(int64_t)b * a.scale_stride + t] = g.s;
    }
}

// ---- launches ----------------------------------------------------------------------------------------------
static bool aligned(const void *p, uintptr_t n) { return !(reinterpret_cast<uintptr_t>(p) & (n - 1)); }

static bool quant_vectorised(const QuantArgs &a) {
    return a.H % 8 == 0 && a.x_stride % 8 == 0 && a.q_stride % 8 == 0 && aligned(a.x, 16) && aligned(a.q, 8);
}

bool norm_quant_vectorised(const QuantArgs &a) {
    return quant_vectorised(a) && a.H <= 8 * 2048 && aligned(a.weight, 16) &&
           (!a.residual || (a.res_stride % 8 == 0 && aligned(a.residual, 16)));
}

template <typename AT, bool SILU>
static hipError_t quant_at(const QuantArgs &a, hipStream_t stream) {
    const int64_t groups = (a.H + FP8_GROUP - 1) / FP8_GROUP;
    if (!quant_vectorised(a)) {
        const int64_t blocks = ((int64_t)a.T * groups + QT / 64 - 1) / (QT / 64);
        hipLaunchKernelGGL((quant_scalar_kernel<AT, SILU>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(QT), 0,
                           stream, a);
        return hipGetLastError();
    }
    const int64_t cols = (a.H / 8 + QT - 1) / QT;
    const bool many = cols * a.T >= 8192;
    const int64_t rows = many ? 4 : 1, gy = ((int64_t)a.T + rows - 1) / rows;
    // grid.y holds 65535 blocks: longer batches run as several launches
    for (int64_t y0 = 0; y0 < gy; y0 += 65535) {
        QuantArgs b = a;
        const int64_t t0 = y0 * rows, left = a.T - t0, ny = gy - y0 < 65535 ? gy - y0 : 65535;
        b.x = static_cast<const uint16_t *>(a.x) + t0 * a.x_stride;
        b.q = static_cast<uint8_t *>(a.q) + t0 * a.q_stride;
        b.scales = a.scales + t0;
        b.T = (int)(left < ny * rows ? left : ny * rows);
        const dim3 grid((unsigned)cols, (unsigned)ny);
        if (many) hipLaunchKernelGGL((quant_vec_kernel<AT, SILU, 4>), grid, dim3(QT), 0, stream, b);
        else hipLaunchKernelGGL((quant_vec_kernel<AT, SILU, 1>), grid, dim3(QT), 0, stream, b);
    }
    return hipGetLastError();
}

hipError_t launch_group_quant(const QuantArgs &a, hipStream_t stream) {
    if (a.T == 0 || a.H == 0) return hipSuccess;
    return a.dtype == PQ_DTYPE_BF16 ? quant_at<bf16_t, false>(a, stream) : quant_at<fp16_t, false>(a, stream);
}

hipError_t launch_silu_quant(const QuantArgs &a, hipStream_t stream) {
    if (a.T == 0 || a.H == 0) return hipSuccess;
    return a.dtype == PQ_DTYPE_BF16 ? quant_at<bf16_t, true>(a, stream) : quant_at<fp16_t, true>(a, stream);
}

template <typename AT, bool ADD>
static hipError_t norm_quant_at(const QuantArgs &a, hipStream_t stream) {
    const dim3 grid((unsigned)a.T);
    if (!norm_quant_vectorised(a)) {
        hipLaunchKernelGGL((norm_quant_scalar_kernel<AT, ADD>), grid, dim3(QT), (size_t)a.H * 4, stream, a);
        return hipGetLastError();
    }
    const int nvec = a.H / 8;
#define PQ_NQ(THREADS, NV) hipLaunchKernelGGL((norm_quant_kernel<AT, THREADS, NV, ADD>), grid, dim3(THREADS), 0, stream, a)
    if (nvec <= 128) PQ_NQ(128, 1);
    else if (nvec <= 256) PQ_NQ(256, 1);
    else if (nvec <= 512) PQ_NQ(512, 1);
    else if (nvec <= 1024) PQ_NQ(1024, 1);
    else PQ_NQ(1024, 2);
#undef PQ_NQ
    return hipGetLastError();
}

hipError_t launch_norm_quant(const QuantArgs &a, hipStream_t stream) {
    if (a.T == 0 || a.H == 0) return hipSuccess;
    const bool add = a.residual != nullptr;
    if (a.dtype == PQ_DTYPE_BF16) return add ? norm_quant_at<bf16_t, true>(a, stream) : norm_quant_at<bf16_t, false>(a, stream);
    return add ? norm_quant_at<fp16_t, true>(a, stream) : norm_quant_at<fp16_t, false>(a, stream);
}

}  // namespace pq
