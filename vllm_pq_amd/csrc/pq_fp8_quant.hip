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
// values (one 16-byte load, at any alignment; the last piece of a row may be shorter), 16 neighbouring lanes a group: its
// maximum is four lane exchanges, nothing passes through LDS.  Measured: 4096 x 14336 bf16 32.3 us (5.4 TB/s of the bytes named
// above; a plain copy reaches 5.0), silu_and_mul 52 us (5.6 TB/s), the norm with a residual of 4096 x 8192 fp16 42.3 us
// (5.6 TB/s); 16 rows of 4096 2.6 to 3.4 us, which is what an empty launch takes.
#include <hip/hip_runtime.h>

#include "pq_common.cuh"
#include "pq_fp8_scale.cuh"
#include "pq_kernels.h"

namespace pq {

constexpr int QT = 256;                  // threads per block of the quantising kernels without a norm
constexpr int QV = FP8_GROUP / 8;        // threads per group

// maximum over the 16 lanes of a group, in all of them: rotations within a row of lanes, part of the maximum's instruction
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
    m = umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, false));   // row_ror:8
    m = umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, false));
    m = umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, false));
    return umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, false));
}

// silu(g) * u = g u / (1 + exp(-g)) in fp32.  The product of two act-dtype values is exact in fp32 and the quotient correctly
// rounded (one Newton step on its residual), so the error is that of the exponential: 2^t, t = -g log2(e), where what t's
// rounding leaves out (up to |t| 2^-24 of the result) is put back to first order.  Numerator and denominator carry a factor of
// 2^-8, so that g u stays finite wherever the result does.  A NaN in g comes through.
//
// FAR is for gates beyond 88 on either side, of which there are none in most waves:
//   - the exponential takes g as at most 128, where it is far below 1's last place, so that t stays finite at the type's
//     largest value;
//   - below -87.5 numerator and denominator carry a further 2^-125: 2^t itself leaves fp32 from -88.7 on;
//   - below -174 g counts as 0: |silu(g) u| < 2^-115 for every finite u, less than half of the smallest value that e4m3 holds
//     beside the floor's scale (2^-9 * 2^-96 / 448), so the type's lowest value gives nothing;
//   - an infinity in g comes through u, as NaN.
// For the other gates it computes the same bits.  4096 x 14336 with such a gate in every wave 68 us, without any 55 (back to back).
template <bool FAR>
__device__ __forceinline__ float silu_mul(float g, float u) {
    constexpr float L = 1.4426950408889634f * 256, L_LO = (float)(1.4426950408889634074 * 256 - (double)L), LN2 = 0.6931471805599453f;
    constexpr float S = 0x1p-8f;
    const float x = FAR && g < -174.0f ? 0.0f : g * S, y = FAR && x > 128.0f * S ? 128.0f * S : x;
    const bool low = FAR && x < -87.5f * S;
    const float one = low ? 0x1p-125f : 1.0f, t = -y * L, rest = __builtin_fmaf(-y, L_LO, __builtin_fmaf(-y, L, -t));
    const float e = __builtin_amdgcn_exp2f(low ? t - 125.0f : t);
    const float d = (one + __builtin_fmaf(e * rest, LN2, e)) * S, r = __builtin_amdgcn_rcpf(d);
    const float p = FAR ? x * __builtin_fmaf(g, 0.0f, u) * one : x * u, q = p * r;
    return __builtin_fmaf(__builtin_fmaf(-d, q, p), r, q);
}
// f = silu(f) * u for 8 values
__device__ __forceinline__ void silu_mul8(float *f, const float *u) {
    float far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) far = fmaxf(far, __builtin_fabsf(f[j]));
    if (__builtin_amdgcn_ballot_w64(far > 87.5f)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = silu_mul<true>(f[j], u[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = silu_mul<false>(f[j], u[j]);
    }
}

// 8 act-dtype values from any address; WHOLE: all of a row's pieces have 8, else the first `valid` and zeros behind, nothing
// read behind them.  ONCE: no one reads them again (past the caches)
template <bool WHOLE, bool ONCE>
__device__ __forceinline__ u32x4 raw8(const uint16_t *p, int valid) {
    typedef u32x4 u32x4_any __attribute__((aligned(2)));
    if (WHOLE || valid >= 8) {
        if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
        else return *reinterpret_cast<const u32x4_any *>(p);
    }
    u32x4 a{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < valid) a[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
    return a;
}
template <typename AT>
__device__ __forceinline__ void unpack8(const u32x4 &a, float *f) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[2 * w] = Act<AT>::to_f32((uint16_t)a[w]);
        f[2 * w + 1] = Act<AT>::to_f32((uint16_t)(a[w] >> 16));
    }
}
// the first `valid` of 8 quotients as e4m3, to any address
template <bool WHOLE>
__device__ __forceinline__ void store8(uint8_t *q, int valid, const float *f, const GroupScale &g) {
    const u32x2 v{pack4(f, g), pack4(f + 4, g)};
    if (WHOLE || valid >= 8) __builtin_memcpy(q, &v, 8);
    else
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) q[j] = (uint8_t)(v[j >> 2] >> (8 * (j & 3)));
}
__device__ __forceinline__ uint32_t amax8(const float *f) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = umax(m, abs_bits(f[j]));
    return m;
}

// ---- without a norm: groups are independent ------------------------------------------------------------
// A block takes 2048 features of R consecutive rows, all R requested before the first is worked on (rows and features past
// the end read the last row's first piece again and are not stored).
template <typename AT, bool SILU, int R, bool WHOLE>
__global__ __launch_bounds__(QT) void quant_kernel(QuantArgs a) {
    const int v = blockIdx.x * QT + threadIdx.x, H = a.H, valid = H - v * 8;
    const int64_t t0 = (int64_t)blockIdx.y * R;
    const uint16_t *x = static_cast<const uint16_t *>(a.x) + (valid > 0 ? v * 8 : 0);
    uint8_t *q = static_cast<uint8_t *>(a.q) + v * 8;
    u32x4 first[R], second[SILU ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const uint16_t *row = x + (t0 + i < a.T ? t0 + i : a.T - 1) * a.x_stride;
        first[i] = raw8<WHOLE, true>(row, valid);
        if constexpr (SILU) second[i] = raw8<WHOLE, true>(row + H, valid);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t t = t0 + i;
        float f[8];
        unpack8<AT>(first[i], f);
        if constexpr (SILU) {
            float u[8];
            unpack8<AT>(second[i], u);
            silu_mul8(f, u);
        }
        const GroupScale g = group_scale(group_max(valid > 0 ? amax8(f) : 0u));
        if (valid > 0 && t < a.T) {
            store8<WHOLE>(q + t * a.q_stride, valid, f, g);
            if (threadIdx.x % QV == 0) a.scales[(int64_t)(v / QV) * a.scale_stride + t] = g.s;
        }
    }
}

// ---- with a norm -----------------------------------------------------------------------------------------
// One block of THREADS per token row; the row stays in registers between the sum of squares and the scaling, as in
// rms_norm_kernel.  ADD: z = x + residual, the residual becomes the rounded sum (the norm uses the unrounded one).
// 1 / rms = 2^e f, f in [1, 2), is a factor of a group's values and of its scale alike, so the quotients are taken with its
// power of two alone, which rounds nothing,
//   q = e4m3(u / (max |u| / 448)),  s = max |u| / 448 f,  u = 2^e z w:
// one rounding less per value.  The floor 2^-96 holds for max |u| f, the normed values, and becomes 2^-96 / f in the quotients;
// 2^e keeps u within a factor of 2 of them, so that a row of small values leaves no quotient of subnormal numbers.
template <typename AT, int THREADS, int NV, bool ADD, bool WHOLE>
__global__ __launch_bounds__(THREADS) void norm_quant_kernel(QuantArgs a) {
    __shared__ float s_part[THREADS / 64];
    const int64_t t = blockIdx.x;
    const uint16_t *xr = static_cast<const uint16_t *>(a.x) + t * a.x_stride;
    uint16_t *rr = ADD ? static_cast<uint16_t *>(a.residual) + t * a.res_stride : nullptr;
    float z[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = i * THREADS + threadIdx.x, valid = a.H - v * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[i][j] = 0.f;
        if (valid > 0) {
            unpack8<AT>(raw8<WHOLE, true>(xr + v * 8, valid), z[i]);
            if constexpr (ADD) {
                float r[8];
                unpack8<AT>(raw8<WHOLE, false>(rr + v * 8, valid), r);
                u32x4 o;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    z[i][2 * w] += r[2 * w];
                    z[i][2 * w + 1] += r[2 * w + 1];
                    o[w] = Act<AT>::pack2(z[i][2 * w], z[i][2 * w + 1]);
                }
                if (WHOLE || valid >= 8) __builtin_memcpy(rr + v * 8, &o, 16);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < valid) rr[v * 8 + j] = (uint16_t)(o[j >> 1] >> (16 * (j & 1)));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(z[i][j], z[i][j], ss);
        }
    }
    const float rs = rsqrtf(block_sum<THREADS>(ss, s_part) / (float)a.H + a.eps);
    const bool plain = __builtin_isnormal(rs);     // 0, infinite or NaN: the values take it as it is
    const float pow2 = plain ? __uint_as_float(__float_as_uint(rs) & 0x7f800000u) : rs;
    const float frac = plain ? __uint_as_float((__float_as_uint(rs) & 0x007fffffu) | 0x3f800000u) : 1.f;
    uint8_t *qr = static_cast<uint8_t *>(a.q) + t * a.q_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = i * THREADS + threadIdx.x, valid = a.H - v * 8;
        if (valid > 0) {
            float w[8];
            unpack8<AT>(raw8<WHOLE, false>(static_cast<const uint16_t *>(a.weight) + v * 8, valid), w);
#pragma unroll
            for (int j = 0; j < 8; ++j) z[i][j] = z[i][j] * pow2 * w[j];
        }
        const float floor = __uint_as_float(AMAX_MIN_BITS), m = __uint_as_float(group_max(amax8(z[i]))), amax = m * frac;
        const bool low = amax < floor;                            // (a NaN is not low)
        const GroupScale g = scale_of(low ? floor / frac : m);
        if (valid > 0) {
            store8<WHOLE>(qr + v * 8, valid, z[i], g);
            if (threadIdx.x % QV == 0) a.scales[(int64_t)(v / QV) * a.scale_stride + t] = (low ? floor : amax) / FP8_MAX;
        }
    }
}

// ---- launches ----------------------------------------------------------------------------------------------
template <typename AT, bool SILU, bool WHOLE>
static hipError_t quant_at(const QuantArgs &a, hipStream_t stream) {
    const int64_t cols = (a.H + 8 * QT - 1) / (8 * QT);
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
        if (many) hipLaunchKernelGGL((quant_kernel<AT, SILU, 4, WHOLE>), grid, dim3(QT), 0, stream, b);
        else hipLaunchKernelGGL((quant_kernel<AT, SILU, 1, WHOLE>), grid, dim3(QT), 0, stream, b);
    }
    return hipGetLastError();
}

template <bool SILU>
static hipError_t quant_any(const QuantArgs &a, hipStream_t stream) {
    if (a.T == 0 || a.H == 0) return hipSuccess;
    const bool bf16 = a.dtype == PQ_DTYPE_BF16;
    if (a.H % 8 == 0) return bf16 ? quant_at<bf16_t, SILU, true>(a, stream) : quant_at<fp16_t, SILU, true>(a, stream);
    return bf16 ? quant_at<bf16_t, SILU, false>(a, stream) : quant_at<fp16_t, SILU, false>(a, stream);
}
hipError_t launch_group_quant(const QuantArgs &a, hipStream_t stream) { return quant_any<false>(a, stream); }
hipError_t launch_silu_quant(const QuantArgs &a, hipStream_t stream) { return quant_any<true>(a, stream); }

template <typename AT, bool ADD, bool WHOLE>
static hipError_t norm_quant_at(const QuantArgs &a, hipStream_t stream) {
    const dim3 grid((unsigned)a.T);
    const int nvec = (a.H + 7) / 8;
#define PQ_NQ(THREADS, NV) hipLaunchKernelGGL((norm_quant_kernel<AT, THREADS, NV, ADD, WHOLE>), grid, dim3(THREADS), 0, stream, a)
    if (nvec <= 128) PQ_NQ(128, 1);
    else if (nvec <= 256) PQ_NQ(256, 1);
    else if (nvec <= 512) PQ_NQ(512, 1);
    // a block of 1024 threads has the whole row under way at once, which is what few rows need (in a graph, 16 x 8192 3.74 against
    // 3.82 us); four blocks of 512 a CU overlap one's barrier with the others' loads (1024 x 8192 12.1 against 12.8 us, 4096 x 8192
    // 41.2 against 43.7)
    else if (nvec <= 1024 && a.T > 512) PQ_NQ(512, 2);
    else if (nvec <= 1024) PQ_NQ(1024, 1);
    else PQ_NQ(1024, 2);
#undef PQ_NQ
    return hipGetLastError();
}

template <typename AT>
static hipError_t norm_quant_any(const QuantArgs &a, hipStream_t stream) {
    if (a.H % 8 == 0) return a.residual ? norm_quant_at<AT, true, true>(a, stream) : norm_quant_at<AT, false, true>(a, stream);
    return a.residual ? norm_quant_at<AT, true, false>(a, stream) : norm_quant_at<AT, false, false>(a, stream);
}

hipError_t launch_norm_quant(const QuantArgs &a, hipStream_t stream) {
    if (a.T == 0 || a.H == 0) return hipSuccess;
    return a.dtype == PQ_DTYPE_BF16 ? norm_quant_any<bf16_t>(a, stream) : norm_quant_any<fp16_t>(a, stream);
}

}  // namespace pq
