// Matrix product of 8-bit floating point (e4m3) activations and weights with a scale per block of 128:
//   y[t][n] = round( sum over blocks b of  xs[t][b] * ws[n / 128][b] * sum_{k in b} q[t][k] * w[n][k]   + bias[n] )
// One v_mfma_f32_16x16x128_f8f6f4 is exactly one block's inner sum for 16 rows x 16 tokens, in fp32 from zero; the scaled
// sum over the blocks is one fp32 FMA per value and block.  The weight rows are the MFMA's rows and the tokens its
// columns, so a lane holds 4 consecutive output features of ONE token and needs one token scale per block.
//
// Both operands give a lane the same features (16 at 16 c and 16 at 64 + 16 c of the block, c = lane / 16): the order inside
// the block does not matter to the sum, and four lanes read 64 contiguous bytes of a row.
#include <hip/hip_runtime.h>
#include <string.h>

#include "pq_common.cuh"
#include "pq_fp8_mfma.cuh"
#include "pq_kernels.h"

namespace pq {

template <bool ALIGNED>
__device__ __forceinline__ u32x4 load16(const uint8_t *p) {
    if constexpr (ALIGNED) return *reinterpret_cast<const u32x4 *>(p);
    u32x4 v;
    memcpy(&v, p, 16);
    return v;
}
// the first `valid` of 16 bytes, zeros behind them; reads nothing behind the valid bytes
template <bool ALIGNED>
__device__ __forceinline__ u32x4 load16_upto(const uint8_t *p, int valid) {
    if (valid >= 16) return load16<ALIGNED>(p);
    u32x4 v{0u, 0u, 0u, 0u};
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (4 * w + j < valid) v[w] |= (uint32_t)p[4 * w + j] << (8 * j);
    return v;
}

// ---- operands straight from memory into registers -------------------------------------------------------------
// For what the other two kernels do not take: fewer than 16 features, rows that the tiles' DMA cannot address, a long K
// without scratch.  Bound by the loads: shaped like the matrix operand they bring a CU 38 GB/s (512 tokens of 4096 x 4097 174 us).
// One block per tile of 16 NF rows x 16 TF tokens; its WK waves take the blocks of K in turn (wave w: w, w + WK, ...), so
// that together they walk the rows contiguously, and add their sums in wave order at the end.
template <typename AT, int NF, int TF, int WK, int U, bool ALIGNED>
__global__ __launch_bounds__(WK * 64) void fp8_gemm_direct_kernel(Fp8GemmArgs a) {
    constexpr int RS = 16 * NF + 4;              // floats between two tokens of a wave's sums in LDS
    __shared__ float s_sum[WK * 16 * RS];
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16 * NF, t0 = blockIdx.y * 16 * TF;
    const int KB = (a.K + FP8_GROUP - 1) / FP8_GROUP, full = a.K / FP8_GROUP;

    const uint8_t *wrow[NF], *xrow[TF];          // rows past the end read the last one; their sums are not stored
    const float *xs[TF], *ws[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const int n = n0 + 16 * f;
        wrow[f] = static_cast<const uint8_t *>(a.w) + (int64_t)min(n + r, a.N - 1) * a.w_stride + 16 * c;
        ws[f] = a.ws + (int64_t)(min(n, a.N - 1) / FP8_GROUP) * a.ws_stride;
    }
#pragma unroll
    for (int f = 0; f < TF; ++f) {
        const int64_t t = min(t0 + 16 * f + r, a.T - 1);
        xrow[f] = static_cast<const uint8_t *>(a.q) + t * a.q_stride + 16 * c;
        xs[f] = a.xs + t * a.xs_token;
    }
    f32x4 acc[NF][TF];
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < TF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int kb0 = wave; kb0 < KB; kb0 += WK * U) {
        i32x8 wv[U][NF], xv[U][TF];
        float xsv[U][TF], wsv[U][NF];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = kb0 + u * WK, k = kb * FP8_GROUP, left = a.K - k - 16 * c;
            if (kb < full) {
#pragma unroll
                for (int f = 0; f < NF; ++f) wv[u][f] = join(load16<ALIGNED>(wrow[f] + k), load16<ALIGNED>(wrow[f] + k + 64));
#pragma unroll
                for (int f = 0; f < TF; ++f) xv[u][f] = join(load16<ALIGNED>(xrow[f] + k), load16<ALIGNED>(xrow[f] + k + 64));
            } else if (kb < KB) {
#pragma unroll
                for (int f = 0; f < NF; ++f)
                    wv[u][f] = join(load16_upto<ALIGNED>(wrow[f] + k, left), load16_upto<ALIGNED>(wrow[f] + k + 64, left - 64));
#pragma unroll
                for (int f = 0; f < TF; ++f)
                    xv[u][f] = join(load16_upto<ALIGNED>(xrow[f] + k, left), load16_upto<ALIGNED>(xrow[f] + k + 64, left - 64));
            }
            if (kb < KB) {
#pragma unroll
                for (int f = 0; f < NF; ++f) wsv[u][f] = ws[f][kb];
#pragma unroll
                for (int f = 0; f < TF; ++f) xsv[u][f] = xs[f][kb * a.xs_group];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kb0 + u * WK < KB) {
#pragma unroll
                for (int i = 0; i < NF; ++i)
#pragma unroll
                    for (int j = 0; j < TF; ++j) {
                        const f32x4 p = mfma_block(wv[u][i], xv[u][j]);
                        const float s = xsv[u][j] * wsv[u][i];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(s, p[e], acc[i][j][e]);
                    }
            }
        }
    }

    // the waves' sums, added in wave order; a thread then holds 4 consecutive features of one token
    const bool vec = a.y_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7) == 0;
#pragma unroll
    for (int j = 0; j < TF; ++j) {
        if (j) __syncthreads();
#pragma unroll
        for (int i = 0; i < NF; ++i) *reinterpret_cast<f32x4 *>(&s_sum[(wave * 16 + r) * RS + 16 * i + 4 * c]) = acc[i][j];
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * 4 * NF; e += WK * 64) {
            const int tl = e / (4 * NF), nl = e % (4 * NF) * 4, n = n0 + nl;
            const int64_t t = t0 + 16 * j + tl;
            if (t >= a.T || n >= a.N) continue;
            f32x4 v = *reinterpret_cast<const f32x4 *>(&s_sum[tl * RS + nl]);
#pragma unroll
            for (int w = 1; w < WK; ++w) {
                const f32x4 o = *reinterpret_cast<const f32x4 *>(&s_sum[(w * 16 + tl) * RS + nl]);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += o[k];
            }
            const uint16_t *bias = static_cast<const uint16_t *>(a.bias);
            uint16_t *y = static_cast<uint16_t *>(a.y) + t * a.y_stride + n;
            if (vec && n + 4 <= a.N) {
                if (bias)
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] += Act<AT>::to_f32(bias[n + k]);
                *reinterpret_cast<u32x2 *>(y) = u32x2{Act<AT>::pack2(v[0], v[1]), Act<AT>::pack2(v[2], v[3])};
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n + k < a.N) y[k] = Act<AT>::from_f32(v[k] + (bias ? Act<AT>::to_f32(bias[n + k]) : 0.f));
            }
        }
    }
}

// y = round(sum of the K ranges' sums + bias): 4 features of one token per thread, the ranges in order.  Two ranges of 128 tokens
// x 4096 features: 3.8 us, most of it the launch.
template <typename AT>
__global__ __launch_bounds__(256) void fp8_join_kernel(const float *part, int split, int T, int N, int64_t np, const uint16_t *bias,
                                                       uint16_t *y, int64_t y_stride) {
    const int64_t per = np / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= T * per) return;
    const int64_t t = i / per;
    const int n = (int)(i - t * per) * 4;
    f32x4 v = *reinterpret_cast<const f32x4 *>(part + t * np + n);
    for (int k = 1; k < split; ++k) v += *reinterpret_cast<const f32x4 *>(part + ((int64_t)k * T + t) * np + n);
    uint16_t *row = y + t * y_stride + n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < N) row[e] = Act<AT>::from_f32(v[e] + (bias ? Act<AT>::to_f32(bias[n + e]) : 0.f));
}

hipError_t launch_fp8_join(const Fp8GemmArgs &a, const float *part, int ranges, int64_t np, hipStream_t stream) {
    const dim3 grid((unsigned)((a.T * (np / 4) + 255) / 256)), block(256);
    const uint16_t *bias = static_cast<const uint16_t *>(a.bias);
    uint16_t *y = static_cast<uint16_t *>(a.y);
    if (a.dtype == PQ_DTYPE_BF16) hipLaunchKernelGGL((fp8_join_kernel<bf16_t>), grid, block, 0, stream, part, ranges, a.T, a.N, np, bias, y, a.y_stride);
    else hipLaunchKernelGGL((fp8_join_kernel<fp16_t>), grid, block, 0, stream, part, ranges, a.T, a.N, np, bias, y, a.y_stride);
    return hipGetLastError();
}

template <typename AT, int NF, int TF, int U>
static hipError_t direct_at(const Fp8GemmArgs &a, hipStream_t stream) {
    constexpr int WK = 8;
    const dim3 grid((unsigned)((a.N + 16 * NF - 1) / (16 * NF)), (unsigned)((a.T + 16 * TF - 1) / (16 * TF)));
    const bool aligned = a.q_stride % 16 == 0 && a.w_stride % 16 == 0 && !((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.w)) & 15);
    if (aligned) hipLaunchKernelGGL((fp8_gemm_direct_kernel<AT, NF, TF, WK, U, true>), grid, dim3(WK * 64), 0, stream, a);
    else hipLaunchKernelGGL((fp8_gemm_direct_kernel<AT, NF, TF, WK, U, false>), grid, dim3(WK * 64), 0, stream, a);
    return hipGetLastError();
}

// ---- a K that is no multiple of 4, more than 16 tokens ----------------------------------------------------------
// Rows of such a K start at any byte and the tiles' DMA reads dwords.  Both operands are copied to rows of K rounded up to 16
// with zeros behind them, 16 bytes per thread, and the tiles run on the copies.  The copy moves the weights twice; even so, against
// the direct kernel: 17 tokens of 4096 x 4099 21.6 us against 26.1, 64 tokens of 28672 x 4095 92 against 195, 512 tokens of
// 4096 x 4097 32 against 174, 4096 tokens of 8192 x 4097 180 against 2681.
__global__ __launch_bounds__(256) void fp8_pad_kernel(const uint8_t *w, int64_t w_stride, uint32_t w_pieces, const uint8_t *q,
                                                      int64_t q_stride, uint32_t pieces, int K, uint32_t row_pieces, uint8_t *out) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const uint32_t row = i / row_pieces, k = (i - row * row_pieces) * 16, w_rows = w_pieces / row_pieces;
    const uint8_t *from = row < w_rows ? w + (int64_t)row * w_stride : q + (int64_t)(row - w_rows) * q_stride;
    *reinterpret_cast<u32x4 *>(out + (int64_t)i * 16) = load16_upto<false>(from + k, K - (int)k);
}

static int padded(int K) { return K % 4 ? (K + 15) / 16 * 16 : K; }
static size_t pad_bytes(int T, int N, int K) { return K % 4 && K >= 16 ? ((size_t)T + N) * padded(K) : 0; }

static bool pad_supported(const Fp8GemmArgs &a) {
    const size_t bytes = pad_bytes(a.T, a.N, a.K);
    return bytes && a.tmp && a.tmp_bytes >= bytes && bytes / 16 < (1u << 31);
}
static Fp8GemmArgs padded_args(const Fp8GemmArgs &a) {
    Fp8GemmArgs b = a;
    const size_t bytes = pad_bytes(a.T, a.N, a.K);
    b.K = padded(a.K);
    b.w = a.tmp;
    b.q = static_cast<const uint8_t *>(a.tmp) + (size_t)a.N * b.K;
    b.w_stride = b.q_stride = b.K;
    b.tmp = static_cast<uint8_t *>(a.tmp) + bytes;
    b.tmp_bytes = a.tmp_bytes - bytes;
    return b;
}
static hipError_t launch_pad(const Fp8GemmArgs &a, hipStream_t stream) {
    const uint32_t row = padded(a.K) / 16, pieces = ((uint32_t)a.T + a.N) * row;
    hipLaunchKernelGGL(fp8_pad_kernel, dim3((pieces + 255) / 256), dim3(256), 0, stream, static_cast<const uint8_t *>(a.w), a.w_stride,
                       (uint32_t)a.N * row, static_cast<const uint8_t *>(a.q), a.q_stride, pieces, a.K, row,
                       static_cast<uint8_t *>(a.tmp));
    return hipGetLastError();
}

template <typename AT>
static hipError_t fp8_gemm_at(const Fp8GemmArgs &a, hipStream_t stream) {
    if (fp8_gemm_stream_supported(a)) return launch_fp8_gemm_stream(a, stream);
    if (fp8_gemm_tiled_supported(a)) return launch_fp8_gemm_tiled(a, stream);
    if (a.T > 16 && pad_supported(a)) {
        const Fp8GemmArgs b = padded_args(a);
        if (fp8_gemm_tiled_supported(b)) {
            const hipError_t e = launch_pad(a, stream);
            return e != hipSuccess ? e : launch_fp8_gemm_tiled(b, stream);
        }
    }
    if (a.T <= 16) return direct_at<AT, 1, 1, 4>(a, stream);
    return direct_at<AT, 2, 4, 1>(a, stream);
}

// scratch the launch of this problem uses when it gets it (every layout)
size_t fp8_gemm_tmp_bytes(int T, int N, int K) {
    return T <= 16 ? fp8_gemm_stream_tmp_bytes(T, N, K) : pad_bytes(T, N, K) + fp8_gemm_tiled_plan(T, N, padded(K), SIZE_MAX).part_bytes;
}

hipError_t launch_fp8_gemm(const Fp8GemmArgs &a, hipStream_t stream) {
    // grid.y holds 65535 token tiles: longer batches run as several launches
    constexpr int MAX_T = 65535 * 16;
    for (int64_t t0 = 0; t0 < a.T; t0 += MAX_T) {
        Fp8GemmArgs b = a;
        b.q = static_cast<const uint8_t *>(a.q) + t0 * a.q_stride;
        b.xs = a.xs + t0 * a.xs_token;
        b.y = static_cast<uint16_t *>(a.y) + t0 * a.y_stride;
        b.T = (int)(a.T - t0 < MAX_T ? a.T - t0 : MAX_T);
        const hipError_t e = a.dtype == PQ_DTYPE_BF16 ? fp8_gemm_at<bf16_t>(b, stream) : fp8_gemm_at<fp16_t>(b, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace pq
