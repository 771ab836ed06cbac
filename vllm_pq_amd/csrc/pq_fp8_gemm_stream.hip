// Block-scaled e4m3 product for up to 16 tokens: the weights streamed once from HBM straight into registers
// (pq_fp8_gemm.hip has the formula).
//
// A block of 8 waves walks row tiles of 16 features; wave w owns the scale blocks w, w + 8, w + 16 and w + 24 of K, so the
// block reads rows contiguously, and keeps its part of the ACTIVATIONS in registers for all tiles.  What moves in the loop is
// weights alone, the next tile's requested before the present ones are multiplied: the loads never drain.  A load shaped
// like the matrix operand (lanes of a quad on four rows) runs at a quarter of a CU's rate, 38 GB/s measured, which is
// still 1.5 times a CU's share of HBM.  The waves' sums meet in LDS once per tile, added in wave order.  A K of more than 32
// scale blocks is cut into ranges (gridDim.y) whose sums are added by a second launch.  Bound by the weights' bytes: in a graph,
// 16 tokens of 28672 x 4096 25.3 to 27.8 us with weights from HBM (4.2 to 4.6 TB/s), 22.0 where the last-level cache holds them; 1
// token of 6144 x 4096 10.8 us (2.3 TB/s, launch included) and 8.7.
//
// FUSED takes fp16 / bf16 activations: the block quantises them itself into LDS while its first weights are on their way
// (the same arithmetic as fp8_group_quant, so the same values), which saves a launch where there are few.
#include <hip/hip_runtime.h>
#include <type_traits>

#include "pq_common.cuh"
#include "pq_fp8_mfma.cuh"
#include "pq_fp8_scale.cuh"
#include "pq_kernels.h"

namespace pq {

constexpr int SM_WAVES = 8, SM_KPW = 4, SM_ROW = 20;   // waves; scale blocks of a wave at most; floats between tokens' sums
constexpr int SM_RANGE = SM_WAVES * SM_KPW;            // scale blocks of a range of K
constexpr size_t SM_SUM_BYTES = 2 * SM_WAVES * 16 * SM_ROW * sizeof(float);
constexpr int SM_MAX_FUSED = 8192;                     // values a block quantises at most (whole groups and scales: up to 9.7 KiB of LDS)

typedef __attribute__((address_space(4))) float const_float;   // memory that no kernel running writes

// 16 bytes from any address: one load, whatever the alignment
__device__ __forceinline__ u32x4 load16u(const uint8_t *p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// part: NULL, or the ranges' sums [gridDim.y][T][np]
template <typename AT, bool FUSED, int KPW>
__global__ __launch_bounds__(SM_WAVES * 64, 4) void fp8_gemm_stream_kernel(Fp8GemmArgs a, int tiles, int range, float *part, int64_t np) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    float *const s_sum = reinterpret_cast<float *>(smem);
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int KB = (a.K + FP8_GROUP - 1) / FP8_GROUP, tail = a.K % FP8_GROUP;
    const int kb0 = blockIdx.y * range + wave, kb_end = min(KB, (int)(blockIdx.y + 1) * range);   // this wave's first, the range's end

    // This lane's two pieces of a row in its wave's scale block i, at 16 c and 64 + 16 c.  In a short last block a piece that
    // reaches behind the end is the last 16 features of the row instead (back); what it holds twice or should not hold
    // counts as zero on the activations' side (keep).  Blocks behind the range read its last one again and count as zero.
    auto block = [&](int i) { return min(kb0 + SM_WAVES * i, kb_end - 1); };
    const uint32_t back0 = tail && 16 * c + 16 > tail ? 16 * c + 16 - tail : 0, back1 = tail && 16 * c + 80 > tail ? 16 * c + 80 - tail : 0;
    auto piece = [&](int i, int h) {      // 16 bytes further, for bases 16 lower: the offset stays unsigned
        return 16 + 16 * c + 64 * h - (block(i) == KB - 1 ? (h ? back1 : back0) : 0);
    };
    auto keep = [&](int i, int h, int e) {
        const int kb = kb0 + SM_WAVES * i, end = kb >= kb_end ? 0 : kb == KB - 1 && tail ? tail : FP8_GROUP;
        const int drop = 64 * h + 16 * c + 16 - end - 4 * e;      // leading bytes of dword e that do not count
        return drop <= 0 ? -1 : drop >= 4 ? 0 : (int)(0xffffffffu << (8 * drop));
    };
    const uint8_t *const w = static_cast<const uint8_t *>(a.w) - 16;
    auto load = [&](int tile, i32x8 *to) {
        const uint8_t *base = w + (int64_t)tile * 16 * a.w_stride;
        const uint32_t row = (uint32_t)min(r, a.N - 1 - tile * 16) * (uint32_t)a.w_stride;
#pragma unroll
        for (int i = 0; i < KPW; ++i) {
            const uint8_t *bk = base + block(i) * FP8_GROUP;
            to[i] = join(load16u(bk + (row + piece(i, 0))), load16u(bk + (row + piece(i, 1))));
        }
    };
    i32x8 wv[2][KPW];
    int tile = blockIdx.x;
    load(tile, wv[0]);

    // ---- the activations of this wave's scale blocks
    i32x8 xv[KPW];
    float xs[KPW];
    uint32_t own[KPW];
    if constexpr (FUSED) {
        // 32 lanes x 4 values take a group
        uint8_t *const s_q = smem + SM_SUM_BYTES;
        float *const s_s = reinterpret_cast<float *>(s_q + (size_t)a.T * KB * FP8_GROUP);
        const int groups = a.T * KB, l = threadIdx.x & 31;
        constexpr int TAKE = 4;               // groups requested together
        for (int g0 = threadIdx.x >> 5; g0 < groups; g0 += TAKE * SM_WAVES * 2) {
            u32x2 v[TAKE];
#pragma unroll
            for (int i = 0; i < TAKE; ++i) {
                const int g = g0 + i * SM_WAVES * 2, t = g / KB, k = (g - t * KB) * FP8_GROUP + 4 * l;
                v[i] = u32x2{0u, 0u};
                if (g < groups && k < a.K) __builtin_memcpy(&v[i], static_cast<const uint16_t *>(a.q) + (int64_t)t * a.q_stride + k, 8);
            }
#pragma unroll
            for (int i = 0; i < TAKE; ++i) {
                const int g = g0 + i * SM_WAVES * 2;
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = Act<AT>::to_f32((uint16_t)(v[i][e >> 1] >> (16 * (e & 1))));
                uint32_t m = umax(umax(abs_bits(f[0]), abs_bits(f[1])), umax(abs_bits(f[2]), abs_bits(f[3])));
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) m = umax(m, (uint32_t)__shfl_xor((int)m, off, 64));
                const GroupScale gs = group_scale(m);
                if (g < groups) {
                    *reinterpret_cast<uint32_t *>(s_q + g * FP8_GROUP + 4 * l) = pack4(f, gs);
                    if (l == 0) s_s[g] = gs.s;
                }
            }
        }
        __syncthreads();
        const int t = min(r, a.T - 1);
#pragma unroll
        for (int i = 0; i < KPW; ++i) {
            const uint8_t *row = s_q + (t * KB + block(i)) * FP8_GROUP - 16;
            xv[i] = join(*reinterpret_cast<const u32x4 *>(row + piece(i, 0)), *reinterpret_cast<const u32x4 *>(row + piece(i, 1)));
            xs[i] = s_s[t * KB + block(i)];
        }
    } else {
        const int t = min(r, a.T - 1);
        const uint8_t *row = static_cast<const uint8_t *>(a.q) + (int64_t)t * a.q_stride - 16;
#pragma unroll
        for (int i = 0; i < KPW; ++i) {
            const uint8_t *bk = row + block(i) * FP8_GROUP;
            xv[i] = join(load16u(bk + piece(i, 0)), load16u(bk + piece(i, 1)));
            xs[i] = a.xs[t * a.xs_token + block(i) * a.xs_group];
        }
    }
#pragma unroll
    for (int i = 0; i < KPW; ++i) {
        own[i] = kb0 + SM_WAVES * i < kb_end ? ~0u : 0u;   // scales behind the range count as 0 (no 0 x infinity)
        asm("" : "+v"(own[i]));                            // (a mask: no branch around a load)
#pragma unroll
        for (int e = 0; e < 8; ++e) xv[i][e] &= keep(i, e >> 2, e & 3);
    }

    // ---- the tiles
    const uint16_t *bias = static_cast<const uint16_t *>(a.bias);
    int parity = 0;
    auto run_tile = [&](auto now_t, auto more_t) {
        constexpr int now = decltype(now_t)::value;           // buffer of this tile's weights
        constexpr bool more = decltype(more_t)::value;        // there is a next tile
        const int next = tile + gridDim.x;
        // read through the scalar cache: a load per wave and not per lane, asked for before the next weights
        const const_float *ws = (const const_float *)(uintptr_t)(a.ws + (int64_t)(tile * 16 / FP8_GROUP) * a.ws_stride);
        float wscale[KPW];
#pragma unroll
        for (int i = 0; i < KPW; ++i) wscale[i] = ws[block(i)];
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
        if (more) load(next, wv[now ^ 1]);
#pragma unroll
        for (int i = 0; i < KPW; ++i) {
            const f32x4 p = mfma_block(wv[now][i], xv[i]);
            const float s = __uint_as_float(__float_as_uint(xs[i] * wscale[i]) & own[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(s, p[e], acc[e]);
        }
        // two areas in turn: whoever writes one again has passed the barrier behind its last reading
        float *const area = s_sum + parity * SM_WAVES * 16 * SM_ROW;
        *reinterpret_cast<f32x4 *>(area + (wave * 16 + r) * SM_ROW + 4 * c) = acc;
        __syncthreads();
        const int t = threadIdx.x >> 4, n = tile * 16 + (threadIdx.x & 15);
        if (t < a.T && n < a.N) {
            float v = area[t * SM_ROW + (threadIdx.x & 15)];
#pragma unroll
            for (int k = 1; k < SM_WAVES; ++k) v += area[(k * 16 + t) * SM_ROW + (threadIdx.x & 15)];
            if (part) part[((int64_t)blockIdx.y * a.T + t) * np + n] = v;
            else {
                if (bias) v += Act<AT>::to_f32(bias[n]);
                static_cast<uint16_t *>(a.y)[(int64_t)t * a.y_stride + n] = Act<AT>::from_f32(v);
            }
        }
        parity ^= 1;
        tile = next;
    };
    const std::integral_constant<int, 0> even{};
    const std::integral_constant<int, 1> odd{};
    while (tile + 2 * (int)gridDim.x < tiles) {
        run_tile(even, std::true_type{});
        run_tile(odd, std::true_type{});
    }
    if (tile + (int)gridDim.x < tiles) {
        run_tile(even, std::true_type{});
        run_tile(odd, std::false_type{});
    } else run_tile(even, std::false_type{});
}

template <typename AT, bool FUSED>
static hipError_t stream_at(const Fp8GemmArgs &a, hipStream_t stream) {
    const int kb = (a.K + FP8_GROUP - 1) / FP8_GROUP, ranges = (kb + SM_RANGE - 1) / SM_RANGE, range = (kb + ranges - 1) / ranges;
    const size_t lds = SM_SUM_BYTES + (FUSED ? a.T * kb * (FP8_GROUP + sizeof(float)) : 0);
    const int tiles = (a.N + 15) / 16, slots = 512 / ranges;   // two blocks a CU, each with every so-manieth tile
    const int64_t np = ((int64_t)a.N + 3) / 4 * 4;
    float *part = ranges > 1 ? static_cast<float *>(a.tmp) : nullptr;
    const dim3 grid((unsigned)(tiles < slots ? tiles : slots), (unsigned)ranges);
    // as many blocks of K per wave as there are: those behind the end are fetched and multiplied all the same.  With 4 always:
    // 16 tokens of 4096 x 1000 5.2 us against 4.0, 8 of 4096 x 2048 6.3 against 5.3, 1 of 8192 x 1536 8.6 against 6.3
    auto kern = range <= SM_WAVES       ? fp8_gemm_stream_kernel<AT, FUSED, 1>
                : range <= 2 * SM_WAVES ? fp8_gemm_stream_kernel<AT, FUSED, 2>
                : range <= 3 * SM_WAVES ? fp8_gemm_stream_kernel<AT, FUSED, 3>
                                        : fp8_gemm_stream_kernel<AT, FUSED, SM_KPW>;
    hipLaunchKernelGGL(kern, grid, dim3(SM_WAVES * 64), lds, stream, a, tiles, range, part, np);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || !part ? e : launch_fp8_join(a, part, ranges, np, stream);
}

size_t fp8_gemm_stream_tmp_bytes(int T, int N, int K) {
    const size_t ranges = ((size_t)(K + FP8_GROUP - 1) / FP8_GROUP + SM_RANGE - 1) / SM_RANGE;
    return ranges > 1 ? ranges * T * (((size_t)N + 3) / 4 * 4) * sizeof(float) : 0;
}

bool fp8_gemm_stream_supported(const Fp8GemmArgs &a) {
    const size_t tmp = fp8_gemm_stream_tmp_bytes(a.T, a.N, a.K);
    return a.T <= 16 && a.K >= 16 && a.K <= SM_RANGE * 128 * FP8_GROUP && a.w_stride < (1 << 26) &&   // (32-bit offsets inside a tile)
           (tmp == 0 || (a.tmp && a.tmp_bytes >= tmp));
}

// Every block quantises for itself, which beats a launch in front while it takes less than that.  Inside against apart, in a
// graph with weights from HBM: 1 token of 28672 x 4096 25.1 us against 27.3, 2 tokens 25.7 against 28.5, 8 of 4096 x 1024 5.4
// against 6.0, 4 of 8192 x 2048 8.3 against 8.5, 2 of 6144 x 4096 11.9 against 11.7; with 16384 values (4 of 6144 x 4096) the
// product alone grows from 9.1 to 13.5, more than the 2.8 of the launch.
bool fp8_linear_fused(int T, int K) { return T <= 16 && K >= 16 && K % 16 == 0 && K <= SM_RANGE * FP8_GROUP && T * K <= SM_MAX_FUSED; }

hipError_t launch_fp8_gemm_stream(const Fp8GemmArgs &a, hipStream_t stream) {
    return a.dtype == PQ_DTYPE_BF16 ? stream_at<bf16_t, false>(a, stream) : stream_at<fp16_t, false>(a, stream);
}
hipError_t launch_fp8_linear_fused(const Fp8GemmArgs &a, hipStream_t stream) {
    return a.dtype == PQ_DTYPE_BF16 ? stream_at<bf16_t, true>(a, stream) : stream_at<fp16_t, true>(a, stream);
}

}  // namespace pq
