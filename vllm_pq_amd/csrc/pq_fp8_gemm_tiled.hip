// Block-scaled e4m3 product for many tokens: tiles of both operands through LDS (pq_fp8_gemm.hip has the formula and the
// kernel for few tokens or awkward layouts).
//
// A block owns BN weight rows x BT tokens and walks K one scale block (128 features, 128 bytes of a row) per step.  Both
// tiles and the step's scales come in by LDS-DMA, STAGES - 1 steps ahead, so no register holds them on the way.  A wave owns
// (BN / WN) x (BT / WT) of the tile: NF x TF matrix instructions a step, each one block's inner sum from zero, and behind
// each the scaled sum: 4 FMAs, which the vector unit runs beside the matrix unit (half its time: 4 x 4 against 32 cycles).
//
// LDS rows are 128 bytes, the 16-byte piece p of row r at slot p ^ ((r / 2) mod 8): the 16 lanes that ds_read_b128 serves in
// one cycle ({0-3, 12-15, 20-27} and the like: rows 0-3 and 12-15 at piece c, rows 4-11 at piece c ^ 1) fall on 16
// different groups of banks.  The DMA writes 64 lanes x 16 bytes in lane order, so it is the lanes' GLOBAL addresses that are
// permuted; the 8 lanes of a row still read one 128-byte line.
//
// Measured over several devices, in a graph: 4096 tokens of 28672 x 4096 404 to 440 us with the weights in the last-level cache
// (2.2 to 2.4 PFLOP/s), 419 to 450 us from HBM; the first 20 calls after idleness 456 to 492.  Of 421 us the matrix
// instructions alone take 268, with the LDS reads 296, with the sums 325; the rest is DMA and stores in the way of
// both, at 1.9 GHz, which is what the power limit leaves of the clock.  512 tokens of 4096 x 4096 15.2 to 15.8 us (5 us of
// it to start and end one round) and 18 from HBM; 128 tokens of 4096 x 14336 16.5 to 18.4 us and 4 for adding the two ranges, 27 in
// all from HBM (a block has 48 KiB of weights under way, and memory answers in 1.9 us).
#include <hip/hip_runtime.h>
#include <atomic>
#include <math.h>
#include <type_traits>

#include "pq_common.cuh"
#include "pq_fp8_mfma.cuh"
#include "pq_kernels.h"

namespace pq {

// 64 lanes x 16 (4) bytes from global memory straight into LDS at `lds` (wave-uniform) + lane * 16 (4)
__device__ __forceinline__ void dma16(uint32_t lds, uint32_t voff, const void *base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(voff), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma4(uint32_t lds, uint32_t voff, const void *base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(voff), "s"(base) : "memory", "m0");
}

// KG groups of WN x WT waves share a tile: group g takes the steps g, g + KG, ..., each through stages of its own
template <int BN, int BT, int WN, int WT, int KG, int STAGES>
struct Fp8Tile {
    static constexpr int THREADS = WN * WT * KG * 64, WAVES = WN * WT;   // WAVES: of one group
    static constexpr int NF = BN / WN / 16, TF = BT / WT / 16;
    static constexpr int RA = BN / (WAVES * 8), RB = BT / (WAVES * 8);   // DMA rounds of a stage: 8 rows a wave and round
    static constexpr int LOADS = RA + RB + 1;                            // DMA instructions of a wave and stage
    static constexpr int XS = (BN + BT) * 128, WS = XS + BT * 4;         // byte offsets of the scales in a stage
    static constexpr int STAGE = WS + 256;
    static constexpr int LDS = KG * STAGES * STAGE;
    static_assert(RA * WAVES * 8 == BN && RB * WAVES * 8 == BT && WAVES > BT / 64 && BT % 64 == 0, "");
    static_assert(KG == 1 || (KG == 2 && BN * BT * 4 <= LDS), "the second group's sums go through LDS");
};

// part: NULL, or the fp32 sums [gridDim.y][T][np] of launches that cut K into gridDim.y ranges of kb_split steps
template <typename AT, int BN, int BT, int WN, int WT, int KG, int STAGES>
__global__ __launch_bounds__(WN * WT * KG * 64) void fp8_gemm_tiled_kernel(Fp8GemmArgs a, int tiles_n, int tiles_t, int per_xcd,
                                                                           int kb_split, float *part, int64_t np) {
    typedef Fp8Tile<BN, BT, WN, WT, KG, STAGES> C;
    constexpr int NF = C::NF, TF = C::TF;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wave_all % C::WAVES, group = wave_all / C::WAVES;
    unsigned char *const stages = smem + group * STAGES * C::STAGE;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)stages;

    // tile: blocks b, b + 8, ... share an XCD and its L2; each XCD takes a contiguous run of tiles, ordered in columns of
    // 8 row tiles by all token tiles, so that the blocks that run together share operands
    const int tile = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || tile >= tiles_n * tiles_t) return;
    const int col = tile / (8 * tiles_t), in_col = tile - col * 8 * tiles_t;
    const int width = min(8, tiles_n - 8 * col);
    const int n0 = (8 * col + in_col % width) * BN, t0 = in_col / width * BT;
    const int wn = wave / WT, wt = wave % WT;

    // ---- what this lane fetches: row 8 (round * WAVES + wave) + lane / 8, slot lane % 8 of each tile
    // steps of this block: scale blocks [k_begin, k_end) of KB; step st of a group is block kb(st), or nothing behind the end
    const int KB = (a.K + FP8_GROUP - 1) / FP8_GROUP;
    const int k_begin = blockIdx.y * kb_split, k_end = min(KB, k_begin + kb_split), steps = (k_end - k_begin + KG - 1) / KG;
    const int row8 = lane >> 3, piece = (lane & 7) ^ ((((wave & 1) * 8 + row8) >> 1) & 7);
    uint32_t va[C::RA], vb[C::RB];
#pragma unroll
    for (int i = 0; i < C::RA; ++i)   // rows past the end read the last one; their sums are not stored
        va[i] = (uint32_t)(min(n0 + 8 * (i * C::WAVES + wave) + row8, a.N - 1) - n0) * (uint32_t)a.w_stride + piece * 16 + 16;
#pragma unroll
    for (int i = 0; i < C::RB; ++i)
        vb[i] = (uint32_t)(min(t0 + 8 * (i * C::WAVES + wave) + row8, a.T - 1) - t0) * (uint32_t)a.q_stride + piece * 16 + 16;
    // (the offsets are unsigned and the last step takes up to 16 p + 12 off them: bases 16 lower, offsets 16 higher)
    const uint8_t *wbase = static_cast<const uint8_t *>(a.w) + (int64_t)n0 * a.w_stride - 16;
    const uint8_t *xbase = static_cast<const uint8_t *>(a.q) + (int64_t)t0 * a.q_stride - 16;
    // scales: the first BT / 64 waves fetch the tokens', the others (all the same) the row blocks'
    const bool xw = wave < BT / 64;
    const int nb0 = n0 / FP8_GROUP, nbs = (a.N + FP8_GROUP - 1) / FP8_GROUP;
    const uint32_t vs = xw ? (uint32_t)(min(t0 + wave * 64 + lane, a.T - 1) - t0) * (uint32_t)a.xs_token * 4
                           : (uint32_t)(min(nb0 + lane % (BN > 128 ? BN / 128 : 1), nbs - 1) - nb0) * (uint32_t)a.ws_stride * 4;
    const float *sbase = xw ? a.xs + (int64_t)t0 * a.xs_token : a.ws + (int64_t)nb0 * a.ws_stride;
    const int64_t sstep = xw ? a.xs_group : 1;
    const uint32_t sdst = xw ? C::XS + wave * 256 : C::WS;
    // the last step of a K that is no multiple of 128: a piece that reaches behind the end reads the last 16 features of
    // the row instead; what it holds twice or should not hold at all counts as zero (mask)
    const int tail = a.K % FP8_GROUP;
    const uint32_t back = tail && piece * 16 + 16 > tail ? piece * 16 + 16 - tail : 0;

    // The XCDs start in different parts of K: rows of weights are often a power of two apart, and reading the same columns all
    // at once they would meet in the same memory channels (64 tokens of 28672 x 4096 31.2 -> 25.8 us, 128 tokens 38.5 -> 33.6).
    // Not where the last step is a special one.
    const int first = tail || (k_end - k_begin) % KG ? 0 : (int)(blockIdx.x & 7) * steps / 8;
    auto block_of = [&](int st) {
        const int from = st + first;
        return k_begin + (from < steps ? from : from - steps) * KG + group;
    };
    // DMA instruction m of the stage of step st
    auto fetch = [&](int st, int m) {
        const uint32_t dst = lds0 + (st % STAGES) * C::STAGE;
        const int kb = min(block_of(st), k_end - 1);
        if (m < C::RA) dma16(dst + (m * C::WAVES + wave) * 1024, va[m], wbase + (int64_t)kb * FP8_GROUP);
        else if (m < C::RA + C::RB)
            dma16(dst + BN * 128 + ((m - C::RA) * C::WAVES + wave) * 1024, vb[m - C::RA], xbase + (int64_t)kb * FP8_GROUP);
        else dma4(dst + sdst, vs, sbase + kb * sstep);
    };
    // In front of the first DMA instruction of step st's weights (tokens); no branch: sums would sink past it
    auto fetch_last = [&](int st, bool weights, bool tokens) {
        const uint32_t less = min(block_of(st), k_end - 1) == KB - 1 ? back : 0;
#pragma unroll
        for (int i = 0; i < C::RA; ++i) va[i] -= weights ? less : 0;
#pragma unroll
        for (int i = 0; i < C::RB; ++i) vb[i] -= tokens ? less : 0;
    };

    f32x4 acc[NF][TF];
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < TF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // a lane's two pieces of a fragment row: c and 4 + c, at the same place in every fragment
    const uint32_t p0 = r * 128 + ((c ^ (r >> 1)) & 7) * 16, p1 = r * 128 + (((4 + c) ^ (r >> 1)) & 7) * 16;
    const int arow = wn * (BN / WN), brow = wt * (BT / WT);

    // ---- the pipeline.  In step st the tile's last two weight fragments are multiplied BEHIND the barrier that ends
    // the reading of its stage (at SYNC): all of a wave's operands for them are in registers by then, so the matrix unit has
    // work while the next step's first fragments are read (at a barrier between the steps every wave would wait for LDS at
    // once).  Behind that barrier the stage is free for step st + STAGES.
    // The tokens' part of it has been read long before: with two stages a second barrier at the head of the step (EARLY) gives
    // its DMA most of a step more.  The DMA instructions go out one per matrix instruction: a CU's memory path takes 64 bytes
    // a cycle, so issued all together they would hold up every wave.
    // The sums run DEPTH matrix instructions behind their products, across the steps.  The scheduling barriers keep this order.
    constexpr int DEPTH = 2, COUNT = NF * TF, SYNC = COUNT - 2 * TF;
    constexpr bool EARLY = STAGES == 2 && TF + C::RB < SYNC;
    constexpr int NEWER = (STAGES - 2) * C::LOADS + (EARLY ? C::RB + 1 : 0);   // DMA instructions that are younger than step st + 1's at SYNC
    i32x8 wv[2], xv[TF];
    float s[TF], s_last[DEPTH], xs_next[TF], ws_next;
    f32x4 p[DEPTH];
    auto wfrag = [&](int st, int i) {
        const unsigned char *f = stages + (st % STAGES) * C::STAGE + arow * 128 + i * 2048;
        return join(*reinterpret_cast<const u32x4 *>(f + p0), *reinterpret_cast<const u32x4 *>(f + p1));
    };
    auto xfrag = [&](int st, int j) {
        const unsigned char *f = stages + (st % STAGES) * C::STAGE + (BN + brow) * 128 + j * 2048;
        return join(*reinterpret_cast<const u32x4 *>(f + p0), *reinterpret_cast<const u32x4 *>(f + p1));
    };
    auto mask = [&](int st) {                   // behind the end of K the token fragments count as zero
        const int kb = block_of(st), end = kb >= k_end ? 0 : kb == KB - 1 && tail ? tail : FP8_GROUP;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int keep = 4 * (e & 3) >= (e < 4 ? 16 * c : 64 + 16 * c) + 16 - end ? -1 : 0;   // (K is a multiple of 4)
#pragma unroll
            for (int j = 0; j < TF; ++j) xv[j][e] &= keep;
        }
    };
    auto scales = [&](int st) {
        const unsigned char *f = stages + (st % STAGES) * C::STAGE;
#pragma unroll
        for (int j = 0; j < TF; ++j) xs_next[j] = reinterpret_cast<const float *>(f + C::XS)[brow + 16 * j + r];
        ws_next = reinterpret_cast<const float *>(f + C::WS)[BN > 128 ? arow / 128 : 0];
    };
    enum { MAIN, DRAIN, LAST };     // DRAIN: nothing to fetch any more; LAST: no next step either
    auto step = [&](int st, auto mode_t) {
        constexpr int mode = decltype(mode_t)::value;
#pragma unroll
        for (int k = 0; k < COUNT; ++k) {
            const int i = k / TF, j = k % TF;
            if (EARLY && k == TF && mode == MAIN) {     // every wave has its token fragments and scales
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                fetch_last(st + STAGES, false, true);
            }
            if (k == SYNC && mode != LAST) {
                // the next stage has landed (later ones may be on their way) and this wave has read all of the present one
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(mode == DRAIN ? 0 : NEWER) : "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (mode == MAIN) fetch_last(st + STAGES, true, !EARLY);
            }
            if (k == 0) {
#pragma unroll
                for (int e = 0; e < TF; ++e) s[e] = xs_next[e] * ws_next;
                if (KG > 1 && mode == LAST) {               // (no 0 x infinity where the second group has no block left)
                    const bool has = block_of(st) < k_end;
#pragma unroll
                    for (int e = 0; e < TF; ++e) s[e] = has ? s[e] : 0.f;
                }
            }
            p[k % DEPTH] = [&] {
                const f32x4 prev = p[k % DEPTH];
                const f32x4 next = mfma_block(wv[i & 1], xv[j]);
                const int kp = (k + COUNT - DEPTH) % COUNT;   // the product that is summed now
                const float sc = k < DEPTH ? s_last[k] : s[kp % TF];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[kp / TF][kp % TF][e] = __builtin_fmaf(sc, prev[e], acc[kp / TF][kp % TF][e]);
                return next;
            }();
            if (k == COUNT - 1) {
#pragma unroll
                for (int e = 0; e < DEPTH; ++e) s_last[e] = s[(COUNT - DEPTH + e) % TF];
            }
            if (j == TF - 1 && i + 2 < NF) wv[i & 1] = wfrag(st, i + 2);
            if (mode != LAST) {
                if (k == SYNC + TF - 1) wv[0] = wfrag(st + 1, 0);
                if (k >= SYNC + TF) xv[j] = xfrag(st + 1, j);
                if (k == COUNT - 1) {
                    wv[1] = wfrag(st + 1, 1);
                    scales(st + 1);
                }
            }
            if (mode == MAIN) {
                constexpr int BEHIND = EARLY ? C::RA : C::LOADS;      // instructions behind SYNC, spread over the rest of the step
#pragma unroll
                for (int m = 0; m < C::LOADS; ++m)
                    if (k == (EARLY && m >= C::RA ? TF + m - C::RA : SYNC + m * 2 * TF / BEHIND)) fetch(st + STAGES, m);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (mode != LAST && mode != MAIN) mask(st + 1);
    };
    static_assert(NF % 2 == 0 && NF >= 2, "");

#pragma unroll
    for (int k = 0; k < STAGES; ++k)
        if (k < steps) {
            fetch_last(k, true, true);
#pragma unroll
            for (int m = 0; m < C::LOADS; ++m) fetch(k, m);
        }
    if (steps >= STAGES) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * C::LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    wv[0] = wfrag(0, 0);
    wv[1] = wfrag(0, 1);
#pragma unroll
    for (int j = 0; j < TF; ++j) xv[j] = xfrag(0, j);
    scales(0);
    mask(0);
#pragma unroll
    for (int e = 0; e < DEPTH; ++e) {
        p[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        s_last[e] = 0.f;
    }
    int st = 0;
    for (; st + STAGES < steps; ++st) step(st, std::integral_constant<int, MAIN>{});
    for (; st < steps - 1; ++st) step(st, std::integral_constant<int, DRAIN>{});
    step(st, std::integral_constant<int, LAST>{});
#pragma unroll
    for (int e = 0; e < DEPTH; ++e) {
        const int kp = COUNT - DEPTH + e;
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[kp / TF][kp % TF][x] = __builtin_fmaf(s_last[e], p[e][x], acc[kp / TF][kp % TF][x]);
    }

    // (the sums stay in front of the stores' branches: sunk behind them the products would have to be kept)
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < TF; ++j) asm volatile("" : "+v"(acc[i][j]));

    if constexpr (KG > 1) {           // the groups' sums, added in group order
        f32x4 *sums = reinterpret_cast<f32x4 *>(smem) + wave * COUNT * 64 + lane;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();              // every wave has read its last stage
        if (group) {
#pragma unroll
            for (int i = 0; i < NF; ++i)
#pragma unroll
                for (int j = 0; j < TF; ++j) sums[(i * TF + j) * 64] = acc[i][j];
        }
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int j = 0; j < TF; ++j) acc[i][j] += sums[(i * TF + j) * 64];
    }
    const int nw = n0 + arow;
    if (part) {
#pragma unroll
        for (int j = 0; j < TF; ++j) {
            const int t = t0 + brow + 16 * j + r;
            if (t >= a.T) continue;
            float *row = part + ((int64_t)blockIdx.y * a.T + t) * np;
#pragma unroll
            for (int i = 0; i < NF; ++i)
                if (nw + 16 * i + 4 * c < np) *reinterpret_cast<f32x4 *>(row + nw + 16 * i + 4 * c) = acc[i][j];
        }
        return;
    }

    // ---- a lane holds 4 consecutive features of one token per fragment.  Where the wave's rows are all there and y takes
    // 16-byte stores, neighbouring lane rows swap halves of two fragments: a lane then holds 8 consecutive features and a
    // store covers 64 contiguous bytes of 16 tokens, else 4 and 32
    const uint16_t *bias = static_cast<const uint16_t *>(a.bias);
    const bool wide = nw + BN / WN <= a.N && a.y_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
    if (bias) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float b = Act<AT>::to_f32(bias[min(nw + 16 * i + 4 * c + e, a.N - 1)]);
#pragma unroll
                for (int j = 0; j < TF; ++j) acc[i][j][e] += b;
            }
    }
#pragma unroll
    for (int j = 0; j < TF; ++j) {
        const int t = t0 + brow + 16 * j + r;
        uint16_t *y = static_cast<uint16_t *>(a.y) + (int64_t)t * a.y_stride + nw;
        if (wide) {
            uint16_t *yl = y + 16 * (c & 1) + 8 * (c >> 1);
#pragma unroll
            for (int i = 0; i < NF; i += 2) {
                const f32x4 &u = acc[i][j], &v = acc[i + 1][j];
                const auto lo = __builtin_amdgcn_permlane16_swap(Act<AT>::pack2(u[0], u[1]), Act<AT>::pack2(v[0], v[1]), false, false);
                const auto hi = __builtin_amdgcn_permlane16_swap(Act<AT>::pack2(u[2], u[3]), Act<AT>::pack2(v[2], v[3]), false, false);
                if (t < a.T) *reinterpret_cast<u32x4 *>(yl + 16 * i) = u32x4{lo[0], hi[0], lo[1], hi[1]};
            }
        } else if (t < a.T) {
#pragma unroll
            for (int i = 0; i < NF; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (nw + 16 * i + 4 * c + e < a.N) y[16 * i + 4 * c + e] = Act<AT>::from_f32(acc[i][j][e]);
        }
    }
}

template <typename AT, int BN, int BT, int WN, int WT, int KG, int STAGES>
static hipError_t tiled_at(const Fp8GemmArgs &a, int split, hipStream_t stream) {
    typedef Fp8Tile<BN, BT, WN, WT, KG, STAGES> C;
    auto kern = fp8_gemm_tiled_kernel<AT, BN, BT, WN, WT, KG, STAGES>;
    static std::atomic<uint64_t> ready{0};   // one bit per device: the attribute is set once
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
        if (e != hipSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    const int tn = (a.N + BN - 1) / BN, tt = (a.T + BT - 1) / BT, kb = (a.K + FP8_GROUP - 1) / FP8_GROUP;
    const int64_t tiles = (int64_t)tn * tt, per_xcd = (tiles + 7) / 8, np = ((int64_t)a.N + 3) / 4 * 4;
    const int kb_split = (kb + split - 1) / split;
    split = (kb + kb_split - 1) / kb_split;   // no empty range
    float *part = split > 1 ? static_cast<float *>(a.tmp) : nullptr;
    hipLaunchKernelGGL(kern, dim3((unsigned)(per_xcd * 8), (unsigned)split), dim3(C::THREADS), C::LDS, stream, a, tn, tt, (int)per_xcd,
                       kb_split, part, np);
    e = hipGetLastError();
    return e != hipSuccess || !part ? e : launch_fp8_join(a, part, split, np, stream);
}

bool fp8_gemm_tiled_supported(const Fp8GemmArgs &a) {
    // the DMA reads dwords; 32-bit offsets inside a tile of up to 256 rows; tile numbers in 31 bits
    return a.K >= 16 && a.K % 4 == 0 && a.q_stride % 4 == 0 && a.w_stride % 4 == 0 &&
           !((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.w)) & 3) && a.q_stride < (1 << 23) &&
           a.w_stride < (1 << 23) && a.xs_token < (1 << 21) && a.ws_stride < (1 << 21) &&
           (int64_t)((a.N + 63) / 64) * ((a.T + 63) / 64) < (1 << 28);
}

// Tile shape and number of K ranges.  A launch lasts about  base + rounds * (round + steps * step)  us, rounds of 256 blocks
// (a CU holds one).  A step of the only round is longer the more blocks fetch weights of their own (load: the memory's latency
// under load is what a block waits for), one of several rounds by `crowd` (clock and caches are shared by work at full rate).
// K ranges make more blocks of fewer steps and cost a second launch and the partial sums' way through memory; and no
// launch beats its weights' bytes.  Fitted to 468 shapes of 20 to 4096 tokens, 512 to 28672 features and 512 to 14336 inputs
// with weights that come from HBM, all tile shapes with 1 to 8 ranges each: 9 % rms from the measurements, the pick on
// average 0.7 % from the best (95 % of the shapes within 4 %, worst 1.29x: 20 tokens, 6144 x 8192).
struct TileShape { int bn, bt; double base, round, step, crowd, load; };
constexpr TileShape TILE_SHAPES[] = {{256, 256, 0.0, 7.0, 1.29, 1.21, 0.21}, {128, 128, 1.5, 3.1, 0.49, 1.18, 0.61},
                                     {128, 64, 1.7, 2.8, 0.343, 1.11, 1.15}, {64, 64, 1.5, 2.45, 0.21, 1.12, 0.93}};
constexpr size_t MAX_PART_BYTES = (size_t)64 << 20;

static Fp8Plan tiled_plan(int T, int N, int K, size_t tmp_bytes) {
    const int kb = (K + FP8_GROUP - 1) / FP8_GROUP;
    const double np = (N + 3) / 4 * 4.0, weights_us = (double)N * K / 5.2e6 + 4.5;
    Fp8Plan best{0, 1, 0};
    double best_us = 1e30;
    for (int i = 0; i < 4; ++i) {
        const TileShape &s = TILE_SHAPES[i];
        const double tiles_t = (T + s.bt - 1) / s.bt, tiles = (double)((N + s.bn - 1) / s.bn) * tiles_t;
        for (int split = 1; split <= 8; split *= 2) {
            const int steps = (kb + split - 1) / split, ranges = (kb + steps - 1) / steps;
            const double part = ranges > 1 ? ranges * (double)T * np * 4 : 0;
            if (ranges > 1 && (steps < 4 || tiles * ranges > 600 || part > (double)tmp_bytes)) break;
            const double rounds = ceil(tiles * ranges / 256);
            const double slower = rounds > 1 ? s.crowd : 1 + s.load * tiles * ranges / 256 / tiles_t;
            double us = s.base + rounds * (s.round + steps * s.step * slower);
            if (us < weights_us) us = weights_us;
            if (ranges > 1) us += 2.9 + 2 * part / 4.6e6;
            if (us < best_us) {
                best_us = us;
                best = Fp8Plan{i, ranges, (size_t)part};
            }
        }
    }
    return best;
}

Fp8Plan fp8_gemm_tiled_plan(int T, int N, int K, size_t tmp_bytes) {
    return tiled_plan(T, N, K, tmp_bytes < MAX_PART_BYTES ? tmp_bytes : MAX_PART_BYTES);
}

template <typename AT>
static hipError_t tiled_dtype(const Fp8GemmArgs &a, hipStream_t stream) {
    const Fp8Plan p = fp8_gemm_tiled_plan(a.T, a.N, a.K, a.tmp ? a.tmp_bytes : 0);
    switch (p.shape) {
    case 0: return tiled_at<AT, 256, 256, 2, 4, 1, 2>(a, p.ranges, stream);
    case 1: return tiled_at<AT, 128, 128, 4, 2, 1, 4>(a, p.ranges, stream);
    case 2: return tiled_at<AT, 128, 64, 2, 2, 2, 3>(a, p.ranges, stream);
    default: return tiled_at<AT, 64, 64, 2, 2, 2, 4>(a, p.ranges, stream);
    }
}

hipError_t launch_fp8_gemm_tiled(const Fp8GemmArgs &a, hipStream_t stream) {
    return a.dtype == PQ_DTYPE_BF16 ? tiled_dtype<bf16_t>(a, stream) : tiled_dtype<fp16_t>(a, stream);
}

}  // namespace pq
