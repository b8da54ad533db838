// tree_tc.cu -- the dense range of tree attention (tree.cu) on the tcgen05
// tensor cores, with fp32 accuracy.
//
// Every fp32 operand x is used as a pair of fp16 values: with a power of two s
// that brings the largest |x| of its group into [2^11, 2^15),
//   hi = fp16(x s),  lo = fp16(x s - hi),
// so that hi + lo keeps 22 bits of x (or 2^-36 of the group's largest value,
// where that is more), and a b is the sum of the products hi hi, lo hi and
// hi lo, each exact in the fp32 accumulator; lo lo (2^-22 of the product) is
// left out.  bf16 pairs would keep 16 bits, a tf32 pair costs twice the tensor
// time.  Groups: a query row; 8 cache rows of K; 8 cache rows of V.
//
// One CTA takes up to 256 query rows of one KV head as two lanes A and B of
// 128 and walks its split of the cache in tiles of 64 rows, each K and V row
// read and split once for both lanes; with at most 128 query rows and several
// tiles both lanes serve the same rows, tile t on lane t & 1 (ALT), and join
// their sums at the end:
//   * loader warps 8-11 bring 8-row chunks in with cp.async (four in flight per
//     warp, 64 KB per SM), split them and write the K-major operand tiles;
//   * warp 12, one thread, issues S = Q K^T (Q pairs stay in TMEM) and, once a
//     lane's weights are in TMEM over its scores, O = P V into the shared O
//     columns, so one lane's softmax runs under the other's products;
//   * warps 0-3 (A) and 4-7 (B), a thread per query row: online softmax, P
//     pairs, and the sum of the tiles' O in fp32 registers: a sum over all
//     tiles in TMEM would add up the tensor core's cut-off bits.
// Every wait is bounded; on a timeout the kernel records an error and leaves.
#include <cuda_fp16.h>
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "tree.cuh"
#include "umma.cuh"

namespace gncx {

constexpr int kTtThreads = 512;
constexpr int kTtLoadWarp = 8, kTtMmaWarp = 12;
// Registers per thread: softmax, loaders, products (whose warpgroup is filled
// up by idle warps); together the 512 x 128 that the block is launched with.
constexpr int kTtSoftmaxRegs = 184, kTtLoadRegs = 96, kTtMmaRegs = 48;
static_assert(2 * kTtSoftmaxRegs + kTtLoadRegs + kTtMmaRegs <= 4 * 128, "a split that can be had");
constexpr int kTtKStride = 64 * 16 + 16;  // bytes between 8-column chunks of the K tile: shifted by a bank group
constexpr int kTtStages = 2;              // K and V operand tiles
constexpr int kTtScales = 4;              // tiles whose scales are kept
// Weights are held as 2^(score - reference + kTtShift), with the score at most
// kTtHead above the reference: up to 2^14 in fp16, and 2^-34 of a weight of 1 is
// still seen.
constexpr int kTtShift = 10, kTtHead = 4;
// ALT from so many tiles per CTA.  16 heads, 8 KV heads of 128, 16 nodes: 8192
// rows (7 tiles) 28.5 us with both lanes, 30.5 with one; 32 heads, 32 nodes, 32768
// rows (28 tiles) 80.4 and 90; with 4 tiles the joining costs as much as it saves
// (32 heads, 24 nodes, 4096 rows: 24.3 and 23.8).
constexpr int kTtAltTiles = 6;
// TMEM columns
constexpr int kTtQ = 0, kTtS = 256, kTtO = 384, kTtCols = 512;

template <int HD>
struct TtLayout {
    static constexpr int kPart = HD / 8 * kTtKStride;  // one of K hi, K lo, V hi, V lo
    static constexpr int kStage = 4 * kPart;
    static constexpr int kChunk = 8 * HD * 4;
    static constexpr int oStaging = kTtStages * kStage;
    static constexpr int oScale = oStaging + 16 * kChunk;     // int [kTtScales][2][8]
    static constexpr int oBar = oScale + kTtScales * 2 * 8 * 4;
    static constexpr int kBars = 4 * kTtStages + 2 + 6 + 2;
    static constexpr int oState = oBar + kBars * 8;    // lane 1's reference and sum of each row: float [2][128]
    static constexpr int kBytes = oState + 2 * 128 * 4;
    static_assert(kStage >= 128 * HD * 4, "a lane's output fits an operand stage");
    // more than half of an SM's shared memory, so one CTA per SM owns all of TMEM
    static constexpr int kAlloc = kBytes > 120 * 1024 ? kBytes : 120 * 1024;
};

__device__ __forceinline__ void cp_async16_row(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}
// The first `bytes` of 16, zeros behind them.
__device__ __forceinline__ void cp_async16_row(void* smem, const void* gmem, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(bytes) : "memory");
}

__device__ __forceinline__ float pow2i(int n) { return __int_as_float((n + 127) << 23); }  // -126 <= n <= 127

// Exponent s with max * 2^s in [2^11, 2^15) for the largest magnitude `max`
// (its bits), a multiple of 4 up to 124.
__device__ __forceinline__ int scale_exp(uint32_t bits) {
    const int s = 14 - ((int)(bits >> 23) - 127);
    return min(s & ~3, 124);
}

// A pair of fp32 values in one 64-bit register, and two operations at once on it.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// hi = fp16(x), lo = fp16(x - hi) of two values
__device__ __forceinline__ void split2(f32x2 x, uint32_t& hi, uint32_t& lo) {
    const float2 v = unpack2(x);
    const __half2 h = __floats2half2_rn(v.x, v.y);
    const float2 f = __half22float2(h);
    const float2 r = unpack2(fma2(pack2(f.x, f.y), pack2(-1.0f, -1.0f), x));
    const __half2 l = __floats2half2_rn(r.x, r.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Bits of the largest finite magnitude of the warp's values; inf(i) is called
// for an infinite x[i].
template <int N, class Inf>
__device__ __forceinline__ uint32_t warp_max_bits(float (&x)[N], Inf inf) {
    float m = 0.0f, m1 = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        m = fmaxf(m, fmaxf(fabsf(x[i]), fabsf(x[i + 1])));
        m1 = fmaxf(m1, fmaxf(fabsf(x[i + 2]), fabsf(x[i + 3])));
    }
    m = fmaxf(m, m1);
    uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    if (b == 0x7F800000u) {
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (fabsf(x[i]) == INFINITY) inf(i);
            else m = fmaxf(m, fabsf(x[i]));
        }
        b = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    }
    return b;
}

// ALT: at most 128 query rows, both lanes on them, tile t on lane t & 1.
template <int HD, bool ALT>
__global__ void __launch_bounds__(kTtThreads, 1) tree_tc_kernel(const TreeArgs a) {
    using L = TtLayout<HD>;
    extern __shared__ __align__(128) uint8_t sm[];
    int* scales = reinterpret_cast<int*>(sm + L::oScale);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + L::oBar);
    uint64_t* kempty = kfull + kTtStages;
    uint64_t* vfull = kempty + kTtStages;
    uint64_t* vempty = vfull + kTtStages;
    uint64_t* sfull = vempty + kTtStages;  // [lane]
    uint64_t* pfull = sfull + 2;
    uint64_t* ofull = pfull + 2;
    uint64_t* oempty = ofull + 2;
    uint64_t* qfull = oempty + 1;
    uint64_t* joined = qfull + 1;
    uint64_t* done = joined + 1;
    __shared__ uint32_t tmem_slot;
    // columns of V with an infinity, positive and negative ones: left out of the
    // products, where its lo part and a zero weight would make it a NaN, and set
    // in the records
    __shared__ unsigned infinite[2][HD / 32];
    __shared__ int any_infinite;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, kvh = blockIdx.y, r0 = blockIdx.z * kTcTreeRows;
    const int rows = a.n_tok * a.G;
    const int nl = !ALT && rows - r0 > 128 ? 2 : 1;  // row blocks of 128
    const int j0 = a.lo + split * a.per, j1 = min(a.pos0, j0 + a.per);
    const int n_tiles = (j1 - j0 + kTcTreeKeys - 1) / kTcTreeKeys;
    auto phase = [](int t) { return (uint32_t)(ALT ? t >> 1 : t) & 1; };  // of a lane's barriers

    if (tid == 0) {
        for (int i = 0; i < kTtStages; ++i) {
            mbar_init(&kfull[i], 4);
            mbar_init(&kempty[i], 1);
            mbar_init(&vfull[i], 4);
            mbar_init(&vempty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sfull[i], 2);
            mbar_init(&pfull[i], 128);
            mbar_init(&ofull[i], 1);
        }
        mbar_init(oempty, 128);
        mbar_init(qfull, 128 * nl);
        mbar_init(joined, 128);
        mbar_init(done, 1);
        any_infinite = 0;
        fence_barrier_init();
    }
    if (tid < HD / 16) infinite[0][tid] = 0;
    if (warp == kTtMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(kTtCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();
    pdl_launch_dependents();  // after the wait: the second kernel reads inputs before it waits for this one
    constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's, so they start at 0
    // False when a wait ran out: the role leaves its loop, and the roles that wait for it run out too.
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
        const bool ok = mbar_wait(bar, parity);
        if (!ok) record_error(a.err, kErrTimeout);
        return __all_sync(0xffffffffu, ok) != 0;
    };
    // Several barriers, asked at once; the slow path one by one.
    auto wait_all3 = [&](uint64_t* b0, uint32_t p0, uint64_t* b1, uint32_t p1, uint64_t* b2, uint32_t p2) {
        const bool r0 = mbar_test(b0, p0), r1 = mbar_test(b1, p1), r2 = mbar_test(b2, p2);
        if (__all_sync(0xffffffffu, r0 && r1 && r2)) return true;
        return wait_warp(b0, p0) && wait_warp(b1, p1) && wait_warp(b2, p2);
    };

    if (warp >= kTtMmaWarp) {
        regs_dec<kTtMmaRegs>();
        if (warp == kTtMmaWarp) {
            // ---------------- products: the warp waits, one thread issues ----------------
            constexpr uint32_t idesc_s = umma_idesc_f16(128, kTcTreeKeys), idesc_o = umma_idesc_f16(128, HD) | kUmmaTransB;
            const uint32_t sbase = smem_u32(sm);
            auto scores = [&](int x, int t) {  // S_x = Q_x K(t)^T
                const uint32_t hi = umma_desc_lo(sbase + (t & 1) * L::kStage, kTtKStride), lo = hi + (L::kPart >> 4);
                const uint32_t q = tmem + kTtQ + (ALT ? 0 : x * 128), d = tmem + kTtS + x * 64;
                constexpr uint32_t step = 2 * kTtKStride >> 4, rest = umma_desc_hi(128);
                if (elect_one()) {
                    mbar_arrive(&sfull[x]);  // orders the loaders' scales before the lane's reads
                    umma_f16_ts<false>(d, q + HD / 2, hi, rest, idesc_s);
#pragma unroll
                    for (int i = 1; i < HD / 16; ++i) umma_f16_ts<true>(d, q + HD / 2 + 8 * i, hi + i * step, rest, idesc_s);
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) umma_f16_ts<true>(d, q + 8 * i, lo + i * step, rest, idesc_s);
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) umma_f16_ts<true>(d, q + 8 * i, hi + i * step, rest, idesc_s);
                    umma_commit(&sfull[x]);
                }
                __syncwarp();
            };
            auto values = [&](int x, int t) {  // O = P_x V(t)
                // V's rows are the reduction here: 8 x 16-byte core matrices as K's, transposed
                const uint32_t hi = umma_desc_lo(sbase + (t & 1) * L::kStage + 2 * L::kPart, 128), lo = hi + (L::kPart >> 4);
                const uint32_t p = tmem + kTtS + x * 64, d = tmem + kTtO;
                constexpr uint32_t step = 16 * 16 >> 4, rest = umma_desc_hi(kTtKStride);
                // P's block of 16 rows i: columns 16 i .. + 7 hold the hi parts, + 8 .. + 15 the lo parts
                if (elect_one()) {
                    umma_f16_ts<false>(d, p + 8, hi, rest, idesc_o);
#pragma unroll
                    for (int i = 1; i < 4; ++i) umma_f16_ts<true>(d, p + 16 * i + 8, hi + i * step, rest, idesc_o);
#pragma unroll
                    for (int i = 0; i < 4; ++i) umma_f16_ts<true>(d, p + 16 * i, lo + i * step, rest, idesc_o);
#pragma unroll
                    for (int i = 0; i < 4; ++i) umma_f16_ts<true>(d, p + 16 * i, hi + i * step, rest, idesc_o);
                    umma_commit(&ofull[x]);
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (elect_one()) umma_commit(bar);
                __syncwarp();
            };
            constexpr int kAhead = ALT ? 2 : 1;  // a lane's next tile
            bool ok = wait_warp(qfull, 0);
            for (int t = 0; ok && t < min(kAhead, n_tiles); ++t) {
                ok = wait_warp(&kfull[t], 0);
                if (!ok) break;
                tc_fence_after();
                for (int x = 0; x < nl; ++x) scores(ALT ? t : x, t);
                commit(&kempty[t]);
            }
            int n_o = 0;                    // products into O so far
            for (int t = 0; ok && t < n_tiles; ++t)
                for (int i = 0; ok && i < nl; ++i) {
                    const int x = ALT ? t & 1 : i;
                    // before the first product into O, oempty's phase "before 0" counts as complete
                    ok = wait_all3(&pfull[x], phase(t), &vfull[t & 1], (t >> 1) & 1, oempty, (n_o - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    values(x, t);
                    ++n_o;
                    if (i == nl - 1) commit(&vempty[t & 1]);
                    const int t2 = t + kAhead;
                    if (t2 < n_tiles) {
                        if (i == 0) ok = wait_warp(&kfull[t2 & 1], (t2 >> 1) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        scores(x, t2);
                        if (i == nl - 1) commit(&kempty[t2 & 1]);
                    }
                }
            commit(done);  // nothing of this CTA's is in flight when TMEM is freed
            if (!mbar_wait(done, 0)) record_error(a.err, kErrTimeout);
        }
    } else if (warp >= kTtLoadWarp) {
        // ---------------- loaders: warp w takes rows 16 w .. 16 w + 15 of each tile ----------------
        regs_dec<kTtLoadRegs>();
        const int lw = warp - kTtLoadWarp;
        const size_t pstride = (size_t)a.n_kv * a.hd;
        const float* src[2] = {a.kc + (size_t)kvh * a.hd, a.vc + (size_t)kvh * a.hd};
        uint8_t* staging = sm + L::oStaging + lw * 4 * L::kChunk;
        // chunk i of tile t: K rows 0-7, 8-15, V rows 0-7, 8-15 of the warp's 16;
        // float4 c of a row per lane, rows sub, sub + RS, ..
        constexpr int LPR = HD / 4, RS = 32 / LPR;
        const int c = lane % LPR, sub = lane / LPR;
        auto row_of = [&](int t, int i) { return j0 + kTcTreeKeys * t + 16 * lw + 8 * (i & 1); };
        auto issue = [&](int t, int i) {
            const int row = row_of(t, i) + sub;
            const float* g = src[i >> 1] + (size_t)row * pstride + 4 * c;
            float* d = reinterpret_cast<float*>(staging + i * L::kChunk) + sub * HD + 4 * c;
            if (t < n_tiles && row_of(t, i) + 8 <= j1 && 4 * c < a.hd) {
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) cp_async16_row(d + RS * k * HD, g + (size_t)(RS * k) * pstride);
            } else if (t < n_tiles) {  // zeros past the last row and column
#pragma unroll 1
                for (int k = 0; k < HD / 16; ++k) {
                    const bool some = row + RS * k < j1 && 4 * c < a.hd;
                    cp_async16_row(d + RS * k * HD, some ? g + (size_t)(RS * k) * pstride : src[0], some ? 16 : 0);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = 0; i < 4; ++i) issue(0, i);
        bool ok = true;
        for (int t = 0; t < n_tiles && ok; ++t) {
            uint8_t* tile = sm + (t & 1) * L::kStage;
            int* sc = scales + (t & (kTtScales - 1)) * 16;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                asm volatile("cp.async.wait_group 3;" ::: "memory");
                __syncwarp();
                const float* st = reinterpret_cast<const float*>(staging + i * L::kChunk);
                const int chunk = 2 * lw + (i & 1);
                float x[HD / 4];
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const float4 v = *reinterpret_cast<const float4*>(st + (sub + RS * k) * HD + 4 * c);
                    x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w;
                }
                const int s = scale_exp(warp_max_bits(x, [&](int e) {
                    if (i < 2) return;
                    const int col = 4 * c + (e & 3);
                    atomicOr(&infinite[x[e] < 0.0f][col >> 5], 1u << (col & 31));
                    any_infinite = 1;
                    x[e] = 0.0f;
                }));
                issue(t + 1, i);  // the chunk is in registers
                const f32x2 f = pack2(pow2i(s), pow2i(s));
                if ((i & 1) == 0 && t >= kTtStages) ok = wait_warp(i ? &vempty[t & 1] : &kempty[t & 1], ((t >> 1) - 1) & 1);
                if (!ok) break;
                uint8_t* d = tile + (i >> 1) * 2 * L::kPart + (c >> 1) * kTtKStride + (8 * chunk + sub) * 16 + (c & 1) * 8;
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    uint2 hi, lo;
                    split2(mul2(pack2(x[4 * k], x[4 * k + 1]), f), hi.x, lo.x);
                    split2(mul2(pack2(x[4 * k + 2], x[4 * k + 3]), f), hi.y, lo.y);
                    *reinterpret_cast<uint2*>(d + RS * k * 16) = hi;
                    *reinterpret_cast<uint2*>(d + L::kPart + RS * k * 16) = lo;
                }
                if (lane == 0) sc[8 * (i >> 1) + chunk] = s;
                if (i & 1) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(i == 1 ? &kfull[t & 1] : &vfull[t & 1]);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if ((warp >> 2) < nl || ALT) {
        // ---------------- softmax and output: a thread per query row (and lane) ----------------
        regs_inc<kTtSoftmaxRegs>();
        const int x = warp >> 2;
        const int first = r0 + (ALT ? 0 : 128 * x) + 32 * (warp & 3), row = first + lane;
        const bool active = first < rows;  // of the warp
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t tq = tmem + lanes + kTtQ + x * 128, ts = tmem + lanes + kTtS + x * 64, to = tmem + lanes + kTtO;
        int sq = 0;
        if (active) {
            const bool some = row < rows;
            const float* qp = a.q + ((size_t)(some ? row / a.G : 0) * a.n_heads + kvh * a.G + (some ? row % a.G : 0)) * a.hd;
            float v[HD];  // the whole row in flight at once
#pragma unroll
            for (int c = 0; c < HD / 4; ++c) {
                const float4 w = some && 4 * c < a.hd ? *reinterpret_cast<const float4*>(qp + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[4 * c] = w.x; v[4 * c + 1] = w.y; v[4 * c + 2] = w.z; v[4 * c + 3] = w.w;
            }
            float m = 0.0f;
#pragma unroll
            for (int c = 0; c < HD; ++c) m = fmaxf(m, fabsf(v[c]) < INFINITY ? fabsf(v[c]) : 0.0f);
            sq = scale_exp(__float_as_uint(m));
            if (x == 0 || !ALT) {
                const f32x2 f = pack2(pow2i(sq), pow2i(sq));
#pragma unroll
                for (int b = 0; b < HD / 32; ++b) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) split2(mul2(pack2(v[32 * b + 2 * c], v[32 * b + 2 * c + 1]), f), hi[c], lo[c]);
                    tmem_st16(tq + 16 * b, hi);
                    tmem_st16(tq + HD / 2 + 16 * b, lo);
                }
                tmem_wait_st();
            }
        }
        tc_fence_before();
        if (x == 0 || !ALT) mbar_arrive(qfull);

        float T = -INFINITY, l = 0.0f;
        f32x2 o[HD / 2];
#pragma unroll
        for (int d = 0; d < HD / 2; ++d) o[d] = 0;
        bool ok = true;
#pragma unroll 1
        for (int t = ALT ? x : 0; t < n_tiles; t += ALT ? 2 : 1) {
            ok = wait_warp(&sfull[x], phase(t));
            if (!ok) break;
            float alpha = 1.0f, beta = 1.0f;
            if (active) {
                tc_fence_after();
                const int4* sc = reinterpret_cast<const int4*>(scales + (t & (kTtScales - 1)) * 16);
                const int valid = j1 - j0 - kTcTreeKeys * t;
                const int4 k0 = sc[0], k1 = sc[1];
                // 2^(-sq - sk) may need two factors
                auto factor = [&](int sk) {
                    const int n = -sq - sk, h = n >> 1;
                    return a.scale2 * pow2i(h) * pow2i(n - h);
                };
                const bool even_k = k0.x == k0.y && k0.x == k0.z && k0.x == k0.w && k0.x == k1.x && k0.x == k1.y &&
                                    k0.x == k1.z && k0.x == k1.w;
                const float c0 = factor(k0.x);
                float tm = -INFINITY;
                if (even_k && valid >= kTcTreeKeys && c0 >= 0.0f) {
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        float s[32];
                        tmem_ld32f(ts + 32 * h, s);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) tm = fmaxf(tm, fmaxf(s[j], s[j + 1]));
                    }
                    tm *= c0;
                } else {
#pragma unroll 1
                    for (int b = 0; b < 4; ++b) {
                        float s[16];
                        tmem_ld16f(ts + 16 * b, s);
                        const int* sk = reinterpret_cast<const int*>(sc) + 2 * b;
                        const float ca = factor(sk[0]), cb = factor(sk[1]);
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (16 * b + j < valid) tm = fmaxf(tm, s[j] * (j < 8 ? ca : cb));
                    }
                }
                // the reference follows the maximum only when that has grown by more
                // than kTtHead: a rescaling of o for every new maximum would come in
                // most tiles of 32 rows
                if (tm > T + kTtHead || T == -INFINITY) {
                    alpha = T == -INFINITY ? 0.0f : ex2(T - tm);
                    T = tm;
                }
                const float ref = T == -INFINITY ? 0.0f : T;
                // V's scales: the products of this tile count in units of its largest rows
                ok = wait_warp(&vfull[t & 1], (t >> 1) & 1);
                if (!ok) break;
                const int4 v0 = sc[2], v1 = sc[3];
                const int U = min(min(min(v0.x, v0.y), min(v0.z, v0.w)), min(min(v1.x, v1.y), min(v1.z, v1.w)));
                const bool even_v = U == max(max(max(v0.x, v0.y), max(v0.z, v0.w)), max(max(v1.x, v1.y), max(v1.z, v1.w)));
                beta = pow2i(-U);
                const float shift = kTtShift - ref;
                f32x2 sum = 0;
                if (even_k && even_v && valid >= kTcTreeKeys) {
                    const f32x2 c02 = pack2(c0, c0), shift2 = pack2(shift, shift);
#pragma unroll 1
                    for (int b = 0; b < 4; ++b) {
                        float s[16];
                        uint32_t p[16];
                        tmem_ld16f(ts + 16 * b, s);
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const float2 z = unpack2(fma2(pack2(s[j], s[j + 1]), c02, shift2));
                            const f32x2 e = pack2(ex2(z.x), ex2(z.y));
                            sum = add2(sum, e);
                            split2(e, p[j / 2], p[8 + j / 2]);
                        }
                        tmem_st16(ts + 16 * b, p);
                    }
                } else {
#pragma unroll 1
                    for (int b = 0; b < 4; ++b) {
                        float s[16];
                        uint32_t p[16];
                        tmem_ld16f(ts + 16 * b, s);
                        const int* sk = reinterpret_cast<const int*>(sc) + 2 * b;
                        const float ca = factor(sk[0]), cb = factor(sk[1]);
                        const float wa = pow2i(max(-126, U - sk[8])), wb = pow2i(max(-126, U - sk[9]));
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const float c = j < 8 ? ca : cb, w = j < 8 ? wa : wb;
                            const float e0 = 16 * b + j < valid ? ex2(fmaf(s[j], c, shift)) : 0.0f;
                            const float e1 = 16 * b + j + 1 < valid ? ex2(fmaf(s[j + 1], c, shift)) : 0.0f;
                            sum = add2(sum, pack2(e0, e1));
                            split2(pack2(e0 * w, e1 * w), p[j / 2], p[8 + j / 2]);
                        }
                        tmem_st16(ts + 16 * b, p);
                    }
                }
                const float2 parts = unpack2(sum);
                l = fmaf(l, alpha, parts.x + parts.y);
                tmem_wait_st();
                tc_fence_before();
            }
            mbar_arrive(&pfull[x]);
            ok = wait_warp(&ofull[x], phase(t));
            if (!ok) break;
            if (active) {
                tc_fence_after();
                const f32x2 beta2 = pack2(beta, beta);
                if (__any_sync(0xffffffffu, alpha != 1.0f)) {
                    const f32x2 alpha2 = pack2(alpha, alpha);
#pragma unroll
                    for (int d = 0; d < HD / 2; ++d) o[d] = mul2(o[d], alpha2);
                }
#pragma unroll
                for (int b = 0; b < HD / 32; ++b) {
                    float v[32];
                    tmem_ld32f(to + 32 * b, v);
#pragma unroll
                    for (int d = 0; d < 32; d += 2) o[16 * b + d / 2] = fma2(pack2(v[d], v[d + 1]), beta2, o[16 * b + d / 2]);
                }
                tc_fence_before();
            }
            mbar_arrive(oempty);
        }
        if (ALT && ok) {
            // lane 1's state of each row joins lane 0's, its output through the second
            // operand stage: the odd tiles', whose products are through
            float* other = reinterpret_cast<float*>(sm + L::kStage) + 32 * (warp & 3) + lane;
            float* state = reinterpret_cast<float*>(sm + L::oState) + 32 * (warp & 3) + lane;
            if (x == 1) {
                if (active) {
                    state[0] = T;
                    state[128] = l;
#pragma unroll
                    for (int d = 0; d < HD / 2; ++d) {
                        const float2 v = unpack2(o[d]);
                        other[2 * d * 128] = v.x;
                        other[(2 * d + 1) * 128] = v.y;
                    }
                }
                mbar_arrive(joined);
            } else {
                ok = wait_warp(joined, 0);
                if (active && ok) {
                    const float T1 = state[0], Tn = fmaxf(T, T1);
                    const float f = T == -INFINITY ? 0.0f : ex2(T - Tn), g = T1 == -INFINITY ? 0.0f : ex2(T1 - Tn);
                    T = Tn;
                    l = fmaf(l, f, state[128] * g);
                    const f32x2 f2 = pack2(f, f), g2 = pack2(g, g);
#pragma unroll
                    for (int d = 0; d < HD / 2; ++d)
                        o[d] = fma2(o[d], f2, mul2(pack2(other[2 * d * 128], other[(2 * d + 1) * 128]), g2));
                }
            }
        }
        if (any_infinite) {
#pragma unroll
            for (int d = 0; d < HD / 2; ++d) {
                auto of = [&](int c) {
                    const float up = infinite[0][c >> 5] >> (c & 31) & 1 ? INFINITY : 0.0f;
                    return infinite[1][c >> 5] >> (c & 31) & 1 ? up - INFINITY : up;
                };
                o[d] = add2(o[d], pack2(of(2 * d), of(2 * d + 1)));
            }
        }
        if (row < rows && !(ALT && x == 1)) {
            float* rec = a.part + (((size_t)kvh * rows + row) * a.splits + split) * (a.hd + 4);
            const float f = pow2i(-kTtShift);
            *reinterpret_cast<float2*>(rec) = make_float2(T, l * f);
#pragma unroll
            for (int d = 0; d < HD; d += 4)
                if (d < a.hd) {
                    const float2 x0 = unpack2(o[d / 2]), x1 = unpack2(o[d / 2 + 1]);
                    *reinterpret_cast<float4*>(rec + 4 + d) = make_float4(x0.x * f, x0.y * f, x1.x * f, x1.y * f);
                }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kTtMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTtCols));
}

bool tree_tc_ok(int hd) { return hd <= 128 && hd % 16 == 0; }

cudaError_t tree_tc_launch(const TreeArgs& a, cudaStream_t st) {
    const dim3 grid(a.splits, a.n_kv, (a.n_tok * a.G + kTcTreeRows - 1) / kTcTreeRows);
    auto go = [&](auto k, size_t smem) {
        const cudaError_t e = set_smem_limit(k, smem);
        if (e != cudaSuccess) return e;
        return launch_after(k, grid, dim3(kTtThreads), smem, st, a);
    };
    const bool alt = a.n_tok * a.G <= 128 && a.per >= kTtAltTiles * kTcTreeKeys;
    if (a.hd <= 64) return alt ? go(tree_tc_kernel<64, true>, TtLayout<64>::kAlloc) : go(tree_tc_kernel<64, false>, TtLayout<64>::kAlloc);
    return alt ? go(tree_tc_kernel<128, true>, TtLayout<128>::kAlloc) : go(tree_tc_kernel<128, false>, TtLayout<128>::kAlloc);
}

}  // namespace gncx
