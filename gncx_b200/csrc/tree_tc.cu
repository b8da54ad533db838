// tree_tc.cu -- the dense range of tree attention (tree.cu) on the tcgen05
// tensor cores, with fp32 accuracy.
//
// Every fp32 operand x is used as a pair of fp16 values: with a power of two s
// that brings the largest |x| of its row into [2^3, 2^15),
//   hi = fp16(x s),  lo = fp16(x s - hi),
// so that hi + lo keeps 22 bits of x (or 2^-25 / s, where that is more: at least 2^-28
// of the row's largest value), and a b is the sum of the products hi hi, lo hi and
// hi lo, each exact in the fp32 accumulator; lo lo (2^-22 of the product) is
// left out.  bf16 pairs would keep 16 bits, a tf32 pair costs twice the tensor
// time.  A query row has a scale of its own; K's rows share one in a CTA, and V's, and
// the rows that it does not suit have scales of their own.  The weights are split in a
// unit that goes by the largest weight times V of the tile.
//
// One CTA takes up to 256 query rows of one KV head as two lanes A and B of
// 128 and walks its split of the cache in tiles of 64 rows, each K and V row
// read and split once for both lanes; with at most 128 query rows and several
// tiles both lanes serve the same rows, tile t on lane t & 1 (ALT), and join
// their sums at the end:
//   * loader warps 8-11 bring chunks of 8 rows in with cp.async (four in flight per
//     warp, 64 KB per SM), split them and write the K-major operand tiles;
//   * warps 13 and 14 give rows of K and V that are small or large by the CTA's scale
//     their own, in the chunks whose loader found a thread without a large value in one
//     of its rows, or with too large a one (hardly any of ordinary data);
//   * warp 12, one thread, issues S = Q K^T (Q pairs stay in TMEM) and, once a
//     lane's weights are in TMEM over its scores, O = P V into the shared O
//     columns, so one lane's softmax runs under the other's products;
//   * warps 0-3 (A) and 4-7 (B), a thread per query row: online softmax, P
//     pairs, and the sum of the tiles' O in fp32 registers: a sum over all
//     tiles in TMEM would add up the tensor core's cut-off bits.
// Head sizes above 128 (WIDE): 128 query rows and tiles of 32 rows, as Q's pairs
// take all of its TMEM columns and a tile as much shared memory; lane A computes
// the weights, and each lane sums half of the output's columns.
// Every wait is bounded; on a timeout the kernel records an error and leaves.
//
// What bounds it: latency, with the tensor pipe, shared memory and the issue slots
// each about half busy.  64 nodes, 32 heads, 8 KV heads of 128, 32768 rows: 114 us
// with the merge (2.4 TB/s; three fp16 products at 910 TFLOP/s, of which the
// pipe alone would need 60 us), tensor pipe 50 % of its cycles, issue 46 %.  1 node:
// 72 to 76 us, 3.6 TB/s.  16 heads, 4 KV heads of 256, 64 nodes, 32768 rows: 152 us
// (tree.cu's CUDA-core kernel: 3799 us).  Where rows need scales of their own the tile
// takes 3 to 4 times as long (all rows of random sizes over 2^12, the first case: 408 to
// 460 us).  Slower, each against the kernel of its day (114 to 118 us): two threads per
// row with 16 softmax warps (128 us for the first case), lanes of different tiles in CTAs
// of 128 rows with 8 loader warps (147 us), Q's lo parts in shared memory for a second S
// buffer (121 us), a weight reference without the pass for the maximum (118 us).
#include <cuda_fp16.h>
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "rows.cuh"
#include "tree.cuh"
#include "umma.cuh"

namespace gncx {

constexpr int kTtThreads = 512;
constexpr int kTtLoadWarp = 8, kTtMmaWarp = 12, kTtSizeWarp = 13;  // and 14
// Registers per thread: softmax, loaders, products (whose warpgroup is filled
// up by the warps of the rows' scales); together at most the 512 x 128 that the block
// is launched with.  64 nodes, 32 heads, 8 KV heads of 128, 32768 rows: 115.0 us; with
// 176, 120 and 40 124.0, with 184, 104 and 40 122.8.  Head size 256 (16 heads, 4 KV heads,
// 64 nodes, 32768 rows): 151.8 us, 148.3 and 157.1.
constexpr int kTtSoftmaxRegs = 176, kTtLoadRegs = 112, kTtMmaRegs = 48;
static_assert(2 * kTtSoftmaxRegs + kTtLoadRegs + kTtMmaRegs <= 4 * 128, "a split that can be had");
constexpr int kTtStages = 2;              // K and V operand tiles
constexpr int kTtScales = 4;              // tiles whose rows' scales are kept
// Weights are 2^(score - reference), with the score at most kTtHead above the
// reference.  A tile's product with V has a unit of its own for each query row: 2^-n
// with the weights times 2^(n - V's scale), the largest of them about 2^kTtTop.  So fp16
// pairs lose nothing of the rows that make up the tile's output, whatever the weights
// and sizes of V's other rows are: what is cut is below 2^-26 of the largest weight
// times V.
constexpr int kTtHead = 4, kTtTop = 14;
// K's rows share one scale in a CTA, and V's, by the largest value of the first chunks;
// a row whose largest value is not in [kTtSmall, kTtLarge) in it has a scale of its
// own.  (Scales by chunks, in steps of 2^4, make the tiles uneven where ordinary values
// lie around a step: 64 nodes over 32768 rows, 32 heads, 8 KV heads of 128, 147 us.)
constexpr float kTtSmall = 8.0f, kTtLarge = 32768.0f;
// ALT from so many tiles per CTA.  16 heads, 8 KV heads of 128, 16 nodes: 8192
// rows (7 tiles) 29.5 us with both lanes, 31.7 with one; 32 heads, 32 nodes, 32768
// rows (28 tiles) 79.2 and 87.5; with 4 tiles the joining costs as much as it saves
// (32 heads, 24 nodes, 4096 rows: 23.3 and 23.2).
constexpr int kTtAltTiles = 6;
// Rows of a warp above which Q and the records go through shared memory, so that a
// load or store touches 8 rows or fewer: 33 nodes, 32 heads, 8 KV heads of 128, 4097
// rows 27.1 us against 28.4 without, 58 nodes, 3 heads, one KV head of 256, 102 rows
// 16.5 against 22.0; with few rows it costs more than it saves (5 nodes, 16 heads, 8
// KV heads, 511 rows: 11.6 against 10.3).
constexpr int kTtTurn = 16;
// TMEM columns: Q pairs, scores, (head sizes above 128: weights), outputs
constexpr int kTtQ = 0, kTtS = 256, kTtP = 320, kTtO = 384, kTtCols = 512;

template <int HD>
struct TtLayout {
    static constexpr int kKeys = tree_tc_keys(HD);
    static constexpr int kRows = kKeys / 8;             // of a chunk: the rows that a loader warp takes at a time
    static constexpr int kStride = kKeys * 16 + 16;     // bytes between 8-column chunks of a tile: shifted by a bank group
    static constexpr int kPart = HD / 8 * kStride;      // one of K hi, K lo, V hi, V lo
    static constexpr int kStage = 4 * kPart;
    static constexpr int kChunk = kRows * HD * 4;
    static constexpr int oStaging = kTtStages * kStage;
    static constexpr int oFlags = oStaging + 16 * kChunk;  // of the chunks: uint8_t [kTtScales][2][8]
    // of the rows, in flagged tiles: int [kTtScales][2][kKeys]; whether any differs from the CTA's: [kTtScales][2]
    static constexpr int oRows = oFlags + kTtScales * 2 * 8;
    static constexpr int oDiffer = oRows + kTtScales * 2 * kKeys * 4;
    static constexpr int oBar = oDiffer + kTtScales * 2 * 4;
    static constexpr int kBars = 6 * kTtStages + 2 + 6 + 2;
    static constexpr int oState = oBar + kBars * 8;    // what the lanes tell each other of each row: float [2][128]
    static constexpr int oTurn = oState + 2 * 128 * 4;  // per softmax warp: 16 columns of its 32 rows of Q
    static constexpr int kTurn = 32 * 20 * 4;
    static constexpr int kBytes = oTurn + 8 * kTurn;
    static_assert(kBytes <= 227 * 1024 - 1024, "shared memory");
    static_assert(HD > 128 || kStage >= 128 * HD * 4, "a lane's output fits an operand stage");
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

// Exponent s with max * 2^s in [2^11, 2^12) for the largest magnitude `max` (its
// bits), up to 124.
__device__ __forceinline__ int scale_exp(uint32_t bits) { return min(11 + 127 - (int)(bits >> 23), 124); }

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

// The largest magnitude of this lane's values; `even` and `odd`: the least of its even
// and odd fours' largest.
template <int N>
__device__ __forceinline__ float lane_max(const float (&x)[N], float& even, float& odd) {
    float m = 0.0f;
    even = odd = INFINITY;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float y = fmaxf(fmaxf(fabsf(x[i]), fabsf(x[i + 1])), fmaxf(fabsf(x[i + 2]), fabsf(x[i + 3])));
        m = fmaxf(m, y);
        (i & 4 ? odd : even) = fminf(i & 4 ? odd : even, y);
    }
    return m;
}

// ALT: at most 128 query rows, both lanes on them, tile t on lane t & 1.
// HD 256 (WIDE): both lanes on 128 rows, lane 0 with columns 0-127 of the output,
// lane 1 with the others.
template <int HD, bool ALT>
__global__ void __launch_bounds__(kTtThreads, 1) tree_tc_kernel(const TreeArgs a) {
    using L = TtLayout<HD>;
    constexpr bool WIDE = HD > 128;
    static_assert(!(WIDE && ALT), "one way to share rows");
    constexpr int KEYS = L::kKeys, CR = L::kRows;
    constexpr int HO = WIDE ? 128 : HD;  // columns of a lane's output
    constexpr bool kShared = ALT || WIDE;  // both lanes on the same rows, S of tile t in block t & 1
    extern __shared__ __align__(128) uint8_t sm[];
    uint8_t* flags = sm + L::oFlags;  // chunks with rows that may need scales of their own
    int* row_scales = reinterpret_cast<int*>(sm + L::oRows);
    int* rows_differ = reinterpret_cast<int*>(sm + L::oDiffer);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + L::oBar);
    uint64_t* kempty = kfull + kTtStages;
    uint64_t* vfull = kempty + kTtStages;
    uint64_t* vempty = vfull + kTtStages;
    uint64_t* ksized = vempty + kTtStages;  // rows have the scales they need
    uint64_t* vsized = ksized + kTtStages;
    uint64_t* sfull = vsized + kTtStages;  // [lane]
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
    __shared__ unsigned first_top[2];  // bits of the largest value of K's and V's first chunks
    __shared__ int cta_scale[2];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, kvh = blockIdx.y, r0 = blockIdx.z * tree_tc_rows(HD);
    const int rows = a.n_tok * a.G;
    const int nl = WIDE || (!ALT && rows - r0 > 128) ? 2 : 1;  // products into O per tile
    const int j0 = a.lo + split * a.per, j1 = min(a.pos0, j0 + a.per);
    const int n_tiles = (j1 - j0 + KEYS - 1) / KEYS;
    auto phase = [](int t) { return (uint32_t)(ALT ? t >> 1 : t) & 1; };        // of a lane's barriers
    auto phase_s = [](int t) { return (uint32_t)(kShared ? t >> 1 : t) & 1; };  // of the scores'

    if (tid == 0) {
        for (int i = 0; i < kTtStages; ++i) {
            mbar_init(&kfull[i], 4);
            mbar_init(&kempty[i], 1);
            mbar_init(&vfull[i], 4);
            mbar_init(&vempty[i], 1);
            mbar_init(&ksized[i], 1);
            mbar_init(&vsized[i], 1);
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
        first_top[0] = first_top[1] = 0;
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
            constexpr uint32_t idesc_s = umma_idesc_f16(128, KEYS), idesc_o = umma_idesc_f16(128, HO) | kUmmaTransB;
            const uint32_t sbase = smem_u32(sm);
            auto scores = [&](int x, int t) {  // S_x = Q_x K(t)^T, or Q K(t)^T
                const uint32_t hi = umma_desc_lo(sbase + (t & 1) * L::kStage, L::kStride), lo = hi + (L::kPart >> 4);
                const uint32_t q = tmem + kTtQ + (kShared ? 0 : x * 128), d = tmem + kTtS + x * KEYS;
                constexpr uint32_t step = 2 * L::kStride >> 4, rest = umma_desc_hi(128);
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
            auto values = [&](int x, int t) {  // O = P_x V(t), or P V(t)'s columns 128 x ..
                // V's rows are the reduction here: 8 x 16-byte core matrices as K's, transposed
                const uint32_t hi = umma_desc_lo(sbase + (t & 1) * L::kStage + 2 * L::kPart + (WIDE ? x * 16 * L::kStride : 0), 128), lo = hi + (L::kPart >> 4);
                const uint32_t p = tmem + (WIDE ? kTtP + (t & 1) * KEYS : kTtS + x * 64), d = tmem + kTtO;
                constexpr uint32_t step = 16 * 16 >> 4, rest = umma_desc_hi(L::kStride);
                // P's block of 16 rows i: columns 16 i .. + 7 hold the hi parts, + 8 .. + 15 the lo parts
                if (elect_one()) {
                    umma_f16_ts<false>(d, p + 8, hi, rest, idesc_o);
#pragma unroll
                    for (int i = 1; i < KEYS / 16; ++i) umma_f16_ts<true>(d, p + 16 * i + 8, hi + i * step, rest, idesc_o);
#pragma unroll
                    for (int i = 0; i < KEYS / 16; ++i) umma_f16_ts<true>(d, p + 16 * i, lo + i * step, rest, idesc_o);
#pragma unroll
                    for (int i = 0; i < KEYS / 16; ++i) umma_f16_ts<true>(d, p + 16 * i, hi + i * step, rest, idesc_o);
                    umma_commit(&ofull[x]);
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (elect_one()) umma_commit(bar);
                __syncwarp();
            };
            constexpr int kAhead = ALT ? 2 : 1;  // the next tile into the same S
            bool ok = wait_warp(qfull, 0);
            for (int t = 0; ok && t < min(kAhead, n_tiles); ++t) {
                ok = wait_warp(&ksized[t], 0);
                if (!ok) break;
                tc_fence_after();
                for (int x = 0; x < (kShared ? 1 : nl); ++x) scores(kShared ? t : x, t);
                commit(&kempty[t]);
            }
            int n_o = 0;                    // products into O so far
            for (int t = 0; ok && t < n_tiles; ++t)
                for (int i = 0; ok && i < nl; ++i) {
                    const int x = ALT ? t & 1 : i;
                    // before the first product into O, oempty's phase "before 0" counts as complete
                    ok = wait_all3(&pfull[x], phase(t), &vsized[t & 1], (t >> 1) & 1, oempty, (n_o - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    values(x, t);
                    ++n_o;
                    if (i == nl - 1) commit(&vempty[t & 1]);
                    const int t2 = t + kAhead;
                    if (t2 < n_tiles && !(WIDE && i == 1)) {  // WIDE: lane 1 was through with tile t2 - 2 before oempty
                        if (i == 0) ok = wait_warp(&ksized[t2 & 1], (t2 >> 1) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        scores(WIDE ? t2 & 1 : x, t2);
                        if (WIDE || i == nl - 1) commit(&kempty[t2 & 1]);
                    }
                }
            commit(done);  // nothing of this CTA's is in flight when TMEM is freed
            if (!mbar_wait(done, 0)) record_error(a.err, kErrTimeout);
        } else if (warp <= kTtSizeWarp + 1) {
            // ---------------- small and large rows of K, of V get scales of their own, in the chunks that are flagged ----------------
            const int kind = warp - kTtSizeWarp;  // 0: K, 1: V
            for (int t = 0; t < n_tiles && wait_warp(kind ? &vfull[t & 1] : &kfull[t & 1], (t >> 1) & 1); ++t) {
                const int slot = 2 * (t & (kTtScales - 1)) + kind;
                const unsigned flagged = __ballot_sync(0xffffffffu, lane < 8 && flags[8 * slot + (lane & 7)]);
                if (flagged) {
                    int* of_row = row_scales + slot * KEYS;
                    for (int j = lane; j < KEYS; j += 32) of_row[j] = cta_scale[kind];
                    __syncwarp();
                    uint8_t* tile = sm + (t & 1) * L::kStage + 2 * kind * L::kPart;
                    bool apart = false;
#pragma unroll 1
                    for (unsigned left = flagged; left; left &= left - 1) {
                        const int c = __ffs(left) - 1;
                        constexpr int G = 32 / CR;  // lanes per row
                        float most = 0.0f;
#pragma unroll 1
                        for (int p = lane % G; p < HD / 8; p += G) {
                            const uint4 h = *reinterpret_cast<const uint4*>(tile + p * L::kStride + (CR * c + lane / G) * 16);
                            auto abs2 = [](uint32_t u) { u &= 0x7FFF7FFFu; return *reinterpret_cast<const __half2*>(&u); };
                            const float2 m = __half22float2(__hmax2(__hmax2(abs2(h.x), abs2(h.y)), __hmax2(abs2(h.z), abs2(h.w))));
                            most = fmaxf(most, fmaxf(m.x, m.y));
                        }
                        const unsigned larges = __ballot_sync(0xffffffffu, most >= kTtSmall);
                        const unsigned too_large = __ballot_sync(0xffffffffu, most >= kTtLarge);
                        unsigned todo = 0;  // the rows to do again
#pragma unroll
                        for (int r = 0; r < CR; ++r) {
                            const unsigned group = ((1u << G) - 1) << r * G;
                            todo |= (unsigned)(!(larges & group) || (too_large & group)) << r;
                        }
                        apart |= todo != 0;
                        constexpr int B = HD > 128 ? 2 : 4, NC = (HD + 127) / 128;  // rows at a time, float4s of a lane
#pragma unroll 1
                        while (todo) {
                            int r[B];
                            float4 y[B][NC];
#pragma unroll
                            for (int b = 0; b < B; ++b) {
                                r[b] = CR * c + __ffs(todo) - 1;
                                const bool some = todo != 0;
                                todo &= todo - 1;
#pragma unroll
                                for (int i = 0; i < NC; ++i) {
                                    const int d = 4 * (lane + 32 * i);
                                    const float* g = (kind ? a.vc : a.kc) + ((size_t)min(j0 + KEYS * t + r[b], j1 - 1) * a.n_kv + kvh) * a.hd + d;
                                    y[b][i] = some && d < a.hd ? *reinterpret_cast<const float4*>(g) : make_float4(0.f, 0.f, 0.f, 0.f);
                                }
                                if (!some) r[b] = -1;
                            }
#pragma unroll
                            for (int b = 0; b < B; ++b) {
                                if (r[b] < 0) break;
                                float m = 0.0f;
                                auto finite = [&](float& z, int col) {
                                    if (fabsf(z) < INFINITY) m = fmaxf(m, fabsf(z));
                                    if (fabsf(z) == INFINITY && kind) {
                                        atomicOr(&infinite[z < 0.0f][col >> 5], 1u << (col & 31));
                                        any_infinite = 1;
                                        z = 0.0f;
                                    }
                                };
#pragma unroll
                                for (int i = 0; i < NC; ++i) {
                                    const int col = 4 * (lane + 32 * i);
                                    finite(y[b][i].x, col), finite(y[b][i].y, col + 1), finite(y[b][i].z, col + 2), finite(y[b][i].w, col + 3);
                                }
                                const int s = scale_exp(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
                                const f32x2 f = pack2(pow2i(s), pow2i(s));
#pragma unroll
                                for (int i = 0; i < NC; ++i) {
                                    const int d4 = lane + 32 * i;
                                    uint8_t* to = tile + (d4 >> 1) * L::kStride + r[b] * 16 + (d4 & 1) * 8;
                                    uint2 hi, lo;
                                    split2(mul2(pack2(y[b][i].x, y[b][i].y), f), hi.x, lo.x);
                                    split2(mul2(pack2(y[b][i].z, y[b][i].w), f), hi.y, lo.y);
                                    if (4 * d4 < HD) {
                                        *reinterpret_cast<uint2*>(to) = hi;
                                        *reinterpret_cast<uint2*>(to + L::kPart) = lo;
                                    }
                                }
                                if (lane == 0) of_row[r[b]] = s;
                            }
                        }
                    }
                    if (lane == 0) rows_differ[slot] = apart;
                    fence_async_smem();
                    __syncwarp();
                }
                if (lane == 0) mbar_arrive(kind ? &vsized[t & 1] : &ksized[t & 1]);
            }
        }
    } else if (warp >= kTtLoadWarp) {
        // ---------------- loaders: warp w takes two of the eight chunks of rows of each tile ----------------
        regs_dec<kTtLoadRegs>();
        const int lw = warp - kTtLoadWarp;
        const size_t pstride = (size_t)a.n_kv * a.hd;
        const float* src[2] = {a.kc + (size_t)kvh * a.hd, a.vc + (size_t)kvh * a.hd};
        uint8_t* staging = sm + L::oStaging + lw * 4 * L::kChunk;
        float scale_k = 0.0f, scale_v = 0.0f;  // the CTA's
        const bool in1 = 4 * (WIDE ? lane + 32 : lane % (HD / 4)) < a.hd;  // the lane's columns (WIDE: of its odd fours) are there
        // chunk i of tile t: the warp's first and second rows of K, of V; a lane's
        // k-th float4 of a chunk is float4 col(k) of its row at(k)
        constexpr int LPR = HD / 4, NK = CR * HD / 128;
        auto at = [&](int k) { return WIDE ? k >> 1 : lane / LPR + 32 / LPR * k; };
        auto col = [&](int k) { return WIDE ? lane + 32 * (k & 1) : lane % LPR; };
        auto row_of = [&](int t, int i) { return j0 + KEYS * t + 2 * CR * lw + CR * (i & 1); };
        auto issue = [&](int t, int i) {
            const int row = row_of(t, i);
            const float* g = src[i >> 1] + (size_t)row * pstride;
            float* d = reinterpret_cast<float*>(staging + i * L::kChunk);
            if (t < n_tiles && row + CR <= j1 && 4 * col(NK - 1) < a.hd) {
#pragma unroll
                for (int k = 0; k < NK; ++k) cp_async16_row(d + at(k) * HD + 4 * col(k), g + (size_t)at(k) * pstride + 4 * col(k));
            } else if (t < n_tiles) {  // zeros past the last column; past the last row that row again, so that none is small there
#pragma unroll 1
                for (int k = 0; k < NK; ++k) {
                    const bool some = 4 * col(k) < a.hd;
                    cp_async16_row(d + at(k) * HD + 4 * col(k), some ? src[i >> 1] + (size_t)min(row + at(k), j1 - 1) * pstride + 4 * col(k) : src[0], some ? 16 : 0);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = 0; i < 4; ++i) issue(0, i);
        bool ok = true;
        for (int t = 0; t < n_tiles && ok; ++t) {
            uint8_t* tile = sm + (t & 1) * L::kStage;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                asm volatile("cp.async.wait_group 3;" ::: "memory");
                __syncwarp();
                const float* st = reinterpret_cast<const float*>(staging + i * L::kChunk);
                const int chunk = 2 * lw + (i & 1);
                float x[4 * NK];
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    const float4 v = *reinterpret_cast<const float4*>(st + at(k) * HD + 4 * col(k));
                    x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w;
                }
                float even, odd;
                const float most = lane_max(x, even, odd);
                if (t == 0 && (i & 1) == 0) {
                    const unsigned top = __reduce_max_sync(0xffffffffu, most < INFINITY ? __float_as_uint(most) : 0u);
                    if (lane == 0) atomicMax(&first_top[i >> 1], top);
                    asm volatile("bar.sync 2, 128;" ::: "memory");
                    const int s = scale_exp(first_top[i >> 1]);
                    (i ? scale_v : scale_k) = pow2i(s);
                    if (lane == 0) cta_scale[i >> 1] = s;  // all four warps the same
                }
                issue(t + 1, i);  // the chunk is in registers
                const float fs = i < 2 ? scale_k : scale_v;
                const f32x2 f = pack2(fs, fs);
                if ((i & 1) == 0 && t >= kTtStages) ok = wait_warp(i ? &vempty[t & 1] : &kempty[t & 1], ((t >> 1) - 1) & 1);
                if (!ok) break;
                uint8_t* d = tile + (i >> 1) * 2 * L::kPart + CR * chunk * 16;
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    uint8_t* dk = d + (col(k) >> 1) * L::kStride + at(k) * 16 + (col(k) & 1) * 8;
                    uint2 hi, lo;
                    split2(mul2(pack2(x[4 * k], x[4 * k + 1]), f), hi.x, lo.x);
                    split2(mul2(pack2(x[4 * k + 2], x[4 * k + 3]), f), hi.y, lo.y);
                    *reinterpret_cast<uint2*>(dk) = hi;
                    *reinterpret_cast<uint2*>(dk + L::kPart) = lo;
                }
                // rows that may be small, or large: in most chunks each lane sees in each of its rows a value
                // that is not small, and one vote tells
                const float least = WIDE ? fminf(even, in1 ? odd : INFINITY) : in1 ? fminf(even, odd) : INFINITY;
                const bool apart = __any_sync(0xffffffffu, least * fs < kTtSmall || most * fs >= kTtLarge);
                if (lane == 0) flags[(2 * (t & (kTtScales - 1)) + (i >> 1)) * 8 + chunk] = apart;
                if (i & 1) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(i == 1 ? &kfull[t & 1] : &vfull[t & 1]);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if ((warp >> 2) < nl || kShared) {
        // ---------------- softmax and output: a thread per query row (and lane) ----------------
        regs_inc<kTtSoftmaxRegs>();
        const int x = warp >> 2;
        const int first = r0 + (kShared ? 0 : 128 * x) + 32 * (warp & 3), row = first + lane;
        const bool active = first < rows;  // of the warp
        const bool many = rows - first > kTtTurn;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t tq = tmem + lanes + kTtQ + x * (WIDE ? 64 : 128), to = tmem + lanes + kTtO;
        constexpr int kQlo = HD / 2;  // columns from Q's hi to its lo parts
        const int c0 = WIDE ? 128 * x : 0;  // the lane's first column
        int sq = 0;
        float v[HO];  // the lane's columns of the row
        float qm = 0.0f;
        if (active && many) {
            // four lanes per row, 16 columns at a time, then turned into a row per thread:
            // a load touches 8 rows' lines instead of 32
            float4 w[HO / 4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int of = first + 8 * k + lane / 4;
                const bool some = of < rows;
                const float* qp = a.q + ((size_t)(some ? of / a.G : 0) * a.n_heads + kvh * a.G + (some ? of % a.G : 0)) * a.hd + c0;
#pragma unroll
                for (int b = 0; b < HO / 16; ++b) {
                    const int col = 16 * b + 4 * (lane % 4);
                    w[4 * b + k] = some && c0 + col < a.hd ? *reinterpret_cast<const float4*>(qp + col) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            float* turn = reinterpret_cast<float*>(sm + L::oTurn + L::kTurn * warp);
#pragma unroll
            for (int b = 0; b < HO / 16; ++b) {
#pragma unroll
                for (int k = 0; k < 4; ++k) *reinterpret_cast<float4*>(turn + (8 * k + lane / 4) * 20 + 4 * (lane % 4)) = w[4 * b + k];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 y = *reinterpret_cast<const float4*>(turn + lane * 20 + 4 * i);
                    v[16 * b + 4 * i] = y.x; v[16 * b + 4 * i + 1] = y.y; v[16 * b + 4 * i + 2] = y.z; v[16 * b + 4 * i + 3] = y.w;
                }
                __syncwarp();
            }
        } else if (active) {
            const bool some = row < rows;
            const float* qp = a.q + ((size_t)(some ? row / a.G : 0) * a.n_heads + kvh * a.G + (some ? row % a.G : 0)) * a.hd + c0;
#pragma unroll
            for (int c = 0; c < HO / 4; ++c) {
                const float4 w = some && c0 + 4 * c < a.hd ? *reinterpret_cast<const float4*>(qp + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[4 * c] = w.x; v[4 * c + 1] = w.y; v[4 * c + 2] = w.z; v[4 * c + 3] = w.w;
            }
        }
        if (active) {
#pragma unroll
            for (int c = 0; c < HO; ++c) qm = fmaxf(qm, fabsf(v[c]) < INFINITY ? fabsf(v[c]) : 0.0f);
        }
        if (WIDE) {  // the other columns' maximum
            float* most = reinterpret_cast<float*>(sm + L::oState) + 32 * (warp & 3) + lane;
            most[128 * x] = qm;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            qm = fmaxf(qm, most[128 * (x ^ 1)]);
        }
        if (active) {
            sq = scale_exp(__float_as_uint(qm));
            if (x == 0 || !ALT) {
                const f32x2 f = pack2(pow2i(sq), pow2i(sq));
#pragma unroll
                for (int b = 0; b < HO / 32; ++b) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) split2(mul2(pack2(v[32 * b + 2 * c], v[32 * b + 2 * c + 1]), f), hi[c], lo[c]);
                    tmem_st16(tq + 16 * b, hi);
                    tmem_st16(tq + kQlo + 16 * b, lo);
                }
                tmem_wait_st();
            }
        }
        tc_fence_before();
        if (x == 0 || !ALT) mbar_arrive(qfull);

        // The least scale of K with scores of up to 2^22 (the products' sum is 2^38 at most): beyond, the rounding
        // of one takes its distance from the reference out of fp16's range where that is not taken last.
        const int tame = 16 + (int)(__float_as_uint(fabsf(a.scale2)) >> 23) - 126 - __reduce_min_sync(0xffffffffu, sq);
        float T = -INFINITY, l = 0.0f;
        f32x2 o[HO / 2];
#pragma unroll
        for (int d = 0; d < HO / 2; ++d) o[d] = 0;
        bool ok = true;
#pragma unroll 1
        for (int t = ALT ? x : 0; t < n_tiles; t += ALT ? 2 : 1) {
            // V is mostly there when the scores are: its flags are then looked at before the first pass
            bool v_in = __all_sync(0xffffffffu, mbar_test(&vfull[t & 1], (t >> 1) & 1));
            ok = wait_warp(&sfull[WIDE ? t & 1 : x], phase_s(t));
            if (!ok) break;
            float alpha = 1.0f, beta = 1.0f;
            const uint32_t ts = tmem + lanes + kTtS + (WIDE ? (t & 1) * KEYS : x * 64), tp = WIDE ? tmem + lanes + kTtP + (t & 1) * KEYS : ts;
            // the weights; WIDE: by lane 0, the other needs their reference alone.  The products of tile t - 2 have read this block of it, as they
            // were issued before the one of tile t - 1 that lane 0 has waited for
            const bool writes = !WIDE || x == 0;
            if (active) {
                tc_fence_after();
                const int valid = j1 - j0 - KEYS * t;
                // 2^(-sq - sk) may need two factors
                auto factor = [&](int sk) {
                    const int n = -sq - sk, h = n >> 1;
                    return a.scale2 * pow2i(h) * pow2i(n - h);
                };
                // The flags are not written again before this warp is through with the tile, so that its
                // threads agree; the rows' own scales are there with the scores (K), with vsized (V).
                const int slot = 2 * (t & (kTtScales - 1));
                auto flagged = [&](int kind) {
                    const uint2 c = *reinterpret_cast<const uint2*>(flags + 8 * (slot + kind));
                    return (c.x | c.y) != 0;
                };
                auto apart = [&](int kind) { return flagged(kind) && rows_differ[slot + kind]; };
                const float f0 = factor(cta_scale[0]);
                const bool even_k = !flagged(0) && cta_scale[0] >= tame;
                int V = 0;
                bool even_v = false;
                auto look = [&] {
                    V = cta_scale[1];
                    even_v = !flagged(1);
                };
                if (v_in) look();
                float tm = -INFINITY;
                if (even_k && f0 >= 0.0f) {  // behind the last row it is there again
#pragma unroll 1
                    for (int h = 0; h < KEYS / 32; ++h) {
                        float s[32];
                        tmem_ld32f(ts + 32 * h, s);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) tm = fmaxf(tm, fmaxf(s[j], s[j + 1]));
                    }
                    tm *= f0;
                } else {
                    const bool own_k = apart(0);
#pragma unroll 1
                    for (int b = 0; b < min(KEYS, valid); b += 4) {
                        float s[4];
                        tmem_ld4f(ts + b, s);
#pragma unroll
                        for (int j = 0; j < 4; ++j) tm = fmaxf(tm, s[j] * (own_k ? factor(row_scales[slot * KEYS + b + j]) : f0));
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
                if (!v_in) {
                    ok = wait_warp(&vfull[t & 1], (t >> 1) & 1);
                    if (!ok) break;
                    look();
                }
                if (!even_v) {
                    ok = wait_warp(&vsized[t & 1], (t >> 1) & 1);
                    if (!ok) break;
                    even_v = !rows_differ[slot + 1];
                }
                // The unit 2^-n.  With the CTA's scales, 2^V for V's rows, the weights are taken
                // times 2^m, m = n - V; else each times 2^(n - its row's scale).
                float back = 1.0f;  // 2^-m
                f32x2 sum = 0;
                if (even_v && (even_k || (!apart(0) && cta_scale[0] >= tame))) {
                    // a whole number by rounding in the last place of 1.5 * 2^23; at most what 2^-m and 2^-n can be
                    const float magic = 12582912.0f;
                    const int zero = __float_as_int(magic), r = min(__float_as_int(fmaxf((float)kTtTop + (ref - tm), 0.0f) + magic), zero + 126 - max(V, 0));
                    const int m = r - zero;
                    const float shift = (__int_as_float(r) - magic) - ref;
                    back = pow2i(-m);
                    beta = pow2i(-m - V);
                    if (writes && valid >= KEYS) {
                        const f32x2 f02 = pack2(f0, f0), shift2 = pack2(shift, shift);
#pragma unroll 1
                        for (int b = 0; b < KEYS / 16; ++b) {
                            float s[16];
                            uint32_t p[16];
                            tmem_ld16f(ts + 16 * b, s);
#pragma unroll
                            for (int j = 0; j < 16; j += 2) {
                                const float2 z = unpack2(fma2(pack2(s[j], s[j + 1]), f02, shift2));
                                const f32x2 e = pack2(ex2(z.x), ex2(z.y));
                                sum = add2(sum, e);
                                split2(e, p[j / 2], p[8 + j / 2]);
                            }
                            tmem_st16(tp + 16 * b, p);
                        }
                    } else if (writes) {
#pragma unroll 1
                        for (int b = 0; b < KEYS / 16; ++b) {
                            float s[16];
                            uint32_t p[16];
                            tmem_ld16f(ts + 16 * b, s);
#pragma unroll
                            for (int j = 0; j < 16; j += 2) {
                                float e[2] = {0.0f, 0.0f};
#pragma unroll
                                for (int y = j; y < j + 2; ++y)
                                    if (16 * b + y < valid)
                                        e[y - j] = ex2(fmaf(s[y], f0, shift));
                                const f32x2 e2 = pack2(e[0], e[1]);
                                sum = add2(sum, e2);
                                split2(e2, p[j / 2], p[8 + j / 2]);
                            }
                            tmem_st16(tp + 16 * b, p);
                        }
                    }
                } else {
                    const int* of_row = row_scales + slot * KEYS;
                    const bool own_k = flagged(0), own_v = flagged(1);
                    auto factor_k = [&](int j) { return own_k ? factor(of_row[j]) : f0; };
                    auto scale_v = [&](int j) { return (float)(own_v ? of_row[KEYS + j] : V); };
                    float most = -INFINITY;  // exponent of the largest weight times V
#pragma unroll 1
                    for (int b = 0; b < min(KEYS, valid); b += 4) {  // behind the last row it is there again
                        float s[4];
                        tmem_ld4f(ts + b, s);
#pragma unroll
                        for (int j = 0; j < 4; ++j) most = fmaxf(most, (__fmul_rn(s[j], factor_k(b + j)) - ref) - scale_v(b + j));
                    }
                    const float n = floorf(fminf(fmaxf((float)kTtTop - most, -126.0f), 126.0f));
                    beta = pow2i(-(int)n);
                    if (writes)
#pragma unroll 1
                        for (int b = 0; b < KEYS; b += 16) {
                            float s[16];
                            uint32_t p[16];
                            tmem_ld16f(ts + b, s);
#pragma unroll
                            for (int j = 0; j < 16; j += 2) {
                                float e[2] = {0.0f, 0.0f}, w[2] = {0.0f, 0.0f};
#pragma unroll
                                for (int y = j; y < j + 2; ++y)
                                    if (b + y < valid) {
                                        const float z = __fmul_rn(s[y], factor_k(b + y)) - ref;
                                        e[y - j] = ex2(z);
                                        w[y - j] = ex2(z + (n - scale_v(b + y)));
                                    }
                                sum = add2(sum, pack2(e[0], e[1]));
                                split2(pack2(w[0], w[1]), p[j / 2], p[8 + j / 2]);
                            }
                            tmem_st16(tp + b, p);
                        }
                }
                const float2 parts = unpack2(sum);
                l = fmaf(l, alpha, (parts.x + parts.y) * back);
                tmem_wait_st();
                tc_fence_before();
            }
            // WIDE: lane 1's arrival says that it has asked for this tile's barriers, which may
            // go on to their next phases once its products are through
            mbar_arrive(&pfull[x]);
            ok = wait_warp(&ofull[x], phase(t));
            if (!ok) break;
            if (active) {
                tc_fence_after();
                const f32x2 beta2 = pack2(beta, beta);
                if (__any_sync(0xffffffffu, alpha != 1.0f)) {
                    const f32x2 alpha2 = pack2(alpha, alpha);
#pragma unroll
                    for (int d = 0; d < HO / 2; ++d) o[d] = mul2(o[d], alpha2);
                }
#pragma unroll
                for (int b = 0; b < HO / 32; ++b) {
                    float w[32];
                    tmem_ld32f(to + 32 * b, w);
#pragma unroll
                    for (int d = 0; d < 32; d += 2) o[16 * b + d / 2] = fma2(pack2(w[d], w[d + 1]), beta2, o[16 * b + d / 2]);
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
            for (int d = 0; d < HO / 2; ++d) {
                auto of = [&](int c) {
                    const float up = infinite[0][c >> 5] >> (c & 31) & 1 ? INFINITY : 0.0f;
                    return infinite[1][c >> 5] >> (c & 31) & 1 ? up - INFINITY : up;
                };
                o[d] = add2(o[d], pack2(of(c0 + 2 * d), of(c0 + 2 * d + 1)));
            }
        }
        if (active && !(ALT && x == 1)) {
            constexpr int C = HD > 64 ? 32 : 16, LR = C / 4;  // columns at a time, lanes per row
            static_assert(32 * (C + 4) * 4 <= 2 * L::kChunk, "a warp's share of the staging");
            auto record = [&](int of) { return a.part + (((size_t)kvh * rows + of) * a.splits + split) * (a.hd + 4); };
            if (row < rows && (!WIDE || x == 0)) *reinterpret_cast<float2*>(record(row)) = make_float2(T, l);
            if (many) {
                // a thread's row is turned into rows of the warp through its part of the loaders'
                // staging, which they are through with: whole lines are written
                float* turn = reinterpret_cast<float*>(sm + L::oStaging + 2 * L::kChunk * warp);
#pragma unroll
                for (int b = 0; b < HO / C; ++b) {
#pragma unroll
                    for (int i = 0; i < LR; ++i) {
                        const float2 x0 = unpack2(o[b * C / 2 + 2 * i]), x1 = unpack2(o[b * C / 2 + 2 * i + 1]);
                        *reinterpret_cast<float4*>(turn + lane * (C + 4) + 4 * i) = make_float4(x0.x, x0.y, x1.x, x1.y);
                    }
                    __syncwarp();
                    const int col = c0 + b * C + 4 * (lane % LR);
#pragma unroll
                    for (int k = 0; k < LR; ++k) {
                        const int of = 32 / LR * k + lane / LR;
                        if (first + of < rows && col < a.hd)
                            *reinterpret_cast<float4*>(record(first + of) + 4 + col) =
                                *reinterpret_cast<const float4*>(turn + of * (C + 4) + 4 * (lane % LR));
                    }
                    __syncwarp();
                }
            } else if (row < rows) {
#pragma unroll
                for (int d = 0; d < HO; d += 4)
                    if (c0 + d < a.hd) {
                        const float2 x0 = unpack2(o[d / 2]), x1 = unpack2(o[d / 2 + 1]);
                        *reinterpret_cast<float4*>(record(row) + 4 + c0 + d) = make_float4(x0.x, x0.y, x1.x, x1.y);
                    }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kTtMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTtCols));
}

bool tree_tc_ok(int hd) { return hd <= 256 && hd % 16 == 0; }

cudaError_t tree_tc_launch(const TreeArgs& a, cudaStream_t st) {
    const int block = tree_tc_rows(a.hd);
    const dim3 grid(a.splits, a.n_kv, (a.n_tok * a.G + block - 1) / block);
    auto go = [&](auto k, size_t smem) {
        const cudaError_t e = set_smem_limit(k, smem);
        if (e != cudaSuccess) return e;
        return launch_after(k, grid, dim3(kTtThreads), smem, st, a);
    };
    if (a.hd > 128) return go(tree_tc_kernel<256, false>, TtLayout<256>::kAlloc);
    const bool alt = a.n_tok * a.G <= 128 && a.per >= kTtAltTiles * tree_tc_keys(a.hd);
    if (a.hd > 64) return alt ? go(tree_tc_kernel<128, true>, TtLayout<128>::kAlloc) : go(tree_tc_kernel<128, false>, TtLayout<128>::kAlloc);
    return alt ? go(tree_tc_kernel<64, true>, TtLayout<64>::kAlloc) : go(tree_tc_kernel<64, false>, TtLayout<64>::kAlloc);
}

}  // namespace gncx
