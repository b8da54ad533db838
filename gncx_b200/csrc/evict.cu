// evict.cu -- a KV cache held to a budget by accumulated attention weight:
// the decode attention step that sums the weight each cache row receives, and
// the eviction of the rows with the least.  No reference counterpart (the
// reference's cache only grows; its decode step is
// csrc/gncx_llm_kernels.cpp:1887-1994).
//
// Step: for each query head p = softmax(scale q.K), out = p V, and
// weight[kv][t] += sum of p[t] over the KV head's group.  p[t] is known only
// when the whole row of scores is, so
//   * weights_part_kernel streams K and V once (each warp walks batches of
//     rows through registers, with an online softmax), and leaves the scores
//     (4 bytes per (head, row) against the 8 hd per (KV head, row) read) and a
//     {max, sum, o} record per range of rows;
//   * weights_merge_kernel merges the records and turns the scores into
//     weights, one CTA per 1024 rows of a KV head, more CTAs for the outputs.
// A short cache is done in one launch: a cluster of 8 CTAs per KV head keeps the
// scores in shared memory and merges through distributed shared memory.
// Bound by HBM where long: 32 heads, 8 KV heads of 128, 32768 rows (268 MB) 49.9 us
// in a graph, 5.4 TB/s, of which 47.3 us are the first kernel; by latency where
// short: 512 rows 4.9 us, 7 us a call.
//
// Eviction: per KV head the rows are ranked (protected ones first, each kind by
// weight, a NaN weight last, equal weights by row), the first n_keep stay.
// The i-th free row below n_keep takes the i-th row that stays from behind
// it: rows that are read and rows that are written are disjoint, so the cache
// is compacted in place, in parallel, and no row moves that need not.
//   * evict_select_kernel, a CTA or a cluster of CTAs per KV head: radix
//     selection of the n_keep-th key over keys in registers, then the lists of
//     free and of moving rows by prefix sums;
//   * evict_move_kernel copies the rows (few rows: the selecting kernel does).
// The selection is a chain of dependent steps (under ncu 17 us of 8 KV heads' 32768
// rows: a read, then per digit a histogram, a cluster barrier, the other CTAs' counts
// and a scan), the moves are bound by HBM (23 us there for 54 MB read and as much
// written): 32768 -> 8192 rows 34 us in a graph, 42 where more rows are protected than
// stay and the first digit is looked at again.  One row of 4097: 3.6 us, two dependent
// reads.  Above 131072 rows one CTA per KV head selects, reading the weights four times:
// 262144 -> 65536 rows 681 us, of which the selection takes 529 (131072 -> 32768 rows
// with a cluster 107 us); one row of 262144 441 us.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "rows.cuh"
#include "tma.cuh"

namespace gncx {

// ---------------------------------------------------------------- decode step with weight sums
constexpr int kWsThreads = 256;
constexpr int kWsWarps = kWsThreads / 32;
constexpr int kWsRows = 1024;      // rows per CTA of the merge kernel's weight part
constexpr int kWsMaxParts = 256;
constexpr int kWsCluster = 8;      // CTAs per KV head that do the whole step for few rows

struct WeightsArgs {
    const float* q;
    const float* new_k;  // null: the row is in the cache
    const float* new_v;
    float* kc;
    float* vc;
    int pos, token_pos;
    int n_heads, n_kv, hd, G;
    float scale;
    float* out;
    float* weight;
    int32_t* positions;
    int row_stride;
    int parts, ppc;      // ranges per KV head, rows per range
    float* part;         // records [head][parts][hd + 4]
    float* scores;       // [head][score_ld]
    size_t score_ld;
};

// The rest of the step in one cluster: the warps' states as the CTA's record, the
// records' maxima and sums through distributed shared memory, then this CTA's
// share of the outputs and the weights of its rows.
template <int GT>
__device__ __forceinline__ void weights_cluster_end(const WeightsArgs& a, float* ost, const float* scores, const float (&mst)[kWsWarps][GT],
                                                    const float (&lst)[kWsWarps][GT], int kvh, int rank, int heads, int p0, int p1) {
    __shared__ float2 s_ml[GT];
    __shared__ float s_M[GT], s_inv[GT], s_f[GT][kWsCluster];
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* wt = a.weight + (size_t)kvh * a.row_stride;
    const int t0 = p0 + tid;
    const float old = t0 < p1 ? wt[t0] : 0.0f;  // on its way while the records are merged
    for (int t = tid; t < heads * a.hd; t += kWsThreads) {
        const int g = t / a.hd, d = t - g * a.hd;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWsWarps; ++w) M = fmaxf(M, mst[w][g]);
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < kWsWarps; ++w) {
            const float f = mst[w][g] == -INFINITY ? 0.0f : __expf(mst[w][g] - M);
            L = fmaf(lst[w][g], f, L);
            O = fmaf(ost[(size_t)(w * GT + g) * a.hd + d], f, O);
        }
        ost[(size_t)g * a.hd + d] = O;  // in place of warp 0's, which this thread alone reads
        if (d == 0) s_ml[g] = make_float2(M, L);
    }
    cluster.sync();
    if (warp < heads) {
        const float2 ml = lane < kWsCluster ? *cluster.map_shared_rank(&s_ml[warp], lane) : make_float2(-INFINITY, 0.0f);
        float M = ml.x;
#pragma unroll
        for (int o = kWsCluster / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float f = ml.x == -INFINITY ? 0.0f : __expf(ml.x - M);
        float L = ml.y * f;  // a NaN stays
#pragma unroll
        for (int o = kWsCluster / 2; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (lane < kWsCluster) s_f[warp][lane] = f;
        if (lane == 0) {
            s_M[warp] = M;
            s_inv[warp] = 1.0f / L;
        }
    }
    __syncthreads();
    for (int t = rank * kWsThreads + tid; t < heads * a.hd; t += kWsCluster * kWsThreads) {
        const int g = t / a.hd;
        float o = 0.0f;
#pragma unroll
        for (int r = 0; r < kWsCluster; ++r) o = fmaf(*cluster.map_shared_rank(&ost[t], r), s_f[g][r], o);
        a.out[(size_t)kvh * a.G * a.hd + t] = o * s_inv[g];
    }
    for (int t = t0; t < p1; t += kWsThreads) {
        float w = 0.0f;
        for (int g = 0; g < heads; ++g) w = fmaf(__expf(scores[g * a.ppc + t - p0] - s_M[g]), s_inv[g], w);
        const bool fresh = a.new_k && t == a.pos;  // the new row's sum starts here
        wt[t] = fresh ? w : (t == t0 ? old : wt[t]) + w;
        if (fresh && a.positions) a.positions[(size_t)kvh * a.row_stride + t] = a.token_pos;
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
}

// LPR lanes hold a row (NJ float4 each; columns past hd are zero), 32 / LPR
// rows side by side in a warp, B rows per lane and batch, GT query heads.  ONE: a
// cluster of kWsCluster CTAs per KV head does the whole step, the scores and
// records in its shared memory.
template <int LPR, int NJ, int GT, int B, bool ONE>
__global__ void __launch_bounds__(kWsThreads, 2) weights_part_kernel(const WeightsArgs a) {
    constexpr int SUB = 32 / LPR;
    constexpr int NV = B * GT;
    constexpr int SH = ilog2(LPR) - ilog2(NV);
    constexpr int LG = ilog2(GT);
    constexpr int RB = B * SUB;  // rows per warp and batch
    static_assert(NV <= LPR, "one total per lane");
    extern __shared__ __align__(16) float ost[];  // [warp][GT][hd], with ONE also scores [GT][ppc]
    float* own_scores = ost + (size_t)kWsWarps * GT * a.hd;
    __shared__ float wsh[kWsWarps][SUB * NV + GT];
    __shared__ float mst[kWsWarps][GT], lst[kWsWarps][GT];
    const int part = blockIdx.x, kvh = blockIdx.y, h0 = kvh * a.G + blockIdx.z * GT;
    const int heads = min(GT, a.G - (int)blockIdx.z * GT);
    const int len = a.pos + 1;
    const int p0 = part * a.ppc, p1 = min(len, p0 + a.ppc);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / LPR, lr = lane % LPR;
    const size_t ps = (size_t)a.n_kv * a.hd;
    float* kbase = a.kc + (size_t)kvh * a.hd;
    float* vbase = a.vc + (size_t)kvh * a.hd;
    bool on[NJ];
    int col[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        col[j] = 4 * (lr + j * LPR);
        on[j] = col[j] < a.hd;
    }
    pdl_wait();
    if (!ONE) pdl_launch_dependents();
    float4 q[GT][NJ], o[GT][NJ];
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            q[g][j] = ld_row(a.q + (size_t)(h0 + min(g, heads - 1)) * a.hd + col[j], on[j]);
            o[g][j] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    // the new row: stored by the lanes that read it below (each reads back what it stored itself)
    if (a.new_k && a.pos >= p0 && a.pos < p1) {
        const int r = a.pos - p0;
        if (warp == (r / RB) % kWsWarps && sub == (r % RB) / B) {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (on[j]) {
                    const size_t at = (size_t)a.pos * ps + col[j];
                    *reinterpret_cast<float4*>(kbase + at) = ld_row(a.new_k + (size_t)kvh * a.hd + col[j], true);
                    *reinterpret_cast<float4*>(vbase + at) = ld_row(a.new_v + (size_t)kvh * a.hd + col[j], true);
                }
        }
    }
    float m = -INFINITY, l = 0.0f;  // of head ((lane % LPR) >> SH) % GT
    const int my = lr >> SH;
    for (int b0 = p0 + warp * RB; b0 < p1; b0 += kWsWarps * RB) {
        const int r0 = b0 + sub * B;
        float4 kr[B][NJ], vr[B][NJ];
#pragma unroll
        for (int p = 0; p < B; ++p)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const size_t at = (size_t)min(r0 + p, p1 - 1) * ps + col[j];
                kr[p][j] = ld_row(kbase + at, on[j] && r0 + p < p1);
                vr[p][j] = ld_row(vbase + at, on[j] && r0 + p < p1);
            }
        float v[NV];
#pragma unroll
        for (int p = 0; p < B; ++p)
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                float c = 0.0f;
#pragma unroll
                for (int j = 0; j < NJ; ++j) c = dot4(q[g][j], kr[p][j], c);
                v[p * GT + g] = c;
            }
        float sc = lanes_reduce<NV, LPR>(v, lane) * a.scale;
        const int mp = my / GT, mg = my % GT;
        const bool live = r0 + mp < p1;
        const bool lead = (lr & ((1 << SH) - 1)) == 0;
        if (live && lead && mg < heads) {
            if (ONE) own_scores[mg * a.ppc + r0 + mp - p0] = sc;
            else a.scores[(size_t)(h0 + mg) * a.score_ld + r0 + mp] = sc;
        }
        if (!live) sc = -INFINITY;
        float bm = sc;
#pragma unroll
        for (int off = 16; off >= (1 << (SH + LG)); off >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, off));
        const float m_new = fmaxf(m, bm);
        // a batch holds at least one live row, so m_new > -inf unless its scores are
        const float e = sc == -INFINITY ? 0.0f : __expf(sc - m_new);
        const float corr = m == -INFINITY ? 0.0f : __expf(m - m_new);
        float bs = e;
#pragma unroll
        for (int off = 16; off >= (1 << (SH + LG)); off >>= 1) bs += __shfl_xor_sync(0xffffffffu, bs, off);
        l = fmaf(l, corr, bs);
        m = m_new;
        float* wr = wsh[warp];
        if (lead) wr[sub * NV + my] = e;
        if (sub == 0 && lead && my < GT) wr[SUB * NV + my] = corr;
        __syncwarp();
        float w[NV], cg[GT];
#pragma unroll
        for (int i = 0; i < NV; ++i) w[i] = wr[sub * NV + i];
#pragma unroll
        for (int g = 0; g < GT; ++g) cg[g] = wr[SUB * NV + g];
        __syncwarp();
#pragma unroll
        for (int g = 0; g < GT; ++g)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                float4 c = o[g][j];
                c.x *= cg[g]; c.y *= cg[g]; c.z *= cg[g]; c.w *= cg[g];
#pragma unroll
                for (int p = 0; p < B; ++p) {
                    const float ww = w[p * GT + g];
                    c.x = fmaf(ww, vr[p][j].x, c.x);
                    c.y = fmaf(ww, vr[p][j].y, c.y);
                    c.z = fmaf(ww, vr[p][j].z, c.z);
                    c.w = fmaf(ww, vr[p][j].w, c.w);
                }
                o[g][j] = c;
            }
    }
    // the warps' states as one record per head
    if (sub == 0 && (lr & ((1 << SH) - 1)) == 0 && my < GT) {
        mst[warp][my] = m;
        lst[warp][my] = l;
    }
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float4 c = o[g][j];
#pragma unroll
            for (int off = 16; off >= LPR; off >>= 1) {
                c.x += __shfl_xor_sync(0xffffffffu, c.x, off);
                c.y += __shfl_xor_sync(0xffffffffu, c.y, off);
                c.z += __shfl_xor_sync(0xffffffffu, c.z, off);
                c.w += __shfl_xor_sync(0xffffffffu, c.w, off);
            }
            if (sub == 0 && on[j]) *reinterpret_cast<float4*>(ost + (size_t)(warp * GT + g) * a.hd + col[j]) = c;
        }
    __syncthreads();
    if constexpr (ONE) {
        weights_cluster_end<GT>(a, ost, own_scores, mst, lst, kvh, part, heads, p0, p1);
    } else {
        for (int t = threadIdx.x; t < heads * a.hd; t += kWsThreads) {
            const int g = t / a.hd, d = t - g * a.hd;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWsWarps; ++w) M = fmaxf(M, mst[w][g]);
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < kWsWarps; ++w) {
                const float f = mst[w][g] == -INFINITY ? 0.0f : __expf(mst[w][g] - M);
                L = fmaf(lst[w][g], f, L);
                O = fmaf(ost[(size_t)(w * GT + g) * a.hd + d], f, O);
            }
            float* rec = a.part + ((size_t)(h0 + g) * a.parts + part) * (a.hd + 4);
            rec[4 + d] = O;
            if (d == 0) {
                rec[0] = M;
                rec[1] = L;
            }
        }
    }
}

// Maximum and sum of one head's records; one warp.
__device__ __forceinline__ void head_max_sum(const WeightsArgs& a, int h, int lane, float& M, float& L) {
    const float* rec = a.part + (size_t)h * a.parts * (a.hd + 4);
    M = -INFINITY;
    L = 0.0f;
    for (int p = lane; p < a.parts; p += 32) M = fmaxf(M, rec[(size_t)p * (a.hd + 4)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    for (int p = lane; p < a.parts; p += 32) {
        const float m = rec[(size_t)p * (a.hd + 4)];
        // the sum of a range without a maximum is 0, or NaN, which stays
        L = fmaf(rec[(size_t)p * (a.hd + 4) + 1], m == -INFINITY ? 0.0f : __expf(m - M), L);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
}

// blockIdx.x < row_ctas: the weights of rows [1024 x, ..) of KV head y;
// else the output of the group's head x - row_ctas.
__global__ void __launch_bounds__(kWsThreads) weights_merge_kernel(const WeightsArgs a, int row_ctas) {
    __shared__ float s_M[kWsWarps], s_inv[kWsWarps];
    __shared__ float s_f[kWsMaxParts];
    const int kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    if ((int)blockIdx.x >= row_ctas) {
        const int h = kvh * a.G + (int)blockIdx.x - row_ctas;
        float M, L;
        if (warp == 0) {
            head_max_sum(a, h, lane, M, L);
            if (lane == 0) {
                s_M[0] = M;
                s_inv[0] = 1.0f / L;
            }
        }
        __syncthreads();
        M = s_M[0];
        const float* rec = a.part + (size_t)h * a.parts * (a.hd + 4);
        for (int p = tid; p < a.parts; p += kWsThreads) {
            const float m = rec[(size_t)p * (a.hd + 4)];
            s_f[p] = m == -INFINITY ? 0.0f : __expf(m - M);
        }
        __syncthreads();
        for (int d = tid; d < a.hd; d += kWsThreads) {
            float o = 0.0f;
#pragma unroll 8
            for (int p = 0; p < a.parts; ++p) o = fmaf(rec[(size_t)p * (a.hd + 4) + 4 + d], s_f[p], o);
            a.out[(size_t)h * a.hd + d] = o * s_inv[0];
        }
        return;
    }
    constexpr int kPer = kWsRows / kWsThreads;
    const int t0 = blockIdx.x * kWsRows + tid;
    float w[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) w[i] = 0.0f;
    // the first heads' scores and the sums are on their way while the maxima are formed
    constexpr int kEarly = 4;
    const float* s0 = a.scores + (size_t)kvh * a.G * a.score_ld;
    float* wt = a.weight + (size_t)kvh * a.row_stride;
    float early[kEarly][kPer], old[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int t = t0 + i * kWsThreads;
        old[i] = t <= a.pos ? wt[t] : 0.0f;
#pragma unroll
        for (int g = 0; g < kEarly; ++g) early[g][i] = t <= a.pos && g < a.G ? s0[g * a.score_ld + t] : 0.0f;
    }
    for (int g0 = 0; g0 < a.G; g0 += kWsWarps) {
        __syncthreads();
        if (g0 + warp < a.G) {
            float M, L;
            head_max_sum(a, kvh * a.G + g0 + warp, lane, M, L);
            if (lane == 0) {
                s_M[warp] = M;
                s_inv[warp] = 1.0f / L;
            }
        }
        __syncthreads();
        if (g0 == 0) {
#pragma unroll
            for (int g = 0; g < kEarly; ++g)
                if (g < a.G) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) w[i] = fmaf(__expf(early[g][i] - s_M[g]), s_inv[g], w[i]);
                }
        }
        for (int g = g0 == 0 ? kEarly : 0; g < min(kWsWarps, a.G - g0); ++g) {
            const float* s = s0 + (size_t)(g0 + g) * a.score_ld;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int t = t0 + i * kWsThreads;
                if (t <= a.pos) w[i] = fmaf(__expf(s[t] - s_M[g]), s_inv[g], w[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int t = t0 + i * kWsThreads;
        if (t > a.pos) continue;
        const bool fresh = a.new_k && t == a.pos;  // the new row's sum starts here
        wt[t] = fresh ? w[i] : old[i] + w[i];
        if (fresh && a.positions) a.positions[(size_t)kvh * a.row_stride + t] = a.token_pos;
    }
}

// Ranges per KV head: about two CTAs per SM, at least 32 rows each.
static int weights_parts(int len, int n_kv, int zgroups, int sm_count) {
    int parts = (2 * sm_count + n_kv * zgroups - 1) / (n_kv * zgroups);
    const int most = (len + 31) / 32;
    if (parts > most) parts = most;
    if (parts > kWsMaxParts) parts = kWsMaxParts;
    return parts < 1 ? 1 : parts;
}
// Whether one launch, a cluster per KV head, does the step: 16 heads, 8 KV heads of
// 128, 512 rows 4.8 us against 5.2 with two kernels (called one by one 6.8 against
// 9.3, a launch less); 2048 rows 8.2 against 9.1; 64 columns, 2048 rows on one KV head
// 5.8 against 7.4; 256 columns, 2048 rows on one KV head 15.4 against 10.4.
static bool weights_one(int len, int hd, int zgroups) {
    return zgroups == 1 && len <= 4096 && len * hd <= (hd > 128 ? 1 << 17 : 1 << 18);
}
static int weights_group(int G) { return G >= 3 ? 4 : G; }  // query heads a CTA serves

size_t weights_workspace_bytes(int pos, int n_heads, int n_kv, int hd, int sm_count) {
    const int G = n_heads / n_kv, GT = weights_group(G);
    const int parts = weights_parts(pos + 1, n_kv, (G + GT - 1) / GT, sm_count);
    const size_t rec = ((size_t)n_heads * parts * (hd + 4) * 4 + 255) / 256 * 256;
    return rec + (size_t)n_heads * (((size_t)pos + 1 + 31) / 32 * 32) * 4;
}

template <int LPR, int NJ>
static cudaError_t launch_weights_part(const WeightsArgs& a, dim3 grid, int GT, bool one, cudaStream_t st) {
    const size_t smem = ((size_t)kWsWarps * GT * a.hd + (one ? GT * a.ppc : 0)) * 4;
    auto go = [&](auto k, auto k_one) {
        const cudaError_t e = set_smem_limit(one ? k_one : k, smem);
        if (e != cudaSuccess) return e;
        return launch_early(one ? k_one : k, grid, dim3(kWsThreads), smem, st, one ? kWsCluster : 1, a);
    };
    constexpr int B = NJ == 1 ? 4 : 2;
    switch (GT) {
        case 1: return go(weights_part_kernel<LPR, NJ, 1, B, false>, weights_part_kernel<LPR, NJ, 1, B, true>);
        case 2: return go(weights_part_kernel<LPR, NJ, 2, B, false>, weights_part_kernel<LPR, NJ, 2, B, true>);
        default: return go(weights_part_kernel<LPR, NJ, 4, B, false>, weights_part_kernel<LPR, NJ, 4, B, true>);
    }
}

int weights_step_launch(const float* q, const float* new_k, const float* new_v, float* kc, float* vc, int pos,
                        int token_pos, int n_heads, int n_kv, int hd, float scale, float* out, float* weight,
                        int32_t* positions, int row_stride, void* ws, cudaStream_t st) {
    const int G = n_heads / n_kv, GT = weights_group(G), z = (G + GT - 1) / GT, len = pos + 1;
    WeightsArgs a{};
    a.q = q;
    a.new_k = new_k;
    a.new_v = new_v;
    a.kc = kc;
    a.vc = vc;
    a.pos = pos;
    a.token_pos = token_pos;
    a.n_heads = n_heads;
    a.n_kv = n_kv;
    a.hd = hd;
    a.G = G;
    a.scale = scale;
    a.out = out;
    a.weight = weight;
    a.positions = positions;
    a.row_stride = row_stride;
    const bool one = weights_one(len, hd, z);
    a.parts = one ? kWsCluster : weights_parts(len, n_kv, z, device_info().sm_count);
    a.ppc = (len + a.parts - 1) / a.parts;
    if (!one) a.parts = (len + a.ppc - 1) / a.ppc;
    a.part = static_cast<float*>(ws);
    a.scores = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + ((size_t)n_heads * a.parts * (hd + 4) * 4 + 255) / 256 * 256);
    a.score_ld = ((size_t)len + 31) / 32 * 32;
    const dim3 grid(a.parts, n_kv, z);
    const cudaError_t e = hd <= 64    ? launch_weights_part<16, 1>(a, grid, GT, one, st)
                          : hd <= 128 ? launch_weights_part<32, 1>(a, grid, GT, one, st)
                                      : launch_weights_part<32, 2>(a, grid, GT, one, st);
    if (e != cudaSuccess) return kErrCuda;
    if (one) return kOk;
    const int row_ctas = (len + kWsRows - 1) / kWsRows;
    return launch_after(weights_merge_kernel, dim3(row_ctas + G, n_kv), dim3(kWsThreads), 0, st, a, row_ctas) == cudaSuccess
               ? kOk
               : kErrCuda;
}

// ---------------------------------------------------------------- eviction
constexpr int kEvThreads = 1024;
constexpr int kEvSpread = 8192;  // rows above which a cluster of 8 CTAs selects instead of one CTA
constexpr int kEvOne = 65536;    // rows up to which one CTA looks for the one row to evict
constexpr int kEvHere = 256;     // moves up to which the selecting kernel makes them
constexpr int kEvBins = 2048;

struct EvictArgs {
    float* kc;
    float* vc;
    const float* weight;
    const int32_t* positions;  // null: nothing is protected
    int row_stride, n_rows, n_keep, recent_pos, n_kv, hd;
    float* weight_out;
    int32_t* positions_out;
    int out_stride;
    int32_t* moves;  // per KV head: count, then max_moves free rows, then max_moves moving rows
    int max_moves;
    uint32_t* masks;  // many rows, per KV head: words of "above the threshold", then of "at the threshold"
    int words;
    bool here;  // the selecting kernel moves the rows too
};

// The weights in order, from 0x007FFFFF (-inf) to 0xFF800000 (+inf); 0: NaN.
__device__ __forceinline__ uint32_t evict_weight_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);  // -0 as +0
    return w != w ? 0u : u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
// Greater keys stay.  32 bits hold protection and weight, because one of them
// decides: where at most n_keep rows are protected all of those stay, under the one
// key kEvProtected, and the others are ranked by weight; where more are (`crowded`)
// no other row stays (0), and the protected ones are ranked by weight.
constexpr uint32_t kEvProtected = 0xFFFFFFFFu;
constexpr uint32_t kEvProtectedBin = ~0u << 21;  // its first digit, which no weight has
__device__ __forceinline__ uint32_t evict_key(float w, bool late, bool crowded = false) {
    const uint32_t k = evict_weight_key(w);
    if (crowded) return late ? max(k, 1u) : 0u;
    return late ? kEvProtected : k;
}
__device__ __forceinline__ uint32_t evict_key(const EvictArgs& a, int h, int i, bool crowded) {
    const float w = a.weight[(size_t)h * a.row_stride + i];
    return evict_key(w, a.positions && a.positions[(size_t)h * a.row_stride + i] >= a.recent_pos, crowded);
}
// The keys key_of(weight, protected) of rows row0 + i * kEvThreads + thread (0 past
// the last row); the sums and positions of those below n_keep go to the outputs at
// once, where the rows that move in write theirs later.
template <int KPT, class Key, class KeyOf>
__device__ __forceinline__ void evict_load(const EvictArgs& a, int h, int row0, Key (&key)[KPT], KeyOf key_of) {
    float w[KPT];
    int32_t p[KPT];
    const size_t base = (size_t)h * a.row_stride;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
        const int row = row0 + i * kEvThreads + threadIdx.x;
        w[i] = row < a.n_rows ? a.weight[base + row] : 0.0f;
        p[i] = row < a.n_rows && a.positions ? a.positions[base + row] : 0;
    }
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
        const int row = row0 + i * kEvThreads + threadIdx.x;
        key[i] = row < a.n_rows ? key_of(w[i], a.positions && p[i] >= a.recent_pos) : Key(0);
        if (row < a.n_keep) {
            if (a.weight_out != a.weight) a.weight_out[(size_t)h * a.out_stride + row] = w[i];
            if (a.positions && a.positions_out != a.positions) a.positions_out[(size_t)h * a.out_stride + row] = p[i];
        }
    }
}

// Exclusive prefix sum of one value per thread over the CTA (32 warps), and the
// total; s_warp holds 32 values, and the next scan uses another array.
template <class T>
__device__ __forceinline__ T cta_scan(T v, T* s_warp, T& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    T w = s_warp[lane];  // every warp sums the warps' totals for itself
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const T before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    return x - v + (warp ? before : T(0));
}

// Copy rows of KV head h: the i-th free row takes the i-th moving row, for i0,
// i0 + step, .. below n, kEvMoveRows at a time; one warp.
constexpr int kEvMoveRows = 2;
__device__ __forceinline__ void evict_move_rows(const EvictArgs& a, int h, const int32_t* to, const int32_t* from, int n,
                                                int i0, int lane) {
    const int hd4 = a.hd / 4;
    const size_t ps = (size_t)a.n_kv * a.hd;
    int f[kEvMoveRows], t[kEvMoveRows];
#pragma unroll
    for (int r = 0; r < kEvMoveRows; ++r) {
        const int i = min(i0 + r, n - 1);
        f[r] = from[i];
        t[r] = to[i];
    }
    for (int c = lane; c < hd4; c += 32) {
        float4 k[kEvMoveRows], v[kEvMoveRows];
#pragma unroll
        for (int r = 0; r < kEvMoveRows; ++r) {
            const size_t at = (size_t)f[r] * ps + (size_t)h * a.hd + 4 * c;
            k[r] = __ldcs(reinterpret_cast<const float4*>(a.kc + at));
            v[r] = __ldcs(reinterpret_cast<const float4*>(a.vc + at));
        }
#pragma unroll
        for (int r = 0; r < kEvMoveRows; ++r)
            if (i0 + r < n) {
                const size_t at = (size_t)t[r] * ps + (size_t)h * a.hd + 4 * c;
                *reinterpret_cast<float4*>(a.kc + at) = k[r];
                *reinterpret_cast<float4*>(a.vc + at) = v[r];
            }
    }
    if (lane < kEvMoveRows && i0 + lane < n) {
        const int ff = from[i0 + lane], tt = to[i0 + lane];
        a.weight_out[(size_t)h * a.out_stride + tt] = a.weight[(size_t)h * a.row_stride + ff];
        if (a.positions) a.positions_out[(size_t)h * a.out_stride + tt] = a.positions[(size_t)h * a.row_stride + ff];
    }
}

// One cluster per KV head, each CTA a run of kEvThreads * KPT rows, their keys in
// registers.  Counts are summed over the cluster through distributed shared
// memory.
template <int KPT, int SIZE>
__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(const EvictArgs a) {
    constexpr int kWords = 32 * KPT;  // of 32 rows, per CTA
    static_assert(kEvThreads == 1024, "32 warps, and a word per thread where KPT is 32");
    // counts of two bins per word, bin 2 i in the low half: at most 16384 rows per CTA
    __shared__ uint32_t hist[4][kEvBins / 2];  // of each pass, and of a first pass that is done again
    static_assert(kEvThreads * KPT < 65536, "a count fits 16 bits");
    __shared__ int s_scan[5][32];
    __shared__ u_int64_t s_scan2[32];
    __shared__ uint32_t s_gt[kWords], s_eq[kWords];
    __shared__ uint32_t s_prefix[4];
    __shared__ int s_need[4], s_ties;  // need of each pass; how many rows have the last key
    __shared__ int2 s_count;           // of this CTA: free rows, moving rows
    __shared__ u_int64_t s_base[kWords];
    __shared__ int32_t s_to[kEvHere], s_from[kEvHere];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = SIZE > 1 ? (int)cluster.block_rank() : 0;
    auto meet = [&] {
        if (SIZE > 1) cluster.sync();
        else __syncthreads();
    };
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row0 = rank * kEvThreads * KPT;
    for (int i = tid; i < 4 * kEvBins / 2; i += kEvThreads) hist[0][i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    uint32_t key[KPT];
    evict_load(a, h, row0, key, [](float w, bool late) { return evict_key(w, late); });
    __syncthreads();
    // The n_keep-th largest key by digits of 11, 11 and 10 bits from the top:
    // each pass counts the keys that share the digits found so far.
    uint32_t prefix = 0;
    int need = a.n_keep;  // how many of the keys that share the prefix stay
    int shift = 32;
    int crowded = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int at = pass + crowded;  // this pass's arrays
        const int bits = pass < 2 ? 11 : 10;
        const uint32_t high = shift == 32 ? 0u : ~0u << shift;  // the digits found so far
        shift -= bits;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const bool in = row0 + i * kEvThreads + tid < a.n_rows && (key[i] & high) == prefix;
            const uint32_t d = (key[i] >> shift) & ((1u << bits) - 1);
            const unsigned act = __ballot_sync(0xffffffffu, in);
            if (!act) continue;
            // rows of equal digits (equal weights, a shared exponent): one addition for the warp
            const uint32_t d0 = __shfl_sync(0xffffffffu, d, __ffs(act) - 1);
            const unsigned same = __ballot_sync(0xffffffffu, in && d == d0);
            if (lane == 0) atomicAdd(&hist[at][d0 >> 1], (uint32_t)__popc(same) << 16 * (d0 & 1));
            if (in && d != d0) atomicAdd(&hist[at][d >> 1], 1u << 16 * (d & 1));
        }
        meet();
        // bins from the top: thread t holds bins 2047 - 2t and 2046 - 2t
        const int b1 = kEvBins - 1 - 2 * tid, b0 = b1 - 1;
        int c0 = 0, c1 = 0;
        uint32_t c[SIZE];
        if (SIZE == 1) {
            c[0] = hist[at][b0 / 2];
        } else {
#pragma unroll
            for (int r = 0; r < SIZE; ++r) c[r] = *cluster.map_shared_rank(&hist[at][b0 / 2], r);
        }
#pragma unroll
        for (int r = 0; r < SIZE; ++r) {
            c0 += c[r] & 0xFFFFu;
            c1 += c[r] >> 16;
        }
        int total;
        const int before = cta_scan(c1 + c0, s_scan[at], total);
        if (before < need && need <= before + c1) {
            s_prefix[at] = prefix | (uint32_t)b1 << shift;
            s_need[at] = need - before;
            s_ties = c1;
        } else if (before + c1 < need && need <= before + c1 + c0) {
            s_prefix[at] = prefix | (uint32_t)b0 << shift;
            s_need[at] = need - before - c1;
            s_ties = c0;
        }
        __syncthreads();
        prefix = s_prefix[at];
        need = s_need[at];
        if (pass == 0 && !crowded && prefix == kEvProtectedBin && need < s_ties) {
            // more rows are protected than stay: once more, with the protected ones' weights
            crowded = 1;
#pragma unroll
            for (int i = 0; i < KPT; ++i)
                key[i] = key[i] == kEvProtected
                             ? evict_key(a.weight[(size_t)h * a.row_stride + row0 + i * kEvThreads + tid], true, true)
                             : 0u;
            prefix = 0;
            need = a.n_keep;
            shift = 32;
            pass = -1;
        }
    }
    // prefix is the n_keep-th largest key; the first `need` of the s_ties rows that have it stay
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
        const bool some = row0 + i * kEvThreads + tid < a.n_rows;
        const unsigned gt = __ballot_sync(0xffffffffu, some && key[i] > prefix);
        const unsigned eq = __ballot_sync(0xffffffffu, some && key[i] == prefix);
        if (lane == 0) {
            s_gt[32 * i + warp] = gt;
            s_eq[32 * i + warp] = eq;
        }
    }
    __syncthreads();
    // a word per thread
    uint32_t keep = tid < kWords ? s_gt[tid] : 0u;
    const uint32_t eq = tid < kWords ? s_eq[tid] : 0u;
    if (need == s_ties) {
        keep |= eq;
    } else {
        int total;
        int before = cta_scan(__popc(eq), s_scan[4], total);
        // the rows of the CTAs before this one that have the key: their bin of the last pass
        if (SIZE > 1)
            for (int r = 0; r < rank; ++r)
                before += *cluster.map_shared_rank(&hist[2 + crowded][(prefix & 1023u) >> 1], r) >> 16 * (prefix & 1) & 0xFFFFu;
        uint32_t left = eq;
        for (int r = min(__popc(eq), max(0, need - before)); r > 0; --r) {
            keep |= left & (0u - left);
            left &= left - 1;
        }
    }
    // rows of this word below n_keep, and rows that exist
    const int i0 = row0 + tid * 32;
    const uint32_t low = i0 >= a.n_keep ? 0u : a.n_keep - i0 >= 32 ? ~0u : (1u << (a.n_keep - i0)) - 1;
    const uint32_t free_bits = tid < kWords ? low & ~keep : 0u, move_bits = keep & ~low;
    u_int64_t total;
    const u_int64_t pre = cta_scan((u_int64_t)__popc(free_bits) << 32 | __popc(move_bits), s_scan2, total);
    if (tid < kWords) {
        s_base[tid] = pre;
        s_gt[tid] = free_bits;
        s_eq[tid] = move_bits;
    }
    int n_to = (int)(total >> 32), pt0 = 0, pf0 = 0;  // of the whole head (= the moving rows); of the CTAs before
    if (SIZE > 1) {
        if (tid == 0) s_count = make_int2((int)(total >> 32), (int)(uint32_t)total);
        cluster.sync();
        int2 c[SIZE];
#pragma unroll
        for (int r = 0; r < SIZE; ++r) c[r] = *cluster.map_shared_rank(&s_count, r);
        n_to = 0;
#pragma unroll
        for (int r = 0; r < SIZE; ++r) {
            if (r < rank) {
                pt0 += c[r].x;
                pf0 += c[r].y;
            }
            n_to += c[r].x;
        }
    } else {
        __syncthreads();
    }
    int32_t* count = a.moves + (size_t)h * (1 + 2 * (size_t)a.max_moves);
    int32_t* to = count + 1;
    int32_t* from = to + a.max_moves;
    if (a.here && SIZE == 1) {
        to = s_to;
        from = s_from;
    }
    for (int w = warp; w < kWords; w += kEvThreads / 32) {  // a word per warp, a row per lane
        const uint32_t f = s_gt[w], m = s_eq[w], below = (1u << lane) - 1;
        const u_int64_t at = s_base[w];
        const int row = row0 + 32 * w + lane;
        if (f >> lane & 1) to[pt0 + (int)(at >> 32) + __popc(f & below)] = row;
        if (m >> lane & 1) from[pf0 + (int)(uint32_t)at + __popc(m & below)] = row;
    }
    if (tid == 0 && rank == 0) *count = n_to;
    if (a.here) {  // few rows: moved by the cluster itself
        meet();
        for (int i = (warp * SIZE + rank) * kEvMoveRows; i < n_to; i += 32 * SIZE * kEvMoveRows)
            evict_move_rows(a, h, to, from, n_to, i, lane);
    } else if (SIZE > 1) {
        cluster.sync();  // no CTA leaves while another may read its counts
    }
}

// One row to evict, the steady state of a full cache: the row with the least key
// (of equal ones the last) is overwritten by the row behind the first n_keep.
// One CTA per KV head.
__global__ void __launch_bounds__(kEvThreads) evict_one_kernel(const EvictArgs a) {
    constexpr int KPT = 4;
    __shared__ u_int64_t s_least[32];
    const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    u_int64_t least = ~(u_int64_t)0;
    for (int row0 = 0; row0 < a.n_rows; row0 += kEvThreads * KPT) {
        // protection, weight and, of equal ones, the last row
        u_int64_t key[KPT];
        evict_load(a, h, row0, key, [](float w, bool late) { return (u_int64_t)late << 63 | (u_int64_t)evict_weight_key(w) << 31; });
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int row = row0 + i * kEvThreads + tid;
            const u_int64_t k = key[i] | (0x7FFFFFFFu - (uint32_t)row);
            if (row < a.n_rows && k < least) least = k;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u_int64_t y = __shfl_xor_sync(0xffffffffu, least, o);
        least = y < least ? y : least;
    }
    if (lane == 0) s_least[warp] = least;
    __syncthreads();
    if (warp > 0) return;
    least = s_least[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u_int64_t y = __shfl_xor_sync(0xffffffffu, least, o);
        least = y < least ? y : least;
    }
    const int32_t to = (int32_t)(0x7FFFFFFFu - ((uint32_t)least & 0x7FFFFFFFu)), from = a.n_keep;
    if (to < a.n_keep) evict_move_rows(a, h, &to, &from, 1, 0, lane);
}

// Any number of rows: one CTA per KV head, which reads the weights in every pass.
__global__ void __launch_bounds__(kEvThreads) evict_select_many_kernel(const EvictArgs a) {
    __shared__ int hist[kEvBins];
    __shared__ int s_warp[32];
    __shared__ u_int64_t s_warp2[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, s_ties;
    pdl_launch_dependents();
    const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t prefix = 0;
    int need = a.n_keep;
    int shift = 32;
    bool crowded = false;
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10;
        const uint32_t high = shift == 32 ? 0u : ~0u << shift;
        shift -= bits;
        for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = 0;
        __syncthreads();
        for (int base = 0; base < a.n_rows; base += kEvThreads) {
            const int i = base + tid;
            const uint32_t k = i < a.n_rows ? evict_key(a, h, i, crowded) : 0u;
            const bool in = i < a.n_rows && (k & high) == prefix;
            const uint32_t d = (k >> shift) & ((1u << bits) - 1);
            const unsigned act = __ballot_sync(0xffffffffu, in);
            if (!act) continue;
            const uint32_t d0 = __shfl_sync(0xffffffffu, d, __ffs(act) - 1);
            const unsigned same = __ballot_sync(0xffffffffu, in && d == d0);
            if (lane == 0) atomicAdd(&hist[d0], __popc(same));
            if (in && d != d0) atomicAdd(&hist[d], 1);
        }
        __syncthreads();
        const int b1 = kEvBins - 1 - 2 * tid, b0 = b1 - 1;
        const int c1 = hist[b1], c0 = hist[b0];
        int total;
        const int before = cta_scan(c1 + c0, s_warp, total);
        if (before < need && need <= before + c1) {
            s_prefix = prefix | (uint32_t)b1 << shift;
            s_need = need - before;
            s_ties = c1;
        } else if (before + c1 < need && need <= before + c1 + c0) {
            s_prefix = prefix | (uint32_t)b0 << shift;
            s_need = need - before - c1;
            s_ties = c0;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        const int ties = s_ties;
        __syncthreads();
        if (pass == 0 && !crowded && prefix == kEvProtectedBin && need < ties) {  // as in evict_select_kernel
            crowded = true;
            prefix = 0;
            need = a.n_keep;
            shift = 32;
            pass = -1;
        }
    }
    uint32_t* above = a.masks + (size_t)h * 2 * a.words;
    uint32_t* at = above + a.words;
    for (int w = warp; w < a.words; w += kEvThreads / 32) {
        const int i = w * 32 + lane;
        const uint32_t k = i < a.n_rows ? evict_key(a, h, i, crowded) : 0u;
        const unsigned gt = __ballot_sync(0xffffffffu, i < a.n_rows && k > prefix);
        const unsigned eq = __ballot_sync(0xffffffffu, i < a.n_rows && k == prefix);
        if (lane == 0) {
            above[w] = gt;
            at[w] = eq;
        }
    }
    for (int i = tid; i < a.n_keep; i += kEvThreads) {
        if (a.weight_out != a.weight)
            a.weight_out[(size_t)h * a.out_stride + i] = a.weight[(size_t)h * a.row_stride + i];
        if (a.positions && a.positions_out != a.positions)
            a.positions_out[(size_t)h * a.out_stride + i] = a.positions[(size_t)h * a.row_stride + i];
    }
    __syncthreads();
    int32_t* count = a.moves + (size_t)h * (1 + 2 * (size_t)a.max_moves);
    int32_t* to = count + 1;
    int32_t* from = to + a.max_moves;
    int ties = 0, n_to = 0, n_from = 0;  // before this tile of words
    for (int base = 0; base < a.words; base += kEvThreads) {
        const int w = base + tid;
        uint32_t keep = w < a.words ? above[w] : 0u;
        const uint32_t eq = w < a.words ? at[w] : 0u;
        int total;
        const int before = ties + cta_scan(__popc(eq), s_warp, total);
        ties += total;
        uint32_t left = eq;
        for (int r = min(__popc(eq), max(0, need - before)); r > 0; --r) {
            keep |= left & (0u - left);
            left &= left - 1;
        }
        const int i0 = w * 32;
        const uint32_t low = i0 >= a.n_keep ? 0u : a.n_keep - i0 >= 32 ? ~0u : (1u << (a.n_keep - i0)) - 1;
        uint32_t free_bits = w < a.words ? low & ~keep : 0u;
        uint32_t move_bits = keep & ~low;
        const u_int64_t mine = (u_int64_t)__popc(free_bits) << 32 | __popc(move_bits);
        u_int64_t sum;
        const u_int64_t pre = cta_scan(mine, s_warp2, sum);
        int pt = n_to + (int)(pre >> 32), pf = n_from + (int)(uint32_t)pre;
        n_to += (int)(sum >> 32);
        n_from += (int)(uint32_t)sum;
        __syncthreads();  // the scans' arrays are read
        for (; free_bits; free_bits &= free_bits - 1) to[pt++] = i0 + __ffs(free_bits) - 1;
        for (; move_bits; move_bits &= move_bits - 1) from[pf++] = i0 + __ffs(move_bits) - 1;
    }
    if (tid == 0) *count = n_to;  // = n_from
}

constexpr int kEvMoveThreads = 256;

__global__ void __launch_bounds__(kEvMoveThreads) evict_move_kernel(const EvictArgs a) {
    const int h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    const int32_t* count = a.moves + (size_t)h * (1 + 2 * (size_t)a.max_moves);
    const int32_t* to = count + 1;
    const int32_t* from = to + a.max_moves;
    const int n = *count;
    for (int i0 = (blockIdx.x * (kEvMoveThreads / 32) + warp) * kEvMoveRows; i0 < n;
         i0 += gridDim.x * (kEvMoveThreads / 32) * kEvMoveRows)
        evict_move_rows(a, h, to, from, n, i0, lane);
}

static int evict_max_moves(int n_rows, int n_keep) { return n_keep < n_rows - n_keep ? n_keep : n_rows - n_keep; }

size_t evict_workspace_bytes(int n_rows, int n_keep, int n_kv) {
    const size_t moves = ((size_t)n_kv * (1 + 2 * (size_t)evict_max_moves(n_rows, n_keep)) * 4 + 255) / 256 * 256;
    return moves + (size_t)n_kv * 2 * ((size_t)(n_rows + 31) / 32) * 4;
}

int evict_launch(float* kc, float* vc, const float* weight, const int32_t* positions, int row_stride, int n_rows,
                 int n_keep, int recent_pos, int n_kv, int hd, float* weight_out, int32_t* positions_out,
                 int out_stride, void* ws, cudaStream_t st) {
    EvictArgs a{kc, vc, weight, positions, row_stride, n_rows, n_keep, recent_pos, n_kv, hd, weight_out, positions_out,
                out_stride, static_cast<int32_t*>(ws), evict_max_moves(n_rows, n_keep), nullptr, (n_rows + 31) / 32, false};
    a.masks = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(ws) +
                                          ((size_t)n_kv * (1 + 2 * (size_t)a.max_moves) * 4 + 255) / 256 * 256);
    if (n_rows - n_keep == 1 && n_rows <= kEvOne) {
        return launch_after(evict_one_kernel, dim3(n_kv), dim3(kEvThreads), 0, st, a) == cudaSuccess ? kOk : kErrCuda;
    }
    const int cluster = n_rows <= kEvSpread ? 1 : 8;
    const int64_t per_thread = ((int64_t)n_rows + cluster * kEvThreads - 1) / (cluster * kEvThreads);
    if (per_thread > 16) {
        evict_select_many_kernel<<<n_kv, kEvThreads, 0, st>>>(a);
        if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    } else {
        a.here = a.max_moves <= kEvHere;
        auto go = [&](auto k) { return launch_early(k, dim3(cluster, n_kv), dim3(kEvThreads), 0, st, cluster, a); };
        const cudaError_t e = cluster == 1 ? (per_thread <= 4 ? go(evict_select_kernel<4, 1>) : go(evict_select_kernel<8, 1>))
                              : per_thread <= 4 ? go(evict_select_kernel<4, 8>)
                              : per_thread <= 8 ? go(evict_select_kernel<8, 8>)
                                                : go(evict_select_kernel<16, 8>);
        if (e != cudaSuccess) return kErrCuda;
        if (a.here) return kOk;
    }
    if (a.max_moves == 0) return kOk;
    const int per_cta = kEvMoveThreads / 32 * kEvMoveRows;
    const int gx = (a.max_moves + per_cta - 1) / per_cta;
    return launch_after(evict_move_kernel, dim3(gx, n_kv), dim3(kEvMoveThreads), 0, st, a) == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace gncx
