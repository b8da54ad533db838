// tree.cu -- attention of a tree of drafted tokens over the KV cache
// (verification step of speculative decoding; no reference counterpart: the
// reference attends with one query per call, csrc/gncx_llm_kernels.cpp:1887-1994).
//
// Drafted node i has its K/V row at cache row pos0 + i, its parent at
// parents[i] < i (-1: the last cached token) and the position
// pos0 + depth(i).  Its query sees the cached rows 0 .. pos0 - 1 and its
// ancestors and itself, with a sliding window W only rows whose position is
// above its own minus W:
//   o = sum_j softmax_j(scale q.k_j) v_j over those rows.
//
// The rows that every node sees are one dense range [lo, pos0) (lo = 0, or with
// a window the first row that even the deepest possible node, at position
// pos0 + n_tok - 1, sees).  tree_dense_kernel computes that range split over
// CTAs, with no mask, and leaves a record {max, sum, o} per (query row,
// split).  tree_merge_kernel, a CTA per (node, KV head) or part of the head's
// group, walks the node's remaining rows one by one -- window rows below lo, then
// its ancestors, whose list it builds from the parents -- and merges the records.
// Rows that a node does not see are never read for it, so what they hold (NaN,
// infinities, another branch) cannot reach its output.
//
// tree_tc.cu has the dense range's kernel on the tensor cores, for head sizes that
// are multiples of 16; tree_dense_kernel serves the others.  It is bound by
// shared memory: a 16-byte read per 4 (values) to 13 (scores) multiply-adds; 12
// heads, 4 KV heads of 136, 16 nodes over 8192 rows: 112 us with the merge, 0.32 TB/s.
// (The tensor-core kernel loads, pads and stores in steps of four columns, so that it
// could take these sizes too; it has not been measured on them.)  The merge
// is bound by the latency of its dependent reads (parents, rows, records: 10 us
// alone and cold, under ncu, for 33 nodes and 8 KV heads), so all that comes before the
// records runs before it waits for the dense kernel, and a thread has eight
// records in flight: 5 nodes over 511 rows, both kernels 10.2 us.
//
// Few query rows over a short cache take one launch, tree_one_kernel, a cluster
// of CTAs on the CUDA cores: bound by its chain of reads, sums over lanes and
// cluster barriers, and by 0.9 us for each 2 (4) cache rows of a warp.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "rows.cuh"
#include "tma.cuh"
#include "tree.cuh"

namespace gncx {

// ---------------------------------------------------------------- dense range, CUDA cores
constexpr int kTdRows = 32;     // query rows (node, head of the group) per CTA
constexpr int kTdKeys = 32;     // cache rows per tile
constexpr int kTdThreads = 256; // 8 threads per query row

static size_t tree_dense_smem(int hd) {
    return ((size_t)(kTdRows + 2 * kTdKeys) * (hd + 4) + kTdRows * (kTdKeys + 1)) * 4;
}

__global__ void __launch_bounds__(kTdThreads) tree_dense_kernel(const TreeArgs a) {
    extern __shared__ __align__(16) float sm[];
    const int ld = a.hd + 4, hd4 = a.hd / 4;
    float* qs = sm;
    float* ks = qs + kTdRows * ld;
    float* vs = ks + kTdKeys * ld;
    float* ps = vs + kTdKeys * ld;
    pdl_wait();
    pdl_launch_dependents();  // after the wait: the second kernel reads inputs before it waits for this one
    const int split = blockIdx.x, kvh = blockIdx.y, r0 = blockIdx.z * kTdRows;
    const int rows = a.n_tok * a.G;
    const int tid = threadIdx.x, r = tid >> 3, c = tid & 7;
    const size_t pstride = (size_t)a.n_kv * a.hd;
    for (int i = tid; i < kTdRows * hd4; i += kTdThreads) {
        const int rr = i / hd4, x = i - rr * hd4, row = r0 + rr;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < rows)
            v = *reinterpret_cast<const float4*>(a.q + ((size_t)(row / a.G) * a.n_heads + kvh * a.G + row % a.G) * a.hd + 4 * x);
        *reinterpret_cast<float4*>(qs + rr * ld + 4 * x) = v;
    }
    const int j0 = a.lo + split * a.per, j1 = min(a.pos0, j0 + a.per);
    float m = -INFINITY, l = 0.0f;
    float4 o[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = j0; base < j1; base += kTdKeys) {
        __syncthreads();
        for (int i = tid; i < kTdKeys * hd4; i += kTdThreads) {
            const int jj = i / hd4, x = i - jj * hd4;
            float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
            if (base + jj < j1) {
                const size_t at = (size_t)(base + jj) * pstride + (size_t)kvh * a.hd + 4 * x;
                k = *reinterpret_cast<const float4*>(a.kc + at);
                v = *reinterpret_cast<const float4*>(a.vc + at);
            }
            *reinterpret_cast<float4*>(ks + jj * ld + 4 * x) = k;
            *reinterpret_cast<float4*>(vs + jj * ld + 4 * x) = v;
        }
        __syncthreads();
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int x = 0; x < hd4; ++x) {
            const float4 q4 = *reinterpret_cast<const float4*>(qs + r * ld + 4 * x);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 k4 = *reinterpret_cast<const float4*>(ks + (c + 8 * k) * ld + 4 * x);
                s[k] = fmaf(q4.w, k4.w, fmaf(q4.z, k4.z, fmaf(q4.y, k4.y, fmaf(q4.x, k4.x, s[k]))));
            }
        }
        float bm = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s[k] = base + c + 8 * k < j1 ? s[k] * a.scale2 : -INFINITY;
            bm = fmaxf(bm, s[k]);
        }
#pragma unroll
        for (int x = 4; x > 0; x >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, x));
        const float m_new = fmaxf(m, bm);
        const float corr = m == -INFINITY ? 0.0f : ex2(m - m_new);
        float bs = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float e = s[k] == -INFINITY ? 0.0f : ex2(s[k] - m_new);
            bs += e;
            ps[r * (kTdKeys + 1) + c + 8 * k] = e;
        }
#pragma unroll
        for (int x = 4; x > 0; x >>= 1) bs += __shfl_xor_sync(0xffffffffu, bs, x);
        l = fmaf(l, corr, bs);
        m = m_new;
        __syncwarp();  // a row's eight threads are in one warp
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const int col = c + 8 * x;
            if (col >= hd4) break;
            float4 acc = o[x];
            acc.x *= corr; acc.y *= corr; acc.z *= corr; acc.w *= corr;
            for (int k = 0; k < min(kTdKeys, j1 - base); ++k) {
                const float p = ps[r * (kTdKeys + 1) + k];
                const float4 v4 = *reinterpret_cast<const float4*>(vs + k * ld + 4 * col);
                acc.x = fmaf(p, v4.x, acc.x);
                acc.y = fmaf(p, v4.y, acc.y);
                acc.z = fmaf(p, v4.z, acc.z);
                acc.w = fmaf(p, v4.w, acc.w);
            }
            o[x] = acc;
        }
        __syncwarp();
    }
    if (r0 + r >= rows) return;
    float* rec = a.part + (((size_t)kvh * rows + r0 + r) * a.splits + split) * (a.hd + 4);
    if (c == 0) {
        rec[0] = m;
        rec[1] = l;
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const int col = c + 8 * x;
        if (col < hd4) *reinterpret_cast<float4*>(rec + 4 + 4 * col) = o[x];
    }
}

// ---------------------------------------------------------------- few rows: everything in one launch
constexpr int kToThreads = 256;
constexpr int kToWarps = kToThreads / 32;
constexpr int kToCluster = 8;  // CTAs per KV head and GT query rows
constexpr int kToTok = 64;     // nodes: a bit each

// A cluster takes GT query rows (node, head of the group) of a KV head and all
// rows that any of them sees, the drafted ones too.  A warp holds B cache rows
// across its lanes (NJ float4 each) and scores them against the GT query rows,
// one (cache row, query row) score per lane; what a query row does not see gets
// no weight, and no product with V.  The warps' and the CTAs' sums are joined in
// shared memory.
template <int NJ, int GT, int B>
__global__ void __launch_bounds__(kToThreads, 1) tree_one_kernel(const TreeArgs a) {
    static_assert(GT * B == 32, "a score per lane");
    extern __shared__ __align__(16) float sm[];  // [warp][GT][hd]
    __shared__ int s_up[kToTok], s_first[GT];
    __shared__ unsigned long long s_path[GT];
    __shared__ __align__(16) float wsh[kToWarps][32 + GT];
    __shared__ float mst[kToWarps][GT], lst[kToWarps][GT];
    __shared__ float2 s_ml[GT];
    __shared__ float s_inv[GT], s_f[GT][kToCluster];
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int rank = blockIdx.x, kvh = blockIdx.y, r0 = blockIdx.z * GT;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows = a.n_tok * a.G, heads = min(GT, rows - r0);
    auto row_at = [&](int g) {  // of q and out; the last row again behind the last
        const int r = min(r0 + g, rows - 1);
        return ((size_t)(r / a.G) * a.n_heads + kvh * a.G + r % a.G) * a.hd;
    };
    pdl_wait();
    if (tid < a.n_tok) s_up[tid] = a.parents[tid];
    f32x2 q[GT][2 * NJ], o[GT][2 * NJ];
    {
        int head = r0 % a.G;
        const float* qp = a.q + row_at(0);
#pragma unroll
        for (int g = 0; g < GT; ++g) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int col = 4 * (lane + 32 * j);
                const float4 x = ld_row(qp + col, col < a.hd);
                q[g][2 * j] = pack2(x.x, x.y);
                q[g][2 * j + 1] = pack2(x.z, x.w);
                o[g][2 * j] = o[g][2 * j + 1] = 0;
            }
            if (g + 1 < heads) {
                qp += a.hd;
                if (++head == a.G) {
                    head = 0;
                    qp += (size_t)(a.n_heads - a.G) * a.hd;
                }
            }
        }
    }
    __syncthreads();
    if (tid < GT) {  // what the query row sees: cache rows from `first` on, drafted rows by their bits
        int depth = -1, i = min(r0 + tid, rows - 1) / a.G;
        unsigned long long path = 0;
        while (true) {
            ++depth;
            if (a.window <= 0 || depth < a.window) path |= 1ull << i;
            const int p = s_up[i];
            if (p < -1 || p >= i) record_error(a.err, kErrInvalidArg);
            if (p < 0 || p >= i) break;
            i = p;
        }
        s_path[tid] = path;
        s_first[tid] = a.window > 0 ? max(0, a.pos0 + depth - a.window + 1) : 0;
    }
    __syncthreads();
    const int g_me = lane % GT, p_me = lane / GT, first = s_first[g_me];
    const unsigned long long path = s_path[g_me];
    const int k0 = a.window > 0 ? min(a.pos0, max(0, a.pos0 - a.window + 1)) : 0, k1 = a.pos0 + a.n_tok;
    const int per = (k1 - k0 + kToCluster - 1) / kToCluster;
    const int p0 = k0 + rank * per, p1 = min(k1, p0 + per);
    const size_t ps = (size_t)a.n_kv * a.hd;
    const float* kb = a.kc + (size_t)kvh * a.hd;
    const float* vb = a.vc + (size_t)kvh * a.hd;
    float m = -INFINITY, l = 0.0f;  // of query row g_me
    // the scores of batch b0 that count, and the rows that any of them needs
    auto seen_at = [&](int b0) {
        const int key = b0 + p_me;
        return key < p1 && (key < a.pos0 ? key >= first : (path >> (key - a.pos0) & 1) != 0);
    };
    float4 k[B][NJ], v[B][NJ];
    auto load = [&](int b0, unsigned mask) {
#pragma unroll
        for (int p = 0; p < B; ++p)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int col = 4 * (lane + 32 * j);
                const bool some = col < a.hd && (mask >> (p * GT) & ((1u << GT) - 1));
                k[p][j] = ld_row(kb + (size_t)(b0 + p) * ps + col, some);
                v[p][j] = ld_row(vb + (size_t)(b0 + p) * ps + col, some);
            }
    };
    bool seen = seen_at(p0 + warp * B);
    unsigned mask = __ballot_sync(0xffffffffu, seen);
    load(p0 + warp * B, mask);
#pragma unroll 1
    for (int b0 = p0 + warp * B; b0 < p1;) {
        f32x2 kk[B][2 * NJ], vv[B][2 * NJ];
#pragma unroll
        for (int p = 0; p < B; ++p)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                kk[p][2 * j] = pack2(k[p][j].x, k[p][j].y);
                kk[p][2 * j + 1] = pack2(k[p][j].z, k[p][j].w);
                vv[p][2 * j] = pack2(v[p][j].x, v[p][j].y);
                vv[p][2 * j + 1] = pack2(v[p][j].z, v[p][j].w);
            }
        const bool seen_now = seen;
        const unsigned now = mask;
        b0 += kToWarps * B;
        seen = seen_at(b0);
        mask = __ballot_sync(0xffffffffu, seen);
        load(b0, mask);  // the next batch, under this one's arithmetic
        if (!now) continue;
        float d[32];
#pragma unroll
        for (int p = 0; p < B; ++p)
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                f32x2 c = mul2(q[g][0], kk[p][0]);
#pragma unroll
                for (int j = 1; j < 2 * NJ; ++j) c = fma2(q[g][j], kk[p][j], c);
                const float2 s = unpack2(c);
                d[p * GT + g] = s.x + s.y;
            }
        float sc = lanes_reduce<32, 32>(d, lane) * a.scale2;
        if (!seen_now) sc = -INFINITY;
        float bm = sc;
#pragma unroll
        for (int off = 16; off >= GT; off >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, off));
        const float m_new = fmaxf(m, bm);
        const float e = sc == -INFINITY ? 0.0f : ex2(sc - m_new);
        const float corr = m == -INFINITY ? 0.0f : ex2(m - m_new);
        float bs = e;
#pragma unroll
        for (int off = 16; off >= GT; off >>= 1) bs += __shfl_xor_sync(0xffffffffu, bs, off);
        l = fmaf(l, corr, bs);
        m = m_new;
        float* wr = wsh[warp];
        wr[lane] = e;
        if (lane < GT) wr[32 + lane] = corr;
        __syncwarp();
        if (__any_sync(0xffffffffu, corr != 1.0f)) {
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const f32x2 c = pack2(wr[32 + g], wr[32 + g]);
#pragma unroll
                for (int j = 0; j < 2 * NJ; ++j) o[g][j] = mul2(o[g][j], c);
            }
        }
#pragma unroll
        for (int p = 0; p < B; ++p)
#pragma unroll
            for (int g = 0; g < GT; g += 4) {
                const float4 w4 = *reinterpret_cast<const float4*>(wr + p * GT + g);
                const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (now >> (p * GT + g + x) & 1) {  // of the warp
                        const f32x2 w2 = pack2(w[x], w[x]);
#pragma unroll
                        for (int j = 0; j < 2 * NJ; ++j) o[g + x][j] = fma2(w2, vv[p][j], o[g + x][j]);
                    }
            }
        __syncwarp();
    }
    if (lane < GT) {
        mst[warp][lane] = m;
        lst[warp][lane] = l;
    }
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int col = 4 * (lane + 32 * j);
            const float2 x = unpack2(o[g][2 * j]), y = unpack2(o[g][2 * j + 1]);
            if (col < a.hd) *reinterpret_cast<float4*>(sm + (size_t)(warp * GT + g) * a.hd + col) = make_float4(x.x, x.y, y.x, y.y);
        }
    __syncthreads();
    // the warps' states as the CTA's record, in place of warp 0's outputs
    for (int t = tid; t < heads * a.hd; t += kToThreads) {
        const int g = t / a.hd;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kToWarps; ++w) M = fmaxf(M, mst[w][g]);
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < kToWarps; ++w) {
            const float f = mst[w][g] == -INFINITY ? 0.0f : ex2(mst[w][g] - M);
            L = fmaf(lst[w][g], f, L);  // a NaN stays
            O = fmaf(sm[(size_t)w * GT * a.hd + t], f, O);
        }
        sm[t] = O;
        if (t == g * a.hd) s_ml[g] = make_float2(M, L);
    }
    cluster.sync();
    for (int g = warp; g < heads; g += kToWarps) {
        const float2 ml = lane < kToCluster ? *cluster.map_shared_rank(&s_ml[g], lane) : make_float2(-INFINITY, 0.0f);
        float M = ml.x;
#pragma unroll
        for (int off = kToCluster / 2; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
        const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
        float L = ml.y * f;
#pragma unroll
        for (int off = kToCluster / 2; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
        if (lane < kToCluster) s_f[g][lane] = f;
        if (lane == 0) s_inv[g] = 1.0f / L;
    }
    __syncthreads();
    for (int t = rank * kToThreads + tid; t < heads * a.hd; t += kToCluster * kToThreads) {
        const int g = t / a.hd;
        float out = 0.0f;
#pragma unroll
        for (int r = 0; r < kToCluster; ++r) out = fmaf(*cluster.map_shared_rank(&sm[t], r), s_f[g][r], out);
        a.out[row_at(g) + t - g * a.hd] = out * s_inv[g];
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
}

// ---------------------------------------------------------------- ancestors and merge
constexpr int kTmThreads = 256;
constexpr int kTmWarps = kTmThreads / 32;
constexpr int kTmHeads = 4;  // query heads of the group at a time

// NJ float4 columns per lane: head_dim <= 128 * NJ
template <int NJ>
__global__ void __launch_bounds__(kTmThreads) tree_merge_kernel(const TreeArgs a) {
    extern __shared__ __align__(16) float sm[];
    float* os = sm;                                                // [warp][kTmHeads][hd]
    int* up = reinterpret_cast<int*>(os + kTmWarps * kTmHeads * a.hd); // parents, then
    int* chain = up + a.n_tok;                                     // the path from the node up
    __shared__ float s_m[kTmWarps][kTmHeads], s_l[kTmWarps][kTmHeads];
    __shared__ float2 ml_g[kTmThreads];
    __shared__ int s_len;
    const int node = blockIdx.x, kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows = a.n_tok * a.G, rl = a.hd + 4;
    // What is read before the wait is read from L2: the kernels before the dense one
    // have completed, as it has waited for them before it let this one start.
    for (int i = tid; i <= node; i += kTmThreads) up[i] = __ldcg(a.parents + i);
    __syncthreads();
    if (tid == 0) {  // parents are below their children, so the walk ends
        int n = 0, i = node;
        while (true) {
            chain[n++] = i;
            const int p = up[i];
            if (p < -1 || p >= i) record_error(a.err, kErrInvalidArg);
            if (p < 0 || p >= i) break;
            i = p;
        }
        s_len = n;
    }
    __syncthreads();
    const int depth = s_len - 1;                // of this node
    const int first = a.window > 0 ? max(0, a.pos0 + depth - a.window + 1) : 0;  // lowest position seen
    const int n_win = max(0, min(a.lo, a.pos0) - first);                     // cached rows below the dense range
    const int n_anc = min(depth + 1, a.pos0 + depth - first + 1);            // of the path, from the node up
    const int n_keys = n_win + n_anc;
    const size_t pstride = (size_t)a.n_kv * a.hd;
    const float* kb = a.kc + (size_t)kvh * a.hd;
    const float* vb = a.vc + (size_t)kvh * a.hd;
    bool waited = false;
    const int g_end = min(a.G, ((int)blockIdx.z + 1) * a.merge_heads);
    for (int g0 = blockIdx.z * a.merge_heads; g0 < g_end; g0 += kTmHeads) {
        const int heads = min(kTmHeads, g_end - g0);
        float4 q[kTmHeads][NJ], o[kTmHeads][NJ];
        float m[kTmHeads], l[kTmHeads];
#pragma unroll
        for (int g = 0; g < kTmHeads; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.0f;
            const float* qp = a.q + ((size_t)node * a.n_heads + kvh * a.G + g0 + min(g, heads - 1)) * a.hd;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int col = 4 * (lane + 32 * j);
                q[g][j] = col < a.hd ? __ldcg(reinterpret_cast<const float4*>(qp + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
                o[g][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        for (int x = warp; x < n_keys; x += kTmWarps) {
            const int row = x < n_win ? first + x : a.pos0 + chain[x - n_win];
            float4 k[NJ], v[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int col = 4 * (lane + 32 * j);
                k[j] = v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (col < a.hd) {
                    k[j] = __ldcg(reinterpret_cast<const float4*>(kb + (size_t)row * pstride + col));
                    v[j] = __ldcg(reinterpret_cast<const float4*>(vb + (size_t)row * pstride + col));
                }
            }
            float s[kTmHeads];
#pragma unroll
            for (int g = 0; g < kTmHeads; ++g) {
                s[g] = 0.0f;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    s[g] = fmaf(q[g][j].w, k[j].w, fmaf(q[g][j].z, k[j].z, fmaf(q[g][j].y, k[j].y, fmaf(q[g][j].x, k[j].x, s[g]))));
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1)
#pragma unroll
                for (int g = 0; g < kTmHeads; ++g) s[g] += __shfl_xor_sync(0xffffffffu, s[g], w);
#pragma unroll
            for (int g = 0; g < kTmHeads; ++g) {
                const float sc = s[g] * a.scale2;
                const float mn = fmaxf(m[g], sc);
                const float e = sc == -INFINITY ? 0.0f : ex2(sc - mn);
                const float corr = m[g] == -INFINITY ? 0.0f : ex2(m[g] - mn);
                m[g] = mn;
                l[g] = fmaf(l[g], corr, e);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    o[g][j].x = fmaf(e, v[j].x, o[g][j].x * corr);
                    o[g][j].y = fmaf(e, v[j].y, o[g][j].y * corr);
                    o[g][j].z = fmaf(e, v[j].z, o[g][j].z * corr);
                    o[g][j].w = fmaf(e, v[j].w, o[g][j].w * corr);
                }
            }
        }
        if (lane == 0)
#pragma unroll
            for (int g = 0; g < kTmHeads; ++g) {
                s_m[warp][g] = m[g];
                s_l[warp][g] = l[g];
            }
#pragma unroll
        for (int g = 0; g < kTmHeads; ++g)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int col = 4 * (lane + 32 * j);
                if (col < a.hd) *reinterpret_cast<float4*>(os + (warp * kTmHeads + g) * a.hd + col) = o[g][j];
            }
        __syncthreads();
        if (!waited) pdl_wait();  // the dense kernel's records
        waited = true;
        // Four columns per thread; where there are threads to spare, groups of them
        // take every groups-th record, group 0 the warps' states too.  Each thread
        // merges with a maximum of its own, so that all its loads are in flight at once.
        const int hd4 = a.hd / 4, items = heads * hd4;
        const int groups = min(8, max(1, kTmThreads / items));
        const int grp = tid / items, it = tid - grp * items;
        const int g = it / hd4, c = it - g * hd4;
        float M = -INFINITY, sum = 0.0f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto join = [&](float m, float l, const float4& v) {
            const float Mn = fmaxf(M, m);
            const float f = M == -INFINITY ? 0.0f : ex2(M - Mn), e = m == -INFINITY ? 0.0f : ex2(m - Mn);
            // a record without a weight may hold no number: NaN sums (and no others) count all the same
            M = Mn;
            sum = fmaf(sum, f, l * e);
            acc.x = fmaf(acc.x, f, v.x * e);
            acc.y = fmaf(acc.y, f, v.y * e);
            acc.z = fmaf(acc.z, f, v.z * e);
            acc.w = fmaf(acc.w, f, v.w * e);
        };
        if (grp < groups) {
            constexpr int kBatch = 8;
            const float* rec = a.part + ((size_t)kvh * rows + node * a.G + g0 + g) * a.splits * rl;
            for (int s0 = grp; s0 < a.splits; s0 += kBatch * groups) {
                float2 ml[kBatch];
                float4 v[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int s = min(s0 + i * groups, a.splits - 1);
                    ml[i] = *reinterpret_cast<const float2*>(rec + (size_t)s * rl);
                    v[i] = *reinterpret_cast<const float4*>(rec + (size_t)s * rl + 4 + 4 * c);
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (s0 + i * groups < a.splits) join(ml[i].x, ml[i].y, v[i]);
            }
            if (grp == 0)
#pragma unroll
                for (int w = 0; w < kTmWarps; ++w)
                    join(s_m[w][g], s_l[w][g], *reinterpret_cast<const float4*>(os + (w * kTmHeads + g) * a.hd + 4 * c));
        }
        if (groups > 1) {
            __syncthreads();  // the warps' states are merged: their place holds the groups'
            float4* sums = reinterpret_cast<float4*>(os);
            if (grp > 0 && grp < groups) {
                sums[tid - items] = acc;
                ml_g[tid - items] = make_float2(M, sum);
            }
            __syncthreads();
            if (grp == 0)
                for (int k = 0; k < groups - 1; ++k) join(ml_g[k * items + it].x, ml_g[k * items + it].y, sums[k * items + it]);
        }
        if (grp == 0) {
            const float f = 1.0f / sum;
            *reinterpret_cast<float4*>(a.out + ((size_t)node * a.n_heads + kvh * a.G + g0 + g) * a.hd + 4 * c) =
                make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host
// First row of the dense range, its splits and rows per split.
static void tree_geometry(TreeArgs& a, int sm_count) {
    const int64_t lo = a.window > 0 ? (int64_t)a.pos0 + a.n_tok - a.window : 0;
    a.lo = lo < 0 ? 0 : lo > a.pos0 ? a.pos0 : (int)lo;
    const int len = a.pos0 - a.lo;
    a.tc = tree_tc_ok(a.hd);
    const int qrows = a.tc ? tree_tc_rows(a.hd) : kTdRows, keys = a.tc ? tree_tc_keys(a.hd) : kTdKeys;
    const int64_t ctas = (int64_t)a.n_kv * ((a.n_tok * a.G + qrows - 1) / qrows);  // per split
    // CUDA cores: about two CTAs per SM; tensor cores: one per SM, in one wave
    int want = (int)(a.tc ? sm_count / ctas : (2 * (int64_t)sm_count + ctas - 1) / ctas);
    if (want < 1) want = 1;
    const int most = (len + keys - 1) / keys;
    if (want > most) want = most;
    a.splits = a.max_splits = want;
    a.per = 0;
    if (want > 0) {
        a.per = ((len + want - 1) / want + keys - 1) / keys * keys;
        a.splits = (len + a.per - 1) / a.per;
    }
}

// Query rows per cluster where one launch does everything, 0 where not: the clusters
// run side by side (15 of 8 CTAs do, 16 took twice the time) and the cache is short.
// One launch against the two kernels: 16 heads, 8 KV heads of 128, 4 nodes (8 query
// rows): 10 cache rows 5.8 us and 10.6, 511 rows 8.1 and 10.1, 700 rows 8.7 and
// 10.5; on 2 KV heads of 64, 700 rows 7.9 and 8.4, 1000 rows 8.9 and 8.7.  5 nodes
// (16 rows per cluster): 256 rows 9.0 and 10.0, 384 rows 9.9 and 10.2, 511 rows 10.9
// and 10.4.  Head size 256: 128 rows 8.3 and 11.0, 256 rows 10.1 and 11.1, 384 rows 10.9
// and 11.2.
static int tree_one_rows(const TreeArgs& a, int sm_count) {
    const int64_t len = (int64_t)a.pos0 + a.n_tok - (a.window > 0 ? max(0, a.pos0 - a.window + 1) : 0);
    const int64_t fit = sm_count * 13 / 16 / kToCluster / a.n_kv;  // clusters per KV head
    const int rows = a.n_tok * a.G;
    if (a.n_tok > kToTok) return 0;
    if (rows <= 8 * fit) return len <= (a.hd > 128 ? 256 : 768) ? 8 : 0;
    return rows <= 16 * fit && a.hd <= 128 && len <= 384 ? 16 : 0;
}

static TreeArgs tree_args(int pos0, int n_tok, int n_heads, int n_kv, int hd, int window) {
    TreeArgs a{};
    a.pos0 = pos0;
    a.n_tok = n_tok;
    a.n_heads = n_heads;
    a.n_kv = n_kv;
    a.hd = hd;
    a.G = n_heads / n_kv;
    a.window = window;
    tree_geometry(a, device_info().sm_count);
    return a;
}

size_t tree_workspace_bytes(int pos0, int n_tok, int n_heads, int n_kv, int hd, int window) {
    const TreeArgs a = tree_args(pos0, n_tok, n_heads, n_kv, hd, window);
    return (size_t)n_heads * n_tok * a.max_splits * (hd + 4) * 4;
}

int tree_launch(const float* q, const float* kc, const float* vc, const int32_t* parents, int pos0, int n_tok,
                int n_heads, int n_kv, int hd, float scale, int window, float* out, void* ws, int32_t* err,
                cudaStream_t st) {
    TreeArgs a = tree_args(pos0, n_tok, n_heads, n_kv, hd, window);
    a.q = q;
    a.kc = kc;
    a.vc = vc;
    a.parents = parents;
    a.scale2 = scale * 1.4426950408889634f;
    a.part = static_cast<float*>(ws);
    a.out = out;
    a.err = err;
    if (const int gt = tree_one_rows(a, device_info().sm_count)) {
        auto one = [&](auto k) {
            const size_t smem = (size_t)kToWarps * gt * hd * 4;
            if (set_smem_limit(k, smem) != cudaSuccess) return kErrCuda;
            const dim3 grid(kToCluster, n_kv, (n_tok * a.G + gt - 1) / gt);
            return launch_early(k, grid, dim3(kToThreads), smem, st, kToCluster, a) == cudaSuccess ? kOk : kErrCuda;
        };
        return hd > 128 ? one(tree_one_kernel<2, 8, 4>) : gt == 8 ? one(tree_one_kernel<1, 8, 4>) : one(tree_one_kernel<1, 16, 2>);
    }
    if (a.splits > 0 && a.tc) {
        if (tree_tc_launch(a, st) != cudaSuccess) return kErrCuda;
    } else if (a.splits > 0) {
        const size_t smem = tree_dense_smem(hd);
        if (set_smem_limit(tree_dense_kernel, smem) != cudaSuccess) return kErrCuda;
        const int tiles = (n_tok * a.G + kTdRows - 1) / kTdRows;
        if (launch_after(tree_dense_kernel, dim3(a.splits, n_kv, tiles), dim3(kTdThreads), smem, st, a) != cudaSuccess)
            return kErrCuda;
    }
    const size_t msm = ((size_t)kTmWarps * kTmHeads * hd + 2 * n_tok) * 4;
    // Heads of a group share the CTA that walks a node's rows; spread over more
    // CTAs only as far as these fit the SMs (8 heads on one KV head, 16 nodes,
    // 65536 rows, 147 records each: 64 us with the 8 together, 34 apart; 16 heads, 4
    // KV heads, 25 nodes, window 1024: 10.2 us as it is, 13.0 with 200 CTAs).
    a.merge_heads = a.G;
    const auto ctas = [&](int heads) { return (int64_t)n_tok * n_kv * ((a.G + heads - 1) / heads); };
    while (a.merge_heads > 1 && ctas((a.merge_heads + 1) / 2) <= device_info().sm_count) a.merge_heads = (a.merge_heads + 1) / 2;
    const dim3 grid(n_tok, n_kv, (a.G + a.merge_heads - 1) / a.merge_heads);
    auto go = [&](auto k) {
        if (set_smem_limit(k, msm) != cudaSuccess) return kErrCuda;
        if (a.splits > 0) return launch_after(k, grid, dim3(kTmThreads), msm, st, a) == cudaSuccess ? kOk : kErrCuda;
        k<<<grid, kTmThreads, msm, st>>>(a);
        return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
    };
    return hd <= 128 ? go(tree_merge_kernel<1>) : go(tree_merge_kernel<2>);
}

}  // namespace gncx
