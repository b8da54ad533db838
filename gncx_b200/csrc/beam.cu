// beam.cu -- beam search's selection over beams and vocabulary, and the
// in-place reordering of per-slot state that follows it (and that follows the
// verification of a drafted tree).  No reference counterpart: the reference
// samples one sequence greedily (lua/gncx_streamer.lua:1229-1273).
//
// Selection.  Beam b's candidates are its tokens t with the score
//   c(b, t) = scores[b] + (x[b][t] - L_b),  L_b = log sum_t exp(x[b][t]),
// in double precision; an ended beam has the one candidate (eos, scores[b]).
// The order is total: score descending, then beam, then logit descending,
// then token, so that the chosen parents and tokens do not depend on how the
// work was split.
//   * beam_part_kernel: one CTA per (part of the vocabulary, beam) reads its
//     logits once.  It keeps sum exp(x - ref) per thread (terms and sums in
//     double: an error of 1e-7 in L_b, as fp32 terms give, could swap two
//     beams' candidates) and a list of the part's best n_out logits: a
//     threshold T that at least n_out seen elements reach, at first from the
//     threads' maxima, filters what is appended.  It writes the list sorted.
//   * beam_merge_kernel: one CTA forms the L_b and walks the sorted lists, a
//     thread (or several) per list, past a threshold from their first entries, until no
//     list has an entry that reaches it; then it ranks what it found.
// The first kernel is bound by instruction issue (about 60 % busy, 45 instructions a
// logit, a third of them the exponential): 25.8 us for 64 beams of 151936 logits, 9
// of them ended, 1.3 TB/s.  The merge is one CTA's chain of dependent reads and
// barriers, alone and cold, under ncu, 10 us for 4 beams and 13 for 64.  Both: 30.7 us;
// 4 beams 12.8 us.  Slower:
// appending by a ballot per logit (48.7 us against 34.7 then), two CTAs per SM
// (31.3 us), more than fit it (4: 9 % slower).
#include <cuda_runtime.h>
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "tma.cuh"

namespace gncx {

constexpr int kBsThreads = 256;
constexpr int kBsPer = 16;
constexpr int kBsTile = kBsThreads * kBsPer;
constexpr int kBsSort = 1024;             // largest list that is sorted
constexpr int kBsList = kBsSort + kBsTile;
constexpr int kBsCtasPerSm = 3;           // that a vocabulary is split for, and that fit one
// From fewer than so many parts for each beam the division follows the number of
// beams that have not ended: 64 beams, 9 of them ended, 30.7 us against 34.4 (none
// ended: 34.8 and 34.0); with more parts it gains less than reading the flags costs.
constexpr int kBsShare = 16;
constexpr int kBmThreads = 1024;
constexpr int kBmList = 2 * kBmThreads;

using u64 = unsigned long long;

// fp32 as an unsigned integer in the same order (-0 as +0; a NaN anywhere)
__device__ __forceinline__ uint32_t ord32(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unord32(uint32_t o) {
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
// The greater value; NaN if one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ u64 ord64(double x) {
    const u64 u = (u64)__double_as_longlong(x + 0.0);
    return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double unord64(u64 o) {
    return __longlong_as_double((long long)(o ^ ((o >> 63) ? 1ull << 63 : ~0ull)));
}

// Descending bitonic sort of list[0, P), P a power of two; whole CTA.
template <class Key>
__device__ __forceinline__ void bitonic_desc(Key* list, int P) {
    for (int k = 2; k <= P; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < P / 2; i += blockDim.x) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const Key x = list[a], y = list[b];
                const bool down = (a & k) == 0;
                if ((x < y) == down) {
                    list[a] = y;
                    list[b] = x;
                }
            }
        }
    __syncthreads();
}

// How the vocabulary is divided: into `parts` for each beam or, where `share` is
// set, on the device into as many as give at most `room` lists of the beams that
// have not ended.
struct BeamSplit {
    int room, parts, per;
    bool share;
};
__host__ __device__ inline int beam_parts(int live, int vocab, int room) {
    const int tiles = (vocab + kBsTile - 1) / kBsTile, most = room / (live > 1 ? live : 1);
    return tiles < most ? tiles : most > 1 ? most : 1;
}

// The beams that have not ended: their number, and s_beam[i] the i-th of them.
// Whole CTA of at least kBeamMax threads.
__device__ __forceinline__ int beam_live(const int32_t* finished, int n_beam, int* s_beam) {
    __shared__ unsigned s_on[kBeamMax / 32];
    const int tid = threadIdx.x;
    const bool on = tid < n_beam && !__ldcg(finished + tid);
    const unsigned mine = __ballot_sync(0xffffffffu, on);
    if (tid < kBeamMax && (tid & 31) == 0) s_on[tid >> 5] = mine;
    __syncthreads();
    int total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kBeamMax / 32; ++w) {
        const int c = __popc(s_on[w]);
        if (w < tid >> 5) before += c;
        total += c;
    }
    if (on) s_beam[before + __popc(mine & ((1u << (tid & 31)) - 1))] = tid;
    __syncthreads();
    return total;
}

struct BeamPart {
    double sum;  // sum of exp(x - ref) over the part; NaN when a logit is NaN or +inf
    float ref;   // about the part's largest logit; -inf: all are
    int pad;
};

// e^y for y in [-700, 700], off by less than 1e-11 of it: y = n ln2 + r with
// |r| <= ln2 / 2, and the Taylor polynomial of e^r to r^9 (r^10 / 10! < 7e-12).
__device__ __forceinline__ double exp_taylor(double y) {
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double t = fma(y, 1.4426950408889634, magic);
    const double r = fma(t - magic, -0.6931471805599453, y);
    double p = 1.0 / 362880;
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

// e^y for the sums over a vocabulary, with fewer double-precision operations:
// y = n ln2 / 16 + r, |r| <= 0.0217, the polynomial to r^4 (r^5 / 120 < 5e-11)
// and tab[k] = 2^(k / 16).
__device__ __forceinline__ double exp_tab(double y, const double* tab) {
    const double magic = 6755399441055744.0;
    const double t = fma(y, 16 * 1.4426950408889634, magic);
    const double r = fma(t - magic, -0.6931471805599453 / 16, y);
    double p = 1.0 / 24;
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const int n = __double2loint(t);
    p *= tab[n & 15];
    return __hiloint2double(__double2hiint(p) + ((n >> 4) << 20), __double2loint(p));
}

// log l of a sum of exponentials (e^-700 < l < 1e38): a Newton step in double
// from the fp32 logarithm y, log l = y + log(l e^-y), with l e^-y near 1.
__device__ __forceinline__ double log_of_sum(double l) {
    if (!(l > 0.0)) return l == 0.0 ? -INFINITY : NAN;
    const double y = (double)logf((float)l);
    const double d = fma(l, exp_taylor(-y), -1.0);
    return y + (d - 0.5 * d * d);
}

// The k-th largest (k = 1..32) of the warp's values, by a bitonic sort over its lanes.
__device__ __forceinline__ uint32_t warp_kth(uint32_t v, int k, int lane) {
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
        for (int j = n >> 1; j > 0; j >>= 1) {
            const uint32_t o = __shfl_xor_sync(0xffffffffu, v, j);
            const bool up = ((lane & n) == 0) == ((lane & j) == 0);  // this lane keeps the larger
            v = up ? max(v, o) : min(v, o);
        }
    return __shfl_sync(0xffffffffu, v, k - 1);
}

// Keep the n largest of list[0, cnt) (distinct keys, kBsSort < cnt <=
// kBsList), in any order: the n-th largest is found bit by bit.  Returns it.
__device__ u64 beam_keep_n(u64* list, int* s_cnt, int cnt, int n) {
    constexpr int kPer = (kBsList + kBsThreads - 1) / kBsThreads;
    __shared__ int s_count;
    u64 k[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int p = threadIdx.x + i * kBsThreads;
        k[i] = p < cnt ? list[p] : 0;
    }
    u64 t = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const u64 cand = t | (1ull << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) c += k[i] >= cand;
        c = __reduce_add_sync(0xffffffffu, c);
        if (threadIdx.x == 0) s_count = 0;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) atomicAdd(&s_count, c);
        __syncthreads();
        const int total = s_count;
        __syncthreads();
        if (total >= n) t = cand;
        if (total == n) break;
    }
    if (threadIdx.x == 0) *s_cnt = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (k[i] >= t && k[i] != 0) list[atomicAdd(s_cnt, 1)] = k[i];
    __syncthreads();
    return t;
}

// Raise the threshold T of list[0, cnt) (all keys >= T, n < cnt <= kBsSort) to
// the lower edge of the bucket that holds the n-th largest value, of 256
// buckets between T and the maximum, and drop the keys below it.
__device__ u64 beam_tighten(u64* list, int* s_cnt, int cnt, int n, u64 T, int* hist) {
    constexpr int kPer = kBsSort / kBsThreads;
    __shared__ uint32_t s_max;
    __shared__ int s_bucket;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 k[kPer];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int p = tid + i * kBsThreads;
        k[i] = p < cnt ? list[p] : 0;
        top = max(top, (uint32_t)(k[i] >> 32));
    }
    hist[tid] = 0;
    if (tid == 0) s_max = 0;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) atomicMax(&s_max, top);
    __syncthreads();
    const uint32_t low = (uint32_t)(T >> 32);
    const int shift = max(0, 24 - __clz(s_max - low));  // (max - low) >> shift < 256
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (k[i]) atomicAdd(&hist[((uint32_t)(k[i] >> 32) - low) >> shift], 1);
    if (tid == 0) *s_cnt = 0;
    __syncthreads();
    if (warp == 0) {  // lane L: buckets 255 - 8 L .. 248 - 8 L, from the top
        int c[8], mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            c[i] = hist[255 - 8 * lane - i];
            mine += c[i];
        }
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += y;
        }
        before -= mine;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (before < n && n <= before + c[i]) s_bucket = 255 - 8 * lane - i;
            before += c[i];
        }
    }
    __syncthreads();
    T = (u64)(low + ((uint32_t)s_bucket << shift)) << 32;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (k[i] >= T && k[i]) list[atomicAdd(s_cnt, 1)] = k[i];
    __syncthreads();
    return T;
}

// Plain pointers and loads: the kernel may be set up while its predecessor still
// writes the inputs, so they are not constant over its lifetime.
__global__ void __launch_bounds__(kBsThreads) beam_part_kernel(const float* logits,
                                                               const int32_t* finished, int n_beam,
                                                               int vocab, const BeamSplit split, int n,
                                                               u64* keys,
                                                               BeamPart* stats) {
    constexpr int kWarps = kBsThreads / 32;
    extern __shared__ __align__(16) u64 list[];                  // [kBsList]
    float* s_tile = reinterpret_cast<float*>(list + kBsList);    // [kBsTile]
    __shared__ int s_cnt;
    __shared__ __align__(16) int s_hist[2 * kBsThreads + 4];
    __shared__ double s_tab[16];
    __shared__ int s_seen[2 * kBsThreads];
    __shared__ uint32_t s_t[kWarps];
    __shared__ float s_m[kWarps];
    __shared__ double s_l[kWarps];
    __shared__ int s_beam[kBeamMax];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) s_cnt = 0;
    if (tid < 16) s_tab[tid] = exp2(tid / 16.0);
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    int b = blockIdx.y, part = blockIdx.x, per = split.per, at = b * split.parts + part;
    if (split.share) {
        const int live = beam_live(finished, n_beam, s_beam), parts = beam_parts(live, vocab, split.room);
        at = blockIdx.x;
        const int rank = at / parts;
        if (rank >= live) return;
        b = s_beam[rank];
        part = at - rank * parts;
        per = (vocab + parts - 1) / parts;
    } else if (finished && finished[b]) {
        return;  // the merge does not look at an ended beam's lists
    }
    const float* x = logits + (size_t)b * vocab;
    const int i0 = part * per, i1 = min(vocab, i0 + per);
    float m = -INFINITY;  // reference of l, at most 64 below the thread's maximum
    double l = 0.0;
    bool bad = false;
    u64 T = 0;
    float ahead[kBsPer];  // the next tile's logits
    auto load = [&](int base) {
        if (base + kBsTile <= i1) {
#pragma unroll
            for (int j = 0; j < kBsPer; ++j) ahead[j] = x[base + tid + j * kBsThreads];
            return;
        }
#pragma unroll
        for (int j = 0; j < kBsPer; ++j) {
            const int i = base + j * kBsThreads + tid;
            ahead[j] = i < i1 ? x[i] : -INFINITY;
        }
    };
    load(i0);
    for (int base = i0; base < i1; base += kBsTile) {
        float v[kBsPer];
        float tm = -INFINITY;
#pragma unroll
        for (int j = 0; j < kBsPer; ++j) {
            v[j] = ahead[j];
            tm = max_nan(tm, v[j]);
        }
        bad |= !(tm < INFINITY);
        if (base + kBsTile < i1) load(base + kBsTile);
        if (base == i0) {
            // at least n elements reach T: the (n / kWarps)-th largest of each warp's thread maxima
            const uint32_t t = warp_kth(tid < i1 - base ? ord32(tm) : 0u, (n + kWarps - 1) / kWarps, lane);
            if (lane == 0) s_t[warp] = t;
            __syncthreads();
            uint32_t low = s_t[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) low = min(low, s_t[w]);
            T = (u64)low << 32;
        }
        {
            // what reaches T goes to the list: a place per warp, then per lane
            unsigned take = 0;
            const float low = T ? unord32((uint32_t)(T >> 32)) : -INFINITY;
            if (tm >= low) {
#pragma unroll
                for (int j = 0; j < kBsPer; ++j) take |= (unsigned)(v[j] >= low) << j;
                if (base + kBsTile > i1 || (uint32_t)T) {  // a part's end; a T that tells equal values apart
#pragma unroll
                    for (int j = 0; j < kBsPer; ++j) {
                        const int i = base + j * kBsThreads + tid;
                        if (i >= i1 || ((u64)ord32(v[j]) << 32 | (0xFFFFFFFFu - (uint32_t)i)) < T) take &= ~(1u << j);
                    }
                }
            }
            if (__any_sync(0xffffffffu, take != 0)) {
#pragma unroll
                for (int j = 0; j < kBsPer; ++j) s_tile[j * kBsThreads + tid] = v[j];  // to be picked by index
                int to = __popc(take);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, to, o);
                    if (lane >= o) to += y;
                }
                int start = 0;
                if (lane == 31) start = atomicAdd(&s_cnt, to);
                to += __shfl_sync(0xffffffffu, start, 31) - __popc(take);
                for (; take; take &= take - 1) {  // few per thread
                    const int j = __ffs(take) - 1;
                    list[to++] = (u64)ord32(s_tile[j * kBsThreads + tid]) << 32 | (0xFFFFFFFFu - (uint32_t)(base + j * kBsThreads + tid));
                }
            }
        }
        if (tm > m + 64.0f || m == -INFINITY) {
            l *= tm - m < 700.0f ? exp_taylor((double)m - (double)tm) : 0.0;  // m = -inf: l is 0
            m = tm;
        }
        if (m > -INFINITY) {
            // what lies over 700 below counts as e^-700: no branch, so that the
            // chains of several terms run side by side
            const float floor = m - 700.0f;
            const double md = (double)m;
            double part[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int g = 0; g < kBsPer; g += 4) {
                if (base + g * kBsThreads >= i1) break;  // of the CTA: the rest of the tile is empty
#pragma unroll
                for (int j = g; j < g + 4; ++j) {
                    part[j & 3] += exp_tab((double)fmaxf(v[j], floor) - md, s_tab);
                }
            }
            l += (part[0] + part[1]) + (part[2] + part[3]);
        }
        __syncthreads();
        const int cnt = s_cnt;
        __syncthreads();
        if (cnt > kBsSort) T = beam_keep_n(list, &s_cnt, cnt, n);
        else if (cnt > 2 * n + 256 || (cnt > n + n / 4 + 32 && base + kBsTile >= i1)) T = beam_tighten(list, &s_cnt, cnt, n, T, s_hist);
    }
    // the threads' (m, l) as one
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (bad) l = NAN;
    else l = m - M > -700.0f ? l * exp_taylor((double)m - (double)M) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
        s_m[warp] = M;
        s_l[warp] = l;
    }
    __syncthreads();
    const int cnt = s_cnt;
    u64* out = keys + (size_t)at * n;
    if (cnt <= 2 * kBsThreads) {
        // place by the number of larger keys: by their values, and where two values
        // are equal once more by the whole keys
        uint32_t* hi = reinterpret_cast<uint32_t*>(s_hist);  // 2 * kBsThreads values and 4 zeros
        const u64 k0 = tid < cnt ? list[tid] : 0, k1 = tid + kBsThreads < cnt ? list[tid + kBsThreads] : 0;
        const uint32_t h0 = (uint32_t)(k0 >> 32), h1 = (uint32_t)(k1 >> 32);
        hi[tid] = h0;
        hi[tid + kBsThreads] = h1;
        if (tid < 4) hi[2 * kBsThreads + tid] = 0;
        if (tid == 0) list[cnt] = 0;
        s_seen[tid] = s_seen[tid + kBsThreads] = 0;
        __syncthreads();
        int r0 = 0, r1 = 0;
        if (32 * warp < cnt) {
#pragma unroll 4
            for (int i = 0; i < cnt; i += 4) {
                const uint4 k = *reinterpret_cast<const uint4*>(hi + i);
                r0 += (k.x > h0) + (k.y > h0) + (k.z > h0) + (k.w > h0);
            }
            if (cnt > kBsThreads)
#pragma unroll 4
                for (int i = 0; i < cnt; i += 4) {
                    const uint4 k = *reinterpret_cast<const uint4*>(hi + i);
                    r1 += (k.x > h1) + (k.y > h1) + (k.z > h1) + (k.w > h1);
                }
        }
        // equal values have equal ranks
        const bool tie = (k0 && atomicExch(&s_seen[r0], 1)) || (k1 && atomicExch(&s_seen[r1], 1));
        if (__syncthreads_or(tie)) {
            r0 = r1 = 0;
            for (int i = 0; i < cnt; i += 2) {
                const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(list + i);
                r0 += (k.x > k0) + (k.y > k0);
                r1 += (k.x > k1) + (k.y > k1);
            }
        }
        if (k0 && r0 < n) out[r0] = k0;
        if (k1 && r1 < n) out[r1] = k1;
    } else {
        int P = kBsThreads;
        while (P < cnt) P <<= 1;
        for (int i = cnt + tid; i < P; i += kBsThreads) list[i] = 0;
        bitonic_desc(list, P);
        for (int i = tid; i < n; i += kBsThreads) out[i] = list[i];
    }
    for (int i = cnt + tid; i < n; i += kBsThreads) out[i] = 0;
    if (tid == 0) {
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w]);
        double ll = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const double f = s_m[w] - mm > -700.0f ? exp_taylor((double)s_m[w] - (double)mm) : 0.0;
            ll += s_l[w] == s_l[w] ? s_l[w] * f : s_l[w];  // a NaN stays
        }
        stats[at] = BeamPart{ll, mm, 0};
    }
}

// (score, then lo = ~(beam | inverted logit | token)): greater is better; hi = 0 is no candidate
struct BeamKey {
    u64 hi, lo;
    __device__ bool operator<(const BeamKey& o) const { return hi < o.hi || (hi == o.hi && lo < o.lo); }
};

// The candidate that entry e (0: none) of beam b's list stands for.
__device__ __forceinline__ BeamKey beam_key(u64 e, int b, double score, double lse) {
    const uint32_t o = (uint32_t)(e >> 32), token = 0xFFFFFFFFu - (uint32_t)e;
    const double s = score + ((double)unord32(o) - lse);
    return BeamKey{e && s > -INFINITY ? ord64(s) : 0, ~((u64)b << 56 | (u64)~o << 24 | token)};
}
// 32 bits of a score in the same order (equal for near ones), 0 for no candidate.
__device__ __forceinline__ uint32_t beam_key32(u64 hi) { return (uint32_t)(hi >> 32); }

// A value that at least n of the threads' v reach: the lower edge of the bucket
// with the n-th largest, of 256 between the least and the greatest v that is not
// 0; 0 when fewer than n are not.  Whole CTA.
__device__ __forceinline__ uint32_t cta_bound(uint32_t v, int n, int* hist) {
    __shared__ uint32_t s_low, s_top;
    __shared__ int s_bucket;
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < 256) hist[tid] = 0;
    if (tid == 0) {
        s_low = 0xFFFFFFFFu;
        s_top = 0;
        s_bucket = -1;
    }
    __syncthreads();
    const uint32_t low = __reduce_min_sync(0xffffffffu, v ? v : 0xFFFFFFFFu), top = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0 && top) {
        atomicMin(&s_low, low);
        atomicMax(&s_top, top);
    }
    __syncthreads();
    const uint32_t base = s_low;
    const int shift = s_top ? max(0, 24 - __clz(s_top - base)) : 0;
    if (v) atomicAdd(&hist[(v - base) >> shift], 1);
    __syncthreads();
    if (tid < 32) {  // lane L: buckets 255 - 8 L .. 248 - 8 L, from the top
        int c[8], mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            c[i] = hist[255 - 8 * lane - i];
            mine += c[i];
        }
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += y;
        }
        before -= mine;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (before < n && n <= before + c[i]) s_bucket = 255 - 8 * lane - i;
            before += c[i];
        }
    }
    __syncthreads();
    const uint32_t t = s_bucket < 0 ? 0u : base + ((uint32_t)s_bucket << shift);
    __syncthreads();
    return t;
}

__global__ void __launch_bounds__(kBmThreads, 1) beam_merge_kernel(
    const u64* keys, const BeamPart* stats, const float* scores, const int32_t* finished,
    int n_beam, int vocab, const BeamSplit split, int n, int eos, float* out_scores, int32_t* out_parents, int32_t* out_tokens,
    int32_t* out_finished) {
    __shared__ __align__(16) BeamKey list[kBmList];
    __shared__ double s_lse[kBeamMax], s_score[kBeamMax];
    __shared__ int s_rank[kBeamMaxOut * 2], s_seen[kBeamMaxOut * 2];
    __shared__ uint4 s_k32[kBeamMaxOut / 2 + 1];
    __shared__ int s_cnt, s_live, s_full;
    __shared__ int s_beam[kBeamMax];
    const int tid = threadIdx.x;
    if (tid == 0) s_cnt = s_live = s_full = 0;
    // read before the wait, from L2: the first kernel has let this one start after its own
    const int n_live = split.share ? beam_live(finished, n_beam, s_beam) : n_beam;
    const int parts = split.share ? beam_parts(n_live, vocab, split.room) : split.parts;
    pdl_wait();
    // Everything that is read first is asked for at once: the first entries of the
    // lists, a thread per list; the parts' sums, 4 to 32 lanes per beam; the beams' scores.
    // Few lists are shared by 2^sh threads each, which take every 2^sh-th entry:
    // sorted lists again (3 beams of 1000 logits, 200 out: 15.1 us; a thread per list
    // 33.3).
    const int whole = n_live * parts;
    int sh = 0;
    if (whole > 0)
        while (whole << sh < n && whole << (sh + 1) <= kBmThreads) ++sh;
    const int lists = whole << sh;  // <= kBmThreads
    const int at = (tid >> sh) / parts, sub = tid & ((1 << sh) - 1), len = (n - sub + (1 << sh) - 1) >> sh;
    const u64* mine = keys + (size_t)(tid >> sh) * n + sub;
    constexpr int kAhead = 4;  // entries of the list that are loaded together
    u64 ahead[kAhead];
    auto load = [&](int r) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ahead[i] = r + i < len ? mine[(r + i) << sh] : 0;
    };
    auto entry = [&](int r) {
        u64 e = ahead[0];
#pragma unroll
        for (int i = 1; i < kAhead; ++i) e = (r & (kAhead - 1)) == i ? ahead[i] : e;
        return e;
    };
    if (tid < lists) load(0);
    int width = 32;
    while (width > 4 && n_live * width > kBmThreads) width >>= 1;
    const int w = tid / width, wl = tid & (width - 1);
    const BeamPart* st = stats + (size_t)w * parts;
    BeamPart part0{0.0, -INFINITY, 0};
    if (w < n_live && wl < parts) part0 = st[wl];
    // the scores; NaN for a beam without lists (ended, or no candidate can be better than none)
    if (tid < n_beam) {
        const float s = scores[tid];
        const bool live = !(finished && finished[tid]) && s > -INFINITY;
        s_score[tid] = live ? (double)s : NAN;
        if (live) atomicAdd(&s_live, 1);
        else if (s > -INFINITY) list[atomicAdd(&s_cnt, 1)] = BeamKey{ord64((double)s), ~((u64)tid << 56 | (u64)eos)};
    }
    __syncthreads();
    const int b = tid < lists ? split.share ? s_beam[at] : at : 0;
    const bool has = tid < lists && s_score[b] == s_score[b];
    {
        const bool on = w < n_live;
        // a lane's parts as one, then the lanes'
        float M = -INFINITY;
        double l = 0.0;
        auto join = [&](float m, double sum) {
            const float top = fmaxf(M, m);
            // nothing counts for less than e^-700; a NaN sum stays
            const double a = M - top > -700.0f ? exp_taylor((double)M - (double)top) : 0.0;
            const double c = m - top > -700.0f ? exp_taylor((double)m - (double)top) : 0.0;
            l = (l == l ? l * a : l) + (sum == sum ? sum * c : sum);
            M = top;
        };
        if (on && wl < parts) {
            M = part0.ref;
            l = part0.sum;
            for (int p = wl + width; p < parts; p += width) {
                const BeamPart s = st[p];
                join(s.ref, s.sum);
            }
        }
        float top = M;
        for (int o = width / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (l == l) l = M - top > -700.0f ? l * exp_taylor((double)M - (double)top) : 0.0;
        M = top;
        for (int o = width / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (on && wl == 0) s_lse[w] = (double)M + log_of_sum(l);
    }
    __syncthreads();
    const double score = s_score[b], lse = has ? s_lse[at] : 0.0;
    // the lists' first R entries, which with the ended beams are enough unless many are no candidates
    const int live_lists = max(1, s_live * parts << sh), R = min(len, (n + live_lists - 1) / live_lists);
    int r = 0;  // entries of this thread's list that were taken
    bool more = has;
    for (; r < R && more; ++r) {
        if (r && (r & (kAhead - 1)) == 0) load(r);
        const BeamKey k = beam_key(entry(r), b, score, lse);
        more = k.hi != 0;  // the list is sorted: nothing follows an entry that is no candidate
        if (more) list[atomicAdd(&s_cnt, 1)] = k;
    }
    __syncthreads();
    int cnt = s_cnt;  // <= n_beam + live lists + n; where it is over kBmThreads, t1 goes by the first of them
    const uint32_t t1 = cnt >= n ? cta_bound(tid < cnt ? beam_key32(list[tid].hi) : 0u, n, s_rank) : 0u;
    // the rest, while it reaches t1: a few entries per list.  Where the lists hold
    // so many candidates that t1 does not bound them, in rounds with a sort.
    const bool bounded = t1 != 0;
    if (bounded) {
        __syncthreads();
        while (more && r < len) {
            if (r && (r & (kAhead - 1)) == 0) load(r);
            const BeamKey k = beam_key(entry(r), b, score, lse);
            more = k.hi != 0 && beam_key32(k.hi) >= t1;
            if (!more) break;
            const int p = atomicAdd(&s_cnt, 1);
            if (p >= kBmList) {  // no room: this entry and the later ones are for the rounds
                s_full = 1;
                break;
            }
            list[p] = k;
            ++r;
        }
        __syncthreads();
        if (s_full && tid == 0) s_cnt = kBmList;
        __syncthreads();
    }
    BeamKey T{0, 0};
    if (!bounded || s_full) {
        for (bool go = true; go;) {
            cnt = s_cnt;
            __syncthreads();
            if (cnt > kBmList - kBmThreads || (T.hi == 0 && cnt >= n)) {
                int P = 512;
                while (P < cnt) P <<= 1;
                for (int i = cnt + tid; i < P; i += kBmThreads) list[i] = BeamKey{0, 0};
                bitonic_desc(list, P);
                T = list[n - 1];
                if (tid == 0) s_cnt = n;
                __syncthreads();
            }
            more = more && r < len;
            if (more) {
                if (r && (r & (kAhead - 1)) == 0) load(r);
                const BeamKey k = beam_key(entry(r), b, score, lse);
                more = k.hi != 0 && T < k;
                if (more) list[atomicAdd(&s_cnt, 1)] = k;
                ++r;
            }
            go = __syncthreads_or(more);
        }
        __syncthreads();
    }
    cnt = s_cnt;
    BeamKey best{0, 0};  // the tid-th best
    uint32_t t2 = 0;
    if (cnt <= kBmThreads) {
        // only what reaches the n-th best (but for the last bits) is ranked
        const BeamKey k = tid < cnt ? list[tid] : BeamKey{0, 0};
        t2 = cnt > n ? cta_bound(beam_key32(k.hi), n, s_rank) : 0u;
        __syncthreads();
        if (tid == 0) s_cnt = 0;
        __syncthreads();
        if (k.hi && beam_key32(k.hi) >= t2) list[atomicAdd(&s_cnt, 1)] = k;
        __syncthreads();
        cnt = s_cnt;
    }
    if (cnt <= 2 * kBeamMaxOut) {
        // place each by the number of better ones, groups of threads counting shares
        // of them: by 32 bits of the scores, where two are equal by the whole keys
        const int P = max(32, (cnt + 31) & ~31), groups = kBmThreads / P;
        const int i = tid % P, g = tid / P;
        const bool on = g < groups && i < cnt;
        uint32_t* k32 = reinterpret_cast<uint32_t*>(s_k32);
        if (tid < 2 * kBeamMaxOut) {
            s_rank[tid] = 0;
            k32[tid] = tid < cnt ? beam_key32(list[tid].hi) : 0u;
            s_seen[tid] = 0;
        }
        __syncthreads();
        if (on) {
            const uint32_t k = k32[i];
            int better = 0;
            for (int j = 4 * g; j < cnt; j += 4 * groups) {
                const uint4 o = *reinterpret_cast<const uint4*>(k32 + j);
                better += (o.x > k) + (o.y > k) + (o.z > k) + (o.w > k);
            }
            if (better) atomicAdd(&s_rank[i], better);
        }
        __syncthreads();
        if (__syncthreads_or(tid < cnt && atomicExch(&s_seen[s_rank[tid]], 1))) {
            if (tid < 2 * kBeamMaxOut) s_rank[tid] = 0;
            __syncthreads();
            if (on) {
                const BeamKey k = list[i];
                int better = 0;
#pragma unroll 4
                for (int j = g; j < cnt; j += groups) {
                    const BeamKey o = list[j];
                    better += (o.hi > k.hi) | ((o.hi == k.hi) & (o.lo > k.lo));
                }
                if (better) atomicAdd(&s_rank[i], better);
            }
            __syncthreads();
        }
        const BeamKey k = list[tid < cnt ? tid : 0];
        const int rank = tid < cnt ? s_rank[tid] : kBmThreads;
        __syncthreads();
        if (rank < n) list[rank] = k;
        __syncthreads();
        if (tid < min(cnt, n)) best = list[tid];
    } else {
        int P = 512;
        while (P < cnt) P <<= 1;
        for (int i = cnt + tid; i < P; i += kBmThreads) list[i] = BeamKey{0, 0};
        bitonic_desc(list, P);
        if (tid < n) best = list[tid];
    }
    const u64 id = ~best.lo;
    const bool some = tid < n && best.hi != 0;
    const int parent = some ? (int)(id >> 56) : -1;
    const int token = some ? (int)(id & 0xFFFFFFu) : -1;
    const bool end = some && ((finished && finished[parent]) || token == eos);
    __syncthreads();  // the inputs are read: the outputs may be the same arrays
    if (tid < n) {
        out_scores[tid] = some ? (float)unord64(best.hi) : -INFINITY;
        out_parents[tid] = parent;
        out_tokens[tid] = token;
        if (out_finished) out_finished[tid] = end;
    }
}

// The most lists: kBsCtasPerSm CTAs per SM, twice that where the beams outnumber
// the SMs.
static int beam_room(int n_beam, int vocab, int sm_count) {
    const int tiles = (vocab + kBsTile - 1) / kBsTile;
    const int room = min(kBmThreads, (n_beam > sm_count ? 2 : 1) * kBsCtasPerSm * sm_count);
    return max(n_beam, min(room, n_beam * tiles));
}

size_t beam_workspace_bytes(int n_beam, int vocab, int n_out, int sm_count) {
    const size_t lists = beam_room(n_beam, vocab, sm_count);
    return (lists * n_out * sizeof(u64) + 255) / 256 * 256 + lists * sizeof(BeamPart);
}

int beam_select_launch(const float* logits, const float* scores, const int32_t* finished, int n_beam, int vocab,
                       int eos, int n_out, float* out_scores, int32_t* out_parents, int32_t* out_tokens,
                       int32_t* out_finished, void* ws, cudaStream_t st) {
    static_assert(kBeamMaxOut <= kBsThreads && kBeamMaxOut <= kBmThreads / 4, "the lists' capacities");
    static_assert(kBeamMax <= kBsThreads && kBeamMax <= kBmThreads, "a thread per beam");
    const int room = beam_room(n_beam, vocab, device_info().sm_count);
    BeamSplit split{room, beam_parts(n_beam, vocab, room), 0, finished && n_beam * kBsShare > room};
    split.per = (vocab + split.parts - 1) / split.parts;
    u64* keys = static_cast<u64*>(ws);
    BeamPart* stats = reinterpret_cast<BeamPart*>(static_cast<uint8_t*>(ws) + ((size_t)room * n_out * sizeof(u64) + 255) / 256 * 256);
    constexpr size_t smem = kBsList * sizeof(u64) + kBsTile * sizeof(float);
    if (set_smem_limit(beam_part_kernel, smem) != cudaSuccess) return kErrCuda;
    if (launch_after(beam_part_kernel, split.share ? dim3(room) : dim3(split.parts, n_beam), dim3(kBsThreads), smem, st,
                     logits, finished, n_beam, vocab, split, n_out, keys, stats) != cudaSuccess)
        return kErrCuda;
    return launch_after(beam_merge_kernel, dim3(1), dim3(kBmThreads), 0, st, (const u64*)keys, (const BeamPart*)stats,
                        scores, finished, n_beam, vocab, split, n_out, eos, out_scores, out_parents, out_tokens,
                        out_finished) == cudaSuccess
               ? kOk
               : kErrCuda;
}

// ---------------------------------------------------------------- reordering
// new[s][i] = old[s][index[i]] for every state s, in place.  A thread owns one
// column (16 or 4 bytes at one offset of every slot), reads the sources of
// all slots that change before it writes any, so no second buffer and no
// barrier is needed; slots that stay (-1, or their own index) are not touched.
// An index outside [-1, n_slots) leaves its slot and records an error.  Bound by
// HBM: 16 states of 8 slots of 4 MB, every slot's row read once and written once,
// 138 us for 0.88 GB, 6.4 TB/s; where small by latency: 33 slots of 4 KB in 56
// states 3.3 us.  Up to 16 slots a thread's columns are in registers, else in shared
// memory.
struct ReorderArgs {
    uint8_t* state;
    size_t state_stride, slot_stride;
    size_t cols;  // columns per slot
    int n_states, n_slots;
    const int32_t* index;
    int32_t* err;
};

// The (destination, source) pairs of the slots that change; whole CTA.
__device__ __forceinline__ int reorder_moves(const ReorderArgs& a, int2* s_move, int* s_n) {
    if (threadIdx.x == 0) *s_n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_slots; i += blockDim.x) {
        const int j = a.index[i];
        if (j < -1 || j >= a.n_slots) record_error(a.err, kErrInvalidArg);
        else if (j >= 0 && j != i) s_move[atomicAdd(s_n, 1)] = make_int2(i, j);
    }
    __syncthreads();
    return *s_n;
}

constexpr int kReorderRegs = 16;  // slots whose columns a thread holds in registers

template <class V, int N>
__global__ void __launch_bounds__(256) reorder_regs_kernel(const ReorderArgs a) {
    __shared__ int2 s_move[N];
    __shared__ int s_n;
    pdl_wait();
    const int m = reorder_moves(a, s_move, &s_n);
    if (m == 0) return;
    const size_t c = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.cols) return;
    for (int s = blockIdx.y; s < a.n_states; s += gridDim.y) {
        uint8_t* p = a.state + (size_t)s * a.state_stride + c * sizeof(V);
        V v[N];
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < m) v[j] = *reinterpret_cast<const V*>(p + (size_t)s_move[j].y * a.slot_stride);
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < m) *reinterpret_cast<V*>(p + (size_t)s_move[j].x * a.slot_stride) = v[j];
    }
}

template <class V>
__global__ void reorder_smem_kernel(const ReorderArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int2 s_move[kReorderMaxSlots];
    __shared__ int s_n;
    pdl_wait();
    const int m = reorder_moves(a, s_move, &s_n);
    if (m == 0) return;
    const size_t c = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.cols) return;
    V* hold = reinterpret_cast<V*>(smem) + threadIdx.x;
    for (int s = blockIdx.y; s < a.n_states; s += gridDim.y) {
        uint8_t* p = a.state + (size_t)s * a.state_stride + c * sizeof(V);
#pragma unroll 8
        for (int j = 0; j < m; ++j) hold[j * blockDim.x] = *reinterpret_cast<const V*>(p + (size_t)s_move[j].y * a.slot_stride);
#pragma unroll 8
        for (int j = 0; j < m; ++j) *reinterpret_cast<V*>(p + (size_t)s_move[j].x * a.slot_stride) = hold[j * blockDim.x];
    }
}

template <class V>
static cudaError_t reorder_launch_v(ReorderArgs a, size_t n_bytes, cudaStream_t st) {
    a.cols = n_bytes / sizeof(V);
    int threads = 256;
    while (threads > 32 && (size_t)threads / 2 >= a.cols) threads >>= 1;
    const int gy = a.n_states < 65535 ? a.n_states : 65535;
    if (a.n_slots <= kReorderRegs) {
        const dim3 grid((unsigned)((a.cols + threads - 1) / threads), gy);
        auto go = [&](auto k) { return launch_after(k, grid, dim3(threads), 0, st, a); };
        return a.n_slots <= 4   ? go(reorder_regs_kernel<V, 4>)
               : a.n_slots <= 8 ? go(reorder_regs_kernel<V, 8>)
                                : go(reorder_regs_kernel<V, kReorderRegs>);
    }
    while (threads > 32 && (size_t)threads * a.n_slots * sizeof(V) > 64 * 1024) threads >>= 1;
    const size_t smem = (size_t)threads * a.n_slots * sizeof(V);
    const cudaError_t e = set_smem_limit(reorder_smem_kernel<V>, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)((a.cols + threads - 1) / threads), gy);
    return launch_after(reorder_smem_kernel<V>, grid, dim3(threads), smem, st, a);
}

int reorder_launch(void* state, int n_states, size_t state_stride, int n_slots, size_t slot_stride, size_t n_bytes,
                   const int32_t* index, int32_t* err, cudaStream_t st) {
    ReorderArgs a{static_cast<uint8_t*>(state), state_stride, slot_stride, 0, n_states, n_slots, index, err};
    if (n_slots == 1) {  // nothing can move: one column of one state looks at the index
        a.n_states = 1;
        n_bytes = 4;
    }
    const bool wide = (((uintptr_t)state | state_stride | slot_stride | n_bytes) & 15) == 0;
    const cudaError_t e = wide ? reorder_launch_v<uint4>(a, n_bytes, st) : reorder_launch_v<uint32_t>(a, n_bytes, st);
    return e == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace gncx
