// The selection of a beam search's next step: of every group's candidates
//     s(b, t) = score_b + logit_bt - log sum_u exp(logit_bu)
// the k best, equal ones by the lowest b * vocab + t.  An ended beam has one candidate, its score with token end_id.  Candidates
// that are not numbers (a row with NaN or +inf, a beam whose score is not finite) count as -inf, as forbidden tokens do, and come
// after all others.
//
// The logits are read once.  Within a beam the order is that of the logits, whatever the sum: k_beam_part takes a stretch of a
// row into registers and leaves its largest logit, its sum of exponentials and its k best logits.  k_beam_merge, a CTA per group,
// joins the sums and orders the candidates in 64 bits.  The sums carry an error of their f32 exponentials and roundings, below
// 2.2e-6; where two beams' candidates lie closer than that could move them, the sums of these beams are formed again in 64 bits.
#include <climits>
#include <type_traits>

#include "beam.h"
#include "rows.cuh"

namespace qb {

namespace {

constexpr int kPartThreads = 256;
constexpr int kMergeThreads = 512;
constexpr int kCap = 1024;  // candidates that pass the threshold; more are taken one at a time
constexpr int kMany = 192;   // candidates that are worth a second threshold before they are ranked
constexpr float kMaxF = 3.402823466e38f;

// Order-preserving keys: of a logit, with the token below so that the lowest one wins; 0 is no candidate.
__device__ __forceinline__ unsigned order(float x) {
    const unsigned b = __float_as_uint(x);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unorder(unsigned k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ unsigned long long key_of(float x, int token) {
    return (unsigned long long)order(x + 0.f) << 32 | (0xffffffffu - unsigned(token));
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return e;
}

// 16 bytes of logits as floats, and their largest (NaN aside).
template <class T>
__device__ __forceinline__ void unpack(uint4 w, float (&x)[16 / sizeof(T)]) {
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(u[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        } else {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
}
template <class T>
__device__ __forceinline__ float largest(uint4 w) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    } else if constexpr (std::is_same<T, __half>::value) {
        const __half2* h = reinterpret_cast<const __half2*>(&w);
        const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
        return fmaxf(f.x, f.y);
    } else {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
        const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
        return fmaxf(f.x, f.y);
    }
}
// Element j of 16 bytes.
template <class T>
__device__ __forceinline__ float pick(uint4 w, int j) {
    constexpr int P = 4 / sizeof(T);  // elements of a word
    const int k = j / P;
    const unsigned u = k == 0 ? w.x : k == 1 ? w.y : k == 2 ? w.z : w.w;
    if constexpr (sizeof(T) == 4) return __uint_as_float(u);
    const unsigned h = u >> (j % P * 16);
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
    else return __uint_as_float(h << 16);
}
// The bits of -inf, twice where the type has 16.
template <class T>
constexpr unsigned kForbidden = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;

// Where the sums and the candidates of stretch s of row r lie: slot r * splits + s.
struct BeamParts {
    double* sum;   // sum of exp(x - top)
    float* top;    // largest logit of the stretch (-inf: none above it)
    unsigned long long* best;  // [k] keys, descending, 0 past the last one
    int splits;
    int pieces;    // 16-byte pieces of a stretch, at most kPartThreads * E / (16 / sizeof(T))
};

// The k-th largest of 32 G values that warp 0 reads (as ordered keys; 0 where there are fewer): with a value of every lane's own
// known against all others, a rank is a count.
template <int G>
__device__ __forceinline__ unsigned kth_of(const unsigned* vals, int k) {
    const int lane = threadIdx.x & 31;
    unsigned v[G];
    int rank[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        v[g] = vals[g * 32 + lane];
        rank[g] = 0;
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const unsigned o = __shfl_sync(0xffffffffu, v[g], j);
#pragma unroll
            for (int h = 0; h < G; ++h) rank[h] += o > v[h];
        }
    unsigned least = 0xffffffffu;
#pragma unroll
    for (int g = 0; g < G; ++g)
        if (rank[g] < k) least = min(least, v[g]);
    return __reduce_min_sync(0xffffffffu, least);
}

// A stretch of kPartThreads * E logits of a row, held as it lies in memory (16 bytes a register quad).  G: 32 G groups of threads whose
// maxima give the threshold that candidates have to reach: the k-th largest of them, so that k candidates reach it and not many
// more.  Instructions bound it next to HBM, so a logit costs about six: half a packed maximum, its conversion, half a packed
// fused y = x log2 e + c, the exponential, half a packed sum, and a comparison only in quads whose maximum reaches the threshold.
// c is the f32 next to -top log2 e; what it lacks is made good in the sum.
template <class T, int E, int G>
__global__ void __launch_bounds__(kPartThreads, E * sizeof(T) == 128 ? 4 : 5)
    k_beam_part(const T* __restrict__ logits, long long stride, int vocab, const float* __restrict__ scores,
                const uint8_t* __restrict__ ended, int k, BeamParts out) {
    constexpr int V = 16 / sizeof(T), N = E / V, W = kPartThreads / 32, GROUP = kPartThreads / (32 * G);
    __shared__ unsigned group_top[32 * G];
    __shared__ float threshold;
    __shared__ int count;
    __shared__ double sums[W];
    __shared__ unsigned long long cand[kCap];
    __shared__ unsigned again[kPartThreads / 2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned slot = blockIdx.x, r = slot / unsigned(out.splits), s = slot - r * unsigned(out.splits);
    pdl_launch_dependents();
    const float score = __ldg(scores + r);
    const int over = ended ? __ldg(ended + r) : 0;
    if (over || !(fabsf(score) <= kMaxF)) return;  // the merge does not look at this row
    const T* row = logits + r * stride;
    // 16-byte pieces as they lie in memory; the row's first one may hold elements that come before it
    const int lead = int(reinterpret_cast<uintptr_t>(row) / sizeof(T) % V), first = int(s) * out.pieces + tid;
    const uint4* base = reinterpret_cast<const uint4*>(row - lead);
    const int t0 = int(s) * out.pieces * V - lead, t1 = t0 + out.pieces * V;  // tokens of the stretch, but for the row's ends
    uint4 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = make_uint4(kForbidden<T>, kForbidden<T>, kForbidden<T>, kForbidden<T>);
    if (t0 >= 0 && t1 <= vocab) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i * kPartThreads + tid < out.pieces) x[i] = __ldcs(base + first + i * kPartThreads);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = (first + i * kPartThreads) * V - lead;  // token of the piece's first element
            if (i * kPartThreads + tid >= out.pieces || e >= vocab) continue;
            if (e >= 0 && e + V <= vocab) {
                x[i] = __ldcs(base + first + i * kPartThreads);
            } else {
                T* v = reinterpret_cast<T*>(&x[i]);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e + j >= 0 && e + j < vocab) v[j] = row[e + j];
            }
        }
    }
    if (tid == 0) count = 0;
    float quad[N], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        quad[i] = largest<T>(x[i]);
        top = fmaxf(top, quad[i]);
    }
    unsigned g = order(top + 0.f);  // (-0 is 0)
#pragma unroll
    for (int o = 1; o < GROUP; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % GROUP == 0) group_top[tid / GROUP] = g;
    __syncthreads();
    unsigned all = 0;
#pragma unroll
    for (int i = 0; i < G; ++i) all = max(all, group_top[i * 32 + lane]);
    all = __reduce_max_sync(0xffffffffu, all);
    const float row_top = unorder(all), ref = row_top == -INFINITY ? 0.f : row_top;
    if (warp == 0) {
        const unsigned t = kth_of<G>(group_top, k);
        if (lane == 0) threshold = unorder(max(t, order(-INFINITY) + 1));  // forbidden tokens are no candidates
    }
    // sums of 2^y, y = x log2 e + c: 8 per thread of at most 8 terms each, then a tree
    const float c = -fmul(ref, kLog2e);
    const bool plain = fabsf(ref) < 1e30f;  // (else x log2 e may leave f32's range)
    unsigned long long part[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) part[j] = f2_pack(0.f, 0.f);
    if (plain) {
        const unsigned long long l2 = f2_pack(kLog2e, kLog2e), c2 = f2_pack(c, c);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[V];
            unpack<T>(x[i], v);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                const float2 y = f2_unpack(f2_fma(f2_pack(v[2 * j], v[2 * j + 1]), l2, c2));
                const int a = V == 8 ? j : (i & 1) * 2 + j;
                part[a] = f2_add(part[a], f2_pack(ex2(y.x), ex2(y.y)));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[V];
            unpack<T>(x[i], v);
#pragma unroll
            for (int j = 0; j < V; ++j) part[0] = f2_add(part[0], f2_pack(ex2((v[j] - ref) * kLog2e), 0.f));
        }
    }
    const float2 pair = f2_unpack(f2_add(f2_add(part[0], part[1]), f2_add(part[2], part[3])));
    double sum = double(pair.x + pair.y);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    const float least = threshold;
    if (top >= least) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (quad[i] >= least) {
                float v[V];
                unpack<T>(x[i], v);
                unsigned pass = 0;
#pragma unroll
                for (int j = 0; j < V; ++j) pass |= unsigned(v[j] >= least) << j;
                for (; pass; pass &= pass - 1) {
                    const int j = __ffs(pass) - 1, at = atomicAdd(&count, 1);
                    if (at < kCap) cand[at] = key_of(pick<T>(x[i], j), (first + i * kPartThreads) * V - lead + j);
                }
            }
    }
    __syncthreads();
    unsigned long long* best = out.best + size_t(slot) * k;
    int n = count;
    if (n > kMany && n <= kCap) {  // the same once more among them, so that fewer have to be ranked
        unsigned long long mine[kCap / kPartThreads];
        unsigned most = 0;
#pragma unroll
        for (int u = 0; u < kCap / kPartThreads; ++u) {
            mine[u] = tid + u * kPartThreads < n ? cand[tid + u * kPartThreads] : 0;
            most = max(most, unsigned(mine[u] >> 32));
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        if ((tid & 1) == 0) again[tid / 2] = most;
        __syncthreads();
        if (tid == 0) count = 0;
        if (warp == 0) {
            const unsigned t = kth_of<4>(again, k);
            if (lane == 0) threshold = unorder(t);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kCap / kPartThreads; ++u)
            if (mine[u] && unsigned(mine[u] >> 32) >= order(threshold)) cand[atomicAdd(&count, 1)] = mine[u];
        __syncthreads();
        n = count;
    }
    if (n <= kCap) {
        for (int a = tid; a < n; a += kPartThreads) {
            const unsigned long long v = cand[a];
            int rank = 0;
            for (int o = 0; o < n; ++o) rank += cand[o] > v;
            if (rank < k) best[rank] = v;
        }
        for (int a = n + tid; a < k; a += kPartThreads) best[a] = 0;
    } else {  // very many equal logits: the best one below the last, k times
        unsigned long long last = ~0ull;
        for (int a = 0; a < k; ++a) {
            unsigned long long v = 0;
            for (int t = max(t0, 0) + tid; t < min(t1, vocab); t += kPartThreads) {
                const float f = to_float(row[t]);
                const unsigned long long w = key_of(f, t);
                if (f >= least && w < last && w > v) v = w;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
            __syncthreads();
            if (lane == 0) cand[warp] = v;
            __syncthreads();
            last = 0;
            for (int w = 0; w < W; ++w) last = max(last, cand[w]);
            if (tid == 0) best[a] = last;
        }
    }
    if (tid == 0) {
        double t = 0;
        for (int w = 0; w < W; ++w) t += sums[w];
        const double off = plain ? double(fmaf(ref, kLog2e, c)) * -0.6931471805599453 : 0.;  // what the terms of `top` lack
        out.sum[slot] = t * (fabs(off) < 1e-5 ? 1. + off + off * off / 2 : exp(off));
        out.top[slot] = row_top;
    }
}

// One candidate in the merge's order: a score and its place in the group.
struct Found {
    double score;
    unsigned at;  // beam * vocab + token
    unsigned pad;
};
__device__ __forceinline__ bool before(double s, unsigned at, double t, unsigned other) { return s > t || (s == t && at < other); }

// Order-preserving key of a score.
__device__ __forceinline__ unsigned long long order64(double x) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(x == 0. ? 0. : x);
    return b ^ (b >> 63 ? ~0ull : 1ull << 63);
}

// e^t for t <= 0 as f32: the rounding of t log2 e made good.
__device__ __forceinline__ float exp_neg(float t) {
    t = fmaxf(t, -150.f);
    const float y = fmul(t, kLog2e), e = ex2(y);
    return fmaf(fmul(e, fmaf(t, kLog2e, -y)), 0.6931471805599453f, e);
}

// log of the sum of exponentials of a row, by a warp, from its stretches; NaN where the row has no candidates.
__device__ double join_sums(const BeamParts& in, size_t slot) {
    constexpr int U = 4;  // stretches of a lane that are read once
    const int lane = threadIdx.x & 31;
    float t[U], top = -INFINITY;
    double v[U], sum = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int s = lane + 32 * u;
        t[u] = s < in.splits ? __ldcg(in.top + slot + s) : -INFINITY;
        v[u] = s < in.splits ? __ldcg(in.sum + slot + s) : 0.;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, t[u]);
    for (int s = lane + 32 * U; s < in.splits; s += 32) top = fmaxf(top, __ldcg(in.top + slot + s));
    top = warp_max(top);
    // (a stretch of forbidden tokens has the sum 0, one with NaN or +inf a NaN)
#pragma unroll
    for (int u = 0; u < U; ++u) sum += v[u] * double(exp_neg(t[u] - top));
    for (int s = lane + 32 * U; s < in.splits; s += 32) sum += __ldcg(in.sum + slot + s) * double(exp_neg(__ldcg(in.top + slot + s) - top));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return top == -INFINITY ? __longlong_as_double(0x7ff8000000000000ll) : double(top) + log(sum);
}

// A CTA per group.  A candidate's key is read once and kept in a register (kHeld of a thread; more are read again).  As in
// k_beam_part, a threshold that at least k + 1 candidates reach comes from the largest of each of 64 (or 128) groups of threads;
// those that reach it are ranked by counting.
constexpr int kHeld = 4;

template <class T>
__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(const T* __restrict__ logits, long long stride, int vocab, int beams,
                                                              const float* __restrict__ scores, const uint8_t* __restrict__ ended,
                                                              int end_id, int k, BeamParts in, unsigned row_magic,
                                                              float* __restrict__ out_scores, int* __restrict__ tokens,
                                                              int* __restrict__ parents) {
    constexpr int W = kMergeThreads / 32;
    // Twice the error of a log sum: of a term 2^-22 (the exponential), ln 2 2^-20 (y below 32), 21 * 1.4e-8 (log2 e as f32); 11 roundings
    // of a thread's sum; 2^-22 of a stretch's weight.  In all below 2.2e-6.
    constexpr double kNear = 5e-6;
    extern __shared__ double lse[];                                     // [beams]; NaN: no candidates of this row
    float* score = reinterpret_cast<float*>(lse + beams);               // [beams]
    unsigned char* again = reinterpret_cast<unsigned char*>(score + beams);  // [beams] rows whose sums are formed again
    __shared__ unsigned group_top[32 * 4];
    __shared__ unsigned threshold;
    __shared__ int count, redo;
    __shared__ Found found[kCap];
    __shared__ Found best[kBeamMaxK + 1];
    __shared__ double sums[W];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = blockIdx.x, r0 = group * beams;
    for (int b = tid; b < beams; b += kMergeThreads) {
        const float sc = __ldg(scores + r0 + b);
        const bool over = ended && __ldg(ended + r0 + b);
        score[b] = sc;
        again[b] = fabsf(sc) <= kMaxF ? over ? 2 : 0 : 3;  // 2: has ended, 3: has no candidates
    }
    if (tid == 0) redo = count = 0;
    __syncthreads();
    pdl_wait();
    const int per_row = in.splits * k, listed = beams * per_row;
    const unsigned long long* lists = in.best + size_t(r0) * per_row;
    unsigned long long held[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int c = tid + u * kMergeThreads;
        held[u] = c < listed ? __ldcg(lists + c) : 0;
    }
    for (int b = warp; b < beams; b += W) {
        const double l = again[b] ? __longlong_as_double(0x7ff8000000000000ll) : join_sums(in, size_t(r0 + b) * in.splits);
        if (lane == 0) lse[b] = l;
    }
    __syncthreads();
    auto row_of = [&](int c) { return row_magic ? int(__umulhi(unsigned(c), row_magic)) : c / per_row; };
    // f(score, place) for every candidate of this thread
    auto each = [&](auto&& f) {
        auto one = [&](int c, unsigned long long key) {
            const int b = row_of(c);
            const double l = lse[b];
            if (key && l == l)
                f(double(score[b]) + (double(unorder(unsigned(key >> 32))) - l), unsigned(b) * unsigned(vocab) + (0xffffffffu - unsigned(key)));
        };
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (tid + u * kMergeThreads < listed) one(tid + u * kMergeThreads, held[u]);
        for (int c = tid + kHeld * kMergeThreads; c < listed; c += kMergeThreads) one(c, __ldcg(lists + c));
        if (ended)
            for (int b = tid; b < beams; b += kMergeThreads)
                if (again[b] == 2) f(double(score[b]), unsigned(b) * unsigned(vocab) + unsigned(end_id));
    };
    int n_best = 0;
    for (int round = 0; round < 2; ++round) {
        unsigned top = 0;  // the upper half of the order is enough for a threshold
        each([&](double sc, unsigned) { top = max(top, unsigned(order64(sc) >> 32)); });
        const bool small = k < 32;
        const int of = kMergeThreads / (small ? 64 : 128);  // threads of a group
        for (int o = 1; o < of; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (tid % of == 0) group_top[tid / of] = top;
        __syncthreads();
        if (warp == 0) {  // one more than k, so that the k-th's distance to the next is known
            const unsigned t = small ? kth_of<2>(group_top, k + 1) : kth_of<4>(group_top, k + 1);
            if (lane == 0) threshold = t;
        }
        __syncthreads();
        const unsigned least = threshold;
        each([&](double sc, unsigned at) {
            if (unsigned(order64(sc) >> 32) >= least) {
                const int i = atomicAdd(&count, 1);
                if (i < kCap) found[i] = Found{sc, at, 0};
            }
        });
        __syncthreads();
        const int n = count;
        n_best = min(n, k + 1);
        if (n <= kCap) {
            for (int c = tid; c < n; c += kMergeThreads) {
                const Found mine = found[c];
                int rank = 0;
                for (int o = 0; o < n; ++o) rank += before(found[o].score, found[o].at, mine.score, mine.at);
                if (rank <= k) best[rank] = mine;
            }
        } else {  // very many equal scores: the best one behind the last, k + 1 times
            Found last{INFINITY, 0, 0};
            for (int i = 0; i <= k; ++i) {
                Found mine{-INFINITY, UINT_MAX, 0};
                each([&](double sc, unsigned at) {
                    if ((i == 0 || before(last.score, last.at, sc, at)) && before(sc, at, mine.score, mine.at)) mine = Found{sc, at, 0};
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const double sc = __shfl_xor_sync(0xffffffffu, mine.score, o);
                    const unsigned at = __shfl_xor_sync(0xffffffffu, mine.at, o);
                    if (before(sc, at, mine.score, mine.at)) mine = Found{sc, at, 0};
                }
                __syncthreads();
                if (lane == 0) found[warp] = mine;
                __syncthreads();
                last = found[0];
                for (int w = 1; w < W; ++w)
                    if (before(found[w].score, found[w].at, last.score, last.at)) last = found[w];
                if (tid == 0) best[i] = last;
            }
        }
        __syncthreads();
        if (round) break;
        for (int i = tid; i + 1 < n_best; i += kMergeThreads) {
            const unsigned a = best[i].at / unsigned(vocab), b = best[i + 1].at / unsigned(vocab);
            if (a != b && best[i].score - best[i + 1].score < kNear) {
                if (again[a] == 0) again[a] = 1;  // (an ended beam's score is exact)
                if (again[b] == 0) again[b] = 1;
                redo = 1;
            }
        }
        if (tid == 0) count = 0;
        __syncthreads();
        if (!redo) break;
        for (int b = 0; b < beams; ++b) {
            if (again[b] != 1) continue;
            const T* row = logits + (r0 + b) * stride;
            float top_f = -INFINITY;
            for (int s = 0; s < in.splits; ++s) top_f = fmaxf(top_f, __ldcg(in.top + size_t(r0 + b) * in.splits + s));
            double sum = 0;
            for (int t = tid; t < vocab; t += kMergeThreads) sum += exp(double(to_float(row[t])) - double(top_f));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sums[warp] = sum;
            __syncthreads();
            if (tid == 0) {
                double t = 0;
                for (int w = 0; w < W; ++w) t += sums[w];
                lse[b] = double(top_f) + log(t);
            }
            __syncthreads();
        }
    }
    const int have = min(n_best, k);
    out_scores += size_t(group) * k;
    tokens += size_t(group) * k;
    parents += size_t(group) * k;
    for (int i = tid; i < have; i += kMergeThreads) {
        const unsigned b = best[i].at / unsigned(vocab);
        out_scores[i] = float(best[i].score);
        parents[i] = int(b);
        tokens[i] = int(best[i].at - b * unsigned(vocab));
    }
    // fewer than k: all that are left are -inf, in order of their places; the first k places hold at most `have` of the best
    if (have < k && warp == 0) {
        int next = have;
        for (int p0 = 0; p0 < 2 * k && next < k; p0 += 32) {
            const unsigned p = unsigned(p0 + lane);
            bool left = true;
            for (int i = 0; i < have; ++i) left &= best[i].at != p;
            const unsigned mask = __ballot_sync(0xffffffffu, left);
            const int i = next + __popc(mask & ((1u << lane) - 1));
            if (left && i < k) {
                out_scores[i] = -INFINITY;
                parents[i] = int(p / unsigned(vocab));
                tokens[i] = int(p % unsigned(vocab));
            }
            next += __popc(mask);
        }
    }
}

// Bytes of a row that a thread takes.  Few rows: short stretches, so that every SM has work; many: long ones, whose fixed costs (about
// 250 instructions a warp) weigh less.
int thread_bytes(const BeamArgs& a) {
    const long long bytes = (long long)a.groups * a.beams * a.vocab * (a.type == KV_F32 ? 4 : 2);
    const long long per_sm = bytes / 148 / kPartThreads;
    return per_sm < 2 * 64 ? 32 : per_sm < 8 * 128 ? 64 : 128;
}
int pieces_of(const BeamArgs& a) {  // 16-byte pieces of a row, one that it shares with what comes before it included
    const int v = a.type == KV_F32 ? 4 : 8;
    return (a.vocab + 2 * (v - 1)) / v;
}
int splits_of(const BeamArgs& a) {
    const int most = kPartThreads * thread_bytes(a) / 16;
    return (pieces_of(a) + most - 1) / most;
}

template <class T, int E>
cudaError_t select_e(const BeamArgs& a, const BeamParts& p, cudaStream_t st) {
    // 32 groups of 8 threads where that gives several times k of them with pieces of their own, else 128 of 2
    auto part = a.k <= 24 && p.pieces >= 16 * a.k ? k_beam_part<T, E, 1> : k_beam_part<T, E, 4>;
    const unsigned rows = unsigned(a.groups) * unsigned(a.beams);
    cudaError_t e = launch_pdl(part, dim3(rows * unsigned(p.splits)), dim3(kPartThreads), 0, st, false, static_cast<const T*>(a.logits),
                               a.stride, a.vocab, a.scores, a.ended, a.k, p);
    if (e != cudaSuccess) return e;
    const int per_row = p.splits * a.k;  // c / per_row = umulhi(c, ceil(2^32 / per_row)) for both below 2^16, per_row > 1
    const unsigned magic = (long long)a.beams * per_row < 65536 && per_row > 1 ? unsigned((0x100000000ULL + per_row - 1) / per_row) : 0;
    return launch_pdl(k_beam_merge<T>, dim3(unsigned(a.groups)), dim3(kMergeThreads), size_t(a.beams) * 13, st, true,
                      static_cast<const T*>(a.logits), a.stride, a.vocab, a.beams, a.scores, a.ended, a.end_id, a.k, p, magic, a.out_scores,
                      a.tokens, a.parents);
}

template <class T>
cudaError_t select_t(const BeamArgs& a, const BeamParts& p, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    switch (thread_bytes(a)) {
        case 32: return select_e<T, 2 * V>(a, p, st);
        case 64: return select_e<T, 4 * V>(a, p, st);
        default: return select_e<T, 8 * V>(a, p, st);
    }
}

}  // namespace

size_t beam_ws_bytes(const BeamArgs& a) { return size_t(a.groups) * a.beams * splits_of(a) * (size_t(a.k) * 8 + 8 + 4); }

cudaError_t launch_beam_select(const BeamArgs& a, void* ws, cudaStream_t st) {
    if (a.groups == 0) return cudaSuccess;
    BeamParts p;
    p.splits = splits_of(a);
    p.pieces = (pieces_of(a) + p.splits - 1) / p.splits;
    const size_t slots = size_t(a.groups) * a.beams * p.splits;
    p.best = static_cast<unsigned long long*>(ws);
    p.sum = reinterpret_cast<double*>(p.best + slots * a.k);
    p.top = reinterpret_cast<float*>(p.sum + slots);
    switch (a.type) {
        case KV_F32: return select_t<float>(a, p, st);
        case KV_F16: return select_t<__half>(a, p, st);
        default: return select_t<__nv_bfloat16>(a, p, st);
    }
}

}  // namespace qb
