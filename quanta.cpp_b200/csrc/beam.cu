// The selection of a beam search's next step: of every group's candidates
//     s(b, t) = score_b + logit_bt - log sum_u exp(logit_bu)
// the k best, equal ones by the lowest b * vocab + t.  An ended beam has one candidate, its score with token end_id.  Candidates
// that are not numbers (a row with NaN or +inf, a beam whose score is not finite) count as -inf, as forbidden tokens do, and come
// after all others.
//
// The logits are read once.  Within a beam the order is that of the logits, whatever the sum: k_beam_part takes a stretch of a
// row into registers and leaves its largest logit, its sum of exponentials and its k best logits.  k_beam_merge, a CTA per group,
// joins the sums and orders the candidates in 64 bits.  Its sums of exponentials carry an error of the f32 exponentials, below
// 2^-20; where two beams' candidates lie closer than that could move them, the sums of these beams are formed again in 64 bits.
#include <climits>

#include "beam.h"
#include "rows.cuh"

namespace qb {

namespace {

constexpr int kPartThreads = 256;
constexpr int kMergeThreads = 256;
constexpr int kCap = 1024;  // candidates that pass the threshold; more are taken one at a time
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

// exp(t) for t <= 0 (NaN stays): 2^y with y = t * log2 e and the rounding of y made good.  Relative error below 2^-22 of the
// hardware's exponential plus |t| * 1.4e-8 of log2 e as f32.
__device__ __forceinline__ float exp_neg(float t) {
    const float log2e = 1.4426950408889634f, ln2 = 0.6931471805599453f;
    t = max_or_nan(t, -150.f);  // (an infinity would leave no rounding to make good)
    const float y = fmul(t, log2e), lo = fmaf(t, log2e, -y);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return fmaf(fmul(e, lo), ln2, e);
}

// Where the sums and the candidates of stretch s of row r lie: slot r * splits + s.
struct BeamParts {
    double* sum;   // sum of exp(x - top)
    float* top;    // largest logit of the stretch (-inf: none above it)
    unsigned long long* best;  // [k] keys, descending, 0 past the last one
    int splits;
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

// A stretch of kPartThreads * E logits of a row.  G: 32 G groups of threads whose maxima give the threshold, at least k of them.
template <class T, int E, int G>
__global__ void __launch_bounds__(kPartThreads) k_beam_part(const T* __restrict__ logits, long long stride, int vocab,
                                                            const float* __restrict__ scores, const uint8_t* __restrict__ ended,
                                                            int k, BeamParts out) {
    constexpr int V = 16 / sizeof(T), N = E / V, W = kPartThreads / 32, GROUP = kPartThreads / (32 * G);
    __shared__ unsigned group_top[32 * G];
    __shared__ float threshold;
    __shared__ int count;
    __shared__ double sums[W];
    __shared__ unsigned long long cand[kCap];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned slot = blockIdx.x, r = slot / unsigned(out.splits), s = slot - r * unsigned(out.splits);
    pdl_launch_dependents();
    if ((ended && __ldg(ended + r)) || !(fabsf(__ldg(scores + r)) <= kMaxF)) return;  // the merge does not look at this row
    const T* row = logits + r * stride;
    // 16-byte pieces as they lie in memory; the row's first one may hold elements that come before it
    const int lead = int(reinterpret_cast<uintptr_t>(row) / sizeof(T) % V), piece0 = int(s) * kPartThreads * N;
    const T* base = row - lead;
    float x[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const long long e = (long long)(piece0 + i * kPartThreads + tid) * V - lead;  // token of the piece's first element
        if (e >= 0 && e + V <= vocab) {
            union {
                uint4 u;
                Pack<T, V> w;
            };
            u = __ldcs(reinterpret_cast<const uint4*>(base) + piece0 + i * kPartThreads + tid);
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = to_float(w.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = e + j >= 0 && e + j < vocab ? to_float(row[e + j]) : -INFINITY;
        }
    }
    if (tid == 0) count = 0;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) top = fmaxf(top, x[i][j]);
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
    float part[V];
#pragma unroll
    for (int j = 0; j < V; ++j) part[j] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) part[j] += exp_neg(x[i][j] - ref);
#pragma unroll
    for (int o = V / 2; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < o; ++j) part[j] += part[j + o];
    double sum = double(part[0]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    const float least = threshold;
    if (top >= least) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (x[i][j] >= least) {
                    const int at = atomicAdd(&count, 1);
                    if (at < kCap) cand[at] = key_of(x[i][j], (piece0 + i * kPartThreads + tid) * V - lead + j);
                }
    }
    __syncthreads();
    unsigned long long* best = out.best + size_t(slot) * k;
    const int n = count;
    if (n <= kCap) {
        for (int c = tid; c < n; c += kPartThreads) {
            const unsigned long long v = cand[c];
            int rank = 0;
            for (int o = 0; o < n; ++o) rank += cand[o] > v;
            if (rank < k) best[rank] = v;
        }
        for (int c = n + tid; c < k; c += kPartThreads) best[c] = 0;
    } else {  // very many equal logits: the best one below the last, k times
        unsigned long long last = ~0ull;
        for (int c = 0; c < k; ++c) {
            unsigned long long v = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (x[i][j] >= least) {
                        const unsigned long long w = key_of(x[i][j], (piece0 + i * kPartThreads + tid) * V - lead + j);
                        if (w < last && w > v) v = w;
                    }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
            __syncthreads();
            if (lane == 0) cand[warp] = v;
            __syncthreads();
            last = 0;
            for (int w = 0; w < W; ++w) last = max(last, cand[w]);
            if (tid == 0) best[c] = last;
        }
    }
    if (tid == 0) {
        double t = 0;
        for (int w = 0; w < W; ++w) t += sums[w];
        out.sum[slot] = t;
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

// A CTA per group.  Dynamic shared memory: [beams] log sums (NaN: the row has no candidates but perhaps itself).
template <class T>
__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(const T* __restrict__ logits, long long stride, int vocab, int beams,
                                                              const float* __restrict__ scores, const uint8_t* __restrict__ ended,
                                                              int end_id, int k, BeamParts in, float* __restrict__ out_scores,
                                                              int* __restrict__ tokens, int* __restrict__ parents) {
    constexpr int W = kMergeThreads / 32;
    constexpr double kNear = 2e-6;  // twice the error of a log sum: 2^-22.x of the exponential and 4 roundings of its f32 sums
    extern __shared__ double lse[];
    unsigned* again = reinterpret_cast<unsigned*>(lse + beams);  // rows whose sums are formed again
    __shared__ unsigned group_top[32 * 4];
    __shared__ unsigned threshold;
    __shared__ int count, redo;
    __shared__ Found found[kCap];
    __shared__ Found best[kBeamMaxK + 1];
    __shared__ double sums[W];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = blockIdx.x, r0 = group * beams;
    pdl_wait();
    for (int b = warp; b < beams; b += W) {
        const float sc = __ldg(scores + r0 + b);
        double l = __longlong_as_double(0x7ff8000000000000ll);
        if (fabsf(sc) <= kMaxF && !(ended && __ldg(ended + r0 + b))) {
            const size_t slot = size_t(r0 + b) * in.splits;
            float top = -INFINITY;
            for (int s = lane; s < in.splits; s += 32) top = fmaxf(top, __ldcg(in.top + slot + s));
            top = warp_max(top);
            double sum = 0;
            for (int s = lane; s < in.splits; s += 32) {
                const float t = __ldcg(in.top + slot + s);
                const double v = __ldcg(in.sum + slot + s);  // NaN where the stretch has NaN or +inf
                sum += t == -INFINITY ? v : v * exp(double(t) - double(top));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l = top == -INFINITY ? l : double(top) + log(sum);
        }
        if (lane == 0) {
            lse[b] = l;
            again[b] = 0;
        }
    }
    if (tid == 0) redo = 0;
    __syncthreads();
    const int per_row = in.splits * k, listed = beams * per_row, total = listed + beams;
    // candidate c of the lists, or of the beams that have ended; false: none
    auto look = [&](int c, double* score, unsigned* at) {
        if (c < listed) {
            const int b = c / per_row;
            const double l = lse[b];
            if (!(l == l)) return false;
            const unsigned long long key = __ldcg(in.best + size_t(r0) * per_row + c);
            if (key == 0) return false;
            *score = double(__ldg(scores + r0 + b)) + (double(unorder(unsigned(key >> 32))) - l);
            *at = unsigned(b) * unsigned(vocab) + (0xffffffffu - unsigned(key));
            return true;
        }
        const int b = c - listed;
        const float sc = __ldg(scores + r0 + b);
        if (!ended || !__ldg(ended + r0 + b) || !(fabsf(sc) <= kMaxF)) return false;
        *score = double(sc);
        *at = unsigned(b) * unsigned(vocab) + unsigned(end_id);
        return true;
    };
    int n_best = 0;
    for (int round = 0; round < 2; ++round) {
        if (tid == 0) count = 0;
        unsigned top = 0;  // upper half of the order: enough for a threshold
        for (int c = tid; c < total; c += kMergeThreads) {
            double sc;
            unsigned at;
            if (look(c, &sc, &at)) top = max(top, unsigned(order64(sc) >> 32));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        if (k < 32) top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int of = k < 32 ? 4 : 2;  // threads of a group: 64 groups, or 128
        if (tid % of == 0) group_top[tid / of] = top;
        __syncthreads();
        if (warp == 0) {  // one more than k, so that the k-th's distance to the next is known
            const unsigned t = k < 32 ? kth_of<2>(group_top, k + 1) : kth_of<4>(group_top, k + 1);
            if (lane == 0) threshold = t;
        }
        __syncthreads();
        const unsigned least = threshold;
        for (int c = tid; c < total; c += kMergeThreads) {
            double sc;
            unsigned at;
            if (look(c, &sc, &at) && unsigned(order64(sc) >> 32) >= least) {
                const int i = atomicAdd(&count, 1);
                if (i < kCap) found[i] = Found{sc, at, 0};
            }
        }
        __syncthreads();
        const int n = count;
        n_best = min(n, k + 1);
        if (n <= kCap) {
            for (int c = tid; c < n; c += kMergeThreads) {
                const double sc = found[c].score;
                const unsigned at = found[c].at;
                int rank = 0;
                for (int o = 0; o < n; ++o) rank += before(found[o].score, found[o].at, sc, at);
                if (rank <= k) best[rank] = found[c];
            }
        } else {  // one at a time
            double last = INFINITY;
            unsigned last_at = 0;
            for (int i = 0; i <= k; ++i) {
                double v = -INFINITY;
                unsigned v_at = UINT_MAX;
                for (int c = tid; c < total; c += kMergeThreads) {
                    double sc;
                    unsigned at;
                    if (look(c, &sc, &at) && (i == 0 || before(last, last_at, sc, at)) && before(sc, at, v, v_at)) {
                        v = sc;
                        v_at = at;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const double ov = __shfl_xor_sync(0xffffffffu, v, o);
                    const unsigned oat = __shfl_xor_sync(0xffffffffu, v_at, o);
                    if (before(ov, oat, v, v_at)) {
                        v = ov;
                        v_at = oat;
                    }
                }
                __syncthreads();
                if (lane == 0) found[warp] = Found{v, v_at, 0};
                __syncthreads();
                last = found[0].score;
                last_at = found[0].at;
                for (int w = 1; w < W; ++w)
                    if (before(found[w].score, found[w].at, last, last_at)) {
                        last = found[w].score;
                        last_at = found[w].at;
                    }
                if (tid == 0) best[i] = Found{last, last_at, 0};
            }
        }
        __syncthreads();
        if (round) break;
        for (int i = tid; i + 1 < n_best; i += kMergeThreads) {
            const unsigned a = best[i].at / unsigned(vocab), b = best[i + 1].at / unsigned(vocab);
            if (a != b && best[i].score - best[i + 1].score < kNear) {
                again[a] = again[b] = 1;
                redo = 1;
            }
        }
        __syncthreads();
        if (!redo) break;
        for (int b = 0; b < beams; ++b) {
            if (!again[b] || !(lse[b] == lse[b])) continue;
            const T* row = logits + (r0 + b) * stride;
            const size_t slot = size_t(r0 + b) * in.splits;
            float top_f = -INFINITY;
            for (int s = 0; s < in.splits; ++s) top_f = fmaxf(top_f, __ldcg(in.top + slot + s));
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
    for (int i = tid; i < have; i += kMergeThreads) {
        const unsigned b = best[i].at / unsigned(vocab);
        out_scores[size_t(group) * k + i] = float(best[i].score);
        parents[size_t(group) * k + i] = int(b);
        tokens[size_t(group) * k + i] = int(best[i].at - b * unsigned(vocab));
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
                out_scores[size_t(group) * k + i] = -INFINITY;
                parents[size_t(group) * k + i] = int(p / unsigned(vocab));
                tokens[size_t(group) * k + i] = int(p % unsigned(vocab));
            }
            next += __popc(mask);
        }
    }
}

// Elements of a thread.  Few rows: short stretches, so that every SM has work; many: long ones, whose fixed costs weigh less.
int elements(const BeamArgs& a) {
    return (long long)a.groups * a.beams * ((a.vocab + 8191) / 8192) < 2 * 148 ? 8 : 32;
}
int splits(const BeamArgs& a, int e) { return (a.vocab + 7 + kPartThreads * e - 1) / (kPartThreads * e); }  // (7: a row's lead)

template <class T, int E>
cudaError_t select_e(const BeamArgs& a, const BeamParts& p, cudaStream_t st) {
    auto part = a.k <= 32 ? k_beam_part<T, E, 1> : k_beam_part<T, E, 4>;
    const unsigned rows = unsigned(a.groups) * unsigned(a.beams);
    cudaError_t e = launch_pdl(part, dim3(rows * unsigned(p.splits)), dim3(kPartThreads), 0, st, false, static_cast<const T*>(a.logits),
                               a.stride, a.vocab, a.scores, a.ended, a.k, p);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_beam_merge<T>, dim3(unsigned(a.groups)), dim3(kMergeThreads), size_t(a.beams) * 12, st, true,
                      static_cast<const T*>(a.logits), a.stride, a.vocab, a.beams, a.scores, a.ended, a.end_id, a.k, p, a.out_scores,
                      a.tokens, a.parents);
}

template <class T>
cudaError_t select_t(const BeamArgs& a, const BeamParts& p, int e, cudaStream_t st) {
    return e == 8 ? select_e<T, 8>(a, p, st) : select_e<T, 32>(a, p, st);
}

}  // namespace

size_t beam_ws_bytes(const BeamArgs& a) {
    const size_t slots = size_t(a.groups) * a.beams * splits(a, elements(a));
    return slots * (size_t(a.k) * 8 + 8 + 4);
}

cudaError_t launch_beam_select(const BeamArgs& a, void* ws, cudaStream_t st) {
    if (a.groups == 0) return cudaSuccess;
    const int e = elements(a);
    BeamParts p;
    p.splits = splits(a, e);
    const size_t slots = size_t(a.groups) * a.beams * p.splits;
    p.best = static_cast<unsigned long long*>(ws);
    p.sum = reinterpret_cast<double*>(p.best + slots * a.k);
    p.top = reinterpret_cast<float*>(p.sum + slots);
    switch (a.type) {
        case KV_F32: return select_t<float>(a, p, e, st);
        case KV_F16: return select_t<__half>(a, p, e, st);
        default: return select_t<__nv_bfloat16>(a, p, e, st);
    }
}

}  // namespace qb
