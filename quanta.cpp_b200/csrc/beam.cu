// The selection of a beam search's next step: of every group's candidates
//     s(b, t) = score_b + logit_bt - log sum_u exp(logit_bu)
// the k best, equal ones by the lowest b * vocab + t.  An ended beam has one candidate, its score with token end_id.  Candidates
// that are not numbers (a row with NaN or +inf, a beam whose score is not finite) count as -inf, as forbidden tokens do, and come
// after all others.
//
// The logits are read once, in tiles of 2 KB.  Within a beam the order is that of the logits, whatever the sum, and the k best
// candidates lie in the k tiles with the best largest candidates (of equal ones the first).  So k_beam_tiles leaves of a tile no
// more than its largest logit and its sum of exponentials: no warp waits for another, nothing is selected on the way.
// k_beam_merge, a CTA per group, joins the sums, ranks the tiles and opens the k best of them.  Scores are formed and compared in
// 64 bits.  The sums carry an error of their f32 exponentials and roundings, below 2.2e-6; where two beams' candidates lie closer
// than that could move them, the sums of these beams are formed again in 64 bits.
#include <climits>
#include <type_traits>

#include "beam.h"
#include "rows.cuh"

namespace qb {

namespace {

constexpr int kTilePieces = 4;       // 16-byte pieces of a lane in a tile
constexpr int kTileThreads = 256;
constexpr int kTileCtas = 6;         // on an SM
constexpr int kMergeThreads = 512;
constexpr int kCap = 1024;           // candidates that pass a threshold; more are taken one at a time
constexpr float kMaxF = 3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f;

// Order-preserving key of a logit.
__device__ __forceinline__ unsigned order(float x) {
    const unsigned b = __float_as_uint(x);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unorder(unsigned k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }

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
// The first of 16 bytes' elements, and the others moved down by one.
template <class T>
__device__ __forceinline__ float first_of(uint4 w) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w.x);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(static_cast<unsigned short>(w.x)));
    else return __uint_as_float(w.x << 16);
}
template <class T>
__device__ __forceinline__ uint4 next_of(uint4 w) {
    if constexpr (sizeof(T) == 4) return make_uint4(w.y, w.z, w.w, 0);
    else return make_uint4(__funnelshift_r(w.x, w.y, 16), __funnelshift_r(w.y, w.z, 16), __funnelshift_r(w.z, w.w, 16), w.w >> 16);
}
// The bits of -inf, twice where the type has 16.
template <class T>
constexpr unsigned kForbidden = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;


// A row as 16-byte pieces as they lie in memory: piece p holds the tokens p * V - lead ..; the first one may hold elements that come
// before the row.  Elements outside the row read as -inf.
template <class T>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    const T* at;
    int lead;
    __device__ __forceinline__ Row(const T* row) : at(row), lead(int(reinterpret_cast<uintptr_t>(row) / sizeof(T) % V)) {}
    __device__ __forceinline__ const uint4* pieces() const { return reinterpret_cast<const uint4*>(at - lead); }
    __device__ __forceinline__ uint4 piece(int p, int vocab) const {
        const int e = p * V - lead;
        if (e >= 0 && e + V <= vocab) return __ldcs(pieces() + p);
        uint4 x = make_uint4(kForbidden<T>, kForbidden<T>, kForbidden<T>, kForbidden<T>);
        T* v = reinterpret_cast<T*>(&x);
        if (e < vocab && e + V > 0)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (e + j >= 0 && e + j < vocab) v[j] = at[e + j];
        return x;
    }
};

// A tile's largest logit (NaN aside; -inf: none above it) and the sum of exp(x - largest), NaN where it holds NaN or +inf.
struct Tile {
    float top, sum;
};

// A warp per tile, one after another.  Bound by HBM; next to it by instructions: a logit costs half a packed maximum, its conversion,
// half a packed fused y = x log2 e + c, the exponential and half a packed sum.  c is the f32 next to -top log2 e, and what it lacks
// is made good in the sum.
template <class T>
__global__ void __launch_bounds__(kTileThreads, kTileCtas)
    k_beam_tiles(const T* __restrict__ logits, long long stride, int vocab, const float* __restrict__ scores,
                 const uint8_t* __restrict__ ended, int row_tiles, int tiles, Tile* __restrict__ out) {
    constexpr int U = kTilePieces, V = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, warps = gridDim.x * (kTileThreads / 32);
    pdl_launch_dependents();
    for (int t = blockIdx.x * (kTileThreads / 32) + (threadIdx.x >> 5); t < tiles; t += warps) {
        const int r = t / row_tiles, j = t - r * row_tiles;
        const float score = __ldg(scores + r);
        const int over = ended ? __ldg(ended + r) : 0;
        if (over || !(fabsf(score) <= kMaxF)) continue;  // the merge does not look at this row
        const Row<T> row(logits + r * stride);
        const int p = j * (32 * U) + lane, e = j * (32 * U * V) - row.lead;
        uint4 x[U];
        if (e >= 0 && e + 32 * U * V <= vocab) {
            const uint4* from = row.pieces() + p;
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = __ldcs(from + 32 * u);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = row.piece(p + 32 * u, vocab);
        }
        float top = largest<T>(x[0]);
#pragma unroll
        for (int u = 1; u < U; ++u) top = fmaxf(top, largest<T>(x[u]));
        top = unorder(__reduce_max_sync(0xffffffffu, order(top + 0.f)));  // (-0 is 0)
        const float ref = top == -INFINITY ? 0.f : top, c = -fmul(ref, kLog2e);
        float sum, off = 0.f;
        if (fabsf(ref) < 1e5f) {  // 8 sums of 4 terms each, then a tree
            unsigned long long part[4];
            const unsigned long long l2 = f2_pack(kLog2e, kLog2e), c2 = f2_pack(c, c);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float v[V];
                unpack<T>(x[u], v);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const float2 y = f2_unpack(f2_fma(f2_pack(v[2 * i], v[2 * i + 1]), l2, c2));
                    const unsigned long long f = f2_pack(ex2(y.x), ex2(y.y));
                    const int a = V == 8 ? i : (u & 1) * 2 + i;
                    part[a] = u < (V == 8 ? 1 : 2) ? f : f2_add(part[a], f);
                }
            }
            const float2 pair = f2_unpack(f2_add(f2_add(part[0], part[1]), f2_add(part[2], part[3])));
            sum = pair.x + pair.y;
            off = fmaf(ref, kLog2e, c) * -0.6931471805599453f;
        } else {  // x log2 e would be too coarse, or leave f32's range
            double all = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll 1
                for (int i = 0; i < V; ++i) {
                    all += double(ex2((first_of<T>(x[u]) - ref) * kLog2e));
                    x[u] = next_of<T>(x[u]);
                }
            sum = float(all);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) out[t] = Tile{top, fmaf(sum, fmaf(off, off * 0.5f, off), sum)};
    }
}

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

// log of the sum of exponentials of a row, by a warp, from its tiles; NaN where the row has no candidates.
__device__ double join_sums(const Tile* tiles, int n) {
    constexpr int N = 8;  // tiles of a lane that are read once
    const int lane = threadIdx.x & 31;
    const float2* in = reinterpret_cast<const float2*>(tiles);
    float2 t[N];
#pragma unroll
    for (int u = 0; u < N; ++u) t[u] = lane + 32 * u < n ? __ldcg(in + lane + 32 * u) : make_float2(-INFINITY, 0.f);
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < N; ++u) top = fmaxf(top, t[u].x);
    for (int i = lane + 32 * N; i < n; i += 32) top = fmaxf(top, __ldcg(in + i).x);
    top = warp_max(top);
    double sum = 0;  // (a tile of forbidden tokens has the sum 0)
#pragma unroll
    for (int u = 0; u < N; ++u) sum += double(t[u].y) * double(exp_neg(t[u].x - top));
    for (int i = lane + 32 * N; i < n; i += 32) {
        const float2 v = __ldcg(in + i);
        sum += double(v.y) * double(exp_neg(v.x - top));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return top == -INFINITY ? __longlong_as_double(0x7ff8000000000000ll) : double(top) + log(sum);
}

struct MergeShared {
    unsigned group_top[32 * 4];
    unsigned threshold;
    int count, redo;
    Found found[kCap];
    Found best[kBeamMaxK + 1];
    double sums[kMergeThreads / 32];
};

// best[0 .. n - 1] = the n = min(k + 1, all) best of the items of the CTA's threads, in order; each(f) calls f(score, place) for every
// item of this thread, the same ones every time.  Items that reach a threshold, the (k + 1)-th largest of the largest of 64 (or 128)
// groups of threads, are ranked by counting.  `floor`: no item below it is wanted.
template <class Each>
__device__ int best_of(MergeShared& sh, int k, double floor, bool has_floor, Each&& each) {
    constexpr int W = kMergeThreads / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned least = 0;
    if (!has_floor) {
        unsigned top = 0;  // the upper half of the order is enough for a threshold
        each([&](double sc, unsigned) { top = max(top, unsigned(order64(sc) >> 32)); });
        const bool small = k < 32;
        const int of = kMergeThreads / (small ? 64 : 128);  // threads of a group
        for (int o = 1; o < of; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (tid % of == 0) sh.group_top[tid / of] = top;
        if (tid == 0) sh.count = 0;
        __syncthreads();
        if (warp == 0) {
            const unsigned t = small ? kth_of<2>(sh.group_top, k + 1) : kth_of<4>(sh.group_top, k + 1);
            if (lane == 0) sh.threshold = t;
        }
        __syncthreads();
        least = sh.threshold;
    } else {
        if (tid == 0) sh.count = 0;
        __syncthreads();
    }
    each([&](double sc, unsigned at) {
        if (has_floor ? sc >= floor : unsigned(order64(sc) >> 32) >= least) {
            const int i = atomicAdd(&sh.count, 1);
            if (i < kCap) sh.found[i] = Found{sc, at, 0};
        }
    });
    __syncthreads();
    const int n = sh.count;
    if (n <= kCap) {
        for (int c = tid; c < n; c += kMergeThreads) {
            const Found mine = sh.found[c];
            int rank = 0;
            for (int o = 0; o < n; ++o) rank += before(sh.found[o].score, sh.found[o].at, mine.score, mine.at);
            if (rank <= k) sh.best[rank] = mine;
        }
    } else {  // very many that reach it: the best one behind the last, k + 1 times
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
            if (lane == 0) sh.found[warp] = mine;
            __syncthreads();
            last = sh.found[0];
            for (int w = 1; w < W; ++w)
                if (before(sh.found[w].score, sh.found[w].at, last.score, last.at)) last = sh.found[w];
            if (tid == 0) sh.best[i] = last;
        }
    }
    __syncthreads();
    return min(n, k + 1);
}

// A CTA per group.
constexpr int kHeld = 4;  // tiles of a thread that are read once

template <class T>
__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(const T* __restrict__ logits, long long stride, int vocab, int beams,
                                                              const float* __restrict__ scores, const uint8_t* __restrict__ ended,
                                                              int end_id, int k, const Tile* __restrict__ tiles, int row_tiles,
                                                              unsigned row_magic, float* __restrict__ out_scores,
                                                              int* __restrict__ tokens, int* __restrict__ parents) {
    constexpr int U = kTilePieces, V = 16 / sizeof(T), W = kMergeThreads / 32;
    // Twice the error of a log sum: of a term 2^-22 (the exponential), ln 2 2^-20 (y above -32), 21 * 1.4e-8 (log2 e as f32); 12 roundings
    // of a tile's sum; 2^-22 of its weight.  In all below 2.2e-6.
    constexpr double kNear = 5e-6;
    extern __shared__ double lse[];                                          // [beams]; NaN: no candidates of this row
    float* score = reinterpret_cast<float*>(lse + beams);                    // [beams]
    unsigned char* state = reinterpret_cast<unsigned char*>(score + beams);  // [beams] 1: the sum is formed again, 2: exactly known, 3: none
    __shared__ MergeShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = blockIdx.x, r0 = group * beams;
    for (int b = tid; b < beams; b += kMergeThreads) {
        const float sc = __ldg(scores + r0 + b);
        const bool over = ended && __ldg(ended + r0 + b);
        score[b] = sc;
        state[b] = fabsf(sc) <= kMaxF ? over ? 2 : 0 : 3;
    }
    if (tid == 0) sh.redo = 0;
    __syncthreads();
    pdl_wait();
    const int n_tiles = beams * row_tiles;
    const Tile* mine = tiles + size_t(r0) * row_tiles;
    float held[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int c = tid + u * kMergeThreads;
        held[u] = c < n_tiles ? __ldcg(&mine[c].top) : -INFINITY;
    }
    for (int b = warp; b < beams; b += W) {
        const double l = state[b] ? __longlong_as_double(0x7ff8000000000000ll) : join_sums(mine + size_t(b) * row_tiles, row_tiles);
        if (lane == 0) lse[b] = l;
    }
    __syncthreads();
    auto row_of = [&](unsigned c) { return row_magic ? int(__umulhi(c, row_magic)) : int(c / unsigned(row_tiles)); };
    // the largest candidates of the group's tiles, with their numbers
    auto each_tile = [&](auto&& f) {
        auto one = [&](int c, float top) {
            const int b = row_of(c);
            const double l = lse[b];
            if (l == l && top != -INFINITY) f(double(score[b]) + (double(top) - l), unsigned(c));
        };
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (tid + u * kMergeThreads < n_tiles) one(tid + u * kMergeThreads, held[u]);
        for (int c = tid + kHeld * kMergeThreads; c < n_tiles; c += kMergeThreads) one(c, __ldcg(&mine[c].top));
        if (ended)
            for (int b = tid; b < beams; b += kMergeThreads)
                if (state[b] == 2 && lse[b] != lse[b]) f(double(score[b]), unsigned(b) * unsigned(row_tiles));
    };
    // Whether two beams' candidates lie too close to each other in best[0 .. n - 1]; then their sums are formed again.
    auto settle = [&](int n, unsigned per_row) {
        for (int i = tid; i + 1 < n; i += kMergeThreads) {
            const unsigned a = sh.best[i].at / per_row, b = sh.best[i + 1].at / per_row;
            if (a != b && sh.best[i].score - sh.best[i + 1].score < kNear) {
                if (state[a] == 0) state[a] = 1, sh.redo = 1;
                if (state[b] == 0) state[b] = 1, sh.redo = 1;
            }
        }
        __syncthreads();
        if (!sh.redo) return false;
        for (int b = 0; b < beams; ++b) {
            if (state[b] != 1) continue;
            const T* row = logits + (r0 + b) * stride;
            float top = -INFINITY;
            for (int i = 0; i < row_tiles; ++i) top = fmaxf(top, __ldcg(&mine[size_t(b) * row_tiles + i].top));
            double sum = 0;
            for (int t = tid; t < vocab; t += kMergeThreads) sum += exp(double(to_float(row[t])) - double(top));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sh.sums[warp] = sum;
            __syncthreads();
            if (tid == 0) {
                double t = 0;
                for (int w = 0; w < W; ++w) t += sh.sums[w];
                lse[b] = double(top) + log(t);
                state[b] = 2;
            }
            __syncthreads();
        }
        if (tid == 0) sh.redo = 0;
        __syncthreads();
        return true;
    };
    int n = best_of(sh, k, 0., false, each_tile);
    if (settle(n, unsigned(row_tiles))) n = best_of(sh, k, 0., false, each_tile);
    // the candidates of the k best tiles that reach the last one's largest
    const int open = min(n, k);
    bool bounded = n >= k;
    const double floor = bounded ? sh.best[k - 1].score : 0.;
    __shared__ unsigned tile_of[kBeamMaxK];
    for (int i = tid; i < open; i += kMergeThreads) tile_of[i] = sh.best[i].at;
    __syncthreads();
    auto each_token = [&](auto&& f) {
        for (int c = tid; c < open * 32 * U; c += kMergeThreads) {
            const unsigned tile = tile_of[c / (32 * U)];
            const int b = row_of(tile), j = int(tile) - b * row_tiles;
            const double l = lse[b], sc = double(score[b]);
            if (l != l) {  // an ended beam
                if (c % (32 * U) == 0) f(sc, unsigned(b) * unsigned(vocab) + unsigned(end_id));
                continue;
            }
            const Row<T> row(logits + (r0 + b) * stride);
            const int p = j * (32 * U) + c % (32 * U);
            uint4 x = row.piece(p, vocab);
            const float top = largest<T>(x);
            if (top == -INFINITY || (bounded && sc + (double(top) - l) < floor)) continue;
#pragma unroll 1
            for (int i = 0; i < V; ++i) {
                const float v = first_of<T>(x);
                if (v != -INFINITY) f(sc + (double(v) - l), unsigned(b) * unsigned(vocab) + unsigned(p * V - row.lead + i));
                x = next_of<T>(x);
            }
        }
    };
    n = best_of(sh, k, floor, bounded, each_token);
    if (settle(n, unsigned(vocab))) {
        bounded = false;  // (the sums have moved a little)
        n = best_of(sh, k, 0., false, each_token);
    }
    const int have = min(n, k);
    out_scores += size_t(group) * k;
    tokens += size_t(group) * k;
    parents += size_t(group) * k;
    for (int i = tid; i < have; i += kMergeThreads) {
        const unsigned b = sh.best[i].at / unsigned(vocab);
        out_scores[i] = float(sh.best[i].score);
        parents[i] = int(b);
        tokens[i] = int(sh.best[i].at - b * unsigned(vocab));
    }
    // fewer than k: all that are left are -inf, in order of their places; the first k places hold at most `have` of the best
    if (have < k && warp == 0) {
        int next = have;
        for (int p0 = 0; p0 < 2 * k && next < k; p0 += 32) {
            const unsigned p = unsigned(p0 + lane);
            bool left = true;
            for (int i = 0; i < have; ++i) left &= sh.best[i].at != p;
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

int row_tiles_of(const BeamArgs& a) {  // (a row shares its first piece with what comes before it)
    const int v = a.type == KV_F32 ? 4 : 8, tile = 32 * kTilePieces * v;
    return (a.vocab + v - 1 + tile - 1) / tile;
}

template <class T>
cudaError_t select_t(const BeamArgs& a, Tile* ws, cudaStream_t st) {
    const int row_tiles = row_tiles_of(a), tiles = a.groups * a.beams * row_tiles, warps = kTileThreads / 32;
    const int ctas = (tiles + warps - 1) / warps, most = 148 * kTileCtas;
    cudaError_t e = launch_pdl(k_beam_tiles<T>, dim3(unsigned(ctas < most ? ctas : most)), dim3(kTileThreads), 0, st, false,
                               static_cast<const T*>(a.logits), a.stride, a.vocab, a.scores, a.ended, row_tiles, tiles, ws);
    if (e != cudaSuccess) return e;
    // c / row_tiles = umulhi(c, ceil(2^32 / row_tiles)) for both below 2^16, row_tiles > 1
    const bool small = (long long)a.beams * row_tiles < 65536 && row_tiles > 1;
    return launch_pdl(k_beam_merge<T>, dim3(unsigned(a.groups)), dim3(kMergeThreads), size_t(a.beams) * 13, st, true,
                      static_cast<const T*>(a.logits), a.stride, a.vocab, a.beams, a.scores, a.ended, a.end_id, a.k,
                      static_cast<const Tile*>(ws), row_tiles, small ? unsigned((0x100000000ULL + row_tiles - 1) / row_tiles) : 0u,
                      a.out_scores, a.tokens, a.parents);
}

}  // namespace

size_t beam_ws_bytes(const BeamArgs& a) { return size_t(a.groups) * a.beams * row_tiles_of(a) * sizeof(Tile); }

cudaError_t launch_beam_select(const BeamArgs& a, void* ws, cudaStream_t st) {
    if (a.groups == 0) return cudaSuccess;
    Tile* t = static_cast<Tile*>(ws);
    switch (a.type) {
        case KV_F32: return select_t<float>(a, t, st);
        case KV_F16: return select_t<__half>(a, t, st);
        default: return select_t<__nv_bfloat16>(a, t, st);
    }
}

}  // namespace qb
