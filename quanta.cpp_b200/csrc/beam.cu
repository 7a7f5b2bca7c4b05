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
// 64 bits.  The sums carry an error of their f32 exponentials and roundings, below 2.7e-6; where two beams' candidates lie closer
// than that could move them, the sums of these beams are formed again in 64 bits, by their group's CTA, a row after the other: rare
// between beams of their own, but with beams that are alike (copies of one prompt with equal scores) it is all of them, 50 to 80 us
// for each row of 151936 (64 x 4 bf16 610 us, 1 x 16 800, where unlike ones take 21 and 10.5).
#include <climits>
#include <type_traits>

#include "beam.h"
#include "rows.cuh"

namespace qb {

namespace {

constexpr int kTilePieces = 4;       // 16-byte pieces of a lane in a tile
constexpr int kTileThreads = 256;
constexpr int kTileCtas = 8;         // on an SM
constexpr int kMergeThreads = 1024;  // at most
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
// 256 rows of 151936 bf16 logits: 15.6 us, 5.0 TB/s, where a loop that only reads them takes 13.7 to 14.4 (4 CTAs per SM 17.0 us, the
// next tile through cp.async 16.7; candidates picked on the way, with thresholds from the tiles before, 30 us and more a call).
template <class T>
__global__ void __launch_bounds__(kTileThreads, kTileCtas)
    k_beam_tiles(const T* __restrict__ logits, long long stride, int vocab, const float* __restrict__ scores,
                 const uint8_t* __restrict__ ended, int row_tiles, int tiles, Tile* __restrict__ out) {
    constexpr int U = kTilePieces, V = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, warps = gridDim.x * (kTileThreads / 32);
    pdl_wait();
    pdl_launch_dependents();  // (only now: the merge reads the scores before its own wait)
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

// A candidate, or the largest one of a tile: its score, its place in the group (which breaks ties) and its row.
struct Found {
    double score;
    unsigned at;
    int row;
};
__device__ __forceinline__ bool before(const Found& a, const Found& b) { return a.score > b.score || (a.score == b.score && a.at < b.at); }

// Order-preserving key of a score, its upper half: enough for a threshold.
__device__ __forceinline__ unsigned order_hi(double x) {
    const unsigned b = unsigned(__double2hiint(x == 0. ? 0. : x));
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

// The least score whose key's upper half is `key` or more; all scores for 0.
__device__ __forceinline__ double least_of(unsigned key) {
    if (key == 0) return __longlong_as_double(0xfff0000000000000ll);
    return key >> 31 ? __hiloint2double(int(key ^ 0x80000000u), 0) : __hiloint2double(int(~key), -1);
}

// Twice the error of a log sum: of a term 2^-22 (the exponential), ln 2 2^-20 (y above -32), 21 * 1.4e-8 (log2 e as f32); 12 roundings
// of a tile's sum; 2^-22 of its weight, at its exact distance from the row's largest, and 8 roundings in the row's.  In all below 2.7e-6.
constexpr double kNear = 6e-6;

// e^(x - top) for x <= top as f32: what the difference loses (up to 2^-20 where it counts, all of it in one direction in a row whose
// tiles are alike) and the rounding of its product with log2 e are made good.
__device__ __forceinline__ float exp_below(float x, float top) {
    const float d = fsub(x, top), back = fsub(d, x);
    const float lost = fsub(fsub(x, fsub(d, back)), fadd(top, back));  // x - top = d + lost
    const float t = fmaxf(d, -150.f), y = fmul(t, kLog2e), e = ex2(y);
    const float more = fmaf(t, kLog2e, -y) + (d > -150.f ? fmul(lost, kLog2e) : 0.f);
    return fmaf(fmul(e, more), 0.6931471805599453f, e);
}

// log of the sum of exponentials of a row, by a warp, from its tiles; NaN where the row has no candidates.
__device__ __forceinline__ double join_sums(const Tile* tiles, int n) {
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
    top = unorder(__reduce_max_sync(0xffffffffu, order(top)));
    float part = 0.f;  // (a tile of forbidden tokens has the sum 0)
#pragma unroll
    for (int u = 0; u < N; ++u) part = fmaf(t[u].y, exp_below(t[u].x, top), part);
    double sum = double(part);
    for (int i = lane + 32 * N; i < n; i += 32) {
        const float2 v = __ldcg(in + i);
        sum += double(v.y) * double(exp_below(v.x, top));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return top == -INFINITY ? __longlong_as_double(0x7ff8000000000000ll) : double(top) + log(sum);
}

struct MergeShared {
    unsigned group_top[128];
    unsigned threshold;
    int count, redo;
    Found found[kCap];
    Found best[kBeamMaxK + 1];
    double sums[kMergeThreads / 32];
};

// A threshold that at least k + 1 of the CTA's items reach, if there are so many, and not many more: the (k + 1)-th largest of the
// largest items of 32 (or 128) groups of threads, whose keys are made different by their groups' numbers in the lowest bits; and less
// by kNear, so that what the sums' errors could lift above the k-th best passes too.
// `top`: the key of the largest item of this thread, 0: none.
__device__ __forceinline__ double threshold_of(MergeShared& sh, int k, unsigned top) {
    const int tid = threadIdx.x, groups = k < 16 ? 32 : 128, of = blockDim.x / groups;
    for (int o = 1; o < of; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (tid % of == 0) sh.group_top[tid / of] = (top & ~127u) | unsigned(tid / of);
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (tid < groups) {
        const unsigned mine = sh.group_top[tid];
        const uint4* all = reinterpret_cast<const uint4*>(sh.group_top);
        int rank = 0;
#pragma unroll 8
        for (int g = 0; g < groups / 4; ++g) {
            const uint4 v = all[g];
            rank += (v.x > mine) + (v.y > mine) + (v.z > mine) + (v.w > mine);
        }
        if (rank == k) sh.threshold = mine & ~127u;
    }
    __syncthreads();
    return least_of(sh.threshold) - kNear;
}

__device__ __forceinline__ void push(MergeShared& sh, double score, unsigned at, int row) {
    const int i = atomicAdd(&sh.count, 1);
    if (i < kCap) sh.found[i] = Found{score, at, row};
}

// best[0 .. n - 1] = the n = min(k + 1, all) best of the items that have been pushed, in order; where they are too many, of all that
// each(f) calls f(score, place, row) for.  A warp ranks an item by counting, and calls close(row, other row) where an item among the k
// best and one of another row lie within kNear of each other.  Ends synchronised.
template <class Each, class Close>
__device__ __forceinline__ int rank_found(MergeShared& sh, int k, Each&& each, Close&& close) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
    __syncthreads();
    const int n = sh.count;
    if (n <= kCap) {
        for (int c = warp; c < n; c += warps) {
            const Found mine = sh.found[c];
            int rank = 0;
            bool near = false;
            for (int o = lane; o < n; o += 32) {
                const Found f = sh.found[o];
                rank += before(f, mine);
                near |= f.row != mine.row && fabs(f.score - mine.score) < kNear;
            }
            rank = __reduce_add_sync(0xffffffffu, rank);
            if (rank <= k && lane == 0) sh.best[rank] = mine;
            if (near && rank < k)
                for (int o = lane; o < n; o += 32)
                    if (fabs(sh.found[o].score - mine.score) < kNear) close(sh.found[o].row, mine.row);
        }
    } else {  // very many that reach the threshold: the best one behind the last, k + 1 times
        Found last{INFINITY, 0, 0};
        for (int i = 0; i <= k; ++i) {
            Found mine{-INFINITY, UINT_MAX, 0};
            each([&](double score, unsigned at, int row) {
                const Found f{score, at, row};
                if ((i == 0 || before(last, f)) && before(f, mine)) mine = f;
            });
#pragma unroll 1
            for (int o = 16; o > 0; o >>= 1) {
                const Found f{__shfl_xor_sync(0xffffffffu, mine.score, o), __shfl_xor_sync(0xffffffffu, mine.at, o),
                              __shfl_xor_sync(0xffffffffu, mine.row, o)};
                if (before(f, mine)) mine = f;
            }
            __syncthreads();
            if (lane == 0) sh.found[warp] = mine;
            __syncthreads();
            last = sh.found[0];
            for (int w = 1; w < warps; ++w)
                if (before(sh.found[w], last)) last = sh.found[w];
            if (tid == 0) sh.best[i] = last;
        }
        __syncthreads();
        for (int i = 0; i < min(n, k); ++i) {
            const Found kept = sh.best[i];
            each([&](double score, unsigned, int row) {
                if (row != kept.row && fabs(score - kept.score) < kNear) close(row, kept.row);
            });
        }
    }
    __syncthreads();
    return min(n, k + 1);
}

// A CTA per group; bound by the latency of its ten or so steps, one behind the other: 5.8 us for one group of 4 rows of 151936 bf16
// logits, 6.5 us for 64 (close candidates looked for in steps of their own: 6.4 and 7.2).  The k best tiles' ranking is a step of its
// own: opening every tile above a threshold instead took as long on ordinary groups and 377 us where few beams live and their tiles
// lie together.
template <class T>
__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(const T* __restrict__ logits, long long stride, int vocab, int beams,
                                                              const float* __restrict__ scores, const uint8_t* __restrict__ ended,
                                                              int end_id, int k, const Tile* __restrict__ tiles, int row_tiles,
                                                              unsigned row_magic, float* __restrict__ out_scores,
                                                              int* __restrict__ tokens, int* __restrict__ parents) {
    constexpr int U = kTilePieces, V = 16 / sizeof(T), kHeld = 2;  // tiles of a thread whose scores are formed once
    extern __shared__ double lse[];                                          // [beams]; NaN: no candidates of this row
    float* score = reinterpret_cast<float*>(lse + beams);                    // [beams]
    unsigned char* state = reinterpret_cast<unsigned char*>(score + beams);  // [beams] 1: the sum is formed again, 2: exactly known, 3: none
    __shared__ MergeShared sh;
    __shared__ Found tile_of[kBeamMaxK];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, threads = blockDim.x, warps = threads >> 5;
    const int group = blockIdx.x, r0 = group * beams;
    for (int b = tid; b < beams; b += threads) {
        const float sc = __ldcg(scores + r0 + b);  // (from L2: an older call's line may be nearer)
        const bool over = ended && __ldcg(ended + r0 + b);
        score[b] = sc;
        state[b] = fabsf(sc) <= kMaxF ? over ? 2 : 0 : 3;
    }
    if (tid == 0) sh.redo = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int n_tiles = beams * row_tiles;
    const Tile* mine = tiles + size_t(r0) * row_tiles;
    auto row_of = [&](int c) { return row_magic ? int(__umulhi(unsigned(c), row_magic)) : c / row_tiles; };
    float held_top[kHeld];
    int held_row[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int c = tid + u * threads;
        held_row[u] = row_of(c);
        held_top[u] = c < n_tiles ? __ldcg(&mine[c].top) : -INFINITY;
    }
    for (int b = warp; b < beams; b += warps) {
        const double l = state[b] ? __longlong_as_double(0x7ff8000000000000ll) : join_sums(mine + size_t(b) * row_tiles, row_tiles);
        if (lane == 0) lse[b] = l;
    }
    __syncthreads();
    // the score of a tile's largest logit; NaN: none
    auto value = [&](int row, float x) {
        return x == -INFINITY ? __longlong_as_double(0x7ff8000000000000ll) : double(score[row]) + (double(x) - lse[row]);
    };
    // Two beams' candidates that lie too close to each other, one of them kept: their sums are formed again.
    auto close = [&](int a, int b) {
        if (a == b) return;
        if (state[a] == 0) state[a] = 1, sh.redo = 1;
        if (state[b] == 0) state[b] = 1, sh.redo = 1;
    };
    auto settle = [&] {  // (behind rank_found's barrier)
        if (!sh.redo) return false;
        for (int b = 0; b < beams; ++b) {
            if (state[b] != 1) continue;
            const T* row = logits + (r0 + b) * stride;
            float top = -INFINITY;
            for (int i = 0; i < row_tiles; ++i) top = fmaxf(top, __ldcg(&mine[size_t(b) * row_tiles + i].top));
            double sum = 0;
            for (int t = tid; t < vocab; t += threads) sum += exp(double(to_float(row[t])) - double(top));
#pragma unroll 1
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sh.sums[warp] = sum;
            __syncthreads();
            if (tid == 0) {
                double t = 0;
                for (int w = 0; w < warps; ++w) t += sh.sums[w];
                lse[b] = double(top) + log(t);
                state[b] = 2;
            }
            __syncthreads();
        }
        if (tid == 0) sh.redo = 0;
        __syncthreads();
        return true;
    };
    // the best tiles, by their largest candidates; an ended beam counts as a tile of one candidate
    int n;
    bool again;
    do {
        double held[kHeld];
        unsigned top = 0;
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            held[u] = tid + u * threads < n_tiles ? value(held_row[u], held_top[u]) : __longlong_as_double(0x7ff8000000000000ll);
            if (held[u] == held[u]) top = max(top, order_hi(held[u]));
        }
        auto others = [&](auto&& f) {
            for (int c = tid + kHeld * threads; c < n_tiles; c += threads) {
                const int row = row_of(c);
                const double v = value(row, __ldcg(&mine[c].top));
                if (v == v) f(v, unsigned(c), row);
            }
            if (ended)
                for (int b = tid; b < beams; b += threads)
                    if (state[b] == 2 && lse[b] != lse[b]) f(double(score[b]), unsigned(b) * unsigned(row_tiles), b);
        };
        others([&](double v, unsigned, int) { top = max(top, order_hi(v)); });
        const double least = threshold_of(sh, k, top);
        auto all = [&](auto&& f) {
#pragma unroll
            for (int u = 0; u < kHeld; ++u)
                if (held[u] == held[u]) f(held[u], unsigned(tid + u * threads), held_row[u]);
            others(f);
        };
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (held[u] >= least) push(sh, held[u], unsigned(tid + u * threads), held_row[u]);
        others([&](double v, unsigned at, int row) {
            if (v >= least) push(sh, v, at, row);
        });
        n = rank_found(sh, k, all, close);
        again = settle();
    } while (again);
    // the candidates of the k best tiles that reach the last one's largest
    const int open = min(n, k);
    bool bounded = n >= k;
    const double floor = bounded ? sh.best[k - 1].score - kNear : 0.;
    for (int i = tid; i < open; i += threads) tile_of[i] = sh.best[i];
    __syncthreads();
    auto each_token = [&](auto&& f) {
        for (int c = tid; c < open * 32 * U; c += threads) {
            const Found& tile = tile_of[c / (32 * U)];
            const int b = tile.row, j = int(tile.at) - b * row_tiles;
            const double l = lse[b], sc = double(score[b]);
            if (l != l) {  // an ended beam
                if (c % (32 * U) == 0) f(sc, unsigned(b) * unsigned(vocab) + unsigned(end_id), b);
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
                if (v != -INFINITY) f(sc + (double(v) - l), unsigned(b) * unsigned(vocab) + unsigned(p * V - row.lead + i), b);
                x = next_of<T>(x);
            }
        }
    };
    for (;; bounded = false) {  // (when the sums have moved a little, so may the bound)
        if (bounded) {
            if (tid == 0) sh.count = 0;
            __syncthreads();
            each_token([&](double v, unsigned at, int row) {
                if (v >= floor) push(sh, v, at, row);
            });
        } else {
            unsigned top = 0;
            each_token([&](double v, unsigned, int) { top = max(top, order_hi(v)); });
            const double least = threshold_of(sh, k, top);
            each_token([&](double v, unsigned at, int row) {
                if (v >= least) push(sh, v, at, row);
            });
        }
        n = rank_found(sh, k, each_token, close);
        if (!settle()) break;
    }
    const int have = min(n, k);
    out_scores += size_t(group) * k;
    tokens += size_t(group) * k;
    parents += size_t(group) * k;
    for (int i = tid; i < have; i += threads) {
        const Found f = sh.best[i];
        out_scores[i] = float(f.score);
        parents[i] = f.row;
        tokens[i] = int(f.at - unsigned(f.row) * unsigned(vocab));
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
    cudaError_t e = launch_pdl(k_beam_tiles<T>, dim3(unsigned(ctas < most ? ctas : most)), dim3(kTileThreads), 0, st, true,
                               static_cast<const T*>(a.logits), a.stride, a.vocab, a.scores, a.ended, row_tiles, tiles, ws);
    if (e != cudaSuccess) return e;
    // c / row_tiles = umulhi(c, ceil(2^32 / row_tiles)) for both below 2^16, row_tiles > 1
    const bool small = (long long)a.beams * row_tiles + 2 * kMergeThreads < 65536 && row_tiles > 1;
    // threads for a tile or two each, as far as that leaves the SMs a CTA per group
    const int work = a.beams * row_tiles > 128 * a.k ? a.beams * row_tiles : 128 * a.k;
    const int threads = work > 1024 && a.groups <= 2 * 148 ? 1024 : work > 512 ? 512 : 256;
    return launch_pdl(k_beam_merge<T>, dim3(unsigned(a.groups)), dim3(unsigned(threads)), size_t(a.beams) * 13, st, true,
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
