// Attention over the paged 8-bit KV cache (kv_cache.h has the layout).
//
// Query i of a sequence's m queries sits at position p = len - m + i and sees the keys max(0, p - window + 1) .. p
// (window 0: all up to p).  With kc, vc the int8 codes and ks, vs the scales of key j's block of 16 tokens:
//     s_j = scale * ks_j * (q . kc_j);   out = sum_j softmax(s)_j * vs_j * vc_j;   lse = log sum_j exp(s_j)
// A query that sees no key gets out = 0 and lse = -inf.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "kv_cache.h"
#include "tcgen05.cuh"

namespace qb {

namespace {

__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// ---------------------------------------------------------------- few query rows per kv head (decode)
//
//   S^T [128 keys][3 digits x RM rows] = K tile [128][HD] . Q digits     int8 tensor cores, K codes as they lie in the cache
//   O^T [HD dims][pieces x RM rows]   += V tile [HD][128] . W pieces     bf16 tensor cores, W = exp(s - ref) vs
// A query row is split into three balanced base-256 digits, x = 65536 x2 + 256 x1 + x0 with |x| <= 127 * 65536: its rounding
// is 2^-24 of the row's largest value, and the int32 sums are exact.  A weight is the sum of three bf16 pieces (24 bits;
// two, 16 bits, where the result is a 16-bit type): bf16 has f32's range, so a weight keeps its relative precision however
// far it is below the largest, and V codes are exact in it.  (Weights in fixed point, on the int8 tensor cores like S, lost
// the small ones beside a much larger one.)  V codes become bf16 on their way through registers.
// The softmax reference `ref` of a row is the score of the last key that it sees in its first tile (so the largest weight is
// at least 1), raised only when a score passes it by 2^32: f32 and bf16 have the range, most tiles need no maximum over the
// CTA, and O stays in TMEM; every 16 tiles (float32: 4) it joins f32 registers, which bounds the accumulation error.
//
// The work of all (sequence, kv head) units, in order, is dealt evenly to the CTAs (`even`), whatever the lengths; a
// unit cut between CTAs leaves partial sums in the workspace and k_kv_join adds them up in CTA order.  Where the host's
// bound on the lengths keeps a unit short, every CTA takes one unit and nothing is joined.
//   softmax warps  thread = key: scores, weights; then thread = dim: O.  Up to 4 rows: 4 warps; else 8, half of the rows each, which
//                  also take the V codes (copied one tile ahead) to bf16
//   4 V warps      (up to 4 rows) that instead
//   last warp      loads K (cp.async; bulk copies of the pages' pieces measured about 0.15 us each, whatever their size) and
//                  the tile's page list two tiles ahead, and issues the MMAs
//
// Bound by: instructions and their latency.  The codes are read once, at HBM's rate a tile would take 0.35 us of an SM (HD 64),
// and the MMAs are short; but a tile's codes, scores and weights pass through about 3800 warp instructions (HD 128, 4 rows; a
// quarter of them turn V codes into bf16), issued at 43 to 60 % of the SM's rate.  Measured (HBM figures of the codes and scales):
//   192 sequences up to 8191, bf16, 4 rows of 128:  115 us, 3.1 TB/s (the V codes in 8 softmax warps: 123, in 4: 141)
//   1 sequence of 131071, f16, 7 rows of 64:         25.3 us with the join
//   256 sequences of 640, f32, 7 rows of 64:         32.8 us (V warps beside 4 softmax warps of 8 rows, which spill: 47)
//   1 sequence of 130, f32:                         10.2 us, start (4 us), two tiles and the outputs one after the other
constexpr int kTileKeys = 128;
constexpr float kDigitMax = 8323072.0f;  // 127 * 256^2: three digits
constexpr float kLog2e = 1.4426950408889634f;
// Tiles whose O stays in TMEM before registers take it over: the tensor cores add with their sums cut off, not rounded, a bias of
// about 2^-26 for each of a tile's 8 steps.  (float32, 5 tiles: 5.5e-7 of the result; 16 tiles pass what 16-bit results show.)
template <class T> constexpr int kFlush = sizeof(T) == 4 ? 4 : 16;
constexpr float kShift = 32.f;           // log2: weights are exp(s - ref) 2^kShift, so that none that f32 can hold is flushed
constexpr float kRaise = 32.f;           // log2: how far a score may pass the reference

template <int HD, int RM, class T>
struct Dec {
    static constexpr int NP = sizeof(T) == 4 ? 3 : 2;                  // pieces of a weight
    static constexpr int NC = (3 * RM + 15) / 16 * 16;                 // columns of S
    static constexpr int WC = (NP * RM + 15) / 16 * 16;                // columns of O
    static constexpr bool v_warps = RM == 4;
    static constexpr int soft = v_warps ? 128 : 256;                   // threads of the softmax warps
    static constexpr int v_threads = v_warps ? 128 : soft;             // threads that take V codes to bf16
    static constexpr int threads = soft + (v_warps ? v_threads : 0) + 32;
    static constexpr int stages = 3;                                   // K tiles
    static constexpr int ctas = HD == 64 && RM <= 8 ? 3 : 2;           // per SM: shared memory, registers
    static constexpr int k_bytes = kTileKeys * HD;
    static constexpr int v_half = HD * 128;                            // bf16: two halves of 64 keys, [HD rows][128 bytes] swizzled
    static constexpr int w_half = WC * 128;                            // the same of the weights, [WC rows][128 bytes]
    static constexpr int q_bytes = (HD * NC + 1023) / 1024 * 1024;     // [NC rows][HD bytes] swizzled, as K's rows
    static constexpr int smem = stages * k_bytes + k_bytes + 2 * v_half + q_bytes + 2 * w_half + 1024;
    static constexpr int s_cols = NC <= 16 ? 16 : NC <= 32 ? 32 : 64;  // TMEM column pitch of an S buffer
    static constexpr int tmem_need = 2 * s_cols + WC;
    static constexpr int tmem_cols = tmem_need <= 64 ? 64 : tmem_need <= 128 ? 128 : 256;
    static constexpr int items = HD * 8 / v_threads;                   // V pieces (a dim's 16 tokens) of a thread
    static constexpr uint32_t idesc_s = (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(NC >> 3) << 17) | (uint32_t(kTileKeys >> 4) << 24);
    static constexpr uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(WC >> 3) << 17) | (uint32_t(HD >> 4) << 24);
    static_assert(tmem_need <= 256, "TMEM allocation");
};

struct DecPlan {
    int even;       // 1: tiles dealt evenly over the CTAs, 0: one unit per CTA
    int4* info;     // [CTAs] of the cut unit that a CTA begins: its last CTA, first token, queries, kv head; x = -1: none
    float* ml;      // [2 CTAs][RM][2] maximum (log2 units) and sum of a partial
    float* o;       // [2 CTAs][RM][HD]
};

// A call's sequence j: its rows and the keys that they see together.
struct SeqWork {
    // keys [lo, len), in tiles of 128 from lo & ~127; tiles >= 1 where m > 0.  A sequence that the call cannot have (reported)
    // has m = 0 like one without rows, and seq 0, so that its row of the page table may be read.
    int seq, t0, m, len, lo, tiles;
};

__device__ __forceinline__ SeqWork seq_work(const KvView& c, const KvAttnArgs& a, const KvCall& call, int j) {
    SeqWork w;
    const int t0 = __ldg(call.starts + j), t1 = __ldg(call.starts + j + 1), seq = __ldg(call.seqs + j);
    const bool known = seq >= 0 && seq < c.max_seqs;
    const int len = min(max(__ldg(c.lens + (known ? seq : 0)), 0), c.max_pages << c.pt_shift);
    w.t0 = t0;
    w.m = t0 < 0 ? 0 : max(min(t1, call.n_tok) - t0, 0);
    w.seq = known ? seq : 0;
    if (w.m > 0 && (!known || w.m > a.max_q)) {
        set_error(c.status, ERR_BAD_POS);
        w.m = 0;
    }
    w.len = w.m > 0 ? len : 0;
    w.lo = a.window ? max(0, w.len - w.m + 1 - a.window) : 0;
    w.tiles = w.m == 0 ? 0 : w.len > 0 ? (w.len - 1) / kTileKeys - w.lo / kTileKeys + 1 : 1;
    return w;
}
// The next sequence of the call, after j, that has tiles; j becomes its number.  (The last one's where there is none: tiles 0.)
__device__ __forceinline__ SeqWork next_work(const KvView& c, const KvAttnArgs& a, const KvCall& call, int& j) {
    SeqWork w;
    do {
        do ++j;  // without rows: passed by the starts alone
        while (j < call.n - 1 && __ldg(call.starts + j + 1) <= __ldg(call.starts + j));
        w = seq_work(c, a, call, j);
    } while (w.tiles == 0 && j < call.n - 1);
    return w;
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float ex2_full(float x) {  // results below 2^-126 too
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float warp_max_redux(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
// E consecutive elements; VEC: they lie aligned (E at most 16 bytes).
template <bool VEC, class T, int E>
__device__ __forceinline__ void load_row(const T* p, T (&x)[E]) {
    if constexpr (VEC) {
        struct alignas(E * sizeof(T)) V {
            T v[E];
        };
        const V w = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int z = 0; z < E; ++z) x[z] = w.v[z];
    } else {
#pragma unroll
        for (int z = 0; z < E; ++z) x[z] = p[z];
    }
}

// warp_wait in little code (it stands in a dozen places): a wait that gives up only sets the abort flag, which the kernel turns
// into its error bit when it ends.
__device__ __forceinline__ bool wait_warp(uint64_t* b, unsigned parity, volatile int* abort_flag) {
#pragma unroll 1
    for (unsigned i = 0; !__all_sync(0xffffffffu, mbar_try(b, parity)); ++i)
        if (__any_sync(0xffffffffu, *abort_flag != 0) || i == kWaitLimit) {
            *abort_flag = 1;
            return false;
        }
    return true;
}

// Barrier of the softmax threads; true for all of them if `bad` holds for one, so that they leave a loop together.
template <int THREADS>
__device__ __forceinline__ bool bar_any(bool bad) {
    unsigned r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(bad ? 1u : 0u), "n"(THREADS)
        : "memory");
    return r != 0;
}

// The value whose digits' dots are (d2, d1, d0).  |d2 * 256 + d1| < 2^30.
__device__ __forceinline__ float join_digits(int d2, int d1, int d0) { return fmaf(float(d2 * 256 + d1), 256.f, float(d0)); }

// 4 int8 codes -> 4 bf16, exactly: 128 + the low 7 bits, less 128 (or 256 for a negative code).
__device__ __forceinline__ uint2 codes_bf16(unsigned w) {
    const unsigned low = w & 0x7F7F7F7Fu, sign = w & 0x80808080u;
    const unsigned a0 = __byte_perm(low, 0x43434343u, 0x4140), b0 = __byte_perm(sign, 0x43434343u, 0x4140);
    const unsigned a1 = __byte_perm(low, 0x43434343u, 0x4342), b1 = __byte_perm(sign, 0x43434343u, 0x4342);
    const __nv_bfloat162 x = __hsub2(reinterpret_cast<const __nv_bfloat162&>(a0), reinterpret_cast<const __nv_bfloat162&>(b0));
    const __nv_bfloat162 y = __hsub2(reinterpret_cast<const __nv_bfloat162&>(a1), reinterpret_cast<const __nv_bfloat162&>(b1));
    return make_uint2(reinterpret_cast<const unsigned&>(x), reinterpret_cast<const unsigned&>(y));
}

// What the loading warp tells the others about a unit and about a tile.
struct UnitRec {
    int t0, m, len, lo, head;
    int first;  // this CTA has the unit's first tile
    int cut;    // and not all of them
    int owner;  // if cut: the CTA that has its last tile
};
struct TileRec {
    long long kt[8];  // of the tile's 8 blocks of 16 tokens: the K tile number (KvView::at), 0 where no key is seen
    int key0, unit, head_of_unit, tail_of_unit;
};

// The call's work is dealt in units of a tile's time: a unit's first tile counts 1 + kUnitCost (its queries, sums and outputs
// take about as long as kUnitCost tiles), the others 1.  CTA x has [x base + min(x, rem), ...) of it, and the tiles that start
// there.
constexpr int kUnitCost = 1;
struct Deal {
    int base, rem;
    __device__ __forceinline__ int begin(int x) const { return x * base + min(x, rem); }
    __device__ __forceinline__ int owner(int t) const {
        return t < rem * (base + 1) ? t / (base + 1) : rem + (t - rem * (base + 1)) / base;
    }
};
// Tiles of a unit that start in the first `part` of its cost.
__device__ __forceinline__ int tiles_before(int part, int tiles) { return part <= 0 ? 0 : min(tiles, max(1, part - kUnitCost)); }

template <int HD, int RM, class T>
__global__ void __launch_bounds__(Dec<HD, RM, T>::threads, Dec<HD, RM, T>::ctas) k_kv_decode(KvView c, KvAttnArgs a, KvCall call, DecPlan plan) {
    using C = Dec<HD, RM, T>;
    constexpr int NP = C::NP, last = C::threads / 32 - 1;  // the loading warp
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* vb = smem + C::stages * C::k_bytes;
    unsigned char* wb = vb + 2 * C::v_half;
    unsigned char* qd = wb + 2 * C::w_half;
    unsigned char* vc = qd + C::q_bytes;  // V codes of the next tile, each thread's pieces in its own places
    __shared__ uint64_t k_full[C::stages], listed[4], s_done[2], w_ready[2], o_done, q_ready, fin;
    __shared__ TileRec tile_rec[4];
    __shared__ __align__(16) float scales[4][16];  // of a tile's 8 blocks: K's, V's
    __shared__ UnitRec unit_rec[4];
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag, fresh[2];
    __shared__ __align__(16) float tile_max[4][RM];
    __shared__ __align__(16) float fac[2][RM], first_ref[2][RM], last_ref[RM], sum_part[4][RM];
    __shared__ int row_off[2][RM];  // a row's place in out and lse, from its unit's first
    __shared__ unsigned nan_rows[2];  // by unit: rows that see a V scale which is not finite
    __shared__ int2 scan_part[4];
    __shared__ int start_j, start_head, start_tile, start_at, tiles_from, tiles_to;
    const int tid = threadIdx.x, warp = warp_same(tid >> 5), lane = tid & 31;
    volatile int* ab = &abort_flag;

    if (tid == 0) {
        for (int s = 0; s < C::stages; ++s) mbar_init(&k_full[s], 32);
        for (int s = 0; s < 4; ++s) mbar_init(&listed[s], 32);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&s_done[b], 1);
            mbar_init(&w_ready[b], C::threads - 32);
        }
        mbar_init(&o_done, 1);
        mbar_init(&q_ready, 128);
        mbar_init(&fin, 1);
        abort_flag = 0;
        nan_rows[0] = nan_rows[1] = 0;
        tiles_from = tiles_to = 0;
        if (plan.even) plan.info[blockIdx.x] = make_int4(-1, 0, 0, 0);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == last) tmem_alloc(&tmem_base, C::tmem_cols);
    pdl_wait();
    pdl_launch_dependents();

    // ---- this CTA's tiles of the call's (even), or the tiles of unit blockIdx.x
    Deal deal = {0, 0};
    if (plan.even) {
        const int per = (call.n + 127) / 128, j0 = min(tid * per, call.n), j1 = warp < 4 ? min(j0 + per, call.n) : j0;
        int2 mine = make_int2(0, 0);  // cost and tiles of this thread's sequences
        SeqWork w = {};
#pragma unroll 1
        for (int j = j0; j < j1; ++j) {
            w = seq_work(c, a, call, j);
            if (w.tiles) mine.x += c.n_kv * (w.tiles + kUnitCost);
            mine.y += c.n_kv * w.tiles;
        }
        int2 inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc.x, o), y = __shfl_up_sync(0xffffffffu, inc.y, o);
            if (lane >= o) {
                inc.x += x;
                inc.y += y;
            }
        }
        if (warp < 4 && lane == 31) scan_part[warp] = inc;
        __syncthreads();
        int2 before = make_int2(inc.x - mine.x, inc.y - mine.y);
        int total = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (x < warp) {
                before.x += scan_part[x].x;
                before.y += scan_part[x].y;
            }
            total += scan_part[x].x;
        }
        // a part is never so small that no tile starts in it
        const int parts = max(1, min(int(gridDim.x), total / (kUnitCost + 1)));
        deal.base = total / parts;
        deal.rem = total - deal.base * parts;
        const int begin = deal.begin(blockIdx.x), end = deal.begin(blockIdx.x + 1);
        if (warp < 4 && int(blockIdx.x) < parts && begin < before.x + mine.x && end >= before.x) {  // a bound is in this thread's sequences
#pragma unroll 1
            for (int j = j0; j < j1; ++j) {
                if (j1 - j0 > 1) w = seq_work(c, a, call, j);
                if (w.tiles == 0) continue;
                const int cost = w.tiles + kUnitCost, all = cost * c.n_kv;
                if (begin >= before.x && begin < before.x + all) {
                    const int h = (begin - before.x) / cost, t = tiles_before(begin - before.x - h * cost, w.tiles);
                    start_j = j;  // t == tiles: the first tile is the next unit's
                    start_head = h;
                    start_tile = t;
                    start_at = before.x + h * cost;
                    tiles_from = before.y + h * w.tiles + t;
                }
                if (end > before.x && end <= before.x + all) {
                    const int h = min((end - before.x) / cost, c.n_kv - 1);
                    tiles_to = before.y + h * w.tiles + tiles_before(end - before.x - h * cost, w.tiles);
                }
                before.x += all;
                before.y += w.tiles * c.n_kv;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int first_j, first_head, first_tile = 0, first_at = 0, n_tiles;  // of the first tile
    SeqWork first_w = {};
    if (plan.even) {
        n_tiles = tiles_to - tiles_from;
        first_j = n_tiles > 0 ? start_j : 0;
        first_head = start_head;
        first_tile = start_tile;
        first_at = start_at;
        first_w = seq_work(c, a, call, first_j);
        if (n_tiles > 0 && first_tile == first_w.tiles) {  // this CTA's part begins after the start of that unit's last tile
            first_tile = 0;
            first_at += first_w.tiles + kUnitCost;
            if (++first_head == c.n_kv) {
                first_head = 0;
                first_w = next_work(c, a, call, first_j);
            }
        }
    } else {
        first_j = blockIdx.x / c.n_kv;
        first_head = blockIdx.x % c.n_kv;
        first_w = seq_work(c, a, call, first_j);
        n_tiles = first_w.tiles;
    }
    const uint32_t tmem = uint32_t(warp_same(int(tmem_base)));
    // V pieces of a thread: dim vd of blocks vblk + x * (v_threads / HD)
    const int v_tid = C::v_warps ? tid & 127 : tid, vd = v_tid % HD, vblk = v_tid / HD;
    const int v_shift = c.pt_shift + (HD == 64 ? 6 : 7);  // log2 of a tile's codes
    auto copy_v = [&](int i) {  // (any codes where no key is seen: their weights are 0)
        const uint32_t dst = smem_u32(vc) + v_tid * 16;
#pragma unroll
        for (int x = 0; x < C::items; ++x) {
            const int b = vblk + x * (C::v_threads / HD);
            const int8_t* src = c.codes + (size_t(tile_rec[i & 3].kt[b] + c.n_kv) << v_shift) +
                                (((b * kKvBlock) & (c.pt - 1)) * HD + vd * 16);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + x * C::v_threads * 16), "l"(src) : "memory");
        }
    };
    auto put_v = [&](int x, const uint4& v) {
        const int b = vblk + x * (C::v_threads / HD);
        const uint2 x0 = codes_bf16(v.x), x1 = codes_bf16(v.y), x2 = codes_bf16(v.z), x3 = codes_bf16(v.w);
        unsigned char* dst = vb + (b >> 2) * C::v_half;
        *reinterpret_cast<uint4*>(dst + sw_offset<128>(vd, 2 * (b & 3))) = make_uint4(x0.x, x0.y, x1.x, x1.y);
        *reinterpret_cast<uint4*>(dst + sw_offset<128>(vd, 2 * (b & 3) + 1)) = make_uint4(x2.x, x2.y, x3.x, x3.y);
    };
    const int n_my = warp_same(n_tiles);

    if (warp == last) {
        // ---- loads, two tiles ahead, and MMAs
        constexpr int kLead = C::stages - 1;
        SeqWork w = first_w;
        int j = first_j, head = first_head, tile = first_tile, at = first_at, end = 0, unit = -1;  // of the next tile to load
        int key0 = 0, entry = 0;  // its first key; lane b < 8: the table's entry for block b
        bool live = false;        // and whether a key of it is seen
        bool ok = true, new_unit = true;
        int s_next = 0, q_next = 0;  // next tile whose scores are to be issued, next unit whose queries are to be waited for
        auto look = [&](int left) {  // the page-table entries of the tile, read an iteration before they are used
            if (new_unit) end = min(w.tiles, tile + left);
            key0 = (w.lo / kTileKeys + tile) * kTileKeys;
            const int lo = max(w.lo, key0), hi = min(w.len, key0 + kTileKeys), b0 = key0 + lane * kKvBlock;
            live = lane < 8 && b0 < hi && b0 + kKvBlock > lo;
            // (not under a condition: the load would be waited for where it ends, instead of an iteration later)
            entry = __ldg(c.table + size_t(w.seq) * c.max_pages + (live ? b0 >> c.pt_shift : 0));
        };
        auto next_unit = [&]() {
            tile = 0;
            at += w.tiles + kUnitCost;
            if (++head == c.n_kv) {
                head = 0;
                w = next_work(c, a, call, j);
            }
        };
        if (n_my > 0) look(n_my);
#pragma unroll 1
        for (int it = 0; it < n_my + kLead && ok; ++it) {
            const int t = it - kLead;  // the tile to finish
#pragma unroll 1
            for (; t >= 0 && s_next <= min(t + 1, n_my - 1) && ok; ++s_next) {  // scores of this tile and of the next one
                if (warp_same(tile_rec[s_next & 3].head_of_unit)) {  // its query digits are in place
                    ok = wait_warp(&q_ready, q_next & 1, ab);
                    ++q_next;
                }
                ok = ok && wait_warp(&k_full[s_next % C::stages], (s_next / C::stages) & 1, ab);
                if (!ok) break;
                fence_async_smem();  // the copies were made by the generic proxy
                tc_fence_after();
                const uint32_t kt = sw_lo(uint32_t(warp_same(int(smem_u32(smem + (s_next % C::stages) * C::k_bytes)))));
                const uint32_t qt = sw_lo(uint32_t(warp_same(int(smem_u32(qd)))));
#pragma unroll
                for (int k = 0; k < HD / 32; ++k)
                    mma_i8_sw<sw_hi<HD>, sw_hi<HD>, C::idesc_s>(tmem + (s_next & 1) * C::s_cols, kt + 2 * k, qt + 2 * k, k > 0);
                mma_commit_elect(&s_done[s_next & 1]);
                __syncwarp();
            }
            if (it < n_my && ok) {  // K of tile `it` into stage it % stages (its last user was tile it - stages), its record into it % 4
                if (new_unit) {
                    ++unit;
                    if (lane == 0) {
                        UnitRec& u = unit_rec[unit & 3];
                        u.t0 = w.t0;
                        u.m = w.m;
                        u.len = w.len;
                        u.lo = w.lo;
                        u.head = head;
                        u.first = tile == 0;
                        u.cut = end - tile < w.tiles;
                        u.owner = u.cut ? deal.owner(at + w.tiles - 1 + (w.tiles > 1 ? kUnitCost : 0)) : 0;
                    }
                }
                const bool bad = live && (entry < 0 || entry >= c.n_pages);
                if (bad) set_error(c.status, ERR_BAD_POS);
                const long long kt = live ? (long long)c.at(bad ? 0 : entry, a.layer, 0, head) : 0;
                const unsigned blocks = __ballot_sync(0xffffffffu, live);
                TileRec& rec = tile_rec[it & 3];
                if (lane < 8) rec.kt[lane] = kt;
                if (lane == 0) {
                    rec.key0 = key0;
                    rec.unit = unit & 3;
                    rec.head_of_unit = new_unit;
                    rec.tail_of_unit = tile + 1 == end;
                }
                __syncwarp();
                mbar_arrive(&listed[it & 3]);
                const int s = it % C::stages;
                const uint32_t dst = smem_u32(smem + s * C::k_bytes);
                const int step = c.pt * 16;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {  // lane's keys kk * 32 + lane
                    const int key = kk * 32 + lane;
                    const long long tl = __shfl_sync(0xffffffffu, kt, key / kKvBlock);
                    const int8_t* src = c.codes + (size_t(tl) << (c.pt_shift + (HD == 64 ? 6 : 7))) + (key & (c.pt - 1)) * 16;
                    if (blocks >> (key / kKvBlock) & 1)
#pragma unroll
                        for (int g = 0; g < HD / 16; ++g)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + sw_offset<HD>(key, g)),
                                         "l"(src + g * step)
                                         : "memory");
                }
                {  // lanes 0-7: K's scales of the 8 blocks, lanes 8-15: V's
                    const int b = lane & 7;
                    const size_t tl = size_t(__shfl_sync(0xffffffffu, kt, b)) + (lane & 8 ? c.n_kv : 0);
                    if (lane < 16)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&scales[it & 3][lane])),
                                     "l"(c.scales + (tl << (c.pt_shift - 4)) + ((b * kKvBlock) & (c.pt - 1)) / kKvBlock)
                                     : "memory");
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&k_full[s])) : "memory");
                new_unit = ++tile == end;
                if (it + 1 < n_my) {
                    if (new_unit) next_unit();
                    look(n_my - it - 1);
                }
            }
            if (t < 0) continue;
            ok = ok && wait_warp(&w_ready[t & 1], (t >> 1) & 1, ab);
            if (!ok) break;
            tc_fence_after();
            {
                const uint32_t vt = sw_lo(uint32_t(warp_same(int(smem_u32(vb))))), wt = sw_lo(uint32_t(warp_same(int(smem_u32(wb)))));
                const bool keep = !warp_same(fresh[t & 1]);
#pragma unroll
                for (int k = 0; k < kTileKeys / 16; ++k)  // 4 steps of 32 bytes in each half
                    mma_f16_sw<sw_hi<128>, sw_hi<128>, C::idesc_o>(tmem + 2 * C::s_cols, vt + (k / 4) * (C::v_half >> 4) + 2 * (k % 4),
                                                                   wt + (k / 4) * (C::w_half >> 4) + 2 * (k % 4), keep || k > 0);
                mma_commit_elect(&o_done);
            }
            __syncwarp();
        }
        mma_commit_elect(&fin);
        for (unsigned i = 0; i < kWaitLimit && !__all_sync(0xffffffffu, mbar_try(&fin, 0)); ++i) {
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (C::v_warps && tid >= C::soft) {
        // ---- V codes to bf16
        bool ok = n_my == 0 || wait_warp(&listed[0], 0, ab);
        if (n_my > 0 && ok) copy_v(0);
#pragma unroll 1
        for (int i = 0; i < n_my && ok; ++i) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            uint4 v[C::items];
#pragma unroll
            for (int x = 0; x < C::items; ++x) v[x] = reinterpret_cast<const uint4*>(vc)[x * C::v_threads + v_tid];
            if (i + 1 < n_my) {
                ok = wait_warp(&listed[(i + 1) & 3], ((i + 1) >> 2) & 1, ab);
                if (!ok) break;
                copy_v(i + 1);
            }
            if (i > 0) ok = wait_warp(&o_done, (i - 1) & 1, ab);  // the product of the tile before has read vb
            if (!ok) break;
#pragma unroll
            for (int x = 0; x < C::items; ++x) put_v(x, v[x]);
            fence_async_smem();
            mbar_arrive(&w_ready[i & 1]);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ---- scores, softmax, outputs: thread = key of the tile, then dim of the head
        constexpr int lanes = HD == 64 ? 16 : 32;  // rows of O^T of a warp (M = 64 leaves the upper half of each quadrant unused)
        constexpr int RH = RM * 128 / C::soft;     // rows of a thread: r0 ..
        const int half = warp >> 2, quad = warp & 3, r0 = half * RH, kid = tid & 127;
        const int dim = quad * lanes + lane;
        const uint32_t my_tmem = tmem + (uint32_t(quad * 32) << 16) + r0;
        bool ok = true;   // a wait that gave up is acted on at the next barrier, by all threads together
        int in_tmem = 0;  // tiles whose sum lies in TMEM
        UnitRec u = {};
        int rows = 0, p0 = 0, units = 0;  // rows of the unit, position of its first query, units so far
        unsigned unset = 0;               // rows without a reference: they have seen no key
        float ref[RH], sum[RH], acc[RH], fq[RH];  // ref and fq are the same in all threads of a half
#pragma unroll 1
        for (int i = -1; i < n_my; ++i) {
            // the next tile begins a unit: its query digits, 128 / RM threads per row (loaded here, written below, as soon as
            // this tile's scores are done and qd is free)
            constexpr int per_row = 128 / RM, E = HD / per_row;
            const int qr = kid / per_row, d0 = kid % per_row * E;  // (threads 0-127)
            bool prep = false;
            int q_rows = 0;
            T x[E];
            if (i + 1 < n_my) {
                int nu_t0 = first_w.t0, nu_m = first_w.m, nu_head = first_head;  // the first unit's is known before it is listed
                prep = i < 0;
                if (i >= 0) {
                    ok = wait_warp(&listed[(i + 1) & 3], ((i + 1) >> 2) & 1, ab) && ok;
                    prep = tile_rec[(i + 1) & 3].head_of_unit;
                    const UnitRec& nu = unit_rec[tile_rec[(i + 1) & 3].unit];
                    nu_t0 = nu.t0;
                    nu_m = nu.m;
                    nu_head = nu.head;
                }
                if (prep) {
                    q_rows = nu_m * a.group;
                    // (rows past the unit's read its first: a load under a condition would be waited for right here)
                    const int row = qr < q_rows ? qr : 0;
                    const T* q = static_cast<const T*>(a.q) + (long long)(nu_t0 + row / a.group) * a.q_stride +
                                 (nu_head * a.group + row % a.group) * HD + d0;
                    load_row<false>(q, x);
                }
            }
            float s[RH], vs = 0.f;  // score less ref, log2
            if (i >= 0) {
                const TileRec& rec = tile_rec[i & 3];
                if (rec.head_of_unit) {
                    u = unit_rec[rec.unit];
                    rows = u.m * a.group;
                    p0 = u.len - u.m;
                    unset = (1u << rows) - 1;  // rows <= 16
                    const float* f = fac[units & 1];
                    ++units;
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        ref[r] = sum[r] = acc[r] = 0.f;
                        fq[r] = f[r0 + r];
                    }
                }
                ok = wait_warp(&k_full[i % C::stages], (i / C::stages) & 1, ab) && ok;
                const float ks = scales[i & 3][kid >> 4];
                vs = scales[i & 3][8 + (kid >> 4)];
                ok = wait_warp(&s_done[i & 1], (i >> 1) & 1, ab) && ok;
                tc_fence_after();
                int d2[RH], d1[RH], d0[RH];
                const uint32_t at = my_tmem + (i & 1) * C::s_cols;
                tmem_ld(at, d2);
                tmem_ld(at + RM, d1);
                tmem_ld(at + 2 * RM, d0);
                tmem_ld_wait();
                tmem_ready(d2);
                tmem_ready(d1);
                tmem_ready(d0);
                tc_fence_before();
#pragma unroll
                for (int r = 0; r < RH; ++r) s[r] = fmaf(join_digits(d2[r], d1[r], d0[r]), ks * fq[r], -ref[r]);  // (ref less kShift)
            }
            if (prep && half == 0) {
                struct alignas(E < 4 ? E : 4) Bytes {
                    unsigned char b[E];
                } digit[3];
                float amax = 0.f;
#pragma unroll
                for (int y = 0; y < E; ++y) amax = max_nan(amax, fabsf(to_f(x[y])));
#pragma unroll
                for (int o = per_row / 2; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const bool fine = amax < INFINITY;  // else the row's scores, and with them its result, are NaN
                // very small or large rows are brought near 1 first, exactly, so that the quotient is in range
                const float pre = amax < 0x1p-60f ? 0x1p64f : amax > 0x1p60f ? 0x1p-64f : 1.f;
                const float inv = fine && amax > 0.f ? __fdividef(kDigitMax, amax * pre) : 0.f;
#pragma unroll
                for (int y = 0; y < E; ++y) {
                    const int x3 = fine ? __float2int_rn(to_f(x[y]) * pre * inv) : 0;
                    const unsigned z = (unsigned(x3) + 0x808080u) ^ 0x808080u;
                    digit[0].b[y] = (unsigned char)(z >> 16);
                    digit[1].b[y] = (unsigned char)(z >> 8);
                    digit[2].b[y] = (unsigned char)z;
                }
#pragma unroll
                for (int z = 0; z < 3; ++z)
                    *reinterpret_cast<Bytes*>(qd + sw_offset<HD>(z * RM + qr, d0 / 16) + d0 % 16) = digit[z];
                if (tid < q_rows) row_off[units & 1][tid] = tid / a.group * a.n_heads + tid % a.group;
                if (tid % per_row == 0) fac[units & 1][qr] = fine ? (amax * a.scale) * (kLog2e / kDigitMax) : __int_as_float(0x7fffffff);
                fence_async_smem();
                mbar_arrive(&q_ready);
            }
            if (i < 0) {  // (else: fac and row_off are read after the barrier below)
                if (n_my > 0) ok = wait_warp(&listed[0], 0, ab) && ok;
                if (bar_any<C::soft>(!ok)) break;
            }
            if (i >= 0) {
                const TileRec& rec = tile_rec[i & 3];
                const int key0 = rec.key0, key = key0 + kid;
                const bool tail = rec.tail_of_unit;
                const bool seen = key >= u.lo && key < u.len;  // by some row
                // do all rows see the whole tile?
                const bool whole = key0 >= u.lo && key0 + kTileKeys <= u.len &&
                                   (u.m == 1 || (key0 + kTileKeys - 1 <= p0 && (!a.window || key0 > u.len - 1 - a.window)));
                // queries of this thread's first row; the next row is of the next query after g more
                const int qi0 = u.m == 1 ? 0 : r0 / a.group, g0 = u.m == 1 ? RM : a.group - r0 % a.group;
                if (!whole) {
                    int p = p0 + qi0, g = g0;
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        if (!seen || key > p || (a.window && key <= p - a.window)) s[r] = -INFINITY;
                        if (--g == 0) {
                            g = a.group;
                            ++p;
                        }
                    }
                }
                // a V scale that is not finite stays out of the products (a weight of 0 would be NaN), and is noted for the rows that see it
                if (!(fabsf(vs) < INFINITY)) {
                    vs = 0.f;
                    unsigned hit = 0;
#pragma unroll
                    for (int r = 0; r < RH; ++r) hit |= unsigned(s[r] != -INFINITY) << (r0 + r);
                    if (hit) atomicOr(&nan_rows[units & 1], hit);
                }
                bool high = in_tmem == kFlush<T>;
                const unsigned had = unset;
                if (had) {  // rows without a reference that see a key of this tile take the last one's score
                    unsigned can = 0;
                    int p = p0, g = u.m == 1 ? RM : a.group;
#pragma unroll 1
                    for (int r = 0; r < rows; ++r) {
                        const int last = min(p, key0 + kTileKeys - 1), lo = a.window ? max(p - a.window + 1, key0) : key0;
                        if (last >= lo) can |= 1u << r;
                        if (--g == 0) {
                            g = a.group;
                            ++p;
                        }
                    }
                    can &= had;
                    p = p0 + qi0;
                    g = g0;
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        if ((can >> (r0 + r) & 1) && key == min(p, key0 + kTileKeys - 1)) first_ref[i & 1][r0 + r] = s[r];
                        if (--g == 0) {
                            g = a.group;
                            ++p;
                        }
                    }
                    const bool stop = bar_any<C::soft>(!ok);
#pragma unroll
                    for (int r = 0; r < RH; ++r)
                        if (can >> (r0 + r) & 1) {
                            ref[r] = first_ref[i & 1][r0 + r] - kShift;
                            s[r] -= ref[r];
                        }
                    unset &= ~can;
                    if (stop) break;
                }
#pragma unroll
                for (int r = 0; r < RH; ++r) high = high || s[r] > kRaise + kShift;
                const bool any = bar_any<C::soft>(high || !ok);
                bool waited = false;  // for the product of the tile before, which reads vb and wb
                if (any) {
                    // O leaves TMEM, and the references that a score passed are raised to the tile's maxima
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        const float top = warp_max_redux(s[r]);
                        if (lane == 0) tile_max[quad][r0 + r] = top;
                    }
                    if (i > 0) ok = wait_warp(&o_done, (i - 1) & 1, ab) && ok;
                    tc_fence_after();
                    waited = true;
                    if (bar_any<C::soft>(!ok)) break;
                    if (in_tmem) {
                        int o0[RH], o1[RH], o2[RH];
                        const uint32_t at = my_tmem + 2 * C::s_cols;
                        tmem_ld(at, o0);
                        tmem_ld(at + RM, o1);
                        if constexpr (NP == 3) tmem_ld(at + 2 * RM, o2);
                        tmem_ld_wait();
                        tmem_ready(o0);
                        tmem_ready(o1);
                        if constexpr (NP == 3) tmem_ready(o2);
                        tc_fence_before();
#pragma unroll
                        for (int r = 0; r < RH; ++r) {
                            float o = __int_as_float(o1[r]);
                            if constexpr (NP == 3) o += __int_as_float(o2[r]);
                            acc[r] += o + __int_as_float(o0[r]);
                        }
                        in_tmem = 0;
                    }
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        const int x = r0 + r;
                        const float top = fmaxf(fmaxf(tile_max[0][x], tile_max[1][x]), fmaxf(tile_max[2][x], tile_max[3][x]));
                        if (top > kRaise + kShift) {
                            ref[r] += top - kShift;
                            s[r] -= top - kShift;
                            const float f = ex2(0.5f * (kShift - top));  // by halves: the factor may be below 2^-126
                            acc[r] = acc[r] * f * f;
                            sum[r] = sum[r] * f * f;
                        }
                    }
                }
                unsigned w[RH / 2][NP];  // pieces of rows 2 x, 2 x + 1 of the half
#pragma unroll
                for (int x = 0; x < RH / 2; ++x) {
                    float p[2];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float e = ex2(s[2 * x + y]);
                        sum[2 * x + y] += e;
                        p[y] = e * vs;
                    }
#pragma unroll
                    for (int z = 0; z < NP; ++z) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(p[0], p[1]);
                        w[x][z] = reinterpret_cast<const unsigned&>(h);
                        if (z + 1 < NP) {
                            p[0] -= __uint_as_float(w[x][z] << 16);
                            p[1] -= __uint_as_float(w[x][z] & 0xffff0000u);
                        }
                    }
                }
                if (!waited) {
                    if (i > 0) ok = wait_warp(&o_done, (i - 1) & 1, ab) && ok;
                    tc_fence_after();
                }
                unsigned char* wt = wb + (kid >> 6) * C::w_half + (kid & 7) * 2;
                const int wc = kid >> 3 & 7;  // 16-byte chunk of the rows of 64 keys
#pragma unroll
                for (int x = 0; x < RH / 2; ++x)
#pragma unroll
                    for (int z = 0; z < NP; ++z) {
                        const int row = z * RM + r0 + 2 * x;
                        *reinterpret_cast<unsigned short*>(wt + sw_offset<128>(row, wc)) = (unsigned short)w[x][z];
                        *reinterpret_cast<unsigned short*>(wt + sw_offset<128>(row + 1, wc)) = (unsigned short)(w[x][z] >> 16);
                    }
                if constexpr (!C::v_warps) {
                    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
                    for (int x = 0; x < C::items; ++x) put_v(x, reinterpret_cast<const uint4*>(vc)[x * C::v_threads + v_tid]);
                }
                if (tid == 0) fresh[i & 1] = in_tmem == 0;
                ++in_tmem;
                fence_async_smem();
                mbar_arrive(&w_ready[i & 1]);
                if (tail) {
                    // ---- the unit's sums over this CTA's keys
                    ok = wait_warp(&o_done, i & 1, ab) && ok;
                    tc_fence_after();
                    {
                        int o0[RH], o1[RH], o2[RH];
                        const uint32_t at = my_tmem + 2 * C::s_cols;
                        tmem_ld(at, o0);
                        tmem_ld(at + RM, o1);
                        if constexpr (NP == 3) tmem_ld(at + 2 * RM, o2);
                        // meanwhile the sums: at each step a lane keeps half of its rows
#pragma unroll
                        for (int h = RH / 2, o = 16; h >= 1; h >>= 1, o >>= 1)
#pragma unroll
                            for (int r = 0; r < h; ++r) {
                                const bool up = lane & o;
                                const float mine = up ? sum[r + h] : sum[r], other = up ? sum[r] : sum[r + h];
                                sum[r] = mine + __shfl_xor_sync(0xffffffffu, other, o);
                            }
#pragma unroll
                        for (int o = 16 / RH; o > 0; o >>= 1) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], o);
                        if (lane % (32 / RH) == 0) sum_part[quad][r0 + lane / (32 / RH)] = sum[0];
                        tmem_ld_wait();
                        tmem_ready(o0);
                        tmem_ready(o1);
                        if constexpr (NP == 3) tmem_ready(o2);
                        tc_fence_before();
                        in_tmem = 0;
#pragma unroll
                        for (int r = 0; r < RH; ++r) {
                            float o = __int_as_float(o1[r]);
                            if constexpr (NP == 3) o += __int_as_float(o2[r]);
                            acc[r] += o + __int_as_float(o0[r]);
                            if (kid == 0) last_ref[r0 + r] = ref[r];
                        }
                    }
                    if (bar_any<C::soft>(!ok)) break;
                    const int* off = row_off[(units - 1) & 1];
                    const size_t row0 = size_t(u.t0) * a.n_heads + u.head * a.group;
                    const size_t slot = size_t(2 * blockIdx.x + u.first) * RM;  // if cut
                    const int rr = lane % RM;  // lane r of a warp looks after row r
                    const float l = (sum_part[0][rr] + sum_part[1][rr]) + (sum_part[2][rr] + sum_part[3][rr]);
                    const bool none = (unset >> rr & 1) && l == 0.f;
                    const float inv = nan_rows[units & 1] >> rr & 1 ? __int_as_float(0x7fffffff)
                                      : u.cut ? 1.f : none ? 0.f : __fdividef(1.f, l);
                    if (tid < rows) {
                        if (u.cut) reinterpret_cast<float2*>(plan.ml)[slot + tid] = make_float2(none ? -INFINITY : last_ref[tid], l);
                        else if (a.lse) a.lse[row0 + off[tid]] = none ? -INFINITY : (last_ref[tid] + __log2f(l)) * (1.f / kLog2e);
                    }
                    auto put_rows = [&](auto* out, bool own_order) {
#pragma unroll
                        for (int r = 0; r < RH; ++r) {
                            const int x = r0 + r;
                            const float o = acc[r] * __shfl_sync(0xffffffffu, inv, x);
                            if (x < rows && lane < lanes) put(out + size_t(own_order ? x : off[x]) * HD + dim, o);
                        }
                    };
                    if (u.cut) put_rows(plan.o + slot * HD, true);
                    else put_rows(static_cast<T*>(a.out) + row0 * HD, false);
                    if (tid == 0 && u.first && u.cut)  // the unit's first CTA says which CTAs share it
                        plan.info[blockIdx.x] = make_int4(u.owner, u.t0, u.m, u.head);
                    if (bar_any<C::soft>(!ok)) break;  // last_ref and sum_part are read before the next unit writes them
                    if (tid == 0) nan_rows[units & 1] = 0;  // (for the unit after the next)
                }
            }
            if (!C::v_warps && i + 1 < n_my) copy_v(i + 1);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) set_error(c.status, ERR_WAIT_TIMEOUT);
    if (warp == last) {
        tc_fence_after();
        tmem_free(tmem, C::tmem_cols);
    }
}

// Joins the partial sums of the units that k_kv_decode cut, in CTA order.
// Few partials to a unit (MANY false): CTA x joins the rows of the unit that CTA x of `parts` began, a warp per row.
// Many: CTA (x, r) joins row r of the x-th unit that was cut, its threads spread over the partials.  Its time is that of its
// few loads, one after the other, so that they are as few as can be: the parts' records, then sums and values together.
// (2 units of 222 partials, 7 rows of 64: a CTA per began part and row, most of them without work, 21 us; the maxima, the sums
// and the values read one after the other, 11 us.)
constexpr int kJoinMany = 512, kJoinFew = 256;  // threads

template <int HD, int RM, class T, bool MANY>
__global__ void __launch_bounds__(MANY ? kJoinMany : kJoinFew) k_kv_join(KvAttnArgs a, DecPlan plan, int parts) {
    constexpr int warps = (MANY ? kJoinMany : kJoinFew) / 32, G = MANY ? kJoinMany / HD : 1, E = HD / 32;
    __shared__ float weight[MANY ? kJoinMany : 1], part[G][HD], red[2][warps];
    __shared__ int4 unit;
    __shared__ int unit_first;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    int first = blockIdx.x;
    int4 in;  // last CTA, first token, queries, kv head
    if constexpr (MANY) {  // parts <= kJoinMany
        in = tid < parts ? __ldcg(plan.info + tid) : make_int4(-1, 0, 0, 0);
        if (tid == 0) unit_first = -1;
        const unsigned mask = __ballot_sync(0xffffffffu, in.x >= 0);
        if (lane == 0) red[0][warp] = __int_as_float(__popc(mask));
        __syncthreads();
        const int k = lane < warp ? __float_as_int(red[0][lane]) : 0;
        const int before = __reduce_add_sync(0xffffffffu, k) + __popc(mask & ((1u << lane) - 1));
        if (in.x >= 0 && before == int(blockIdx.x)) {
            unit = in;
            unit_first = tid;
        }
        __syncthreads();
        first = unit_first;
        if (first < 0) return;
        in = unit;
    } else {
        in = __ldcg(plan.info + first);
        if (in.x < 0) return;
    }
    const int n = in.x - first + 1, rows = in.z * a.group;
    auto slot = [&](int x, int r) { return size_t(2 * (first + x) + (x == 0)) * RM + r; };
    auto row_of = [&](int r) { return size_t(in.y + r / a.group) * a.n_heads + in.w * a.group + r % a.group; };
    if constexpr (!MANY) {
        for (int r = warp; r < rows; r += warps) {
            float top = -INFINITY, l = 0.f, o[E] = {};
            for (int x0 = 0; x0 < n; x0 += 32) {  // a partial per lane
                const int k = min(n - x0, 32);
                const float2 ml = lane < k ? __ldcg(reinterpret_cast<const float2*>(plan.ml) + slot(x0 + lane, r))
                                           : make_float2(-INFINITY, 0.f);
                const float t = fmaxf(top, warp_max_redux(ml.x)), ref = t == -INFINITY ? 0.f : t;
                const float w = ex2_full(ml.x - ref), f = ex2_full(top - ref);
                top = t;
                l = l * f + warp_sum(ml.y * w);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll 4
                for (int x = 0; x < k; ++x) {
                    float v[E];
                    load_row<true>(plan.o + slot(x0 + x, r) * HD + lane * E, v);
                    const float wx = __shfl_sync(0xffffffffu, w, x);
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = fmaf(v[e], wx, o[e]);
                }
            }
            const bool none = top == -INFINITY && l == 0.f;
            T* out = static_cast<T*>(a.out) + row_of(r) * HD + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) put(out + e, none ? 0.f : o[e] / l);
            if (a.lse && lane == 0) a.lse[row_of(r)] = none ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
        }
    } else {
        const int d = tid % HD, g = tid / HD, r = blockIdx.y;
        if (r >= rows) return;
        constexpr int U = 32;  // values read along with the sums
        const float2 ml = tid < n ? __ldcg(reinterpret_cast<const float2*>(plan.ml) + slot(tid, r)) : make_float2(-INFINITY, 0.f);
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = __ldcg(plan.o + slot(min(g + u * G, n - 1), r) * HD + d);
        float top = warp_max_redux(ml.x);
        if (lane == 0) red[0][warp] = top;
        __syncthreads();
        top = warp_max_redux(lane < warps ? red[0][lane] : -INFINITY);
        const float w = ex2_full(ml.x - (top == -INFINITY ? 0.f : top));
        weight[tid] = w;
        float l = warp_sum(ml.y * w);
        if (lane == 0) red[1][warp] = l;
        __syncthreads();
        float o = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (g + u * G < n) o = fmaf(v[u], weight[g + u * G], o);
#pragma unroll 4
        for (int x = g + U * G; x < n; x += G) o = fmaf(__ldcg(plan.o + slot(x, r) * HD + d), weight[x], o);
        part[g][d] = o;
        __syncthreads();
        if (g == 0) {
#pragma unroll
            for (int q = 1; q < G; ++q) o += part[q][d];
            l = 0.f;
#pragma unroll
            for (int q = 0; q < warps; ++q) l += red[1][q];
            const bool none = top == -INFINITY && l == 0.f;
            put(static_cast<T*>(a.out) + row_of(r) * HD + d, none ? 0.f : o / l);
            if (a.lse && d == 0) a.lse[row_of(r)] = none ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
        }
    }
}

// ---------------------------------------------------------------- many query rows per kv head (chunks of a prompt, drafts)
//
// A CTA takes 128 WG query rows (token-major: row r is query r / group, head r % group of the kv head) and a stretch of keys,
// 64 at a time.  S = Q K^T and O += W V run on the 16-bit tensor cores; K and V codes become 16-bit numbers, exactly, once per
// tile for all rows.
// A query row is scaled by a power of two that brings its largest value to [1, 2), and is the sum of f16 pieces: two for float32
// (2^-23 of the row's largest value), one for 16-bit types (their 11 bits or fewer, to 2^-25 of the row's largest value).  A weight
// W = exp(s - ref) vs is a sum of bf16 pieces, which have f32's range:
//   float32 queries: three (24 bits).  The tensor cores' sums are cut off, not rounded (12 steps a tile: 1e-6 of the result after 8
//     tiles), so O moves every other tile to a total in shared memory.
//   16-bit queries: two (16 bits; 8 or 11 would cost as much again as the result's own rounding).
// (f16 weights for f16 queries lost small ones: those of keys behind one whose V is 0, and all weights where a block's V, even one
// that the row does not see, was 2^20 times the others'.)
//   warps 0 .. 4 WG - 1  softmax, thread = row: S from TMEM, weights back to TMEM (the A operand of the second product); the
//                        reference of a row is raised only when a score passes it by far (O is then scaled)
//   next 4 warps         codes and scales of the next tile on their way (cp.async into each thread's own places), this one's
//                        to 16-bit operands
//   last warp            issues the MMAs: S of tile i + 1 runs beside the softmax of tile i
//
// Bound by: the softmax's chain per tile (S out of TMEM, maximum, exp, pieces, weights into TMEM: about 3000 cycles for a CTA
// alone) and, with two CTAs to an SM, instructions: about 4200 warp instructions per 128 x 64 scores, half of the issue rate; the
// tensor cores are busy a quarter of the time at most.  Measured:
//   8 prompts of 2048, 32/8 heads of 128:  f16 607 us, bf16 609 us (453 and 451 TFLOP/s of what causal rows need)
//   6 sequences up to 8191 with 5 .. 509 queries, f16, 32/8 heads of 128, window 4096: 89 to 121 us with the sequences' order
//     (every row tile has the same number of stretches, whatever its keys)
//   1 prompt of 512, f32, 14/2 heads of 64: 18.4 to 19.1 us with the join, 112 CTAs of up to 4 tiles
template <int HD, class T, int WG>  // WG row groups of 128 (two of HD 128 and float32 pass TMEM)
struct Chunk {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int QP = F32 ? 2 : 1;               // pieces of a query
    static constexpr int NP = F32 ? 3 : 2;               // pieces of a weight
    static constexpr int flush = F32 ? 2 : 1 << 30;      // tiles whose O stays in TMEM
    static constexpr int rows = 128 * WG;
    static constexpr int threads = 128 * WG + 128 + 32;
    static constexpr int keys = 64;
    // operands in swizzled rows of 128 bytes: of a query piece and of K, HD / 64 slabs of 64 dims; of V, a row per dim
    static constexpr int q_bytes = 128 * HD * 2, kv_bytes = keys * HD * 2;
    static constexpr int total_at = WG * QP * q_bytes + 4 * kv_bytes + 2 * keys * HD;
    static constexpr int smem = total_at + (F32 ? WG * HD * 128 * 4 : 0);
    static constexpr int p_cols = NP * keys / 2;
    static constexpr int s_at = 0, p_at = 64 * WG, o_at = p_at + p_cols * WG;  // TMEM columns
    static constexpr int tmem_cols = o_at + HD * WG <= 256 ? 256 : 512;
    // per SM, with 1 KB static and 1 KB of the system's each.  (float32: two would leave a thread 96 registers, which it spills:
    // 31 us instead of 25 for 512 queries of 14 heads of 64 over 512 keys.)
    static constexpr int ctas = !F32 && smem <= 112 * 1024 && tmem_cols == 256 ? 2 : 1;
    static constexpr uint32_t idesc_s = (1u << 4) | (uint32_t(keys >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    static constexpr uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(HD >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    // log2.  Weights carry 2^shift; a row's reference follows its scores when one passes it by more than raise (every raise has
    // the warp's O pass through its registers: with 4 every other tile did, 1.3 times the time).
    static constexpr float shift = kShift, raise = 10.f;
    static_assert(o_at + HD * WG <= 512, "TMEM");
};

struct ChunkPlan {
    int splits;  // stretches of keys per row tile
    float* ml;   // [n_tok * n_heads][splits][2] maximum (log2) and sum, if splits > 1
    float* o;    // [n_tok * n_heads][splits][HD]
};

__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 4 int8 codes -> 4 f16, exactly: 1024 + (code + 128), less 1152.
__device__ __forceinline__ uint2 codes_f16(unsigned w) {
    w ^= 0x80808080u;
    const unsigned a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 x = __hsub2(reinterpret_cast<const __half2&>(a), off), y = __hsub2(reinterpret_cast<const __half2&>(b), off);
    return make_uint2(reinterpret_cast<const unsigned&>(x), reinterpret_cast<const unsigned&>(y));
}

template <int HD, class T, int WG>
__global__ void __launch_bounds__(Chunk<HD, T, WG>::threads, Chunk<HD, T, WG>::ctas) k_kv_chunk(KvView c, KvAttnArgs a, KvCall call, ChunkPlan plan) {
    using C = Chunk<HD, T, WG>;
    constexpr int QP = C::QP, NP = C::NP;
    constexpr bool F32 = C::F32;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* kb = smem + WG * QP * C::q_bytes;   // 2 buffers
    unsigned char* vb = kb + 2 * C::kv_bytes;          // 2 buffers
    unsigned char* codes = vb + 2 * C::kv_bytes;       // of the next tile: K's pieces, V's pieces, 16 bytes each, by thread
    // A wait on a phase's parity must come before the phase after it ends.  The softmax warps wait on scales_full, which comes
    // round every 4 tiles (converted at most 2 ahead of the weights), and not on k_full: K of tile i + 2 may be there as soon as
    // the scores of tile i are, however late a softmax warp is to look.
    __shared__ uint64_t q_full[WG], k_full[2], v_full[2], k_free[2], v_free[2], scales_full[4], s_full[WG], s_free[WG], p_full[WG], o_done[WG], fin;
    __shared__ __align__(16) float scales[4][8];       // of a tile's 4 blocks: K's, V's
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = warp_same(tid >> 5), lane = tid & 31;
    volatile int* ab = &abort_flag;

    // ---- this CTA's rows and keys
    const int split = blockIdx.x % plan.splits, r0 = int(blockIdx.x / plan.splits) * C::rows, head = blockIdx.y;
    const SeqWork w = seq_work(c, a, call, blockIdx.z);
    const int rows = w.m * a.group;
    if (r0 >= rows) return;
    const int p0 = w.len - w.m;  // position of the sequence's first query
    const int hi = p0 + (min(r0 + C::rows, rows) - 1) / a.group + 1;                    // keys [lo, hi) are seen by some row
    const int lo = a.window ? max(0, p0 + r0 / a.group - a.window + 1) : 0;
    const int all = hi > lo ? (hi - 1) / C::keys - lo / C::keys + 1 : 0;
    const int from = int((long long)all * split / plan.splits), nt = warp_same(int((long long)all * (split + 1) / plan.splits) - from);
    const int key_base = (lo / C::keys + from) * C::keys;
    const int wgs = warp_same(min(WG, (rows - r0 + 127) / 128));  // row groups with rows

    if (tid == 0) {
        for (int g = 0; g < WG; ++g) {
            mbar_init(&q_full[g], 128);
            mbar_init(&s_full[g], 1);
            mbar_init(&s_free[g], 128);
            mbar_init(&p_full[g], 128);
            mbar_init(&o_done[g], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&k_full[b], 128);
            mbar_init(&v_full[b], 128);
            mbar_init(&k_free[b], 1);
            mbar_init(&v_free[b], 1);
        }
        for (int b = 0; b < 4; ++b) mbar_init(&scales_full[b], 4);
        mbar_init(&fin, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4 * WG + 4) tmem_alloc(&tmem_base, C::tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uint32_t(warp_same(int(tmem_base)));
    pdl_launch_dependents();

    if (warp == 4 * WG + 4) {
        // ---- MMAs
        bool ok = true;
        for (int g = 0; g < wgs && nt > 0; ++g) ok = ok && wait_warp(&q_full[g], 0, ab);
#pragma unroll 1
        for (int i = 0; i <= nt && ok && nt > 0; ++i) {
            if (i < nt) {
                ok = wait_warp(&k_full[i & 1], (i >> 1) & 1, ab);
#pragma unroll 1
                for (int g = 0; g < wgs && ok; ++g) {
                    if (i > 0) ok = wait_warp(&s_free[g], (i - 1) & 1, ab);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t qt = sw_lo(uint32_t(warp_same(int(smem_u32(smem + g * QP * C::q_bytes)))));
                    const uint32_t kt = sw_lo(uint32_t(warp_same(int(smem_u32(kb + (i & 1) * C::kv_bytes)))));
#pragma unroll
                    for (int z = 0; z < QP; ++z)
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k)  // 4 steps of 32 bytes in each slab
                            mma_f16_sw<sw_hi<128>, sw_hi<128>, C::idesc_s>(
                                tmem + C::s_at + g * 64, qt + ((z * C::q_bytes + (k / 4) * 128 * 128) >> 4) + 2 * (k % 4),
                                kt + ((k / 4) * C::keys * 128 >> 4) + 2 * (k % 4), z > 0 || k > 0);
                    mma_commit_elect(&s_full[g]);
                    if (g == wgs - 1) mma_commit_elect(&k_free[i & 1]);
                }
            }
            if (i > 0 && ok) {
                const int t = i - 1;
                ok = wait_warp(&v_full[t & 1], (t >> 1) & 1, ab);
#pragma unroll 1
                for (int g = 0; g < wgs && ok; ++g) {
                    ok = wait_warp(&p_full[g], t & 1, ab);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t vt = sw_lo(uint32_t(warp_same(int(smem_u32(vb + (t & 1) * C::kv_bytes)))));
#pragma unroll
                    for (int z = 0; z < NP; ++z)
#pragma unroll
                        for (int k = 0; k < C::keys / 16; ++k)
                            mma_f16_ts<sw_hi<128>, C::idesc_o>(tmem + C::o_at + g * HD,
                                                               tmem + C::p_at + g * C::p_cols + z * (C::keys / 2) + k * 8, vt + 2 * k,
                                                               t % C::flush > 0 || z > 0 || k > 0);
                    mma_commit_elect(&o_done[g]);
                    if (g == wgs - 1) mma_commit_elect(&v_free[t & 1]);
                }
            }
        }
        mma_commit_elect(&fin);
        for (unsigned i = 0; i < kWaitLimit && !__all_sync(0xffffffffu, mbar_try(&fin, 0)); ++i) {
        }
    } else if (warp >= 4 * WG) {
        // ---- codes to operands
        constexpr int pieces = HD / 32;  // of K and of V, each thread
        const int ct = tid - 128 * WG, k_shift = c.pt_shift + (HD == 64 ? 6 : 7);
        const uint32_t mine = smem_u32(codes) + ct * 16;
        // (loads are not made under a condition: they would be waited for where it ends)
        int entry = 0;             // lane b < 4 (and every 4th): the table's entry for block b of the next tile to copy
        bool seen = false;         // and whether a key of it is seen (what lies in the cache beyond may be anything)
        float ks = 0.f, vs = 0.f;  // the copied tile's scales, where seen
        bool scaled = false;
        auto look = [&](int i) {
            const int k = key_base + i * C::keys + (lane & 3) * kKvBlock;
            seen = i < nt && k < hi && k + kKvBlock > lo;
            entry = __ldg(c.table + size_t(w.seq) * c.max_pages + (seen ? k >> c.pt_shift : 0));
        };
        auto copy = [&](int i) {
            const int key0 = key_base + i * C::keys;
            const bool bad = seen && (entry < 0 || entry >= c.n_pages);
            if (bad) set_error(c.status, ERR_BAD_POS);
            const size_t kt = c.at(seen && !bad ? entry : 0, a.layer, 0, head);
            const int in_page = ((key0 + (lane & 3) * kKvBlock) & (c.pt - 1)) / kKvBlock;
            const float* sc = c.scales + (kt << (c.pt_shift - 4)) + in_page;
            ks = __ldg(sc);
            vs = __ldg(sc + (c.n_kv << (c.pt_shift - 4)));
            scaled = seen;
#pragma unroll
            for (int x = 0; x < pieces; ++x) {
                const int key = ct % 64, g = ct / 64 + 2 * x;  // K piece: 16 dims of a key
                const size_t tl = __shfl_sync(0xffffffffu, (long long)kt, key / kKvBlock);
                const int8_t* src = c.codes + (tl << k_shift) + (size_t(g) * c.pt + ((key0 + key) & (c.pt - 1))) * 16;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + x * 2048), "l"(src) : "memory");
            }
#pragma unroll
            for (int x = 0; x < pieces; ++x) {
                const int d = ct % HD, b = ct / HD + x * (128 / HD);  // V piece: 16 keys of a dim
                const size_t tl = __shfl_sync(0xffffffffu, (long long)kt, b) + c.n_kv;
                const int8_t* src = c.codes + (tl << k_shift) + (size_t((key0 + b * kKvBlock) & (c.pt - 1)) * HD + d * 16);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + (pieces + x) * 2048), "l"(src) : "memory");
            }
        };
        auto convert = [&](unsigned char* to, int row, int chunk, const uint4& v, bool bf16) {  // 16 codes -> 16-byte chunks `chunk`, + 1 of a row
            uint2 x[4];
            const unsigned w4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int z = 0; z < 4; ++z) x[z] = bf16 ? codes_bf16(w4[z]) : codes_f16(w4[z]);
            *reinterpret_cast<uint4*>(to + sw_offset<128>(row, chunk)) = make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
            *reinterpret_cast<uint4*>(to + sw_offset<128>(row, chunk + 1)) = make_uint4(x[2].x, x[2].y, x[3].x, x[3].y);
        };
        bool ok = true;
        if (nt > 0) {
            look(0);
            copy(0);
            look(1);
        }
#pragma unroll 1
        for (int i = 0; i < nt && ok; ++i) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            uint4 kc[pieces], vc[pieces];
#pragma unroll
            for (int x = 0; x < pieces; ++x) {
                kc[x] = reinterpret_cast<const uint4*>(codes)[x * 128 + ct];
                vc[x] = reinterpret_cast<const uint4*>(codes)[(pieces + x) * 128 + ct];
            }
            if (ct < 4) {
                scales[i & 3][ct] = scaled ? ks : 0.f;
                scales[i & 3][4 + ct] = scaled ? vs : 0.f;
                mbar_arrive(&scales_full[i & 3]);
            }
            if (i + 1 < nt) copy(i + 1);
            look(i + 2);
            if (i >= 2) ok = wait_warp(&k_free[i & 1], ((i >> 1) - 1) & 1, ab);
            unsigned char* kt = kb + (i & 1) * C::kv_bytes;
#pragma unroll
            for (int x = 0; x < pieces; ++x) {  // dims 16 g .. of key ct % 64
                const int g = ct / 64 + 2 * x;
                convert(kt + (g / 4) * C::keys * 128, ct % 64, 2 * (g % 4), kc[x], false);
            }
            fence_async_smem();
            mbar_arrive(&k_full[i & 1]);
            if (i >= 2) ok = ok && wait_warp(&v_free[i & 1], ((i >> 1) - 1) & 1, ab);
            unsigned char* vt = vb + (i & 1) * C::kv_bytes;
#pragma unroll
            for (int x = 0; x < pieces; ++x) convert(vt, ct % HD, 2 * (ct / HD + x * (128 / HD)), vc[x], true);
            fence_async_smem();
            mbar_arrive(&v_full[i & 1]);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp < 4 * wgs) {
        // ---- softmax: thread = row
        const int g = warp >> 2, rt = tid & 127, r = r0 + g * 128 + rt;
        const bool valid = r < rows, busy = r0 + g * 128 + (warp & 3) * 32 < rows;  // busy: the warp has rows
        const int qi = valid ? r / a.group : 0, qh = head * a.group + (valid ? r % a.group : 0), pos = p0 + qi;
        const uint32_t my = tmem + (uint32_t((warp & 3) * 32) << 16);
        float fac = fabsf(a.scale) * kLog2e;  // score = S * fac * ks, log2 (the queries carry the scale's sign)
        const float sign = copysignf(1.f, a.scale);
        if (nt > 0) {
            // the warp's 32 rows, one after the other (coalesced), 8 in flight; lane = HD / 32 dims
            constexpr int E = HD / 32;
            unsigned char* qt = smem + g * QP * C::q_bytes + (lane * E / 64) * 128 * 128;
            const T* q_mine = static_cast<const T*>(a.q) + (long long)(w.t0 + qi) * a.q_stride + (long long)qh * HD;  // this lane's row
            const bool vec = !((reinterpret_cast<uintptr_t>(a.q) | uintptr_t(a.q_stride * sizeof(T))) & (E * sizeof(T) - 1));
            auto rows_in = [&](auto aligned) {  // 8 at a time (rows past the end read some other row)
#pragma unroll 1
                for (int r8 = 0; r8 < 32; r8 += 8) {
                    T x[8][E];
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        load_row<decltype(aligned)::value>(
                            reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(q_mine), r8 + y)) + lane * E, x[y]);
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        float f[E], amax = 0.f;
#pragma unroll
                        for (int z = 0; z < E; ++z) {
                            f[z] = to_f(x[y][z]);
                            amax = fmaxf(amax, fabsf(f[z]));
                        }
                        // a power of two brings the row's largest value to [1, 2); 255: not finite, its scores are NaN
                        const int e = int(__float_as_uint(warp_max_redux(amax)) >> 23);
                        const int up = e == 255 ? 127 : min(max(254 - e, 1), 253);  // its biased exponent
                        const float pre = __uint_as_float(unsigned(up) << 23) * sign;
                        if (lane == r8 + y) fac *= e == 255 ? __int_as_float(0x7fffffff) : __uint_as_float(unsigned(254 - up) << 23);
#pragma unroll
                        for (int z = 0; z < E; ++z) f[z] *= pre;
                        const int row = (warp & 3) * 32 + r8 + y;
                        unsigned char* to = qt + sw_offset<128>(row, lane * E % 64 / 8) + lane * E % 8 * 2;
#pragma unroll
                        for (int z = 0; z < QP; ++z) {
                            unsigned o[E / 2];
#pragma unroll
                            for (int k = 0; k < E / 2; ++k) {
                                const __half2 h = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
                                o[k] = reinterpret_cast<const unsigned&>(h);
                                const float2 b = __half22float2(h);
                                f[2 * k] -= b.x;
                                f[2 * k + 1] -= b.y;
                            }
                            if constexpr (E == 2) *reinterpret_cast<unsigned*>(to + z * C::q_bytes) = o[0];
                            else *reinterpret_cast<uint2*>(to + z * C::q_bytes) = make_uint2(o[0], o[1]);
                        }
                    }
                }
            };
            if (vec) rows_in(std::true_type{});
            else rows_in(std::false_type{});
            fence_async_smem();
            mbar_arrive(&q_full[g]);
        }
        float* total = reinterpret_cast<float*>(smem + C::total_at) + g * HD * 128 + rt;  // (float32) [dim][row]
        float ref = -INFINITY, sum = 0.f;
        bool ok = true, sees_nan = false;
#pragma unroll 1
        for (int i = 0; i < nt && ok; ++i) {
            const int key0 = key_base + i * C::keys;
            ok = wait_warp(&scales_full[i & 3], (i >> 2) & 1, ab) && wait_warp(&s_full[g], i & 1, ab);
            if (!ok) break;
            tc_fence_after();
            const float4 ks = *reinterpret_cast<const float4*>(scales[i & 3]), vs = *reinterpret_cast<const float4*>(scales[i & 3] + 4);
            float vr[4] = {vs.x, vs.y, vs.z, vs.w};
            if (!(fabsf((vs.x + vs.y) + (vs.z + vs.w)) < INFINITY)) {
                // a V scale that is not finite stays out of the products (a weight of 0 would be NaN); rows that see it are NaN
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (!(fabsf(vr[b]) < INFINITY)) {
                        const int k = key0 + b * kKvBlock;
                        sees_nan = sees_nan || (k <= pos && (!a.window || k + kKvBlock - 1 > pos - a.window));
                        vr[b] = 0.f;
                    }
            }
            int s0[32], s1[32];
            tmem_ld(my + C::s_at + g * 64, s0);
            tmem_ld(my + C::s_at + g * 64 + 32, s1);
            tmem_ld_wait();
            tmem_ready(s0);
            tmem_ready(s1);
            tc_fence_before();
            mbar_arrive(&s_free[g]);
            float f[4] = {ks.x * fac, ks.y * fac, ks.z * fac, ks.w * fac};
            float s[64];  // scores less the factor f of their 16 keys
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                s[k] = __int_as_float(s0[k]);
                s[k + 32] = __int_as_float(s1[k]);
            }
            // do all of the warp's rows see the whole tile, and is no factor below 0 (none that an append makes), so that the
            // maximum may be taken before it?  (rows past the end do as they like)
            const bool whole = key0 + C::keys - 1 <= pos && (!a.window || key0 > pos - a.window) &&
                               fminf(fminf(ks.x, ks.y), fminf(ks.z, ks.w)) >= 0.f;
            if (!__all_sync(0xffffffffu, whole)) {
                const int last = pos - key0, first = a.window ? last - a.window + 1 : -1;
#pragma unroll
                for (int k = 0; k < 64; ++k) s[k] = k > last || k < first ? -INFINITY : s[k] * f[k / 16];
                f[0] = f[1] = f[2] = f[3] = 1.f;
            }
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float m = s[16 * b];
#pragma unroll
                for (int k = 1; k < 15; k += 2) m = fmaxf(fmaxf(m, s[16 * b + k]), s[16 * b + k + 1]);
                top = fmaxf(top, fmaxf(m, s[16 * b + 15]) * f[b]);
            }
            const bool up = top > ref + C::raise;
            const float now = up ? top : ref;
            float factor = up ? ex2(0.5f * (ref - now)) : 1.f;  // the square root of O's: that may be below 2^-126
            if (ref == -INFINITY) factor = 0.f;  // (an infinite score as the first reference)
            ref = now;
            sum = sum * factor * factor;
            if (i > 0) {  // the product of the last tile has read the weights and written O
                ok = wait_warp(&o_done[g], (i - 1) & 1, ab);
                if (!ok) break;
                tc_fence_after();
                const bool out = F32 && i % C::flush == 0;  // O moves to the total: the next product starts anew
                if ((out || __any_sync(0xffffffffu, up)) && busy) {
#pragma unroll 1
                    for (int x = 0; x < HD; x += 16) {
                        int o[16];
                        tmem_ld(my + C::o_at + g * HD + x, o);
                        tmem_ld_wait();
                        tmem_ready(o);
                        unsigned n[16];
                        float* tt = total + x * 128;
#pragma unroll
                        for (int z = 0; z < 16; ++z) {
                            float y = __int_as_float(o[z]);
                            if constexpr (F32) {
                                const float t = i > C::flush ? tt[z * 128] : 0.f;
                                if (out) y += t;
                                if (i > C::flush || out) tt[z * 128] = (out ? y : t) * factor * factor;
                            }
                            n[z] = __float_as_uint(y * factor * factor);
                        }
                        if (!out) tmem_st(my + C::o_at + g * HD + x, n);
                    }
                }
            }
            if (busy) {
                const float base = (ref == -INFINITY ? 0.f : ref) - C::shift;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float p[16];
                    const unsigned long long f2 = f2_pack(f[b], f[b]), base2 = f2_pack(-base, -base), vr2 = f2_pack(vr[b], vr[b]);
                    unsigned long long part[2] = {0, 0};  // two keys at a time
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float2 x = f2_unpack(f2_fma(f2_pack(s[16 * b + k], s[16 * b + k + 1]), f2, base2));
                        const unsigned long long e = f2_pack(ex2(x.x), ex2(x.y));
                        part[k / 2 & 1] = f2_add(part[k / 2 & 1], e);
                        const float2 y = f2_unpack(f2_mul(e, vr2));
                        p[k] = y.x;
                        p[k + 1] = y.y;
                    }
                    const float2 both = f2_unpack(f2_add(part[0], part[1]));
                    sum += both.x + both.y;
#pragma unroll
                    for (int z = 0; z < NP; ++z) {
                        unsigned o[8];
#pragma unroll
                        for (int y = 0; y < 8; ++y) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(p[2 * y], p[2 * y + 1]);
                            o[y] = reinterpret_cast<const unsigned&>(h);
                            if (z + 1 < NP) {
                                const float2 left = f2_unpack(f2_add(f2_pack(p[2 * y], p[2 * y + 1]),
                                                                     f2_pack(-__uint_as_float(o[y] << 16), -__uint_as_float(o[y] & 0xffff0000u))));
                                p[2 * y] = left.x;
                                p[2 * y + 1] = left.y;
                            }
                        }
                        tmem_st(my + C::p_at + g * C::p_cols + z * (C::keys / 2) + b * 8, o);
                    }
                }
                tmem_st_wait();
            }
            tc_fence_before();
            mbar_arrive(&p_full[g]);
        }
        // ---- results
        if (nt > 0) ok = ok && wait_warp(&o_done[g], (nt - 1) & 1, ab);
        tc_fence_after();
        const bool none = sum == 0.f && ref == -INFINITY;
        const size_t row = size_t(w.t0 + qi) * a.n_heads + qh;
        const bool direct = plan.splits == 1;
        const float factor = sees_nan ? __int_as_float(0x7fffffff) : direct ? none ? 0.f : 1.f / sum : 1.f;
        if (ok && busy) {
            // 32 rows x 32 dims at a time through shared memory (the queries are no longer read), so that rows leave whole
            float* turn = reinterpret_cast<float*>(smem + g * QP * C::q_bytes) + (warp & 3) * 1024;
            const unsigned write = __ballot_sync(0xffffffffu, valid && (direct || !none));
            const long long to_mine = direct ? (long long)row * HD : ((long long)row * plan.splits + split) * HD;
#pragma unroll 1
            for (int x = 0; x < HD; x += 32) {
                int o[32];
                if (nt > 0) {
                    tmem_ld(my + C::o_at + g * HD + x, o);
                    tmem_ld_wait();
                    tmem_ready(o);
                }
                if (F32 && nt > C::flush) {
#pragma unroll
                    for (int z = 0; z < 32; ++z) o[z] = __float_as_int(__int_as_float(o[z]) + total[(x + z) * 128]);
                }
#pragma unroll
                for (int z = 0; z < 32; ++z) turn[lane * 32 + (z ^ lane)] = none ? 0.f : __int_as_float(o[z]) * factor;
                __syncwarp();
                auto rows_out = [&](auto* out) {
#pragma unroll 1
                    for (int y8 = 0; y8 < 32; y8 += 8) {
                        float v[8];
                        long long to[8];
#pragma unroll
                        for (int y = 0; y < 8; ++y) {
                            v[y] = turn[(y8 + y) * 32 + (lane ^ (y8 + y))];
                            to[y] = __shfl_sync(0xffffffffu, to_mine, y8 + y);
                        }
#pragma unroll
                        for (int y = 0; y < 8; ++y)
                            if (write >> (y8 + y) & 1) put(out + to[y] + x + lane, v[y]);
                    }
                };
                if (!direct) rows_out(plan.o);
                else rows_out(static_cast<T*>(a.out));
                __syncwarp();
            }
            if (valid) {
                if (!direct)
                    reinterpret_cast<float2*>(plan.ml)[row * plan.splits + split] =
                        make_float2(none ? -INFINITY : ref - C::shift, sum);
                else if (a.lse)
                    a.lse[row] = none ? -INFINITY : (ref - C::shift + log2f(sum)) * (1.f / kLog2e);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) set_error(c.status, ERR_WAIT_TIMEOUT);
    if (warp == 4 * WG + 4) {
        tc_fence_after();
        tmem_free(tmem, C::tmem_cols);
    }
}

// Joins the stretches of k_kv_chunk: a warp per (token, head), in order.  Stretches without a key have sum 0 and no O.
// (476 tokens of 32 heads of 128, 2 stretches: 7.7 us, latency.)
template <int HD, class T>
__global__ void __launch_bounds__(256) k_kv_chunk_join(KvAttnArgs a, ChunkPlan plan, long long n_rows) {
    pdl_wait();
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= n_rows) return;
    constexpr int E = HD / 32;
    // a stretch per lane (splits <= 32)
    const float2 ml = lane < plan.splits ? __ldcg(reinterpret_cast<const float2*>(plan.ml) + row * plan.splits + lane)
                                         : make_float2(-INFINITY, 0.f);
    const unsigned live = __ballot_sync(0xffffffffu, !(ml.x == -INFINITY && ml.y == 0.f));
    const float top = warp_max_redux(ml.x), w = ex2_full(ml.x - (top == -INFINITY ? 0.f : top)), l = warp_sum(ml.y * w);
    const float* src = plan.o + row * plan.splits * HD + lane * E;
    float o[E] = {};
#pragma unroll 2
    for (int x = 0; x < plan.splits; ++x) {
        float v[E];
        load_row<true>(src + x * HD, v);
        const float wx = __shfl_sync(0xffffffffu, w, x);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = live >> x & 1 ? fmaf(v[e], wx, o[e]) : o[e];
    }
    const bool none = top == -INFINITY && l == 0.f;
    const float inv = none ? 0.f : 1.f / l;
    struct alignas(E * sizeof(T)) Out {
        T v[E];
    } out;
#pragma unroll
    for (int e = 0; e < E; ++e) put(&out.v[e], none ? 0.f : o[e] * inv);
    *reinterpret_cast<Out*>(static_cast<T*>(a.out) + row * HD + lane * E) = out;
    if (a.lse && lane == 0) a.lse[row] = none ? -INFINITY : (top + log2f(l)) * (1.f / kLog2e);
}

// ---------------------------------------------------------------- host side

constexpr int kDecRows = 16;  // most query rows (queries x heads of a kv head) of k_kv_decode

// (256 x 640 f32, 14 rows of 64: 46 us against k_kv_chunk's 103; 64 x 4000 bf16, 16 rows of 128: 200 against 336.)
bool takes_decode(const KvAttnArgs& a) { return (long long)a.max_q * a.group <= kDecRows; }

int dec_rm(const KvAttnArgs& a) {
    const int rows = a.max_q * a.group;
    return rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
}

struct DecLaunch {
    int even, grid;
    size_t units;
};

DecLaunch dec_launch(const KvView& c, const KvAttnArgs& a, const KvCall& call) {
    DecLaunch l;
    l.units = size_t(call.n) * c.n_kv;
    // a unit's tiles, at most: never more with a window (which may begin and end within a tile) than without
    const auto tiles_of = [](long long keys) { return std::max(1LL, (keys + kTileKeys - 1) / kTileKeys); };
    const long long tiles = std::min(tiles_of(a.max_len), a.window ? tiles_of((long long)a.window + a.max_q) + 1 : LLONG_MAX);
    const int ctas = c.hd == 64 && dec_rm(a) <= 8 ? 3 : 2;  // per SM, as the kernel's
    // Units of up to 8 tiles are not dealt: cutting them costs more than an uneven last wave (32 x 2 units of 640 keys: 19.3 us, dealt
    // 21.5; 256 x 2: 34.9, dealt 39.9; of 1100 keys 25.4 either way; of 1500 dealt 25.6, a CTA each 29.7; of 2000 27.6, 36.8).
    l.even = tiles > 8;
    l.grid = int(l.even ? std::min<long long>(148 * ctas, std::max<long long>(1, (long long)l.units * tiles / 2)) : (long long)l.units);
    return l;
}

template <int HD, int RM, class T>
cudaError_t decode_t(const KvView& c, const KvAttnArgs& a, const KvCall& call, void* ws, cudaStream_t st) {
    using C = Dec<HD, RM, T>;
    const DecLaunch l = dec_launch(c, a, call);
    DecPlan p{};
    p.even = l.even;
    if (l.even) {
        p.o = static_cast<float*>(ws);
        p.ml = p.o + size_t(l.grid) * 2 * RM * HD;
        p.info = reinterpret_cast<int4*>(p.ml + size_t(l.grid) * 2 * RM * 2);
    }
    static_assert(C::smem > 48 * 1024, "launch_pdl raises the limit");
    cudaError_t e = launch_pdl(k_kv_decode<HD, RM, T>, dim3(unsigned(l.grid)), dim3(C::threads), C::smem, st, false, c, a, call, p);
    if (e != cudaSuccess || !l.even) return e;
    // more than 32 partials to a unit: a CTA per row, else a warp
    static_assert(148 * C::ctas <= kJoinMany, "a record per thread");
    if (size_t(l.grid) > l.units * 32)
        return launch_pdl(k_kv_join<HD, RM, T, true>, dim3(unsigned(l.units), unsigned(a.max_q * a.group)), dim3(kJoinMany), 0,
                          st, true, a, p, int(l.grid));
    return launch_pdl(k_kv_join<HD, RM, T, false>, dim3(unsigned(l.grid)), dim3(kJoinFew), 0, st, true, a, p, int(l.grid));
}

struct ChunkLaunch {
    int wg, splits;
};

// Row groups of 128 per CTA and stretches of keys per row tile.  Two groups share the conversion of K and V, but leave half as
// many CTAs: taken where those fill the SMs (8 prompts of 2048, f16, 8 kv heads of 128: 607 us, one group 674; 16 of 512, f32,
// 2 of 64: 88, 117; a single one, f32: 23.5 with one group, 27.6 with two).  Stretches: as many as fill the SMs twice, of at least
// 4 key tiles (a prompt of 512, 2 kv heads of 64: f32 23.5 us, of at least 8 tiles 27.4; f16 23.6, 24.6).
ChunkLaunch chunk_launch(const KvView& c, const KvAttnArgs& a, const KvCall& call) {
    ChunkLaunch l;
    const long long rows = (long long)call.n_tok * a.group;
    auto units = [&](int wg) { return c.n_kv * ((rows + 128 * wg - 1) / (128 * wg) + call.n - 1); };  // a part-filled tile per sequence
    const long long span = a.window && a.window < a.max_len ? std::min<long long>(a.max_len, (long long)a.window + a.max_q) : a.max_len;
    l.wg = (a.type == KV_F32 && c.hd == 128) || units(2) < 148 ? 1 : 2;
    const long long u = units(l.wg);
    l.splits = int(std::max<long long>(1, std::min<long long>({(span / 64 + 3) / 4, (2 * 148 + u - 1) / u, 32})));
    return l;
}

template <int HD, class T, int WG>
cudaError_t chunk_w(const KvView& c, const KvAttnArgs& a, const KvCall& call, int splits, void* ws, cudaStream_t st) {
    using C = Chunk<HD, T, WG>;
    ChunkPlan p{};
    p.splits = splits;
    const long long n_rows = (long long)call.n_tok * a.n_heads;
    if (p.splits > 1) {
        p.o = static_cast<float*>(ws);
        p.ml = p.o + n_rows * p.splits * HD;
    }
    const long long tiles = ((long long)std::min(a.max_q, call.n_tok) * a.group + C::rows - 1) / C::rows;
    cudaError_t e = launch_pdl(k_kv_chunk<HD, T, WG>, dim3(unsigned(tiles * p.splits), unsigned(c.n_kv), unsigned(call.n)), dim3(C::threads),
                               C::smem, st, false, c, a, call, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_pdl(k_kv_chunk_join<HD, T>, dim3(unsigned((n_rows + 7) / 8)), dim3(256), 0, st, true, a, p, n_rows);
}

template <int HD, class T>
cudaError_t attn_t(const KvView& c, const KvAttnArgs& a, const KvCall& call, void* ws, cudaStream_t st) {
    if (takes_decode(a)) {
        const int rm = dec_rm(a);
        return rm == 4 ? decode_t<HD, 4, T>(c, a, call, ws, st) : rm == 8 ? decode_t<HD, 8, T>(c, a, call, ws, st)
                                                                        : decode_t<HD, 16, T>(c, a, call, ws, st);
    }
    const ChunkLaunch l = chunk_launch(c, a, call);
    if constexpr (sizeof(T) == 2 || HD == 64)
        if (l.wg == 2) return chunk_w<HD, T, 2>(c, a, call, l.splits, ws, st);
    return chunk_w<HD, T, 1>(c, a, call, l.splits, ws, st);
}

template <class T>
cudaError_t attn_hd(const KvView& c, const KvAttnArgs& a, const KvCall& call, void* ws, cudaStream_t st) {
    return c.hd == 64 ? attn_t<64, T>(c, a, call, ws, st) : attn_t<128, T>(c, a, call, ws, st);
}

}  // namespace

size_t kv_attn_ws_bytes(const KvView& c, const KvAttnArgs& a, const KvCall& call) {
    if (!takes_decode(a)) {
        const int splits = chunk_launch(c, a, call).splits;
        return splits > 1 ? size_t(call.n_tok) * a.n_heads * splits * (c.hd + 2) * 4 : 0;
    }
    const DecLaunch l = dec_launch(c, a, call);
    return l.even ? size_t(l.grid) * (2 * dec_rm(a) * (c.hd + 2) * 4 + sizeof(int4)) : 0;
}

cudaError_t launch_kv_attention(const KvView& c, const KvAttnArgs& a, const KvCall& call, void* ws, cudaStream_t st) {
    if (call.n == 0 || call.n_tok == 0) return cudaSuccess;
    return a.type == KV_F32 ? attn_hd<float>(c, a, call, ws, st)
         : a.type == KV_F16 ? attn_hd<__half>(c, a, call, ws, st) : attn_hd<__nv_bfloat16>(c, a, call, ws, st);
}

}  // namespace qb
