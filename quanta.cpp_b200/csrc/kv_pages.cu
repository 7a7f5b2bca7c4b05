// The paged 8-bit KV cache: appending tokens, reading values back, and the page operations (kv_cache.h has the layout).
//
// Rounding of an append, for each block of 16 tokens that it touches, K or V, head (f32, round to nearest):
//     a = max |x| over the new tokens of the block and the head's dims;  old = the block's scale if the block holds
//     earlier tokens, else 0;  d = max(old, a * RN(1 / 127))
//     earlier codes c <- rint(c * (old / d));  new codes = rint(x * (1 / d)) in [-127, 127]
// A scale only grows, so a block's codes are rounded again at most when a larger value arrives, and appending the same
// tokens again changes nothing.  A non-finite input makes d non-finite; the codes are then 0 and the block reads as NaN.
// (d so small that 1 / d is infinite, below 2^-128: the codes are 0.)  Positions of the block past the sequence's end get 0.
#include <cuda_bf16.h>
#include <climits>

#include "kv_cache.h"

namespace qb {

namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The page of position pos of sequence seq, or -1 (and an error bit) where the table has none.
__device__ __forceinline__ int kv_page(const KvView& c, int seq, int pos) {
    const int k = pos >> c.pt_shift;
    const int p = pos >= 0 && k < c.max_pages ? __ldg(c.table + size_t(seq) * c.max_pages + k) : -1;
    if (p < 0 || p >= c.n_pages) {
        set_error(c.status, ERR_BAD_POS);
        return -1;
    }
    return p;
}

// ---------------------------------------------------------------- append

// A warp takes one (block of 16 tokens, K or V, head) after another.  A lane holds 8 dims of HD / 16 tokens that follow one
// another, so that the new values are read once, in whole rows, and a lane's codes already make 8 bytes of a token's dims (K)
// or 4 or 8 of a dim's tokens (V); through shared memory (rows padded by 16 bytes) they leave as the layout's 16-byte pieces.
// VEC: a lane's dims are read in 16-byte loads (aligned rows).
// 32 prompts of up to 4093 bf16 tokens, 8 heads of 128: 48 us, 4.4 TB/s (a byte at a time through shared memory: 250 us; 3 CTAs
// per SM instead of 4: 66 us; a task per warp: 77 us, the look-up of the page takes as long as the task).
constexpr int kAppendWarps = 4;

// |x| of 8 values, the largest (a NaN if one is), as f32
__device__ __forceinline__ float amax8(const float (&a)[8], float m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(a[i]));
    return m;
}
__device__ __forceinline__ __half2 amax8(const __half (&a)[8], __half2 m) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = __hmax2_nan(m, __habs2(__halves2half2(a[i], a[i + 1])));
    return m;
}
__device__ __forceinline__ __nv_bfloat162 amax8(const __nv_bfloat16 (&a)[8], __nv_bfloat162 m) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = __hmax2_nan(m, __habs2(__halves2bfloat162(a[i], a[i + 1])));
    return m;
}
__device__ __forceinline__ float amax_of(float m) { return m; }
__device__ __forceinline__ float amax_of(__half2 m) { return max_nan(__low2float(m), __high2float(m)); }
__device__ __forceinline__ float amax_of(__nv_bfloat162 m) { return max_nan(__low2float(m), __high2float(m)); }
template <class T> struct AmaxType { using t = float; };
template <> struct AmaxType<__half> { using t = __half2; };
template <> struct AmaxType<__nv_bfloat16> { using t = __nv_bfloat162; };

template <class T, int HD, bool VEC>
__global__ void __launch_bounds__(32 * kAppendWarps, 4) k_kv_append(KvView c, int layer, const T* __restrict__ k,
                                                                 const T* __restrict__ v, long long k_stride,
                                                                 long long v_stride, KvCall call, int max_new, int group) {
    constexpr int TPL = HD / 16, LPR = HD / 8;  // tokens of a lane, lanes of a row
    struct alignas(16) Row {
        T a[8];
    };
    __shared__ __align__(16) unsigned char tiles[kAppendWarps][HD * 18];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int j = blockIdx.y;
    const int t0 = __ldg(call.starts + j), m = min(__ldg(call.starts + j + 1), call.n_tok) - t0, seq = __ldg(call.seqs + j);
    if (m <= 0 || t0 < 0) return;
    if (seq < 0 || seq >= c.max_seqs) {
        set_error(c.status, ERR_BAD_POS);
        return;
    }
    const int p1 = __ldg(c.lens + seq), p0 = p1 - m;  // the new tokens' positions [p0, p1)
    if (p0 < 0 || m > max_new) {  // more tokens than the sequence has positions, or than the grid covers
        set_error(c.status, ERR_BAD_POS);
        return;
    }
    const int block0 = p0 / kKvBlock + int(blockIdx.x) * group, blocks = min(group, (p1 - 1) / kKvBlock + 1 - block0);
    if (blocks <= 0) return;
    const int tasks = blocks * 2 * c.n_kv, step = gridDim.z * kAppendWarps;
    unsigned char* tile = tiles[warp];
    const int d0 = lane % LPR * 8, tb = lane / LPR * TPL;

#pragma unroll 1
    for (int task = blockIdx.z * kAppendWarps + warp; task < tasks; task += step) {
        const int b0 = (block0 + task / (2 * c.n_kv)) * kKvBlock, kh = task % (2 * c.n_kv), kind = kh >= c.n_kv;
        const int head = kind ? kh - c.n_kv : kh;
        const int page = kv_page(c, seq, b0);
        if (page < 0) continue;  // reported
        const int in_page = b0 & (c.pt - 1), kept = max(p0 - b0, 0), end = min(p1 - b0, kKvBlock);  // tokens [kept, end) are new
        const size_t at = c.at(page, layer, kind, head);
        int8_t* codes = c.codes + at * c.tile();
        float* scale = c.scales + at * (c.pt / kKvBlock) + in_page / kKvBlock;
        const float before = *scale;
        const T* src = (kind ? v : k) + head * HD + d0;
        const long long stride = kind ? v_stride : k_stride;
        Row raw[TPL];
        typename AmaxType<T>::t most = {};
#pragma unroll
        for (int u = 0; u < TPL; ++u) {
            // (tokens that are not new read the nearest one: a load under a condition would be waited for right here)
            const int t = min(max(tb + u, kept), end - 1);
            const T* row = src + (long long)(t0 + b0 + t - p0) * stride;
            if constexpr (VEC) raw[u] = *reinterpret_cast<const Row*>(row);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[u].a[i] = row[i];
        }
        const float old = kept ? before : 0.f;
#pragma unroll
        for (int u = 0; u < TPL; ++u) most = amax8(raw[u].a, most);
        float amax = amax_of(most);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float d = max_nan(old, fmul(amax, 1.0f / 127.0f));
        const float inv = d > 0.f ? __frcp_rn(d) : 0.f;
        const bool fine = d > 0.f && d < INFINITY && inv < INFINITY;
        // the block's 16-byte pieces: K: dims 16 (i / 16) .. of token i % 16, V: dim i's tokens
        const int pitch = kind ? HD : c.pt, first = kind ? in_page / kKvBlock * HD : in_page;
        auto piece = [&](int i) {
            return reinterpret_cast<uint4*>(kind ? codes + size_t(first + i) * 16
                                                 : codes + (size_t(i / 16) * pitch + first + i % 16) * 16);
        };
        auto in_tile = [&](int i) { return tile + i * 16 + (kind ? i / 8 : i / 16) * 16; };
        __syncwarp();
        if (kept) {
            const float ratio = fine ? fdiv(old, d) : 0.f;
#pragma unroll
            for (int u = 0; u < HD / 32; ++u) {
                const int i = u * 32 + lane;
                uint4 w = *piece(i);
                if (d != old) {
                    int8_t* b = reinterpret_cast<int8_t*>(&w);
#pragma unroll
                    for (int z = 0; z < 16; ++z) b[z] = int8_t(__float2int_rn(fmul(float(b[z]), ratio)));
                }
                *reinterpret_cast<uint4*>(in_tile(i)) = w;
            }
            __syncwarp();
        }
        // A code is the low byte of 1.5 * 2^23 + x * (1 / d), rounded to an integer by that sum.  |x / d| <= 127 (1 + 2^-20), also
        // where d is subnormal (1 / d is finite from 2^-128 on): it never rounds to 128.
        const int used = fine ? end : 0;  // the later tokens' codes are 0
        unsigned q[TPL][8];
#pragma unroll
        for (int u = 0; u < TPL; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) q[u][i] = __float_as_uint(fadd(fmul(to_f(raw[u].a[i]), inv), 12582912.f));
        auto pack = [](unsigned a, unsigned b, unsigned e, unsigned f) {
            return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(e, f, 0x0040), 0x5410);
        };
        auto below = [](int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1; };  // mask of the first n bytes
        if (kind == 0) {
#pragma unroll
            for (int u = 0; u < TPL; ++u) {
                const unsigned on = tb + u < used ? ~0u : 0u;
                if (tb + u >= kept)
                    *reinterpret_cast<uint2*>(in_tile(d0 / 16 * 16 + tb + u) + d0 % 16) =
                        make_uint2(pack(q[u][0], q[u][1], q[u][2], q[u][3]) & on, pack(q[u][4], q[u][5], q[u][6], q[u][7]) & on);
            }
        } else {
#pragma unroll
            for (int h = 0; h < TPL / 4; ++h) {
                const unsigned on = below(used - tb - 4 * h), stay = below(kept - tb - 4 * h);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    unsigned* to = reinterpret_cast<unsigned*>(in_tile(d0 + i) + tb) + h;
                    unsigned w = pack(q[4 * h][i], q[4 * h + 1][i], q[4 * h + 2][i], q[4 * h + 3][i]) & on;
                    if (kept) w = (w & ~stay) | (*to & stay);
                    *to = w;
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < HD / 32; ++u) {
            const int i = u * 32 + lane;
            *piece(i) = *reinterpret_cast<const uint4*>(in_tile(i));
        }
        if (lane == 0) *scale = d;
    }
}

// ---------------------------------------------------------------- read

constexpr int kReadRows = 32, kReadWarps = 16;

__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// One CTA per 32 output rows.  Rows of one block of 16 tokens make a segment; a warp takes (segment, K or V, head): a lane reads
// its dims of all tokens before it writes the first, and rows are written whole by the warp (HD = 64: two K rows at a time).
// 35k rows of 8 heads of 128 to f32: 63 us, 4.7 TB/s (64 rows, K and V to one warp of 8, loads between the stores: 99 us).

// 4 codes -> f32, exactly: 2^23 + 128 + code in the mantissa, less 2^23 + 128
__device__ __forceinline__ void codes_f32(unsigned w, float (&x)[4]) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540 + i)) - 8388736.f;
}
template <class T, int N>
struct alignas(N * sizeof(T)) Vals {
    T a[N];
};

template <class T, int HD>
__global__ void __launch_bounds__(32 * kReadWarps) k_kv_read(KvView c, int layer, const int* __restrict__ first, KvCall call,
                                                             T* __restrict__ k_out, T* __restrict__ v_out) {
    __shared__ int page_of[kReadRows], pos_of[kReadRows], seg_row[kReadRows + 1], pivot[32 * kReadWarps];
    __shared__ int n_seg;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = blockIdx.x * kReadRows, rows = min(kReadRows, call.n_tok - row0);
    // the sequence of a row is the last with starts[j] <= row: among every `per`-th start first
    const int per = (call.n + 32 * kReadWarps - 1) / (32 * kReadWarps);
    pivot[tid] = tid * per < call.n ? __ldg(call.starts + tid * per) : INT_MAX;
    __syncthreads();
    if (tid < rows) {
        const int r = row0 + tid;
        int lo = 0;
#pragma unroll
        for (int step = 16 * kReadWarps; step > 0; step >>= 1)
            if (pivot[lo + step] <= r) lo += step;
        lo *= per;
        for (int hi = min(lo + per, call.n) - 1; lo < hi;) {
            const int mid = (lo + hi + 1) >> 1;
            if (__ldg(call.starts + mid) <= r) lo = mid;
            else hi = mid - 1;
        }
        const int seq = __ldg(call.seqs + lo), i = r - __ldg(call.starts + lo), i1 = __ldg(call.starts + lo + 1), p0 = __ldg(first + lo);
        const bool known = seq >= 0 && seq < c.max_seqs && i >= 0 && p0 >= 0 && r < i1;
        const int pos = p0 + i, k = known ? pos >> c.pt_shift : 0;
        const int len = __ldg(c.lens + (known ? seq : 0));
        int page = __ldg(c.table + size_t(known ? seq : 0) * c.max_pages + min(max(k, 0), c.max_pages - 1));
        if (!known || pos < 0 || pos >= len || k >= c.max_pages || page < 0 || page >= c.n_pages) {
            set_error(c.status, ERR_BAD_POS);
            page = -1;
        }
        page_of[tid] = page;
        pos_of[tid] = pos;
    }
    __syncthreads();
    if (warp == 0) {  // a segment starts where the block of 16 tokens does, or another sequence
        int n = 0;
        for (int g = 0; g < rows; g += 32) {
            const int r = g + lane;
            const bool start = r < rows && (r == 0 || (pos_of[r] & 15) == 0 || pos_of[r] != pos_of[r - 1] + 1 ||
                                            (page_of[r] < 0) != (page_of[r - 1] < 0) || page_of[r] != page_of[r - 1]);
            const unsigned mask = __ballot_sync(0xffffffffu, start);
            if (start) seg_row[n + __popc(mask & ((1u << lane) - 1))] = r;
            n += __popc(mask);
        }
        if (lane == 0) {
            seg_row[n] = rows;
            n_seg = n;
        }
    }
    __syncthreads();
    const size_t pitch = size_t(c.n_kv) * HD;
    for (int task = warp; task < n_seg * 2 * c.n_kv; task += kReadWarps) {
        const int s = task / (2 * c.n_kv), kh = task % (2 * c.n_kv), kind = kh >= c.n_kv, head = kind ? kh - c.n_kv : kh;
        const int r0 = seg_row[s], m = seg_row[s + 1] - r0;
        const int page = page_of[r0], in_page = pos_of[r0] & (c.pt - 1), t0 = in_page & 15;
        T* out = (kind ? v_out : k_out) + (size_t(row0 + r0) * c.n_kv + head) * HD;
        if (page < 0) {  // reported; the rows read as 0
            for (int t = 0; t < m; ++t)
                for (int d = lane; d < HD; d += 32) put(out + t * pitch + d, 0.f);
            continue;
        }
        const size_t at = c.at(page, layer, kind, head);
        const int8_t* codes = c.codes + at * c.tile();
        const float scale = __ldg(c.scales + at * (c.pt / kKvBlock) + in_page / kKvBlock);
        if (kind == 0) {
            constexpr int R = 128 / HD;  // rows at a time
            const int d = lane * 4 % HD, up = lane * 4 / HD;
            unsigned w[kKvBlock / R];
#pragma unroll
            for (int u = 0; u < kKvBlock / R; ++u)
                w[u] = *reinterpret_cast<const unsigned*>(codes + (size_t(d / 16) * c.pt + in_page + min(u * R + up, m - 1)) * 16 + d % 16);
#pragma unroll
            for (int u = 0; u < kKvBlock / R; ++u) {
                float x[4];
                codes_f32(w[u], x);
                Vals<T, 4> o;
#pragma unroll
                for (int i = 0; i < 4; ++i) put(&o.a[i], fmul(x[i], scale));
                if (u * R + up < m) *reinterpret_cast<Vals<T, 4>*>(out + (u * R + up) * pitch + d) = o;
            }
        } else {
            constexpr int N = HD / 32;  // dims of a lane
            uint4 w[N];
#pragma unroll
            for (int i = 0; i < N; ++i)
                w[i] = *reinterpret_cast<const uint4*>(codes + (size_t(in_page / 16) * HD + lane * N + i) * 16);
#pragma unroll
            for (int h = 0; h < 4; ++h) {  // 4 tokens at a time
                float x[N][4];
#pragma unroll
                for (int i = 0; i < N; ++i) codes_f32(h == 0 ? w[i].x : h == 1 ? w[i].y : h == 2 ? w[i].z : w[i].w, x[i]);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int t = h * 4 + z - t0;
                    Vals<T, N> o;
#pragma unroll
                    for (int i = 0; i < N; ++i) put(&o.a[i], fmul(x[i][z], scale));
                    if (t >= 0 && t < m) *reinterpret_cast<Vals<T, N>*>(out + t * pitch + lane * N) = o;
                }
            }
        }
    }
}

// ---------------------------------------------------------------- page bookkeeping

// The planning kernels are one CTA each: what they look over (a reference count per page, a mark per sequence) is small, and the
// lowest free pages, in order, are a prefix sum.  Bound by latency: about 10 dependent rounds of loads and barriers.  Measured:
// free of 64 sequences and reserve for 256 in a pool of 32768 pages 17 us a pair with the host's part (kernels 4 and 10 us);
// fork of 4 sequences to 64: 18.6 us (plan 7.5, copies of 25 MB 12 us); compact of 2048 pages of 393 KB with 1229 in use: 81 us
// (plan 7.6), moves at 5.4 TB/s of HBM, 16 KB of a page to a CTA.
constexpr int kPlanThreads = 1024;

// Exclusive prefix sum of one value per thread of the CTA; *total gets the sum.
__device__ __forceinline__ int cta_scan(int x, int* total) {
    __shared__ int part[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    const int p = lane < int(blockDim.x >> 5) ? part[lane] : 0;
    *total = __reduce_add_sync(0xffffffffu, p);
    return __reduce_add_sync(0xffffffffu, lane < warp ? p : 0) + inc - x;
}

// words[g] = bit i set where page 32 g + i is free (pages past the pool are not).
__device__ __forceinline__ void free_bitmap(const KvView& c, unsigned* words, int n_words) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    constexpr int U = 16;  // loads in flight
    for (int g0 = warp * U; g0 < n_words; g0 += warps * U) {
        int r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = (g0 + u) * 32 + lane;
            r[u] = p < c.n_pages ? __ldcg(c.refs + p) : 1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned mask = __ballot_sync(0xffffffffu, r[u] <= 0);
            if (lane == 0 && g0 + u < n_words) words[g0 + u] = mask;
        }
    }
}

// list[r] = the r-th free page for r < want; returns how many pages are free.  All threads of the CTA; ends synchronised.
__device__ int lowest_free(const KvView& c, unsigned* words, int want, int* list) {
    const int n_words = (c.n_pages + 31) / 32, per = (n_words + blockDim.x - 1) / int(blockDim.x);
    free_bitmap(c, words, n_words);
    __syncthreads();
    const int w0 = min(int(threadIdx.x) * per, n_words), w1 = min(w0 + per, n_words);
    int mine = 0, total;
    for (int w = w0; w < w1; ++w) mine += __popc(words[w]);
    int r = cta_scan(mine, &total);
    if (total >= want)
        for (int w = w0; w < w1 && r < want; ++w)
            for (unsigned b = words[w]; b && r < want; b &= b - 1) list[r++] = w * 32 + __ffs(b) - 1;
    __syncthreads();
    return total;
}

// Dynamic shared memory of the planning kernels: [n_words] free pages, [max_seqs] marks, [n] bases.
__host__ __device__ inline size_t plan_words(const KvView& c) { return size_t(c.n_pages + 31) / 32; }

// lens[seq] += extra and the pages for it.  A call that names a sequence twice or out of range, asks for a negative or too
// large length, or for more pages than are free, changes nothing and sets its error bit.
__global__ void __launch_bounds__(kPlanThreads) k_kv_reserve(KvView c, const int* __restrict__ seqs,
                                                             const int* __restrict__ extra, int n, int* __restrict__ list) {
    extern __shared__ __align__(16) unsigned smem[];
    unsigned* words = smem;
    int* mark = reinterpret_cast<int*>(words + plan_words(c));
    int* base = mark + c.max_seqs;
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    for (int s = threadIdx.x; s < c.max_seqs; s += blockDim.x) mark[s] = 0;
    __syncthreads();
    const int per = (n + int(blockDim.x) - 1) / int(blockDim.x);
    const int i0 = min(int(threadIdx.x) * per, n), i1 = min(i0 + per, n);
    int mine = 0;
    for (int i = i0; i < i1; ++i) {
        const int s = seqs[i], x = extra[i];
        if (s < 0 || s >= c.max_seqs || x < 0 || atomicExch(mark + s, 1)) {
            bad = 1;
            continue;
        }
        const long long len = (long long)c.lens[s] + x;
        if (len > (long long)c.max_pages << c.pt_shift) {
            bad = 1;
            continue;
        }
        const int have = (c.lens[s] + c.pt - 1) >> c.pt_shift;
        mine += int((len + c.pt - 1) >> c.pt_shift) - have;
        base[i] = mine;  // inclusive within the thread, for now
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) set_error(c.status, ERR_BAD_POS);
        return;
    }
    int want;
    const int before = cta_scan(mine, &want);
    for (int i = i0; i < i1; ++i) base[i] += before;  // pages of requests 0 .. i
    __syncthreads();
    if (want > 0 && lowest_free(c, words, want, list) < want) {
        if (threadIdx.x == 0) set_error(c.status, ERR_CAPACITY);
        return;
    }
    for (int r = threadIdx.x; r < want; r += blockDim.x) {
        int lo = 0, hi = n - 1;  // the first request with base > r
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (base[mid] > r) hi = mid;
            else lo = mid + 1;
        }
        const int s = seqs[lo], have = (c.lens[s] + c.pt - 1) >> c.pt_shift, page = list[r];
        c.table[size_t(s) * c.max_pages + have + r - (lo ? base[lo - 1] : 0)] = page;
        c.refs[page] = 1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) c.lens[seqs[i]] += extra[i];
}

// Fork, first half: fresh[i] = the page for the part-filled last page of pair i (-1: none needed); ok[0] = 1, or 0 for a
// call that is refused (a sequence out of range, a dst that is named twice, is not empty or is also a src, no pages left).
__global__ void __launch_bounds__(kPlanThreads) k_kv_fork_plan(KvView c, const int* __restrict__ src,
                                                               const int* __restrict__ dst, int n, int* __restrict__ ok,
                                                               int* __restrict__ fresh, int* __restrict__ list) {
    extern __shared__ __align__(16) unsigned smem[];
    pdl_launch_dependents();
    unsigned* words = smem;
    int* mark = reinterpret_cast<int*>(words + plan_words(c));
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    for (int s = threadIdx.x; s < c.max_seqs; s += blockDim.x) mark[s] = 0;
    __syncthreads();
    const int per = (n + int(blockDim.x) - 1) / int(blockDim.x);
    const int i0 = min(int(threadIdx.x) * per, n), i1 = min(i0 + per, n);
    int mine = 0;
    for (int i = i0; i < i1; ++i) {
        const int s = src[i], d = dst[i];
        if (s < 0 || s >= c.max_seqs || d < 0 || d >= c.max_seqs || atomicExch(mark + d, 1) || c.lens[d] != 0) {
            bad = 1;
            continue;
        }
        mine += (c.lens[s] & (c.pt - 1)) != 0;
    }
    __syncthreads();
    if (!bad)
        for (int i = i0; i < i1; ++i)
            if (mark[src[i]]) bad = 1;
    int want;
    int r = cta_scan(mine, &want);  // synchronises
    int status = bad ? int(ERR_BAD_POS) : 0;
    if (!status && want > 0 && lowest_free(c, words, want, list) < want) status = int(ERR_CAPACITY);
    if (threadIdx.x == 0) {
        ok[0] = status == 0;
        if (status) set_error(c.status, unsigned(status));
    }
    if (status) return;
    for (int i = i0; i < i1; ++i) fresh[i] = (c.lens[src[i]] & (c.pt - 1)) ? list[r++] : -1;
}

constexpr int kPagePart = 16384;  // bytes of a page that a CTA copies

// Copies a page's codes and scales, all layers; part `part` of `parts`.
__device__ __forceinline__ void copy_page(const KvView& c, int from, int to, int part, int parts) {
    const size_t n16 = c.page_codes() / 16;
    const uint4* a = reinterpret_cast<const uint4*>(c.codes + size_t(from) * c.page_codes());
    uint4* b = reinterpret_cast<uint4*>(c.codes + size_t(to) * c.page_codes());
    const size_t per = (n16 + parts - 1) / parts, i0 = size_t(part) * per, i1 = min(i0 + per, n16);
    constexpr int U = 4;  // 256 threads read a part of 16 KB at once
    for (size_t i = i0 + threadIdx.x; i < i1; i += size_t(U) * blockDim.x) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + size_t(u) * blockDim.x < i1) w[u] = __ldcs(a + i + size_t(u) * blockDim.x);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + size_t(u) * blockDim.x < i1) __stcs(b + i + size_t(u) * blockDim.x, w[u]);
    }
    const int ns = c.page_scales();
    for (int i = part * int(blockDim.x) + int(threadIdx.x); i < ns; i += parts * int(blockDim.x))
        c.scales[size_t(to) * ns + i] = c.scales[size_t(from) * ns + i];
}

// Fork, second half: grid (parts of a page, pairs); part 0 also writes the pair's table row and counts its pages.  The plan
// changes neither the sources' lengths nor their pages, so a part of at most 16 KB is read while the plan still runs.
constexpr int kForkThreads = 256;

__global__ void __launch_bounds__(kForkThreads) k_kv_fork(KvView c, const int* __restrict__ src, const int* __restrict__ dst,
                                                          const int* __restrict__ ok, const int* __restrict__ fresh) {
    constexpr int U = kPagePart / 16 / kForkThreads;
    const int i = blockIdx.y, s = src[i], d = dst[i], s0 = s >= 0 && s < c.max_seqs ? s : 0;  // (a bad one is refused by the plan)
    const int len = c.lens[s0], parts = gridDim.x;
    const int* from = c.table + size_t(s0) * c.max_pages;
    const int last = from[min(max(len >> c.pt_shift, 0), c.max_pages - 1)];  // the part-filled page, if there is one
    const bool known = last >= 0 && last < c.n_pages;
    const size_t n16 = c.page_codes() / 16, per = (n16 + parts - 1) / parts, i0 = blockIdx.x * per, i1 = min(i0 + per, n16);
    const uint4* codes = reinterpret_cast<const uint4*>(c.codes + size_t(known ? last : 0) * c.page_codes());
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = __ldcs(codes + min(i0 + u * kForkThreads + threadIdx.x, i1 - 1));
    pdl_wait();
    const int go = __ldcg(ok), to = __ldcg(fresh + i);
    if (!go) return;
    const int full = min(len >> c.pt_shift, to >= 0 ? c.max_pages - 1 : c.max_pages);
    if (to >= 0) {
        if (known) {
            uint4* out = reinterpret_cast<uint4*>(c.codes + size_t(to) * c.page_codes());
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * kForkThreads + threadIdx.x < i1) __stcs(out + i0 + u * kForkThreads + threadIdx.x, w[u]);
            const int ns = c.page_scales();
            for (int x = blockIdx.x * kForkThreads + threadIdx.x; x < ns; x += parts * kForkThreads)
                c.scales[size_t(to) * ns + x] = c.scales[size_t(last) * ns + x];
        } else if (threadIdx.x == 0) {
            set_error(c.status, ERR_BAD_POS);
        }
    }
    if (blockIdx.x == 0) {
        int* row = c.table + size_t(d) * c.max_pages;
        for (int k = threadIdx.x; k < full; k += blockDim.x) {
            const int p = from[k];
            row[k] = p;
            if (p >= 0 && p < c.n_pages) atomicAdd(c.refs + p, 1);
        }
        if (threadIdx.x == 0) {
            if (to >= 0) {
                row[full] = to;
                c.refs[to] = 1;
            }
            c.lens[d] = len;
        }
    }
}

// Sequences give their pages back.  Every CTA looks the whole list over (a list with a sequence out of range or named twice
// is refused as a whole), then takes sequences blockIdx.x, blockIdx.x + gridDim.x, ...
__global__ void __launch_bounds__(256) k_kv_free(KvView c, const int* __restrict__ seqs, int n) {
    extern __shared__ __align__(16) unsigned smem[];
    int* mark = reinterpret_cast<int*>(smem);
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    for (int s = threadIdx.x; s < c.max_seqs; s += blockDim.x) mark[s] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = seqs[i];
        if (s < 0 || s >= c.max_seqs || atomicExch(mark + s, 1)) bad = 1;
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0 && blockIdx.x == 0) set_error(c.status, ERR_BAD_POS);
        return;
    }
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int s = seqs[i], used = min((c.lens[s] + c.pt - 1) >> c.pt_shift, c.max_pages);
        int* row = c.table + size_t(s) * c.max_pages;
        for (int k = threadIdx.x; k < used; k += blockDim.x) {
            const int p = row[k];
            if (p >= 0 && p < c.n_pages) atomicSub(c.refs + p, 1);
            row[k] = -1;
        }
        __syncthreads();  // every thread has read the length
        if (threadIdx.x == 0) c.lens[s] = 0;
    }
}

// Compaction, first half: with L pages in use, the used pages at index >= L move to the free pages below L, both in
// ascending order: moves[0] = how many, moves[1] = L, from[r] -> to[r]; map[p] = the new index of every page p >= L.
__global__ void __launch_bounds__(kPlanThreads) k_kv_compact_plan(KvView c, int* __restrict__ moves, int* __restrict__ from,
                                                                  int* __restrict__ to, int* __restrict__ map) {
    extern __shared__ __align__(16) unsigned smem[];
    pdl_launch_dependents();
    unsigned* words = smem;
    const int n_words = int(plan_words(c)), per = (n_words + int(blockDim.x) - 1) / int(blockDim.x);
    free_bitmap(c, words, n_words);
    __syncthreads();
    const int w0 = min(int(threadIdx.x) * per, n_words), w1 = min(w0 + per, n_words);
    int mine = 0, n_free;
    for (int w = w0; w < w1; ++w) mine += __popc(words[w]);
    const int free0 = cta_scan(mine, &n_free), live = c.n_pages - n_free;
    // free pages below `live` = used pages at or past it
    int f = free0;
    __shared__ int n_moves;
    if (threadIdx.x == 0) n_moves = 0;
    __syncthreads();
    for (int w = w0; w < w1; ++w) {
        const unsigned b = words[w];
        if (w == live / 32) n_moves = f + __popc(b & ((1u << (live % 32)) - 1));  // free pages below live
        f += __popc(b);
    }
    __syncthreads();
    if (live == n_words * 32 && threadIdx.x == 0) n_moves = n_free;  // every word is below it
    __syncthreads();
    const int n_mv = n_moves;
    f = free0;
    for (int w = w0; w < w1; ++w) {
        for (int i = 0; i < 32; ++i) {
            const int p = w * 32 + i;
            if (p >= c.n_pages) break;
            const bool is_free = (words[w] >> i) & 1;
            if (p < live) {
                if (is_free) to[f] = p;
            } else if (!is_free) {
                const int r = (p - f) - (live - n_mv);  // used pages in [live, p)
                from[r] = p;
            } else {
                map[p] = p;
            }
            f += is_free;
        }
    }
    __syncthreads();  // to[] is complete
    for (int r = threadIdx.x; r < n_mv; r += blockDim.x) map[from[r]] = to[r];
    if (threadIdx.x == 0) {
        moves[0] = n_mv;
        moves[1] = live;
    }
}

__global__ void __launch_bounds__(256) k_kv_compact(KvView c, const int* __restrict__ moves, const int* __restrict__ from,
                                                    const int* __restrict__ to, const int* __restrict__ map, int parts) {
    pdl_wait();
    const int n = __ldcg(moves);
    for (long long task = blockIdx.x; task < (long long)n * parts; task += gridDim.x) {
        const int r = int(task / parts), a = __ldcg(from + r), b = __ldcg(to + r);
        copy_page(c, a, b, int(task % parts), parts);
        if (task % parts == 0 && threadIdx.x == 0) {
            c.refs[b] = c.refs[a];
            c.refs[a] = 0;
        }
    }
    if (n == 0) return;
    const int live = __ldcg(moves + 1);
    const size_t total = size_t(c.max_seqs) * c.max_pages;
    for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += size_t(gridDim.x) * blockDim.x) {
        const int p = c.table[i];
        if (p >= live && p < c.n_pages) c.table[i] = __ldcg(map + p);
    }
}

__global__ void __launch_bounds__(256) k_kv_copy(KvView c, const int* __restrict__ src, const int* __restrict__ dst) {
    const int a = src[blockIdx.y], b = dst[blockIdx.y];
    if (a < 0 || a >= c.n_pages || b < 0 || b >= c.n_pages) {
        if (threadIdx.x == 0) set_error(c.status, ERR_BAD_POS);
        return;
    }
    if (a != b) copy_page(c, a, b, blockIdx.x, gridDim.x);
}

// A planning kernel's launch; large pools and many sequences pass the default limit of shared memory (48 KB, static included).
template <class... KArgs, class... Args>
cudaError_t launch_plan(void (*kernel)(KArgs...), int ctas, int threads, size_t smem, cudaStream_t st, Args... args) {
    if (smem > 32 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kernel, dim3(unsigned(ctas)), dim3(unsigned(threads)), smem, st, false, args...);
}

size_t plan_smem(const KvView& c, int n) { return plan_words(c) * 4 + size_t(c.max_seqs) * 4 + size_t(n) * 4; }

// A page in parts of about 16 KB, so that one page's copy spreads over several SMs.
int page_parts(const KvView& c) { return int((c.page_codes() + kPagePart - 1) / kPagePart); }

template <class T, int HD>
cudaError_t append_t(const KvView& c, int layer, const void* k, const void* v, long long ks, long long vs, const KvCall& call,
                     int max_new, cudaStream_t st) {
    const bool vec = !((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | uintptr_t(ks * sizeof(T)) |
                        uintptr_t(vs * sizeof(T))) % 16);
    // a CTA takes up to 4 blocks of all heads, where that leaves CTAs enough; else a block of kAppendWarps tasks
    const long long blocks = (max_new + kKvBlock - 1) / kKvBlock + 1;
    const bool many = blocks * call.n >= 4 * 4 * 148;
    const int group = many ? 4 : 1;
    const dim3 grid(unsigned((blocks + group - 1) / group), unsigned(call.n),
                    many ? 1u : unsigned((2 * c.n_kv + kAppendWarps - 1) / kAppendWarps));
    auto kern = vec ? k_kv_append<T, HD, true> : k_kv_append<T, HD, false>;
    return launch_pdl(kern, grid, dim3(32 * kAppendWarps), 0, st, false, c, layer, static_cast<const T*>(k),
                      static_cast<const T*>(v), ks, vs, call, max_new, group);
}

template <class T, int HD>
cudaError_t read_t(const KvView& c, int layer, const int* first, const KvCall& call, void* k, void* v, cudaStream_t st) {
    return launch_pdl(k_kv_read<T, HD>, dim3(unsigned((call.n_tok + kReadRows - 1) / kReadRows)), dim3(32 * kReadWarps), 0, st,
                      false, c, layer, first, call, static_cast<T*>(k), static_cast<T*>(v));
}

}  // namespace

cudaError_t launch_kv_append(const KvView& c, int layer, const void* k, const void* v, KvType type, long long k_stride,
                             long long v_stride, const KvCall& call, int max_new, cudaStream_t st) {
    if (call.n == 0 || call.n_tok == 0 || max_new == 0) return cudaSuccess;
    const bool wide = c.hd == 128;
    switch (type) {
        case KV_F32: return (wide ? append_t<float, 128> : append_t<float, 64>)(c, layer, k, v, k_stride, v_stride, call, max_new, st);
        case KV_F16: return (wide ? append_t<__half, 128> : append_t<__half, 64>)(c, layer, k, v, k_stride, v_stride, call, max_new, st);
        default:
            return (wide ? append_t<__nv_bfloat16, 128> : append_t<__nv_bfloat16, 64>)(c, layer, k, v, k_stride, v_stride, call,
                                                                                      max_new, st);
    }
}

cudaError_t launch_kv_read(const KvView& c, int layer, const int* first, const KvCall& call, void* k_out, void* v_out,
                           KvType type, cudaStream_t st) {
    if (call.n == 0 || call.n_tok == 0) return cudaSuccess;
    const bool wide = c.hd == 128;
    switch (type) {
        case KV_F32: return (wide ? read_t<float, 128> : read_t<float, 64>)(c, layer, first, call, k_out, v_out, st);
        case KV_F16: return (wide ? read_t<__half, 128> : read_t<__half, 64>)(c, layer, first, call, k_out, v_out, st);
        default: return (wide ? read_t<__nv_bfloat16, 128> : read_t<__nv_bfloat16, 64>)(c, layer, first, call, k_out, v_out, st);
    }
}

// reserve: [n_pages] list.  fork: ok, [max_seqs] fresh, [n_pages] list.  compact: 2 counts, from, to, map [n_pages] each.
size_t kv_page_ws_bytes(const KvView& c) { return (size_t(c.n_pages) * 3 + size_t(c.max_seqs) + 4) * 4; }

cudaError_t launch_kv_reserve(const KvView& c, const int* seqs, const int* extra, int n, void* ws, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    return launch_plan(k_kv_reserve, 1, kPlanThreads, plan_smem(c, n), st, c, seqs, extra, n, static_cast<int*>(ws));
}

cudaError_t launch_kv_fork(const KvView& c, const int* src, const int* dst, int n, void* ws, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    int* ok = static_cast<int*>(ws);
    int* fresh = ok + 4;
    int* list = fresh + c.max_seqs;
    cudaError_t e = launch_plan(k_kv_fork_plan, 1, kPlanThreads, plan_smem(c, 0), st, c, src, dst, n, ok, fresh, list);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_kv_fork, dim3(unsigned(page_parts(c)), unsigned(n)), dim3(kForkThreads), 0, st, true, c, src, dst,
                      static_cast<const int*>(ok), static_cast<const int*>(fresh));
}

cudaError_t launch_kv_free(const KvView& c, const int* seqs, int n, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    return launch_plan(k_kv_free, n < 148 ? n : 148, 256, size_t(c.max_seqs) * 4, st, c, seqs, n);
}

cudaError_t launch_kv_compact(const KvView& c, void* ws, cudaStream_t st) {
    int* moves = static_cast<int*>(ws);
    int* from = moves + 4;
    int* to = from + c.n_pages;
    int* map = to + c.n_pages;
    cudaError_t e = launch_plan(k_kv_compact_plan, 1, kPlanThreads, plan_words(c) * 4, st, c, moves, from, to, map);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_kv_compact, dim3(148 * 8), dim3(256), 0, st, true, c, static_cast<const int*>(moves),
                      static_cast<const int*>(from), static_cast<const int*>(to), static_cast<const int*>(map), page_parts(c));
}

cudaError_t launch_kv_copy(const KvView& c, const int* src, const int* dst, int n, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    return launch_pdl(k_kv_copy, dim3(unsigned(page_parts(c)), unsigned(n)), dim3(256), 0, st, false, c, src, dst);
}

}  // namespace qb
