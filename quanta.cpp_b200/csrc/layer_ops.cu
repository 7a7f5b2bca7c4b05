// RMS norm with the residual's addition and 8-bit rows out, values of 8-bit rows, rotary positions (layer_ops.h).
#include <type_traits>

#include "layer_ops.h"
#include "rows.cuh"

namespace qb {

namespace {

bool aligned_to(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// ---------------------------------------------------------------- RMS norm to 8-bit rows

// With h = x + r (r: the residual row, h rounded once into it):
//     y = h * (1 / sqrt(mean h^2 + eps)) * w;  per 32 values: d = max |y| / 127, q = y / d to the nearest, halves away from 0
// A row stays in registers between the sum and the rounding: every byte crosses HBM once (rows above 16384 values, and above 8192 with
// a f32 residual, are spilled in part).  A thread holds R chunks of 8 consecutive
// values, so that a block of 32 is 4 neighbouring lanes and its maximum two shuffles.  Sums in f32: per thread, then per warp, then
// over warps (an error of a few 2^-24).  A block with a value that is not finite gets a NaN for its scale, every block of a row whose
// sum is not finite does.  Next to HBM, and without a residual more than HBM (8192 rows of 4096 bf16: 23.7 us, 16.4 of them for the
// bytes), instructions bound it.  So values go in pairs (f32x2), and a code is the low byte of y * u + 1.5 * 2^23, one operation whose
// rounding is that to the nearest integer; u is 1 / d one step up, so that halves go away from 0.
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// max |.| that keeps a NaN
__device__ __forceinline__ float max3_or_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 1 / d of a normal d below 2^126: an approximation and a step of Newton's method, within a unit in the last place.
__device__ __forceinline__ float reciprocal(float d) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return fmaf(r, fmaf(-d, r, 1.f), r);
}

// 8 elements as they are in memory, as 4 pairs of f32, and back with one rounding.
template <class T>
struct Raw8 {
    uint4 v[sizeof(T) / 2];
};
template <class T, bool VEC>
__device__ __forceinline__ Raw8<T> load_raw(const T* p) {
    Raw8<T> r;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
        T* e = reinterpret_cast<T*>(r.v);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
    return r;
}
template <class T>
__device__ __forceinline__ void to_pairs(const Raw8<T>& r, unsigned long long (&x)[4]) {
    const T* e = reinterpret_cast<const T*>(r.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = f2_pack(to_float(e[2 * i]), to_float(e[2 * i + 1]));
}
template <class T>
__device__ __forceinline__ void store_pairs(T* p, const unsigned long long (&x)[4], bool aligned) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = f2_unpack(x[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
    store_row(p, v, aligned);
}

// RES: there is a residual.  Rows blockIdx.x, blockIdx.x + gridDim.x, ...: a CTA keeps the weights in registers from row to row, and
// its next row is on its way while one is worked on.  8192 rows of 4096 with their residual: bf16 38.2 us, 6.3 TB/s (a CTA per row
// reads its weights, twice as many bytes as a 16-bit row, from L2 each time: 46 us), f32 68.0 us, 6.5 TB/s.
template <class T, class RT, int R, int THREADS, bool RES, bool VEC>
__global__ void __launch_bounds__(THREADS)
    k_rms_norm_q8(const T* __restrict__ x, long long x_stride, RT* __restrict__ residual, long long residual_stride,
                  const float* __restrict__ weight, float eps, int n_tok, int n, int8_t* __restrict__ q, float* __restrict__ d) {
    constexpr int C = 8;
    __shared__ float part[2][32];
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, chunks = n / C, threads = blockDim.x;
    Raw8<T> rx[R];
    Raw8<RT> rr[R];
    auto load = [&](int row) {
        const T* xr = x + row * x_stride;
        const RT* res = residual + row * residual_stride;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = r * threads + tid;
            if (c < chunks) {
                rx[r] = load_raw<T, VEC>(xr + c * C);
                if constexpr (RES) rr[r] = load_raw<RT, VEC>(res + c * C);
            }
        }
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {  // (chunks that the row does not have are zeros)
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) rx[r].v[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < int(sizeof(RT) / 2); ++i) rr[r].v[i] = make_uint4(0, 0, 0, 0);
    }
    load(blockIdx.x);
    unsigned long long w[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = r * threads + tid;
        if (c < chunks) to_pairs(load_raw<float, VEC>(weight + c * C), w[r]);
        else w[r][0] = w[r][1] = w[r][2] = w[r][3] = 0;
    }
    for (int row = blockIdx.x, turn = 0; row < n_tok; row += gridDim.x, turn ^= 1) {
        unsigned long long h[R][4], squares = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            to_pairs(rx[r], h[r]);
            if constexpr (RES) {
                unsigned long long b[4];
                to_pairs(rr[r], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[r][i] = f2_add(h[r][i], b[i]);
            }
            unsigned long long s = f2_mul(h[r][0], h[r][0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) s = f2_fma(h[r][i], h[r][i], s);
            squares = r ? f2_add(squares, s) : s;
        }
        if (row + gridDim.x < n_tok) load(row + gridDim.x);
        if constexpr (RES) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int c = r * threads + tid;
                if (c < chunks) store_pairs(residual + row * residual_stride + c * C, h[r], VEC);
            }
        }
        const float2 both = f2_unpack(squares);
        float sum = warp_sum(both.x + both.y);
        if (threads > 32) {
            if (lane == 0) part[turn][warp] = sum;
            __syncthreads();  // (the other half is written again only after the next one)
            constexpr int W = THREADS / 32;  // (every lane ends with the sum of all)
            sum = (lane & (W - 1)) < threads >> 5 ? part[turn][lane & (W - 1)] : 0.f;
#pragma unroll
            for (int o = W / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        // (an infinite sum is an infinite value's or an overflow: NaN, where 1 / sqrt would make the row's other blocks zeros)
        const float inv = sum <= 3.402823466e38f ? __frsqrt_rn(sum / float(n) + eps) : __int_as_float(0x7fc00000);
        const unsigned long long inv2 = f2_pack(inv, inv), magic = f2_pack(12582912.f, 12582912.f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = r * threads + tid;
            const bool in = c < chunks;
            unsigned long long y[4];
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                y[i] = f2_mul(f2_mul(h[r][i], inv2), w[r][i]);
                const float2 v = f2_unpack(y[i]);
                top = max3_or_nan(top, fabsf(v.x), fabsf(v.y));
            }
            top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float scale = div127(top);
            const float up = scale >= 1.17549435e-38f ? __uint_as_float(__float_as_uint(reciprocal(scale)) + 1) : 0.f;
            const unsigned long long up2 = f2_pack(up, up);
            unsigned b[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = f2_unpack(f2_fma(y[i], up2, magic));
                b[2 * i] = __float_as_uint(t.x);
                b[2 * i + 1] = __float_as_uint(t.y);
            }
            if (in) {
                uint2 codes;
                codes.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
                codes.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
                *reinterpret_cast<uint2*>(q + size_t(row) * n + c * C) = codes;
                if ((lane & 3) == 0) d[size_t(row) * (n / QK) + c / 4] = top <= 3.402823466e38f ? scale : __int_as_float(0x7fc00000);
            }
        }
    }
}

template <class T, class RT, bool RES, bool VEC>
cudaError_t norm_r(const NormQ8Args& a, cudaStream_t st) {
    // Two chunks a thread halve a row's shuffles and its barrier: 8192 rows of 4096 bf16 with their residual 38.2 us (one chunk: 49,
    // four: 59), 16384 of 2048 38.0 (one: 46.4).  One has the shorter chain where rows are few: 256 of 896 f32 1.9 us (two: 2.3), 1000
    // of 1024 3.2 (3.3), 600 of 2048 bf16 3.0 (2.9).  Four are for rows above 16384, the longest that 1024 threads hold in two; their
    // registers spill (128 to 1220 bytes a thread, two with 1024 threads and a f32 residual 8 to 40): 1024 rows of 32768 bf16 29.6 us,
    // 67.6 with their residual, f32 with it 289, where 2048 of 16384 take 25.0, 39.5 and 74.5 for as many bytes.
    const int chunks = a.n / 8;
    const bool many = chunks > 32 && (long long)a.n_tok * chunks >= 148 * 1024;
    const int r = chunks <= 256 && !many ? 1 : chunks <= 2048 ? 2 : 4;
    const int threads = ((chunks + r - 1) / r + 31) / 32 * 32;
    auto kern = r == 1           ? k_rms_norm_q8<T, RT, 1, 256, RES, VEC>
                : r == 4         ? k_rms_norm_q8<T, RT, 4, 1024, RES, VEC>
                : threads <= 512 ? k_rms_norm_q8<T, RT, 2, 512, RES, VEC>
                                 : k_rms_norm_q8<T, RT, 2, 1024, RES, VEC>;
    // CTAs for 2048 threads an SM.  Two chunks a thread take 58 to 80 registers, so that half of these run at a time, or less (of 256
    // threads 4 of 8 an SM; f32 with its residual 3): the rows go in two or three waves, and each CTA reads the weights for its share.
    const int most = 148 * (2048 / threads > 16 ? 16 : 2048 / threads);
    return launch_pdl(kern, dim3(unsigned(a.n_tok < most ? a.n_tok : most)), dim3(unsigned(threads)), 0, st, true,
                      static_cast<const T*>(a.x), a.x_stride, static_cast<RT*>(a.residual), a.residual_stride, a.weight, a.eps, a.n_tok,
                      a.n, a.q, a.d);
}

template <class T, class RT>
cudaError_t norm_t(const NormQ8Args& a, cudaStream_t st) {
    const bool vec = aligned_to(a.x, 16) && a.x_stride * sizeof(T) % 16 == 0 && aligned_to(a.residual, 16) &&
                     a.residual_stride * sizeof(RT) % 16 == 0 && aligned_to(a.weight, 16);
    if (!a.residual) return vec ? norm_r<T, T, false, true>(a, st) : norm_r<T, T, false, false>(a, st);
    return vec ? norm_r<T, RT, true, true>(a, st) : norm_r<T, RT, true, false>(a, st);
}

// ---------------------------------------------------------------- values of 8-bit rows

// 16 bytes of output a thread and step, so that a warp writes whole lines; kDequantAhead steps in flight.  Bound by HBM: 8192 rows of
// 4096 to bf16 17.3 us, 6.1 TB/s.
constexpr int kDequantAhead = 4;

template <class T>
__global__ void __launch_bounds__(256) k_dequantize_q8(const int8_t* __restrict__ q, const float* __restrict__ d, long long pieces,
                                                       T* __restrict__ out) {
    constexpr int V = 16 / sizeof(T);
    using Codes = typename std::conditional<V == 8, uint2, unsigned>::type;
    pdl_wait();
    pdl_launch_dependents();
    const long long first = (long long)blockIdx.x * (256 * kDequantAhead) + threadIdx.x;
    Codes w[kDequantAhead];
    float s[kDequantAhead];
#pragma unroll
    for (int u = 0; u < kDequantAhead; ++u) {
        const long long i = first + u * 256;
        if (i < pieces) {
            w[u] = __ldg(reinterpret_cast<const Codes*>(q) + i);
            s[u] = __ldg(d + i / (QK / V));
        }
    }
#pragma unroll
    for (int u = 0; u < kDequantAhead; ++u) {
        const long long i = first + u * 256;
        if (i >= pieces) continue;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            unsigned word;
            if constexpr (V == 8) word = j < 4 ? w[u].x : w[u].y;
            else word = w[u];
            v[j] = fmul(float(int8_t(word >> (j % 4 * 8))), s[u]);
        }
        store_row(out + i * V, v, true);
    }
}

template <class T>
cudaError_t dequantize_t(const int8_t* q, const float* d, long long n, void* out, cudaStream_t st) {
    const long long pieces = n * sizeof(T) / 16, per = 256 * kDequantAhead;
    return launch_pdl(k_dequantize_q8<T>, dim3(unsigned((pieces + per - 1) / per)), dim3(256), 0, st, true, q, d, pieces,
                      static_cast<T*>(out));
}

// ---------------------------------------------------------------- rotary positions

// Pair (a, b) of a head's first rotary_dim dims at position p: (a cos - b sin, a sin + b cos) * scale at p * turns[i] revolutions;
// pairs are (i, i + rotary_dim / 2) or (2 i, 2 i + 1).  The revolution count is formed in 64 bits and only its fraction becomes
// f32: an angle is off by 1e-7 at the start, and by 4e-7 more at position 2^31 (the 64-bit roundings of a turn and its product).  A
// thread has a token and a unit of its heads (interleaved: V dims of 16 bytes; half layout: V dims and the V that they turn with),
// forms these pairs' cosines and sines once and takes one head after another, 64 bytes of them in flight; `slots` threads share the
// heads of a token.  Bound by HBM: 8192 tokens of 32 + 8 heads of 128: bf16 28.9 us, 5.8 TB/s, f32 56.8 us, 5.9 TB/s (128 bytes in
// flight: 44, too many registers; without streaming stores 44; cosines and sines of a CTA's tokens in shared memory and a task of any
// head: 57).
constexpr int kRopeThreads = 128;

// VEC: V elements are one access; else they are read one by one.
template <class T, int V, bool VEC>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    if constexpr (VEC) {
        return *reinterpret_cast<const Pack<T, V>*>(p);
    } else {
        Pack<T, V> w;
#pragma unroll
        for (int i = 0; i < V; ++i) w.v[i] = p[i];
        return w;
    }
}
template <class T, int V, bool VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& w) {
    if constexpr (VEC && sizeof(w) == 16) {
        __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&w));
    } else if constexpr (VEC) {
        *reinterpret_cast<Pack<T, V>*>(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = w.v[i];
    }
}

template <class T, int V, bool INTER, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) k_rope(RopeHeads qh, RopeHeads kh, int head_dim, int rotary_dim, int n_tok, int slots,
                                                       const int* __restrict__ positions, const double* __restrict__ turns, float scale,
                                                       int units) {
    constexpr int P = INTER ? V / 2 : V, AHEAD = INTER ? 4 : 2;  // pairs of a unit, heads in flight
    pdl_wait();
    pdl_launch_dependents();
    const int pairs = rotary_dim / 2, n_rot = INTER ? rotary_dim / V : pairs / V;
    // thread -> token, slot, unit; units: rotated ones first, then ones (half layout: two) of V dims that are only copied
    const long long id = (long long)blockIdx.x * kRopeThreads + threadIdx.x;
    const int per = slots * units, t = int(id / per), in_tok = int(id - (long long)t * per), slot = in_tok / units, u = in_tok - slot * units;
    if (t >= n_tok) return;
    const bool rot = u < n_rot;
    const int at = rot ? u * V : rotary_dim + (u - n_rot) * V, other = rot ? pairs : (units - n_rot) * V;
    const bool two = !INTER && at + other < head_dim;
    float c[P], s[P];
    if (rot) {
        const double p = double(__ldg(positions + t));
        const double* turn = turns + (INTER ? at / 2 : at);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const double n = p * __ldg(turn + i);
            sincospif(2.f * float(n - rint(n)), &s[i], &c[i]);
            c[i] *= scale;
            s[i] *= scale;
        }
    }
    auto heads = [&](const RopeHeads& h) {
        const T* from = static_cast<const T*>(h.in) + t * h.in_stride + at;
        T* to = static_cast<T*>(h.out) + t * h.out_stride + at;
#pragma unroll 1
        for (int h0 = slot; h0 < h.heads; h0 += slots * AHEAD) {
            Pack<T, V> lo[AHEAD], hi[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (h0 + a * slots < h.heads) {
                    const T* x = from + (h0 + a * slots) * head_dim;
                    lo[a] = load_pack<T, V, VEC>(x);
                    if (two) hi[a] = load_pack<T, V, VEC>(x + other);
                }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (h0 + a * slots < h.heads) {
                    T* y = to + (h0 + a * slots) * head_dim;
                    if (rot) {
                        float x[V], z[V];
                        to_floats(lo[a], x);
                        if constexpr (INTER) {
#pragma unroll
                            for (int i = 0; i < P; ++i) {
                                const float v = x[2 * i], w = x[2 * i + 1];
                                x[2 * i] = fmaf(v, c[i], -(w * s[i]));
                                x[2 * i + 1] = fmaf(v, s[i], w * c[i]);
                            }
                        } else {
                            to_floats(hi[a], z);
#pragma unroll
                            for (int i = 0; i < P; ++i) {
                                const float v = x[i], w = z[i];
                                x[i] = fmaf(v, c[i], -(w * s[i]));
                                z[i] = fmaf(v, s[i], w * c[i]);
                            }
                            hi[a] = from_floats(z, T());
                        }
                        lo[a] = from_floats(x, T());
                    }
                    store_pack<T, V, VEC>(y, lo[a]);
                    if (two) store_pack<T, V, VEC>(y + other, hi[a]);
                }
        }
    };
    heads(qh);
    heads(kh);
}

template <class T, int V, bool INTER, bool VEC>
cudaError_t rope_v(const RopeArgs& a, cudaStream_t st) {
    const int most = a.q.heads > a.k.heads ? a.q.heads : a.k.heads;
    const int copied = a.q.in == a.q.out && a.k.in == a.k.out ? 0 : (a.head_dim - a.rotary_dim) / V;
    const int units = INTER ? a.rotary_dim / V + copied : a.rotary_dim / 2 / V + (copied + 1) / 2;
    int slots = 1;  // threads that share a token's heads: until there are threads enough for every SM
    while (slots < most && (long long)a.n_tok * slots * units < 148 * 1024) slots *= 2;
    if (slots > most) slots = most;
    const long long threads = (long long)a.n_tok * slots * units, ctas = (threads + kRopeThreads - 1) / kRopeThreads;
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_pdl(k_rope<T, V, INTER, VEC>, dim3(unsigned(ctas)), dim3(kRopeThreads), 0, st, true, a.q, a.k, a.head_dim, a.rotary_dim,
                      a.n_tok, slots, a.positions, a.turns, a.scale, units);
}

template <class T, int V>
bool rope_fits(const RopeArgs& a) {
    if ((a.interleaved ? a.rotary_dim : a.rotary_dim / 2) % V || (a.head_dim - a.rotary_dim) % V || a.head_dim % V) return false;
    for (const RopeHeads* h : {&a.q, &a.k})
        if (h->heads && (!aligned_to(h->in, V * sizeof(T)) || !aligned_to(h->out, V * sizeof(T)) || h->in_stride % V || h->out_stride % V))
            return false;
    return true;
}

// Accesses of 16 bytes, of 8 where sizes or addresses do not allow that, else of an element.
template <class T, bool INTER>
cudaError_t rope_t(const RopeArgs& a, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (rope_fits<T, V>(a)) return rope_v<T, V, INTER, true>(a, st);
    if (rope_fits<T, V / 2>(a)) return rope_v<T, V / 2, INTER, true>(a, st);
    return rope_v<T, INTER ? 2 : 1, INTER, false>(a, st);
}

}  // namespace

cudaError_t launch_rms_norm_q8(const NormQ8Args& a, cudaStream_t st) {
    if (a.n_tok == 0) return cudaSuccess;
    switch (a.type) {
        case KV_F32: return norm_t<float, float>(a, st);
        case KV_F16: return a.residual && a.residual_f32 ? norm_t<__half, float>(a, st) : norm_t<__half, __half>(a, st);
        default: return a.residual && a.residual_f32 ? norm_t<__nv_bfloat16, float>(a, st) : norm_t<__nv_bfloat16, __nv_bfloat16>(a, st);
    }
}

cudaError_t launch_dequantize_q8(const int8_t* q, const float* d, long long n, void* out, KvType type, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    switch (type) {
        case KV_F32: return dequantize_t<float>(q, d, n, out, st);
        case KV_F16: return dequantize_t<__half>(q, d, n, out, st);
        default: return dequantize_t<__nv_bfloat16>(q, d, n, out, st);
    }
}

cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
    if (a.n_tok == 0 || a.q.heads + a.k.heads == 0) return cudaSuccess;
    switch (a.type) {
        case KV_F32: return (a.interleaved ? rope_t<float, true> : rope_t<float, false>)(a, st);
        case KV_F16: return (a.interleaved ? rope_t<__half, true> : rope_t<__half, false>)(a, st);
        default: return (a.interleaved ? rope_t<__nv_bfloat16, true> : rope_t<__nv_bfloat16, false>)(a, st);
    }
}

}  // namespace qb
