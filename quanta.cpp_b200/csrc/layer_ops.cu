// RMS norm with the residual's addition and 8-bit rows out, values of 8-bit rows, rotary positions (layer_ops.h).
#include "layer_ops.h"
#include "rows.cuh"

namespace qb {

namespace {

bool aligned_to(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// ---------------------------------------------------------------- RMS norm to 8-bit rows

// With h = x + r (r: the residual row, h rounded once into it):
//     y = h * (1 / sqrt(mean h^2 + eps)) * w;  per 32 values: d = max |y| / 127, q = y * (1 / d) to the nearest, halves away from 0
// A CTA per row, which stays in registers between the sum and the rounding: every byte crosses HBM once.  A thread holds R chunks
// of 8 consecutive values, so that a block of 32 is 4 neighbouring lanes and its maximum two shuffles.  Sums in f32: per thread,
// then per warp, then over warps (an error of a few 2^-24).  A block with a value that is not finite gets a scale that is not and
// codes 0: it reads as NaN.
template <class T, class RT, int R, bool VEC>
__global__ void __launch_bounds__(1024) k_rms_norm_q8(const T* __restrict__ x, long long x_stride, RT* __restrict__ residual,
                                                      long long residual_stride, const float* __restrict__ weight, float eps,
                                                      int n, int8_t* __restrict__ q, float* __restrict__ d) {
    constexpr int C = 8;
    __shared__ float part[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, chunks = n / C;
    const T* xr = x + blockIdx.x * x_stride;
    RT* rr = residual ? residual + blockIdx.x * residual_stride : nullptr;
    float h[R][C], w[R][C];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = r * int(blockDim.x) + tid;
        if (c < chunks) {
            load_row(xr + c * C, h[r], VEC);
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i) h[r][i] = 0.f;
        }
    }
    if (rr) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = r * int(blockDim.x) + tid;
            if (c < chunks) {
                float b[C];
                load_row(rr + c * C, b, VEC);
#pragma unroll
                for (int i = 0; i < C; ++i) h[r][i] = fadd(h[r][i], b[i]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = r * int(blockDim.x) + tid;
        if (c < chunks) load_row(weight + c * C, w[r], VEC);
    }
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < C; ++i) s = fmaf(h[r][i], h[r][i], s);
        sum += s;
    }
    sum = warp_sum(sum);
    if (blockDim.x > 32) {
        if (lane == 0) part[warp] = sum;
        __syncthreads();
        sum = warp_sum(lane < int(blockDim.x >> 5) ? part[lane] : 0.f);
    }
    const float inv = __frsqrt_rn(sum / float(n) + eps);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = r * int(blockDim.x) + tid;
        const bool in = c < chunks;
        float top = 0.f, y[C];
        if (in && rr) store_row(rr + c * C, h[r], VEC);
#pragma unroll
        for (int i = 0; i < C; ++i) {
            y[i] = in ? h[r][i] * inv * w[r][i] : 0.f;
            top = max_or_nan(top, fabsf(y[i]));
        }
        top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float scale = div127(top), up = scale > 0.f ? __frcp_rn(scale) : 0.f;
        const bool fine = top <= 3.402823466e38f && up <= 3.402823466e38f;
        uint2 codes = make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const unsigned b = unsigned(fine ? round_away(fmul(y[i], up)) : 0) & 0xff;
            (i < 4 ? codes.x : codes.y) |= b << (i % 4 * 8);
        }
        if (in) {
            *reinterpret_cast<uint2*>(q + size_t(blockIdx.x) * n + c * C) = codes;
            if ((lane & 3) == 0) d[size_t(blockIdx.x) * (n / QK) + c / 4] = scale;
        }
    }
}

template <class T, class RT, bool VEC>
cudaError_t norm_r(const NormQ8Args& a, cudaStream_t st) {
    const int chunks = a.n / 8, r = chunks <= 256 ? 1 : chunks <= 1024 ? 2 : 4;
    const int threads = ((chunks + r - 1) / r + 31) / 32 * 32;
    auto kern = r == 1 ? k_rms_norm_q8<T, RT, 1, VEC> : r == 2 ? k_rms_norm_q8<T, RT, 2, VEC> : k_rms_norm_q8<T, RT, 4, VEC>;
    return launch_pdl(kern, dim3(unsigned(a.n_tok)), dim3(unsigned(threads)), 0, st, false, static_cast<const T*>(a.x), a.x_stride,
                      static_cast<RT*>(a.residual), a.residual_stride, a.weight, a.eps, a.n, a.q, a.d);
}

template <class T, class RT>
cudaError_t norm_t(const NormQ8Args& a, cudaStream_t st) {
    const bool vec = aligned_to(a.x, 16) && a.x_stride * sizeof(T) % 16 == 0 && aligned_to(a.residual, 16) &&
                     a.residual_stride * sizeof(RT) % 16 == 0 && aligned_to(a.weight, 16);
    return vec ? norm_r<T, RT, true>(a, st) : norm_r<T, RT, false>(a, st);
}

// ---------------------------------------------------------------- values of 8-bit rows

// 16 codes (half a block) a thread.
template <class T>
__global__ void __launch_bounds__(256) k_dequantize_q8(const int8_t* __restrict__ q, const float* __restrict__ d, long long halves,
                                                       T* __restrict__ out) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= halves) return;
    const uint4 w = __ldcs(reinterpret_cast<const uint4*>(q) + i);
    const float s = __ldcs(d + i / 2);
    const unsigned words[4] = {w.x, w.y, w.z, w.w};
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = fmul(float(int8_t(words[j / 4] >> (j % 4 * 8))), s);
    store_row(out + i * 16, v, true);
}

template <class T>
cudaError_t dequantize_t(const int8_t* q, const float* d, long long n, void* out, cudaStream_t st) {
    const long long halves = n / 16;
    return launch_pdl(k_dequantize_q8<T>, dim3(unsigned((halves + 255) / 256)), dim3(256), 0, st, false, q, d, halves,
                      static_cast<T*>(out));
}

// ---------------------------------------------------------------- rotary positions

// Pair (a, b) of a head's first rotary_dim dims at position p: (a cos - b sin, a sin + b cos) * scale at p * turns[i] revolutions;
// pairs are (i, i + rotary_dim / 2) or (2 i, 2 i + 1).  The revolution count is formed in 64 bits and only its fraction becomes
// f32, so that an angle is as exact at position 2^31 as at the start.  A CTA takes a few tokens: their cosines and sines go to
// shared memory once, then all heads of q and k pass through registers, V elements of 16 bytes at a time.  Bound by HBM.
constexpr int kRopeThreads = 256;
constexpr int kRopeAhead = 4;  // tasks of a thread whose loads are in flight together

// d = quotient: by a multiplication where the numbers are small (magic != 0), see rope_v.
__device__ __forceinline__ int quotient(int n, int d, unsigned magic) { return magic ? int(__umulhi(unsigned(n), magic)) : n / d; }

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
    if constexpr (VEC) {
        *reinterpret_cast<Pack<T, V>*>(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = w.v[i];
    }
}

template <class T, int V, bool INTER, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) k_rope(RopeHeads qh, RopeHeads kh, int head_dim, int rotary_dim, int n_tok,
                                                       int tok_per_cta, const int* __restrict__ positions,
                                                       const double* __restrict__ turns, float scale, int units,
                                                       unsigned units_magic, unsigned heads_magic) {
    extern __shared__ float2 cs[];  // [tok_per_cta][rotary_dim / 2]
    const int pairs = rotary_dim / 2, t0 = blockIdx.x * tok_per_cta, toks = min(tok_per_cta, n_tok - t0);
    for (int t = 0; t < toks; ++t) {
        const double p = double(__ldg(positions + t0 + t));
        for (int i = threadIdx.x; i < pairs; i += kRopeThreads) {
            const double turn = p * __ldg(turns + i);
            float s, c;
            sincospif(2.f * float(turn - rint(turn)), &s, &c);
            cs[t * pairs + i] = make_float2(c * scale, s * scale);
        }
    }
    __syncthreads();
    // a task: a unit of a head; units: rotated ones first (INTER: V elements, else V elements of either half), then V elements that
    // are only copied
    const int heads = qh.heads + kh.heads, n_rot = INTER ? rotary_dim / V : pairs / V, tasks = toks * heads * units;
    for (int task0 = threadIdx.x; task0 < tasks; task0 += kRopeThreads * kRopeAhead) {
        Pack<T, V> lo[kRopeAhead], hi[kRopeAhead];
        T* to[kRopeAhead];
        int trig[kRopeAhead];  // -1: copied
#pragma unroll
        for (int a = 0; a < kRopeAhead; ++a) {
            const int task = task0 + a * kRopeThreads;
            if (task >= tasks) break;
            const int row = quotient(task, units, units_magic), u = task - row * units;
            const int t = quotient(row, heads, heads_magic), h = row - t * heads;
            const bool is_q = h < qh.heads, rot = u < n_rot;
            const int at = (is_q ? h : h - qh.heads) * head_dim + (rot ? u * V : rotary_dim + (u - n_rot) * V);
            const T* from = static_cast<const T*>(is_q ? qh.in : kh.in) + (t0 + t) * (is_q ? qh.in_stride : kh.in_stride) + at;
            to[a] = static_cast<T*>(is_q ? qh.out : kh.out) + (t0 + t) * (is_q ? qh.out_stride : kh.out_stride) + at;
            trig[a] = rot ? t * pairs + (INTER ? u * V / 2 : u * V) : -1;
            lo[a] = load_pack<T, V, VEC>(from);
            if (!INTER && rot) hi[a] = load_pack<T, V, VEC>(from + pairs);
        }
#pragma unroll
        for (int a = 0; a < kRopeAhead; ++a) {
            if (task0 + a * kRopeThreads >= tasks) break;
            if (trig[a] >= 0) {
                if constexpr (INTER) {
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        const float2 r = cs[trig[a] + i / 2];
                        const float x = to_float(lo[a].v[i]), y = to_float(lo[a].v[i + 1]);
                        lo[a].v[i] = from_float<T>(fmaf(x, r.x, -(y * r.y)));
                        lo[a].v[i + 1] = from_float<T>(fmaf(x, r.y, y * r.x));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float2 r = cs[trig[a] + i];
                        const float x = to_float(lo[a].v[i]), y = to_float(hi[a].v[i]);
                        lo[a].v[i] = from_float<T>(fmaf(x, r.x, -(y * r.y)));
                        hi[a].v[i] = from_float<T>(fmaf(x, r.y, y * r.x));
                    }
                    store_pack<T, V, VEC>(to[a] + pairs, hi[a]);
                }
            }
            store_pack<T, V, VEC>(to[a], lo[a]);
        }
    }
}

template <class T, int V, bool INTER, bool VEC>
cudaError_t rope_v(const RopeArgs& a, cudaStream_t st) {
    const int heads = a.q.heads + a.k.heads, pairs = a.rotary_dim / 2;
    const bool in_place = a.q.in == a.q.out && a.k.in == a.k.out;
    const int units = (INTER ? a.rotary_dim : pairs) / V + (in_place ? 0 : (a.head_dim - a.rotary_dim) / V);
    int per = 1;  // tokens of a CTA: until every SM has several CTAs of it, while a CTA's tasks are few
    while (per < 8 && a.n_tok / (2 * per) >= 8 * 148 && 2 * per * heads * units <= 8 * kRopeThreads) per *= 2;
    const bool small = per * heads * units < 65536;  // n / d = umulhi(n, ceil(2^32 / d)) for n, d < 2^16, d > 1
    const unsigned um = small && units > 1 ? unsigned((0x100000000ULL + units - 1) / units) : 0;
    const unsigned hm = small && heads > 1 ? unsigned((0x100000000ULL + heads - 1) / heads) : 0;
    return launch_pdl(k_rope<T, V, INTER, VEC>, dim3(unsigned((a.n_tok + per - 1) / per)), dim3(kRopeThreads),
                      size_t(per) * pairs * sizeof(float2), st, false, a.q, a.k, a.head_dim, a.rotary_dim, a.n_tok, per, a.positions,
                      a.turns, a.scale, units, um, hm);
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
        case KV_F16: return a.residual_f32 ? norm_t<__half, float>(a, st) : norm_t<__half, __half>(a, st);
        default: return a.residual_f32 ? norm_t<__nv_bfloat16, float>(a, st) : norm_t<__nv_bfloat16, __nv_bfloat16>(a, st);
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
