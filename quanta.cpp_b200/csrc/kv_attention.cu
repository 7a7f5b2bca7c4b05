// Attention over the paged 8-bit KV cache (kv_cache.h has the layout).
//
// Query i of a sequence's m queries sits at position p = len - m + i and sees the keys max(0, p - window + 1) .. p
// (window 0: all up to p).  With kc, vc the int8 codes and ks, vs the scales of key j's block of 16 tokens:
//     s_j = scale * ks_j * (q . kc_j);   out = sum_j softmax(s)_j * vs_j * vc_j;   lse = log sum_j exp(s_j)
// A query that sees no key gets out = 0 and lse = -inf.
#include <cuda_bf16.h>

#include "kv_cache.h"

namespace qb {

namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// One warp per (token, head), 32 keys at a time: lane l scores key l, then lane l sums dims l, l + 32, ...
template <class T, int HD>
__global__ void __launch_bounds__(128) k_kv_attn(KvView c, KvAttnArgs a, KvCall call) {
    __shared__ float sq[4][HD], sw[4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int j = blockIdx.y;
    const int t0 = __ldg(call.starts + j), m = min(__ldg(call.starts + j + 1), call.n_tok) - t0, seq = __ldg(call.seqs + j);
    if (t0 < 0 || m <= 0) return;
    if (seq < 0 || seq >= c.max_seqs || m > a.max_q) {
        set_error(c.status, ERR_BAD_POS);
        return;
    }
    const int len = min(__ldg(c.lens + seq), c.max_pages << c.pt_shift);
    for (int row = blockIdx.x * 4 + warp; row < m * a.n_heads; row += gridDim.x * 4) {
        const int i = row / a.n_heads, h = row % a.n_heads, head = h / a.group, pos = len - m + i;
        const T* q = static_cast<const T*>(a.q) + (long long)(t0 + i) * a.q_stride + h * HD;
        __syncwarp();
        for (int d = lane; d < HD; d += 32) sq[warp][d] = to_f(q[d]);
        __syncwarp();
        float top = -INFINITY, sum = 0.f, o[HD / 32] = {};
        const int j0 = a.window ? max(0, pos - a.window + 1) : 0;
        for (int k0 = j0 & ~31; k0 <= pos; k0 += 32) {
            const int k = k0 + lane;
            float s = -INFINITY, vs = 0.f;
            if (k >= j0 && k <= pos) {
                int page = __ldg(c.table + size_t(seq) * c.max_pages + (k >> c.pt_shift));
                if (page < 0 || page >= c.n_pages) {
                    set_error(c.status, ERR_BAD_POS);
                    page = 0;
                }
                const int t = k & (c.pt - 1);
                const size_t ak = c.at(page, a.layer, 0, head), av = c.at(page, a.layer, 1, head);
                float acc = 0.f;
                for (int g = 0; g < HD / 16; ++g) {
                    const uint4 w = *reinterpret_cast<const uint4*>(c.codes + ak * c.tile() + (size_t(g) * c.pt + t) * 16);
                    const int8_t* b = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
                    for (int z = 0; z < 16; ++z) acc += sq[warp][16 * g + z] * float(b[z]);
                }
                s = acc * (a.scale * __ldg(c.scales + ak * (c.pt / 16) + t / 16));
                vs = __ldg(c.scales + av * (c.pt / 16) + t / 16);
            }
            float now = s;
#pragma unroll
            for (int z = 16; z > 0; z >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, z));
            now = fmaxf(now, top);
            const float keep = top == -INFINITY ? 0.f : expf(top - now);
            const float p = s == -INFINITY ? 0.f : expf(s - now);
            top = now;
            sum = sum * keep + p;
            __syncwarp();
            sw[warp][lane] = p * vs;
            __syncwarp();
#pragma unroll
            for (int u = 0; u < HD / 32; ++u) o[u] *= keep;
            for (int z = 0; z < 32; z += 16) {
                if (k0 + z > pos || k0 + z + 16 <= j0) continue;
                int page = __ldg(c.table + size_t(seq) * c.max_pages + ((k0 + z) >> c.pt_shift));
                if (page < 0 || page >= c.n_pages) page = 0;
                const int8_t* tile = c.codes + c.at(page, a.layer, 1, head) * c.tile() + size_t(((k0 + z) & (c.pt - 1)) / 16) * HD * 16;
                for (int u = 0; u < HD / 32; ++u) {
                    const uint4 w = *reinterpret_cast<const uint4*>(tile + (lane + 32 * u) * 16);
                    const int8_t* b = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
                    for (int y = 0; y < 16; ++y) o[u] += k0 + z + y <= pos && k0 + z + y >= j0 ? sw[warp][z + y] * float(b[y]) : 0.f;
                }
            }
        }
#pragma unroll
        for (int z = 16; z > 0; z >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, z);
        const bool none = pos < 0;
        T* out = static_cast<T*>(a.out) + (size_t(t0 + i) * a.n_heads + h) * HD;
#pragma unroll
        for (int u = 0; u < HD / 32; ++u) put(out + lane + 32 * u, none ? 0.f : o[u] / sum);
        if (a.lse && lane == 0) a.lse[size_t(t0 + i) * a.n_heads + h] = none ? -INFINITY : top + logf(sum);
    }
}

template <class T>
cudaError_t attn_t(const KvView& c, const KvAttnArgs& a, const KvCall& call, cudaStream_t st) {
    const dim3 grid(unsigned((a.max_q * a.n_heads + 3) / 4), unsigned(call.n));
    return launch_pdl(c.hd == 128 ? k_kv_attn<T, 128> : k_kv_attn<T, 64>, grid, dim3(128), 0, st, false, c, a, call);
}

}  // namespace

size_t kv_attn_ws_bytes(const KvView&, const KvAttnArgs&, const KvCall&) { return 0; }

cudaError_t launch_kv_attention(const KvView& c, const KvAttnArgs& a, const KvCall& call, void*, cudaStream_t st) {
    if (call.n == 0 || call.n_tok == 0) return cudaSuccess;
    return a.type == KV_F32 ? attn_t<float>(c, a, call, st)
         : a.type == KV_F16 ? attn_t<__half>(c, a, call, st) : attn_t<__nv_bfloat16>(c, a, call, st);
}

}  // namespace qb
