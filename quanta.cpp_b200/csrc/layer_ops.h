// Operators around the quantized products of a decoder layer (layer_ops.cu): RMS norm with the residual's addition and 8-bit
// rows out, values of 8-bit rows, rotary positions.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.h"

namespace qb {

constexpr int kNormMax = 32768;  // longest row of the norm

struct NormQ8Args {
    const void* x;      // token t at x + t * x_stride (elements)
    long long x_stride;
    void* residual;     // or null: h = x + residual, written back
    long long residual_stride;
    const float* weight;
    float eps;
    int n_tok, n;
    int8_t* q;  // [n_tok][n]
    float* d;   // [n_tok][n / 32]
    KvType type;
    bool residual_f32;  // else of x's type
};
cudaError_t launch_rms_norm_q8(const NormQ8Args& a, cudaStream_t st);

cudaError_t launch_dequantize_q8(const int8_t* q, const float* d, long long n_values, void* out, KvType type, cudaStream_t st);

// Heads of one kind: token t, head h, dim i at t * stride + h * head_dim + i (elements), in and out.
struct RopeHeads {
    const void* in;
    void* out;
    long long in_stride, out_stride;
    int heads;
};
struct RopeArgs {
    RopeHeads q, k;
    int head_dim, rotary_dim, n_tok;
    const int* positions;  // [n_tok]
    const double* turns;   // [rotary_dim / 2] revolutions a position
    float scale;           // on the rotated values
    bool interleaved;
    KvType type;
};
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st);

}  // namespace qb
