// The paged 8-bit KV cache: device view and launchers (kv_pages.cu, kv_attention.cu).
//
// Codes are int8, one f32 scale for each block of 16 tokens of a page, K or V, layer and kv head; value = code * scale.
// A page holds page_tokens positions of every layer and kv head:
//   codes  [page][layer][2: K, V][kv head][page_tokens * head_dim]
//            K tile [head_dim / 16][page_tokens][16 dims], V tile [page_tokens / 16][head_dim][16 tokens]
//   scales [page][layer][2][kv head][page_tokens / 16]
// Both tiles are made of 16-byte pieces along the contraction of the product that reads them: K's of a token's dims, V's of a
// dim's tokens.  A piece goes to its place in the tensor cores' K-major operand with one copy (K codes as they are, as int8; V
// codes as bf16 or f16), pieces that follow one another are read by lanes that do, and an append writes whole pieces.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace qb {

constexpr int kKvBlock = 16;          // tokens that share a scale
constexpr int kKvMaxSeqs = 8192;      // rows of the page table
constexpr int kKvMaxPages = 1 << 20;  // pages of the pool

enum KvType : int { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };

struct KvView {
    int8_t* codes;
    float* scales;
    int* refs;   // [n_pages] sequences that use the page (0: free)
    int* table;  // [max_seqs][max_pages] page of positions k * page_tokens .., -1: none
    int* lens;   // [max_seqs]
    unsigned* status;
    int n_layers, n_kv, hd, pt, pt_shift;
    int n_pages, max_seqs, max_pages;

    __host__ __device__ size_t tile() const { return size_t(pt) * hd; }                         // codes of (page, layer, K or V, head)
    __host__ __device__ size_t page_codes() const { return size_t(n_layers) * 2 * n_kv * tile(); }
    __host__ __device__ int page_scales() const { return n_layers * 2 * n_kv * (pt / kKvBlock); }
    // tile number of (page, layer, K or V, head): codes at * tile(), scales at * (pt / 16)
    __host__ __device__ size_t at(int page, int layer, int kind, int head) const {
        return ((size_t(page) * n_layers + layer) * 2 + kind) * n_kv + head;
    }
};

// Tokens [starts[j], starts[j + 1]) of a call belong to sequence seqs[j] (device arrays, n sequences, n_tok tokens).
struct KvCall {
    const int* seqs;
    const int* starts;
    int n, n_tok;
};

// k, v: token t, head h, dim d at t * stride + h * hd + d (elements of the type).  max_new bounds a sequence's tokens.
cudaError_t launch_kv_append(const KvView& c, int layer, const void* k, const void* v, KvType type, long long k_stride,
                             long long v_stride, const KvCall& call, int max_new, cudaStream_t st);
// Values of positions first[j] + i of sequence seqs[j] into rows starts[j] + i of k_out, v_out [n_tok][n_kv][hd].
cudaError_t launch_kv_read(const KvView& c, int layer, const int* first, const KvCall& call, void* k_out, void* v_out,
                           KvType type, cudaStream_t st);

// Page operations; ws: kv_page_ws_bytes(c) bytes.
size_t kv_page_ws_bytes(const KvView& c);
cudaError_t launch_kv_reserve(const KvView& c, const int* seqs, const int* extra, int n, void* ws, cudaStream_t st);
cudaError_t launch_kv_fork(const KvView& c, const int* src, const int* dst, int n, void* ws, cudaStream_t st);
// Sequence seqs[i] becomes what seqs[i - i % group + parents[i]] was (kv_reorder_ws_bytes(c) bytes of ws).
size_t kv_reorder_ws_bytes(const KvView& c);
cudaError_t launch_kv_reorder(const KvView& c, const int* seqs, const int* parents, int n, int group, void* ws, cudaStream_t st);
cudaError_t launch_kv_free(const KvView& c, const int* seqs, int n, cudaStream_t st);
cudaError_t launch_kv_compact(const KvView& c, void* ws, cudaStream_t st);
cudaError_t launch_kv_copy(const KvView& c, const int* src, const int* dst, int n, cudaStream_t st);

struct KvAttnArgs {
    const void* q;  // token t, head h, dim d at t * q_stride + h * hd + d
    long long q_stride;
    void* out;      // [n_tok][n_heads][hd]
    float* lse;     // [n_tok][n_heads] or null
    KvType type;    // of q and out
    int layer, n_heads, group;
    int window;  // 0: none, else below max_pages * pt
    float scale;
    int max_q, max_len;  // host bounds: queries of a sequence, length of a sequence
};
// Workspace of a call (0: none needed); n_tok and the bounds as in the call.
size_t kv_attn_ws_bytes(const KvView& c, const KvAttnArgs& a, const KvCall& call);
cudaError_t launch_kv_attention(const KvView& c, const KvAttnArgs& a, const KvCall& call, void* ws, cudaStream_t st);

}  // namespace qb
