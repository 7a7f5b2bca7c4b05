// extern "C" layer of the paged 8-bit KV cache (include/quanta_b200.h, qnt_kv_*): argument checks and launches.
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "quanta_b200.h"
#include "capi_util.h"
#include "kv_cache.h"

namespace {

using namespace qnt_capi;

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Checks a cache description and makes the device view; QNT_OK or an error.
int make_view(const qnt_kv_cache* c, qb::KvView* v) {
    if (!c || !c->codes || !c->scales || !c->refs || !c->table || !c->lens || !c->status)
        return set_err(QNT_ERR_INVALID, "kv cache: null array");
    if (c->n_layers <= 0 || c->n_kv_heads <= 0 || c->n_pages <= 0 || c->max_seqs <= 0 || c->max_pages <= 0)
        return set_err(QNT_ERR_INVALID, "kv cache: sizes must be positive");
    if (c->head_dim != 64 && c->head_dim != 128) return set_err(QNT_ERR_UNSUPPORTED, "kv cache: head_dim must be 64 or 128");
    const int pt = c->page_tokens;
    if (pt != 16 && pt != 32 && pt != 64 && pt != 128)
        return set_err(QNT_ERR_UNSUPPORTED, "kv cache: page_tokens must be 16, 32, 64 or 128");
    if (c->n_pages > qb::kKvMaxPages || c->max_seqs > qb::kKvMaxSeqs)
        return set_err(QNT_ERR_UNSUPPORTED, "kv cache: at most 1048576 pages and 8192 sequences");
    if ((long long)c->max_pages * pt > (1 << 30) || (long long)c->max_pages * c->max_seqs > (1 << 30) ||
        (long long)c->n_layers * c->n_kv_heads > (1 << 20))
        return set_err(QNT_ERR_UNSUPPORTED, "kv cache: page table or sequence too long");
    if (!aligned(c->codes, 16) || !aligned(c->scales, 4) || !aligned(c->refs, 4) || !aligned(c->table, 4) || !aligned(c->lens, 4) ||
        !aligned(c->status, 4))
        return set_err(QNT_ERR_INVALID, "kv cache: codes must be 16-byte aligned, the other arrays to their elements");
    v->codes = c->codes;
    v->scales = c->scales;
    v->refs = c->refs;
    v->table = c->table;
    v->lens = c->lens;
    v->status = c->status;
    v->n_layers = c->n_layers;
    v->n_kv = c->n_kv_heads;
    v->hd = c->head_dim;
    v->pt = pt;
    v->pt_shift = pt == 16 ? 4 : pt == 32 ? 5 : pt == 64 ? 6 : 7;
    v->n_pages = c->n_pages;
    v->max_seqs = c->max_seqs;
    v->max_pages = c->max_pages;
    return QNT_OK;
}

int make_type(int dtype, qb::KvType* t) {
    switch (dtype) {
        case QNT_F32: *t = qb::KV_F32; return QNT_OK;
        case QNT_F16: *t = qb::KV_F16; return QNT_OK;
        case QNT_BF16: *t = qb::KV_BF16; return QNT_OK;
    }
    return set_err(QNT_ERR_UNSUPPORTED, "dtype must be QNT_F32, QNT_F16 or QNT_BF16");
}

uintptr_t size_of(qb::KvType t) { return t == qb::KV_F32 ? 4 : 2; }

int check_layer(const qb::KvView& v, int layer) {
    return layer >= 0 && layer < v.n_layers ? QNT_OK : set_err(QNT_ERR_INVALID, "layer out of range");
}

int check_call(const qb::KvView& v, const int* seqs, const int* starts, int n, int n_tok) {
    if (n < 0 || n_tok < 0 || n > v.max_seqs) return set_err(QNT_ERR_INVALID, "bad count of sequences or tokens");
    if (n > 0 && (!seqs || !starts)) return set_err(QNT_ERR_INVALID, "null sequence list");
    if (!aligned(seqs, 4) || !aligned(starts, 4)) return set_err(QNT_ERR_INVALID, "sequence lists must be aligned to their elements");
    return QNT_OK;
}

int check_list(const qb::KvView& v, const void* a, const void* b, int n) {
    if (n < 0 || n > v.max_seqs) return set_err(QNT_ERR_INVALID, "bad count of sequences");
    if (n > 0 && (!a || !b)) return set_err(QNT_ERR_INVALID, "null sequence list");
    if (!aligned(a, 4) || !aligned(b, 4)) return set_err(QNT_ERR_INVALID, "sequence lists must be aligned to their elements");
    return QNT_OK;
}

int done(cudaError_t e, const char* what) { return e == cudaSuccess ? QNT_OK : cuda_err(e, what); }

cudaStream_t stream_of(void* s) { return static_cast<cudaStream_t>(s); }

int check_ws(const void* ws, size_t have, size_t need) {
    if (need == 0) return QNT_OK;
    if (!ws || !aligned(ws, 16) || have < need)
        return set_err(QNT_ERR_INVALID, "workspace: need " + std::to_string(need) + " bytes, 16-byte aligned");
    return QNT_OK;
}

int attn_args(const qb::KvView& v, int layer, const void* q, int dtype, long long q_stride, int n_heads, int n, int n_tok,
              int max_q, int max_len, float scale, int window, void* out, float* lse, qb::KvAttnArgs* a) {
    if (int r = check_layer(v, layer)) return r;
    if (int r = make_type(dtype, &a->type)) return r;
    if (n_heads <= 0 || n_heads > 65536 || n_heads % v.n_kv)
        return set_err(QNT_ERR_INVALID, "n_heads must be a positive multiple of n_kv_heads");
    if (max_q < 0 || max_len < 0 || window < 0 || (n_tok > 0 && n > 0 && max_q == 0))
        return set_err(QNT_ERR_INVALID, "bad max_q, max_len or window");
    if (n_tok > 0 && q_stride < (long long)n_heads * v.hd && n_tok > 1)
        return set_err(QNT_ERR_INVALID, "q_stride is smaller than a token's heads");
    if ((long long)n * v.n_kv * ((long long)v.max_pages * v.pt / 128 + 2) > 0x7fffffffLL)
        return set_err(QNT_ERR_UNSUPPORTED, "sequences x heads x longest length is too large for one call");
    a->q = q;
    a->q_stride = q_stride;
    a->out = out;
    a->lse = lse;
    a->layer = layer;
    a->n_heads = n_heads;
    a->group = n_heads / v.n_kv;
    // a window that holds every position a sequence can have is none (and sums with it stay in range)
    a->window = window >= v.max_pages * v.pt ? 0 : window;
    a->scale = scale;
    a->max_q = max_q;
    a->max_len = max_len;
    return QNT_OK;
}

}  // namespace

extern "C" {

int qnt_kv_append(const qnt_kv_cache* cache, int layer, const void* k, const void* v, int dtype, long long k_stride,
                  long long v_stride, const int* seqs, const int* starts, int n, int n_tok, int max_new, void* stream) {
    qb::KvView c;
    qb::KvType t;
    if (int r = make_view(cache, &c)) return r;
    if (int r = check_layer(c, layer)) return r;
    if (int r = make_type(dtype, &t)) return r;
    if (int r = check_call(c, seqs, starts, n, n_tok)) return r;
    if (n == 0 || n_tok == 0) return QNT_OK;
    if (!k || !v || max_new <= 0) return set_err(QNT_ERR_INVALID, "null rows or max_new <= 0");
    if (n_tok > 1 && (k_stride < (long long)c.n_kv * c.hd || v_stride < (long long)c.n_kv * c.hd))
        return set_err(QNT_ERR_INVALID, "k_stride or v_stride is smaller than a token's heads");
    if (!aligned(k, size_of(t)) || !aligned(v, size_of(t))) return set_err(QNT_ERR_INVALID, "k and v must be aligned to their elements");
    return done(qb::launch_kv_append(c, layer, k, v, t, k_stride, v_stride, qb::KvCall{seqs, starts, n, n_tok},
                                     max_new < n_tok ? max_new : n_tok, stream_of(stream)), "kv append");
}

int qnt_kv_read(const qnt_kv_cache* cache, int layer, const int* seqs, const int* first, const int* starts, int n, int n_tok,
                void* k_out, void* v_out, int dtype, void* stream) {
    qb::KvView c;
    qb::KvType t;
    if (int r = make_view(cache, &c)) return r;
    if (int r = check_layer(c, layer)) return r;
    if (int r = make_type(dtype, &t)) return r;
    if (int r = check_call(c, seqs, starts, n, n_tok)) return r;
    if (n == 0 || n_tok == 0) return QNT_OK;
    if (!first || !k_out || !v_out || !aligned(first, 4) || !aligned(k_out, 16) || !aligned(v_out, 16))
        return set_err(QNT_ERR_INVALID, "first and outputs: not null, outputs 16-byte aligned, first to its elements");
    return done(qb::launch_kv_read(c, layer, first, qb::KvCall{seqs, starts, n, n_tok}, k_out, v_out, t, stream_of(stream)),
                "kv read");
}

size_t qnt_kv_attention_workspace(const qnt_kv_cache* cache, int n_heads, int n, int n_tok, int max_q, int max_len) {
    qb::KvView c;
    size_t need = 0;
    if (make_view(cache, &c) || n < 0 || n_tok < 0 || n > c.max_seqs) return 0;
    if (n == 0 || n_tok == 0) return 0;
    for (int dtype : {QNT_F32, QNT_F16}) {  // whichever type and window the call will have: a window never needs more
        qb::KvAttnArgs a;
        if (attn_args(c, 0, nullptr, dtype, (long long)n_heads * c.hd, n_heads, n, n_tok, max_q, max_len, 1.f, 0, nullptr, nullptr, &a))
            return 0;
        const size_t b = qb::kv_attn_ws_bytes(c, a, qb::KvCall{nullptr, nullptr, n, n_tok});
        if (b > need) need = b;
    }
    return need;
}

int qnt_kv_attention(const qnt_kv_cache* cache, int layer, const void* q, int dtype, long long q_stride, int n_heads,
                     const int* seqs, const int* starts, int n, int n_tok, int max_q, int max_len, float scale, int window,
                     void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    qb::KvView c;
    qb::KvAttnArgs a;
    if (int r = make_view(cache, &c)) return r;
    if (int r = check_call(c, seqs, starts, n, n_tok)) return r;
    if (int r = attn_args(c, layer, q, dtype, q_stride, n_heads, n, n_tok, max_q, max_len, scale, window, out, lse, &a)) return r;
    if (n == 0 || n_tok == 0) return QNT_OK;
    if (!q || !out || !aligned(out, 16)) return set_err(QNT_ERR_INVALID, "null q, or out not 16-byte aligned");
    if (!aligned(q, size_of(a.type)) || !aligned(lse, 4)) return set_err(QNT_ERR_INVALID, "q and lse must be aligned to their elements");
    const qb::KvCall call{seqs, starts, n, n_tok};
    if (int r = check_ws(workspace, workspace_bytes, qb::kv_attn_ws_bytes(c, a, call))) return r;
    return done(qb::launch_kv_attention(c, a, call, workspace, stream_of(stream)), "kv attention");
}

size_t qnt_kv_page_workspace(const qnt_kv_cache* cache) {
    qb::KvView c;
    return make_view(cache, &c) ? 0 : qb::kv_page_ws_bytes(c);
}

int qnt_kv_reserve(const qnt_kv_cache* cache, const int* seqs, const int* extra, int n, void* workspace, size_t workspace_bytes,
                   void* stream) {
    qb::KvView c;
    if (int r = make_view(cache, &c)) return r;
    if (int r = check_list(c, seqs, extra, n)) return r;
    if (int r = check_ws(workspace, workspace_bytes, qb::kv_page_ws_bytes(c))) return r;
    return done(qb::launch_kv_reserve(c, seqs, extra, n, workspace, stream_of(stream)), "kv reserve");
}

int qnt_kv_fork(const qnt_kv_cache* cache, const int* src, const int* dst, int n, void* workspace, size_t workspace_bytes,
                void* stream) {
    qb::KvView c;
    if (int r = make_view(cache, &c)) return r;
    if (int r = check_list(c, src, dst, n)) return r;
    if (int r = check_ws(workspace, workspace_bytes, qb::kv_page_ws_bytes(c))) return r;
    return done(qb::launch_kv_fork(c, src, dst, n, workspace, stream_of(stream)), "kv fork");
}

int qnt_kv_free(const qnt_kv_cache* cache, const int* seqs, int n, void* stream) {
    qb::KvView c;
    if (int r = make_view(cache, &c)) return r;
    if (int r = check_list(c, seqs, seqs, n)) return r;
    return done(qb::launch_kv_free(c, seqs, n, stream_of(stream)), "kv free");
}

int qnt_kv_compact(const qnt_kv_cache* cache, void* workspace, size_t workspace_bytes, void* stream) {
    qb::KvView c;
    if (int r = make_view(cache, &c)) return r;
    if (int r = check_ws(workspace, workspace_bytes, qb::kv_page_ws_bytes(c))) return r;
    return done(qb::launch_kv_compact(c, workspace, stream_of(stream)), "kv compact");
}

int qnt_kv_copy(const qnt_kv_cache* cache, const int* src, const int* dst, int n, void* stream) {
    qb::KvView c;
    if (int r = make_view(cache, &c)) return r;
    if (n < 0 || n > 65535 || (n > 0 && (!src || !dst)) || !aligned(src, 4) || !aligned(dst, 4)) return set_err(QNT_ERR_INVALID, "bad page list (at most 65535 pages)");
    return done(qb::launch_kv_copy(c, src, dst, n, stream_of(stream)), "kv copy");
}

int qnt_kv_check(const qnt_kv_cache* cache, void* stream) {
    qb::KvView c;
    if (int r = make_view(cache, &c)) return r;
    unsigned bits = 0;
    cudaError_t e = cudaMemcpyAsync(&bits, c.status, sizeof bits, cudaMemcpyDeviceToHost, stream_of(stream));
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream_of(stream));
    if (e == cudaSuccess && bits) e = cudaMemsetAsync(c.status, 0, sizeof bits, stream_of(stream));
    if (e != cudaSuccess) return cuda_err(e, "qnt_kv_check");
    if (!bits) return QNT_OK;
    std::string why = "kv cache: error bits " + std::to_string(bits);
    if (bits & qb::ERR_BAD_POS) why += " (a sequence, length or page-table entry out of range)";
    if (bits & qb::ERR_CAPACITY) why += " (no free pages left)";
    if (bits & qb::ERR_WAIT_TIMEOUT) why += " (a bounded wait gave up)";
    return set_err(QNT_ERR_DEVICE, why);
}

}  // extern "C"
