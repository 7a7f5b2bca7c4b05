// extern "C" layer of the operators around a decoder layer and a beam search (include/quanta_b200.h: qnt_rms_norm_q8,
// qnt_dequantize_q8, qnt_rope, qnt_beam_*): argument checks and launches.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "quanta_b200.h"
#include "beam.h"
#include "capi_util.h"
#include "layer_ops.h"

namespace {

using namespace qnt_capi;

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int make_type(int dtype, qb::KvType* t) {
    switch (dtype) {
        case QNT_F32: *t = qb::KV_F32; return QNT_OK;
        case QNT_F16: *t = qb::KV_F16; return QNT_OK;
        case QNT_BF16: *t = qb::KV_BF16; return QNT_OK;
    }
    return set_err(QNT_ERR_UNSUPPORTED, "dtype must be QNT_F32, QNT_F16 or QNT_BF16");
}

uintptr_t size_of(qb::KvType t) { return t == qb::KV_F32 ? 4 : 2; }

using Wide = __int128;  // (strides are the caller's)

// Rows of `row` bytes, `stride` bytes from each other.
struct Rows {
    const void* at;
    Wide stride, row;
};

// Whether rows of a and of b share a byte.  Where the strides differ and there are several rows, only the first ones are compared.
bool overlap(const Rows& a, const Rows& b, int n) {
    const Wide d = Wide(reinterpret_cast<uintptr_t>(b.at)) - Wide(reinterpret_cast<uintptr_t>(a.at));
    if (d < a.row && d > -b.row) return true;
    if (n <= 1 || a.stride != b.stride) return false;
    if (d >= (n - 1) * a.stride + a.row || -d >= (n - 1) * b.stride + b.row) return false;
    // row j of b lies d + (j - i) stride behind row i of a: the largest such distance below a.row, with |j - i| < n
    const Wide room = a.row - 1 - d;
    Wide k = room / a.stride - (room < 0 && room % a.stride ? 1 : 0);
    if (k > n - 1) k = n - 1;
    return k > -Wide(n) && d + k * a.stride > -b.row;
}

int done(cudaError_t e, const char* what) { return e == cudaSuccess ? QNT_OK : cuda_err(e, what); }

cudaStream_t stream_of(void* s) { return static_cast<cudaStream_t>(s); }

int check_heads(const char* name, const qb::RopeHeads& h, int head_dim, int n_tok, uintptr_t size) {
    if (h.heads == 0) return QNT_OK;
    if (!h.in || !h.out) return set_err(QNT_ERR_INVALID, std::string("rope: null ") + name);
    if (!aligned(h.in, size) || !aligned(h.out, size)) return set_err(QNT_ERR_INVALID, std::string("rope: ") + name + " must be aligned to its elements");
    const long long row = (long long)h.heads * head_dim;
    if (n_tok > 1 && (h.in_stride < row || h.out_stride < row))
        return set_err(QNT_ERR_INVALID, std::string("rope: a stride of ") + name + " is smaller than a token's heads");
    if (h.in == h.out && h.in_stride != h.out_stride && n_tok > 1)
        return set_err(QNT_ERR_INVALID, std::string("rope: ") + name + " in place with two strides");
    return QNT_OK;
}

int beam_args(int groups, int beams, int vocab, int k, qb::BeamArgs* a) {
    if (groups < 0 || beams <= 0 || vocab <= 0 || k <= 0) return set_err(QNT_ERR_INVALID, "beam select: sizes must be positive");
    if (k > qb::kBeamMaxK || beams > 1024) return set_err(QNT_ERR_UNSUPPORTED, "beam select: at most 64 candidates and 1024 beams");
    if ((long long)beams * vocab < k) return set_err(QNT_ERR_INVALID, "beam select: fewer than k candidates");
    if (vocab > 1 << 30 || (long long)beams * vocab > 0x7fffffffLL || (long long)groups * beams * (vocab / 512 + 2) > 0x3fffffffLL)
        return set_err(QNT_ERR_UNSUPPORTED, "beam select: groups x beams x vocab is too large for one call");
    a->groups = groups;
    a->beams = beams;
    a->vocab = vocab;
    a->k = k;
    return QNT_OK;
}

}  // namespace

extern "C" {

int qnt_rms_norm_q8(const void* x, int dtype, long long x_stride, void* residual, int residual_dtype, long long residual_stride,
                    const float* weight, float eps, int n_tok, int n, int8_t* q, float* d, void* stream) {
    qb::NormQ8Args a{};
    if (int r = make_type(dtype, &a.type)) return r;
    if (n_tok < 0 || n <= 0 || n % 32) return set_err(QNT_ERR_INVALID, "rms norm: n must be a positive multiple of 32");
    if (n > qb::kNormMax) return set_err(QNT_ERR_UNSUPPORTED, "rms norm: rows of at most 32768 values");
    if (!(eps >= 0.f)) return set_err(QNT_ERR_INVALID, "rms norm: eps must not be negative");
    if (n_tok == 0) return QNT_OK;
    if (!x || !weight || !q || !d) return set_err(QNT_ERR_INVALID, "rms norm: null array");
    if (!aligned(x, size_of(a.type)) || !aligned(weight, 4) || !aligned(q, 16) || !aligned(d, 16))
        return set_err(QNT_ERR_INVALID, "rms norm: x and weight must be aligned to their elements, q and d to 16 bytes");
    if (n_tok > 1 && x_stride < n) return set_err(QNT_ERR_INVALID, "rms norm: x_stride is smaller than a row");
    if (residual) {
        if (residual_dtype != dtype && residual_dtype != QNT_F32)
            return set_err(QNT_ERR_UNSUPPORTED, "rms norm: the residual must have x's dtype or QNT_F32");
        a.residual_f32 = residual_dtype == QNT_F32;
        if (!aligned(residual, a.residual_f32 ? 4 : size_of(a.type)))
            return set_err(QNT_ERR_INVALID, "rms norm: the residual must be aligned to its elements");
        if (n_tok > 1 && residual_stride < n) return set_err(QNT_ERR_INVALID, "rms norm: residual_stride is smaller than a row");
        if (residual == x) return set_err(QNT_ERR_INVALID, "rms norm: the residual must not be x");
        const Wide xb = size_of(a.type), rb = a.residual_f32 ? 4 : xb;
        if (overlap({x, x_stride * xb, n * xb}, {residual, residual_stride * rb, n * rb}, n_tok))
            return set_err(QNT_ERR_INVALID, "rms norm: the residual must not overlap x");
    }
    a.x = x;
    a.x_stride = x_stride;
    a.residual = residual;
    a.residual_stride = residual_stride;
    a.weight = weight;
    a.eps = eps;
    a.n_tok = n_tok;
    a.n = n;
    a.q = q;
    a.d = d;
    return done(qb::launch_rms_norm_q8(a, stream_of(stream)), "rms norm");
}

int qnt_dequantize_q8(const int8_t* q, const float* d, int n_tok, int n, void* out, int dtype, void* stream) {
    qb::KvType t;
    if (int r = make_type(dtype, &t)) return r;
    if (n_tok < 0 || n <= 0 || n % 32) return set_err(QNT_ERR_INVALID, "dequantize: n must be a positive multiple of 32");
    if ((long long)n_tok * n > (1LL << 40)) return set_err(QNT_ERR_UNSUPPORTED, "dequantize: too many values for one call");
    if (n_tok == 0) return QNT_OK;
    if (!q || !d || !out || !aligned(q, 16) || !aligned(d, 4) || !aligned(out, 16))
        return set_err(QNT_ERR_INVALID, "dequantize: arrays not null, q and out 16-byte aligned, d to its elements");
    return done(qb::launch_dequantize_q8(q, d, (long long)n_tok * n, out, t, stream_of(stream)), "dequantize");
}

int qnt_rope(const void* q, long long q_stride, void* q_out, long long q_out_stride, int n_heads, const void* k, long long k_stride,
             void* k_out, long long k_out_stride, int n_kv_heads, int dtype, int head_dim, int rotary_dim, int interleaved,
             const double* turns, float scale, const int* positions, int n_tok, void* stream) {
    qb::RopeArgs a{};
    if (int r = make_type(dtype, &a.type)) return r;
    if (head_dim <= 0 || head_dim > 1024 || head_dim % 2 || rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 2)
        return set_err(QNT_ERR_INVALID, "rope: an even head_dim of at most 1024, an even rotary_dim within it");
    if (n_tok < 0 || n_heads < 0 || n_kv_heads < 0 || n_heads > 4096 || n_kv_heads > 4096)
        return set_err(QNT_ERR_INVALID, "rope: bad count of tokens or heads (at most 4096)");
    if (n_heads) a.q = qb::RopeHeads{q, q_out, q_stride, q_out_stride, n_heads};
    if (n_kv_heads) a.k = qb::RopeHeads{k, k_out, k_stride, k_out_stride, n_kv_heads};
    if (n_tok > 0) {
        if (int r = check_heads("q", a.q, head_dim, n_tok, size_of(a.type))) return r;
        if (int r = check_heads("k", a.k, head_dim, n_tok, size_of(a.type))) return r;
        const Wide b = size_of(a.type);
        const auto in = [&](const qb::RopeHeads& h) { return Rows{h.in, h.in_stride * b, h.heads * head_dim * b}; };
        const auto out = [&](const qb::RopeHeads& h) { return Rows{h.out, h.out_stride * b, h.heads * head_dim * b}; };
        const bool both = a.q.heads && a.k.heads;
        if ((both && (overlap(out(a.q), out(a.k), n_tok) || overlap(out(a.q), in(a.k), n_tok) || overlap(in(a.q), out(a.k), n_tok))) ||
            (a.q.heads && a.q.in != a.q.out && overlap(in(a.q), out(a.q), n_tok)) ||
            (a.k.heads && a.k.in != a.k.out && overlap(in(a.k), out(a.k), n_tok)))
            return set_err(QNT_ERR_INVALID, "rope: an output must not overlap the other or an input that it is not");
    }
    if (n_tok == 0 || a.q.heads + a.k.heads == 0) return QNT_OK;
    if (!turns || !positions || !aligned(turns, 8) || !aligned(positions, 4))
        return set_err(QNT_ERR_INVALID, "rope: turns and positions not null and aligned to their elements");
    a.head_dim = head_dim;
    a.rotary_dim = rotary_dim;
    a.n_tok = n_tok;
    a.positions = positions;
    a.turns = turns;
    a.scale = scale;
    a.interleaved = interleaved != 0;
    return done(qb::launch_rope(a, stream_of(stream)), "rope");
}

size_t qnt_beam_workspace(int groups, int beams, int vocab, int k) {
    qb::BeamArgs a{};
    if (beam_args(groups, beams, vocab, k, &a)) return 0;
    size_t need = 0;
    for (qb::KvType t : {qb::KV_F32, qb::KV_F16}) {  // whichever type the call will have
        a.type = t;
        const size_t b = qb::beam_ws_bytes(a);
        if (b > need) need = b;
    }
    return need;
}

int qnt_beam_select(const void* logits, int dtype, long long stride, const float* scores, const uint8_t* ended, int end_id,
                    int groups, int beams, int vocab, int k, float* out_scores, int* tokens, int* parents, void* workspace,
                    size_t workspace_bytes, void* stream) {
    qb::BeamArgs a{};
    if (int r = make_type(dtype, &a.type)) return r;
    if (int r = beam_args(groups, beams, vocab, k, &a)) return r;
    if (groups == 0) return QNT_OK;
    if (!logits || !scores || !out_scores || !tokens || !parents) return set_err(QNT_ERR_INVALID, "beam select: null array");
    if (!aligned(logits, size_of(a.type)) || !aligned(scores, 4) || !aligned(out_scores, 4) || !aligned(tokens, 4) || !aligned(parents, 4))
        return set_err(QNT_ERR_INVALID, "beam select: arrays must be aligned to their elements");
    if ((long long)groups * beams > 1 && stride < vocab) return set_err(QNT_ERR_INVALID, "beam select: stride is smaller than a row");
    if (ended && (end_id < 0 || end_id >= vocab)) return set_err(QNT_ERR_INVALID, "beam select: ended beams need an end_id within the vocabulary");
    const size_t need = qb::beam_ws_bytes(a);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
        return set_err(QNT_ERR_INVALID, "workspace: need " + std::to_string(need) + " bytes, 16-byte aligned");
    a.logits = logits;
    a.stride = stride;
    a.scores = scores;
    a.ended = ended;
    a.end_id = end_id;
    a.out_scores = out_scores;
    a.tokens = tokens;
    a.parents = parents;
    return done(qb::launch_beam_select(a, workspace, stream_of(stream)), "beam select");
}

}  // extern "C"
