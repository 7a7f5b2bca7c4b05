// The operators on torch tensors as a CPython extension: argument checks, output tensors and the call of the C ABI
// (include/quanta_b200.h) in a microsecond or two of host time, which is what a call on a few rows costs next to its launch
// (through ctypes and torch's Python calls 8 to 12 us).  quanta_b200.py has the functions' documentation.  Every function works on
// torch's current stream and returns its result, or a negative QNT_ERR_* as an int; wrong types raise TypeError, more tokens than an
// int counts ValueError, tensors that would be written in place although a gradient is recorded through them RuntimeError.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/core/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <mutex>

#include "quanta_b200.h"

namespace {

struct Refused {
    PyObject* type;
    const char* message;
};
[[noreturn]] void refuse(const char* message) { throw Refused{PyExc_TypeError, message}; }

const at::Tensor* tensor_or_null(PyObject* o) { return o != Py_None && THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int dtype_of(const at::Tensor& t) {  // -1: none of ours
    switch (t.scalar_type()) {
        case at::kFloat: return QNT_F32;
        case at::kHalf: return QNT_F16;
        case at::kBFloat16: return QNT_BF16;
        default: return -1;
    }
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, at::Device device) {
    return at::Tensor(at::detail::empty_cuda(size, type, device, std::nullopt));
}

// A tensor that a call writes in place.  The operators have no gradients, so none may be recorded through it; and what autograd has
// saved of it learns that it is stale (written()).
void will_write(const at::Tensor& t) {
    if ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined())
        throw Refused{PyExc_RuntimeError, "a tensor that requires a gradient cannot be written in place (no gradient is recorded)"};
}
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* pair(PyObject* a, PyObject* b) {
    PyObject* t = a && b ? PyTuple_Pack(2, a, b) : nullptr;
    Py_XDECREF(a);
    Py_XDECREF(b);
    return t;
}

// Runs f between Python and C++: exceptions become Python's.
template <class F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(e.type, e.message);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

bool arguments(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return false;
}

bool to_double(PyObject* o, double* v) {
    *v = PyFloat_AsDouble(o);
    return !(*v == -1. && PyErr_Occurred());
}
bool to_long(PyObject* o, long long* v) {
    *v = PyLong_AsLongLong(o);
    return !(*v == -1 && PyErr_Occurred());
}

// A call of the C ABI without Python's lock: a launch waits while a thousand others are queued before it, and what those wait for may
// be another of Python's threads.  Calls of several launches that share a workspace stay in one piece (between_calls).
std::mutex between_calls;
template <class... P, class... A>
int unlocked(bool several, int (*call)(P...), A... args) {
    PyThreadState* state = PyEval_SaveThread();
    if (several) between_calls.lock();
    const int rc = call(args...);
    if (several) between_calls.unlock();
    PyEval_RestoreThread(state);
    return rc;
}

// A size or a number as the C ABI takes it; what does not fit becomes one that the C ABI refuses.
int narrow(int64_t n) { return n > INT32_MAX ? INT32_MAX : n < INT32_MIN ? INT32_MIN : int(n); }

// A count of tokens: any that fits is as good as another.
int token_count(int64_t n) {
    if (n > INT32_MAX) throw Refused{PyExc_ValueError, "at most 2147483647 tokens in one call"};
    return int(n);
}

// x, weight, eps, residual or None -> (q, d)
PyObject* rms_norm_q8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    double eps;
    if (!arguments(n_args, 4) || !to_double(a[2], &eps)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = tensor_or_null(a[0]), *w = tensor_or_null(a[1]), *r = tensor_or_null(a[3]);
        if (!x || !x->is_cuda() || dtype_of(*x) < 0 || x->dim() != 2 || x->stride(1) != 1)
            refuse("x must be a float32, float16 or bfloat16 CUDA tensor [tokens, n] whose rows are contiguous");
        const int64_t m = token_count(x->size(0)), n = x->size(1);
        if (!w || w->scalar_type() != at::kFloat || w->device() != x->device() || w->dim() != 1 || w->size(0) != n || !w->is_contiguous())
            refuse("weight must be a contiguous float32 CUDA tensor [n] on x's device");
        if (a[3] != Py_None && (!r || r->dim() != 2 || r->size(0) != m || r->size(1) != n || r->device() != x->device() || r->stride(1) != 1 ||
                                (r->scalar_type() != x->scalar_type() && r->scalar_type() != at::kFloat)))
            refuse("residual must be a CUDA tensor of x's shape, on its device, of its type or float32, whose rows are contiguous");
        if (r) will_write(*r);
        const c10::cuda::CUDAGuard on(x->device());
        at::Tensor q = empty({m, n}, at::kChar, x->device()), d = empty({m, n / 32}, at::kFloat, x->device());
        const int rc = unlocked(false, qnt_rms_norm_q8, x->const_data_ptr(), dtype_of(*x), x->stride(0), r ? r->mutable_data_ptr() : nullptr,
                                r ? dtype_of(*r) : 0, r ? r->stride(0) : 0, static_cast<const float*>(w->const_data_ptr()), float(eps), int(m),
                                narrow(n), static_cast<int8_t*>(q.mutable_data_ptr()), static_cast<float*>(d.mutable_data_ptr()),
                                c10::cuda::getCurrentCUDAStream(x->device().index()).stream());
        if (rc) return PyLong_FromLong(rc);
        if (r) written(*r);
        return pair(wrap(std::move(q)), wrap(std::move(d)));
    });
}

// q, d, dtype's number -> values
PyObject* dequantize_q8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    long long dtype;
    if (!arguments(n_args, 3) || !to_long(a[2], &dtype)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *q = tensor_or_null(a[0]), *d = tensor_or_null(a[1]);
        if (!q || !d || !q->is_cuda() || q->scalar_type() != at::kChar || q->dim() != 2 || !q->is_contiguous() ||
            d->scalar_type() != at::kFloat || d->device() != q->device() || !d->is_contiguous() || d->dim() != 2 || q->size(1) % 32 ||
            d->size(0) != q->size(0) || d->size(1) != q->size(1) / 32)
            refuse("q must be a contiguous int8 CUDA tensor [tokens, n], d a contiguous float32 one [tokens, n / 32] on its device");
        const int n_tok = token_count(q->size(0));
        const c10::cuda::CUDAGuard on(q->device());
        at::Tensor out = empty(q->sizes(), dtype == QNT_F32 ? at::kFloat : dtype == QNT_F16 ? at::kHalf : at::kBFloat16, q->device());
        const int rc = unlocked(false, qnt_dequantize_q8, static_cast<const int8_t*>(q->const_data_ptr()),
                                static_cast<const float*>(d->const_data_ptr()), n_tok, narrow(q->size(1)), out.mutable_data_ptr(), int(dtype),
                                c10::cuda::getCurrentCUDAStream(q->device().index()).stream());
        return rc ? PyLong_FromLong(rc) : wrap(std::move(out));
    });
}

// q, k or None, positions, turns, rotary_dim, interleaved, scale, inplace -> (q, k)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    long long rotary_dim, interleaved, inplace;
    double scale;
    if (!arguments(n_args, 8) || !to_long(a[4], &rotary_dim) || !to_long(a[5], &interleaved) || !to_double(a[6], &scale) ||
        !to_long(a[7], &inplace))
        return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *q = tensor_or_null(a[0]), *k = tensor_or_null(a[1]), *p = tensor_or_null(a[2]), *t = tensor_or_null(a[3]);
        if (!t || !t->is_cuda() || t->scalar_type() != at::kDouble || !t->is_contiguous() || rotary_dim < 0 || t->numel() != rotary_dim / 2)
            refuse("the table of turns must be a contiguous float64 CUDA tensor [rotary_dim / 2]");
        if (!p || p->scalar_type() != at::kInt || p->device() != t->device() || p->dim() != 1 || !p->is_contiguous())
            refuse("positions must be a contiguous int32 CUDA tensor [tokens] on the table's device");
        const auto fits = [&](const at::Tensor* x) {
            return x && x->dim() == 3 && x->stride(2) == 1 && (x->stride(1) == x->size(2) || x->size(1) == 1) && x->size(0) == p->size(0) &&
                   x->device() == t->device();
        };
        if (!fits(q) || dtype_of(*q) < 0 || (a[1] != Py_None && (!fits(k) || k->scalar_type() != q->scalar_type() || k->size(2) != q->size(2))))
            refuse("q and k must be CUDA tensors [tokens, heads, head_dim] of one type, float32, float16 or bfloat16, on the table's device, "
                   "whose heads are contiguous within a token");
        const int n_tok = token_count(p->size(0));
        if (inplace) {
            will_write(*q);
            if (k) will_write(*k);
        }
        const c10::cuda::CUDAGuard on(q->device());
        at::Tensor q_out = inplace ? *q : empty(q->sizes(), q->scalar_type(), q->device()), k_out;
        if (k) k_out = inplace ? *k : empty(k->sizes(), k->scalar_type(), k->device());
        // (of a single head the stride between heads says nothing)
        const int rc = unlocked(false, qnt_rope, q->const_data_ptr(), q->stride(0), q_out.mutable_data_ptr(), q_out.stride(0),
                                narrow(q->size(1)), k ? k->const_data_ptr() : nullptr, k ? k->stride(0) : 0,
                                k ? k_out.mutable_data_ptr() : nullptr, k ? k_out.stride(0) : 0, k ? narrow(k->size(1)) : 0, dtype_of(*q),
                                narrow(q->size(2)), narrow(rotary_dim), int(interleaved), static_cast<const double*>(t->const_data_ptr()),
                                float(scale), static_cast<const int*>(p->const_data_ptr()), n_tok,
                                c10::cuda::getCurrentCUDAStream(q->device().index()).stream());
        if (rc) return PyLong_FromLong(rc);
        if (inplace) {
            written(*q);
            if (k) written(*k);
        }
        if (!k) Py_INCREF(Py_None);
        return pair(wrap(std::move(q_out)), k ? wrap(std::move(k_out)) : Py_None);
    });
}

// logits, scores, ended or None, end_id, k, workspace -> (scores, tokens, parents)
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    long long end_id, k;
    if (!arguments(n_args, 6) || !to_long(a[3], &end_id) || !to_long(a[4], &k)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = tensor_or_null(a[0]), *s = tensor_or_null(a[1]), *e = tensor_or_null(a[2]), *ws = tensor_or_null(a[5]);
        if (!x || !x->is_cuda() || dtype_of(*x) < 0 || x->dim() != 3 || (x->stride(2) != 1 && x->size(2) != 1))
            refuse("logits must be a float32, float16 or bfloat16 CUDA tensor [groups, beams, vocab] whose rows are contiguous");
        const int64_t g = x->size(0), b = x->size(1), v = x->size(2), row = b > 1 ? x->stride(1) : x->stride(0);
        if (g > 1 && b > 1 && x->stride(0) != b * row) refuse("the rows of logits must lie at one distance from each other");
        if (!s || s->scalar_type() != at::kFloat || s->device() != x->device() || s->dim() != 2 || s->size(0) != g || s->size(1) != b ||
            !s->is_contiguous())
            refuse("scores must be a contiguous float32 CUDA tensor [groups, beams] on the logits' device");
        if (a[2] != Py_None && (!e || (e->scalar_type() != at::kBool && e->scalar_type() != at::kByte) || e->device() != x->device() ||
                                e->dim() != 2 || e->size(0) != g || e->size(1) != b || !e->is_contiguous()))
            refuse("ended must be a contiguous bool or uint8 CUDA tensor [groups, beams] on the logits' device");
        if (!ws || ws->device() != x->device() || !ws->is_contiguous()) refuse("workspace");
        const c10::cuda::CUDAGuard on(x->device());
        const int64_t width = k < 0 ? 0 : k > 64 ? 64 : k;  // (any other k is refused below)
        at::Tensor out = empty({g, width}, at::kFloat, x->device()), tokens = empty({g, width}, at::kInt, x->device()),
                   parents = empty({g, width}, at::kInt, x->device());
        const int rc = unlocked(true, qnt_beam_select, x->const_data_ptr(), dtype_of(*x), row, static_cast<const float*>(s->const_data_ptr()),
                                e ? static_cast<const uint8_t*>(e->const_data_ptr()) : nullptr, narrow(end_id), narrow(g), narrow(b),
                                narrow(v), narrow(k), static_cast<float*>(out.mutable_data_ptr()), static_cast<int*>(tokens.mutable_data_ptr()),
                                static_cast<int*>(parents.mutable_data_ptr()), ws->mutable_data_ptr(), size_t(ws->nbytes()),
                                c10::cuda::getCurrentCUDAStream(x->device().index()).stream());
        if (rc) return PyLong_FromLong(rc);
        PyObject *o = wrap(std::move(out)), *t = wrap(std::move(tokens)), *p = wrap(std::move(parents));
        PyObject* all = o && t && p ? PyTuple_Pack(3, o, t, p) : nullptr;
        Py_XDECREF(o);
        Py_XDECREF(t);
        Py_XDECREF(p);
        return all;
    });
}

// the address of a qnt_kv_cache, seqs, parents, group or None, workspace -> 0
PyObject* kv_reorder(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    long long cache, group = -1;
    if (!arguments(n_args, 5) || !to_long(a[0], &cache) || (a[3] != Py_None && !to_long(a[3], &group))) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *s = tensor_or_null(a[1]), *p = tensor_or_null(a[2]), *ws = tensor_or_null(a[4]);
        if (!ws) refuse("workspace");
        for (const at::Tensor* t : {s, p})
            if (!t || t->scalar_type() != at::kInt || t->device() != ws->device() || !t->is_contiguous())
                refuse("sequence lists must be contiguous int32 CUDA tensors on the cache's device");
        const int64_t n = s->numel();
        if (p->numel() != n) {
            PyErr_SetString(PyExc_ValueError, "one parent per sequence");
            return nullptr;
        }
        const c10::cuda::CUDAGuard on(ws->device());
        return PyLong_FromLong(unlocked(true, qnt_kv_reorder, reinterpret_cast<const qnt_kv_cache*>(intptr_t(cache)),
                                        static_cast<const int*>(s->const_data_ptr()), static_cast<const int*>(p->const_data_ptr()), narrow(n),
                                        a[3] == Py_None ? narrow(n) : narrow(group), ws->mutable_data_ptr(), size_t(ws->nbytes()),
                                        c10::cuda::getCurrentCUDAStream(ws->device().index()).stream()));
    });
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"rms_norm_q8", fast(rms_norm_q8), METH_FASTCALL, nullptr},
                         {"dequantize_q8", fast(dequantize_q8), METH_FASTCALL, nullptr},
                         {"rope", fast(rope), METH_FASTCALL, nullptr},
                         {"beam_select", fast(beam_select), METH_FASTCALL, nullptr},
                         {"kv_reorder", fast(kv_reorder), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "quanta_b200_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit_quanta_b200_torch() { return PyModule_Create(&module); }
