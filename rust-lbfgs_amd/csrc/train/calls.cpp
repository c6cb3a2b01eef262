// rust-lbfgs_amd/csrc/train/calls.cpp -- the ordinary calls of losses.py and directions.py as one native function each.
//
// A small batch is done in less time on the GPU than Python takes to check seven tensors, allocate three and go through ctypes.  The host's
// side of a call, of which a launch is 3 us: log-probabilities 5.3 us (11.3 in Python), preference 6.0 (11.4), policy 7.0 (12.5).  These functions take the arguments as Python has them, and where every tensor is as the operator
// wants it -- dense, of the right type and shape, on the current device -- they allocate the results, call include/lbfgs_train.h and return
// the results.  For anything else they return None and have done nothing: the caller then goes through its own checks and copies, which
// also say what is wrong.  A whole number is the status of a refused call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/lbfgs_train.h"

namespace {

#ifndef LBFGS_TRAIN_CALLS_BUILD_ID
#define LBFGS_TRAIN_CALLS_BUILD_ID "unstamped"
#endif
extern "C" __attribute__((used, visibility("default"))) const char lbfgs_train_calls_id[] = "LBFGS_TRAIN_CALLS_BUILD_ID=" LBFGS_TRAIN_CALLS_BUILD_ID;

// the library's functions and torch's current stream, from bind()
struct Library {
    decltype(&lbfgs_train_token_logprobs_workspace) logprobs_workspace;
    decltype(&lbfgs_train_token_logprobs) logprobs;
    decltype(&lbfgs_train_token_logprobs_grad) logprobs_grad;
    decltype(&lbfgs_train_sequences_workspace) sequences_workspace;
    decltype(&lbfgs_train_preference) preference;
    decltype(&lbfgs_train_policy) policy;
    decltype(&lbfgs_train_orthogonalize_workspace) orthogonalize_workspace;
    decltype(&lbfgs_train_orthogonalize) orthogonalize;
    PyObject* stream;
} L;

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kDouble: return LBFGS_TRAIN_F64;
        case at::kFloat: return LBFGS_TRAIN_F32;
        case at::kBFloat16: return LBFGS_TRAIN_BF16;
        case at::kHalf: return LBFGS_TRAIN_F16;
        default: return -1;
    }
}
at::ScalarType wide(at::ScalarType t) { return t == at::kDouble ? at::kDouble : at::kFloat; }

// a tensor as the kernels want it, or NULL: dense, plain (no subclass that has a say in what happens to it), with its sign applied and
// without a forward-mode derivative
const at::Tensor* tensor(PyObject* o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || !t.is_contiguous() || t.is_neg() || t.key_set().has(c10::DispatchKey::Python) || t._fw_grad(0).defined())
        return nullptr;
    return &t;
}
const at::Tensor* floating(PyObject* o) {
    const at::Tensor* t = tensor(o);
    return t && type_of(t->scalar_type()) >= 0 ? t : nullptr;
}
bool like(const at::Tensor* t, const at::Tensor& what, at::ScalarType type, at::IntArrayRef sizes) {
    return t && t->scalar_type() == type && t->device() == what.device() && t->sizes() == sizes;
}
bool number(PyObject* o, double* v) {
    if (PyFloat_Check(o)) {
        *v = PyFloat_AS_DOUBLE(o);
        return true;
    }
    if (!PyLong_CheckExact(o)) return false;
    *v = PyLong_AsDouble(o);
    if (*v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
bool whole(PyObject* o, int64_t* v) {
    if (!PyLong_CheckExact(o)) return false;
    int over;
    *v = PyLong_AsLongLongAndOverflow(o, &over);
    return !over;
}
// the current stream of the tensors' device, if that is the current one
bool stream_of(const at::Tensor& t, void** stream) {
    const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
    if (guard.getDevice().index() != t.device().index()) return false;
    PyObject* index = PyLong_FromLong(t.device().index());
    PyObject* s = index ? PyObject_CallOneArg(L.stream, index) : nullptr;
    Py_XDECREF(index);
    if (s) *stream = PyLong_AsVoidPtr(s);
    Py_XDECREF(s);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
at::Tensor make(const at::Tensor& like_, at::IntArrayRef sizes, at::ScalarType type) { return at::empty(sizes, at::TensorOptions().device(like_.device()).dtype(type)); }
struct Workspace {
    at::Tensor t;
    void* data = nullptr;
    uint64_t bytes;
    Workspace(const at::Tensor& like_, uint64_t bytes_) : bytes(bytes_) {
        if (bytes) t = make(like_, {(int64_t)bytes}, at::kByte), data = t.data_ptr();
    }
};
template <class F>
int without_lock(F f) {  // (a full queue makes a launch wait: not the other threads of Python)
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = f();
    Py_END_ALLOW_THREADS return rc;
}
template <class... T>
PyObject* results(int rc, T&&... t) {
    if (rc) return PyLong_FromLong(rc);
    PyObject* out = PyTuple_New(sizeof...(T));
    if (!out) return nullptr;
    Py_ssize_t k = 0;
    bool whole_ = true;
    auto add = [&](at::Tensor&& x) {
        PyObject* o = THPVariable_Wrap(std::move(x));
        whole_ &= o != nullptr;
        PyTuple_SET_ITEM(out, k++, o);
    };
    (add(std::move(t)), ...);
    if (whole_) return out;
    Py_DECREF(out);
    return nullptr;
}
// what torch throws -- no memory, above all -- as it would have come through torch's own functions
template <class F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const c10::OutOfMemoryError& e) {
        PyObject *torch = PyImport_ImportModule("torch"), *type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        PyErr_Clear();
        PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
bool arguments(Py_ssize_t have, Py_ssize_t want) {
    if (have != want) PyErr_Format(PyExc_TypeError, "%zd arguments, %zd are taken", have, want);
    return have == want;
}

bool rows_of(const at::Tensor* x, const at::Tensor* y, int64_t ignore, lbfgs_train_rows* r) {
    if (!x || !y || x->dim() < 1 || x->size(-1) < 1 || y->scalar_type() != at::kLong || y->device() != x->device() || y->sizes() != x->sizes().slice(0, x->dim() - 1)) return false;
    const int64_t v = x->size(-1);
    *r = {x->data_ptr(), (const int64_t*)y->data_ptr(), type_of(x->scalar_type()), 0, 1, y->numel(), v, 0, v, ignore};
    return true;
}
at::DimVector pairs_of(const at::Tensor& y) {
    at::DimVector sizes(y.sizes().begin(), y.sizes().end());
    sizes.push_back(2);
    return sizes;
}

// logprobs(logits, targets, temperature, ignore_index) -> (logps, lse)
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 4)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = floating(a[0]), *y = tensor(a[1]);
        double tau;
        int64_t ignore;
        lbfgs_train_rows r;
        void* s;
        if (!number(a[2], &tau) || !whole(a[3], &ignore) || !rows_of(x, y, ignore, &r) || !stream_of(*x, &s)) Py_RETURN_NONE;
        at::Tensor logps = make(*x, y->sizes(), wide(x->scalar_type())), lse = make(*x, pairs_of(*y), at::kDouble);
        const Workspace w(*x, L.logprobs_workspace(r.dtype, r.inner, r.vocab));
        const int rc = without_lock([&] { return L.logprobs(&r, tau, logps.data_ptr(), (double*)lse.data_ptr(), w.data, w.bytes, s); });
        return results(rc, std::move(logps), std::move(lse));
    });
}
// logprobs_grad(logits, targets, lse, grad, temperature, ignore_index) -> (dlogits,)
PyObject* logprobs_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 6)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = floating(a[0]), *y = tensor(a[1]), *lse = tensor(a[2]), *g = tensor(a[3]);
        double tau;
        int64_t ignore;
        lbfgs_train_rows r;
        void* s;
        if (!number(a[4], &tau) || !whole(a[5], &ignore) || !rows_of(x, y, ignore, &r) || !like(lse, *x, at::kDouble, pairs_of(*y)) ||
            !like(g, *x, wide(x->scalar_type()), y->sizes()) || !stream_of(*x, &s))
            Py_RETURN_NONE;
        at::Tensor out = make(*x, x->sizes(), x->scalar_type());
        const int rc = without_lock([&] { return L.logprobs_grad(&r, tau, (const double*)lse->data_ptr(), g->data_ptr(), out.data_ptr(), s); });
        return results(rc, std::move(out));
    });
}

// The sequences of a call, its offsets and mask; others: tensors like logps, NULL where there is none.
bool sequences_of(const at::Tensor* x, PyObject* offsets, PyObject* mask, lbfgs_train_sequences* q) {
    if (!x) return false;
    const at::Tensor *o = nullptr, *m = nullptr;
    if (offsets != Py_None) {
        o = tensor(offsets);
        if (!o || o->device() != x->device() || (o->scalar_type() != at::kInt && o->scalar_type() != at::kLong) || o->dim() != 1 || o->size(0) < 2 || x->dim() != 1) return false;
    } else if (x->dim() != 2 || x->size(0) < 1) {
        return false;
    }
    if (mask != Py_None) {
        m = tensor(mask);
        if (!like(m, *x, at::kBool, x->sizes())) return false;
    }
    *q = {o ? o->data_ptr() : nullptr, m ? (const uint8_t*)m->data_ptr() : nullptr, !o ? 0 : o->scalar_type() == at::kInt ? 32 : 64, type_of(x->scalar_type()), x->numel(),
          o ? o->size(0) - 1 : x->size(0)};
    return true;
}
// a tensor of the type and shape of x, or None: *t is left NULL
bool another(PyObject* o, const at::Tensor& x, const at::Tensor** t) {
    if (o == Py_None) return true;
    *t = tensor(o);
    return like(*t, x, x.scalar_type(), x.sizes());
}
const void* data(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// preference(logps, ref_logps, offsets, mask, beta, label_smoothing, kind, normalize_lengths) -> (f, rewards, grad); WIDE: the gradient in
// the wide type
template <bool WIDE>
PyObject* preference(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 8)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = floating(a[0]), *ref = nullptr;
        lbfgs_train_sequences q;
        double beta, smoothing;
        int64_t kind;
        void* s;
        if (!sequences_of(x, a[2], a[3], &q) || !another(a[1], *x, &ref) || !number(a[4], &beta) || !number(a[5], &smoothing) || !whole(a[6], &kind) || !PyBool_Check(a[7]) ||
            !stream_of(*x, &s))
            Py_RETURN_NONE;
        const bool normalize = a[7] == Py_True;
        at::Tensor f = make(*x, {}, wide(x->scalar_type())), rewards = make(*x, {q.count}, wide(x->scalar_type())), grad = make(*x, x->sizes(), WIDE ? wide(x->scalar_type()) : x->scalar_type());
        if (WIDE) q.dtype |= LBFGS_TRAIN_WIDE_GRAD;
        const Workspace w(*x, L.sequences_workspace(q.tokens, q.count));
        const int rc = without_lock([&] {
            return L.preference(&q, x->data_ptr(), data(ref), beta, smoothing, (int32_t)kind, normalize, f.data_ptr(), rewards.data_ptr(), grad.data_ptr(), w.data, w.bytes, s);
        });
        return results(rc, std::move(f), std::move(rewards), std::move(grad));
    });
}
// policy(logps, old_logps, advantages, ref_logps, offsets, mask, clip_low, clip_high, kl_coef, by_sequence) -> (f, kl, clip_fraction, grad)
template <bool WIDE>
PyObject* policy(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 10)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor *x = floating(a[0]), *old = nullptr, *adv = tensor(a[2]), *ref = nullptr;
        lbfgs_train_sequences q;
        double low, high, kl_coef;
        int64_t by_sequence;
        void* s;
        if (!sequences_of(x, a[4], a[5], &q) || !another(a[1], *x, &old) || !old || !another(a[3], *x, &ref) || !number(a[6], &low) || !number(a[7], &high) ||
            !number(a[8], &kl_coef) || !whole(a[9], &by_sequence))
            Py_RETURN_NONE;
        const int64_t each[2] = {q.count, 1};
        const bool per_token = !(adv && adv->sizes() == at::IntArrayRef(each, 2));
        if (!like(adv, *x, x->scalar_type(), per_token ? x->sizes() : at::IntArrayRef(each, 2)) || (kl_coef != 0 && !ref) || !stream_of(*x, &s)) Py_RETURN_NONE;
        const at::ScalarType out = wide(x->scalar_type());
        at::Tensor f = make(*x, {}, out), kl = make(*x, {}, out), clipped = make(*x, {}, out), grad = make(*x, x->sizes(), WIDE ? out : x->scalar_type());
        if (WIDE) q.dtype |= LBFGS_TRAIN_WIDE_GRAD;
        const Workspace w(*x, L.sequences_workspace(q.tokens, q.count));
        const int rc = without_lock([&] {
            return L.policy(&q, x->data_ptr(), old->data_ptr(), data(ref), adv->data_ptr(), per_token, low, high, kl_coef, (int32_t)by_sequence, f.data_ptr(), kl.data_ptr(),
                            clipped.data_ptr(), grad.data_ptr(), w.data, w.bytes, s);
        });
        return results(rc, std::move(f), std::move(kl), std::move(clipped), std::move(grad));
    });
}
// orthogonalize(update, steps, a, b, c) -> (direction,)
PyObject* orthogonalize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 5)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor* x = floating(a[0]);
        int64_t steps;
        double p[3];
        void* s;
        if (!x || x->scalar_type() == at::kDouble || x->dim() < 2 || x->numel() == 0 || !whole(a[1], &steps) || steps < 0 || steps > 1000 || !number(a[2], p) || !number(a[3], p + 1) ||
            !number(a[4], p + 2) || !stream_of(*x, &s))
            Py_RETURN_NONE;
        const int64_t rows = x->size(-2), cols = x->size(-1), batch = x->numel() / (rows * cols);
        const int type = type_of(x->scalar_type());
        at::Tensor out = make(*x, x->sizes(), x->scalar_type());
        const Workspace w(*x, L.orthogonalize_workspace(type, batch, rows, cols));
        const int rc = without_lock([&] { return L.orthogonalize(type, batch, rows, cols, x->data_ptr(), out.data_ptr(), (int32_t)steps, p[0], p[1], p[2], w.data, w.bytes, s); });
        return results(rc, std::move(out));
    });
}

// bind(the eight functions' addresses in the order of Library, torch's current-stream function)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!arguments(n, 9)) return nullptr;
    void* f[8];
    for (int k = 0; k < 8; k++) {
        f[k] = PyLong_AsVoidPtr(a[k]);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_INCREF(a[8]);
    Py_XDECREF(L.stream);
    L = {(decltype(L.logprobs_workspace))f[0], (decltype(L.logprobs))f[1], (decltype(L.logprobs_grad))f[2], (decltype(L.sequences_workspace))f[3], (decltype(L.preference))f[4],
         (decltype(L.policy))f[5], (decltype(L.orthogonalize_workspace))f[6], (decltype(L.orthogonalize))f[7], a[8]};
    Py_RETURN_NONE;
}

#define METHOD(name, ...) {#name, (PyCFunction)(void (*)(void))__VA_ARGS__, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind, bind), METHOD(logprobs, logprobs), METHOD(logprobs_grad, logprobs_grad), METHOD(preference, preference<false>),
                         METHOD(preference_wide, preference<true>), METHOD(policy, policy<false>), METHOD(policy_wide, policy<true>),
                         METHOD(orthogonalize, orthogonalize), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "liblbfgs_train_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_liblbfgs_train_calls() { return PyModule_Create(&module); }
