// tokens_fast.cpp -- the ordinary calls of tensorium_b200/tokens.py without its checks' and
// allocations' cost in Python: a decoding step's kernels take 4 to 10 us, the same call through Python and ctypes
// 10 to 18 us of host time, through here 5 to 7. Without this extension tokens.py does the same through ctypes.
//
// Each function takes (context handle, device, the context's stream, tensors and numbers) and returns its result,
// the library's negative status as an int, or None for anything that is not plain: wrong types, shapes or
// devices, strides, another current stream. tokens.py then goes its own way, which also says what is wrong. No
// arithmetic is done here: every function is one call of the C ABI.
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/tensorium_b200.h"

#include <initializer_list>

namespace {

int64_t elem(const at::Tensor& t) {
    switch (t.scalar_type()) {
    case at::kFloat: return TB_F32;
    case at::kBFloat16: return TB_BF16;
    case at::kHalf: return TB_F16;
    default: return -1;
    }
}

// A call's context: the first three arguments.
struct Call {
    tb_ctx* ctx = nullptr;
    int64_t device = -1;
    bool ok = false;
    explicit Call(PyObject* const* a) {
        if (!PyLong_Check(a[0]) || !PyLong_Check(a[1]) || !PyLong_Check(a[2])) return;
        ctx = static_cast<tb_ctx*>(PyLong_AsVoidPtr(a[0]));
        device = PyLong_AsLongLong(a[1]);
        const void* stream = PyLong_AsVoidPtr(a[2]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return;
        }
        ok = ctx && device >= 0 && c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream() == stream;
    }
    // a plain tensor of this GPU, or null
    const at::Tensor* tensor(PyObject* o) const {
        if (!THPVariable_CheckExact(o)) return nullptr;
        const at::Tensor& t = THPVariable_Unpack(o);
        return t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided ? &t : nullptr;
    }
    const at::Tensor* matrix(PyObject* o) const {
        const at::Tensor* t = tensor(o);
        return t && t->dim() == 2 && (t->stride(1) == 1 || t->size(1) <= 1) ? t : nullptr;
    }
    // n contiguous values; *ok is cleared where they are not
    const void* vector(PyObject* o, at::ScalarType type, int64_t n, bool* good) const {
        const at::Tensor* t = tensor(o);
        if (!t || t->scalar_type() != type || t->dim() != 1 || t->size(0) != n || (n > 1 && t->stride(0) != 1)) {
            *good = false;
            return nullptr;
        }
        return t->data_ptr();
    }
    const void* vector_or_none(PyObject* o, at::ScalarType type, int64_t n, bool* good) const {
        return o == Py_None ? nullptr : vector(o, type, n, good);
    }
};

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }
int64_t pitch(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (row_stride(t) + 15) / 16 * 16; }

bool whole(PyObject* o, int64_t* v) {
    if (!PyLong_CheckExact(o)) return false;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

PyObject* none() { Py_RETURN_NONE; }

template <typename F> PyObject* guarded(F&& f) {  // no C++ exception leaves through Python's C frames
    try {
        return f();
    } catch (const std::exception&) {
        return none();  // allocation failures and the like: tokens.py meets, and reports, them again
    }
}

// (handle, device, stream, x, w, w_scales, bias or None, activation) -> y
PyObject* int8_connected(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 8) return none();
    return guarded([&]() -> PyObject* {
        const Call c(a);
        if (!c.ok) return none();
        const at::Tensor *x = c.matrix(a[3]), *w = c.matrix(a[4]);
        int64_t act;
        if (!x || !w || elem(*x) < 0 || w->scalar_type() != at::kChar || x->size(1) != w->size(1) || !whole(a[7], &act)) return none();
        const int64_t m = x->size(0), k = x->size(1), ch = w->size(0);
        bool good = true;
        const void* scales = c.vector(a[5], at::kFloat, ch, &good);
        const void* bias = c.vector_or_none(a[6], at::kFloat, ch, &good);
        if (!good) return none();
        at::Tensor y = at::empty({m, ch}, x->options());
        const int rc = tb_int8_connected_fwd(c.ctx, m, ch, k, x->data_ptr(), elem(*x), row_stride(*x), static_cast<const int8_t*>(w->data_ptr()),
                                             pitch(*w), static_cast<const float*>(scales), static_cast<const float*>(bias), act, y.data_ptr(),
                                             elem(y), ch);
        return rc < 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(y));
    });
}

// (handle, device, stream, logits, tokens or None, top, temperature) -> (stats, top_logprobs or None, top_tokens or None)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7) return none();
    return guarded([&]() -> PyObject* {
        const Call c(a);
        if (!c.ok) return none();
        const at::Tensor* l = c.matrix(a[3]);
        int64_t top;
        if (!l || elem(*l) < 0 || !whole(a[5], &top) || !PyFloat_CheckExact(a[6])) return none();
        const int64_t rows = l->size(0), vocab = l->size(1);
        if (top < 0 || top > vocab) return none();
        bool good = true;
        const void* tokens = c.vector_or_none(a[4], at::kLong, rows, &good);
        if (!good) return none();
        at::Tensor stats = at::empty({5, rows}, l->options().dtype(at::kFloat)), lp, tok;
        if (top) {
            lp = at::empty({rows, top}, stats.options());
            tok = at::empty({rows, top}, l->options().dtype(at::kLong));
        }
        float* s = stats.data_ptr<float>();
        const int rc = tb_token_logprobs_fwd(c.ctx, rows, vocab, l->data_ptr(), elem(*l), row_stride(*l), static_cast<const int64_t*>(tokens),
                                             (float)PyFloat_AS_DOUBLE(a[6]), top, s, s + rows, s + 2 * rows, s + 3 * rows, s + 4 * rows,
                                             top ? lp.data_ptr<float>() : nullptr, top ? tok.data_ptr<int64_t>() : nullptr);
        if (rc < 0) return PyLong_FromLong(rc);
        PyObject* r = PyTuple_New(3);
        if (!r) return nullptr;
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(stats)));
        PyTuple_SET_ITEM(r, 1, top ? THPVariable_Wrap(std::move(lp)) : none());
        PyTuple_SET_ITEM(r, 2, top ? THPVariable_Wrap(std::move(tok)) : none());
        return r;
    });
}

// (handle, device, stream, logits, tokens or None, stats, grad_logprobs or None, grad_entropy or None, temperature) -> gradient
PyObject* token_logprobs_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 9) return none();
    return guarded([&]() -> PyObject* {
        const Call c(a);
        if (!c.ok) return none();
        const at::Tensor *l = c.matrix(a[3]), *stats = c.matrix(a[5]);
        if (!l || !stats || elem(*l) < 0 || !PyFloat_CheckExact(a[8])) return none();
        const int64_t rows = l->size(0), vocab = l->size(1);
        if (stats->scalar_type() != at::kFloat || stats->size(0) != 5 || stats->size(1) != rows || !stats->is_contiguous()) return none();
        if (a[6] != Py_None && a[4] == Py_None) return none();
        bool good = true;
        const void* tokens = c.vector_or_none(a[4], at::kLong, rows, &good);
        const void* gl = c.vector_or_none(a[6], at::kFloat, rows, &good);
        const void* gh = c.vector_or_none(a[7], at::kFloat, rows, &good);
        if (!good) return none();
        at::Tensor d = at::empty({rows, vocab}, l->options());
        const float* s = stats->data_ptr<float>();
        const int rc = tb_token_logprobs_bwd(c.ctx, rows, vocab, l->data_ptr(), elem(*l), row_stride(*l), static_cast<const int64_t*>(tokens),
                                             (float)PyFloat_AS_DOUBLE(a[8]), s + 3 * rows, s + 4 * rows, s + rows, static_cast<const float*>(gl),
                                             static_cast<const float*>(gh), d.data_ptr(), vocab);
        return rc < 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(d));
    });
}

PyMethodDef methods[] = {
    {"int8_connected", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(int8_connected)), METH_FASTCALL, nullptr},
    {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(token_logprobs)), METH_FASTCALL, nullptr},
    {"token_logprobs_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(token_logprobs_backward)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tokens_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tokens_fast() { return PyModule_Create(&module); }
