// The host side of the per-token operators (aimet_b200.int4, aimet_b200.kv_cache) for arguments that need no
// preparation: checks, output from torch's allocator, one call of the C ABI.  A decode step makes a few of these
// calls per layer, and from Python the checks, the allocation and ctypes cost two to three times the launch.
//
// Every function returns None for whatever is not its plain case (a layout that has to be copied, an argument
// that has to be refused, another device than the current one): the Python code then does the work or
// raises.  So this file decides nothing and can be left out.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/aimet_b200.h"

namespace {

decltype(&aimet_b200_int4_linear) g_linear;
decltype(&aimet_b200_kv_append) g_append;
decltype(&aimet_b200_kv_gather) g_gather;
decltype(&aimet_b200_kv_attention) g_attention;
decltype(&aimet_b200_kv_attention_scratch_bytes) g_scratch;

int code_of(at::ScalarType t) {
    return t == at::kFloat ? AB_F32 : t == at::kHalf ? AB_F16 : t == at::kBFloat16 ? AB_BF16 : -1;
}
// a plain tensor on the current device `index` that autograd does not have to follow, backwards or forwards; else nullptr
const at::Tensor *plain(PyObject *o, int64_t index) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != index) return nullptr;
    if (t.requires_grad() && c10::GradMode::is_enabled()) return nullptr;
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()) return nullptr;
    return &t;
}
const at::Tensor *lengths(PyObject *o, int64_t index, int64_t n) {
    const at::Tensor *t = plain(o, index);
    return t && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && (n <= 1 || t->stride(0) == 1) ? t : nullptr;
}
const at::Tensor *block_table(PyObject *o, int64_t index, int64_t n) {
    const at::Tensor *t = plain(o, index);
    return t && t->scalar_type() == at::kInt && t->dim() == 2 && t->size(0) == n && (t->size(1) <= 1 || t->stride(1) == 1) ? t : nullptr;
}
// [sequences, tokens, heads, dim] with the last dim contiguous, nothing empty
bool tokens4(const at::Tensor *t, int64_t dim) {
    return t && t->dim() == 4 && t->size(3) == dim && t->stride(3) == 1 && t->numel() > 0 && code_of(t->scalar_type()) >= 0;
}
void *current_stream(int64_t index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }
bool current(int64_t index) { return c10::cuda::current_device() == index; }
int64_t integer(PyObject *o) { return (int64_t)PyLong_AsLongLong(o); }
void *address(PyObject *o) { return PyLong_AsVoidPtr(o); }

// A refusal of the C ABI, and an allocation that fails, are left to the Python code, which does the same again and raises.
#define BODY_BEGIN try {
#define BODY_END                                \
    }                                           \
    catch (const std::exception &) {            \
        if (PyErr_Occurred()) return nullptr;   \
        Py_RETURN_NONE;                         \
    }

PyObject *init(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 5) return PyErr_Format(PyExc_TypeError, "init: five addresses");
    g_linear = (decltype(g_linear))address(a[0]);
    g_append = (decltype(g_append))address(a[1]);
    g_gather = (decltype(g_gather))address(a[2]);
    g_attention = (decltype(g_attention))address(a[3]);
    g_scratch = (decltype(g_scratch))address(a[4]);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// linear(input, bias, descriptor, index, status)
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    BODY_BEGIN
    if (n != 5) return PyErr_Format(PyExc_TypeError, "linear: 5 arguments");
    const auto *w = static_cast<const ab_int4_weight *>(address(a[2]));
    const int64_t index = integer(a[3]);
    auto *status = static_cast<volatile int32_t *>(address(a[4]));
    const at::Tensor *x = plain(a[0], index);
    if (!x || !current(index) || x->dim() < 1 || x->size(-1) != w->k || x->numel() == 0 || !x->is_contiguous()) Py_RETURN_NONE;
    const int code = code_of(x->scalar_type());
    const int64_t tokens = x->numel() / w->k;
    if (code < 0 || *status) Py_RETURN_NONE;
    const void *bias = nullptr;
    if (a[1] != Py_None) {
        const at::Tensor *b = plain(a[1], index);
        if (!b || b->scalar_type() != x->scalar_type() || b->dim() != 1 || b->size(0) != w->n || !b->is_contiguous()) Py_RETURN_NONE;
        bias = b->data_ptr();
    }
    // what the tensor-core kernel would read unaligned is copied first
    at::Tensor padded;
    int64_t pitch = w->k;
    if (tokens > 16 && code != AB_F32 && (w->k % 8 || reinterpret_cast<uintptr_t>(x->data_ptr()) % 16)) {
        pitch = (w->k + 7) / 8 * 8;
        padded = at::empty({tokens, pitch}, x->options().requires_grad(false));
        padded.narrow(1, 0, w->k).copy_(x->detach().view({tokens, w->k}));
        x = &padded;
    }
    const at::Tensor &input = THPVariable_Unpack(a[0]);
    c10::SmallVector<int64_t, 6> shape(input.sizes().begin(), input.sizes().end());
    shape.back() = w->n;
    at::Tensor y = at::empty(shape, x->options().requires_grad(false));
    if (g_linear(w, x->data_ptr(), pitch, bias, y.data_ptr(), w->n, tokens, code, const_cast<int32_t *>(status), current_stream(index)) != AB_OK)
        Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
    BODY_END
}

// append(key, value, table, context, new or None, descriptor, index)
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    BODY_BEGIN
    if (n != 7) return PyErr_Format(PyExc_TypeError, "append: 7 arguments");
    const auto *c = static_cast<const ab_kv_cache *>(address(a[5]));
    const int64_t index = integer(a[6]);
    const at::Tensor *k = plain(a[0], index), *v = plain(a[1], index);
    if (!tokens4(k, c->head_dim) || !tokens4(v, c->head_dim) || !current(index) || k->scalar_type() != v->scalar_type() ||
        k->sizes() != v->sizes() || k->size(2) != c->num_heads)
        Py_RETURN_NONE;
    const int64_t seqs = k->size(0);
    const at::Tensor *t = block_table(a[2], index, seqs), *ctx = lengths(a[3], index, seqs);
    const at::Tensor *len = a[4] == Py_None ? nullptr : lengths(a[4], index, seqs);
    if (!t || !ctx || (a[4] != Py_None && !len)) Py_RETURN_NONE;
    if (g_append(c, k->data_ptr(), v->data_ptr(), k->strides().data(), v->strides().data(), seqs, k->size(1),
                 static_cast<const int32_t *>(t->data_ptr()), t->stride(0), t->size(1), static_cast<const int32_t *>(ctx->data_ptr()),
                 len ? static_cast<const int32_t *>(len->data_ptr()) : nullptr, code_of(k->scalar_type()), current_stream(index)) != AB_OK)
        Py_RETURN_NONE;
    Py_RETURN_TRUE;
    BODY_END
}

// gather(table, lens, length (-1: the table's), dtype code, descriptor, index)
PyObject *gather(PyObject *, PyObject *const *a, Py_ssize_t n) {
    BODY_BEGIN
    if (n != 6) return PyErr_Format(PyExc_TypeError, "gather: 6 arguments");
    const auto *c = static_cast<const ab_kv_cache *>(address(a[4]));
    const int64_t index = integer(a[5]);
    int64_t length = integer(a[2]);
    const int code = (int)integer(a[3]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor *l = plain(a[1], index);
    if (!l || l->dim() != 1 || l->size(0) == 0 || !current(index)) Py_RETURN_NONE;
    const int64_t seqs = l->size(0);
    const at::Tensor *t = block_table(a[0], index, seqs);
    if (!t || !lengths(a[1], index, seqs)) Py_RETURN_NONE;
    if (length < 0) length = t->size(1) * c->page_size;
    if (length == 0) Py_RETURN_NONE;
    const auto options = l->options().dtype(code == AB_F32 ? at::kFloat : code == AB_F16 ? at::kHalf : at::kBFloat16);
    at::Tensor k = at::empty({seqs, length, c->num_heads, c->head_dim}, options), v = at::empty({seqs, length, c->num_heads, c->head_dim}, options);
    if (g_gather(c, k.data_ptr(), v.data_ptr(), seqs, length, static_cast<const int32_t *>(t->data_ptr()), t->stride(0), t->size(1),
                 static_cast<const int32_t *>(l->data_ptr()), code, current_stream(index)) != AB_OK)
        Py_RETURN_NONE;
    PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v)), *both = PyTuple_Pack(2, pk, pv);
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return both;
    BODY_END
}

// attention(query, table, context, lens or None, causal, window, scale, return_lse, descriptor, index)
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    BODY_BEGIN
    if (n != 10) return PyErr_Format(PyExc_TypeError, "attention: 10 arguments");
    const auto *c = static_cast<const ab_kv_cache *>(address(a[8]));
    const int64_t index = integer(a[9]);
    const at::Tensor *q = plain(a[0], index);
    if (!tokens4(q, c->head_dim) || !current(index) || q->size(2) % c->num_heads) Py_RETURN_NONE;
    const int64_t seqs = q->size(0), tokens = q->size(1), heads = q->size(2), group = heads / c->num_heads;
    const at::Tensor *t = block_table(a[1], index, seqs), *ctx = lengths(a[2], index, seqs);
    const at::Tensor *len = a[3] == Py_None ? nullptr : lengths(a[3], index, seqs);
    if (!t || !ctx || (a[3] != Py_None && !len)) Py_RETURN_NONE;
    const int causal = PyObject_IsTrue(a[4]), with_lse = PyObject_IsTrue(a[7]);  // (-1 with an error set)
    const int64_t window = integer(a[5]);
    const double scale = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred()) return nullptr;
    const int code = code_of(q->scalar_type());
    const int64_t need = g_scratch(c, seqs, tokens, group, t->size(1), code);
    if (need < 0) Py_RETURN_NONE;
    const auto options = q->options().requires_grad(false);
    at::Tensor out = at::empty({seqs, tokens, heads, q->size(3)}, options), lse, part;
    if (with_lse) lse = at::empty({seqs, tokens, heads}, options.dtype(at::kFloat));
    // scratch from the caching allocator, call by call: buffers of two streams, or of two captured graphs, are never shared
    if (need) part = at::empty({need}, options.dtype(at::kByte));
    if (g_attention(c, q->data_ptr(), q->strides().data(), out.data_ptr(), with_lse ? static_cast<float *>(lse.data_ptr()) : nullptr, seqs, tokens,
                    group, static_cast<const int32_t *>(t->data_ptr()), t->stride(0), t->size(1),
                    static_cast<const int32_t *>(ctx->data_ptr()), len ? static_cast<const int32_t *>(len->data_ptr()) : nullptr, causal, window,
                    scale, code, need ? part.data_ptr() : nullptr, need, current_stream(index)) != AB_OK)
        Py_RETURN_NONE;
    PyObject *po = THPVariable_Wrap(std::move(out));
    if (!with_lse) return po;
    PyObject *pl = THPVariable_Wrap(std::move(lse)), *both = PyTuple_Pack(2, po, pl);
    Py_XDECREF(po);
    Py_XDECREF(pl);
    return both;
    BODY_END
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(init), METHOD(linear), METHOD(append), METHOD(gather), METHOD(attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
