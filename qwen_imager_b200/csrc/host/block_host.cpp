// The host side of a block operator's ordinary call, in C++: checks, output
// allocation and the C entry point (include/qmm_block.h).
//
// A small operator's time is the time of its call: on B200 a one-token linear
// (7.1 us on the device) took 14 us through the Python checks and ctypes.  Each function
// here takes exactly the operands that need no conversion and returns its outputs;
// for anything else (another type, device or layout, an argument error) it returns
// None, and the Python function goes its general way, which converts or raises.  A
// status other than QMM_OK is returned as an int, for the caller to raise.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "qmm_block.h"

namespace {

// Entry points of libqmm, bound once by address (the library is loaded by ctypes).
struct Entries {
    decltype(&qmm_mx4_linear) linear;
    decltype(&qmm_mx4_linear_workspace_bytes) linear_workspace;
    decltype(&qmm_mx4_quantize) quantize;
    decltype(&qmm_mx4_dequantize) dequantize;
    decltype(&qmm_qk_norm_rotary) rotary;
    decltype(&qmm_gated_residual_norm) norm;
} g;

const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// None, or a tensor; false for anything else.
bool optional_tensor(PyObject *o, const at::Tensor **out) {
    *out = nullptr;
    if (o == Py_None) return true;
    *out = tensor(o);
    return *out != nullptr;
}

int elem_of(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return QMM_ELEM_BF16;
        case at::kFloat: return QMM_ELEM_F32;
        case at::kHalf: return QMM_ELEM_F16;
        default: return -1;
    }
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    return at::detail::empty_cuda(sizes, type, device, std::nullopt);
}

void *current_stream(at::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

// x as rows of its last dimension: false unless they are evenly spaced, apart, and their columns consecutive.
struct Rows {
    int64_t rows, cols, stride;
};
bool rows_of(const at::Tensor &x, Rows *r) {
    const int64_t dim = x.dim();
    if (dim == 0) return false;
    r->cols = x.size(-1);
    if (r->cols == 0) return false;
    if (dim == 2) {
        if (x.stride(1) != 1) return false;
        r->rows = x.size(0);
        r->stride = x.stride(0);
        return r->stride >= r->cols || r->rows <= 1;
    }
    if (!x.is_contiguous()) return false;
    r->rows = x.numel() / r->cols;
    r->stride = r->cols;
    return true;
}

// On the current CUDA device.
bool here(const at::Tensor &t) { return t.is_cuda() && t.device().index() == c10::cuda::current_device(); }

PyObject *wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject *pair(at::Tensor a, at::Tensor b) {
    PyObject *x = wrap(std::move(a)), *y = wrap(std::move(b));
    PyObject *t = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}
PyObject *failed(qmm_status s) { return PyLong_FromLong(s); }

// C++ exceptions (an allocation that fails) become Python ones.
template <typename F>
PyObject *guarded(F f) {
    try {
        return f();
    } catch (const c10::OutOfMemoryError &e) {
        PyObject *torch = PyImport_ImportModule("torch"), *type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        if (type) PyErr_SetString(type, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

#define ARITY(n)                                                                              \
    if (nargs != (n)) {                                                                       \
        PyErr_Format(PyExc_TypeError, "%s takes %d arguments, not %zd", __func__, n, nargs);  \
        return nullptr;                                                                       \
    }

// mx_quantize(x) -> (codes, scales)
PyObject *mx_quantize(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    ARITY(1)
    return guarded([&]() -> PyObject * {
        const at::Tensor *x = tensor(args[0]);
        Rows r;
        if (!x || !here(*x) || elem_of(x->scalar_type()) < 0 || !rows_of(*x, &r) || r.rows == 0) Py_RETURN_NONE;
        const at::Device d = x->device();
        const int64_t blocks = (r.cols + 31) / 32;
        at::Tensor codes = empty({r.rows, blocks * 16}, at::kByte, d);
        at::Tensor scales = empty({(r.rows + 127) / 128 * ((r.cols + 255) / 256) * 1024}, at::kByte, d);
        const qmm_status s = g.quantize(x->const_data_ptr(), elem_of(x->scalar_type()), r.rows, r.cols, r.stride, codes.mutable_data_ptr<uint8_t>(),
                                        scales.mutable_data_ptr<uint8_t>(), current_stream(d));
        return s != QMM_OK ? failed(s) : pair(std::move(codes), std::move(scales));
    });
}

// mx_dequantize(codes, scales, rows, k) -> bf16 [rows, k]
PyObject *mx_dequantize(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    ARITY(4)
    return guarded([&]() -> PyObject * {
        const at::Tensor *codes = tensor(args[0]), *scales = tensor(args[1]);
        const int64_t rows = PyLong_AsLongLong(args[2]), k = PyLong_AsLongLong(args[3]);
        if (PyErr_Occurred()) return nullptr;
        if (!codes || !scales || !here(*codes) || rows <= 0) Py_RETURN_NONE;
        at::Tensor out = empty({rows, k}, at::kBFloat16, codes->device());
        const qmm_mx4 w{codes->const_data_ptr<uint8_t>(), scales->const_data_ptr<uint8_t>(), rows, k};
        const qmm_status s = g.dequantize(&w, out.mutable_data_ptr(), QMM_ELEM_BF16, current_stream(codes->device()));
        return s != QMM_OK ? failed(s) : wrap(std::move(out));
    });
}

// bf16, contiguous, n values, on the device: a vector that needs no conversion.
bool plain_vector(const at::Tensor *v, int64_t n, at::Device d) {
    return !v || (v->scalar_type() == at::kBFloat16 && v->numel() == n && v->is_contiguous() && v->device() == d);
}

// mx_linear(x, x_scales or None, codes, scales, n, k, bias, gate, residual, activation) -> y
// x: a matrix, or with x_scales the codes of an MXFP4 matrix.
PyObject *mx_linear(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    ARITY(10)
    return guarded([&]() -> PyObject * {
        const at::Tensor *x = tensor(args[0]), *xs, *codes = tensor(args[2]), *scales = tensor(args[3]), *bias, *gate, *res;
        const int64_t n = PyLong_AsLongLong(args[4]), k = PyLong_AsLongLong(args[5]);
        if (!x || !codes || !scales || !optional_tensor(args[1], &xs) || !optional_tensor(args[6], &bias) || !optional_tensor(args[7], &gate) ||
            !optional_tensor(args[8], &res))
            Py_RETURN_NONE;
        const int64_t act = PyLong_AsLongLong(args[9]);
        if (PyErr_Occurred()) return nullptr;
        const at::Device d = codes->device();
        if (x->device() != d || !here(*x)) Py_RETURN_NONE;
        qmm_mx4_linear_args a{};
        at::Tensor y, work;
        if (xs) {
            a.m = x->size(0);
            a.x_codes = x->const_data_ptr<uint8_t>();
            a.x_scales = xs->const_data_ptr<uint8_t>();
            if (a.m == 0) Py_RETURN_NONE;
            y = empty({a.m, n}, at::kBFloat16, d);
        } else {
            Rows r;
            a.x_elem = elem_of(x->scalar_type());
            if (a.x_elem < 0 || !rows_of(*x, &r) || r.cols != k || r.rows == 0) Py_RETURN_NONE;
            a.m = r.rows;
            a.x = x->const_data_ptr();
            a.x_row_stride = r.stride;
            if (x->dim() == 2) {
                y = empty({a.m, n}, at::kBFloat16, d);
            } else {
                c10::SmallVector<int64_t, 6> sizes(x->sizes().begin(), x->sizes().end());
                sizes.back() = n;
                y = empty(sizes, at::kBFloat16, d);
            }
            a.workspace_bytes = g.linear_workspace(a.m, n, k);
            if (a.workspace_bytes) {
                work = empty({(int64_t)a.workspace_bytes}, at::kByte, d);
                a.workspace = work.mutable_data_ptr();
            }
        }
        if (!plain_vector(bias, n, d) || !plain_vector(gate, n, d)) Py_RETURN_NONE;
        if (res && (!plain_vector(res, a.m * n, d) || res->size(-1) != n || reinterpret_cast<uintptr_t>(res->const_data_ptr()) % 16)) Py_RETURN_NONE;
        a.w = qmm_mx4{codes->const_data_ptr<uint8_t>(), scales->const_data_ptr<uint8_t>(), n, k};
        auto bits = [](const at::Tensor *t) { return t ? static_cast<const uint16_t *>(t->const_data_ptr()) : nullptr; };
        a.bias = bits(bias);
        a.gate = bits(gate);
        a.residual = bits(res);
        a.y = static_cast<uint16_t *>(y.mutable_data_ptr());
        a.activation = (int32_t)act;
        const qmm_status s = g.linear(&a, current_stream(d));
        return s != QMM_OK ? failed(s) : wrap(std::move(y));
    });
}

// qk_norm_rotary(q, k or None, positions, turns, axis, axes, adjacent, q_weight, k_weight, eps) -> (q', k') or q'
PyObject *qk_norm_rotary(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    ARITY(10)
    return guarded([&]() -> PyObject * {
        const at::Tensor *q = tensor(args[0]), *k, *pos = tensor(args[2]), *turns = tensor(args[3]), *axis = tensor(args[4]), *qw, *kw;
        if (!q || !pos || !turns || !axis || !optional_tensor(args[1], &k) || !optional_tensor(args[7], &qw) || !optional_tensor(args[8], &kw))
            Py_RETURN_NONE;
        qmm_rotary_args a{};
        a.axes = (int32_t)PyLong_AsLong(args[5]);
        a.adjacent = (int32_t)PyLong_AsLong(args[6]);
        a.eps = (float)PyFloat_AsDouble(args[9]);
        if (PyErr_Occurred()) return nullptr;
        const at::Device d = q->device();
        const int64_t nd = q->dim();
        if (!here(*q) || (nd != 3 && nd != 4) || (a.elem = elem_of(q->scalar_type())) < 0) Py_RETURN_NONE;
        const int64_t tokens = q->size(nd - 3), dim = q->size(nd - 1), batch = nd == 4 ? q->size(0) : 1;
        if (q->stride(nd - 1) != 1 || pos->device() != d || turns->device() != d || !pos->is_contiguous() || pos->dim() != 2 || pos->size(0) != tokens ||
            pos->size(1) != a.axes || dim > 256 || 2 * turns->size(0) > dim || q->numel() == 0)
            Py_RETURN_NONE;
        switch (pos->scalar_type()) {
            case at::kInt: a.pos_kind = 0; break;
            case at::kLong: a.pos_kind = 1; break;
            case at::kFloat: a.pos_kind = 2; break;
            default: Py_RETURN_NONE;
        }
        auto weight = [&](const at::Tensor *w, const void **p) {
            *p = w ? w->const_data_ptr() : nullptr;
            return !w || (w->scalar_type() == q->scalar_type() && w->numel() == dim && w->is_contiguous() && w->device() == d);
        };
        if (!weight(qw, &a.q_weight) || !weight(kw, &a.k_weight)) Py_RETURN_NONE;
        auto strides = [&](const at::Tensor &t, int64_t (&s)[3]) {
            s[0] = nd == 4 ? t.stride(0) : 0;
            s[1] = t.stride(nd - 3);
            s[2] = t.stride(nd - 2);
        };
        at::Tensor qo = empty(q->sizes(), q->scalar_type(), d), ko;
        strides(*q, a.q_stride);
        strides(qo, a.q_out_stride);
        a.q = q->const_data_ptr();
        a.q_out = qo.mutable_data_ptr();
        a.q_heads = (int32_t)q->size(nd - 2);
        if (k) {
            if (k->dim() != nd || k->size(nd - 1) != dim || k->size(nd - 3) != tokens || (nd == 4 && k->size(0) != batch) || k->scalar_type() != q->scalar_type() ||
                k->device() != d || k->stride(nd - 1) != 1 || k->numel() == 0)
                Py_RETURN_NONE;
            ko = empty(k->sizes(), k->scalar_type(), d);
            strides(*k, a.k_stride);
            strides(ko, a.k_out_stride);
            a.k = k->const_data_ptr();
            a.k_out = ko.mutable_data_ptr();
            a.k_heads = (int32_t)k->size(nd - 2);
        }
        a.positions = pos->const_data_ptr();
        a.turns = turns->const_data_ptr<float>();
        a.axis = axis->const_data_ptr<uint8_t>();
        a.batch = batch;
        a.tokens = tokens;
        a.dim = (int32_t)dim;
        a.pairs = (int32_t)turns->size(0);
        const qmm_status s = g.rotary(&a, current_stream(d));
        if (s != QMM_OK) return failed(s);
        return k ? pair(std::move(qo), std::move(ko)) : wrap(std::move(qo));
    });
}

// gated_norm(x, branch, post, post_weight, gate, residual_scale, pre, pre_weight, scale, shift, eps, quantize, same)
//   -> (x', n) or (x', codes, scales); same: x' is x itself
PyObject *gated_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    ARITY(13)
    return guarded([&]() -> PyObject * {
        const at::Tensor *x = tensor(args[0]), *branch, *pw, *gate, *qw, *scale, *shift;
        if (!x || !optional_tensor(args[1], &branch) || !optional_tensor(args[3], &pw) || !optional_tensor(args[4], &gate) ||
            !optional_tensor(args[7], &qw) || !optional_tensor(args[8], &scale) || !optional_tensor(args[9], &shift))
            Py_RETURN_NONE;
        qmm_gated_norm_args a{};
        a.post = (int32_t)PyLong_AsLong(args[2]);
        a.residual_scale = (float)PyFloat_AsDouble(args[5]);
        a.pre = (int32_t)PyLong_AsLong(args[6]);
        a.eps = (float)PyFloat_AsDouble(args[10]);
        const int quantize = PyObject_IsTrue(args[11]), same = PyObject_IsTrue(args[12]);
        if (PyErr_Occurred()) return nullptr;
        if (a.post < 0 || a.pre < 0) Py_RETURN_NONE;
        const at::Device d = x->device();
        Rows r, rb{};
        if (!here(*x) || (a.x_elem = elem_of(x->scalar_type())) < 0 || !rows_of(*x, &r) || r.rows == 0) Py_RETURN_NONE;
        a.x = x->const_data_ptr();
        a.x_stride = r.stride;
        a.rows = r.rows;
        a.hidden = r.cols;
        if (branch) {
            if (branch->sizes() != x->sizes() || branch->device() != d || (a.branch_elem = elem_of(branch->scalar_type())) < 0 || !rows_of(*branch, &rb))
                Py_RETURN_NONE;
            a.branch = branch->const_data_ptr();
            a.branch_stride = rb.stride;
        }
        // vectors of one type, [hidden] or [groups, hidden] with the same number of groups or one
        int elem = -1;
        a.groups = 1;
        for (const at::Tensor *v : {gate, scale, shift})
            if (v && v->dim() == 2) a.groups = std::max(a.groups, v->size(0));
        if (a.groups == 0 || r.rows % a.groups) Py_RETURN_NONE;
        auto vector = [&](const at::Tensor *v, bool grouped, const void **p, int64_t *stride) {
            if (!v) return true;
            const int64_t nd = v->dim();
            if (v->device() != d || nd < 1 || nd > (grouped ? 2 : 1) || v->size(-1) != r.cols || (r.cols > 1 && v->stride(-1) != 1)) return false;
            const int e = elem_of(v->scalar_type());
            if (e < 0 || (elem >= 0 && e != elem)) return false;
            elem = e;
            if (nd == 2 && v->size(0) != 1 && v->size(0) != a.groups) return false;
            *stride = nd == 2 && v->size(0) > 1 ? v->stride(0) : 0;
            *p = v->const_data_ptr();
            return true;
        };
        int64_t none = 0;
        if (!vector(pw, false, &a.post_weight, &none) || !vector(qw, false, &a.pre_weight, &none) || !vector(gate, true, &a.gate, &a.gate_stride) ||
            !vector(scale, true, &a.scale, &a.scale_stride) || !vector(shift, true, &a.shift, &a.shift_stride))
            Py_RETURN_NONE;
        a.vec_elem = elem < 0 ? 0 : elem;
        at::Tensor xn, n, scales;
        if (same) {
            xn = *x;
        } else {
            xn = empty(x->sizes(), x->scalar_type(), d);
            a.x_out = xn.mutable_data_ptr();
            a.x_out_stride = r.cols;
        }
        if (quantize) {
            n = empty({r.rows, (r.cols + 31) / 32 * 16}, at::kByte, d);
            scales = empty({(r.rows + 127) / 128 * ((r.cols + 255) / 256) * 1024}, at::kByte, d);
            a.n_codes = n.mutable_data_ptr<uint8_t>();
            a.n_scales = scales.mutable_data_ptr<uint8_t>();
        } else {
            n = empty(x->sizes(), x->scalar_type(), d);
            a.n_out = n.mutable_data_ptr();
            a.n_out_stride = r.cols;
        }
        const qmm_status s = g.norm(&a, current_stream(d));
        if (s != QMM_OK) return failed(s);
        if (!quantize) return pair(std::move(xn), std::move(n));
        PyObject *t[3] = {wrap(std::move(xn)), wrap(std::move(n)), wrap(std::move(scales))};
        PyObject *out = t[0] && t[1] && t[2] ? PyTuple_Pack(3, t[0], t[1], t[2]) : nullptr;
        for (PyObject *o : t) Py_XDECREF(o);
        return out;
    });
}

// bind(addresses of the entry points, in the order of Entries)
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    ARITY(6)
    void *p[6];
    for (int i = 0; i < 6; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
    g = Entries{reinterpret_cast<decltype(g.linear)>(p[0]),     reinterpret_cast<decltype(g.linear_workspace)>(p[1]),
                reinterpret_cast<decltype(g.quantize)>(p[2]),   reinterpret_cast<decltype(g.dequantize)>(p[3]),
                reinterpret_cast<decltype(g.rotary)>(p[4]),     reinterpret_cast<decltype(g.norm)>(p[5])};
    Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(mx_quantize), FAST(mx_dequantize), FAST(mx_linear), FAST(qk_norm_rotary), FAST(gated_norm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_qmm_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// What this file was built from and for; the package loads no other (build.py).
#ifndef QMM_HOST_KEY
#define QMM_HOST_KEY ""
#endif

PyMODINIT_FUNC PyInit__qmm_host(void) {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "key", QMM_HOST_KEY) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
