// The operators on torch tensors: checks of the arguments, outputs and workspaces from torch's allocator, torch's current stream, and the entry
// points of include/tatara_b200.h.  tatara_b200/ops.py documents the functions and calls these.
//
// In Python the checks, allocations and the foreign call cost 13 to 24 us of a call, several times what the kernels of a small problem take; here 2 to 5 beside
// the launches.
// Every function takes all of its arguments by position; None stands for a tensor that is not given.  Wrong arguments raise
// tatara_b200.TrainerError, what torch raises (memory) stays as it is.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <initializer_list>
#include <math.h>
#include <stdarg.h>
#include <string>

#include "../../include/tatara_b200.h"

namespace {

PyObject* g_error = nullptr;  // TrainerError

struct Refused {};
[[noreturn]] void refuse(const char* fmt, ...) {
    char text[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, text);
    throw Refused();
}

#define BODY_BEGIN HANDLE_TH_ERRORS try {
#define BODY_END                    \
    }                               \
    catch (const Refused&) {        \
        return nullptr;             \
    }                               \
    END_HANDLE_TH_ERRORS

void arguments(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) refuse("%zd arguments are needed (got %zd)", want, got);
}
int type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TB_TYPE_F32;
        case at::kHalf: return TB_TYPE_F16;
        case at::kBFloat16: return TB_TYPE_BF16;
        default: return -1;
    }
}
std::string shape_text(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + ")";
}
// a tensor whose memory does not hold its values: a negated view, or zeros without memory
void in_memory(const at::Tensor& t, const char* name) {
    if (t.is_neg() || t._is_zerotensor()) refuse("%s must hold its values in memory (resolve_neg, clone)", name);
}
const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse("%s must be a CUDA tensor", name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided) refuse("%s must be a CUDA tensor", name);
    in_memory(t, name);
    return t;
}
const at::Tensor& typed(PyObject* o, const char* name) {
    const at::Tensor& t = cuda_tensor(o, name);
    if (type_of(t) < 0) refuse("%s must be float32, float16 or bfloat16 (got %s)", name, c10::toString(t.scalar_type()));
    return t;
}
// the row stride of a [rows, n] tensor with adjacent columns
int64_t rows_of(const at::Tensor& t, const char* name) {
    if (t.dim() != 2) refuse("%s must have two dimensions (got %d)", name, (int)t.dim());
    const int64_t rows = t.size(0), n = t.size(1);
    if (n > 1 && t.stride(1) != 1) refuse("%s must have adjacent columns", name);
    if (rows <= 1) return n;
    if (t.stride(0) < n) refuse("rows of %s overlap", name);
    return t.stride(0);
}
// the address of a contiguous tensor beside `like`; NULL for None
void* vector_of(PyObject* o, const char* name, const at::Tensor& like, at::IntArrayRef shape, at::ScalarType type = at::kFloat, bool needed = false) {
    if (o == Py_None) {
        if (needed) refuse("%s must be a tensor", name);
        return nullptr;
    }
    if (!THPVariable_Check(o)) refuse("%s must be a tensor on %s", name, like.device().str().c_str());
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.device() != like.device()) refuse("%s must be on %s", name, like.device().str().c_str());
    in_memory(t, name);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous())
        refuse("%s must be a contiguous %s tensor of shape %s", name, c10::toString(type), shape_text(shape).c_str());
    return t.data_ptr();
}
at::Tensor make(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType type) { return at::detail::empty_cuda(shape, type, like.device(), std::nullopt); }
// Small results of one call from one allocation (one each costs 0.5 us): places of 128 bytes' alignment, and the tensors there.
struct Shared {
    int64_t bytes = 0;
    at::Tensor base;
    int64_t place(int64_t elements) {  // 32-bit ones
        const int64_t at = bytes;
        bytes += (elements * 4 + 127) / 128 * 128;
        return at;
    }
    void allocate(const at::Tensor& like) { base = make(like, {bytes}, at::kByte); }
    at::Tensor tensor(int64_t at, at::IntArrayRef shape, at::ScalarType type) const {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_storage_offset(at / 4);
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
        return t;
    }
};
// `out`, which has to match `like`, or a new tensor
at::Tensor output(PyObject* out, const at::Tensor& like) {
    if (out == Py_None) return make(like, like.sizes(), like.scalar_type());
    const at::Tensor& t = cuda_tensor(out, "out");
    if (t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type() || t.device() != like.device()) refuse("out must match the input");
    return t;
}
// A caller's tensor has been written: what automatic differentiation has saved of it is no longer there, as after any operation in place.
void written(PyObject* o) {
    if (o == Py_None) return;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse("%s must be a number", name);
    }
    return v;
}
int whole(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse("%s must be a whole number", name);
    }
    if (v < INT32_MIN || v > INT32_MAX) refuse("%s is out of range (got %lld)", name, v);
    return (int)v;
}
bool truth(PyObject* o, const char* name) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        refuse("%s must be a truth value", name);
    }
    return v == 1;
}
int side(int64_t v, const char* name) {
    if (v > INT32_MAX) refuse("%s is out of range (got %lld)", name, (long long)v);
    return (int)v;
}

// a tensor's device made current, and torch's stream there
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    cudaStream_t stream;
    explicit On(const at::Tensor& t) {
        guard.set_device(t.device());
        stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
    }
};
struct Work {
    at::Tensor t;
    int64_t bytes;
    Work(const at::Tensor& like, int64_t size) : bytes(size > 0 ? size : 0) {
        if (size > 0) t = make(like, {size}, at::kByte);
    }
    void* at() const { return bytes ? t.data_ptr() : nullptr; }
};
void check(int rc, const char* what, const char* err) {
    if (rc != TB_OK) refuse("%s failed (%d): %s", what, rc, err);
}

PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
    PyObject* t = PyTuple_New((Py_ssize_t)tensors.size());
    if (!t) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor& x : tensors) {
        PyObject* o = THPVariable_Wrap(x);
        if (!o) {
            Py_DECREF(t);
            return nullptr;
        }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}

// x, weight, bias, eps, out
PyObject* layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    BODY_BEGIN
    arguments(n_args, 5);
    const at::Tensor& x = typed(a[0], "x");
    const int64_t xs = rows_of(x, "x"), rows = x.size(0), n = x.size(1);
    const float* w = static_cast<float*>(vector_of(a[1], "weight", x, {n}));
    const float* b = static_cast<float*>(vector_of(a[2], "bias", x, {n}));
    const double eps = number(a[3], "eps");
    const On on(x);
    const at::Tensor y = output(a[4], x);
    Shared both;
    const int64_t mean_at = both.place(rows), rstd_at = both.place(rows);
    both.allocate(x);
    const at::Tensor mean = both.tensor(mean_at, {rows}, at::kFloat), rstd = both.tensor(rstd_at, {rows}, at::kFloat);
    char err[256];
    check(tb_layer_norm_forward(x.data_ptr(), xs, w, b, (float)eps, type_of(x), rows, side(n, "n"), y.data_ptr(), rows_of(y, "out"), mean.data_ptr<float>(),
                                rstd.data_ptr<float>(), on.stream, err, sizeof err),
          "tb_layer_norm_forward", err);
    written(a[4]);
    return tuple_of({y, mean, rstd});
    BODY_END
}

// dy, x, mean, rstd, weight, out
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    BODY_BEGIN
    arguments(n_args, 6);
    const at::Tensor &x = typed(a[1], "x"), &dy = typed(a[0], "dy");
    const int64_t xs = rows_of(x, "x"), gs = rows_of(dy, "dy"), rows = x.size(0), n = x.size(1);
    if (dy.sizes() != x.sizes() || dy.scalar_type() != x.scalar_type() || dy.device() != x.device()) refuse("dy must match x");
    const float* m = static_cast<float*>(vector_of(a[2], "mean", x, {rows}, at::kFloat, true));
    const float* r = static_cast<float*>(vector_of(a[3], "rstd", x, {rows}, at::kFloat, true));
    const float* w = static_cast<float*>(vector_of(a[4], "weight", x, {n}));
    const On on(x);
    const at::Tensor dx = output(a[5], x);
    Shared both;
    const int64_t w_at = both.place(n), b_at = both.place(n);
    both.allocate(x);
    const at::Tensor dweight = both.tensor(w_at, {n}, at::kFloat), dbias = both.tensor(b_at, {n}, at::kFloat);
    const Work work(x, tb_layer_norm_backward_workspace(rows, side(n, "n")));
    char err[256];
    check(tb_layer_norm_backward(dy.data_ptr(), gs, x.data_ptr(), xs, m, r, w, type_of(x), rows, (int)n, dx.data_ptr(), rows_of(dx, "out"),
                                 dweight.data_ptr<float>(), dbias.data_ptr<float>(), work.at(), work.bytes, on.stream, err, sizeof err),
          "tb_layer_norm_backward", err);
    written(a[5]);
    return tuple_of({dx, dweight, dbias});
    BODY_END
}

const uint8_t* mask_of(PyObject* o, const at::Tensor& like) {
    const bool bytes = o != Py_None && THPVariable_Check(o) && THPVariable_Unpack(o).scalar_type() == at::kByte;
    return static_cast<uint8_t*>(vector_of(o, "mask", like, {like.size(0)}, bytes ? at::kByte : at::kBool));
}

// logits, k, renormalise, mask
PyObject* route_forward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    BODY_BEGIN
    arguments(n_args, 4);
    const at::Tensor& x = typed(a[0], "logits");
    const int64_t stride = rows_of(x, "logits"), rows = x.size(0), experts = x.size(1);
    const int k = whole(a[1], "k");
    if (k < 1) refuse("k must be positive (got %d)", k);
    const bool renormalise = truth(a[2], "renormalise");
    const uint8_t* mask = mask_of(a[3], x);
    const On on(x);
    const at::Tensor index = make(x, {rows, k}, at::kInt), gate = make(x, {rows, k}, at::kFloat);
    Shared few;
    const int64_t counts_at = few.place(experts), n_at = few.place(1), mean_at = few.place(experts), losses_at = few.place(2);
    few.allocate(x);
    const at::Tensor counts = few.tensor(counts_at, {experts}, at::kInt), n = few.tensor(n_at, {1}, at::kInt), mean = few.tensor(mean_at, {experts}, at::kFloat),
                     losses = few.tensor(losses_at, {2}, at::kFloat);
    const Work work(x, tb_route_forward_workspace(rows, side(experts, "experts")));
    char err[256];
    check(tb_route_forward(x.data_ptr(), stride, type_of(x), rows, (int)experts, k, renormalise, mask, index.data_ptr<int>(), gate.data_ptr<float>(),
                           counts.data_ptr<int>(), n.data_ptr<int>(), mean.data_ptr<float>(), losses.data_ptr<float>(), work.at(), work.bytes, on.stream, err, sizeof err),
          "tb_route_forward", err);
    return tuple_of({index, gate, counts, n, mean, losses});
    BODY_END
}

// logits, index, gate, counts, rows, dgate, dlosses, renormalise, mask
PyObject* route_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    BODY_BEGIN
    arguments(n_args, 9);
    const at::Tensor& x = typed(a[0], "logits");
    const int64_t stride = rows_of(x, "logits"), rows = x.size(0), experts = x.size(1);
    const at::Tensor& ix = cuda_tensor(a[1], "routing.index");
    if (ix.dim() != 2) refuse("routing.index must have two dimensions");
    const int64_t k = ix.size(1);
    const int32_t* index = static_cast<int32_t*>(vector_of(a[1], "routing.index", x, {rows, k}, at::kInt, true));
    const float* gate = static_cast<float*>(vector_of(a[2], "routing.gate", x, {rows, k}, at::kFloat, true));
    const int32_t* counts = static_cast<int32_t*>(vector_of(a[3], "routing.counts", x, {experts}, at::kInt, true));
    const int32_t* n = static_cast<int32_t*>(vector_of(a[4], "routing.rows", x, {1}, at::kInt, true));
    const float* dgate = static_cast<float*>(vector_of(a[5], "dgate", x, {rows, k}));
    const float* dlosses = static_cast<float*>(vector_of(a[6], "dlosses", x, {2}));
    const bool renormalise = truth(a[7], "renormalise");
    const uint8_t* mask = mask_of(a[8], x);
    const On on(x);
    const at::Tensor out = make(x, x.sizes(), x.scalar_type());
    char err[256];
    check(tb_route_backward(x.data_ptr(), stride, type_of(x), rows, side(experts, "experts"), side(k, "k"), renormalise, mask, index, gate, dgate, counts, n, dlosses,
                            out.data_ptr(), experts, on.stream, err, sizeof err),
          "tb_route_backward", err);
    return THPVariable_Wrap(out);
    BODY_END
}

struct Matrices {
    int batch, rows, cols;
    int64_t batch_stride, stride;
};
// a [rows, cols] or [batch, rows, cols] tensor with adjacent columns
Matrices matrices_of(const at::Tensor& t, const char* name) {
    if (t.dim() != 2 && t.dim() != 3) refuse("%s must have two or three dimensions (got %d)", name, (int)t.dim());
    const int64_t rows = t.size(-2), cols = t.size(-1), batch = t.dim() == 3 ? t.size(0) : 1;
    if (rows < 1 || cols < 1) refuse("%s has no elements in a matrix", name);
    if (cols > 1 && t.stride(-1) != 1) refuse("%s must have adjacent columns", name);
    const int64_t stride = rows > 1 ? t.stride(-2) : cols;
    if (stride < cols) refuse("rows of %s overlap", name);
    return {side(batch, "batch"), side(rows, "rows"), side(cols, "cols"), batch > 1 ? t.stride(0) : 0, stride};
}
void coefficients_of(PyObject* o, float (&c)[3]) {
    PyObject* s = PySequence_Fast(o, "");
    if (!s) {
        PyErr_Clear();
        refuse("three coefficients are needed");
    }
    const bool three = PySequence_Fast_GET_SIZE(s) == 3;
    bool numbers = three;
    for (int i = 0; numbers && i < 3; ++i) {
        const double v = PyFloat_AsDouble(PySequence_Fast_GET_ITEM(s, i));
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            numbers = false;
        }
        c[i] = (float)v;
    }
    Py_DECREF(s);
    if (!three) refuse("three coefficients are needed");
    if (!numbers) refuse("coefficients must be numbers");
}

// x, steps, coefficients, eps, out
PyObject* orthogonalise(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    BODY_BEGIN
    arguments(n_args, 5);
    const at::Tensor& x = typed(a[0], "x");
    const Matrices m = matrices_of(x, "x");
    const int steps = whole(a[1], "steps");
    float c[3];
    coefficients_of(a[2], c);
    const double eps = number(a[3], "eps");
    const On on(x);
    const at::Tensor y = output(a[4], x);
    const Matrices o = matrices_of(y, "out");
    const Work work(x, tb_orthogonalise_workspace(type_of(x), m.batch, m.rows, m.cols));
    char err[256];
    check(tb_orthogonalise(x.data_ptr(), m.batch_stride, m.stride, type_of(x), m.batch, m.rows, m.cols, steps, c, (float)eps, y.data_ptr(), o.batch_stride, o.stride,
                           work.at(), work.bytes, on.stream, err, sizeof err),
          "tb_orthogonalise", err);
    written(a[4]);
    return THPVariable_Wrap(y);
    BODY_END
}

// weight, momentum, grad, weight_out, momentum_out, steps, nesterov, coefficients, eps, lr, beta, weight_decay, scale (None: by the shape), clip
PyObject* muon_step(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    BODY_BEGIN
    arguments(n_args, 14);
    const at::Tensor& w = typed(a[0], "weight");
    const Matrices m = matrices_of(w, "weight");
    const float* weight = static_cast<float*>(vector_of(a[0], "weight", w, w.sizes(), at::kFloat, true));
    const float* momentum = static_cast<float*>(vector_of(a[1], "momentum", w, w.sizes(), at::kFloat, true));
    const at::Tensor& g = typed(a[2], "grad");
    const void* grad = vector_of(a[2], "grad", w, w.sizes(), g.scalar_type(), true);
    PyObject *wo = a[3] == Py_None ? a[0] : a[3], *mo = a[4] == Py_None ? a[1] : a[4];
    float* weight_out = static_cast<float*>(vector_of(wo, "weight_out", w, w.sizes(), at::kFloat, true));
    float* momentum_out = static_cast<float*>(vector_of(mo, "momentum_out", w, w.sizes(), at::kFloat, true));
    float c[3];
    coefficients_of(a[7], c);
    tb_muon cfg;
    cfg.struct_size = (int32_t)sizeof cfg;
    cfg.steps = whole(a[5], "steps");
    cfg.nesterov = truth(a[6], "nesterov");
    cfg.a = c[0];
    cfg.b = c[1];
    cfg.c = c[2];
    cfg.eps = (float)number(a[8], "eps");
    cfg.lr = (float)number(a[9], "lr");
    cfg.beta = (float)number(a[10], "beta");
    cfg.weight_decay = (float)number(a[11], "weight_decay");
    cfg.scale = a[12] == Py_None ? (float)sqrt(fmax(1.0, (double)m.rows / m.cols)) : (float)number(a[12], "scale");
    cfg.clip = (float)number(a[13], "clip");
    const On on(w);
    const Work work(w, tb_muon_step_workspace(m.batch, m.rows, m.cols));
    char err[256];
    check(tb_muon_step(&cfg, weight, momentum, grad, type_of(g), m.batch, m.rows, m.cols, weight_out, momentum_out, work.at(), work.bytes, on.stream, err, sizeof err),
          "tb_muon_step", err);
    written(wo);
    written(mo);
    return PyTuple_Pack(2, wo, mo);
    BODY_END
}

PyObject* set_error(PyObject*, PyObject* type) {
    Py_INCREF(type);
    Py_XDECREF(g_error);
    g_error = type;
    Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FAST(layer_norm_forward), FAST(layer_norm_backward), FAST(route_forward), FAST(route_backward), FAST(orthogonalise), FAST(muon_step),
                           {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops", "the operators on torch tensors", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&g_module); }
