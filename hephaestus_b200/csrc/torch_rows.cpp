// torch_rows.cpp — the torch boundary of the row operators as a CPython module
// (hephaestus_b200/_torch_rows.so): checks the tensors, allocates the outputs
// with torch's allocator and calls the C ABI on the current torch stream.
//
// The operators of a decoding step run for a few microseconds.  The same
// checks, allocations and a ctypes call from Python take 11-19 us a call on a
// B200 host, this module 3.6-5.3 us.
//
// torch_ops.py documents the functions; their arguments here are positional.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <sstream>
#include <string>

#include "heph/heph.h"

namespace {

PyObject *g_refusal = nullptr;  // core.InvalidConfiguration
PyObject *g_check = nullptr;    // core.check

// A Python exception is set; unwinds to the module function.
struct Raised {};

[[noreturn]] void refuse(const std::string &message) {
    PyObject *error = PyObject_CallFunction(g_refusal, "s", message.c_str());
    if (error) {
        PyErr_SetObject(g_refusal, error);
        Py_DECREF(error);
    }
    throw Raised();
}

void check(heph_status status) {
    if (status == HEPH_OK) return;
    PyObject *none = PyObject_CallFunction(g_check, "i", (int)status);
    Py_XDECREF(none);
    throw Raised();
}

template <typename T> std::string text(const T &v) {
    std::ostringstream s;
    s << v;
    return s.str();
}

const char *dtype_name(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        case at::kDouble: return "torch.float64";
        default: return c10::toString(t);
    }
}

bool row_dtype(at::ScalarType t, heph_row_dtype *out) {
    if (t == at::kFloat) *out = HEPH_ROW_F32;
    else if (t == at::kBFloat16) *out = HEPH_ROW_BF16;
    else if (t == at::kHalf) *out = HEPH_ROW_F16;
    else return false;
    return true;
}

// --------------------------------------------------------------- arguments

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a torch tensor");
    return THPVariable_Unpack(o);
}
// Null for None.
const at::Tensor *maybe_tensor(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }

double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}
int64_t whole(PyObject *o, const char *name, int64_t low, int64_t high) {
    PyObject *index = PyNumber_Index(o);
    if (!index) throw Raised();
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(index, &overflow);
    Py_DECREF(index);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    if (overflow || v < low || v > high) refuse(std::string(name) + " is out of range");
    return v;
}

void check_grad(const char *name, const at::Tensor &t) {
    if (t.requires_grad() && c10::GradMode::is_enabled())
        refuse(std::string(name) + " asks for a gradient, which these calls do not record: detach it, or use torch.no_grad()");
    // A dual tensor of forward-mode differentiation, which no_grad() does not turn off (level 0 is the only one).
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
        refuse(std::string(name) + " has a tangent, which these calls do not carry: take its primal (torch.autograd.forward_ad.unpack_dual)");
}

// What the tensor holds is what its memory says.
void check_plain(const char *name, const at::Tensor &t) {
    if (t.layout() != at::kStrided || t.is_neg()) refuse(std::string(name) + " must be a strided tensor of plain values");
}

// A tensor as rows of adjacent columns.
struct Matrix {
    const void *ptr = nullptr;
    int64_t rows = 0, cols = 0, stride = 0;
};

// dtype: any row type where it is Undefined.  shape: any where it is null.
Matrix rows_of(const char *name, const at::Tensor &t, at::ScalarType dtype = at::ScalarType::Undefined,
               const at::IntArrayRef *shape = nullptr) {
    const at::ScalarType have = t.scalar_type();
    heph_row_dtype code;
    if (dtype == at::ScalarType::Undefined) {
        if (!row_dtype(have, &code)) refuse(std::string(name) + " must be f32, bf16 or f16, not " + dtype_name(have));
    } else if (have != dtype) {
        refuse(std::string(name) + " must be " + dtype_name(dtype) + ", not " + dtype_name(have));
    }
    check_plain(name, t);
    const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
    if (shape && sizes != *shape) refuse(std::string(name) + " has shape " + text(sizes) + ", not " + text(*shape));
    const int64_t dims = t.dim();
    if (dims < 2) refuse(std::string(name) + " must have rows and columns");
    Matrix m;
    m.cols = sizes[dims - 1];
    m.rows = 1;
    for (int64_t d = 0; d < dims - 1; ++d) m.rows *= sizes[d];
    if (strides[dims - 1] != 1 && m.cols > 1) refuse(std::string(name) + " must have adjacent columns");
    // Leading dimensions are one of equal distances, or are refused.
    if (m.rows > 1 && m.cols > 0) {
        int64_t upto = 1;  // rows that the dimensions seen so far make
        for (int64_t d = dims - 2; d >= 0; --d) {
            if (sizes[d] == 1) continue;
            if (upto == 1) m.stride = strides[d];
            else if (strides[d] != m.stride * upto) refuse(std::string(name) + " has leading dimensions that do not form rows at equal distances");
            upto *= sizes[d];
        }
    }
    if (m.rows <= 1) m.stride = m.cols;  // one row: as good as contiguous
    check_grad(name, t);
    m.ptr = t.const_data_ptr();
    return m;
}

const void *vector_of(const char *name, const at::Tensor &t, int64_t length, std::initializer_list<at::ScalarType> dtypes) {
    bool known = false;
    for (const at::ScalarType d : dtypes) known = known || t.scalar_type() == d;
    if (!known) {
        std::string names;
        for (const at::ScalarType d : dtypes) names += (names.empty() ? "" : " or ") + std::string(dtype_name(d));
        refuse(std::string(name) + " must be " + names + ", not " + dtype_name(t.scalar_type()));
    }
    check_plain(name, t);
    if (t.dim() != 1 || t.size(0) != length || (t.stride(0) != 1 && length > 1))
        refuse(std::string(name) + " must be a vector of " + std::to_string(length) + " adjacent elements");
    check_grad(name, t);
    return t.const_data_ptr();
}

// The CUDA device of all operands (null: absent).
int device_of(std::initializer_list<const at::Tensor *> operands) {
    int at = -1;
    for (const at::Tensor *t : operands) {
        if (!t) continue;
        if (!t->is_cuda()) refuse("hephaestus_b200.torch_ops needs CUDA tensors");
        if (at >= 0 && t->get_device() != at) refuse("operands are on different devices");
        at = (int)t->get_device();
    }
    return at;
}

heph_stream stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

at::Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, int device) {
    return at::Tensor(at::detail::empty_cuda(shape, dtype, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt));
}

// The leading dimensions of t, and `last` columns.
c10::SmallVector<int64_t, 6> with_columns(const at::Tensor &t, int64_t last) {
    c10::SmallVector<int64_t, 6> shape(t.sizes().begin(), t.sizes().end());
    shape.back() = last;
    return shape;
}

PyObject *one(const at::Tensor &t) { return THPVariable_Wrap(t); }

PyObject *tuple(std::initializer_list<const at::Tensor *> tensors) {
    PyObject *out = PyTuple_New((Py_ssize_t)tensors.size());
    if (!out) throw Raised();
    Py_ssize_t i = 0;
    for (const at::Tensor *t : tensors) {
        PyObject *v = t ? THPVariable_Wrap(*t) : Py_NewRef(Py_None);
        if (!v) {
            Py_DECREF(out);
            throw Raised();
        }
        PyTuple_SET_ITEM(out, i++, v);
    }
    return out;
}

// --------------------------------------------------------------- operators

struct NormOperands {
    Matrix x, other;
    const void *weight = nullptr;
    heph_row_dtype dtype, weight_dtype;
    int device;
};

// other: the residual, or the gradient of the norm; null where there is none.
NormOperands norm_operands(const char *name, const at::Tensor &x, const at::Tensor *weight, const char *other_name,
                           const at::Tensor *other, const at::Tensor *third = nullptr) {
    NormOperands o;
    o.x = rows_of(name, x);
    row_dtype(x.scalar_type(), &o.dtype);
    o.weight_dtype = o.dtype;
    const at::IntArrayRef shape = x.sizes();
    if (other) o.other = rows_of(other_name, *other, x.scalar_type(), &shape);
    if (weight) {
        o.weight = vector_of("weight", *weight, o.x.cols, {x.scalar_type(), at::kFloat});
        row_dtype(weight->scalar_type(), &o.weight_dtype);
    }
    if (third) rows_of("dsum", *third, x.scalar_type(), &shape);
    o.device = device_of({&x, other, weight, third});
    return o;
}

// rms_norm(x, weight, eps, residual)
PyObject *rms_norm(PyObject *const *args) {
    const at::Tensor &x = tensor(args[0], "x");
    const at::Tensor *weight = maybe_tensor(args[1], "weight"), *residual = maybe_tensor(args[3], "residual");
    const double eps = number(args[2]);
    const NormOperands o = norm_operands("x", x, weight, "residual", residual);
    at::Tensor y = empty(x.sizes(), x.scalar_type(), o.device), s;
    if (residual) s = empty(x.sizes(), x.scalar_type(), o.device);
    check(heph_rms_norm(o.device, o.dtype, o.x.ptr, o.x.stride, residual ? o.other.ptr : nullptr, o.other.stride, o.weight,
                        o.weight_dtype, eps, o.x.rows, o.x.cols, y.data_ptr(), residual ? s.data_ptr() : nullptr,
                        stream_of(o.device)));
    return residual ? tuple({&y, &s}) : one(y);
}

// rms_norm_fp8(x, weight, eps, residual, group)
PyObject *rms_norm_fp8(PyObject *const *args) {
    const at::Tensor &x = tensor(args[0], "x");
    const at::Tensor *weight = maybe_tensor(args[1], "weight"), *residual = maybe_tensor(args[3], "residual");
    const double eps = number(args[2]);
    int64_t group = 0;
    if (args[4] != Py_None) {
        group = whole(args[4], "group", INT64_MIN, INT64_MAX);
        if (group < 16 || group > (1 << 30) || (group & (group - 1))) refuse("group must be a power of two of 16 or more");
    }
    const NormOperands o = norm_operands("x", x, weight, "residual", residual);
    const int64_t groups = group ? std::max<int64_t>(1, (o.x.cols + group - 1) / group) : 1;
    at::Tensor q = empty(x.sizes(), at::kFloat8_e4m3fn, o.device), scales = empty(with_columns(x, groups), at::kFloat, o.device), s;
    if (residual) s = empty(x.sizes(), x.scalar_type(), o.device);
    check(heph_rms_norm_fp8(o.device, o.dtype, o.x.ptr, o.x.stride, residual ? o.other.ptr : nullptr, o.other.stride, o.weight,
                            o.weight_dtype, eps, o.x.rows, o.x.cols, (uint32_t)group, (uint8_t *)q.data_ptr(),
                            (float *)scales.data_ptr(), residual ? s.data_ptr() : nullptr, stream_of(o.device)));
    return residual ? tuple({&q, &scales, &s}) : tuple({&q, &scales});
}

// rms_norm_backward(dy, s, weight, eps, dsum)
PyObject *rms_norm_backward(PyObject *const *args) {
    const at::Tensor &dy = tensor(args[0], "dy"), &s = tensor(args[1], "s");
    const at::Tensor *weight = maybe_tensor(args[2], "weight"), *dsum = maybe_tensor(args[4], "dsum");
    const double eps = number(args[3]);
    const NormOperands o = norm_operands("s", s, weight, "dy", &dy, dsum);
    const Matrix d = dsum ? rows_of("dsum", *dsum, s.scalar_type()) : Matrix();
    at::Tensor ds = empty(s.sizes(), s.scalar_type(), o.device), dw, work;
    uint64_t bytes = 0;
    if (weight) {
        check(heph_rms_norm_backward_workspace(o.device, o.x.rows, o.x.cols, &bytes));
        work = empty({(int64_t)bytes}, at::kByte, o.device);
        dw = empty({o.x.cols}, weight->scalar_type(), o.device);
    }
    check(heph_rms_norm_backward(o.device, o.dtype, o.other.ptr, o.other.stride, o.x.ptr, o.x.stride, d.ptr, d.stride, o.weight,
                                 o.weight_dtype, eps, o.x.rows, o.x.cols, ds.data_ptr(), weight ? dw.data_ptr() : nullptr,
                                 weight ? work.data_ptr() : nullptr, bytes, stream_of(o.device)));
    return tuple({&ds, weight ? &dw : nullptr});
}

heph_route_score route_score(PyObject *o) {
    const char *name = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    PyErr_Clear();
    if (name && !strcmp(name, "softmax")) return HEPH_ROUTE_SOFTMAX;
    if (name && !strcmp(name, "sigmoid")) return HEPH_ROUTE_SIGMOID;
    refuse("unknown routing score" + (name ? " '" + std::string(name) + "'" : std::string()));
}

// Before the numbers become 32-bit ones of the C ABI.
void check_choice(const char *op, int64_t k, int64_t experts) {
    if (experts < 1 || experts > 1024 || k < 1 || k > 32 || k > experts)
        refuse(std::string(op) + " chooses 1 to 32 of up to 1024 experts, not " + std::to_string(k) + " of " + std::to_string(experts));
}

// route_experts(logits, k, score, bias, groups, groups_kept, group_top, renormalize, scale)
PyObject *route_experts(PyObject *const *args) {
    const at::Tensor &logits = tensor(args[0], "logits");
    const at::Tensor *bias = maybe_tensor(args[3], "bias");
    const heph_route_score score = route_score(args[2]);
    const Matrix m = rows_of("logits", logits);
    heph_row_dtype dtype;
    row_dtype(logits.scalar_type(), &dtype);
    const int64_t k = whole(args[1], "k", INT64_MIN, INT64_MAX);
    check_choice("route_experts", k, m.cols);
    const void *b = bias ? vector_of("bias", *bias, m.cols, {at::kFloat}) : nullptr;
    const uint32_t groups = (uint32_t)whole(args[4], "groups", 0, UINT32_MAX), kept = (uint32_t)whole(args[5], "groups_kept", 0, UINT32_MAX);
    const uint32_t top = (uint32_t)whole(args[6], "group_top", 0, UINT32_MAX);
    const int renormalize = PyObject_IsTrue(args[7]);
    if (renormalize < 0) throw Raised();
    const double scale = number(args[8]);
    const int device = device_of({&logits, bias});
    const auto shape = with_columns(logits, k);
    at::Tensor weights = empty(shape, at::kFloat, device), picks = empty(shape, at::kInt, device);
    check(heph_route_experts(device, dtype, m.ptr, m.stride, (const float *)b, m.rows, (uint32_t)m.cols, (uint32_t)k, score,
                             groups, kept, top, renormalize, (float)scale, (float *)weights.data_ptr(),
                             (int32_t *)picks.data_ptr(), stream_of(device)));
    return tuple({&weights, &picks});
}

// route_experts_backward(dweights, logits, experts, score, renormalize, scale)
PyObject *route_experts_backward(PyObject *const *args) {
    const at::Tensor &dweights = tensor(args[0], "dweights"), &logits = tensor(args[1], "logits"), &experts = tensor(args[2], "experts");
    const heph_route_score score = route_score(args[3]);
    const Matrix m = rows_of("logits", logits);
    heph_row_dtype dtype;
    row_dtype(logits.scalar_type(), &dtype);
    if (experts.dim() != logits.dim()) refuse("experts must have the logits' leading dimensions");
    check_choice("route_experts_backward", experts.size(-1), m.cols);
    const auto shape = with_columns(logits, experts.size(-1));
    const at::IntArrayRef want(shape);
    const Matrix g = rows_of("dweights", dweights, at::kFloat, &want), p = rows_of("experts", experts, at::kInt, &want);
    const int renormalize = PyObject_IsTrue(args[4]);
    if (renormalize < 0) throw Raised();
    const double scale = number(args[5]);
    const int device = device_of({&logits, &dweights, &experts});
    at::Tensor dlogits = empty(logits.sizes(), logits.scalar_type(), device);
    check(heph_route_experts_backward(device, dtype, (const float *)g.ptr, g.stride, m.ptr, m.stride, (const int32_t *)p.ptr,
                                      p.stride, m.rows, (uint32_t)m.cols, (uint32_t)p.cols, score, renormalize, (float)scale,
                                      dlogits.data_ptr(), stream_of(device)));
    return one(dlogits);
}

// expert_order(experts, num_experts)
PyObject *expert_order(PyObject *const *args) {
    const at::Tensor &experts = tensor(args[0], "experts");
    if (experts.scalar_type() != at::kInt) refuse(std::string("experts must be torch.int32, not ") + dtype_name(experts.scalar_type()));
    check_plain("experts", experts);
    if (!experts.is_contiguous()) refuse("experts must be contiguous");
    const int64_t num = whole(args[1], "num_experts", INT64_MIN, INT64_MAX);
    if (num < 1 || num > 1024) refuse("expert_order takes 1 to 1024 experts, not " + std::to_string(num));
    const int device = device_of({&experts});
    const int64_t count = experts.numel();
    at::Tensor offsets = empty({num + 1}, at::kInt, device), order = empty({count}, at::kInt, device);
    at::Tensor slot = empty(experts.sizes(), at::kInt, device), work;
    uint64_t bytes = 0;
    check(heph_expert_order_workspace((uint64_t)count, (uint32_t)num, &bytes));
    if (bytes) work = empty({(int64_t)bytes}, at::kByte, device);
    check(heph_expert_order(device, (const int32_t *)experts.const_data_ptr(), (uint64_t)count, (uint32_t)num,
                            (int32_t *)offsets.data_ptr(), (int32_t *)order.data_ptr(), (int32_t *)slot.data_ptr(),
                            bytes ? work.data_ptr() : nullptr, bytes, stream_of(device)));
    return tuple({&offsets, &order, &slot});
}

// One number, or a tensor of one per row.
struct Setting {
    const at::Tensor *t = nullptr;
    const void *rows = nullptr;
    double all = 0.0;
    Setting(PyObject *o, const char *name, int64_t count, at::ScalarType dtype) {
        if (THPVariable_Check(o)) {
            t = &THPVariable_Unpack(o);
            rows = vector_of(name, *t, count, {dtype});
        } else if (dtype == at::kInt) {
            all = (double)whole(o, name, INT32_MIN, INT32_MAX);
        } else {
            all = number(o);
        }
    }
};

// sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)
PyObject *sample_tokens(PyObject *const *args) {
    const at::Tensor &logits = tensor(args[0], "logits"), &uniform = tensor(args[1], "uniform");
    const Matrix m = rows_of("logits", logits);
    heph_row_dtype dtype;
    row_dtype(logits.scalar_type(), &dtype);
    if (logits.dim() != 2 || !m.cols || m.cols > UINT32_MAX) refuse("logits must be [rows, vocabulary]");
    const void *u = vector_of("uniform", uniform, m.rows, {at::kFloat});
    const Setting t(args[2], "temperature", m.rows, at::kFloat), k(args[3], "top_k", m.rows, at::kInt);
    const Setting p(args[4], "top_p", m.rows, at::kFloat), least(args[5], "min_p", m.rows, at::kFloat);
    const int device = device_of({&logits, &uniform, t.t, k.t, p.t, least.t});
    at::Tensor tokens = empty({m.rows}, at::kLong, device), probs = empty({m.rows}, at::kFloat, device);
    check(heph_sample_tokens(device, dtype, m.ptr, m.stride, m.rows, (uint32_t)m.cols, (const float *)u, (const float *)t.rows,
                             t.all, (const int32_t *)k.rows, (int32_t)k.all, (const float *)p.rows, p.all,
                             (const float *)least.rows, least.all, (int64_t *)tokens.data_ptr(), (float *)probs.data_ptr(),
                             stream_of(device)));
    return tuple({&tokens, &probs});
}

// ------------------------------------------------------------------ module

template <PyObject *(*F)(PyObject *const *), int N> PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != N) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, count);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Raised &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

template <PyObject *(*F)(PyObject *const *), int N> PyMethodDef method(const char *name) {
    return {name, (PyCFunction)(void (*)())entry<F, N>, METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<rms_norm, 4>("rms_norm"),
                           method<rms_norm_fp8, 5>("rms_norm_fp8"),
                           method<rms_norm_backward, 5>("rms_norm_backward"),
                           method<route_experts, 9>("route_experts"),
                           method<route_experts_backward, 6>("route_experts_backward"),
                           method<expert_order, 2>("expert_order"),
                           method<sample_tokens, 6>("sample_tokens"),
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_rows", "torch boundary of the row operators", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_rows(void) {
    PyObject *core = PyImport_ImportModule("hephaestus_b200.core");
    if (!core) return nullptr;
    g_refusal = PyObject_GetAttrString(core, "InvalidConfiguration");
    g_check = PyObject_GetAttrString(core, "check");
    Py_DECREF(core);
    if (!g_refusal || !g_check) return nullptr;
    return PyModule_Create(&g_module);
}
