// The host side of the float operators' calls (mamba_int.ops: add_rms_norm,
// add_rms_norm_quant, causal_conv, selective_scan, w4_matvec, sample_tokens, adapter_add,
// gated_scan): checks of the tensors, outputs, the call of the C ABI, and gated_scan's node
// of autograd, as a Python module.  Through ctypes and checks in Python a call took 9 to
// 18 us of host time, several times what its kernel takes on a decode step's rows.
//
// The entry points come as addresses (the library is loaded once, by _lib), the
// stream as its handle and device.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <stdarg.h>

#include <array>

#include "mamba_int.h"

namespace {

using at::Tensor;

decltype(&mi_add_rms_norm) g_norm;
decltype(&mi_causal_conv) g_conv;
decltype(&mi_selective_scan) g_scan;
decltype(&mi_selective_scan_workspace_size) g_scan_size;
decltype(&mi_w4_matvec) g_w4;
decltype(&mi_sample_workspace_size) g_sample_size;
decltype(&mi_sample_tokens) g_sample;
decltype(&mi_adapter_workspace_size) g_adapter_size;
decltype(&mi_adapter_add) g_adapter;
decltype(&mi_gated_scan_sizes) g_gated_sizes;
decltype(&mi_gated_scan) g_gated;
decltype(&mi_gated_scan_backward) g_gated_backward;
decltype(&mi_last_error_string) g_last_error;
PyObject *g_mi_error;   // _lib.MIError

thread_local long t_device;   // the current device: the stream's, and the one that all tensors have to be on

struct Raised {};       // a Python error is set

[[noreturn]] void raise(PyObject *type, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw Raised{};
}

void check(const char *fn, int status) {
    if (status == MI_OK) return;
    PyObject *e = PyObject_CallFunction(g_mi_error, "sis", fn, status, g_last_error());
    if (e) {
        PyErr_SetObject(g_mi_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

std::string text(at::IntArrayRef v) {
    std::string s = "(";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + ")";
}

const char *type_name(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "float32";
        case at::kBFloat16: return "bfloat16";
        case at::kHalf: return "float16";
        case at::kInt: return "int32";
        case at::kLong: return "int64";
        case at::kByte: return "uint8";
        default: return c10::toString(t);
    }
}

const Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s must be a torch.Tensor", name);
    return THPVariable_Unpack(o);
}

int float_type(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return MI_F32;
        case at::kBFloat16: return MI_BF16;
        case at::kHalf: return MI_F16;
        default: raise(PyExc_TypeError, "%s must be float32, bfloat16 or float16, got %s", name, type_name(t.scalar_type()));
    }
}

const Tensor &like(PyObject *o, at::IntArrayRef shape, at::ScalarType type, const char *name) {
    const Tensor &t = tensor(o, name);
    if (t.scalar_type() != type) raise(PyExc_TypeError, "%s must be %s, got %s", name, type_name(type), type_name(t.scalar_type()));
    if (t.sizes() != shape) raise(PyExc_ValueError, "%s must be %s, got %s", name, text(shape).c_str(), text(t.sizes()).c_str());
    if (!t.is_cuda()) raise(PyExc_ValueError, "%s must be a device tensor (libmamba_int has no host path)", name);
    if (t.device().index() != t_device)
        raise(PyExc_ValueError, "%s is on cuda:%d, but the call runs on the stream of the current device, cuda:%ld", name,
              (int)t.device().index(), t_device);
    if (t.requires_grad() && c10::GradMode::is_enabled())
        raise(PyExc_ValueError, "%s requires a gradient; the float operators are forward only", name);
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        raise(PyExc_ValueError, "%s carries a tangent; the float operators are forward only", name);
    if (t.is_neg()) raise(PyExc_ValueError, "%s is a negated view of other values; resolve_neg() makes them", name);
    return t;
}

// Rows of a tensor [rows, dim] or [batch, len, dim]: any strides between rows, the
// elements of a row adjacent; those of an output do not overlap.
struct Rows {
    void *p = nullptr;
    int64_t ld = 0, bs = 0;
};
Rows rows(PyObject *o, at::IntArrayRef shape, at::ScalarType type, const char *name, bool out = false) {
    const Tensor &t = like(o, shape, type, name);
    const auto st = t.strides();
    const int n = (int)shape.size();
    if (st[n - 1] != 1 && shape[n - 1] > 1)
        raise(PyExc_ValueError, "%s: the elements of a row must be adjacent (strides %s)", name, text(st).c_str());
    Rows r{t.data_ptr(), st[n - 2], n == 3 ? st[0] : 0};
    if (!out) return r;
    int64_t span = shape[n - 1];
    for (int i = n - 2; i >= 0; --i) {
        if (shape[i] > 1 && st[i] < span) raise(PyExc_ValueError, "%s: output rows overlap (strides %s)", name, text(st).c_str());
        span = std::max(span, st[i] * shape[i]);
    }
    // the stride of a dimension of one element is free: the library asks for a row's length
    if (shape[n - 2] <= 1) r.ld = shape[n - 1];
    if (shape[0] <= 1) r.bs = 0;
    return r;
}

// A contiguous tensor of this shape; None: NULL.
template <class T>
T *vec(PyObject *o, at::IntArrayRef shape, at::ScalarType type, const char *name) {
    if (o == Py_None) return nullptr;
    const Tensor &t = like(o, shape, type, name);
    if (!t.is_contiguous()) raise(PyExc_ValueError, "%s must be contiguous", name);
    return static_cast<T *>(t.data_ptr());
}

// The call has written a tensor that was passed in (or None): a backward pass that saved
// it has to notice.
void written(PyObject *o) {
    if (o == Py_None) return;
    const Tensor &t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject *empty(at::IntArrayRef shape, const Tensor &x, at::ScalarType type) {
    return THPVariable_Wrap(at::empty(shape, x.options().dtype(type)));
}

// `out` as a new reference, or a new tensor
PyObject *output(PyObject *out, at::IntArrayRef shape, const Tensor &x) {
    if (out == Py_None) return empty(shape, x, x.scalar_type());
    Py_INCREF(out);
    return out;
}

struct Ref {
    PyObject *p;
    explicit Ref(PyObject *o) : p(o) {
        if (!o) throw Raised{};
    }
    ~Ref() { Py_XDECREF(p); }
    PyObject *release() {
        PyObject *o = p;
        p = nullptr;
        return o;
    }
};

void count(Py_ssize_t n, Py_ssize_t want, const char *fn) {
    if (n != want) raise(PyExc_TypeError, "%s takes %zd arguments, got %zd", fn, want, n);
}
void *address(PyObject *o) {
    void *p = PyLong_AsVoidPtr(o);
    if (PyErr_Occurred()) throw Raised{};
    return p;
}
int64_t int_of(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}
// (handle of the current stream, its device)
void *stream_of(PyObject *o) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) raise(PyExc_TypeError, "the stream must be a tuple of its handle and device");
    if (at::tracer::impl::is_dispatch_enabled())
        raise(PyExc_RuntimeError, "the float operators cannot be traced: the trace would hold their results as constants");
    t_device = (long)int_of(PyTuple_GET_ITEM(o, 1));
    return address(PyTuple_GET_ITEM(o, 0));
}
int size_of(int64_t v, const char *name) {
    if (v < 0 || v > INT32_MAX) raise(PyExc_ValueError, "%s=%lld is out of range", name, (long long)v);
    return (int)v;
}

// (stream, x, weight, residual, eps, residual_out, out, unit): unit 0 returns (y,
// residual_out), else (q, scale, residual_out) with q's rows rounded up to unit.
PyObject *add_rms_norm(PyObject *const *a, Py_ssize_t n) {
    count(n, 8, "add_rms_norm");
    void *stream = stream_of(a[0]);
    const Tensor &x = tensor(a[1], "x");
    const int code = float_type(x, "x");
    if (x.dim() != 2) raise(PyExc_ValueError, "x must be [tokens, dim], got %s", text(x.sizes()).c_str());
    const int64_t T = x.size(0), d = x.size(1), unit = int_of(a[7]);
    const auto shape = x.sizes();
    const double eps = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) throw Raised{};
    at::ScalarType rtype = x.scalar_type();
    if (a[3] != Py_None)
        rtype = tensor(a[3], "residual").scalar_type();
    else if (a[5] != Py_None)
        rtype = tensor(a[5], "residual_out").scalar_type();
    if (rtype != x.scalar_type() && rtype != at::kFloat)
        raise(PyExc_TypeError, "the residual must be %s or float32, got %s", type_name(x.scalar_type()), type_name(rtype));
    const int rcode = rtype == at::kFloat ? MI_F32 : code;
    const Rows xr = rows(a[1], shape, x.scalar_type(), "x");
    const Rows rr = a[3] != Py_None ? rows(a[3], shape, rtype, "residual") : Rows{};
    const float *w = vec<float>(a[2], shape.slice(1), at::kFloat, "weight");
    Ref res(a[5] != Py_None || a[3] == Py_None ? (Py_INCREF(a[5]), a[5]) : empty(shape, x, rtype));
    const Rows ro = res.p != Py_None ? rows(res.p, shape, rtype, "residual_out", true) : Rows{};
    Rows yr;
    if (unit == 0) {
        Ref y(output(a[6], shape, x));
        yr = rows(y.p, shape, x.scalar_type(), "out", true);
        check("mi_add_rms_norm", g_norm(xr.p, code, xr.ld, rr.p, rcode, rr.ld, w, (float)eps, yr.p, yr.ld, nullptr, 0,
                                        nullptr, ro.p, ro.ld, size_of(T, "tokens"), size_of(d, "dim"), stream));
        written(a[5]);
        written(a[6]);
        return Py_BuildValue("(NN)", y.release(), res.release());
    }
    if (unit < 1) raise(PyExc_ValueError, "unit=%lld must be at least 1", (long long)unit);
    const int64_t dp = (d + unit - 1) / unit * unit;
    Ref q(empty({T, dp}, x, at::kChar)), scale(empty({T}, x, at::kFloat));
    check("mi_add_rms_norm",
          g_norm(xr.p, code, xr.ld, rr.p, rcode, rr.ld, w, (float)eps, nullptr, 0,
                 static_cast<int8_t *>(THPVariable_Unpack(q.p).data_ptr()), dp,
                 static_cast<float *>(THPVariable_Unpack(scale.p).data_ptr()), ro.p, ro.ld, size_of(T, "tokens"),
                 size_of(d, "dim"), stream));
    written(a[5]);
    return Py_BuildValue("(NNN)", q.release(), scale.release(), res.release());
}

// (stream, x, weight, bias, silu, state_in, state_out, lens, out)
PyObject *causal_conv(PyObject *const *a, Py_ssize_t n) {
    count(n, 9, "causal_conv");
    void *stream = stream_of(a[0]);
    const Tensor &x = tensor(a[1], "x");
    const int code = float_type(x, "x");
    if (x.dim() != 3) raise(PyExc_ValueError, "x must be [batch, len, dim], got %s", text(x.sizes()).c_str());
    const at::ScalarType type = x.scalar_type();
    const auto shape = x.sizes();
    const int64_t B = shape[0], L = shape[1], D = shape[2];
    if (!THPVariable_Check(a[2]) || THPVariable_Unpack(a[2]).dim() != 2)
        raise(PyExc_ValueError, "weight must be a tensor [dim, width]");
    const int64_t W = THPVariable_Unpack(a[2]).size(1);
    const Rows xr = rows(a[1], shape, type, "x");
    const float *w = vec<float>(a[2], {D, W}, at::kFloat, "weight"), *bias = vec<float>(a[3], {D}, at::kFloat, "bias");
    const int64_t st[3] = {B, W - 1, D};
    const void *si = vec<void>(a[5], st, type, "state_in");
    void *so = vec<void>(a[6], st, type, "state_out");
    const int32_t *lens = vec<int32_t>(a[7], {B}, at::kInt, "lens");
    Ref y(output(a[8], shape, x));
    const Rows yr = rows(y.p, shape, type, "out", true);
    check("mi_causal_conv", g_conv(xr.p, xr.ld, xr.bs, code, w, bias, size_of(W, "width"), (int)int_of(a[4]), si, so, lens,
                                   yr.p, yr.ld, yr.bs, size_of(B, "batch"), size_of(L, "len"), size_of(D, "dim"),
                                   stream));
    written(a[6]);
    written(a[8]);
    return y.release();
}

// b or c: [batch, len, states], or [batch, len, groups, states] with adjacent groups
Rows group_rows(PyObject *o, int64_t B, int64_t L, int64_t G, int64_t N, at::ScalarType type, const char *name) {
    if (!THPVariable_Check(o) || THPVariable_Unpack(o).dim() != 4) return rows(o, {B, L, G * N}, type, name);
    const Tensor &t = like(o, {B, L, G, N}, type, name);
    const auto st = t.strides();
    if ((G > 1 && st[2] != N) || (N > 1 && st[3] != 1))
        raise(PyExc_ValueError, "%s: the groups of a row must be adjacent (strides %s)", name, text(st).c_str());
    return {t.data_ptr(), st[1], st[0]};
}

// (stream, u, dt, a, b, c, d_skip, z, dt_bias, dt_softplus, h_in, h_out, lens, out)
PyObject *selective_scan(PyObject *const *a, Py_ssize_t n) {
    count(n, 14, "selective_scan");
    void *stream = stream_of(a[0]);
    const int softplus = PyObject_IsTrue(a[9]);
    if (softplus < 0) throw Raised{};
    const Tensor &u = tensor(a[1], "u");
    const int code = float_type(u, "u");
    if (u.dim() != 3) raise(PyExc_ValueError, "u must be [batch, len, dim], got %s", text(u.sizes()).c_str());
    const at::ScalarType type = u.scalar_type();
    const auto shape = u.sizes();
    const int64_t B = shape[0], L = shape[1], D = shape[2];
    if (!THPVariable_Check(a[3]) || THPVariable_Unpack(a[3]).dim() != 2)
        raise(PyExc_ValueError, "a must be a tensor [dim, states]");
    const int64_t N = THPVariable_Unpack(a[3]).size(1);
    const int64_t G = THPVariable_Check(a[4]) && THPVariable_Unpack(a[4]).dim() == 4 ? THPVariable_Unpack(a[4]).size(2) : 1;
    const Rows br = group_rows(a[4], B, L, G, N, type, "b"), cr = group_rows(a[5], B, L, G, N, type, "c");
    const Rows ur = rows(a[1], shape, type, "u"), tr = rows(a[2], shape, type, "dt");
    const Rows zr = a[7] != Py_None ? rows(a[7], shape, type, "z") : Rows{};
    const float *am = vec<float>(a[3], {D, N}, at::kFloat, "a"), *skip = vec<float>(a[6], {D}, at::kFloat, "d_skip"),
                *bias = vec<float>(a[8], {D}, at::kFloat, "dt_bias");
    const int64_t st[3] = {B, D, N};
    const float *h_in = vec<float>(a[10], st, at::kFloat, "h_in");
    float *h_out = vec<float>(a[11], st, at::kFloat, "h_out");
    const int32_t *lens = vec<int32_t>(a[12], {B}, at::kInt, "lens");
    Ref y(output(a[13], shape, u));
    const Rows yr = rows(y.p, shape, type, "out", true);
    const int bi = size_of(B, "batch"), li = size_of(L, "len"), di = size_of(D, "dim"), ni = size_of(N, "states"),
              gi = size_of(G, "groups");
    size_t bytes = 0;
    check("mi_selective_scan_workspace_size", g_scan_size(bi, li, di, ni, gi, &bytes));
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, u.options().dtype(at::kByte));
    check("mi_selective_scan",
          g_scan(ur.p, ur.ld, ur.bs, tr.p, tr.ld, tr.bs, am, br.p, br.ld, br.bs, cr.p, cr.ld, cr.bs, skip, zr.p, zr.ld,
                 zr.bs, bias, softplus, h_in, h_out, lens, yr.p, yr.ld, yr.bs, code, bi, li, di, ni, gi,
                 bytes ? ws.data_ptr() : nullptr, bytes, stream));
    written(a[11]);
    written(a[13]);
    return y.release();
}

// (stream, x, packed, scales, n, group, zeros, bias, out)
PyObject *w4_matvec(PyObject *const *a, Py_ssize_t n_args) {
    count(n_args, 9, "w4_matvec");
    void *stream = stream_of(a[0]);
    const Tensor &x = tensor(a[1], "x");
    const int code = float_type(x, "x");
    if (x.dim() != 2) raise(PyExc_ValueError, "x must be [rows, k], got %s", text(x.sizes()).c_str());
    const int64_t M = x.size(0), k = x.size(1), n = int_of(a[4]), group = int_of(a[5]);
    if (group != 32 && group != 64 && (group <= 0 || group > INT32_MAX || group % 128))
        raise(PyExc_ValueError, "group=%lld must be 32, 64 or a multiple of 128 below 2^31", (long long)group);
    if (n < 0) raise(PyExc_ValueError, "n=%lld must not be negative", (long long)n);
    const Tensor &scales = tensor(a[3], "scales");
    const at::ScalarType stype = scales.scalar_type();
    if (stype != at::kHalf && stype != at::kFloat)
        raise(PyExc_TypeError, "scales must be a float16 or float32 tensor, got %s", type_name(stype));
    const int64_t nb = (n + 15) / 16, kb = (k + 127) / 128, ng = group < 128 ? kb * 128 / group : (k + group - 1) / group;
    const int64_t vals[3] = {nb, ng, 16}, shape[2] = {M, n};
    const Rows xr = rows(a[1], x.sizes(), x.scalar_type(), "x");
    const uint8_t *packed = vec<uint8_t>(a[2], {nb, kb, 1024}, at::kByte, "packed");
    const void *s = vec<void>(a[3], vals, stype, "scales");
    const uint8_t *zeros = vec<uint8_t>(a[6], vals, at::kByte, "zeros");
    const float *bias = vec<float>(a[7], {n}, at::kFloat, "bias");
    Ref y(output(a[8], shape, x));
    const Rows yr = rows(y.p, shape, x.scalar_type(), "out", true);
    check("mi_w4_matvec", g_w4(xr.p, xr.ld, code, packed, s, stype == at::kHalf ? MI_F16 : MI_F32, zeros, bias, yr.p, yr.ld,
                               size_of(M, "rows"), size_of(n, "n"), size_of(k, "k"), size_of(group, "group"), stream));
    written(a[8]);
    return y.release();
}

// A parameter of every row: a tensor [rows] of this type, or one number for all of them.
template <class T>
const T *each(PyObject *o, int64_t rows, at::ScalarType type, const char *name, T &all) {
    if (THPVariable_Check(o)) return vec<T>(o, {rows}, type, name);
    if constexpr (std::is_same<T, float>::value) {
        all = (float)PyFloat_AsDouble(o);
        if (PyErr_Occurred()) throw Raised{};
    } else {
        all = (T)std::min<int64_t>(std::max<int64_t>(int_of(o), INT32_MIN), INT32_MAX);
    }
    return nullptr;
}

// (stream, logits, u, temperature, top_k, top_p, min_p, scale, logprob, out)
PyObject *sample_tokens(PyObject *const *a, Py_ssize_t n) {
    count(n, 10, "sample_tokens");
    void *stream = stream_of(a[0]);
    const Tensor &x = tensor(a[1], "logits");
    const int code = x.scalar_type() == at::kInt ? (int)MI_I32 : float_type(x, "logits");
    if (x.dim() != 2) raise(PyExc_ValueError, "logits must be [rows, vocab], got %s", text(x.sizes()).c_str());
    const int64_t B = x.size(0), V = x.size(1);
    const double scale = PyFloat_AsDouble(a[7]);
    if (PyErr_Occurred()) throw Raised{};
    const int with_logprob = PyObject_IsTrue(a[8]);
    if (with_logprob < 0) throw Raised{};
    const Rows xr = rows(a[1], x.sizes(), x.scalar_type(), "logits");
    const float *u = vec<float>(a[2], {B}, at::kFloat, "u");
    float t_all = 1.0f, p_all = 1.0f, min_all = 0.0f;
    int32_t k_all = 0;
    const float *t = each<float>(a[3], B, at::kFloat, "temperature", t_all);
    const int32_t *k = each<int32_t>(a[4], B, at::kInt, "top_k", k_all);
    const float *p = each<float>(a[5], B, at::kFloat, "top_p", p_all), *least = each<float>(a[6], B, at::kFloat, "min_p", min_all);
    Ref ids(a[9] != Py_None ? (Py_INCREF(a[9]), a[9]) : empty({B}, x, at::kLong));
    int64_t *ip = vec<int64_t>(ids.p, {B}, at::kLong, "out");
    Ref lp(with_logprob ? empty({B}, x, at::kFloat) : (Py_INCREF(Py_None), Py_None));
    float *lpp = with_logprob ? static_cast<float *>(THPVariable_Unpack(lp.p).data_ptr()) : nullptr;
    const int bi = size_of(B, "rows"), vi = size_of(V, "vocab");
    size_t bytes = 0;
    check("mi_sample_workspace_size", g_sample_size(bi, vi, &bytes));
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check("mi_sample_tokens", g_sample(xr.p, code, xr.ld, scale, u, t, t_all, k, k_all, p, p_all, least, min_all, ip, lpp, bi, vi,
                                       bytes ? ws.data_ptr() : nullptr, bytes, stream));
    written(a[9]);
    return with_logprob ? Py_BuildValue("(NN)", ids.release(), lp.release()) : ids.release();
}

// Rows [batch, len, dim], or [batch, dim] as sequences of one token.
Rows sequences(PyObject *o, bool flat, int64_t B, int64_t L, int64_t D, at::ScalarType type, const char *name, bool out = false) {
    if (!flat) return rows(o, {B, L, D}, type, name, out);
    Rows r = rows(o, {B, D}, type, name, out);
    return {r.p, D, r.ld};
}

// (stream, y, x, a, b, ids, scales, x_scale, lens, out)
PyObject *adapter_add(PyObject *const *a, Py_ssize_t n_args) {
    count(n_args, 10, "adapter_add");
    void *stream = stream_of(a[0]);
    const Tensor &y = tensor(a[1], "y"), &x = tensor(a[2], "x"), &am = tensor(a[3], "a"), &bm = tensor(a[4], "b");
    const int code = float_type(y, "y"), wcode = float_type(am, "a");
    const bool flat = y.dim() == 2, bytes_in = x.scalar_type() == at::kChar;
    if (y.dim() != 2 && y.dim() != 3) raise(PyExc_ValueError, "y must be [batch, dim] or [batch, len, dim], got %s", text(y.sizes()).c_str());
    if (x.dim() != y.dim()) raise(PyExc_ValueError, "x must have y's dimensions, got %s beside %s", text(x.sizes()).c_str(), text(y.sizes()).c_str());
    if (am.dim() != 3) raise(PyExc_ValueError, "a must be [bank, rank, k], got %s", text(am.sizes()).c_str());
    const int64_t B = y.size(0), L = flat ? 1 : y.size(1), N = y.size(-1), bank = am.size(0), R = am.size(1), K = am.size(2);
    const Rows xr = sequences(a[2], flat, B, L, K, bytes_in ? at::kChar : y.scalar_type(), "x");
    const void *ap = vec<void>(a[3], {bank, R, K}, am.scalar_type(), "a"), *bp = vec<void>(a[4], {bank, N, R}, am.scalar_type(), "b");
    const int32_t *ids = vec<int32_t>(a[5], {B}, at::kInt, "ids");
    if (!ids && B > 0) raise(PyExc_TypeError, "ids must be a torch.Tensor");
    const float *scales = vec<float>(a[6], {bank}, at::kFloat, "scales");
    if (bytes_in != (a[7] != Py_None)) raise(PyExc_ValueError, "x_scale goes with int8 rows");
    const float *x_scale = flat ? vec<float>(a[7], {B}, at::kFloat, "x_scale") : vec<float>(a[7], {B, L}, at::kFloat, "x_scale");
    const int32_t *lens = vec<int32_t>(a[8], {B}, at::kInt, "lens");
    Ref out(output(a[9], y.sizes(), y));
    const Rows outr = sequences(out.p, flat, B, L, N, y.scalar_type(), "out", true);
    Rows yr = sequences(a[1], flat, B, L, N, y.scalar_type(), "y");
    if (yr.p && yr.p == outr.p) {
        // (strides of dimensions of one element are free)
        if ((L > 1 && yr.ld != outr.ld) || (B > 1 && yr.bs != outr.bs))
            raise(PyExc_ValueError, "out overlaps y: in place, it must have y's strides");
        yr = outr;
    }
    const int bi = size_of(B, "batch"), li = size_of(L, "len"), ri = size_of(R, "rank");
    size_t bytes = 0;
    check("mi_adapter_workspace_size", g_adapter_size(bi, li, ri, &bytes));
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, y.options().dtype(at::kByte));
    check("mi_adapter_add",
          g_adapter(xr.p, bytes_in ? (int)MI_I8 : code, xr.ld, xr.bs, x_scale, ap, bp, wcode, scales, ids, lens, yr.p, yr.ld, yr.bs,
                    outr.p, outr.ld, outr.bs, code, bi, li, size_of(K, "k"), size_of(N, "n"), ri, size_of(bank, "bank"),
                    bytes ? ws.data_ptr() : nullptr, bytes, stream));
    written(a[9]);
    return out.release();
}

// What a gated recurrence and its backward pass read.
struct Gated {
    int64_t B, L, D;
    at::ScalarType type;
    int code, bi, li, di;
    Rows x, r, i, z;
    const float *decay;
    float rate;
    const int32_t *lens;
    size_t forward_bytes = 0, backward_bytes = 0, saved_bytes = 0;

    Gated(PyObject *xo, PyObject *ro, PyObject *io, PyObject *decay_o, PyObject *zo, PyObject *rate_o, PyObject *lens_o) {
        const Tensor &t = tensor(xo, "x");
        code = float_type(t, "x");
        if (t.dim() != 3) raise(PyExc_ValueError, "x must be [batch, len, dim], got %s", text(t.sizes()).c_str());
        B = t.size(0), L = t.size(1), D = t.size(2), type = t.scalar_type();
        bi = size_of(B, "batch"), li = size_of(L, "len"), di = size_of(D, "dim");
        x = rows(xo, {B, L, D}, type, "x"), r = rows(ro, {B, L, D}, type, "r"), i = rows(io, {B, L, D}, type, "i");
        z = zo != Py_None ? rows(zo, {B, L, D}, type, "z") : Rows{};
        decay = static_cast<const float *>(like(decay_o, {D}, at::kFloat, "decay").data_ptr());
        if (!THPVariable_Unpack(decay_o).is_contiguous()) raise(PyExc_ValueError, "decay must be contiguous");
        rate = (float)PyFloat_AsDouble(rate_o);
        if (PyErr_Occurred()) throw Raised{};
        lens = vec<int32_t>(lens_o, {B}, at::kInt, "lens");
        check("mi_gated_scan_sizes", g_gated_sizes(bi, li, di, &forward_bytes, &backward_bytes, &saved_bytes));
    }
};

// (stream, x, r, i, decay, z, rate, h_in, h_out, lens, out): y, or None where autograd records an input
PyObject *gated_scan(PyObject *const *a, Py_ssize_t n) {
    count(n, 11, "gated_scan");
    void *stream = stream_of(a[0]);
    if (c10::GradMode::is_enabled())
        for (const int k : {1, 2, 3, 4, 5, 7})
            if (THPVariable_Check(a[k]) && THPVariable_Unpack(a[k]).requires_grad()) Py_RETURN_NONE;
    const Gated g(a[1], a[2], a[3], a[4], a[5], a[6], a[9]);
    const Tensor &x = THPVariable_Unpack(a[1]);
    const float *h_in = vec<float>(a[7], {g.B, g.D}, at::kFloat, "h_in");
    float *h_out = vec<float>(a[8], {g.B, g.D}, at::kFloat, "h_out");
    Ref y(output(a[10], x.sizes(), x));
    const Rows yr = rows(y.p, x.sizes(), g.type, "out", true);
    Tensor ws;
    if (g.forward_bytes) ws = at::empty({(int64_t)g.forward_bytes}, x.options().dtype(at::kByte));
    check("mi_gated_scan",
          g_gated(g.x.p, g.x.ld, g.x.bs, g.r.p, g.r.ld, g.r.bs, g.i.p, g.i.ld, g.i.bs, g.decay, g.rate, g.z.p, g.z.ld, g.z.bs, h_in,
                  h_out, g.lens, yr.p, yr.ld, yr.bs, nullptr, g.code, g.bi, g.li, g.di, g.forward_bytes ? ws.data_ptr() : nullptr,
                  g.forward_bytes, stream));
    written(a[8]);
    written(a[10]);
    return y.release();
}

// ------------------------------------------------ the gated recurrence under autograd
// In C++ on both sides: through Python the two passes of a small training step took 60 us of
// host time more than their kernels.  Nothing below touches Python (the backward pass runs on
// the engine's threads); what is wrong raises a C++ error, which torch hands on.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void require(mi_status st, const char *fn) {
    TORCH_CHECK(st == MI_OK, fn, " failed with status ", (int)st, ": ", g_last_error());
}
Rows rows_of(const Tensor &t) { return t.defined() ? Rows{t.data_ptr(), t.stride(1), t.stride(0)} : Rows{}; }
int code_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? MI_F32 : t.scalar_type() == at::kBFloat16 ? MI_BF16 : MI_F16; }
Tensor bytes_of(size_t n, const Tensor &like) {
    return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }

// What was recorded, of tensors that the call has checked; `stream`: a backward pass runs on the
// forward pass's.
variable_list gated_gradients(const Tensor &grad, const variable_list &in, double rate, int64_t stream, const std::array<bool, 6> &needs) {
    const Tensor &x = in[0], &r = in[1], &i = in[2], &decay = in[3], &z = in[4], &lens = in[5], &saved = in[6];
    // (contiguous() keeps an empty tensor's strides)
    const Tensor dy = grad.stride(2) != 1 || grad.is_neg() ? grad.clone(at::MemoryFormat::Contiguous) : grad;
    const int B = (int)x.size(0), L = (int)x.size(1), D = (int)x.size(2);
    size_t forward = 0, backward = 0, keep = 0;
    require(g_gated_sizes(B, L, D, &forward, &backward, &keep), "mi_gated_scan_sizes");
    const auto like_x = [&](bool on) { return on ? at::empty(x.sizes(), x.options()) : Tensor(); };
    const auto floats = [&](bool on, at::IntArrayRef shape) { return on ? at::empty(shape, x.options().dtype(at::kFloat)) : Tensor(); };
    variable_list out{like_x(needs[0]),       like_x(needs[1]), like_x(needs[2]), floats(needs[3], {x.size(2)}), like_x(needs[4]),
                      floats(needs[5], {x.size(0), x.size(2)})};
    const Tensor ws = bytes_of(backward, x);
    const Rows dr = rows_of(dy), xr = rows_of(x), rr = rows_of(r), ir = rows_of(i), zr = rows_of(z);
    require(g_gated_backward(dr.p, dr.ld, dr.bs, xr.p, xr.ld, xr.bs, rr.p, rr.ld, rr.bs, ir.p, ir.ld, ir.bs,
                             static_cast<const float *>(decay.data_ptr()), (float)rate, zr.p, zr.ld, zr.bs,
                             static_cast<const int32_t *>(pointer(lens)), static_cast<const float *>(saved.data_ptr()), pointer(out[0]),
                             pointer(out[1]), pointer(out[2]), pointer(out[4]), static_cast<float *>(pointer(out[3])),
                             static_cast<float *>(pointer(out[5])), code_of(x), B, L, D, pointer(ws), backward,
                             reinterpret_cast<void *>(stream)),
            "mi_gated_scan_backward");
    return out;
}

// The gradients as a node whose own gradient is an error: a second derivative that leaves this
// part out would be wrong without one.
struct GatedGradients : torch::autograd::Function<GatedGradients> {
    static variable_list forward(AutogradContext *, const Tensor &dy, const Tensor &x, const Tensor &r, const Tensor &i,
                                 const Tensor &decay, const Maybe &z, const Maybe &lens, const Tensor &saved, double rate,
                                 int64_t stream, std::array<bool, 6> needs) {
        variable_list out;      // (those there are)
        for (const Tensor &v : gated_gradients(dy, {x, r, i, decay, z.value_or(Tensor()), lens.value_or(Tensor()), saved}, rate, stream, needs))
            if (v.defined()) out.push_back(v);
        return out;
    }
    static variable_list backward(AutogradContext *, const variable_list &) { TORCH_CHECK(false, "gated_scan is differentiable once"); }
};

struct GatedScan : torch::autograd::Function<GatedScan> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &r, const Tensor &i, const Tensor &decay, const Maybe &gate,
                          const Maybe &first, const Maybe &lengths, double rate, int64_t stream) {
        const Tensor z = gate.value_or(Tensor()), h_in = first.value_or(Tensor()), lens = lengths.value_or(Tensor());
        const int B = (int)x.size(0), L = (int)x.size(1), D = (int)x.size(2);
        size_t forward = 0, backward = 0, keep = 0;
        require(g_gated_sizes(B, L, D, &forward, &backward, &keep), "mi_gated_scan_sizes");
        const Tensor y = at::empty(x.sizes(), x.options()), saved = at::empty({(int64_t)(keep / sizeof(float))}, x.options().dtype(at::kFloat)),
                     ws = bytes_of(forward, x);
        const Rows xr = rows_of(x), rr = rows_of(r), ir = rows_of(i), zr = rows_of(z), yr = rows_of(y);
        require(g_gated(xr.p, xr.ld, xr.bs, rr.p, rr.ld, rr.bs, ir.p, ir.ld, ir.bs, static_cast<const float *>(decay.data_ptr()),
                        (float)rate, zr.p, zr.ld, zr.bs, static_cast<const float *>(pointer(h_in)), nullptr,
                        static_cast<const int32_t *>(pointer(lens)), yr.p, std::max(yr.ld, x.size(2)), yr.bs,
                        static_cast<float *>(saved.data_ptr()), code_of(x), B, L, D, pointer(ws), forward, reinterpret_cast<void *>(stream)),
                "mi_gated_scan");
        ctx->save_for_backward({x, r, i, decay, z, lens, saved});
        ctx->saved_data["rate"] = rate;
        ctx->saved_data["stream"] = stream;
        ctx->saved_data["state"] = h_in.defined();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        variable_list out(9);
        if (!grads[0].defined()) return out;
        const variable_list in = ctx->get_saved_variables();
        const double rate = ctx->saved_data["rate"].toDouble();
        const int64_t stream = ctx->saved_data["stream"].toInt();
        // (tensors that were not given are not counted among the node's inputs)
        const bool z = in[4].defined(), state = ctx->saved_data["state"].toBool();
        const std::array<bool, 6> needs{ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2),
                                        ctx->needs_input_grad(3), z && ctx->needs_input_grad(4),
                                        state && ctx->needs_input_grad(z ? 5 : 4)};
        if (!c10::GradMode::is_enabled()) {
            const variable_list got = gated_gradients(grads[0], in, rate, stream, needs);
            std::copy(got.begin(), got.end(), out.begin());
            return out;
        }
        const variable_list got =
            GatedGradients::apply(grads[0], in[0], in[1], in[2], in[3], maybe(in[4]), maybe(in[5]), in[6], rate, stream, needs);
        for (int k = 0, at = 0; k < 6; ++k)
            if (needs[k]) out[k] = got[at++];
        return out;
    }
};

// (stream, x, r, i, decay, z, rate, h_in, lens): y, recorded
PyObject *gated_scan_recorded(PyObject *const *a, Py_ssize_t n) {
    count(n, 9, "gated_scan_recorded");
    void *stream = stream_of(a[0]);
    double rate;
    {
        const c10::AutoGradMode none(false);
        const Gated g(a[1], a[2], a[3], a[4], a[5], a[6], a[8]);
        vec<float>(a[7], {g.B, g.D}, at::kFloat, "h_in");
        rate = PyFloat_AsDouble(a[6]);
    }
    const auto some = [](PyObject *o) { return o == Py_None ? Maybe() : Maybe(THPVariable_Unpack(o)); };
    return THPVariable_Wrap(GatedScan::apply(THPVariable_Unpack(a[1]), THPVariable_Unpack(a[2]), THPVariable_Unpack(a[3]),
                                             THPVariable_Unpack(a[4]), some(a[5]), some(a[7]), some(a[8]), rate,
                                             reinterpret_cast<int64_t>(stream)));
}

// (stream, name, tensor): raises where the tensor is a leaf whose gradient another live graph
// adds up on another stream than this one.
PyObject *check_accumulator(PyObject *const *a, Py_ssize_t n) {
    count(n, 3, "check_accumulator");
    void *stream = stream_of(a[0]);
    const Tensor &t = tensor(a[2], "the input");
    const char *name = PyUnicode_AsUTF8(a[1]);
    if (!name) throw Raised{};
    if (t.requires_grad() && t.is_leaf()) {
        const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
        const auto on = node ? node->stream() : std::nullopt;
        // (a stream object of the current stream is the same as what the node keeps)
        if (on && c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device()) != *on)
            raise(PyExc_RuntimeError,
                  "%s is a leaf of another graph that lives, recorded on another stream: a backward pass captured here would make "
                  "that stream wait for the capture; drop that graph's outputs first", name);
    }
    Py_RETURN_NONE;
}

// (MIError, addresses of the entry points)
PyObject *init(PyObject *const *a, Py_ssize_t n) {
    const auto entry = [&](int i, auto &f) { f = reinterpret_cast<std::decay_t<decltype(f)>>(address(a[i])); };
    count(n, 14, "init");
    entry(1, g_norm);
    entry(2, g_conv);
    entry(3, g_scan_size);
    entry(4, g_scan);
    entry(5, g_w4);
    entry(6, g_sample_size);
    entry(7, g_sample);
    entry(8, g_adapter_size);
    entry(9, g_adapter);
    entry(10, g_gated_sizes);
    entry(11, g_gated);
    entry(12, g_gated_backward);
    entry(13, g_last_error);
    Py_INCREF(a[0]);
    Py_XDECREF(g_mi_error);
    g_mi_error = a[0];
    Py_RETURN_NONE;
}

// No C++ exception leaves a call.
template <PyObject *(*F)(PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *, PyObject *const *a, Py_ssize_t n) {
    try {
        return F(a, n);
    } catch (const Raised &) {
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(init),           METHOD(add_rms_norm), METHOD(causal_conv),
                         METHOD(selective_scan), METHOD(w4_matvec),
                         METHOD(sample_tokens), METHOD(adapter_add), METHOD(gated_scan), METHOD(gated_scan_recorded),
                         METHOD(check_accumulator), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_float_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__float_calls() { return PyModule_Create(&module); }
