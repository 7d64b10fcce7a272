// The host side of the float operators' calls (mamba_int.ops: add_rms_norm,
// add_rms_norm_quant, causal_conv, selective_scan, w4_matvec): checks of the
// tensors, outputs, and the call of the C ABI, as a Python module.  Through ctypes
// and checks in Python a call took 9 to 18 us of host time, several times what its
// kernel takes on a decode step's rows.
//
// The entry points come as addresses (the library is loaded once, by _lib), the
// stream as its handle and device.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdarg.h>

#include "mamba_int.h"

namespace {

using at::Tensor;

decltype(&mi_add_rms_norm) g_norm;
decltype(&mi_causal_conv) g_conv;
decltype(&mi_selective_scan) g_scan;
decltype(&mi_selective_scan_workspace_size) g_scan_size;
decltype(&mi_w4_matvec) g_w4;
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

// (MIError, addresses of the six entry points)
PyObject *init(PyObject *const *a, Py_ssize_t n) {
    count(n, 7, "init");
    void *p[6];
    for (int i = 0; i < 6; ++i) p[i] = address(a[i + 1]);
    g_norm = reinterpret_cast<decltype(g_norm)>(p[0]);
    g_conv = reinterpret_cast<decltype(g_conv)>(p[1]);
    g_scan_size = reinterpret_cast<decltype(g_scan_size)>(p[2]);
    g_scan = reinterpret_cast<decltype(g_scan)>(p[3]);
    g_w4 = reinterpret_cast<decltype(g_w4)>(p[4]);
    g_last_error = reinterpret_cast<decltype(g_last_error)>(p[5]);
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
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(init),           METHOD(add_rms_norm), METHOD(causal_conv),
                         METHOD(selective_scan), METHOD(w4_matvec),    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_float_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__float_calls() { return PyModule_Create(&module); }
