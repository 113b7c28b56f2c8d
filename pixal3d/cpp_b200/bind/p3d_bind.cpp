// Native torch binding of the operators that run in a few microseconds.
//
// A ctypes call with its checks in Python costs the host 9 to 14 us, several
// times the kernels of a single token; here the checks, the output tensor, the
// stream and the call take about 4.  ops.py documents the functions and calls
// them by position; the checks are theirs: ValueError and TypeError for
// tensors that do not fit, P3DError for a status of the library.  The calls
// go through contexts of libp3dcuda.so that share the ctypes binding's fault
// flags and launch counts.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>

#include "p3d.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr int kMaxDevices = 64;
PyObject *g_root_context = nullptr;  // (device) -> handle of the device's first context, which stays
PyObject *g_error = nullptr;         // P3DError(status, message)

// A host thread's contexts, forks of the devices' first ones: no other thread,
// nor the ctypes binding, sets their stream.
struct ThreadContexts {
    p3d_ctx *of[kMaxDevices] = {};
    ~ThreadContexts() {
        for (p3d_ctx *c : of) p3d_ctx_destroy(c);
    }
};
thread_local ThreadContexts t_contexts;

struct Raised {};  // a Python error has been set

[[noreturn]] void fail(PyObject *type, const char *what, const char *message) {
    PyErr_Format(type, "%s: %s", what, message);
    throw Raised();
}
void need(bool ok, const char *what, const char *message) {
    if (!ok) fail(PyExc_ValueError, what, message);
}

const Tensor &tensor(PyObject *o, const char *what, const char *name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: %s must be a tensor", what, name);
        throw Raised();
    }
    return THPVariable_Unpack(o);
}
int device_of(const Tensor &t, const char *what) {
    need(t.is_cuda(), what, "tensors must be on a CUDA device");
    return t.device().index();
}
bool lies_on(const Tensor &t, int device) { return t.is_cuda() && t.device().index() == device; }

int dtype_code(ScalarType t, const char *what) {
    if (t == at::kFloat) return P3D_F32;
    if (t == at::kBFloat16) return P3D_BF16;
    if (t == at::kHalf) return P3D_F16;
    fail(PyExc_TypeError, what, "unsupported dtype (f32, bf16 or f16 wanted)");
}

// Row pitch of a 2-D view of `cols` columns with unit column stride; of a
// single row, `cols` (its stride says nothing).
int64_t matrix(const Tensor &t, int64_t cols, ScalarType type, int device, const char *what, const char *name) {
    if (t.dim() != 2 || t.scalar_type() != type || !lies_on(t, device) || t.size(1) != cols) {
        PyErr_Format(PyExc_ValueError, "%s: %s must be a 2-D %s tensor of %lld columns on cuda:%d", what, name, c10::toString(type),
                     static_cast<long long>(cols), device);
        throw Raised();
    }
    if (cols > 1 && t.stride(1) != 1) {
        PyErr_Format(PyExc_ValueError, "%s: %s must be a row-major view", what, name);
        throw Raised();
    }
    return t.size(0) > 1 ? t.stride(0) : cols;
}

// Pointer of a contiguous 1-D tensor of n elements; null for None.
template <typename T>
T *vector(PyObject *o, int64_t n, ScalarType type, int device, const char *what, const char *name) {
    if (o == Py_None) return nullptr;
    const Tensor &t = tensor(o, what, name);
    if (t.dim() != 1 || t.scalar_type() != type || !lies_on(t, device) || t.size(0) != n || !t.is_contiguous()) {
        PyErr_Format(PyExc_ValueError, "%s: %s must be a contiguous %s vector of %lld on cuda:%d", what, name, c10::toString(type),
                     static_cast<long long>(n), device);
        throw Raised();
    }
    return static_cast<T *>(t.data_ptr());
}

int64_t integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}
int small(PyObject *o) {
    const int64_t v = integer(o);
    if (v < INT32_MIN || v > INT32_MAX) {
        PyErr_SetString(PyExc_OverflowError, "integer argument out of range");
        throw Raised();
    }
    return static_cast<int>(v);
}
float real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return static_cast<float>(v);
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised();
    return v != 0;
}

p3d_ctx *context(int device, const char *what) {
    need(device < kMaxDevices, what, "device index out of range");
    p3d_ctx *&mine = t_contexts.of[device];
    if (!mine) {
        PyObject *h = PyObject_CallFunction(g_root_context, "i", device);
        if (!h) throw Raised();
        void *p = PyLong_AsVoidPtr(h);
        Py_DECREF(h);
        if (!p) throw Raised();
        if (p3d_ctx_fork(static_cast<p3d_ctx *>(p), nullptr, &mine) != P3D_OK) fail(PyExc_MemoryError, what, "no context");
    }
    return mine;
}

// call(ctx) on torch's current stream of the device, without the GIL.
template <typename F>
void launch(int device, const char *what, F &&call) {
    p3d_ctx *ctx = context(device, what);
    void *stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    int rc;
    std::string message;
    Py_BEGIN_ALLOW_THREADS;
    p3d_ctx_set_stream(ctx, stream);
    rc = call(ctx);
    if (rc != P3D_OK) message = p3d_last_error(ctx);
    Py_END_ALLOW_THREADS;
    if (rc != P3D_OK) {
        PyObject *e = PyObject_CallFunction(g_error, "is", rc, message.c_str());
        if (e) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
        throw Raised();
    }
}

Tensor fresh(at::IntArrayRef size, ScalarType type, const Tensor &like) {
    return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}

#define P3D_BIND_BEGIN HANDLE_TH_ERRORS try {
#define P3D_BIND_END                \
    }                               \
    catch (const Raised &) {        \
        return nullptr;             \
    }                               \
    END_HANDLE_TH_ERRORS

#define P3D_ARGS(count, what)                                                       \
    if (nargs != (count)) {                                                         \
        PyErr_Format(PyExc_TypeError, "%s: %d arguments wanted", what, (count));    \
        return nullptr;                                                             \
    }

// x, out, scale -> (out, scale)
PyObject *quantize_rows(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    P3D_BIND_BEGIN
    constexpr const char *what = "quantize_rows";
    P3D_ARGS(3, what)
    const Tensor &x = tensor(a[0], what, "x");
    const int dev = device_of(x, what), dt = dtype_code(x.scalar_type(), what);
    need(x.dim() == 2 && x.size(1) > 0, what, "x must be 2-D with columns");
    const int64_t m = x.size(0), k = x.size(1), ldx = matrix(x, k, x.scalar_type(), dev, what, "x");
    Tensor out, scale;
    int64_t ldq = (k + 15) & ~int64_t(15);
    if (a[1] == Py_None) {
        out = at::detail::empty_strided_cuda({m, k}, {ldq, 1}, at::kChar, x.device());
    } else {
        out = tensor(a[1], what, "out");
        ldq = matrix(out, k, at::kChar, dev, what, "out");
        need(out.size(0) == m, what, "out must be of x's shape");
    }
    float *ps;
    if (a[2] == Py_None) {
        scale = fresh({m}, at::kFloat, x);
        ps = scale.data_ptr<float>();
    } else {
        ps = vector<float>(a[2], m, at::kFloat, dev, what, "scale");
        scale = THPVariable_Unpack(a[2]);
    }
    if (m > 0)
        launch(dev, what, [&](p3d_ctx *c) {
            return p3d_quantize_rows(c, x.data_ptr(), ldx, m, k, dt, static_cast<int8_t *>(out.data_ptr()), ldq, ps);
        });
    PyObject *q = THPVariable_Wrap(std::move(out));
    if (!q) return nullptr;
    PyObject *s = THPVariable_Wrap(std::move(scale));
    if (!s) {
        Py_DECREF(q);
        return nullptr;
    }
    PyObject *both = PyTuple_Pack(2, q, s);
    Py_DECREF(q);
    Py_DECREF(s);
    return both;
    P3D_BIND_END
}

// x, x_scale, w, w_scale, bias, out, out_dtype, epilogue, gate, batch_offsets -> out
PyObject *linear_i8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    P3D_BIND_BEGIN
    constexpr const char *what = "linear_i8";
    P3D_ARGS(10, what)
    const Tensor &x = tensor(a[0], what, "x"), &w = tensor(a[2], what, "w");
    const int dev = device_of(x, what);
    need(x.dim() == 2 && w.dim() == 2, what, "x and w must be 2-D");
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
    need(k > 0 && n > 0, what, "x or w of no elements");
    int64_t ldx = matrix(x, k, at::kChar, dev, what, "x"), ldw = matrix(w, k, at::kChar, dev, what, "w");
    // a lone row has no pitch; the tensor maps want one of whole 16-byte words
    if (m == 1) ldx = (k + 15) & ~int64_t(15);
    if (n == 1) ldw = (k + 15) & ~int64_t(15);
    const int epilogue = small(a[7]);
    Tensor out;
    int64_t ldo = n;
    int dt;
    if (a[5] == Py_None) {
        need(!(epilogue & P3D_EPI_RESIDUAL), what, "the residual epilogue adds into out");
        if (!THPDtype_Check(a[6])) fail(PyExc_TypeError, what, "out_dtype must be a torch dtype");
        const ScalarType type = reinterpret_cast<THPDtype *>(a[6])->scalar_type;
        dt = dtype_code(type, what);
        out = fresh({m, n}, type, x);
    } else {
        out = tensor(a[5], what, "out");
        dt = dtype_code(out.scalar_type(), what);
        ldo = matrix(out, n, out.scalar_type(), dev, what, "out");
        need(out.size(0) == m, what, "out must be [m, n]");
    }
    need(a[1] != Py_None && a[3] != Py_None, what, "x_scale and w_scale are wanted");
    const float *xs = vector<float>(a[1], m, at::kFloat, dev, what, "x_scale");
    const float *ws = vector<float>(a[3], n, at::kFloat, dev, what, "w_scale");
    const float *bias = vector<float>(a[4], n, at::kFloat, dev, what, "bias");
    const float *gate = nullptr;
    const int32_t *offsets = nullptr;
    int64_t ldg = 0;
    int items = 0;
    if (a[8] != Py_None) {
        const Tensor &g = tensor(a[8], what, "gate");
        need(a[9] != Py_None, what, "gate needs batch offsets");
        ldg = matrix(g, n, at::kFloat, dev, what, "gate");
        items = static_cast<int>(g.size(0));
        need(items > 0, what, "gate must have a row an item");
        offsets = vector<int32_t>(a[9], items + 1, at::kInt, dev, what, "batch_offsets");
        gate = static_cast<const float *>(g.data_ptr());
    }
    if (m > 0)
        launch(dev, what, [&](p3d_ctx *c) {
            return p3d_linear_i8(c, static_cast<const int8_t *>(x.data_ptr()), ldx, xs, static_cast<const int8_t *>(w.data_ptr()),
                                 ldw, ws, bias, m, n, k, out.data_ptr(), ldo, dt, epilogue, gate, ldg, offsets, items);
        });
    return THPVariable_Wrap(std::move(out));
    P3D_BIND_END
}

// x, freqs, heads, head_dim, positions, layout, amplitude, position_offset, out -> out
PyObject *rotary(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    P3D_BIND_BEGIN
    constexpr const char *what = "rotary";
    P3D_ARGS(9, what)
    const Tensor &x = tensor(a[0], what, "x"), &f = tensor(a[1], what, "freqs");
    const int dev = device_of(x, what), dt = dtype_code(x.scalar_type(), what);
    const int heads = small(a[2]), head_dim = small(a[3]), layout = small(a[5]);
    need(x.dim() == 2 && f.dim() == 1, what, "x must be 2-D and freqs 1-D");
    const int64_t n = x.size(0), width = x.size(1), half = f.size(0);
    need(heads > 0 && head_dim > 0 && width == static_cast<int64_t>(heads) * head_dim, what, "x must be [n, heads * head_dim]");
    const int64_t ldx = matrix(x, width, x.scalar_type(), dev, what, "x");
    const double *freqs = vector<double>(a[1], half, at::kDouble, dev, what, "freqs");
    const int32_t *positions = vector<int32_t>(a[4], n, at::kInt, dev, what, "positions");
    const float amplitude = real(a[6]);
    const int64_t offset = integer(a[7]);
    Tensor out;
    int64_t ldo = width;
    if (a[8] == Py_None) {
        out = fresh({n, width}, x.scalar_type(), x);
    } else {
        out = tensor(a[8], what, "out");
        ldo = matrix(out, width, x.scalar_type(), dev, what, "out");
        need(out.size(0) == n, what, "out must be like x");
    }
    need(half < 65536, what, "too many frequencies");
    if (n > 0)
        launch(dev, what, [&](p3d_ctx *c) {
            return p3d_rotary(c, x.data_ptr(), ldx, n, heads, head_dim, static_cast<int>(2 * half), layout, positions, offset, freqs,
                              amplitude, out.data_ptr(), ldo, dt);
        });
    return THPVariable_Wrap(std::move(out));
    P3D_BIND_END
}

// q, k, v, cu_q, cu_k, max_q, max_k, heads, scale, kv_heads, causal, prefix,
// doc_q, doc_k, slopes, softcap, out -> out
PyObject *masked_attention(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    P3D_BIND_BEGIN
    constexpr const char *what = "masked_attention";
    P3D_ARGS(17, what)
    const Tensor &q = tensor(a[0], what, "q"), &k = tensor(a[1], what, "k"), &v = tensor(a[2], what, "v");
    const Tensor &cq = tensor(a[3], what, "cu_q");
    tensor(a[4], what, "cu_k");
    const int dev = device_of(q, what);
    const ScalarType type = q.scalar_type();
    need(type == at::kHalf || type == at::kBFloat16, what, "q, k, v must be bf16 or f16");
    const int dt = dtype_code(type, what);
    need(q.dim() == 2 && k.dim() == 2 && v.dim() == 2 && cq.dim() == 1, what, "q, k, v must be 2-D and the offsets 1-D");
    const int heads = small(a[7]), kv = a[9] == Py_None ? heads : small(a[9]);
    const int64_t rows_q = q.size(0), width = q.size(1), rows_k = k.size(0);
    need(heads > 0 && kv > 0 && width > 0 && width % heads == 0, what, "q's columns must be heads * d");
    const int64_t d = width / heads;
    need(d < 65536, what, "head_dim out of range");
    const int64_t ldq = matrix(q, width, type, dev, what, "q"), ldk = matrix(k, kv * d, type, dev, what, "k"),
                  ldv = matrix(v, kv * d, type, dev, what, "v");
    need(v.size(0) == rows_k, what, "k and v must have the same rows");
    const int64_t nseq = cq.size(0) - 1;
    need(nseq >= 0 && nseq < 65536, what, "between 0 and 65535 sequences wanted");
    const int32_t *cu_q = vector<int32_t>(a[3], nseq + 1, at::kInt, dev, what, "cu_q");
    const int32_t *cu_k = vector<int32_t>(a[4], nseq + 1, at::kInt, dev, what, "cu_k");
    need((a[12] == Py_None) == (a[13] == Py_None), what, "doc_q and doc_k go together");
    p3d_attention_rules rules{};
    rules.softcap = real(a[15]);
    rules.causal = truth(a[10]);
    rules.prefix = vector<int32_t>(a[11], nseq, at::kInt, dev, what, "prefix");
    rules.doc_q = vector<int32_t>(a[12], rows_q, at::kInt, dev, what, "doc_q");
    rules.doc_k = vector<int32_t>(a[13], rows_k, at::kInt, dev, what, "doc_k");
    rules.slopes = vector<float>(a[14], heads, at::kFloat, dev, what, "slopes");
    const float scale = real(a[8]);
    const int64_t max_q = std::min(integer(a[5]), rows_q), max_k = std::min(integer(a[6]), rows_k);
    need(max_q >= 0 && max_k >= 0, what, "max_q and max_k must not be negative");
    Tensor out, ws;
    int64_t ldo = width;
    if (a[16] == Py_None) {
        out = fresh({rows_q, width}, type, q);
    } else {
        out = tensor(a[16], what, "out");
        ldo = matrix(out, width, type, dev, what, "out");
        need(out.size(0) == rows_q, what, "out must be like q");
    }
    if (rows_q > 0 && nseq > 0 && max_q > 0) {
        const size_t bytes =
            p3d_masked_attention_workspace(static_cast<int>(nseq), max_q, max_k, rows_q, rows_k, heads, kv, static_cast<int>(d),
                                           rules.doc_k != nullptr);
        if (bytes) ws = fresh({static_cast<int64_t>(bytes)}, at::kByte, q);
        launch(dev, what, [&](p3d_ctx *c) {
            return p3d_masked_attention(c, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, out.data_ptr(), ldo, cu_q, cu_k,
                                        static_cast<int>(nseq), max_q, max_k, rows_q, rows_k, heads, kv, static_cast<int>(d), scale,
                                        &rules, bytes ? ws.data_ptr() : nullptr, bytes, dt);
        });
    }
    return THPVariable_Wrap(std::move(out));
    P3D_BIND_END
}

// root_context(device) -> handle, P3DError
PyObject *setup(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    if (nargs != 2) {
        PyErr_SetString(PyExc_TypeError, "setup: 2 arguments wanted");
        return nullptr;
    }
    Py_INCREF(a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(g_root_context, a[0]);
    Py_XSETREF(g_error, a[1]);
    Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"setup", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(setup)), METH_FASTCALL, nullptr},
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(quantize_rows)), METH_FASTCALL, nullptr},
    {"linear_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(linear_i8)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(rotary)), METH_FASTCALL, nullptr},
    {"masked_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(masked_attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&kModule); }
