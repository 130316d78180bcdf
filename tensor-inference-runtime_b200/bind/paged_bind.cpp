// paged_bind.cpp -- the Python entry points of the paged cache operators: checks
// of torch tensors and the call of the C function, compiled because a decode
// step's calls take the GPU a few microseconds each (interpreted, the checks of a
// norm-and-rotation call took 8 us more than its launch, compiled 1).
//
// The C functions come as addresses from the ctypes library (setup), so this
// module links torch alone.  Errors are raised as tir.TirError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>
#include <string>

#include "../../include/tir.h"

namespace {

struct {
    PyObject *error, *device, *stream;  // TirError, current device, raw current stream of a device
    decltype(&tir_last_error) last_error;
    decltype(&tir_qk_norm_rope) qk_norm_rope;
    decltype(&tir_qk_norm_rope_append) qk_norm_rope_append;
    decltype(&tir_kv_append) kv_append;
    decltype(&tir_kv_gather) kv_gather;
    decltype(&tir_paged_attention) paged_attention;
    decltype(&tir_paged_attention_workspace) workspace;
} S;

// Raised as a Python exception at the module's edge.
struct Raised {};

[[noreturn]] void raise(int status, const std::string& message) {
    if (PyObject* args = Py_BuildValue("(is)", status, message.c_str())) {
        PyErr_SetObject(S.error, args);
        Py_DECREF(args);
    }
    throw Raised();
}

[[noreturn]] void bad(const std::string& message) { raise(TIR_ERR_INVALID_ARG, message); }

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) bad(std::string(what) + " must be a torch tensor");
    return THPVariable_Unpack(o);
}

int32_t act_code(at::ScalarType t, const char* what) {
    switch (t) {
        case at::kFloat: return TIR_DTYPE_F32;
        case at::kHalf: return TIR_DTYPE_F16;
        case at::kBFloat16: return TIR_DTYPE_BF16;
        default:
            raise(TIR_ERR_UNSUPPORTED_DTYPE, std::string(what) + ": activations must be float32, float16 or bfloat16, got " + c10::toString(t));
    }
}

struct Rows {
    void* p;
    int64_t stride, n;
};

// A [tokens, heads, dim] tensor whose heads are adjacent.
Rows rows(const at::Tensor& x, int64_t heads, int64_t dim, at::ScalarType type, int64_t device, const char* what) {
    const auto shape = x.sizes();
    if (shape.size() != 3 || shape[1] != heads || shape[2] != dim)
        bad(std::string(what) + " must be [tokens, " + std::to_string(heads) + ", " + std::to_string(dim) + "]");
    const auto st = x.strides();
    if ((st[2] != 1 && dim > 1) || (st[1] != dim && heads > 1)) bad(std::string(what) + ": a token's heads must be adjacent");
    if (x.scalar_type() != type) bad(std::string(what) + " has another type than q or k: " + c10::toString(x.scalar_type()));
    if (x.get_device() != device) bad(std::string(what) + " is not on device " + std::to_string(device));
    return {x.data_ptr(), shape[0] > 1 ? st[0] : heads * dim, shape[0]};  // one token has no next one
}

// A contiguous int32 vector of at least n values; None: NULL.
const int32_t* ints(PyObject* o, int64_t n, int64_t device, const char* what) {
    if (o == Py_None) return nullptr;
    const at::Tensor& x = tensor(o, what);
    if (x.dim() != 1 || x.scalar_type() != at::kInt || x.size(0) < n || (n > 1 && x.stride(0) != 1))
        bad(std::string(what) + " must be a contiguous int32 vector of " + std::to_string(n) + " values");
    if (x.get_device() != device) bad(std::string(what) + " is not on device " + std::to_string(device));
    return static_cast<const int32_t*>(x.data_ptr());
}

const float* floats(PyObject* o, int64_t n, int64_t device) {
    if (o == Py_None) return nullptr;
    const at::Tensor& x = tensor(o, "a norm weight");
    if (x.dim() != 1 || x.size(0) != n || x.scalar_type() != at::kFloat || (n > 1 && x.stride(0) != 1))
        bad("a norm weight must be a contiguous float32 vector of " + std::to_string(n));
    if (x.get_device() != device) bad("a norm weight is not on device " + std::to_string(device));
    return static_cast<const float*>(x.data_ptr());
}

int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}

int32_t integer32(PyObject* o, const char* what) {
    const int64_t v = integer(o);
    if (v < 0 || v > INT32_MAX) bad(std::string(what) + " is out of range");
    return static_cast<int32_t>(v);
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}

int64_t current_device() {
    PyObject* r = PyObject_CallNoArgs(S.device);
    if (!r) throw Raised();
    const int64_t v = PyLong_AsLongLong(r);
    Py_DECREF(r);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}

int64_t current_stream(int64_t device) {
    PyObject* d = PyLong_FromLongLong(device);
    if (!d) throw Raised();
    PyObject* r = PyObject_CallOneArg(S.stream, d);
    Py_DECREF(d);
    if (!r) throw Raised();
    const int64_t v = static_cast<int64_t>(PyLong_AsUnsignedLongLong(r));
    Py_DECREF(r);
    if (PyErr_Occurred()) throw Raised();
    return v;
}

// The stream to launch on (None: the current one).  The operators run on the
// current device, and their tensors must be there.
void* stream_of(PyObject* o, int64_t device) {
    if (device < 0) bad("the cache and the activations must be on a CUDA device");
    const int64_t now = current_device();
    if (now != device)
        bad("the cache or activations are on device " + std::to_string(device) + ", the current device is " + std::to_string(now));
    return reinterpret_cast<void*>(o == Py_None ? current_stream(device) : integer(o));
}

void check(tir_status st) {
    if (st != TIR_OK) raise(st, S.last_error());
}

// rope, q_weight, k_weight, eps, pairs
tir_qk_norm norm_of(PyObject* const* a, int64_t dim, int64_t device) {
    tir_qk_norm n{};
    if (a[0] != Py_None) {
        const at::Tensor& x = tensor(a[0], "rope");
        if (x.dim() != 3 || x.size(2) != 2 || x.scalar_type() != at::kFloat || !x.is_contiguous())
            bad("rope must be a contiguous float32 [positions, rope_dim / 2, 2] table");
        if (x.get_device() != device) bad("rope is not on device " + std::to_string(device));
        if (x.size(1) > (1 << 20)) bad("rope must have at most 2^20 pairs");
        n.rope = static_cast<const float*>(x.data_ptr());
        n.rope_positions = x.size(0);
        n.rope_dim = static_cast<int32_t>(2 * x.size(1));
    }
    n.q_weight = floats(a[1], dim, device);
    n.k_weight = floats(a[2], dim, device);
    n.eps = static_cast<float>(number(a[3]));
    n.pairs = integer32(a[4], "pairs");
    return n;
}

void same(int64_t n, int64_t m) {
    if (n != m) bad("rows of different token counts");
}

const at::Tensor& query(PyObject* o, const char* what) {
    const at::Tensor& q = tensor(o, what);
    if (q.dim() != 3) bad(std::string(what) + " must be [tokens, heads, dim]");
    return q;
}

// q, k, q_out, k_out, positions, rope, q_weight, k_weight, eps, pairs, stream
void qk_norm_rope(PyObject* const* a) {
    const at::Tensor &q = query(a[0], "q"), &k = query(a[1], "k");
    const auto type = q.scalar_type();
    const int32_t code = act_code(type, "q");
    const int64_t dev = q.get_device(), qh = q.size(1), kh = k.size(1), dim = q.size(2);
    void* st = stream_of(a[10], dev);
    const Rows x = rows(q, qh, dim, type, dev, "q"), y = rows(k, kh, dim, type, dev, "k");
    const Rows xo = rows(tensor(a[2], "q_out"), qh, dim, type, dev, "q_out"), yo = rows(tensor(a[3], "k_out"), kh, dim, type, dev, "k_out");
    same(x.n, y.n), same(x.n, xo.n), same(x.n, yo.n);
    if (qh > INT32_MAX || kh > INT32_MAX || dim > INT32_MAX) bad("q or k is too large");
    const tir_qk_norm n = norm_of(a + 5, dim, dev);
    check(S.qk_norm_rope(x.p, x.stride, y.p, y.stride, xo.p, xo.stride, yo.p, yo.stride, ints(a[4], x.n, dev, "positions"), x.n,
                         static_cast<int32_t>(qh), static_cast<int32_t>(kh), static_cast<int32_t>(dim), code, &n, st));
}

const tir_kv_pages* pages(PyObject* o) { return reinterpret_cast<const tir_kv_pages*>(integer(o)); }

// q, k, v, q_out, kv, device, seqs, positions, rope, q_weight, k_weight, eps, pairs, stream
void qk_norm_rope_append(PyObject* const* a) {
    const at::Tensor& q = query(a[0], "q");
    const tir_kv_pages* kv = pages(a[4]);
    const auto type = q.scalar_type();
    const int32_t code = act_code(type, "q");
    const int64_t dev = integer(a[5]), qh = q.size(1), kh = kv->kv_heads, dim = kv->dim;
    void* st = stream_of(a[13], dev);
    const Rows x = rows(q, qh, dim, type, dev, "q"), y = rows(tensor(a[1], "k"), kh, dim, type, dev, "k");
    const Rows z = rows(tensor(a[2], "v"), kh, dim, type, dev, "v"), xo = rows(tensor(a[3], "q_out"), qh, dim, type, dev, "q_out");
    same(x.n, y.n), same(x.n, z.n), same(x.n, xo.n);
    if (qh > INT32_MAX) bad("q is too large");
    const tir_qk_norm n = norm_of(a + 8, dim, dev);
    check(S.qk_norm_rope_append(x.p, x.stride, y.p, y.stride, z.p, z.stride, xo.p, xo.stride, kv, ints(a[6], x.n, dev, "seqs"),
                                ints(a[7], x.n, dev, "positions"), x.n, static_cast<int32_t>(qh), code, &n, st));
}

// kv, device, k, v, seqs, positions, stream
template <bool kGather>
void move(PyObject* const* a) {
    const char *ks = kGather ? "k_out" : "k", *vs = kGather ? "v_out" : "v";
    const tir_kv_pages* kv = pages(a[0]);
    const int64_t dev = integer(a[1]);
    const at::Tensor& k = tensor(a[2], ks);
    const auto type = k.scalar_type();
    const int32_t code = act_code(type, ks);
    void* st = stream_of(a[6], dev);
    const Rows x = rows(k, kv->kv_heads, kv->dim, type, dev, ks), y = rows(tensor(a[3], vs), kv->kv_heads, kv->dim, type, dev, vs);
    same(x.n, y.n);
    const int32_t *seqs = ints(a[4], x.n, dev, "seqs"), *positions = ints(a[5], x.n, dev, "positions");
    if constexpr (kGather)
        check(S.kv_gather(kv, x.p, x.stride, y.p, y.stride, seqs, positions, x.n, code, st));
    else
        check(S.kv_append(kv, x.p, x.stride, y.p, y.stride, seqs, positions, x.n, code, st));
}

// q, kv, device, seq_lens, out, scale, max_len, window, workspace, stream
void paged_attention(PyObject* const* a) {
    const at::Tensor& q = query(a[0], "q");
    const tir_kv_pages* kv = pages(a[1]);
    const int64_t dev = integer(a[2]);
    const auto type = q.scalar_type();
    const int32_t code = act_code(type, "q");
    void* st = stream_of(a[9], dev);
    const int64_t qh = q.size(1);
    if (qh > INT32_MAX) bad("q is too large");
    const Rows x = rows(q, qh, kv->dim, type, dev, "q"), o = rows(tensor(a[4], "out"), qh, kv->dim, type, dev, "out");
    same(x.n, o.n);
    const int32_t* lens = ints(a[3], x.n, dev, "seq_lens");
    const int64_t max_len = integer(a[6]), window = integer(a[7]);
    void* ws = nullptr;
    int64_t bytes = 0;
    at::Tensor own;  // from torch's allocator: stays until work on the current stream is done with it
    if (a[8] != Py_None) {
        const at::Tensor& w = tensor(a[8], "workspace");
        if (w.get_device() != dev || !w.is_contiguous()) bad("workspace must be a contiguous tensor on device " + std::to_string(dev));
        ws = w.data_ptr();
        bytes = static_cast<int64_t>(w.nbytes());
    } else if (a[9] == Py_None || reinterpret_cast<int64_t>(st) == current_stream(dev)) {
        bytes = S.workspace(kv, x.n, static_cast<int32_t>(qh), max_len, window);
        if (bytes > 0) {
            own = at::empty({bytes}, q.options().dtype(at::kByte));
            ws = own.data_ptr();
        }
    }  // on another stream a call that divides its rows is refused: the allocator would not know of its work
    check(S.paged_attention(x.p, x.stride, kv, lens, o.p, o.stride, x.n, static_cast<int32_t>(qh), code,
                            static_cast<float>(number(a[5])), max_len, window, ws, bytes, st));
}

// kv, rows, q_heads, max_len, window
PyObject* workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
    try {
        if (n != 5) bad("workspace takes 5 arguments");
        const int64_t b = S.workspace(pages(a[0]), integer(a[1]), integer32(a[2], "q_heads"), integer(a[3]), integer(a[4]));
        if (b < 0) bad(S.last_error());
        return PyLong_FromLongLong(b);
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

template <void (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != N) bad("wrong number of arguments");
        F(args);
        Py_RETURN_NONE;
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// TirError, current_device, current_raw_stream, then the C functions' addresses
PyObject* setup(PyObject*, PyObject* args) {
    unsigned long long f[7];
    PyObject *e, *d, *s;
    if (!PyArg_ParseTuple(args, "OOOKKKKKKK", &e, &d, &s, f, f + 1, f + 2, f + 3, f + 4, f + 5, f + 6)) return nullptr;
    Py_INCREF(e), Py_INCREF(d), Py_INCREF(s);
    S.error = e, S.device = d, S.stream = s;
    S.last_error = reinterpret_cast<decltype(S.last_error)>(f[0]);
    S.qk_norm_rope = reinterpret_cast<decltype(S.qk_norm_rope)>(f[1]);
    S.qk_norm_rope_append = reinterpret_cast<decltype(S.qk_norm_rope_append)>(f[2]);
    S.kv_append = reinterpret_cast<decltype(S.kv_append)>(f[3]);
    S.kv_gather = reinterpret_cast<decltype(S.kv_gather)>(f[4]);
    S.paged_attention = reinterpret_cast<decltype(S.paged_attention)>(f[5]);
    S.workspace = reinterpret_cast<decltype(S.workspace)>(f[6]);
    Py_RETURN_NONE;
}

#define ENTRY(name, fn, n) \
    { name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<fn, n>)), METH_FASTCALL, nullptr }

PyMethodDef methods[] = {
    {"setup", setup, METH_VARARGS, nullptr},
    ENTRY("qk_norm_rope", qk_norm_rope, 11),
    ENTRY("qk_norm_rope_append", qk_norm_rope_append, 14),
    ENTRY("kv_append", move<false>, 7),
    ENTRY("kv_gather", move<true>, 7),
    ENTRY("paged_attention", paged_attention, 10),
    {"workspace", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&workspace)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_bind", nullptr, -1, methods};

}  // namespace

// built_for: the torch whose headers this was compiled with
PyMODINIT_FUNC PyInit__paged_bind() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", TIR_BIND_TORCH) < 0) Py_CLEAR(m);
    return m;
}
