// Python binding of the streaming-memory entry points (tcq_rope_axes, tcq_kv8_*) of libtcq_b200.so.
//
// These run once per token and layer, and a call's own work takes a few microseconds: the checks of the arguments and the
// launch are made here rather than through ctypes. The C ABI stays the only interface to the kernels: kernels.py passes the
// addresses of its functions, its error class and its launch counts once, when it is imported.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "tcq_b200.h"

namespace {

decltype(&tcq_status_string) f_status;
decltype(&tcq_rope_axes) f_rope;
decltype(&tcq_kv8_append) f_append;
decltype(&tcq_kv8_read) f_read;
decltype(&tcq_kv8_attention_workspace) f_workspace;
decltype(&tcq_kv8_attention) f_attention;
decltype(&tcq_capture_id) f_capture;
PyObject *g_error, *g_launches, *g_rope_class, *g_cache_class, *s_ref;

struct Refused {};                         // a Python error is set

[[noreturn]] void refuse(const char* what, const char* why) {
    PyErr_Format(g_error, "%s: %s", what, why);
    throw Refused();
}

const at::Tensor& tensor(const char* what, PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: %s must be a tensor", what, name);
        throw Refused();
    }
    return THPVariable_Unpack(o);
}

int dtype_code(const char* what, const at::Tensor& t, bool f32) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return TCQ_DT_BF16;
        case at::kHalf: return TCQ_DT_F16;
        case at::kFloat:
            if (f32) return TCQ_DT_F32;
            [[fallthrough]];
        default: break;
    }
    PyErr_Format(g_error, "%s: dtype %s not supported (expected one of bfloat16, float16%s)", what, c10::toString(t.scalar_type()),
                 f32 ? ", float32" : "");
    throw Refused();
}

// (B, T, W) with contiguous rows on `dev`.
void rows(const char* what, const char* name, const at::Tensor& t, int dev) {
    if (t.dim() != 3 || !t.is_cuda() || t.get_device() != dev || (t.size(2) > 1 && t.stride(2) != 1)) {
        PyErr_Format(g_error, "%s: %s must be a (B, T, heads * D) CUDA tensor with contiguous rows, on one device with the others", what, name);
        throw Refused();
    }
}

const int32_t* ints(const char* what, const char* name, const at::Tensor& t, at::IntArrayRef shape, int dev) {
    if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != dev || !t.is_contiguous() || t.sizes() != shape) {
        std::string s = "(";
        for (int64_t n : shape) s += std::to_string(n) + ", ";
        PyErr_Format(g_error, "%s: %s must be a contiguous int32 CUDA tensor of shape %s), on one device with the others", what, name,
                     s.substr(0, s.size() - 2).c_str());
        throw Refused();
    }
    return t.const_data_ptr<int32_t>();
}

// The C struct of a RopeAxes or KV8Cache, whose tensors have to be on device `dev`.
template <class S>
struct Handle {
    S s;
    int device;
};
template <class S>
const S* handle(const char* what, PyObject* o, PyObject* cls, int dev) {
    if (!PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(cls))) {
        PyErr_Format(PyExc_TypeError, "%s: expected a %s", what, reinterpret_cast<PyTypeObject*>(cls)->tp_name);
        throw Refused();
    }
    PyObject* r = PyObject_GetAttr(o, s_ref);
    if (!r) throw Refused();
    const auto* p = static_cast<const Handle<S>*>(PyLong_AsVoidPtr(r));
    Py_DECREF(r);
    if (!p) throw Refused();
    if (p->device != dev) refuse(what, "the tensors, the cache and the tables must be CUDA tensors on one device");
    return &p->s;
}

// The current stream of the tensors' device, which has to be the current device.
void* stream_of(const char* what, int dev) {
    if (dev != c10::cuda::current_device()) refuse(what, "the tensors are not on the current device");
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
}

void done(int status, const char* what, const char* name) {
    if (status != TCQ_OK) {
        PyErr_Format(g_error, "%s: %s (status %d)", what, f_status(status), status);
        throw Refused();
    }
    PyObject* key = PyUnicode_InternFromString(name);
    PyObject* old = key ? PyDict_GetItemWithError(g_launches, key) : nullptr;
    PyObject* now = key ? PyLong_FromLong((old ? PyLong_AsLong(old) : 0) + 1) : nullptr;
    const bool bad = !now || PyDict_SetItem(g_launches, key, now) < 0;
    Py_XDECREF(key);
    Py_XDECREF(now);
    if (bad) throw Refused();
}

// Truth of an argument; what has none raises its own error.
int flag(PyObject* o) {
    const int t = PyObject_IsTrue(o);
    if (t < 0) throw Refused();
    return t;
}

// Distance of a dimension's steps in elements; nothing steps along one of size one, whatever stride its tensor states.
int64_t step(const at::Tensor& t, int dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

int extent(const char* what, int64_t n) {
    if (n > INT32_MAX) refuse(what, "a size passes 31 bits");
    return static_cast<int>(n);
}

template <class F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F body) {
    HANDLE_TH_ERRORS
    if (given != wanted) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    try {
        return body();
    } catch (const Refused&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// rope_axes(x, pos, rope, inverse, out)
PyObject* rope_axes(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 5, [&]() -> PyObject* {
        const char* me = "rope_axes";
        const at::Tensor &x = tensor(me, a[0], "x"), &pos = tensor(me, a[1], "pos");
        const int inverse = flag(a[3]), dev = x.is_cuda() ? x.get_device() : -1;
        const auto* plan = handle<tcq_rope_plan>(me, a[2], g_rope_class, dev);
        rows(me, "x", x, dev);
        const int64_t B = x.size(0), T = x.size(1), W = x.size(2);
        if (W % plan->head_dim) refuse(me, "x's rows are no multiple of the head width");
        const int dt = dtype_code(me, x, true);
        const int32_t* p = ints(me, "pos", pos, {plan->axes, B, T}, dev);
        at::Tensor made;
        if (a[4] == Py_None) made = at::empty({B, T, W}, x.options());
        const at::Tensor& out = a[4] == Py_None ? made : tensor(me, a[4], "out");
        rows(me, "out", out, dev);
        if (out.sizes() != x.sizes() || out.scalar_type() != x.scalar_type()) refuse(me, "out must have the shape and type of x");
        done(f_rope(x.const_data_ptr(), dt, step(x, 0), step(x, 1), out.data_ptr(), step(out, 0), step(out, 1), p, plan, extent(me, B),
                    extent(me, T), extent(me, W / plan->head_dim), inverse, stream_of(me, dev)),
             "tcq_rope_axes", me);
        if (a[4] == Py_None) return THPVariable_Wrap(made);
        return Py_NewRef(a[4]);
    });
}

// kv8_append(cache, k, v, table, start, count, rope, pos)
PyObject* kv8_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const char* me = "kv8_append";
        const at::Tensor &k = tensor(me, a[1], "k"), &v = tensor(me, a[2], "v"), &table = tensor(me, a[3], "table"), &start = tensor(me, a[4], "start");
        const int dev = k.is_cuda() ? k.get_device() : -1;
        const auto* c = handle<tcq_kv8_cache>(me, a[0], g_cache_class, dev);
        rows(me, "k", k, dev);
        rows(me, "v", v, dev);
        const int64_t B = k.size(0), T = k.size(1);
        if (k.size(2) != (int64_t)c->kv_heads * c->head_dim) refuse(me, "k's rows are not kv_heads * head_dim wide");
        if (v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type()) refuse(me, "k and v must have the same shape and type");
        if ((a[6] == Py_None) != (a[7] == Py_None)) refuse(me, "give rope and pos, or neither");
        const int dt = dtype_code(me, k, false);
        const int64_t blocks = table.dim() == 2 ? table.size(1) : 0;
        const int32_t* tp = ints(me, "table", table, {B, blocks}, dev);
        const int32_t* sp = ints(me, "start", start, {B}, dev);
        const int32_t* cp = a[5] == Py_None ? nullptr : ints(me, "count", tensor(me, a[5], "count"), {B}, dev);
        const auto* plan = a[6] == Py_None ? nullptr : handle<tcq_rope_plan>(me, a[6], g_rope_class, dev);
        const int32_t* pp = plan ? ints(me, "pos", tensor(me, a[7], "pos"), {plan->axes, B, T}, dev) : nullptr;
        done(f_append(c, k.const_data_ptr(), step(k, 0), step(k, 1), v.const_data_ptr(), step(v, 0), step(v, 1), dt, tp, extent(me, blocks), sp,
                      cp, pp, plan, extent(me, B), extent(me, T), stream_of(me, dev)),
             "tcq_kv8_append", me);
        Py_RETURN_NONE;
    });
}

// kv8_read(cache, table, begin, lens, tokens, dtype, out)
PyObject* kv8_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&]() -> PyObject* {
        const char* me = "kv8_read";
        const at::Tensor &table = tensor(me, a[1], "table"), &begin = tensor(me, a[2], "begin"), &lens = tensor(me, a[3], "lens");
        const int64_t T = PyLong_AsLongLong(a[4]);
        if (T == -1 && PyErr_Occurred()) return nullptr;
        const int dev = table.is_cuda() ? table.get_device() : -1;
        const auto* c = handle<tcq_kv8_cache>(me, a[0], g_cache_class, dev);
        const int64_t B = table.dim() == 2 ? table.size(0) : 0, blocks = table.dim() == 2 ? table.size(1) : 0, W = (int64_t)c->kv_heads * c->head_dim;
        const int32_t* tp = ints(me, "table", table, {B, blocks}, dev);
        const int32_t* bp = ints(me, "begin", begin, {B}, dev);
        const int32_t* lp = ints(me, "lens", lens, {B}, dev);
        if (T < 1) refuse(me, "at least one token");
        at::Tensor mk, mv;
        const at::Tensor *k = &mk, *v = &mv;
        if (a[6] == Py_None) {
            if (!THPDtype_Check(a[5])) refuse(me, "dtype must be a torch.dtype");
            const auto opt = table.options().dtype(reinterpret_cast<THPDtype*>(a[5])->scalar_type);
            mk = at::empty({B, T, W}, opt);
            mv = at::empty({B, T, W}, opt);
        } else {
            if (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 2) refuse(me, "out must be a pair of tensors");
            k = &tensor(me, PyTuple_GET_ITEM(a[6], 0), "out[0]");
            v = &tensor(me, PyTuple_GET_ITEM(a[6], 1), "out[1]");
        }
        const std::array<int64_t, 3> want{B, T, W};
        if (k->sizes() != at::IntArrayRef(want) || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() || !k->is_contiguous() ||
            !v->is_contiguous() || !k->is_cuda() || !v->is_cuda() || k->get_device() != dev || v->get_device() != dev)
            refuse(me, "out must be two contiguous CUDA tensors (B, tokens, kv_heads * D) of one type");
        done(f_read(c, k->data_ptr(), v->data_ptr(), dtype_code(me, *k, true), tp, extent(me, blocks), bp, lp, extent(me, B), extent(me, T),
                    stream_of(me, dev)),
             "tcq_kv8_read", me);
        if (a[6] != Py_None) return Py_NewRef(a[6]);
        return Py_BuildValue("(NN)", THPVariable_Wrap(mk), THPVariable_Wrap(mv));
    });
}

// Workspace of the attention for a stream. Outside captures: one per device and stream, grown on demand, replaced in the stream's
// order. In a capture the graph gets one of its own: allocated in the capture, so that it lives in the graph's memory pool, with
// its counters cleared by a node of the graph, so that the graph may be replayed before, after or (on another stream) next to any
// other call. A graph is never handed the stream's own workspace, whose address a later call may change. The capture's is let go by
// the first call on the stream that belongs to another capture or to none; the memory stays with the pool.
// Entries are kept until the process ends (a destructor would run after the CUDA context is gone).
void* workspace(int dev, void* stream, size_t need, size_t& have) {
    struct Entry {
        int dev;
        void* stream;
        unsigned long long capture;
        at::Tensor own, captured;
    };
    static auto* all = new std::vector<Entry>();
    Entry* e = nullptr;
    for (auto& x : *all)
        if (x.dev == dev && x.stream == stream) e = &x;
    if (!e) {
        all->push_back({dev, stream, 0, at::Tensor(), at::Tensor()});
        e = &all->back();
    }
    unsigned long long capture = 0;
    f_capture(stream, &capture);
    if (e->capture != capture) {
        e->captured.reset();
        e->capture = capture;
    }
    at::Tensor& t = capture ? e->captured : e->own;
    if (!t.defined() || static_cast<size_t>(t.numel()) < need) {
        t.reset();
        t = at::empty({static_cast<int64_t>(need)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(dev)));
        t.narrow(0, 0, std::min<int64_t>(t.numel(), TCQ_KV8_ZEROED_BYTES)).zero_();
    }
    have = static_cast<size_t>(t.numel());
    return t.data_ptr();
}

// kv8_attention(q, cache, table, lens, count, causal, scale, out)
PyObject* kv8_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const char* me = "kv8_attention";
        const at::Tensor &q = tensor(me, a[0], "q"), &table = tensor(me, a[2], "table"), &lens = tensor(me, a[3], "lens");
        const int dev = q.is_cuda() ? q.get_device() : -1;
        const auto* c = handle<tcq_kv8_cache>(me, a[1], g_cache_class, dev);
        rows(me, "q", q, dev);
        const int64_t B = q.size(0), T = q.size(1), W = q.size(2), D = c->head_dim, heads = W / D;
        if (W % D || heads % c->kv_heads) refuse(me, "q's rows are no multiple of kv_heads * head_dim");
        const int dt = dtype_code(me, q, false);
        const int64_t blocks = table.dim() == 2 ? table.size(1) : 0;
        const int32_t* tp = ints(me, "table", table, {B, blocks}, dev);
        const int32_t* lp = ints(me, "lens", lens, {B}, dev);
        const int32_t* cp = a[4] == Py_None ? nullptr : ints(me, "count", tensor(me, a[4], "count"), {B}, dev);
        const int causal = flag(a[5]);
        const double scale = a[6] == Py_None ? 1.0 / std::sqrt((double)D) : PyFloat_AsDouble(a[6]);
        if (scale == -1.0 && PyErr_Occurred()) return nullptr;
        at::Tensor made;
        if (a[7] == Py_None) made = at::empty({B, T, W}, q.options());
        const at::Tensor& out = a[7] == Py_None ? made : tensor(me, a[7], "out");
        if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous() || !out.is_cuda() || out.get_device() != dev)
            refuse(me, "out must be contiguous and have the shape, type and device of q");
        void* st = stream_of(me, dev);
        const int b = extent(me, B), t = extent(me, T), h = extent(me, heads), bl = extent(me, blocks);
        size_t have = 0;
        void* ws = workspace(dev, st, f_workspace(b, t, h, c->kv_heads, c->head_dim, bl), have);
        done(f_attention(c, q.const_data_ptr(), dt, step(q, 0), step(q, 1), out.data_ptr(), tp, bl, lp, cp, causal, (float)scale, b, t, h, ws,
                         have, st),
             "tcq_kv8_attention", me);
        if (a[7] == Py_None) return THPVariable_Wrap(made);
        return Py_NewRef(a[7]);
    });
}

// init(addresses of the C functions by name, error class, launch counts, RopeAxes, KV8Cache)
PyObject* init(PyObject*, PyObject* args) {
    PyObject* f;
    if (!PyArg_ParseTuple(args, "O!OO!OO", &PyDict_Type, &f, &g_error, &PyDict_Type, &g_launches, &g_rope_class, &g_cache_class)) return nullptr;
    for (PyObject* o : {g_error, g_launches, g_rope_class, g_cache_class}) Py_INCREF(o);
    auto take = [&](const char* name, auto& fn) {
        PyObject* p = PyDict_GetItemString(f, name);
        void* at = p ? PyLong_AsVoidPtr(p) : nullptr;
        fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(at);
        return at != nullptr;
    };
    if (!take("tcq_status_string", f_status) || !take("tcq_rope_axes", f_rope) || !take("tcq_kv8_append", f_append) || !take("tcq_kv8_read", f_read) ||
        !take("tcq_kv8_attention_workspace", f_workspace) || !take("tcq_kv8_attention", f_attention) ||
        !take("tcq_capture_id", f_capture)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, "a function address is missing");
        return nullptr;
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"init", init, METH_VARARGS, nullptr},
    {"rope_axes", reinterpret_cast<PyCFunction>(rope_axes), METH_FASTCALL, nullptr},
    {"kv8_append", reinterpret_cast<PyCFunction>(kv8_append), METH_FASTCALL, nullptr},
    {"kv8_read", reinterpret_cast<PyCFunction>(kv8_read), METH_FASTCALL, nullptr},
    {"kv8_attention", reinterpret_cast<PyCFunction>(kv8_attention), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "Binding of the streaming-memory entry points (see kernels.py).", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() {
    if (Py_Version >> 16 != PY_VERSION_HEX >> 16) {
        PyErr_Format(PyExc_ImportError, "it is built for Python %d.%d", PY_MAJOR_VERSION, PY_MINOR_VERSION);
        return nullptr;
    }
    s_ref = PyUnicode_InternFromString("ref");
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TCQ_TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
