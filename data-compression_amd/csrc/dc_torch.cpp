// dc_torch.cpp -- the fixed-rate operators of include/dc_gpu.h for torch tensors (module dcamd_torch, used by dcamd.py): checks
// of shapes, types and devices, new outputs and workspaces from torch, launches on torch's current stream.  A CPython
// extension over ATen's headers, because single tokens are bound by the host's side of a call: 8.4 us through ctypes and
// Python for a call with two outputs.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <algorithm>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include "../../include/dc_gpu.h"

namespace {

using at::Tensor;

PyObject* g_error = nullptr;            // dcamd.DCError

#define REFUSE(...) \
    do { \
        PyErr_Format(PyExc_ValueError, __VA_ARGS__); \
        return nullptr; \
    } while (0)
#define ARGS(n) \
    if (count != n) REFUSE("%d arguments are needed", n)

// a Python argument as a tensor (None: nullptr; anything else: an error)
bool tensor_of(PyObject* o, const char* name, bool optional, const Tensor** t) {
    *t = nullptr;
    if (optional && o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: a tensor is needed", name);
        return false;
    }
    *t = &THPVariable_Unpack(o);
    if ((*t)->is_neg()) {                                   // (its memory holds the other sign)
        PyErr_Format(PyExc_ValueError, "%s: a negative view is not taken (resolve_neg() it)", name);
        return false;
    }
    return true;
}
#define TENSOR(i, name, optional) \
    const Tensor* name; \
    if (!tensor_of(args[i], #name, optional, &name)) return nullptr

int code_of(at::ScalarType t) {
    return t == at::kFloat ? DC_F32 : t == at::kHalf ? DC_F16 : t == at::kBFloat16 ? DC_BF16 : -1;
}
bool known(const Tensor& t) {
    if (code_of(t.scalar_type()) >= 0) return true;
    PyErr_SetString(PyExc_ValueError, "dtype: f32, f16 or bf16 is needed");
    return false;
}

// all tensors on one GPU, the library's and the current one.  The library starts on the first call's device, which has to be the
// current one before it does, as starting makes it that; and not in a capture, as starting allocates
bool on_gpu(std::initializer_list<const Tensor*> ts) {
    int dev = dc_get_device();
    const bool starts = dev < 0;
    if (starts && (*ts.begin())->is_cuda()) dev = c10::hip::current_device();
    for (const Tensor* t : ts)
        if (t && (!t->is_cuda() || t->get_device() != dev)) {
            PyErr_SetString(PyExc_ValueError, starts ? "tensors must lie on the GPU, on the current device" : "tensors must lie on the GPU, on the library's device");
            return false;
        }
    if (starts) {
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) {
            PyErr_SetString(PyExc_ValueError, "the library's first call cannot be captured: make one before");
            return false;
        }
        if (dc_init(dev)) {
            PyErr_Format(g_error, "dc_init: %s", dc_last_error());
            return false;
        }
        dev = dc_get_device();                              // (another thread may have been first)
    }
    if (c10::hip::current_device() != dev) {
        PyErr_Format(PyExc_ValueError, "the current device must be the library's (cuda:%d)", dev);
        return false;
    }
    return true;
}
void* stream_of() { return c10::hip::getCurrentHIPStream().stream(); }
PyObject* failed(const char* what, int rc) {
    PyErr_Format(g_error, "%s -> %d: %s", what, rc, dc_last_error());
    return nullptr;
}

// whether two places of a tensor, or of two tensors of these sizes and strides `apart` elements apart, are the same one.  The
// dimensions, ordered by their strides, have to lie within one another (else true: such layouts are not taken)
bool nested(const Tensor& x, int (&order)[4]) {
    int n = 0;
    for (int i = 0; i < 4; i++)
        if (x.size(i) > 1) order[n++] = i;
    for (int i = n; i < 4; i++) order[i] = -1;
    std::sort(order, order + n, [&](int a, int b) { return x.stride(a) < x.stride(b); });
    int64_t reach = 0;                                      // of the dimensions so far
    for (int i = 0; i < n; i++) {
        if (x.stride(order[i]) <= reach) return false;
        reach += (x.size(order[i]) - 1) * x.stride(order[i]);
    }
    return true;
}
bool meets(const Tensor& x, const int (&order)[4], int from, int64_t apart) {
    if (from < 0) return apart == 0;
    if (order[from] < 0) return meets(x, order, from - 1, apart);
    const int64_t s = x.stride(order[from]), most = x.size(order[from]) - 1, c = apart / s;
    for (int64_t k = c - 1; k <= c + 1; k++)
        if (k >= -most && k <= most && meets(x, order, from - 1, apart - k * s)) return true;
    return false;
}

// (batch, tokens, heads, head_dim) rows: their strides; heads 0: any number.  Outputs' rows do not lie on one another
bool rows_of(const Tensor& x, const char* name, int64_t heads, int64_t dim, bool output, long long* s) {
    if (x.dim() != 4 || x.size(3) != dim || (heads && x.size(2) != heads)) {
        if (heads) PyErr_Format(PyExc_ValueError, "%s: (batch, tokens, %lld, %lld) is needed", name, (long long)heads, (long long)dim);
        else PyErr_Format(PyExc_ValueError, "%s: (batch, tokens, heads, %lld) is needed", name, (long long)dim);
        return false;
    }
    const auto st = x.strides();
    if (st[3] != 1 && x.numel()) {
        PyErr_Format(PyExc_ValueError, "%s: a head's values must be consecutive", name);
        return false;
    }
    for (int i = 0; i < 3; i++) s[i] = st[i];
    int order[4];
    if (output && x.numel() && !nested(x, order)) {
        PyErr_Format(PyExc_ValueError, "%s: rows must not lie on one another", name);
        return false;
    }
    return true;
}

bool ints_of(const Tensor& t, const char* name, int64_t batch) {
    if (t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == batch && t.is_contiguous()) return true;
    PyErr_Format(PyExc_ValueError, "%s: contiguous int32 of (%lld,) is needed", name, (long long)batch);
    return false;
}

bool positions_of(const dc_kv_cache& c, int64_t batch, int64_t tokens, const Tensor& start, const char* what, const Tensor* table,
                  const Tensor* lens, bool zero_padding, dc_kv_batch* at) {
    if (batch > INT_MAX || tokens > INT_MAX) {
        PyErr_SetString(PyExc_ValueError, "too many tokens in one call");
        return false;
    }
    if (!ints_of(start, what, batch) || (lens && !ints_of(*lens, "lens", batch))) return false;
    *at = {(int)batch, (int)tokens, (const int*)start.data_ptr(), lens ? (const int*)lens->data_ptr() : nullptr, nullptr, 0, 0, zero_padding};
    if (!table) {
        if (batch <= c.pages) return true;
        PyErr_SetString(PyExc_ValueError, "without a table each sequence has a page");
        return false;
    }
    if (table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != batch || table->size(1) < 1 || table->size(1) > INT_MAX ||
        table->stride(1) != 1 || (batch > 1 && table->stride(0) < table->size(1))) {
        PyErr_Format(PyExc_ValueError, "table: int32 of (%lld, pages of a sequence) with consecutive entries is needed", (long long)batch);
        return false;
    }
    at->table = (const int*)table->data_ptr();
    at->table_width = (int)table->size(1);
    at->table_stride = std::max(table->stride(0), table->size(1));
    return true;
}

// the cache is the address of a dc_kv_cache, held with its buffer by a KVCache
#define CACHE \
    const dc_kv_cache& c = *(const dc_kv_cache*)PyLong_AsVoidPtr(args[0]); \
    if (PyErr_Occurred()) return nullptr; \
    TENSOR(1, buffer, false); \
    if (buffer->data_ptr() != c.data || !buffer->is_contiguous() || \
        buffer->nbytes() < (size_t)c.pages * dc_kv_page_bytes(c.page_size, c.heads, c.head_dim, c.bits)) \
        REFUSE("buffer: the one the cache was made with is needed")

// write(cache, buffer, k, v, start, table, lens)
PyObject* kv_write(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGS(7);
    CACHE;
    TENSOR(2, k, false);
    TENSOR(3, v, false);
    TENSOR(4, start, false);
    TENSOR(5, table, true);
    TENSOR(6, lens, true);
    long long ks[3], vs[3];
    if (!rows_of(*k, "k", c.heads, c.head_dim, false, ks) || !rows_of(*v, "v", c.heads, c.head_dim, false, vs)) return nullptr;
    if (k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type()) REFUSE("k and v differ in shape or type");
    dc_kv_batch at;
    if (!known(*k) || !positions_of(c, k->size(0), k->size(1), *start, "start", table, lens, false, &at) ||
        !on_gpu({buffer, k, v, start, table, lens}))
        return nullptr;
    void* stream = stream_of();
    int rc;
    const void *pk = k->data_ptr(), *pv = v->data_ptr();
    Py_BEGIN_ALLOW_THREADS
    rc = dc_kv_write_device(&c, &at, code_of(k->scalar_type()), pk, ks, pv, vs, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed("kv_write", rc);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// read(cache, buffer, start, tokens, table, lens, dtype code, k, v); k, v None: new ones
PyObject* kv_read(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGS(9);
    CACHE;
    TENSOR(2, start, false);
    const long long tokens = PyLong_AsLongLong(args[3]), code = PyLong_AsLongLong(args[6]);
    if (PyErr_Occurred()) return nullptr;
    TENSOR(4, table, true);
    TENSOR(5, lens, true);
    TENSOR(7, k, true);
    TENSOR(8, v, true);
    if (tokens < 0) REFUSE("tokens is not negative");
    const int64_t batch = start->dim() ? start->size(0) : 0;
    Tensor nk, nv;
    long long ks[3], vs[3];
    dc_kv_batch at;
    if (k || v) {
        if (!k || !v) REFUSE("out: two tensors are needed");
        if (!rows_of(*k, "out", c.heads, c.head_dim, true, ks) || !rows_of(*v, "out", c.heads, c.head_dim, true, vs) || !known(*k)) return nullptr;
        if (k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() || k->size(0) != batch || k->size(1) != tokens ||
            (code >= 0 && code != code_of(k->scalar_type())))
            REFUSE("out: two tensors (batch, tokens, heads, head_dim) of the type asked for are needed");
        int order[4];
        const int64_t apart = (const char*)v->data_ptr() - (const char*)k->data_ptr(), size = (int64_t)k->element_size();
        if (k->numel() && k->strides() == v->strides() && apart % size == 0 && nested(*k, order) && meets(*k, order, 3, apart / size))
            REFUSE("out: keys and values must not lie on one another");
        if (!positions_of(c, batch, tokens, *start, "start", table, lens, false, &at) || !on_gpu({buffer, start, table, lens, k, v}))
            return nullptr;
    } else {
        if (!positions_of(c, batch, tokens, *start, "start", table, lens, true, &at) || !on_gpu({buffer, start, table, lens}))
            return nullptr;
        const auto o = buffer->options().dtype(code == DC_F32 ? at::kFloat : code == DC_F16 ? at::kHalf : at::kBFloat16);
        nk = at::empty({batch, (int64_t)tokens, c.heads, c.head_dim}, o);
        nv = at::empty(nk.sizes(), o);
        for (int i = 0; i < 3; i++) ks[i] = vs[i] = nk.stride(i);
        k = &nk;
        v = &nv;
    }
    void* stream = stream_of();
    int rc;
    void *pk = k->data_ptr(), *pv = v->data_ptr();
    Py_BEGIN_ALLOW_THREADS
    rc = dc_kv_read_device(&c, &at, code_of(k->scalar_type()), pk, ks, pv, vs, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed("kv_read", rc);
    return Py_BuildValue("(NN)", THPVariable_Wrap(*k), THPVariable_Wrap(*v));
    END_HANDLE_TH_ERRORS
}

// attention(cache, buffer, q, context, table, lens, scale, causal, max_context (-1: the table's), out, lse)
PyObject* kv_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGS(11);
    CACHE;
    TENSOR(2, q, false);
    TENSOR(3, context, false);
    TENSOR(4, table, true);
    TENSOR(5, lens, true);
    TENSOR(9, out, true);
    TENSOR(10, lse, true);
    const double scale = PyFloat_AsDouble(args[6]);
    const int causal = PyObject_IsTrue(args[7]);
    long long limit = PyLong_AsLongLong(args[8]);
    if (PyErr_Occurred()) return nullptr;
    long long qs[3], os[3];
    if (!rows_of(*q, "q", 0, c.head_dim, false, qs)) return nullptr;
    const int code = code_of(q->scalar_type());
    if (code != DC_F16 && code != DC_BF16) REFUSE("q: f16 or bf16 is needed");
    const int64_t batch = q->size(0), tokens = q->size(1), heads = q->size(2);
    if (heads < 1 || heads % c.heads || heads > INT_MAX) REFUSE("q: heads in a multiple of the cache's %d are needed", c.heads);
    dc_kv_batch at;
    if (!positions_of(c, batch, tokens, *context, "context", table, lens, !out, &at)) return nullptr;
    const long long capacity = (long long)c.page_size * (table ? at.table_width : 1);
    if (limit < -1) REFUSE("max_context is not negative");
    if (limit < 0 || limit > capacity) limit = capacity;
    if (lse && (lse->scalar_type() != at::kFloat || lse->sizes() != q->sizes().slice(0, 3) || !lse->is_contiguous()))
        REFUSE("lse: contiguous float32 of (batch, tokens, q_heads) is needed");
    if (out) {
        if (!rows_of(*out, "out", 0, c.head_dim, true, os)) return nullptr;
        if (out->sizes() != q->sizes() || out->scalar_type() != q->scalar_type()) REFUSE("out: q's shape and type are needed");
    }
    if (!on_gpu({buffer, q, context, table, lens, lse, out})) return nullptr;
    Tensor made, space;
    if (!out) {
        made = at::empty(q->sizes(), q->options());
        out = &made;
        for (int i = 0; i < 3; i++) os[i] = made.stride(i);
    }
    const size_t need = dc_kv_attention_workspace(&c, (int)batch, (int)tokens, (int)heads, limit);
    if (need) space = at::empty({(int64_t)need}, buffer->options());
    void* stream = stream_of();
    int rc;
    const void* pq = q->data_ptr();
    void *po = out->data_ptr(), *ps = need ? space.data_ptr() : nullptr;
    float* pl = lse ? (float*)lse->data_ptr() : nullptr;
    Py_BEGIN_ALLOW_THREADS
    rc = dc_kv_attention_device(&c, &at, code, (int)heads, pq, qs, (float)scale, causal, limit, po, os, pl, ps, need, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed("kv_attention", rc);
    return THPVariable_Wrap(*out);
    END_HANDLE_TH_ERRORS
}

// x as rows of its last dimension (contiguous: one row); copied if its rows do not lie so
struct Flat {
    Tensor x;
    long long rows, cols, ld;
};
Flat flat(const Tensor& x) {
    const int64_t n = x.numel();
    if (x.is_contiguous()) return {x, 1, n, n};
    const int64_t cols = x.size(-1);
    Tensor y = x.reshape({n / cols, cols});
    if (y.stride(1) != 1 || y.stride(0) < cols) y = y.contiguous();
    return {y, y.size(0), cols, std::max(y.stride(0), cols)};
}
// two of one shape with one's rows: an array in one row takes the other's
void alike(Flat& a, Flat& b) {
    if (a.rows == 1 && b.rows > 1) a.rows = b.rows, a.cols = a.ld = b.cols;
    else if (b.rows == 1 && a.rows > 1) b.rows = a.rows, b.cols = b.ld = a.cols;
}
bool holds(const Tensor* kept, int64_t n) {
    if (!kept || (kept->scalar_type() == at::kByte && kept->is_contiguous() && kept->numel() >= (int64_t)dc_act_bytes(n))) return true;
    PyErr_Format(PyExc_ValueError, "checkpoint: %lld contiguous bytes (uint8) are needed", (long long)dc_act_bytes(n));
    return false;
}
Tensor kept_for(const Tensor& x) { return at::empty({(int64_t)dc_act_bytes(x.numel())}, x.options().dtype(at::kByte)); }

// forward(x, kind, up) -> (y, kept, kept_up); kind 0: the checkpoint alone, y None
PyObject* act_forward(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGS(3);
    TENSOR(0, x, false);
    const long kind = PyLong_AsLong(args[1]);
    if (PyErr_Occurred()) return nullptr;
    TENSOR(2, up, true);
    if (!known(*x)) return nullptr;
    if (up && (up->sizes() != x->sizes() || up->scalar_type() != x->scalar_type())) REFUSE("x and up differ in shape or type");
    if (!on_gpu({x, up})) return nullptr;
    Flat fx = flat(*x), fu = {};
    if (up) {
        fu = flat(*up);
        alike(fx, fu);
    }
    Tensor y, kept = kept_for(*x), kept_up;
    if (kind) y = at::empty(x->sizes(), x->options());
    if (up) kept_up = kept_for(*x);
    void* stream = stream_of();
    int rc;
    const void *px = fx.x.data_ptr(), *pu = up ? fu.x.data_ptr() : nullptr;
    void *py = kind ? y.data_ptr() : nullptr, *pk = kept.data_ptr(), *pv = up ? kept_up.data_ptr() : nullptr;
    const int code = code_of(x->scalar_type());
    Py_BEGIN_ALLOW_THREADS
    rc = dc_act_forward_device((int)kind, code, fx.rows, fx.cols, px, fx.ld, pu, fu.ld, py, fx.cols, pk, pv, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed("act_forward", rc);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(y), THPVariable_Wrap(kept), THPVariable_Wrap(kept_up));   // (undefined: None)
    END_HANDLE_TH_ERRORS
}

// backward(dy, kept, kept_up, kind, recompute) -> (dx[, dup][, y])
PyObject* act_backward(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGS(5);
    TENSOR(0, dy, false);
    TENSOR(1, kept, false);
    TENSOR(2, kept_up, true);
    const long kind = PyLong_AsLong(args[3]);
    const int again = PyObject_IsTrue(args[4]);
    if (PyErr_Occurred()) return nullptr;
    if (!known(*dy) || !holds(kept, dy->numel()) || !holds(kept_up, dy->numel()) || !on_gpu({dy, kept, kept_up})) return nullptr;
    const Flat fd = flat(*dy);
    Tensor dx = at::empty(dy->sizes(), dy->options()), dup, y;
    if (kept_up) dup = at::empty(dy->sizes(), dy->options());
    if (again) y = at::empty(dy->sizes(), dy->options());
    void* stream = stream_of();
    int rc;
    const void *pd = fd.x.data_ptr(), *pk = kept->data_ptr(), *pv = kept_up ? kept_up->data_ptr() : nullptr;
    void *px = dx.data_ptr(), *pu = kept_up ? dup.data_ptr() : nullptr, *py = again ? y.data_ptr() : nullptr;
    const int code = code_of(dy->scalar_type());
    Py_BEGIN_ALLOW_THREADS
    rc = dc_act_backward_device((int)kind, code, fd.rows, fd.cols, pd, fd.ld, pk, pv, px, fd.cols, pu, fd.cols, py, fd.cols, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed("act_backward", rc);
    if (kept_up && again) return Py_BuildValue("(NNN)", THPVariable_Wrap(dx), THPVariable_Wrap(dup), THPVariable_Wrap(y));
    if (kept_up || again) return Py_BuildValue("(NN)", THPVariable_Wrap(dx), THPVariable_Wrap(again ? y : dup));
    return Py_BuildValue("(N)", THPVariable_Wrap(dx));
    END_HANDLE_TH_ERRORS
}

// load(kept, dtype code, shape...) -> x
PyObject* act_load(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count < 2) REFUSE("2 arguments or more are needed");
    TENSOR(0, kept, false);
    const long code = PyLong_AsLong(args[1]);
    c10::SmallVector<int64_t, 6> shape;
    for (Py_ssize_t i = 2; i < count; i++) shape.push_back(PyLong_AsLongLong(args[i]));
    if (PyErr_Occurred()) return nullptr;
    if (!holds(kept, c10::multiply_integers(shape)) || !on_gpu({kept})) return nullptr;
    Tensor x = at::empty(shape, kept->options().dtype(code == DC_F32 ? at::kFloat : code == DC_F16 ? at::kHalf : at::kBFloat16));
    void* stream = stream_of();
    int rc;
    const void* pk = kept->data_ptr();
    void* px = x.data_ptr();
    const long long n = x.numel();
    Py_BEGIN_ALLOW_THREADS
    rc = dc_act_backward_device(DC_ACT_NONE, (int)code, 1, n, nullptr, 0, pk, nullptr, px, n, nullptr, 0, nullptr, 0, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed("act_load", rc);
    return THPVariable_Wrap(x);
    END_HANDLE_TH_ERRORS
}

// status(reset) -> the sticky word after the work queued on torch's current stream
PyObject* kv_status(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGS(1);
    unsigned word = 0;
    const int reset = PyObject_IsTrue(args[0]);
    if (dc_get_device() < 0) return PyLong_FromLong(0);     // (nothing has run)
    void* stream = stream_of();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = dc_kv_status(stream, &word, reset);
    Py_END_ALLOW_THREADS
    if (rc) return failed("kv_status", rc);
    return PyLong_FromUnsignedLong(word);
    END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
    Py_INCREF(cls);
    g_error = cls;
    Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void*)name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(kv_write), FAST(kv_read), FAST(kv_attention), FAST(kv_status), FAST(act_forward), FAST(act_backward),
                         FAST(act_load), {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "dcamd_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dcamd_torch(void) { return PyModule_Create(&module_def); }
