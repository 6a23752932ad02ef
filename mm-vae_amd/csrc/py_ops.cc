// mmvae_amd._ops: the layer operators' calls on torch tensors (mmvae_amd/ops.py holds their
// documentation and the differentiable forms).  A call checks its tensors, allocates its results on
// the current stream of their device and makes the C call of mmvae_capi.h; in C++ because the calls
// of small layers cost more on the host than on the GPU: a norm's forward takes 11.7 us of host time
// through ctypes, its launch 3.3.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <stdexcept>
#include <string>

#include "../../include/mmvae_capi.h"

namespace {

PyObject* g_error = nullptr;  // mmvae_amd.MMVAEError

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
[[noreturn]] void wrong(const std::string& what) { throw Refused(what); }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) wrong(std::string(name) + " must be a CUDA tensor");
    return THPVariable_Unpack(o);
}
int type_code(at::ScalarType t) {
    return t == at::kFloat ? MMVAE_T_F32 : t == at::kBFloat16 ? MMVAE_T_BF16 : t == at::kHalf ? MMVAE_T_F16 : -1;
}

// a tensor as [rows][N] with unit column stride: a view where it is one, else a copy (kept alive here)
struct Rows {
    at::Tensor copy;
    const void* p;
    int64_t M, N, ld;
    int dtype, device;
    Rows(const at::Tensor& t, const char* name) {
        if (!t.is_cuda()) wrong(std::string(name) + " must be a CUDA tensor");
        dtype = type_code(t.scalar_type());
        if (dtype < 0) wrong(std::string(name) + ": float32, bfloat16 or float16");
        const int64_t d = t.dim();
        if (d == 0 || t.size(-1) == 0) wrong(std::string(name) + " needs a last dimension of at least 1");
        device = t.get_device();
        const at::Tensor* q = &t;
        if (t.is_neg()) {  // (a lazily negated view)
            copy = t.resolve_neg();
            q = &copy;
        }
        if (d != 2) {
            copy = q->reshape({-1, t.size(-1)});
            q = &copy;
        }
        if (q->stride(1) != 1 && q->size(1) > 1) {
            copy = q->contiguous();
            q = &copy;
        }
        M = q->size(0);
        N = q->size(1);
        ld = q->stride(0);
        p = q->const_data_ptr();
    }
};

void like(const at::Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type, int device) {
    if (!t.is_cuda() || t.sizes() != sizes || t.scalar_type() != type || t.get_device() != device)
        wrong(std::string(name) + " must have the shape, type and device of the other tensors");
}

struct Weights {
    const void *w = nullptr, *b = nullptr;
    int type = -1;
    at::ScalarType st = at::kFloat;
    void take(PyObject* o, const char* name, const Rows& x, const void** out) {
        if (o == Py_None) return;
        const at::Tensor& t = tensor(o, name);
        if (!t.is_cuda() || t.get_device() != x.device || t.dim() != 1 || t.size(0) != x.N)
            wrong(std::string(name) + " must be a tensor of [" + std::to_string(x.N) + "] on x's device");
        const int c = type_code(t.scalar_type());
        if (c < 0 || (c != x.dtype && c != MMVAE_T_F32)) wrong(std::string(name) + ": x's type or float32");
        if (!t.is_contiguous() || t.is_neg()) wrong(std::string(name) + " must be contiguous");
        if (type >= 0 && type != c) wrong("weight and bias must have one type");
        type = c;
        st = t.scalar_type();
        *out = t.const_data_ptr();
    }
    Weights(PyObject* wo, PyObject* bo, const Rows& x) {
        take(wo, "weight", x, &w);
        take(bo, "bias", x, &b);
        if (type < 0) type = MMVAE_T_F32;
    }
};

const int64_t* state_of(PyObject* o, const Rows& x) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, "state");
    if (!t.is_cuda() || t.get_device() != x.device || t.scalar_type() != at::kLong || t.numel() != 2 || !t.is_contiguous())
        wrong("state must be a contiguous int64 tensor [step, row_offset] on x's device");
    return static_cast<const int64_t*>(t.const_data_ptr());
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1. && PyErr_Occurred()) throw std::exception();
    return v;
}
uint64_t word(PyObject* o) {  // a whole number modulo 2^64
    const uint64_t v = PyLong_AsUnsignedLongLongMask(o);
    if (v == (uint64_t)-1 && PyErr_Occurred()) throw std::exception();
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw std::exception();
    return v != 0;
}

at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType t, int device) {
    return at::Tensor(at::detail::empty_cuda(sizes, at::TensorOptions().dtype(t).device(at::Device(at::kCUDA, (c10::DeviceIndex)device))));
}
void* stream_of(int device) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }
void check(int rc) {
    if (rc != MMVAE_OK) wrong(std::string(mmvae_last_error(nullptr)) + " (" + std::to_string(rc) + ")");
}
PyObject* wrap(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}
PyObject* triple(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) {
    PyObject* t = PyTuple_New(3);
    if (!t) throw std::exception();
    const at::Tensor* v[3] = {&a, &b, &c};
    for (int i = 0; i < 3; ++i) {
        PyObject* o = wrap(*v[i]);
        if (!o) {
            Py_DECREF(t);
            throw std::exception();
        }
        PyTuple_SET_ITEM(t, i, o);
    }
    return t;
}

// no C++ exception leaves a call
template <class F> PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F&& f) {
    if (n != want) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

// (x, weight, bias, eps, relu, p, seed, step, row_offset, state, stats) -> (y, mean, rstd)
PyObject* norm_forward(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 11, [&]() -> PyObject* {
        const at::Tensor& x = tensor(v[0], "x");
        const Rows r(x, "x");
        const Weights w(v[1], v[2], r);
        mmvae_norm_args a;
        std::memset(&a, 0, sizeof(a));
        a.M = r.M;
        a.N = r.N;
        a.x = r.p;
        a.ldx = r.ld;
        a.w = w.w;
        a.b = w.b;
        a.eps = (float)number(v[3]);
        a.relu = truth(v[4]) ? 1 : 0;
        a.p = number(v[5]);
        a.seed = word(v[6]);
        a.step = word(v[7]);
        a.row_offset = word(v[8]);
        a.state = state_of(v[9], r);
        at::Tensor y = fresh(x.sizes(), x.scalar_type(), r.device), mean, rstd;
        if (truth(v[10])) {
            const at::IntArrayRef s = x.sizes().slice(0, x.dim() - 1);
            mean = fresh(s, at::kFloat, r.device);
            rstd = fresh(s, at::kFloat, r.device);
            a.mean = (float*)mean.data_ptr();
            a.rstd = (float*)rstd.data_ptr();
        }
        a.y = y.data_ptr();
        a.ldy = r.N;
        a.stream = stream_of(r.device);
        a.device = r.device;
        a.dtype = r.dtype;
        a.wtype = w.type;
        check(mmvae_layer_norm_fwd(&a));
        return triple(y, mean, rstd);
    });
}

// (dy, x, mean, rstd, weight, bias, relu, p, seed, step, row_offset, state, need0, need1, need2) -> (dx, dw, db)
PyObject* norm_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 15, [&]() -> PyObject* {
        const at::Tensor &dy = tensor(v[0], "dy"), &x = tensor(v[1], "x");
        const Rows r(x, "x");
        like(dy, "dy", x.sizes(), x.scalar_type(), r.device);
        const Rows d(dy, "dy");
        const Weights w(v[4], v[5], r);
        mmvae_norm_args a;
        std::memset(&a, 0, sizeof(a));
        const at::Tensor* st[2] = {&tensor(v[2], "mean"), &tensor(v[3], "rstd")};
        for (const at::Tensor* t : st)
            if (!t->is_cuda() || t->scalar_type() != at::kFloat || t->get_device() != r.device || t->numel() != r.M || !t->is_contiguous())
                wrong("mean and rstd must be the forward's float32 statistics");
        a.M = r.M;
        a.N = r.N;
        a.x = r.p;
        a.ldx = r.ld;
        a.w = w.w;
        a.b = w.b;
        a.mean = (float*)const_cast<void*>(st[0]->const_data_ptr());
        a.rstd = (float*)const_cast<void*>(st[1]->const_data_ptr());
        a.dy = d.p;
        a.lddy = d.ld;
        a.relu = truth(v[6]) ? 1 : 0;
        a.p = number(v[7]);
        a.seed = word(v[8]);
        a.step = word(v[9]);
        a.row_offset = word(v[10]);
        a.state = state_of(v[11], r);
        at::Tensor dx, dw, db, ws;
        if (truth(v[12])) {
            dx = fresh(x.sizes(), x.scalar_type(), r.device);
            a.dx = dx.data_ptr();
        }
        a.lddx = r.N;
        if (truth(v[13])) {
            dw = fresh({r.N}, w.st, r.device);
            a.dw = dw.data_ptr();
        }
        if (truth(v[14])) {
            db = fresh({r.N}, w.st, r.device);
            a.db = db.data_ptr();
        }
        if (a.dw || a.db) {
            a.ws_bytes = mmvae_layer_norm_bwd_ws(r.M, r.N);
            if (a.ws_bytes > 0) {
                ws = fresh({a.ws_bytes}, at::kByte, r.device);
                a.ws = ws.data_ptr();
            }
        }
        a.stream = stream_of(r.device);
        a.device = r.device;
        a.dtype = r.dtype;
        a.wtype = w.type;
        check(mmvae_layer_norm_bwd(&a));
        return triple(dx, dw, db);
    });
}

// (x, p, seed, step, row_offset, state) -> y
PyObject* dropout(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 6, [&]() -> PyObject* {
        const at::Tensor& x = tensor(v[0], "x");
        const Rows r(x, "x");
        mmvae_dropout_args a;
        std::memset(&a, 0, sizeof(a));
        a.M = r.M;
        a.N = r.N;
        a.x = r.p;
        a.ldx = r.ld;
        a.p = number(v[1]);
        a.seed = word(v[2]);
        a.step = word(v[3]);
        a.row_offset = word(v[4]);
        a.state = state_of(v[5], r);
        at::Tensor y = fresh(x.sizes(), x.scalar_type(), r.device);
        a.y = y.data_ptr();
        a.ldy = r.N;
        a.stream = stream_of(r.device);
        a.device = r.device;
        a.dtype = r.dtype;
        check(mmvae_dropout(&a));
        return wrap(y);
    });
}

struct Ids {
    at::Tensor copy;
    const void* p;
    int64_t T;
    int32_t is64;
    Ids(const at::Tensor& t, int device) {
        if ((t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) || !t.is_cuda() || t.get_device() != device)
            wrong("ids must be an int64 or int32 tensor on the table's device");
        const at::Tensor* q = &t;
        if (!t.is_contiguous()) {
            copy = t.contiguous();
            q = &copy;
        }
        p = q->const_data_ptr();
        T = q->numel();
        is64 = t.scalar_type() == at::kLong;
    }
};

// (ids, table, scale, add) -> y
PyObject* embedding_forward(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 4, [&]() -> PyObject* {
        const at::Tensor &ids = tensor(v[0], "ids"), &table = tensor(v[1], "table");
        const Rows t(table, "table");
        if (table.dim() != 2) wrong("table must be [rows, N]");
        const Ids i(ids, t.device);
        c10::SmallVector<int64_t, 6> s(ids.sizes().begin(), ids.sizes().end());
        s.push_back(t.N);
        mmvae_embedding_args a;
        std::memset(&a, 0, sizeof(a));
        at::Tensor y = fresh(s, table.scalar_type(), t.device), add;
        if (v[3] != Py_None) {
            const at::Tensor& d = tensor(v[3], "add");
            like(d, "add", s, table.scalar_type(), t.device);
            const Rows r(d, "add");
            a.add = r.p;
            a.ldadd = r.ld;
            add = r.copy;  // (a copy lives until the call is enqueued)
        }
        a.T = i.T;
        a.N = t.N;
        a.V = t.M;
        a.ids = i.p;
        a.table = t.p;
        a.ldt = t.ld;
        a.y = y.data_ptr();
        a.ldy = t.N;
        a.stream = stream_of(t.device);
        a.device = t.device;
        a.dtype = t.dtype;
        a.ids64 = i.is64;
        a.scale = (float)number(v[2]);
        check(mmvae_embedding_fwd(&a));
        return wrap(y);
    });
}

// (dy, ids, rows, scale) -> dtable
PyObject* embedding_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded(n, 4, [&]() -> PyObject* {
        const at::Tensor &dy = tensor(v[0], "dy"), &ids = tensor(v[1], "ids");
        const Rows d(dy, "dy");
        const Ids i(ids, d.device);
        if (dy.sizes().slice(0, dy.dim() - 1) != ids.sizes()) wrong("dy must be ids' shape and the width");
        const long long V = PyLong_AsLongLong(v[2]);
        if (V == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            wrong("rows must be the table's row count");
        }
        if (V < 0) wrong("rows must be the table's row count");
        mmvae_embedding_args a;
        std::memset(&a, 0, sizeof(a));
        a.T = i.T;
        a.N = d.N;
        a.V = V;
        a.ids = i.p;
        a.dy = d.p;
        a.lddy = d.ld;
        at::Tensor out = fresh({(int64_t)V, d.N}, dy.scalar_type(), d.device), ws;
        a.dtable = out.data_ptr();
        a.ws_bytes = mmvae_embedding_bwd_ws(i.T, d.N, V);
        if (a.ws_bytes > 0) {
            ws = fresh({a.ws_bytes}, at::kByte, d.device);
            a.ws = ws.data_ptr();
        }
        a.stream = stream_of(d.device);
        a.device = d.device;
        a.dtype = d.dtype;
        a.ids64 = i.is64;
        a.scale = (float)number(v[3]);
        check(mmvae_embedding_bwd(&a));
        return wrap(out);
    });
}

PyObject* set_error(PyObject*, PyObject* e) {
    Py_XINCREF(e);
    Py_XDECREF(g_error);
    g_error = e;
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {{"norm_forward", FAST(norm_forward), METH_FASTCALL, nullptr},
                         {"norm_backward", FAST(norm_backward), METH_FASTCALL, nullptr},
                         {"dropout", FAST(dropout), METH_FASTCALL, nullptr},
                         {"embedding_forward", FAST(embedding_forward), METH_FASTCALL, nullptr},
                         {"embedding_backward", FAST(embedding_backward), METH_FASTCALL, nullptr},
                         {"set_error", set_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "mmvae_amd._ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&module); }
