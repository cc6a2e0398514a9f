// The calls of ops.py on torch tensors, without the interpreter's share: a Python extension that reads the tensors' fields, looks
// them over, fills the C structs and calls libptq8's entry points (whose addresses it is given).  Anything out of the ordinary makes
// it return -1 before any call, and ops.py goes through the arguments one by one and says what is wrong with them.
//
// A call of cache_write took 8 us of host time with the same steps in Python, of which this takes one.
//
// The interpreter's lock is given back around the calls of libptq8 and the allocator, as ctypes does: a launch may wait for room in its
// stream's queue, and that stream for a host function that wants the lock.  Meanwhile the tensors are held, whatever other
// threads do with the caller's containers.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "ptq8.h"

namespace {

int (*cache_write_entry)(ptq8_ops*, const ptq8_cache_rows_args*, void*);
int (*cache_read_entry)(ptq8_ops*, const ptq8_cache_rows_args*, void*);
int (*attention_entry)(ptq8_ops*, const ptq8_cache_attention_args*, void*);
long long (*workspace_entry)(ptq8_ops*, const ptq8_cache_attention_args*);
int (*w4_entry)(ptq8_ops*, const ptq8_linear_w4_args*, void*);

// The tensor behind an argument, or null.
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PTQ8_F32;
        case at::kHalf: return PTQ8_F16;
        case at::kBFloat16: return PTQ8_BF16;
        default: return -1;
    }
}

bool on(const at::Tensor& t, int64_t device) { return t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided; }

bool ints(const at::Tensor& t, int64_t n, int64_t device) { return t.scalar_type() == at::kInt && t.numel() == n && t.is_contiguous() && on(t, device); }

// Codes (bytes) or pairs (bf16) of a cache: [pages][heads][page][wide], a head's rows of a page one after another.
bool part(const at::Tensor& t, at::ScalarType type, const int64_t* shape, int64_t wide, int64_t device) {
    return t.dim() == 4 && t.scalar_type() == type && t.size(0) == shape[0] && t.size(1) == shape[1] && t.size(2) == shape[2] && t.size(3) == wide && t.stride(3) == 1 &&
           t.stride(2) == wide && on(t, device);
}

// Tensors that a call reads and writes, kept until it is over.
struct Held {
    at::Tensor tensors[10];
    int n = 0;
    void add(std::initializer_list<const at::Tensor*> more) {
        for (const at::Tensor* t : more)
            if (t) tensors[n++] = *t;
    }
};

// What a call gives, without the interpreter's lock meanwhile.
template <typename F>
auto unlocked(const F& call) {
    PyThreadState* state = PyEval_SaveThread();
    const auto result = call();   // (throws nothing)
    PyEval_RestoreThread(state);
    return result;
}

bool fill(ptq8_cache& c, Held& held, PyObject* cache, PyObject* table_o, PyObject* lengths_o, PyObject* starts_o, int64_t tokens, int64_t device) {
    PyObject* const* items;
    if (PyTuple_Check(cache) && PyTuple_GET_SIZE(cache) == 4)
        items = &PyTuple_GET_ITEM(cache, 0);
    else if (PyList_Check(cache) && PyList_GET_SIZE(cache) == 4)
        items = reinterpret_cast<PyListObject*>(cache)->ob_item;
    else
        return false;
    const at::Tensor *k = tensor(items[0]), *ks = tensor(items[1]), *v = tensor(items[2]), *vs = tensor(items[3]), *table = tensor(table_o), *lengths = tensor(lengths_o);
    if (!k || !ks || !v || !vs || !table || !lengths || k->dim() != 4) return false;
    const int64_t shape[3] = {k->size(0), k->size(1), k->size(2)}, half = k->size(3);
    if (!part(*k, at::kByte, shape, half, device) || !part(*v, at::kByte, shape, half, device) || !part(*ks, at::kBFloat16, shape, 2, device) ||
        !part(*vs, at::kBFloat16, shape, 2, device))
        return false;
    if (table->dim() != 2 || table->scalar_type() != at::kInt || table->stride(1) != 1 || !on(*table, device)) return false;
    const int64_t seqs = table->size(0);
    if (!ints(*lengths, seqs, device)) return false;
    c = ptq8_cache{};
    if (starts_o == Py_None) {
        if (tokens != seqs) return false;
    } else {
        const at::Tensor* starts = tensor(starts_o);
        if (!starts || !ints(*starts, seqs + 1, device)) return false;
        held.add({starts});
        c.starts = static_cast<const int*>(starts->data_ptr());
    }
    constexpr int64_t most = 0x7FFFFFFF;
    if (shape[0] > most || shape[1] > most || shape[2] > most || half > most / 2 || seqs > most || table->size(1) > most) return false;
    c.k = static_cast<uint8_t*>(k->data_ptr());
    c.v = static_cast<uint8_t*>(v->data_ptr());
    c.k_scale = static_cast<uint16_t*>(ks->data_ptr());
    c.v_scale = static_cast<uint16_t*>(vs->data_ptr());
    c.k_page = k->stride(0), c.k_head = k->stride(1), c.v_page = v->stride(0), c.v_head = v->stride(1);
    c.k_scale_page = 2 * ks->stride(0), c.k_scale_head = 2 * ks->stride(1), c.v_scale_page = 2 * vs->stride(0), c.v_scale_head = 2 * vs->stride(1);
    c.table = static_cast<const int*>(table->data_ptr());
    c.table_pitch = table->stride(0);
    c.lengths = static_cast<const int*>(lengths->data_ptr());
    c.pages = shape[0];
    c.table_width = static_cast<int>(table->size(1));
    c.page = static_cast<int>(shape[2]);
    c.kv_heads = static_cast<int>(shape[1]);
    c.head_dim = static_cast<int>(2 * half);
    c.sequences = static_cast<int>(seqs);
    held.add({k, ks, v, vs, table, lengths});
    return true;
}

PyObject* answer(int rc) { return PyLong_FromLong(rc); }

// cache_rows(write, handle, device, cache, k, v, table, lengths, starts, stream)
PyObject* cache_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 10) return answer(-1);
    if (a[1] == Py_None) return answer(-1);   // a closed handle
    const bool write = a[0] == Py_True;
    const int64_t device = PyLong_AsLongLong(a[2]);
    const at::Tensor *k = tensor(a[4]), *v = tensor(a[5]);
    if (!k || !v || k->dim() != 3 || v->dim() != 3 || k->scalar_type() != v->scalar_type()) return answer(-1);
    ptq8_cache_rows_args args{};
    const int64_t tokens = k->size(0);
    Held held;
    held.add({k, v});
    if (!fill(args.cache, held, a[3], a[6], a[7], a[8], tokens, device)) return answer(-1);
    args.type = type_of(*k);
    for (const at::Tensor* t : {k, v})
        if (t->size(0) != tokens || t->size(1) != args.cache.kv_heads || t->size(2) != args.cache.head_dim || t->stride(2) != 1 || !on(*t, device)) return answer(-1);
    if (args.type < 0) return answer(-1);
    args.k = k->data_ptr(), args.v = v->data_ptr();
    args.k_token = k->stride(0), args.k_head = k->stride(1), args.v_token = v->stride(0), args.v_head = v->stride(1);
    args.tokens = tokens;
    auto* ops = static_cast<ptq8_ops*>(PyLong_AsVoidPtr(a[1]));
    void* stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) return nullptr;
    return answer(unlocked([&]() noexcept { return (write ? cache_write_entry : cache_read_entry)(ops, &args, stream); }));
}

// cache_attention(handle, device, q, cache, table, lengths, starts, scale, out, stream), its workspace made here
PyObject* cache_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 10) return answer(-1);
    if (a[0] == Py_None) return answer(-1);   // a closed handle
    const int64_t device = PyLong_AsLongLong(a[1]);
    const at::Tensor *q = tensor(a[2]), *out = tensor(a[8]);
    if (!q || !out || q->dim() != 3 || out->sizes() != q->sizes() || out->scalar_type() != q->scalar_type() || !on(*q, device) || !on(*out, device)) return answer(-1);
    if (q->stride(2) != 1 || out->stride(2) != 1) return answer(-1);
    ptq8_cache_attention_args args{};
    Held held;
    held.add({q, out});
    if (!fill(args.cache, held, a[3], a[4], a[5], a[6], q->size(0), device)) return answer(-1);
    args.type = type_of(*q);
    if (args.type != PTQ8_F16 && args.type != PTQ8_BF16) return answer(-1);
    if (q->size(2) != args.cache.head_dim || q->size(1) > 0x7FFFFFFF) return answer(-1);
    args.q = q->data_ptr(), args.out = out->data_ptr();
    args.q_token = q->stride(0), args.q_head = q->stride(1), args.out_token = out->stride(0), args.out_head = out->stride(1);
    args.tokens = q->size(0);
    args.heads = static_cast<int>(q->size(1));
    args.scale = static_cast<float>(a[7] == Py_None ? std::pow(static_cast<double>(args.cache.head_dim), -0.5) : PyFloat_AsDouble(a[7]));
    auto* ops = static_cast<ptq8_ops*>(PyLong_AsVoidPtr(a[0]));
    void* stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor workspace;
    const auto options = q->options().dtype(at::kByte);
    return answer(unlocked([&]() noexcept {
        const long long need = workspace_entry(ops, &args);
        if (need < 0) return -1;
        if (need) {
            try {
                workspace = at::empty({need}, options);
            } catch (...) {   // out of memory: the way through Python raises torch's own error
                return -1;
            }
            args.workspace = workspace.data_ptr();
            args.workspace_bytes = need;
        }
        return attention_entry(ops, &args, stream);
    }));
}

// linear_w4(handle, device, x, w, w_scale, group, bias, act, out, stream)
PyObject* linear_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 10) return answer(-1);
    if (a[0] == Py_None) return answer(-1);   // a closed handle
    const int64_t device = PyLong_AsLongLong(a[1]), group = PyLong_AsLongLong(a[5]), act = PyLong_AsLongLong(a[7]);
    if (PyErr_Occurred()) {   // no whole numbers
        PyErr_Clear();
        return answer(-1);
    }
    const at::Tensor *x = tensor(a[2]), *w = tensor(a[3]), *s = tensor(a[4]), *y = tensor(a[8]);
    if (!x || !w || !s || !y || group <= 0 || group > 0x7FFFFFFF || (act != PTQ8_EPI_NONE && act != PTQ8_EPI_SWIGLU)) return answer(-1);
    for (const at::Tensor* t : {x, w, s, y})
        if (t->dim() != 2 || t->stride(1) != 1 || !on(*t, device)) return answer(-1);
    ptq8_linear_w4_args args{};
    args.x_type = type_of(*x), args.scale_type = type_of(*s), args.y_type = type_of(*y);
    if (args.x_type < 0 || args.scale_type < 0 || args.y_type < 0 || (w->scalar_type() != at::kByte && w->scalar_type() != at::kChar)) return answer(-1);
    const int64_t rows = x->size(0), k = x->size(1), channels = w->size(0), halves = act == PTQ8_EPI_SWIGLU ? 2 : 1;
    if (k <= 0 || k > 0x7FFFFFFF || channels > 0x7FFFFFFF || channels % halves || w->size(1) != (k + 1) / 2) return answer(-1);
    if (s->size(0) != channels || s->size(1) != (k + group - 1) / group || y->size(0) != rows || y->size(1) != channels / halves) return answer(-1);
    if (a[6] != Py_None) {
        const at::Tensor* b = tensor(a[6]);
        if (!b || b->scalar_type() != at::kFloat || b->numel() != channels || !b->is_contiguous() || !on(*b, device)) return answer(-1);
        args.bias = static_cast<const float*>(b->data_ptr());
    }
    args.x = x->data_ptr(), args.ldx = x->stride(0);
    args.w = w->data_ptr(), args.ldw = w->stride(0);
    args.w_scale = s->data_ptr(), args.lds = s->stride(0);
    args.y = y->data_ptr(), args.ldy = y->stride(0);
    args.rows = rows;
    args.in_features = static_cast<int>(k), args.out_features = static_cast<int>(channels / halves);
    args.group = static_cast<int>(group), args.epilogue = static_cast<int>(act);
    auto* ops = static_cast<ptq8_ops*>(PyLong_AsVoidPtr(a[0]));
    void* stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) return nullptr;
    Held held;
    held.add({x, w, s, y});
    if (a[6] != Py_None) held.add({tensor(a[6])});
    return answer(unlocked([&]() noexcept { return w4_entry(ops, &args, stream); }));
}

// entries(cache_write, cache_read, cache_attention, cache_attention_workspace, linear_w4): addresses
PyObject* entries(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "five addresses");
        return nullptr;
    }
    cache_write_entry = reinterpret_cast<decltype(cache_write_entry)>(PyLong_AsVoidPtr(a[0]));
    cache_read_entry = reinterpret_cast<decltype(cache_read_entry)>(PyLong_AsVoidPtr(a[1]));
    attention_entry = reinterpret_cast<decltype(attention_entry)>(PyLong_AsVoidPtr(a[2]));
    workspace_entry = reinterpret_cast<decltype(workspace_entry)>(PyLong_AsVoidPtr(a[3]));
    w4_entry = reinterpret_cast<decltype(w4_entry)>(PyLong_AsVoidPtr(a[4]));
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// A tensor whose fields cannot be read (it has no memory of its own, or no sizes yet) throws: ops.py meets it then.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* no_throw(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    try {
        return F(self, a, n);
    } catch (...) {
        return answer(-1);
    }
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(no_throw<f>)), METH_FASTCALL

PyMethodDef methods[] = {{"entries", FAST(entries), nullptr},
                         {"cache_rows", FAST(cache_rows), nullptr},
                         {"cache_attention", FAST(cache_attention), nullptr},
                         {"linear_w4", FAST(linear_w4), nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "ptq8_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ptq8_host() { return PyModule_Create(&module); }
