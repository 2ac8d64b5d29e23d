// The host side of the small calls: a quantized linear or an expert on tensors, from the Python call to the library's
// launches.  What a call of one row costs is this path (the kernels run 5-20 us): through ctypes it was 20-33 us -- struct
// and pointer objects for some twenty arguments, seven data_ptr() calls, three tensor methods -- and here it is the
// allocation of the result and the launches (4-bit 1024 x 4096, one row: 21.7 us per call before, 6.5 now, which is the
// kernel's own time).
//
// Every function returns None where it does not cover the arguments (another device, dtype conversions, a layer that has to
// be validated first, an error from the library); the Python code around it then takes the general way and raises what
// there is to raise.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include <ATen/Functions.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/hqq_moe.h"

namespace {

struct Names {
    PyObject *dict, *W_q, *meta, *bias, *plan, *desc, *ready, *expert, *scale_q, *zero_q, *meta_scale, *meta_zero, *scale, *zero, *modules, *w1, *w2, *w3, *axis;
} N;

PyObject* g_scratch = nullptr;        // custom_layers._SCRATCH: {("cuda", index): uint8 tensor}
PyObject* g_grow = nullptr;           // custom_layers._scratch(device, bytes)
PyObject* g_keys[64];                 // ("cuda", index)

// A layer's descriptor (and with it the addresses it was made from) and the workspace of its last row count, as linear
// layer and as w1 of an expert; kept in the layer's __dict__.  It is good for as long as the layer keeps the descriptor it was
// made from (`of`, the layer's _desc, held here so that its address is not given to another) and its tensors stay where they
// are: the addresses alone do not tell a layer that was quantized again, in another format, into recycled memory.  A copied or
// pickled layer gets None and makes its own.  The descriptor is never changed once it is made.
struct Plan {
    PyObject_HEAD
    PyObject* of;
    hqm_weight w;
    int64_t linear_rows, expert_rows;
    size_t linear_bytes, f16_bytes, expert_bytes;
};
void plan_dealloc(PyObject* self) {
    Py_XDECREF(reinterpret_cast<Plan*>(self)->of);
    PyObject_Free(self);
}
PyObject* plan_copy(PyObject*, PyObject*) { Py_RETURN_NONE; }
PyObject* plan_reduce(PyObject*, PyObject*) { return Py_BuildValue("(O())", (PyObject*)Py_TYPE(Py_None)); }
PyMethodDef plan_methods[] = {{"__deepcopy__", plan_copy, METH_O, nullptr},
                              {"__copy__", plan_copy, METH_NOARGS, nullptr},
                              {"__reduce__", plan_reduce, METH_NOARGS, nullptr},
                              {nullptr, nullptr, 0, nullptr}};
PyTypeObject PlanType = {PyVarObject_HEAD_INIT(nullptr, 0) "mixtral_offloading_b200._host.Plan", sizeof(Plan)};

// borrowed reference out of a dict, null if absent (no error set)
PyObject* item(PyObject* dict, PyObject* key) {
    if (dict == nullptr || !PyDict_CheckExact(dict)) return nullptr;
    PyObject* v = PyDict_GetItemWithError(dict, key);
    if (v == nullptr) PyErr_Clear();
    return v;
}
// An owned reference.  A layer's dictionary may drop what it holds while a call is under way (another thread runs wherever
// Python code does: a workspace that grows, a descriptor that is made), so the call holds what it uses.
template <typename T>
struct Held {
    T* p;
    explicit Held(T* owned = nullptr) : p(owned) {}
    Held(const Held&) = delete;
    Held& operator=(const Held&) = delete;
    ~Held() { Py_XDECREF(reinterpret_cast<PyObject*>(p)); }
    T* operator->() const { return p; }
    explicit operator bool() const { return p != nullptr; }
    void take(T* owned) {
        Py_XDECREF(reinterpret_cast<PyObject*>(p));
        p = owned;
    }
};
PyObject* own(PyObject* borrowed) {
    Py_XINCREF(borrowed);
    return borrowed;
}
const void* address(PyObject* t) { return t != nullptr && THPVariable_Check(t) ? THPVariable_Unpack(t).const_data_ptr() : nullptr; }

// The addresses of a layer's seven tensors; false where it is not ready or has another form.
bool addresses_of(PyObject* dict, const void* (&at)[7]) {
    PyObject* meta = item(dict, N.meta);
    PyObject *ms = item(meta, N.meta_scale), *mz = item(meta, N.meta_zero);
    if (item(dict, N.ready) != Py_True || ms == nullptr || mz == nullptr) return false;
    PyObject* t[7] = {item(dict, N.W_q), item(meta, N.scale_q), item(meta, N.zero_q), item(ms, N.scale), item(ms, N.zero), item(mz, N.scale), item(mz, N.zero)};
    for (int i = 0; i < 7; ++i) at[i] = address(t[i]);
    return true;
}

// The plan of a layer whose tensors are where they were when its descriptor was made (new reference); null: not to be had here.
Plan* plan_of(PyObject* layer, PyObject* dict) {
    const void* at[7];
    if (!addresses_of(dict, at)) return nullptr;
    PyObject* kept = item(dict, N.plan);
    if (kept != nullptr && Py_TYPE(kept) == &PlanType) {
        Plan* p = reinterpret_cast<Plan*>(kept);
        if (p->of == item(dict, N.desc) && p->w.W_q == at[0] && p->w.scale_q == at[1] && p->w.zero_q == at[2] && p->w.ms_scale == at[3] && p->w.mz_scale == at[4] &&
            p->w.ms_zero == at[5] && p->w.mz_zero == at[6])
            return reinterpret_cast<Plan*>(own(kept));
    }
    PyObject* axis = item(item(dict, N.meta), N.axis);
    if (axis == nullptr || !PyLong_Check(axis) || PyLong_AsLong(axis) != 0) return nullptr;
    PyObject* d = PyObject_CallMethod(layer, "descriptor", nullptr);      // validates; a ctypes structure
    if (d == nullptr) {
        PyErr_Clear();
        return nullptr;
    }
    Plan* p = nullptr;
    Py_buffer view;
    if (PyObject_GetBuffer(d, &view, PyBUF_SIMPLE) == 0) {
        if (view.len == (Py_ssize_t)sizeof(hqm_weight) && (p = PyObject_New(Plan, &PlanType)) != nullptr) {
            memcpy(&p->w, view.buf, sizeof(hqm_weight));
            p->of = own(item(dict, N.desc));
            p->linear_rows = p->expert_rows = -1;
            p->linear_bytes = p->f16_bytes = p->expert_bytes = 0;
            if (PyDict_SetItem(dict, N.plan, reinterpret_cast<PyObject*>(p)) != 0) {
                Py_DECREF(p);
                p = nullptr;
            }
        }
        PyBuffer_Release(&view);
    }
    Py_DECREF(d);
    PyErr_Clear();
    return p;
}

PyObject* dict_of(PyObject* module) {        // new reference
    PyObject* d = PyObject_GetAttr(module, N.dict);
    if (d == nullptr) PyErr_Clear();
    return d;
}

// x if it is bf16, fp16 or fp32, contiguous, on the current device, last dimension K, at least one row; else null.
const at::Tensor* rows_of(PyObject* obj, int64_t K, int64_t* rows) {
    if (!THPVariable_CheckExact(obj)) return nullptr;
    const at::Tensor& x = THPVariable_Unpack(obj);
    const auto type = x.scalar_type();
    if (!x.is_cuda() || (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat) || x.dim() < 1 || x.size(-1) != K || x.numel() == 0 || !x.is_contiguous() ||
        x.device().index() != c10::cuda::current_device())
        return nullptr;
    *rows = x.numel() / K;
    return &x;
}

// Workspace of the device (the Python module's, grown through it); its address, null on failure.
void* scratch(const at::Tensor& on, size_t bytes, size_t* have) {
    const int dev = on.device().index();
    if (dev < 0 || dev >= 64) return nullptr;
    if (g_keys[dev] == nullptr && (g_keys[dev] = Py_BuildValue("(si)", "cuda", dev)) == nullptr) return nullptr;
    PyObject* t = item(g_scratch, g_keys[dev]);
    if (t != nullptr && THPVariable_Check(t) && (size_t)THPVariable_Unpack(t).numel() >= bytes) {
        *have = (size_t)THPVariable_Unpack(t).numel();
        return THPVariable_Unpack(t).data_ptr();
    }
    PyObject* device = THPDevice_New(on.device());
    t = device == nullptr ? nullptr : PyObject_CallFunction(g_grow, "On", device, (Py_ssize_t)bytes);
    Py_XDECREF(device);
    if (t == nullptr) {
        PyErr_Clear();
        return nullptr;
    }
    void* p = THPVariable_Unpack(t).data_ptr();           // (the module keeps it)
    *have = (size_t)THPVariable_Unpack(t).numel();
    Py_DECREF(t);
    return p;
}

at::Tensor result(const at::Tensor& x, int64_t n) {
    c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    return at::empty(shape, x.options());
}

// linear(layer, x)
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) return PyErr_Format(PyExc_TypeError, "linear(layer, x)");
    try {
        Held<PyObject> dict(dict_of(args[0]));
        Held<Plan> p(dict ? plan_of(args[0], dict.p) : nullptr);
        Held<PyObject> bias(own(item(dict.p, N.bias)));
        int64_t rows = 0;
        const at::Tensor* x = p ? rows_of(args[1], p->w.K, &rows) : nullptr;
        if (x == nullptr) Py_RETURN_NONE;
        c10::InferenceMode guard;
        const auto type = x->scalar_type();
        if (p->linear_rows != rows) {
            p->linear_bytes = hqm_linear_scratch_preferred(rows, &p->w);
            p->f16_bytes = hqm_linear_f16_scratch_bytes(rows, &p->w);
            p->linear_rows = rows;
        }
        const bool f16 = type == at::kHalf && p->f16_bytes != 0;
        at::Tensor converted;
        if (type != at::kBFloat16 && !f16) {
            converted = x->to(at::kBFloat16);
            x = &converted;
        }
        const size_t bytes = f16 ? p->f16_bytes : p->linear_bytes;
        size_t have = 0;
        void* ws = nullptr;
        if (bytes && (ws = scratch(*x, bytes, &have)) == nullptr) Py_RETURN_NONE;
        at::Tensor y = result(*x, p->w.N);
        const uint16_t* b = static_cast<const uint16_t*>(address(bias.p));
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = (f16 ? hqm_linear_f16 : hqm_linear)(static_cast<uint16_t*>(y.data_ptr()), static_cast<const uint16_t*>(x->const_data_ptr()), rows,
                                                 &p->w, b, ws, bytes, c10::cuda::getCurrentCUDAStream(x->device().index()).stream());
        Py_END_ALLOW_THREADS
        if (rc < 0) Py_RETURN_NONE;
        if (y.scalar_type() != type) y = y.to(type);
        return THPVariable_Wrap(std::move(y));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// dequantize(layer, code): the weight in bf16 (0), fp16 (1) or fp32 (2)
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) return PyErr_Format(PyExc_TypeError, "dequantize(layer, code)");
    try {
        const long code = PyLong_AsLong(args[1]);
        Held<PyObject> dict(dict_of(args[0]));
        Held<Plan> p(dict ? plan_of(args[0], dict.p) : nullptr);
        Held<PyObject> wq(own(item(dict.p, N.W_q)));
        if (!p || address(wq.p) != p->w.W_q || code < 0 || code > 2) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        const at::Tensor& like = THPVariable_Unpack(wq.p);
        if (like.device().index() != c10::cuda::current_device()) Py_RETURN_NONE;
        c10::InferenceMode guard;
        at::Tensor out = at::empty({p->w.N, p->w.K}, like.options().dtype(code == 0 ? at::kBFloat16 : code == 1 ? at::kHalf : at::kFloat));
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = hqm_dequantize(out.data_ptr(), (int)code, &p->w, c10::cuda::getCurrentCUDAStream(like.device().index()).stream());
        Py_END_ALLOW_THREADS
        if (rc < 0) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(out));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// The three plans of an expert module.
bool expert_plans(PyObject* module, Held<Plan> (&p)[3]) {
    Held<PyObject> dict(dict_of(module));
    Held<PyObject> modules(own(item(dict.p, N.modules)));
    PyObject* names[3] = {N.w1, N.w2, N.w3};
    for (int i = 0; i < 3; ++i) {
        Held<PyObject> layer(own(item(modules.p, names[i])));
        Held<PyObject> d(layer ? dict_of(layer.p) : nullptr);
        p[i].take(d ? plan_of(layer.p, d.p) : nullptr);
        if (!p[i]) return false;
    }
    return true;
}

int run_expert(const Held<Plan> (&p)[3], const at::Tensor& x, int64_t rows, const int32_t* idx, const float* w, uint16_t* out, int accumulate) {
    if (p[0]->expert_rows != rows) {
        p[0]->expert_bytes = hqm_expert_ffn_scratch_bytes(rows, &p[0]->w, &p[1]->w, &p[2]->w);
        p[0]->expert_rows = rows;
    }
    size_t have = 0;
    void* ws = scratch(x, p[0]->expert_bytes, &have);
    if (ws == nullptr) return -1;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = hqm_expert_ffn(out, static_cast<const uint16_t*>(x.const_data_ptr()), rows, idx, w, accumulate, &p[0]->w, &p[1]->w, &p[2]->w, ws, have,
                        c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
    Py_END_ALLOW_THREADS
    return rc;
}

// expert(module, x): all rows of x
PyObject* expert(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) return PyErr_Format(PyExc_TypeError, "expert(module, x)");
    try {
        Held<Plan> p[3];
        if (!expert_plans(args[0], p)) Py_RETURN_NONE;
        int64_t rows = 0;
        const at::Tensor* x = rows_of(args[1], p[0]->w.K, &rows);
        if (x == nullptr) Py_RETURN_NONE;
        c10::InferenceMode guard;
        const auto type = x->scalar_type();
        at::Tensor converted;
        if (type != at::kBFloat16) {
            converted = x->to(at::kBFloat16);
            x = &converted;
        }
        at::Tensor out = result(*x, p[1]->w.N);
        if (run_expert(p, *x, rows, nullptr, nullptr, static_cast<uint16_t*>(out.data_ptr()), 0) < 0) Py_RETURN_NONE;
        if (type != at::kBFloat16) out = out.to(type);
        return THPVariable_Wrap(std::move(out));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// expert_addresses(experts): the addresses of all layers' descriptors and tensors as bytes; None where a layer has no descriptor
// (its tensors were replaced) or another form.  For as long as the caller holds the descriptors, what it made from them is good
// while this does not change.
PyObject* expert_addresses(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 1 || !PyList_CheckExact(args[0])) return PyErr_Format(PyExc_TypeError, "expert_addresses(list)");
    const Py_ssize_t experts = PyList_GET_SIZE(args[0]);
    Held<PyObject> out(PyBytes_FromStringAndSize(nullptr, experts * 3 * 8 * (Py_ssize_t)sizeof(void*)));
    if (!out) return nullptr;
    char* to = PyBytes_AS_STRING(out.p);
    PyObject* names[3] = {N.w1, N.w2, N.w3};
    for (Py_ssize_t e = 0; e < experts; ++e) {
        if (e >= PyList_GET_SIZE(args[0])) Py_RETURN_NONE;
        Held<PyObject> module(own(PyList_GET_ITEM(args[0], e)));
        Held<PyObject> outer(dict_of(module.p));
        if (PyObject* inner = item(outer.p, N.expert)) module.take(own(inner));       // a wrapper around the expert
        Held<PyObject> dict(dict_of(module.p));
        Held<PyObject> modules(own(item(dict.p, N.modules)));
        for (PyObject* name : names) {
            Held<PyObject> layer(own(item(modules.p, name)));
            Held<PyObject> d(layer ? dict_of(layer.p) : nullptr);
            PyObject* desc = item(d.p, N.desc);
            const void* at[7];
            if (desc == nullptr || desc == Py_None || !addresses_of(d.p, at)) Py_RETURN_NONE;
            memcpy(to, &desc, sizeof(desc));
            memcpy(to + sizeof(desc), at, sizeof(at));
            to += sizeof(desc) + sizeof(at);
        }
    }
    return own(out.p);
}

// ---- a key/value cache in pages (paged.py has the same steps, and the messages for what is refused) ---------------------
// A plain tensor on device `dev` (-1: any CUDA device, and `dev` is set), null otherwise.
const at::Tensor* on_device(PyObject* obj, int& dev) {
    if (!THPVariable_CheckExact(obj)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(obj);
    if (!t.is_cuda()) return nullptr;
    if (dev < 0) dev = t.device().index();
    return t.device().index() == dev ? &t : nullptr;
}
// int32 with contiguous rows
const at::Tensor* ints(PyObject* obj, int& dev, int64_t dims) {
    const at::Tensor* t = on_device(obj, dev);
    if (t == nullptr || t->scalar_type() != at::kInt || t->dim() != dims || (dims > 0 && t->size(dims - 1) > 1 && t->stride(dims - 1) != 1)) return nullptr;
    return t;
}
int32_t* words(const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
bool whole(PyObject* obj, int64_t* v) {
    *v = PyLong_CheckExact(obj) ? PyLong_AsLongLong(obj) : -1;
    if (*v == -1 && PyErr_Occurred()) PyErr_Clear();
    return *v >= 0;
}
cudaStream_t stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

// `n` elements of a vector from `from` on, on the same storage.  (As narrow() does, in a third of its time.)
at::Tensor stretch(const at::Tensor& all, int64_t from, int64_t n) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(from);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(n);
    return t;
}

struct Tables {
    const at::Tensor *table, *lens, *free_pages, *count, *change;
    int64_t B, stride, page;
    bool read(PyObject* const* args) {
        int dev = -1;
        table = ints(args[0], dev, 2);
        lens = ints(args[1], dev, 1);
        free_pages = ints(args[2], dev, 1);
        change = ints(args[4], dev, 1);
        count = on_device(args[3], dev);
        if (!table || !lens || !free_pages || !change || !count || count->scalar_type() != at::kInt || count->numel() != 1 || dev != c10::cuda::current_device() ||
            !whole(args[5], &page) || page > INT32_MAX || free_pages->size(0) > INT32_MAX || table->size(1) > INT32_MAX)
            return false;
        B = table->size(0);
        stride = B > 1 ? table->stride(0) : table->size(1);
        return B <= INT32_MAX && lens->size(0) == B && change->size(0) == B;
    }
    int dev() const { return table->device().index(); }
};

// paged_reserve(block_table, kv_lens, free_pages, free_count, new_lens, page_size, tokens)
PyObject* paged_reserve(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) return PyErr_Format(PyExc_TypeError, "paged_reserve: seven arguments");
    try {
        Tables t;
        int64_t tokens;
        if (!t.read(args) || !whole(args[6], &tokens) || tokens > INT32_MAX) Py_RETURN_NONE;
        at::AutoDispatchBelowADInplaceOrView guard;
        const int64_t B = t.B, sizes[5] = {B + 1, B, tokens, tokens, 1};
        at::Tensor all = at::empty({2 * B + 2 + 2 * tokens}, t.table->options());
        int32_t* at = words(all);
        int32_t *cu = at, *after = cu + B + 1, *positions = after + B, *slots = positions + tokens, *status = slots + tokens;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = hqm_paged_reserve(words(*t.table), t.stride, words(*t.lens), words(*t.free_pages), words(*t.count), words(*t.change), cu, after, positions,
                               slots, status, (int32_t)B, (int32_t)t.table->size(1), (int32_t)t.page, (int32_t)t.free_pages->size(0), tokens, stream_of(t.dev()));
        Py_END_ALLOW_THREADS
        if (rc < 0) Py_RETURN_NONE;
        PyObject* out = PyTuple_New(5);
        int64_t from = 0;
        for (int i = 0; out != nullptr && i < 5; from += sizes[i++]) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(stretch(all, from, sizes[i])));
        return out;
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// paged_truncate(block_table, kv_lens, free_pages, free_count, keep, page_size)
PyObject* paged_truncate(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 6) return PyErr_Format(PyExc_TypeError, "paged_truncate: six arguments");
    try {
        Tables t;
        if (!t.read(args)) Py_RETURN_NONE;
        at::AutoDispatchBelowADInplaceOrView guard;
        at::Tensor status = at::empty({1}, t.table->options());
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = hqm_paged_truncate(words(*t.table), t.stride, words(*t.lens), words(*t.free_pages), words(*t.count), words(*t.change), words(status), (int32_t)t.B,
                                (int32_t)t.table->size(1), (int32_t)t.page, (int32_t)t.free_pages->size(0), stream_of(t.dev()));
        Py_END_ALLOW_THREADS
        if (rc < 0) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(status));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// A tensor of `dims` dimensions like q in type, device and its last one, whose elements are contiguous.
const at::Tensor* like(PyObject* obj, const at::Tensor& q, int64_t dims) {
    int dev = q.device().index();
    const at::Tensor* t = on_device(obj, dev);
    if (t == nullptr || t->scalar_type() != q.scalar_type() || t->dim() != dims || t->size(-1) != q.size(-1) || (t->size(-1) > 1 && t->stride(-1) != 1)) return nullptr;
    return t;
}
const at::Tensor* queries(PyObject* obj) {
    int dev = -1;
    const at::Tensor* q = on_device(obj, dev);
    if (q == nullptr || q->dim() != 3 || (q->scalar_type() != at::kBFloat16 && q->scalar_type() != at::kHalf) || dev != c10::cuda::current_device() ||
        (q->size(2) > 1 && q->stride(2) != 1) || q->size(0) > INT32_MAX)
        return nullptr;
    return q;
}
// strides of (tokens, heads, head_dim); of a dimension of one, what a contiguous tensor has
void strides(const at::Tensor& t, int64_t* token, int64_t* head) {
    *token = t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
    *head = t.size(1) > 1 ? t.stride(1) : t.size(2);
}
struct Pool {
    const at::Tensor *k, *v;
    int64_t pages, heads, page, k_page, v_page;
    bool read(PyObject* k_obj, PyObject* v_obj, const at::Tensor& q) {
        k = like(k_obj, q, 4);
        v = like(v_obj, q, 4);
        if (!k || !v || k->sizes() != v->sizes()) return false;
        pages = k->size(0), heads = k->size(1), page = k->size(2);
        const int64_t D = k->size(3), one = heads * page * D;
        for (const at::Tensor* t : {k, v})
            if ((page > 1 && t->stride(2) != D) || (heads > 1 && t->stride(1) != page * D)) return false;
        k_page = pages > 1 ? k->stride(0) : one;
        v_page = pages > 1 ? v->stride(0) : one;
        return pages <= INT32_MAX && page <= INT32_MAX && heads <= INT32_MAX;
    }
};
// `out`, or a new tensor where it is None; false: of another form than q
bool result_like(PyObject* obj, const at::Tensor& q, at::Tensor* out) {
    if (obj == Py_None) {
        *out = at::empty(q.sizes(), q.options());
        return true;
    }
    const at::Tensor* t = like(obj, q, 3);
    if (t == nullptr || t->sizes() != q.sizes() || !t->is_contiguous()) return false;
    *out = *t;
    return true;
}
bool real(PyObject* obj, double* v) {
    *v = PyFloat_AsDouble(obj);
    if (*v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

// rope_append_paged(q, k, v, k_pages, v_pages, positions, slots, theta, out or None, k_out or None)
PyObject* rope_append_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 10) return PyErr_Format(PyExc_TypeError, "rope_append_paged: ten arguments");
    try {
        const at::Tensor* q = queries(args[0]);
        if (q == nullptr) Py_RETURN_NONE;
        const at::Tensor *k = like(args[1], *q, 3), *v = like(args[2], *q, 3);
        Pool pool;
        int dev = q->device().index();
        const at::Tensor *positions = ints(args[5], dev, 1), *slots = ints(args[6], dev, 1);
        const int64_t T = q->size(0);
        hqm_paged_append a = {};
        double theta;
        if (!k || !v || !positions || !slots || !pool.read(args[3], args[4], *q) || k->sizes() != v->sizes() || k->size(0) != T || k->size(1) != pool.heads ||
            positions->size(0) != T || slots->size(0) != T || !real(args[7], &theta))
            Py_RETURN_NONE;
        a.rope_theta = (float)theta;
        a.rope_theta_low = (float)(theta - a.rope_theta);
        at::AutoDispatchBelowADInplaceOrView guard;
        at::Tensor out;
        if (!result_like(args[8], *q, &out)) Py_RETURN_NONE;
        if (args[9] != Py_None) {
            at::Tensor k_out;
            if (!result_like(args[9], *k, &k_out)) Py_RETURN_NONE;
            a.k_out = k_out.data_ptr();
        }
        a.q_out = out.data_ptr();
        a.q = q->const_data_ptr(), a.k = k->const_data_ptr(), a.v = v->const_data_ptr();
        strides(*q, &a.q_token, &a.q_head);
        strides(*k, &a.k_token, &a.k_head);
        strides(*v, &a.v_token, &a.v_head);
        a.k_pages = pool.k->data_ptr(), a.v_pages = pool.v->data_ptr();
        a.k_page = pool.k_page, a.v_page = pool.v_page;
        a.positions = words(*positions), a.slots = words(*slots);
        a.tokens = T;
        a.n_heads = (int32_t)q->size(1), a.n_kv_heads = (int32_t)pool.heads, a.head_dim = (int32_t)q->size(2);
        a.pages = (int32_t)pool.pages, a.page_size = (int32_t)pool.page;
        a.dtype = q->scalar_type() == at::kHalf;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = hqm_rope_append_paged(&a, stream_of(dev));
        Py_END_ALLOW_THREADS
        if (rc < 0) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(out));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

// attention(q, k, v, cu_seqlens, max_new, scale or None, out or None[, block_table, kv_lens]): with the last two k and v are pages
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7 && n != 9) return PyErr_Format(PyExc_TypeError, "attention: seven or nine arguments");
    try {
        const bool paged = n == 9;
        const at::Tensor* q = queries(args[0]);
        if (q == nullptr) Py_RETURN_NONE;
        int dev = q->device().index();
        const int64_t T = q->size(0);
        hqm_attention c = {};
        const at::Tensor* cu = ints(args[3], dev, 1);
        int64_t most = 0;
        if (cu == nullptr || cu->size(0) < 1 || cu->size(0) > INT32_MAX || !whole(args[4], &most) || most > INT32_MAX) Py_RETURN_NONE;
        c.sequences = (int32_t)(cu->size(0) - 1);
        if (paged) {
            Pool pool;
            const at::Tensor *table = ints(args[7], dev, 2), *lens = ints(args[8], dev, 1);
            if (!table || !lens || !pool.read(args[1], args[2], *q) || table->size(0) != c.sequences || lens->size(0) != c.sequences || table->size(1) > INT32_MAX)
                Py_RETURN_NONE;
            c.k = pool.k->const_data_ptr(), c.v = pool.v->const_data_ptr();
            c.k_page = pool.k_page, c.v_page = pool.v_page;
            c.block_table = words(*table);
            c.table_stride = c.sequences > 1 ? table->stride(0) : table->size(1);
            c.kv_lens = words(*lens);
            c.n_kv_heads = (int32_t)pool.heads, c.pages = (int32_t)pool.pages, c.page_size = (int32_t)pool.page;
            c.max_pages = (int32_t)table->size(1);
        } else {
            const at::Tensor *k = like(args[1], *q, 3), *v = like(args[2], *q, 3);
            if (!k || !v || k->sizes() != v->sizes() || k->size(0) != T) Py_RETURN_NONE;
            c.k = k->const_data_ptr(), c.v = v->const_data_ptr();
            strides(*k, &c.k_token, &c.k_head);
            strides(*v, &c.v_token, &c.v_head);
            c.n_kv_heads = (int32_t)k->size(1);
        }
        double scale = 1.f / std::sqrt((float)std::max<int64_t>(q->size(2), 1));
        if (args[5] != Py_None && !real(args[5], &scale)) Py_RETURN_NONE;
        c.scale = (float)scale;
        at::AutoDispatchBelowADInplaceOrView guard;
        at::Tensor out;
        if (!result_like(args[6], *q, &out)) Py_RETURN_NONE;
        c.out = out.data_ptr();
        c.q = q->const_data_ptr();
        strides(*q, &c.q_token, &c.q_head);
        c.cu_seqlens = words(*cu);
        c.tokens = T;
        c.max_new = (int32_t)most;
        c.n_heads = (int32_t)q->size(1), c.head_dim = (int32_t)q->size(2);
        c.dtype = q->scalar_type() == at::kHalf;
        const size_t bytes = hqm_attention_scratch_bytes(&c);
        at::Tensor ws = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
        void* at = ws.data_ptr();
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = (paged ? hqm_paged_attention : hqm_prompt_attention)(&c, at, bytes, stream_of(dev));
        Py_END_ALLOW_THREADS
        if (rc < 0) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(out));
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) return PyErr_Format(PyExc_TypeError, "setup(scratch, grow)");
    Py_INCREF(args[0]);
    Py_INCREF(args[1]);
    Py_XSETREF(g_scratch, args[0]);
    Py_XSETREF(g_grow, args[1]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, "setup(scratch_dict, grow)"},
    {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, "linear(layer, x) -> tensor or None"},
    {"dequantize", (PyCFunction)(void (*)(void))dequantize, METH_FASTCALL, "dequantize(layer, dtype code) -> tensor or None"},
    {"expert", (PyCFunction)(void (*)(void))expert, METH_FASTCALL, "expert(module, x) -> tensor or None"},
    {"expert_addresses", (PyCFunction)(void (*)(void))expert_addresses, METH_FASTCALL, "expert_addresses(experts) -> bytes or None"},
    {"paged_reserve", (PyCFunction)(void (*)(void))paged_reserve, METH_FASTCALL, "paged_reserve(...) -> five tensors or None"},
    {"paged_truncate", (PyCFunction)(void (*)(void))paged_truncate, METH_FASTCALL, "paged_truncate(...) -> tensor or None"},
    {"rope_append_paged", (PyCFunction)(void (*)(void))rope_append_paged, METH_FASTCALL, "rope_append_paged(...) -> tensor or None"},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, "attention(...) -> tensor or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host path of the quantized layers.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    struct {
        PyObject** to;
        const char* name;
    } all[] = {{&N.dict, "__dict__"}, {&N.W_q, "W_q"},     {&N.meta, "meta"},           {&N.bias, "bias"},           {&N.plan, "_plan"}, {&N.desc, "_desc"}, {&N.ready, "ready"}, {&N.expert, "_expert"},
               {&N.scale_q, "scale_q"}, {&N.zero_q, "zero_q"}, {&N.meta_scale, "meta_scale"}, {&N.meta_zero, "meta_zero"}, {&N.scale, "scale"}, {&N.zero, "zero"},
               {&N.modules, "_modules"}, {&N.w1, "w1"},    {&N.w2, "w2"},               {&N.w3, "w3"}, {&N.axis, "axis"}};
    for (auto& a : all)
        if ((*a.to = PyUnicode_InternFromString(a.name)) == nullptr) return nullptr;
    PlanType.tp_flags = Py_TPFLAGS_DEFAULT;
    PlanType.tp_methods = plan_methods;
    PlanType.tp_dealloc = plan_dealloc;
    if (PyType_Ready(&PlanType) != 0) return nullptr;
    return PyModule_Create(&module);
}
