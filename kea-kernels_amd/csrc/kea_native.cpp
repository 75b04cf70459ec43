// The host side of an operator call in one native call: argument checks on the tensors' own fields, the output and
// workspace allocations and the library's launch, without the Python objects (shape tuples, dictionary keys, ctypes
// conversions) that cost a call more than its two kernel launches. The module extends kea_kernels.lowbit, int8, norms,
// window, int4 and paged: everything it does not take (tensor subclasses and transforms, arguments that would raise) it declines by
// returning None / False, and the caller's Python path, which holds the full checks and their messages, runs instead.
//
// Calls in a row, host bound: Int8MmaLayer.linear at M = 128, N = 4096, K = 1024 (fp16 in and out) 13.2 -> 9.3 us, at one
// row 13.2 -> 9.9, lowbit.quantize + lowbit.gemm with group scales 21.9 -> 12.9, the provider's call on a few rows 18.7 ->
// 11.7; the two HIP launches are about 6 us of each. int8.gemm on one row 15.5 -> 5.1 (one launch), norms.block_norm 23 -> 6.8,
// window.attention (two launches) 27 -> 13.7, paged.write and paged.read (two calls, a launch each) 85 -> 10.7, paged.attention of a few
// tokens (two launches) 27 -> 12.2.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cmath>
#include <cstdint>
#include <list>
#include <unordered_map>

#include "../../include/kea_block.h"
#include "../../include/kea_decode.h"
#include "../../include/kea_lowbit.h"

namespace {

// Library entry points, resolved from the loaded libkea_hip.so by bind().
struct Library {
    decltype(&kea_lowbit_project_launch) project_launch = nullptr;
    decltype(&kea_lowbit_gemm) gemm = nullptr;
    decltype(&kea_lowbit_gemm_residual) gemm_residual = nullptr;
    decltype(&kea_quantize) quantize = nullptr;
    decltype(&kea_int8_gemm) int8_gemm = nullptr;
    decltype(&kea_block_norm) block_norm = nullptr;
    decltype(&kea_window_attention) window = nullptr;
    decltype(&kea_window_attention_workspace) window_workspace = nullptr;
    decltype(&kea_int4_gemm) int4_gemm = nullptr;
    decltype(&kea_paged_write) paged_write = nullptr;
    decltype(&kea_paged_read) paged_read = nullptr;
    decltype(&kea_paged_attention) paged_attention = nullptr;
    decltype(&kea_paged_attention_workspace) paged_workspace = nullptr;
} lib;

// The tensor behind an exact torch.Tensor whose memory a kernel may read as it is: on a GPU, strided, no transform
// (functorch, lazy negation or conjugation), nothing that autograd would have to record or carry on. nullptr otherwise.
const at::Tensor *plain(PyObject *o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) return nullptr;
    constexpr c10::DispatchKeySet transforms({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                              c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                              c10::DispatchKey::Negative, c10::DispatchKey::Conjugate,
                                              c10::DispatchKey::ZeroTensor});
    if (t.key_set().has_any(transforms)) return nullptr;
    if ((t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined()) return nullptr;
    return &t;
}

// Calls made while something records or rewrites operators (dispatch modes, functorch layers, tracing) are not taken.
bool modes_active() {
    const auto &tls = c10::impl::tls_local_dispatch_key_set();
    return tls.included_.has(c10::DispatchKey::Python) || tls.included_.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) ||
           tls.included_.has(c10::DispatchKey::Tracer);
}

int code_of(at::ScalarType t) {
    return t == at::kFloat ? KEA_F32 : t == at::kHalf ? KEA_F16 : t == at::kBFloat16 ? KEA_BF16 : -1;
}

void *stream_of(c10::Device d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

// ---- Replays: an operator's resolved call layouts ----

constexpr int kMaxDim = 4;

struct Key {
    int64_t tag;                // what the operator does with the input (its own numbering)
    int64_t sizes[kMaxDim], strides[kMaxDim];
    const void *norm_w, *norm_b;
    int64_t norm_size[2];       // elements of each; -1: a call without a LayerNorm
    float eps;
    int8_t dim, dtype, out_dtype, device;
    bool operator==(const Key &o) const {
        if (tag != o.tag || dim != o.dim || dtype != o.dtype || out_dtype != o.out_dtype || device != o.device ||
            norm_w != o.norm_w || norm_b != o.norm_b || norm_size[0] != o.norm_size[0] || norm_size[1] != o.norm_size[1] ||
            eps != o.eps)
            return false;
        for (int i = 0; i < dim; ++i)
            if (sizes[i] != o.sizes[i] || strides[i] != o.strides[i]) return false;
        return true;
    }
};
struct KeyHash {
    size_t operator()(const Key &k) const {
        uint64_t h = (uint64_t)k.tag * 0x9E3779B97F4A7C15ull + (uint64_t)(uintptr_t)k.norm_w + ((uint64_t)k.out_dtype << 56);
        for (int i = 0; i < k.dim; ++i) {
            h = (h ^ (uint64_t)k.sizes[i]) * 0x100000001B3ull;
            h = (h ^ (uint64_t)k.strides[i]) * 0x100000001B3ull;
        }
        return (size_t)(h ^ (h >> 29));
    }
};

struct Entry {
    PyObject *owner;  // the Python entry that frees the plan
    const kea_project_plan *plan;
    int64_t need;
    c10::SmallVector<int64_t, 4> shape;
    bool transposed;
    std::list<Key>::iterator order;
};

struct Replays {
    PyObject_HEAD
    std::unordered_map<Key, Entry, KeyHash> *entries;
    std::list<Key> *order;  // oldest first
    Py_ssize_t limit;
};

// The key of input x; false where the call cannot be kept or replayed. norm: the call has a LayerNorm, whose parameters
// must be there.
bool make_key(const at::Tensor &x, PyObject *out_dtype, int64_t tag, bool norm, PyObject *norm_w, PyObject *norm_b, double eps,
              Key *k) {
    if (x.dim() > kMaxDim || !THPDtype_Check(out_dtype)) return false;
    *k = Key{};
    k->tag = tag;
    k->dim = (int8_t)x.dim();
    for (int i = 0; i < k->dim; ++i) {
        k->sizes[i] = x.size(i);
        k->strides[i] = x.stride(i);
    }
    k->dtype = (int8_t)x.scalar_type();
    k->out_dtype = (int8_t)((THPDtype *)out_dtype)->scalar_type;
    k->device = x.device().index();
    k->norm_size[0] = k->norm_size[1] = -1;
    if (norm) {  // LayerNorm parameters are read in place, where the plan was made for
        const at::Tensor *w[2];
        PyObject *const o[2] = {norm_w, norm_b};
        for (int i = 0; i < 2; ++i) {
            if (!THPVariable_Check(o[i])) return false;
            w[i] = &THPVariable_Unpack(o[i]);
            if (!w[i]->defined() || w[i]->scalar_type() != at::kFloat || w[i]->device() != x.device() ||
                w[i]->layout() != at::kStrided || !w[i]->is_contiguous() || !w[i]->has_storage())
                return false;
        }
        k->norm_w = w[0]->const_data_ptr();
        k->norm_b = w[1]->const_data_ptr();
        k->norm_size[0] = w[0]->numel();
        k->norm_size[1] = w[1]->numel();
        k->eps = (float)eps;
    }
    return true;
}

PyObject *replays_new(PyTypeObject *type, PyObject *args, PyObject *) {
    Py_ssize_t limit;
    if (!PyArg_ParseTuple(args, "n", &limit)) return nullptr;
    auto *self = (Replays *)type->tp_alloc(type, 0);
    if (!self) return nullptr;
    self->entries = new (std::nothrow) std::unordered_map<Key, Entry, KeyHash>;
    self->order = new (std::nothrow) std::list<Key>;
    self->limit = limit;
    if (!self->entries || !self->order) {
        Py_DECREF(self);
        return PyErr_NoMemory();
    }
    return (PyObject *)self;
}

void replays_dealloc(PyObject *o) {
    auto *self = (Replays *)o;
    if (self->entries)
        for (auto &e : *self->entries) Py_DECREF(e.second.owner);
    delete self->entries;
    delete self->order;
    Py_TYPE(o)->tp_free(o);
}

// call(x, out_dtype, tag[, norm_weight, norm_bias, eps]) -> the output, or None where this layout is not kept
PyObject *replays_call(PyObject *o, PyObject *const *args, Py_ssize_t n) {
    auto *self = (Replays *)o;
    if (n != 3 && n != 6) Py_RETURN_NONE;
    const at::Tensor *x = plain(args[0]);
    if (!x || modes_active()) Py_RETURN_NONE;
    const int64_t tag = PyLong_AsLongLong(args[2]);
    const double eps = n == 6 ? PyFloat_AsDouble(args[5]) : 0.0;
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    Key k;
    if (!make_key(*x, args[1], tag, n == 6, n == 6 ? args[3] : nullptr, n == 6 ? args[4] : nullptr, eps, &k)) Py_RETURN_NONE;
    const auto it = self->entries->find(k);
    if (it == self->entries->end()) Py_RETURN_NONE;
    try {
        // the plan outlives this call whatever runs meanwhile, and its owner is released however the call ends
        const THPObjectPtr owner(Py_NewRef(it->second.owner));
        const kea_project_plan *plan = it->second.plan;
        const int64_t need = it->second.need;
        const bool transposed = it->second.transposed;
        const auto device = x->device();
        at::Tensor y = at::empty(it->second.shape, at::TensorOptions().device(device).dtype((at::ScalarType)k.out_dtype));
        at::Tensor ws = at::empty({need}, at::TensorOptions().device(device).dtype(at::kByte));
        const int rc = lib.project_launch(plan, x->const_data_ptr(), y.mutable_data_ptr(), ws.mutable_data_ptr(), need,
                                          stream_of(device));
        if (rc != 0) Py_RETURN_NONE;  // the Python path reports it
        return THPVariable_Wrap(transposed ? y.transpose(1, 2) : std::move(y));
    } catch (const std::exception &) {
        Py_RETURN_NONE;  // (an allocation failed: the Python path raises torch's error)
    }
}

// keep(x, out_dtype, tag, norm_weight, norm_bias, eps, owner, plan, need, shape, transposed)
PyObject *replays_keep(PyObject *o, PyObject *args) {
    auto *self = (Replays *)o;
    PyObject *xo, *dtype, *nw, *nb, *owner, *shape;
    long long tag, need;
    unsigned long long plan;
    double eps;
    int transposed;
    if (!PyArg_ParseTuple(args, "OOLOOdOKLO!p", &xo, &dtype, &tag, &nw, &nb, &eps, &owner, &plan, &need, &PyTuple_Type, &shape,
                          &transposed))
        return nullptr;
    const at::Tensor *x = plain(xo);
    Key k;
    if (!x || !make_key(*x, dtype, tag, nw != Py_None || nb != Py_None, nw, nb, eps, &k)) Py_RETURN_NONE;
    Entry e{owner, (const kea_project_plan *)plan, need, {}, transposed != 0, {}};
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(shape); ++i) {
        e.shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i)));
        if (PyErr_Occurred()) return nullptr;
    }
    THPObjectPtr old;  // released last: that may run other code, which may come back here
    try {
        auto it = self->entries->find(k);
        if (it == self->entries->end() && (Py_ssize_t)self->entries->size() >= self->limit) it = self->entries->find(self->order->front());
        if (it != self->entries->end()) {  // replaced, or the oldest makes room
            old = it->second.owner;
            self->order->erase(it->second.order);
            self->entries->erase(it);
        }
        e.order = self->order->insert(self->order->end(), k);
        self->entries->emplace(k, e);
        Py_INCREF(owner);
    } catch (const std::exception &) {
        return PyErr_NoMemory();
    }
    Py_RETURN_NONE;
}

PyMethodDef replays_methods[] = {
    {"call", (PyCFunction)(void (*)())replays_call, METH_FASTCALL, "call(x, out_dtype, tag[, norm_weight, norm_bias, eps])"},
    {"keep", replays_keep, METH_VARARGS, "keep(x, out_dtype, tag, norm_weight, norm_bias, eps, owner, plan, need, shape, transposed)"},
    {nullptr, nullptr, 0, nullptr}};

PyTypeObject ReplaysType = {PyVarObject_HEAD_INIT(nullptr, 0) "kea_native.Replays", sizeof(Replays)};

// ---- quantize and gemm ----

bool as_int(PyObject *o, int64_t *v) {
    *v = PyLong_AsLongLong(o);
    if (!PyErr_Occurred()) return true;
    PyErr_Clear();
    return false;
}

// An optional tensor argument: false where it is neither None nor a plain tensor on `device`.
bool optional(PyObject *o, c10::Device device, const at::Tensor **t) {
    *t = nullptr;
    if (o == Py_None) return true;
    *t = plain(o);
    return *t && (*t)->device() == device;
}

// quantize(x, xb, xt, xk, t, m, k, parts, norm_w, norm_b, eps, silu, qs_dtype, ldq) -> (q, qs) or None. norm_w / norm_b:
// contiguous FP32 tensors on x's device, or None.
PyObject *native_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != 14) Py_RETURN_NONE;
    const at::Tensor *x = plain(args[0]), *w, *b;
    if (!x || modes_active() || !THPDtype_Check(args[12])) Py_RETURN_NONE;
    int64_t xb, xt, xk, t, m, k, parts, silu, ldq;
    if (!as_int(args[1], &xb) || !as_int(args[2], &xt) || !as_int(args[3], &xk) || !as_int(args[4], &t) ||
        !as_int(args[5], &m) || !as_int(args[6], &k) || !as_int(args[7], &parts) || !as_int(args[11], &silu) ||
        !as_int(args[13], &ldq) || !optional(args[8], x->device(), &w) || !optional(args[9], x->device(), &b))
        Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(args[10]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const int xc = code_of(x->scalar_type());
    const auto qs_type = ((THPDtype *)args[12])->scalar_type;
    const int qc = code_of(qs_type);
    if ((xc != KEA_F32 && xc != KEA_F16) || (qc != KEA_F32 && qc != KEA_F16) || m < 1 || k < 1 || t < 1 || xb < 0 ||
        xt < 0 || xk < 0 || parts < 1 || parts > 3 || m > INT32_MAX || k > 8192 || ldq < k || (w != nullptr) != (b != nullptr))
        Py_RETURN_NONE;
    for (const at::Tensor *v : {w, b})
        if (v && (v->scalar_type() != at::kFloat || !v->is_contiguous() || v->numel() != k)) Py_RETURN_NONE;
    // the furthest element any row reads lies in x's storage (each factor is below 2^31 or a stride of x's own storage)
    const int64_t bl = (m - 1) / t, rl = (m - 1) % t;
    const int64_t limit = (int64_t)(x->storage().nbytes() / x->element_size());
    if (xb > limit || xt > limit || xk > limit) Py_RETURN_NONE;
    __int128 far = (__int128)bl * xb + (__int128)rl * xt;
    if (bl >= 1) {
        const __int128 other = (__int128)(bl - 1) * xb + (__int128)(t - 1) * xt;
        if (other > far) far = other;
    }
    far += (__int128)(k - 1) * xk + x->storage_offset();
    if (far >= limit) Py_RETURN_NONE;
    try {
        const auto device = x->device();
        at::Tensor q = at::empty({parts, m, ldq}, at::TensorOptions().device(device).dtype(at::kChar));
        at::Tensor qs = at::empty({parts, m}, at::TensorOptions().device(device).dtype(qs_type));
        const int rc = lib.quantize(x->const_data_ptr(), xc, xb, xt, xk, t, m, k, (int)parts,
                                    w ? (const float *)w->const_data_ptr() : nullptr,
                                    b ? (const float *)b->const_data_ptr() : nullptr, (float)eps, (int)(silu != 0),
                                    (int8_t *)q.mutable_data_ptr(), ldq, qs.mutable_data_ptr(), qc, stream_of(device));
        if (rc != 0) Py_RETURN_NONE;
        PyObject *qo = THPVariable_Wrap(std::move(q)), *so = THPVariable_Wrap(std::move(qs));
        PyObject *r = qo && so ? PyTuple_Pack(2, qo, so) : nullptr;
        Py_XDECREF(qo);
        Py_XDECREF(so);
        return r;
    } catch (const std::exception &) {
        Py_RETURN_NONE;
    }
}

// gemm(wbits, q, qs, words, words_needed, n, k, wscale, bias, y, acc_out, m, flags, split, tile, ws_group, workspace_bytes,
// residual, factor) -> True where the checks of lowbit.gemm hold and the launch went out
PyObject *native_gemm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != 19) Py_RETURN_FALSE;
    const at::Tensor *q = plain(args[1]);
    if (!q || modes_active()) Py_RETURN_FALSE;
    const auto device = q->device();
    const at::Tensor *qs, *words, *ws, *bias, *y, *acc, *res;
    int64_t wbits, words_needed, n, k, m, flags, split, tile, group, need;
    if (!optional(args[2], device, &qs) || !optional(args[3], device, &words) || !optional(args[7], device, &ws) ||
        !optional(args[8], device, &bias) || !optional(args[9], device, &y) || !optional(args[10], device, &acc) ||
        !optional(args[17], device, &res) || !as_int(args[0], &wbits) || !as_int(args[4], &words_needed) ||
        !as_int(args[5], &n) || !as_int(args[6], &k) || !as_int(args[11], &m) || !as_int(args[12], &flags) ||
        !as_int(args[13], &split) || !as_int(args[14], &tile) || !as_int(args[15], &group) || !as_int(args[16], &need))
        Py_RETURN_FALSE;
    const double factor = PyFloat_AsDouble(args[18]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    if (!qs || !words || !ws || (!y && !acc) || (res && !y)) Py_RETURN_FALSE;
    if (q->scalar_type() != at::kChar || q->dim() != 3 || q->stride(2) != 1 || q->stride(1) != q->size(2)) Py_RETURN_FALSE;
    const int64_t parts = q->size(0), ldq = q->size(2);
    const int sc = code_of(qs->scalar_type()), wc = code_of(ws->scalar_type()), bc = bias ? code_of(bias->scalar_type()) : KEA_F32;
    const int yc = y ? code_of(y->scalar_type()) : KEA_F32;
    auto scale = [](int c) { return c == KEA_F32 || c == KEA_F16; };
    const int64_t groups = group > 0 ? (k + group - 1) / group : 1, ny = (flags & KEA_FLAG_GLU) ? n / 2 : n;
    if ((wbits != 1 && wbits != 2) || parts < 1 || parts > 3 || n < 1 || k < 1 || m < 1 || m > q->size(1) || group < 0 ||
        !scale(sc) || !scale(wc) || !scale(bc) || yc < 0 || qs->dim() != 2 || qs->size(0) != parts || qs->size(1) < m ||
        qs->stride(1) != 1 || !ws->is_contiguous() || ws->numel() < n * groups ||
        (bias && (!bias->is_contiguous() || bias->numel() != n)) || !words->is_contiguous() ||
        words->numel() * (int64_t)words->element_size() < 4 * words_needed ||
        (y && (y->dim() != 2 || y->size(0) < m || y->size(1) < ny || y->stride(1) != 1)) ||
        (acc && (acc->scalar_type() != at::kInt || acc->dim() != 3 || acc->size(0) != parts || acc->size(1) != m ||
                 acc->size(2) < n || acc->stride(2) != 1 || acc->stride(0) != m * acc->stride(1))) ||
        (res && (res->scalar_type() != at::kFloat || res->dim() != 2 || res->size(0) < m || res->size(1) < n ||
                 res->stride(1) != 1)))
        Py_RETURN_FALSE;
    try {
        at::Tensor space;
        if (need > 0) space = at::empty({need}, at::TensorOptions().device(device).dtype(at::kByte));
        void *sp = need > 0 ? space.mutable_data_ptr() : nullptr;
        auto run = [&](auto fn, auto... tail) {
            return fn((int)wbits, (const int8_t *)q->const_data_ptr(), q->stride(0), ldq, (int)parts, qs->const_data_ptr(), sc,
                      qs->stride(0), (const uint32_t *)words->const_data_ptr(), n, k, ws->const_data_ptr(), wc, group,
                      bias ? bias->const_data_ptr() : nullptr, bc, y ? y->mutable_data_ptr() : nullptr, yc,
                      y ? y->stride(0) : 0, acc ? (int32_t *)acc->mutable_data_ptr() : nullptr, acc ? acc->stride(1) : 0, m,
                      (int)flags, (int)split, (int)tile, sp, need, tail...);
        };
        const int rc = res ? run(lib.gemm_residual, (const float *)res->const_data_ptr(), (int64_t)res->stride(0), (float)factor,
                                 stream_of(device))
                           : run(lib.gemm, stream_of(device));
        if (rc == 0) Py_RETURN_TRUE;
    } catch (const std::exception &) {
    }
    Py_RETURN_FALSE;
}

// ---- int8.gemm, norms.block_norm, window.attention ----

// Whether launches on `d` can be made from here: the default stream's handle names the current device's.
bool current(c10::Device d) { return d.index() == c10::hip::current_device(); }

bool as_float(PyObject *o, double *v) {
    *v = PyFloat_AsDouble(o);
    if (!PyErr_Occurred()) return true;
    PyErr_Clear();
    return false;
}

// The first dimensions of t as rows of its last one with one stride (of rows: 1 row, any stride), without a copy.
bool rows_of(const at::Tensor &t, int64_t *rows, int64_t *stride) {
    const int64_t dim = t.dim();
    if (dim < 1 || t.size(dim - 1) < 1 || (t.size(dim - 1) > 1 && t.stride(dim - 1) != 1)) return false;
    *rows = 1;
    *stride = t.size(dim - 1);
    for (int64_t i = dim - 2; i >= 0; --i) {
        const int64_t n = t.size(i);
        if (n == 0) return false;
        if (n == 1) continue;
        if (*rows == 1) *stride = t.stride(i);
        else if (t.stride(i) != *stride * *rows) return false;
        *rows *= n;
    }
    return true;
}

// Whether the bytes from a's first element to its last meet b's (or `bytes` at b). (An output that lies between an input's
// rows meets it too; the Python path sorts that out.)
int64_t reach(const at::Tensor &t) {
    int64_t last = 1;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return last * (int64_t)t.element_size();
}
bool meet(const at::Tensor &a, const void *b, int64_t bytes) {
    const uintptr_t from = (uintptr_t)a.const_data_ptr(), other = (uintptr_t)b;
    return b && from < other + bytes && other < from + reach(a);
}
bool meet(const at::Tensor &a, const at::Tensor &b) { return meet(a, b.const_data_ptr(), reach(b)); }

// int8 rows [.., k] that start at multiples of 16 bytes, the last one readable to a multiple of 16 of `k` elements.
bool rows8(const at::Tensor &t, int64_t dim, int64_t k, int64_t *ld) {
    const int64_t m = t.size(dim), w = t.size(dim + 1);
    if (t.scalar_type() != at::kChar || (w > 1 && t.stride(dim + 1) != 1) || (uintptr_t)t.const_data_ptr() % 16) return false;
    *ld = m > 1 ? t.stride(dim) : (w + 15) / 16 * 16;
    return m >= 1 && *ld % 16 == 0 && *ld >= w && t.storage_offset() + (m - 1) * *ld + (k + 15) / 16 * 16 <= (int64_t)t.storage().nbytes();
}

// int8_gemm(q, qs, weight, wscale, bias, out, out_dtype, silu, residual, factor) -> the output, or None
PyObject *native_int8_gemm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != 10) Py_RETURN_NONE;
    const at::Tensor *q = plain(args[0]);
    if (!q || modes_active()) Py_RETURN_NONE;
    const auto device = q->device();
    const at::Tensor *qs, *w, *ws, *bias, *out, *res;
    int64_t silu;
    double factor;
    if (!current(device) || !optional(args[1], device, &qs) || !optional(args[2], device, &w) || !optional(args[3], device, &ws) ||
        !optional(args[4], device, &bias) || !optional(args[5], device, &out) || !optional(args[8], device, &res) ||
        !as_int(args[7], &silu) || !as_float(args[9], &factor) || !THPDtype_Check(args[6]) || !qs || !w || !ws)
        Py_RETURN_NONE;
    const auto type = out ? out->scalar_type() : ((THPDtype *)args[6])->scalar_type;
    const int yc = code_of(type), sc = code_of(qs->scalar_type()), wc = code_of(ws->scalar_type()), bc = bias ? code_of(bias->scalar_type()) : KEA_F32;
    auto scale = [](int c) { return c == KEA_F32 || c == KEA_F16; };
    const int64_t qd = q->dim() - 2;
    if (yc < 0 || !scale(sc) || !scale(wc) || !scale(bc) || (qd != 0 && (qd != 1 || q->size(0) != 1)) || w->dim() != 2) Py_RETURN_NONE;
    const int64_t m = q->size(qd), n = w->size(0), k = w->size(1);
    int64_t ldq, ldw;
    if (m < 1 || n < 1 || k < 1 || k > 131071 || q->size(qd + 1) < k || !rows8(*q, qd, k, &ldq) || !rows8(*w, 0, k, &ldw) ||
        !qs->is_contiguous() || qs->numel() != m || !ws->is_contiguous() || ws->numel() != n ||
        (bias && (!bias->is_contiguous() || bias->numel() != n)) ||
        (res && (res->scalar_type() != at::kFloat || res->dim() != 2 || res->size(0) != m || res->size(1) != n || (n > 1 && res->stride(1) != 1))) ||
        (out && (out->dim() != 2 || out->size(0) != m || out->size(1) != n || (n > 1 && out->stride(1) != 1) || (m > 1 && out->stride(0) < n))))
        Py_RETURN_NONE;
    if (out) {
        const bool same = res && out->const_data_ptr() == res->const_data_ptr() && type == at::kFloat && (m == 1 || out->stride(0) == res->stride(0));
        for (const at::Tensor *t : {q, qs, w, ws, bias, same ? nullptr : res})
            if (t && meet(*out, *t)) Py_RETURN_NONE;
    }
    try {
        at::Tensor y = out ? *out : at::empty({m, n}, at::TensorOptions().device(device).dtype(type));
        const int rc = lib.int8_gemm((const int8_t *)q->const_data_ptr(), ldq, qs->const_data_ptr(), sc, (const int8_t *)w->const_data_ptr(), ldw,
                                     ws->const_data_ptr(), wc, bias ? bias->const_data_ptr() : nullptr, bc, y.mutable_data_ptr(), yc,
                                     m > 1 ? y.stride(0) : n, res ? (const float *)res->const_data_ptr() : nullptr, res && m > 1 ? res->stride(0) : n,
                                     (float)factor, m, n, k, silu ? KEA_FLAG_SILU : 0, stream_of(device));
        if (rc == 0) return THPVariable_Wrap(std::move(y));
    } catch (const std::exception &) {
    }
    Py_RETURN_NONE;
}

// A norm given as (kind, weight, bias, eps) in four arguments; false where autograd would have to record its parameters.
bool norm_of(PyObject *const *args, int64_t d, c10::Device device, kea_norm *n) {
    int64_t kind;
    double eps;
    if (!as_int(args[0], &kind) || !as_float(args[3], &eps)) return false;
    *n = kea_norm{(int)kind, KEA_F32, nullptr, nullptr, (float)eps};
    int type = -1;
    for (int i = 0; i < 2; ++i) {
        if (args[1 + i] == Py_None) continue;
        if (!THPVariable_Check(args[1 + i])) return false;
        const at::Tensor &t = THPVariable_Unpack(args[1 + i]);
        if (!t.defined() || t.device() != device || t.layout() != at::kStrided || !t.has_storage() || !t.is_contiguous() || t.numel() != d ||
            (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined() || t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                                     c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Negative})))
            return false;
        const int c = code_of(t.scalar_type());
        if (c < 0 || (type >= 0 && c != type)) return false;
        type = c;
        (i ? n->b_dev : n->w_dev) = t.const_data_ptr();
    }
    if (type >= 0) n->dtype = type;
    return true;
}

// block_norm(x, block, post x 4, gate, act, factor, pre x 4, quantize, out) -> (y, z) or (y, q, qs), or None. See norm_of.
PyObject *native_block_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != 15) Py_RETURN_NONE;
    const at::Tensor *x = plain(args[0]);
    if (!x || modes_active()) Py_RETURN_NONE;
    const auto device = x->device();
    const at::Tensor *block, *gate, *out;
    int64_t act, quantize, m, ldx, mb, ldb, ldg = 0, gates = 1, my, ldy;
    double factor;
    kea_norm post, pre;
    if (!current(device) || !optional(args[1], device, &block) || !block || !optional(args[6], device, &gate) || !as_int(args[7], &act) ||
        !as_float(args[8], &factor) || !as_int(args[13], &quantize) || !optional(args[14], device, &out) || x->dim() < 1)
        Py_RETURN_NONE;
    const int64_t d = x->size(x->dim() - 1);
    const int xc = code_of(x->scalar_type()), bc = code_of(block->scalar_type());
    if (xc < 0 || bc < 0 || block->sizes() != x->sizes() || d < 1 || d > 32768 || !rows_of(*x, &m, &ldx) || !rows_of(*block, &mb, &ldb) ||
        !norm_of(args + 2, d, device, &post) || !norm_of(args + 9, d, device, &pre) || act < 0 || act > 2)
        Py_RETURN_NONE;
    if (gate && (gate->scalar_type() != block->scalar_type() || gate->dim() < 1 || gate->size(gate->dim() - 1) != d ||
                 !rows_of(*gate, &gates, &ldg) || m % gates))
        Py_RETURN_NONE;
    if (out && (out->scalar_type() != x->scalar_type() || out->sizes() != x->sizes() || !rows_of(*out, &my, &ldy) || ldy < d)) Py_RETURN_NONE;
    if (out) {
        auto same = [&](const at::Tensor &t, int64_t ld) {
            return t.scalar_type() == out->scalar_type() && t.const_data_ptr() == out->const_data_ptr() && (m == 1 || ld == ldy);
        };
        if ((!same(*x, ldx) && meet(*out, *x)) || (!same(*block, ldb) && meet(*out, *block)) || (gate && meet(*out, *gate))) Py_RETURN_NONE;
        for (const kea_norm *n : {&post, &pre}) {
            const int64_t bytes = d * (n->dtype == KEA_F32 ? 4 : 2);
            if (meet(*out, n->w_dev, bytes) || meet(*out, n->b_dev, bytes)) Py_RETURN_NONE;
        }
    }
    try {
        const auto options = at::TensorOptions().device(device);
        at::Tensor y = out ? *out : at::empty(x->sizes(), options.dtype(x->scalar_type())), z, q, qs;
        if (!out) ldy = d;
        const int64_t ldq = (d + 15) / 16 * 16;
        const bool values = !quantize && pre.kind != KEA_NORM_NONE;
        if (values) z = at::empty(x->sizes(), options.dtype(block->scalar_type()));
        if (quantize) {
            q = at::empty({1, m, ldq}, options.dtype(at::kChar));
            qs = at::empty({1, m}, options.dtype(at::kFloat));
        }
        const int rc = lib.block_norm(x->const_data_ptr(), xc, ldx, block->const_data_ptr(), bc, ldb, m, d, &post,
                                      gate ? gate->const_data_ptr() : nullptr, ldg, m / gates, gate ? (int)act : 0, (float)factor,
                                      y.mutable_data_ptr(), ldy, &pre, values ? z.mutable_data_ptr() : nullptr, d,
                                      quantize ? (int8_t *)q.mutable_data_ptr() : nullptr, ldq,
                                      quantize ? (float *)qs.mutable_data_ptr() : nullptr, stream_of(device));
        if (rc != 0) Py_RETURN_NONE;
        const THPObjectPtr yo(THPVariable_Wrap(std::move(y)));
        if (quantize) {
            const THPObjectPtr qo(THPVariable_Wrap(std::move(q))), so(THPVariable_Wrap(std::move(qs)));
            return PyTuple_Pack(3, yo.get(), qo.get(), so.get());
        }
        const THPObjectPtr zo(values ? THPVariable_Wrap(std::move(z)) : Py_NewRef(Py_None));
        return PyTuple_Pack(2, yo.get(), zo.get());
    } catch (const std::exception &) {
        Py_RETURN_NONE;
    }
}

bool heads_of(const at::Tensor &t, at::ScalarType type, int64_t b, int64_t d, kea_heads *h) {
    if (t.scalar_type() != type || t.dim() != 4 || t.size(0) != b || t.size(3) != d || t.stride(3) != 1 || (uintptr_t)t.const_data_ptr() % 16 ||
        t.size(1) > (1 << 30))
        return false;
    const int64_t unit = 16 / (int64_t)t.element_size();
    int64_t s[3];
    for (int i = 0; i < 3; ++i) {
        s[i] = t.size(i) > 1 ? t.stride(i) : 0;
        if (s[i] % unit) return false;
    }
    *h = kea_heads{const_cast<void *>(t.const_data_ptr()), s[0], s[1], s[2]};
    return true;
}

// window_attention(q, k, v, left, right, sinks, scale, kv_lengths, q_starts) -> the output, or None. left, right: None or int.
PyObject *native_window(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != 9) Py_RETURN_NONE;
    const at::Tensor *q = plain(args[0]);
    if (!q || modes_active()) Py_RETURN_NONE;
    const auto device = q->device();
    const at::Tensor *k, *v, *lengths, *starts;
    int64_t left = 1 << 30, right = 1 << 30, sinks;
    double scale;
    if (!current(device) || !optional(args[1], device, &k) || !optional(args[2], device, &v) || !k || !v || !PyLong_CheckExact(args[5]) ||
        !as_int(args[5], &sinks) || (args[3] != Py_None && (!PyLong_CheckExact(args[3]) || !as_int(args[3], &left))) ||
        (args[4] != Py_None && (!PyLong_CheckExact(args[4]) || !as_int(args[4], &right))) || !optional(args[7], device, &lengths) ||
        !optional(args[8], device, &starts) || q->dim() != 4 || k->dim() != 4)
        Py_RETURN_NONE;
    const int64_t b = q->size(0), tq = q->size(1), h = q->size(2), d = q->size(3), tk = k->size(1), hk = k->size(2);
    const int code = code_of(q->scalar_type());
    kea_heads qh, kh, vh;
    if (code < 0 || d < 8 || d % 8 || d > 256 || h < 1 || hk < 1 || h % hk || b < 1 || tq < 1 || left < 0 || right < 0 || sinks < 0 ||
        v->sizes() != k->sizes() || !heads_of(*q, q->scalar_type(), b, d, &qh) || !heads_of(*k, q->scalar_type(), b, d, &kh) ||
        !heads_of(*v, q->scalar_type(), b, d, &vh))
        Py_RETURN_NONE;
    for (const at::Tensor *t : {lengths, starts})
        if (t && (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != b || !t->is_contiguous())) Py_RETURN_NONE;
    if (args[6] == Py_None) scale = 1.0 / std::sqrt((double)d);
    else if (!as_float(args[6], &scale)) Py_RETURN_NONE;
    try {
        at::Tensor y = at::empty({b, tq, h, d}, at::TensorOptions().device(device).dtype(q->scalar_type())), space;
        const kea_heads yh{y.mutable_data_ptr(), tq * h * d, h * d, d};
        const int64_t need = lib.window_workspace(code, b, tq, tk, h, hk, d, left, right, sinks);
        if (need < 0) Py_RETURN_NONE;
        if (need > 0) space = at::empty({need}, at::TensorOptions().device(device).dtype(at::kByte));
        const int rc = lib.window(&qh, &kh, &vh, &yh, code, b, tq, tk, h, hk, d, left, right, sinks, (float)scale,
                                  lengths ? (const int32_t *)lengths->const_data_ptr() : nullptr,
                                  starts ? (const int32_t *)starts->const_data_ptr() : nullptr, need > 0 ? space.mutable_data_ptr() : nullptr, need,
                                  stream_of(device));
        if (rc == 0) return THPVariable_Wrap(std::move(y));
    } catch (const std::exception &) {
    }
    Py_RETURN_NONE;
}

// int4_gemm(q, qs, words, scales, n, k, group, bias, out, out_dtype, silu, residual, factor) -> the output, or None
PyObject *native_int4_gemm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != 13) Py_RETURN_NONE;
    const at::Tensor *q = plain(args[0]);
    if (!q || modes_active()) Py_RETURN_NONE;
    const auto device = q->device();
    const at::Tensor *qs, *w, *ws, *bias, *out, *res;
    int64_t n, k, group, silu;
    double factor;
    if (!current(device) || !optional(args[1], device, &qs) || !optional(args[2], device, &w) || !optional(args[3], device, &ws) ||
        !as_int(args[4], &n) || !as_int(args[5], &k) || !as_int(args[6], &group) || !optional(args[7], device, &bias) ||
        !optional(args[8], device, &out) || !THPDtype_Check(args[9]) || !as_int(args[10], &silu) || !optional(args[11], device, &res) ||
        !as_float(args[12], &factor) || !qs || !w || !ws)
        Py_RETURN_NONE;
    const auto type = out ? out->scalar_type() : ((THPDtype *)args[9])->scalar_type;
    const int yc = code_of(type), sc = code_of(qs->scalar_type()), wc = code_of(ws->scalar_type()), bc = bias ? code_of(bias->scalar_type()) : KEA_F32;
    auto scale = [](int c) { return c == KEA_F32 || c == KEA_F16; };
    const int64_t qd = q->dim() - 2;
    if (yc < 0 || !scale(sc) || !scale(wc) || !scale(bc) || (qd != 0 && (qd != 1 || q->size(0) != 1)) || n < 1 || n > INT32_MAX || k < 1 || k > (1 << 20) ||
        group < 32 || group > (1 << 30) || (group & (group - 1)))
        Py_RETURN_NONE;
    const int64_t m = q->size(qd), tiles = (n + 15) / 16, blocks = (k + 127) / 128, groups = (k + group - 1) / group;
    int64_t ldq;
    if (m < 1 || q->size(qd + 1) < k || !rows8(*q, qd, k, &ldq) || !qs->is_contiguous() || qs->numel() != m ||
        w->scalar_type() != at::kInt || !w->is_contiguous() || w->numel() != tiles * blocks * 256 || (uintptr_t)w->const_data_ptr() % 16 ||
        ws->dim() != 3 || ws->size(0) != tiles || ws->size(1) != groups || ws->size(2) != 16 || !ws->is_contiguous() || (uintptr_t)ws->const_data_ptr() % 16 ||
        (bias && (!bias->is_contiguous() || bias->numel() != n)) ||
        (res && (res->scalar_type() != at::kFloat || res->dim() != 2 || res->size(0) != m || res->size(1) != n || (n > 1 && res->stride(1) != 1) || (m > 1 && res->stride(0) < n))) ||
        (out && (out->dim() != 2 || out->size(0) != m || out->size(1) != n || (n > 1 && out->stride(1) != 1) || (m > 1 && out->stride(0) < n))))
        Py_RETURN_NONE;
    if (out) {
        const bool same = res && out->const_data_ptr() == res->const_data_ptr() && type == at::kFloat && (m == 1 || out->stride(0) == res->stride(0));
        for (const at::Tensor *t : {q, qs, w, ws, bias, same ? nullptr : res})
            if (t && meet(*out, *t)) Py_RETURN_NONE;
    }
    try {
        at::Tensor y = out ? *out : at::empty({m, n}, at::TensorOptions().device(device).dtype(type));
        const int rc = lib.int4_gemm((const int8_t *)q->const_data_ptr(), ldq, qs->const_data_ptr(), sc, (const uint32_t *)w->const_data_ptr(),
                                     ws->const_data_ptr(), wc, group, bias ? bias->const_data_ptr() : nullptr, bc, y.mutable_data_ptr(), yc,
                                     m > 1 ? y.stride(0) : n, res ? (const float *)res->const_data_ptr() : nullptr, res && m > 1 ? res->stride(0) : n,
                                     (float)factor, m, n, k, silu ? KEA_FLAG_SILU : 0, stream_of(device));
        if (rc == 0) return THPVariable_Wrap(std::move(y));
    } catch (const std::exception &) {
    }
    Py_RETURN_NONE;
}

// The cache's tensors (args[0 .. 3]: k, v and their scales) as kea_pages; false where they are not what paged.Cache holds.
struct PagedCache {
    const at::Tensor *t[4];
    kea_pages k, v;
    int64_t pages, heads, size, d;
};
bool cache_of(PyObject *const *args, PagedCache *c) {
    for (int i = 0; i < 4; ++i)
        if (!(c->t[i] = plain(args[i])) || c->t[i]->device() != c->t[0]->device()) return false;
    const at::Tensor &k = *c->t[0];
    if (k.dim() != 4) return false;
    c->pages = k.size(0), c->heads = k.size(1), c->size = k.size(2), c->d = k.size(3);
    for (int i = 0; i < 2; ++i) {
        const at::Tensor &t = *c->t[i], &s = *c->t[2 + i];
        if (t.scalar_type() != at::kChar || t.sizes() != k.sizes() || t.stride(3) != 1 || (uintptr_t)t.const_data_ptr() % 16 || s.scalar_type() != at::kFloat ||
            s.dim() != 3 || s.size(0) != c->pages || s.size(1) != c->heads || s.size(2) != c->size)
            return false;
        int64_t st[6];
        for (int j = 0; j < 3; ++j) {
            st[j] = t.size(j) > 1 ? t.stride(j) : 0;
            st[3 + j] = s.size(j) > 1 ? s.stride(j) : 0;
            if (st[j] % 16) return false;
        }
        (i ? c->v : c->k) = kea_pages{(int8_t *)const_cast<void *>(t.const_data_ptr()), (float *)const_cast<void *>(s.const_data_ptr()), st[0], st[1], st[2], st[3], st[4], st[5]};
    }
    return true;
}

bool index_of(const at::Tensor *t, int64_t n) { return t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous(); }

// The table, lengths and offsets (args[0 .. 2]; offsets may be None) for `tokens` new tokens.
bool paging_of(PyObject *const *args, const PagedCache &c, int64_t tokens, const at::Tensor **t, kea_paging *g) {
    const auto device = c.t[0]->device();
    t[0] = plain(args[0]), t[1] = plain(args[1]);
    if (!t[0] || !t[1] || t[0]->device() != device || t[1]->device() != device || !optional(args[2], device, &t[2])) return false;
    const at::Tensor &table = *t[0];
    if (table.scalar_type() != at::kInt || table.dim() != 2 || (table.size(1) > 1 && table.stride(1) != 1)) return false;
    const int64_t batch = table.size(0), width = table.size(1);
    if (batch < 1 || width * c.size > (1 << 30) || !index_of(t[1], batch) || (t[2] ? !index_of(t[2], batch + 1) : tokens % batch != 0)) return false;
    *g = kea_paging{(const int32_t *)table.const_data_ptr(), (const int32_t *)t[1]->const_data_ptr(), t[2] ? (const int32_t *)t[2]->const_data_ptr() : nullptr,
                    batch > 1 ? table.stride(0) : 0, width, batch, c.pages, c.size, tokens};
    return true;
}

// [tokens][heads][d] of a float type; heads 0: any number.
bool tokens_of(const at::Tensor &t, int64_t heads, int64_t d, kea_heads *h) {
    if (code_of(t.scalar_type()) < 0 || t.dim() != 3 || t.size(0) < 1 || (heads && t.size(1) != heads) || t.size(2) != d || t.stride(2) != 1 || (uintptr_t)t.const_data_ptr() % 16)
        return false;
    const int64_t unit = 16 / (int64_t)t.element_size();
    int64_t s[2];
    for (int i = 0; i < 2; ++i) {
        s[i] = t.size(i) > 1 ? t.stride(i) : 0;
        if (s[i] % unit) return false;
    }
    *h = kea_heads{const_cast<void *>(t.const_data_ptr()), 0, s[0], s[1]};
    return true;
}

// paged_write(cache x 4, k, v, table, kv_lengths, q_offsets) -> True, or None
PyObject *native_paged_write(PyObject *, PyObject *const *args, Py_ssize_t count) {
    PagedCache c;
    const at::Tensor *g[3], *x[2];
    kea_heads h[2];
    kea_paging paging;
    if (count != 9 || modes_active() || !cache_of(args, &c)) Py_RETURN_NONE;
    const auto device = c.t[0]->device();
    if (!current(device) || !optional(args[4], device, &x[0]) || !optional(args[5], device, &x[1]) || !x[0] || !x[1] || x[0]->scalar_type() != x[1]->scalar_type() ||
        x[0]->sizes() != x[1]->sizes() || !tokens_of(*x[0], c.heads, c.d, &h[0]) || !tokens_of(*x[1], c.heads, c.d, &h[1]) ||
        !paging_of(args + 6, c, x[0]->size(0), g, &paging))
        Py_RETURN_NONE;
    for (const at::Tensor *to : c.t)
        for (const at::Tensor *t : {x[0], x[1], g[0], g[1], g[2]})
            if (t && to->numel() && t->numel() && meet(*to, *t)) Py_RETURN_NONE;
    try {
        if (lib.paged_write(&h[0], &h[1], code_of(x[0]->scalar_type()), c.heads, c.d, &c.k, &c.v, &paging, stream_of(device)) == 0) Py_RETURN_TRUE;
    } catch (const std::exception &) {
    }
    Py_RETURN_NONE;
}

// paged_read(cache x 4, table, kv_lengths, length, starts, out_dtype) -> (k, v), or None
PyObject *native_paged_read(PyObject *, PyObject *const *args, Py_ssize_t count) {
    PagedCache c;
    const at::Tensor *g[3], *starts;
    kea_paging paging;
    int64_t length;
    if (count != 9 || modes_active() || !cache_of(args, &c)) Py_RETURN_NONE;
    const auto device = c.t[0]->device();
    PyObject *const index[3] = {args[4], args[5], Py_None};
    if (!current(device) || !paging_of(index, c, 0, g, &paging) || !PyLong_CheckExact(args[6]) || !as_int(args[6], &length) || length < 1 || length > (1 << 30) ||
        !optional(args[7], device, &starts) || (starts && !index_of(starts, paging.batch)) || !THPDtype_Check(args[8]))
        Py_RETURN_NONE;
    const auto type = ((THPDtype *)args[8])->scalar_type;
    if (code_of(type) < 0) Py_RETURN_NONE;
    try {
        const auto options = at::TensorOptions().device(device).dtype(type);
        at::Tensor k = at::empty({paging.batch, length, c.heads, c.d}, options), v = at::empty({paging.batch, length, c.heads, c.d}, options);
        if (lib.paged_read(&c.k, &c.v, &paging, starts ? (const int32_t *)starts->const_data_ptr() : nullptr, length, c.heads, c.d, k.mutable_data_ptr(),
                           v.mutable_data_ptr(), code_of(type), stream_of(device)) != 0)
            Py_RETURN_NONE;
        const THPObjectPtr ko(THPVariable_Wrap(std::move(k))), vo(THPVariable_Wrap(std::move(v)));
        return PyTuple_Pack(2, ko.get(), vo.get());
    } catch (const std::exception &) {
        Py_RETURN_NONE;
    }
}

// paged_attention(cache x 4, q, table, kv_lengths, q_offsets, left, scale) -> the output, or None. left: None or int.
PyObject *native_paged_attention(PyObject *, PyObject *const *args, Py_ssize_t count) {
    PagedCache c;
    const at::Tensor *g[3], *q;
    kea_heads h;
    kea_paging paging;
    int64_t left = 1 << 30;
    double scale;
    if (count != 10 || modes_active() || !cache_of(args, &c)) Py_RETURN_NONE;
    const auto device = c.t[0]->device();
    if (!current(device) || !optional(args[4], device, &q) || !q || !tokens_of(*q, 0, c.d, &h) || q->size(1) < 1 || q->size(1) % c.heads ||
        !paging_of(args + 5, c, q->size(0), g, &paging) || (args[8] != Py_None && (!PyLong_CheckExact(args[8]) || !as_int(args[8], &left) || left < 0)))
        Py_RETURN_NONE;
    if (args[9] == Py_None) scale = 1.0 / std::sqrt((double)c.d);
    else if (!as_float(args[9], &scale)) Py_RETURN_NONE;
    if (left > 1 << 30) left = 1 << 30;
    try {
        const int64_t tokens = q->size(0), heads = q->size(1);
        const int code = code_of(q->scalar_type());
        at::Tensor y = at::empty({tokens, heads, c.d}, at::TensorOptions().device(device).dtype(q->scalar_type())), space;
        const kea_heads yh{y.mutable_data_ptr(), 0, heads * c.d, c.d};
        const int64_t need = lib.paged_workspace(code, paging.batch, tokens, paging.table_width * c.size, heads, c.heads, c.d, left, g[2] != nullptr);
        if (need < 0) Py_RETURN_NONE;
        if (need > 0) space = at::empty({need}, at::TensorOptions().device(device).dtype(at::kByte));
        if (lib.paged_attention(&h, &yh, code, heads, c.heads, c.d, &c.k, &c.v, &paging, left, (float)scale, 1, need > 0 ? space.mutable_data_ptr() : nullptr, need,
                                stream_of(device)) == 0)
            return THPVariable_Wrap(std::move(y));
    } catch (const std::exception &) {
    }
    Py_RETURN_NONE;
}

// bind_decode(int4_gemm, paged_write, paged_read, paged_attention, paged_attention_workspace)
PyObject *native_bind_decode(PyObject *, PyObject *args) {
    unsigned long long g, w, r, a, s;
    if (!PyArg_ParseTuple(args, "KKKKK", &g, &w, &r, &a, &s)) return nullptr;
    lib.int4_gemm = (decltype(lib.int4_gemm))g;
    lib.paged_write = (decltype(lib.paged_write))w;
    lib.paged_read = (decltype(lib.paged_read))r;
    lib.paged_attention = (decltype(lib.paged_attention))a;
    lib.paged_workspace = (decltype(lib.paged_workspace))s;
    Py_RETURN_NONE;
}

// bind_block(int8_gemm, block_norm, window_attention, window_attention_workspace)
PyObject *native_bind_block(PyObject *, PyObject *args) {
    unsigned long long g, n, w, ww;
    if (!PyArg_ParseTuple(args, "KKKK", &g, &n, &w, &ww)) return nullptr;
    lib.int8_gemm = (decltype(lib.int8_gemm))g;
    lib.block_norm = (decltype(lib.block_norm))n;
    lib.window = (decltype(lib.window))w;
    lib.window_workspace = (decltype(lib.window_workspace))ww;
    Py_RETURN_NONE;
}

// bind(project_launch, gemm, gemm_residual, quantize): the library's entry points as integers
PyObject *native_bind(PyObject *, PyObject *args) {
    unsigned long long p, g, r, q;
    if (!PyArg_ParseTuple(args, "KKKK", &p, &g, &r, &q)) return nullptr;
    lib.project_launch = (decltype(lib.project_launch))p;
    lib.gemm = (decltype(lib.gemm))g;
    lib.gemm_residual = (decltype(lib.gemm_residual))r;
    lib.quantize = (decltype(lib.quantize))q;
    Py_RETURN_NONE;
}

PyMethodDef module_methods[] = {
    {"bind", native_bind, METH_VARARGS, nullptr},
    {"bind_block", native_bind_block, METH_VARARGS, nullptr},
    {"bind_decode", native_bind_decode, METH_VARARGS, nullptr},
    {"int4_gemm", (PyCFunction)(void (*)())native_int4_gemm, METH_FASTCALL, nullptr},
    {"paged_write", (PyCFunction)(void (*)())native_paged_write, METH_FASTCALL, nullptr},
    {"paged_read", (PyCFunction)(void (*)())native_paged_read, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)())native_paged_attention, METH_FASTCALL, nullptr},
    {"int8_gemm", (PyCFunction)(void (*)())native_int8_gemm, METH_FASTCALL, nullptr},
    {"block_norm", (PyCFunction)(void (*)())native_block_norm, METH_FASTCALL, nullptr},
    {"window_attention", (PyCFunction)(void (*)())native_window, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void (*)())native_quantize, METH_FASTCALL, nullptr},
    {"gemm", (PyCFunction)(void (*)())native_gemm, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kea_native", nullptr, -1, module_methods};

}  // namespace

PyMODINIT_FUNC PyInit_kea_native(void) {
    ReplaysType.tp_flags = Py_TPFLAGS_DEFAULT;
    ReplaysType.tp_new = replays_new;
    ReplaysType.tp_dealloc = replays_dealloc;
    ReplaysType.tp_methods = replays_methods;
    if (PyType_Ready(&ReplaysType) < 0) return nullptr;
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddObjectRef(m, "Replays", (PyObject *)&ReplaysType) < 0) Py_CLEAR(m);
    return m;
}
