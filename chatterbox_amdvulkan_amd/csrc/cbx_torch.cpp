// cbx_torch.cpp -- the Python front end's way from torch tensors to the C ABI
// for the calls of a decode step: descriptors filled and outputs allocated in
// C++ (a step's call takes 4 to 11 tensors; in Python each descriptor costs
// more than 1 us, these calls 12 to 14 us of host time together with their
// outputs, and 5.4 to 6.5 here, the launch included).
//
// Every function takes its tensors and numbers by position, then the current
// device's index and the current stream's handle.  It returns the outputs; an
// int instead says what the caller has to do first: kInitDevice (cbx_init for
// the device) or kOtherDevice - index (make the tensors' device the current
// one).  Errors raise the front end's exception with the C ABI's status and
// message.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_ops.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <vector>

#include "../../include/cbxops.h"

namespace {

constexpr long kInitDevice = 1, kOtherDevice = -1000;
PyObject* g_error = nullptr;      // CbxError(status, message)

// Thrown where the Python error is set.
struct Raised {};

[[noreturn]] void raise(int status, const std::string& msg) {
    PyObject* e = PyObject_CallFunction(g_error, "is#", status, msg.data(), static_cast<Py_ssize_t>(msg.size()));
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

// The arguments of one call.
struct Call {
    PyObject* const* args;
    int device;                   // the current one
    cbx_stream stream;
    int other = -1;               // the tensors' device, when it is not
    int first = -1;               // of the first tensor
    int used = 0;
    cbx_tensor d[16];

    Call(PyObject* const* a, Py_ssize_t n, Py_ssize_t want) : args(a) {
        if (n != want + 2) raise(CBX_ERR_INVALID_ARG, "wrong number of arguments");
        device = static_cast<int>(integer(want));
        stream = reinterpret_cast<cbx_stream>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(a[want + 1])));
        if (PyErr_Occurred()) throw Raised{};
    }
    bool none(Py_ssize_t i) const { return args[i] == Py_None; }
    int64_t integer(Py_ssize_t i) const {
        const long long v = PyLong_AsLongLong(args[i]);
        if (v == -1 && PyErr_Occurred()) throw Raised{};
        return v;
    }
    int32_t int32(Py_ssize_t i) const {
        const int64_t v = integer(i);
        if (v != static_cast<int32_t>(v)) raise(CBX_ERR_INVALID_ARG, "a number does not fit in 32 bits");
        return static_cast<int32_t>(v);
    }
    float number(Py_ssize_t i) const {
        const double v = PyFloat_AsDouble(args[i]);
        if (v == -1.0 && PyErr_Occurred()) throw Raised{};
        return static_cast<float>(v);
    }
    const void* handle(Py_ssize_t i) const {
        void* p = PyLong_AsVoidPtr(args[i]);
        if (!p && PyErr_Occurred()) throw Raised{};
        return p;
    }
    const at::Tensor& tensor(Py_ssize_t i) const {
        if (!THPVariable_Check(args[i])) raise(CBX_ERR_INVALID_ARG, "argument " + std::to_string(i) + " is not a tensor");
        return THPVariable_Unpack(args[i]);
    }

    // The descriptor of t: ggml's order, byte strides; a dimension of extent
    // 1 gets the stride a contiguous tensor would have.
    cbx_tensor* describe(const at::Tensor& t) {
        if (!t.is_cuda() && first < 0) raise(CBX_ERR_INVALID_ARG, "tensor is not on a ROCm device");
        const int dev = t.is_cuda() ? t.device().index() : -1;
        if (first < 0) first = dev;
        if (dev != first) raise(CBX_ERR_INVALID_ARG, "tensors on cuda:" + std::to_string(first) + " and " + t.device().str());
        if (dev != device) other = dev;
        cbx_tensor* o = &d[used++];
        const auto sizes = t.sizes();
        const auto strides = t.strides();
        const int n = static_cast<int>(sizes.size());
        if (n > 4) raise(CBX_ERR_INVALID_ARG, "more than 4 dims");
        size_t es;
        switch (t.scalar_type()) {
            case at::kFloat: o->type = CBX_TYPE_F32; es = 4; break;
            case at::kHalf: o->type = CBX_TYPE_F16; es = 2; break;
            case at::kInt: o->type = CBX_TYPE_I32; es = 4; break;
            case at::kChar: o->type = CBX_TYPE_I8; es = 1; break;
            default: raise(CBX_ERR_INVALID_ARG, std::string("unsupported dtype ") + c10::toString(t.scalar_type()));
        }
        o->data = t.data_ptr();
        o->reserved = 0;
        const bool nothing = t.numel() == 0;
        size_t next = es;         // a contiguous tensor's stride here
        for (int i = 0; i < 4; i++) {
            o->ne[i] = i < n ? sizes[n - 1 - i] : 1;
            o->nb[i] = i < n && o->ne[i] != 1 && !nothing ? static_cast<size_t>(strides[n - 1 - i]) * es : next;
            next = o->nb[i] * static_cast<size_t>(o->ne[i]);
        }
        return o;
    }
    cbx_tensor* describe(Py_ssize_t i) { return describe(tensor(i)); }
    cbx_tensor* maybe(Py_ssize_t i) { return none(i) ? nullptr : describe(i); }

    // at::empty, past the dispatch on its options (0.8 us of host time down to 0.65).
    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type) const {
        return at::_ops::empty_memory_format::redispatch(c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::fromIntArrayRefSlow(sizes),
                                                         type, at::kStrided, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)),
                                                         false, std::nullopt);
    }
    // Several outputs of one 4-byte type in one allocation, each 16-byte
    // aligned (a tensor over an allocation takes 0.1 us of host time).  Of one
    // type: torch.save refuses tensors of different types over one storage.
    std::vector<at::Tensor> parts(at::ScalarType type, std::initializer_list<at::DimVector> ps) const {
        int64_t total = 0;
        for (const at::DimVector& p : ps) total += (c10::multiply_integers(p) + 3) / 4 * 4;
        const at::Tensor all = empty({total}, type);
        std::vector<at::Tensor> out;
        out.reserve(ps.size());
        int64_t at = 0;
        for (const at::DimVector& p : ps) {
            at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
            t.unsafeGetTensorImpl()->set_sizes_contiguous(p);
            t.unsafeGetTensorImpl()->set_storage_offset(at);
            at += (t.numel() + 3) / 4 * 4;
            out.push_back(std::move(t));
        }
        return out;
    }
    // The tensor at i, or a new one of these sizes.
    at::Tensor or_empty(Py_ssize_t i, at::IntArrayRef sizes, at::ScalarType type) const {
        return none(i) ? empty(sizes, type) : tensor(i);
    }
    // Whether something has to be done before the inputs' device can be used;
    // asked once all inputs are described and nothing is allocated.
    bool elsewhere() const { return other >= 0; }
    // What a status asks of the caller: nothing, the device's init, or an error.
    bool done(int rc) const {
        if (rc == CBX_OK) return true;
        if (rc != CBX_ERR_NOT_INITIALIZED) raise(rc, cbx_last_error());
        return false;
    }
    PyObject* todo() const { return PyLong_FromLong(other >= 0 ? kOtherDevice - other : kInitDevice); }
};

// The C ABI without the interpreter's lock.
template <typename F> int unlocked(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

PyObject* wrap(const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }

PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
    PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
    if (!r) throw Raised{};
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) {
        PyObject* o = wrap(t);
        if (!o) {
            Py_DECREF(r);
            throw Raised{};
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

// n_past, n_new, free_pages, n_free, block_tables, page_size, n_slots, five outputs or five times None
PyObject* paged_append(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 12);
    cbx_tensor *past = c.describe(0), *nw = c.describe(1), *fr = c.describe(2), *nf = c.describe(3), *tab = c.describe(4);
    const int32_t page = c.int32(5), slots = c.int32(6);
    if (slots < 0) raise(CBX_ERR_INVALID_ARG, "cbx_paged_append: n_slots must be >= 0");
    if (c.elsewhere()) return c.todo();
    const int64_t s = past->ne[0];
    std::vector<at::Tensor> out;
    if (c.none(7)) out = c.parts(at::kInt, {{s}, {1}, {s + 1}, {slots}, {slots}});
    else for (int i = 0; i < 5; i++) out.push_back(c.tensor(7 + i));
    cbx_tensor* o[5];
    for (int i = 0; i < 5; i++) o[i] = c.describe(out[i]);
    if (c.elsewhere()) return c.todo();
    if (!c.done(unlocked([&] { return cbx_paged_append(past, nw, fr, nf, tab, page, o[0], o[1], o[2], o[3], o[4], c.stream); }))) {
        return c.todo();
    }
    return tuple_of({out[0], out[1], out[2], out[3], out[4]});
}

// seq_lens, release, block_tables, page_size, free_pages, n_free, two outputs or None each
PyObject* paged_release(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 8);
    cbx_tensor *len = c.describe(0), *rel = c.describe(1), *tab = c.describe(2), *fr = c.describe(4), *nf = c.describe(5);
    const int32_t page = c.int32(3);
    if (c.elsewhere()) return c.todo();
    const at::Tensor lo = c.or_empty(6, {len->ne[0]}, at::kInt), left = c.or_empty(7, {1}, at::kInt);
    cbx_tensor *dl = c.describe(lo), *dn = c.describe(left);
    if (!c.done(unlocked([&] { return cbx_paged_release(len, rel, tab, page, fr, nf, dl, dn, c.stream); }))) return c.todo();
    return tuple_of({lo, left});
}

// k, v, slots, k_cache, v_cache, k_scale, v_scale
PyObject* paged_store(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 7);
    cbx_tensor *k = c.describe(0), *v = c.describe(1), *sl = c.describe(2), *kc = c.describe(3), *vc = c.describe(4),
               *ks = c.maybe(5), *vs = c.maybe(6);
    if (c.elsewhere()) return c.todo();
    if (!c.done(unlocked([&] {
            return ks || vs ? cbx_paged_store_q8(k, v, sl, kc, ks, vc, vs, c.stream) : cbx_paged_store(k, v, sl, kc, vc, c.stream);
        }))) {
        return c.todo();
    }
    Py_RETURN_NONE;
}

// slots, k_cache, v_cache, k_scale, v_scale, F16 (else F32), out_k, out_v
PyObject* paged_load(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 8);
    cbx_tensor *sl = c.describe(0), *kc = c.describe(1), *vc = c.describe(2), *ks = c.maybe(3), *vs = c.maybe(4);
    const int half = PyObject_IsTrue(a[5]);
    if (half < 0) throw Raised{};
    if (c.elsewhere()) return c.todo();
    const at::DimVector rows{sl->ne[0], kc->ne[2], kc->ne[0]};
    const at::Tensor k = c.or_empty(6, rows, half ? at::kHalf : at::kFloat), v = c.or_empty(7, rows, half ? at::kHalf : at::kFloat);
    cbx_tensor *dk = c.describe(k), *dv = c.describe(v);
    if (!c.done(unlocked([&] { return cbx_paged_load(sl, kc, ks, vc, vs, dk, dv, c.stream); }))) return c.todo();
    return tuple_of({k, v});
}

// q, k, gq, gk, eps, pos, rope, out_q, out_k
PyObject* qk_norm_rope(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 9);
    cbx_tensor *q = c.describe(0), *k = c.describe(1), *gq = c.maybe(2), *gk = c.maybe(3), *pos = c.describe(5);
    const float eps = c.number(4);
    const auto* rope = static_cast<const cbx_rope_cache*>(c.handle(6));
    if (c.elsewhere()) return c.todo();
    const at::Tensor &tq = c.tensor(0), &tk = c.tensor(1);
    const at::Tensor yq = c.or_empty(7, tq.sizes(), tq.scalar_type()), yk = c.or_empty(8, tk.sizes(), tk.scalar_type());
    cbx_tensor *dq = c.describe(yq), *dk = c.describe(yk);
    if (!c.done(unlocked([&] { return cbx_qk_norm_rope(q, gq, k, gk, eps, pos, rope, dq, dk, c.stream); }))) return c.todo();
    return tuple_of({yq, yk});
}

// q, k, v, gq, gk, eps, pos, rope, slots, k_cache, v_cache, out_q, k_scale, v_scale
PyObject* qk_norm_rope_store(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 14);
    cbx_tensor *q = c.describe(0), *k = c.describe(1), *v = c.describe(2), *gq = c.maybe(3), *gk = c.maybe(4), *pos = c.describe(6),
               *sl = c.describe(8), *kc = c.describe(9), *vc = c.describe(10), *ks = c.maybe(12), *vs = c.maybe(13);
    const float eps = c.number(5);
    const auto* rope = static_cast<const cbx_rope_cache*>(c.handle(7));
    if (c.elsewhere()) return c.todo();
    const at::Tensor& tq = c.tensor(0);
    const at::Tensor yq = c.or_empty(11, tq.sizes(), tq.scalar_type());
    cbx_tensor* dq = c.describe(yq);
    if (!c.done(unlocked([&] {
            return ks || vs ? cbx_qk_norm_rope_store_q8(q, gq, k, gk, v, eps, pos, rope, sl, dq, kc, ks, vc, vs, c.stream)
                            : cbx_qk_norm_rope_store(q, gq, k, gk, v, eps, pos, rope, sl, dq, kc, vc, c.stream);
        }))) {
        return c.todo();
    }
    return wrap(yq);
}

// Scratch of `bytes`: the caller's (at i) or torch's, on the current stream.
struct Scratch {
    at::Tensor t;
    void* p = nullptr;
    size_t bytes = 0;
};
Scratch scratch(const Call& c, Py_ssize_t i, size_t bytes) {
    Scratch s;
    if (c.none(i)) {
        if (!bytes) return s;
        s.t = c.empty({static_cast<int64_t>(bytes)}, at::kByte);
    } else {
        s.t = c.tensor(i);
        if (!s.t.is_cuda() || s.t.device().index() != c.device || !s.t.is_contiguous()) {
            raise(CBX_ERR_INVALID_ARG, "ws must be a contiguous tensor on the call's device");
        }
    }
    s.p = s.t.data_ptr();
    s.bytes = s.t.nbytes();
    return s;
}

// q, k_cache, v_cache, block_tables, seq_lens, scale, softcap, window, out, ws, k_scale, v_scale
PyObject* paged_attention(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 12);
    cbx_tensor *q = c.describe(0), *k = c.describe(1), *v = c.describe(2), *tab = c.describe(3), *len = c.describe(4),
               *ks = c.maybe(10), *vs = c.maybe(11);
    const float scale = c.number(5), cap = c.number(6);
    const int32_t window = c.int32(7);
    if (c.elsewhere()) return c.todo();
    size_t bytes = 0;
    if (c.none(9) && !c.done(cbx_paged_attention_workspace(q, k, tab, &bytes))) return c.todo();
    const at::Tensor& tq = c.tensor(0);
    const at::Tensor y = c.or_empty(8, tq.sizes(), tq.scalar_type());
    cbx_tensor* dy = c.describe(y);
    const Scratch ws = scratch(c, 9, bytes);
    if (!c.done(unlocked([&] {
            return ks || vs ? cbx_paged_attention_q8(q, k, ks, v, vs, tab, len, scale, cap, window, dy, ws.p, ws.bytes, c.stream)
                            : cbx_paged_attention(q, k, v, tab, len, scale, cap, window, dy, ws.p, ws.bytes, c.stream);
        }))) {
        return c.todo();
    }
    return wrap(y);
}

// q, k_cache, v_cache, block_tables, seq_lens, tok_start, scale, softcap, window, out, ws, k_scale, v_scale
PyObject* paged_prompt_attention(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 13);
    cbx_tensor *q = c.describe(0), *k = c.describe(1), *v = c.describe(2), *tab = c.describe(3), *len = c.describe(4),
               *start = c.describe(5), *ks = c.maybe(11), *vs = c.maybe(12);
    const float scale = c.number(6), cap = c.number(7);
    const int32_t window = c.int32(8);
    if (c.elsewhere()) return c.todo();
    size_t bytes = 0;
    if (c.none(10) && !c.done(cbx_paged_prompt_attention_workspace(q, k, tab, &bytes))) return c.todo();
    const at::Tensor& tq = c.tensor(0);
    const at::Tensor y = c.or_empty(9, tq.sizes(), tq.scalar_type());
    cbx_tensor* dy = c.describe(y);
    const Scratch ws = scratch(c, 10, bytes);
    if (!c.done(unlocked([&] {
            return cbx_paged_prompt_attention(q, k, ks, v, vs, tab, len, start, scale, cap, window, dy, ws.p, ws.bytes, c.stream);
        }))) {
        return c.todo();
    }
    return wrap(y);
}

// q, k_cache, v_cache, block_tables, seq_lens, group_start, shared_lens, scale, softcap, window, out, ws, k_scale, v_scale
PyObject* paged_shared_attention(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 14);
    cbx_tensor *q = c.describe(0), *k = c.describe(1), *v = c.describe(2), *tab = c.describe(3), *len = c.describe(4),
               *start = c.describe(5), *pre = c.describe(6), *ks = c.maybe(12), *vs = c.maybe(13);
    const float scale = c.number(7), cap = c.number(8);
    const int32_t window = c.int32(9);
    if (c.elsewhere()) return c.todo();
    size_t bytes = 0;
    if (c.none(11) && !c.done(cbx_paged_shared_attention_workspace(q, k, tab, start, &bytes))) return c.todo();
    const at::Tensor& tq = c.tensor(0);
    const at::Tensor y = c.or_empty(10, tq.sizes(), tq.scalar_type());
    cbx_tensor* dy = c.describe(y);
    const Scratch ws = scratch(c, 11, bytes);
    if (!c.done(unlocked([&] {
            return cbx_paged_shared_attention(q, k, ks, v, vs, tab, len, start, pre, scale, cap, window, dy, ws.p, ws.bytes, c.stream);
        }))) {
        return c.todo();
    }
    return wrap(y);
}

// logits, ids, top_n, scale, entropy, ws
PyObject* token_log_probs(PyObject* const* a, Py_ssize_t n) {
    Call c(a, n, 6);
    cbx_tensor *x = c.describe(0), *ids = c.maybe(1);
    const int32_t top = c.int32(2);
    const float scale = c.number(3);
    const int entropy = PyObject_IsTrue(a[4]);
    if (entropy < 0) throw Raised{};
    if (top < 0) raise(CBX_ERR_INVALID_ARG, "cbx_token_log_probs: n_top must be >= 0");
    if (c.elsewhere()) return c.todo();
    size_t bytes = 0;
    if (c.none(5) && !c.done(cbx_token_log_probs_workspace(x, top, &bytes))) return c.todo();
    const int64_t rows = x->ne[1];
    const at::Tensor ti = c.empty({rows, top}, at::kInt);
    const std::vector<at::Tensor> out = c.parts(at::kFloat, {{rows, top}, {ids ? rows : 0}, {entropy ? rows : 0}});
    const at::Tensor &tl = out[0], logp = ids ? out[1] : at::Tensor(), ent = entropy ? out[2] : at::Tensor();
    cbx_tensor *dl = ids ? c.describe(logp) : nullptr, *de = entropy ? c.describe(ent) : nullptr;
    cbx_tensor *di = top ? c.describe(ti) : nullptr, *dt = top ? c.describe(tl) : nullptr;
    const Scratch ws = scratch(c, 5, bytes);
    if (!c.done(unlocked([&] { return cbx_token_log_probs(x, ids, scale, dl, de, di, dt, ws.p, ws.bytes, c.stream); }))) return c.todo();
    return tuple_of({logp, ent, ti, tl});
}

// No C++ exception leaves: torch's become its Python ones.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        return F(a, n);
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyObject* setup(PyObject*, PyObject* cls) {
    Py_INCREF(cls);
    Py_XSETREF(g_error, cls);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)> PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<F>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    {"setup", setup, METH_O, nullptr},
    method<paged_append>("paged_append"),
    method<paged_release>("paged_release"),
    method<paged_store>("paged_store"),
    method<paged_load>("paged_load"),
    method<qk_norm_rope>("qk_norm_rope"),
    method<qk_norm_rope_store>("qk_norm_rope_store"),
    method<paged_attention>("paged_attention"),
    method<paged_prompt_attention>("paged_prompt_attention"),
    method<paged_shared_attention>("paged_shared_attention"),
    method<token_log_probs>("token_log_probs"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_cbxtorch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cbxtorch() { return PyModule_Create(&g_module); }
