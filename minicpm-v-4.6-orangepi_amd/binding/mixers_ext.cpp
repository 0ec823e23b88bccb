// mixers_ext.cpp -- the token mixers' Python calls (mixers.py), from torch tensors to the C-ABI.
//
// One decoded token's mixers run 3 to 5 us each on the GPU, so the host's part of a call
// is what counts: the same checks written in Python with a ctypes call of thirty
// arguments took 7 to 9 us, these take under one beside the launch.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <exception>
#include <initializer_list>
#include <string>

#include "mcv_mixers.h"

namespace {

PyObject *g_error, *g_empty_on;                  // McvError, and mixers.py's tensor of another stream
// A function of mixers.py or the package that makes workspaces, the dict of those it keeps, by device, stream and size.
struct Workspaces {
    PyObject *make, *held;
} g_gemm, g_delta;
int64_t g_gemm_sizes[2], g_delta_sizes[2];

struct Failed {};                                // a Python error is set

[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    PyErr_SetString(g_error, text);
    throw Failed{};
}

// The error of a C-ABI call, with its status.
void check(int rc, const char* who) {
    if (rc == MCV_OK) return;
    PyObject* e = PyObject_CallFunction(g_error, "N", PyUnicode_FromFormat("%s failed (status %d): %s", who, rc, mcv_last_error()));
    PyObject* status = e ? PyLong_FromLong(rc) : nullptr;
    if (status && PyObject_SetAttrString(e, "status", status) == 0) PyErr_SetObject(g_error, e);
    Py_XDECREF(status);
    Py_XDECREF(e);
    throw Failed{};
}

const at::Tensor& tensor(const char* who, const char* name, PyObject* o) {
    if (!THPVariable_Check(o)) refuse("%s: %s must be a tensor", who, name);
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(const char* who, const char* name, PyObject* o) {
    return o == Py_None ? nullptr : &tensor(who, name, o);
}

std::string shape(const at::Tensor& t) {
    std::string s = "[";
    for (int64_t n : t.sizes()) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
    return s + "]";
}
bool is_shape(const at::Tensor& t, std::initializer_list<int64_t> want) {
    return t.sizes() == at::IntArrayRef(want.begin(), want.size());
}
double number(PyObject* o, double otherwise) {
    if (o == Py_None) return otherwise;
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Failed{};
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Failed{};
    return v != 0;
}

// The stride of a dimension, none where it has one entry: torch leaves any there.
int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// fp16 [rows][heads][D]: pointer, row stride, head stride.
struct Heads {
    void* p;
    int64_t row, head;
};
Heads heads(const char* who, const char* name, const at::Tensor& t, int64_t rows) {
    if (t.scalar_type() != at::kHalf || t.dim() != 3 || t.stride(2) != 1 || t.size(0) != rows)
        refuse("%s: %s must be fp16 [%lld, heads, D] with contiguous heads, got %s %s", who, name, (long long)rows,
               c10::toString(t.scalar_type()), shape(t).c_str());
    return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1)};
}
// fp16 [pages][page_size][Hkv][D] of `like`'s shape.
struct Cache {
    void* p;
    int64_t page, token, head;
};
Cache cache(const char* who, const char* name, const at::Tensor& t, const at::Tensor& like, int64_t Hkv, int64_t D) {
    if (t.scalar_type() != at::kHalf || t.dim() != 4 || t.sizes() != like.sizes() || t.size(2) != Hkv || t.size(3) != D || t.stride(3) != 1)
        refuse("%s: %s must be fp16 [pages, page_size, %lld, %lld] with contiguous heads, both caches of one shape, got %s %s", who,
               name, (long long)Hkv, (long long)D, c10::toString(t.scalar_type()), shape(t).c_str());
    return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)};
}
void same_device(const char* who, const at::Tensor& t, std::initializer_list<const at::Tensor*> others) {
    for (const at::Tensor* o : others)
        if (o && o->device() != t.device()) refuse("%s: tensors on %s and %s", who, t.device().str().c_str(), o->device().str().c_str());
}
// Kernels read what they are given as device memory.  Asked last, when all tensors are known to be on t's device;
// the device is then the current one until the call ends, its stream and its memory among them.
c10::DeviceGuard on_gpu(const char* who, const at::Tensor& t) {
    if (!t.is_cuda()) refuse("%s: tensors must be on a GPU, got %s", who, t.device().str().c_str());
    return c10::DeviceGuard(t.device());
}
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
PyObject* wrapped(const at::Tensor& t) { return THPVariable_Wrap(t); }

// The handle of `stream` (a torch stream, or None: the current one).
mcv_stream_t handle(PyObject* stream) {
    if (stream == Py_None) return static_cast<mcv_stream_t>(c10::hip::getCurrentHIPStream().stream());
    PyObject* h = PyObject_GetAttrString(stream, "cuda_stream");
    if (!h) throw Failed{};
    void* p = PyLong_AsVoidPtr(h);
    Py_DECREF(h);
    if (!p && PyErr_Occurred()) throw Failed{};
    return static_cast<mcv_stream_t>(p);
}

// An output of a call on `stream`, whose handle is h.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like, PyObject* stream, mcv_stream_t h) {
    if (h == handle(Py_None)) return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
    PyObject* shape = PyTuple_New(static_cast<Py_ssize_t>(sizes.size()));
    if (!shape) throw Failed{};
    for (size_t i = 0; i < sizes.size(); ++i) PyTuple_SET_ITEM(shape, i, PyLong_FromLongLong(sizes[i]));
    PyObject* made = PyObject_CallFunction(g_empty_on, "NisO", shape, int(type == at::kFloat), like.device().str().c_str(), stream);
    if (!made) throw Failed{};
    const at::Tensor t = THPVariable_Unpack(made);
    Py_DECREF(made);
    return t;
}

// A buffer of `size` bytes.  Held ones are looked up here, a reference of that dict is all it takes.
void* workspace(const Workspaces& from, int64_t size, const at::Tensor& t, PyObject* stream, mcv_stream_t h) {
    PyObject* key = Py_BuildValue("(iNL)", int(t.device().index()), PyLong_FromVoidPtr(h), (long long)size);
    if (!key) throw Failed{};
    PyObject* ws = PyDict_GetItemWithError(from.held, key);
    Py_DECREF(key);
    if (ws) return THPVariable_Unpack(ws).data_ptr();
    if (PyErr_Occurred()) throw Failed{};
    PyObject* device = PyUnicode_FromString(t.device().str().c_str());
    PyObject* made = device ? PyObject_CallFunction(from.make, "LOO", (long long)size, device, stream) : nullptr;
    Py_XDECREF(device);
    if (!made) throw Failed{};
    void* p = THPVariable_Unpack(made).data_ptr();
    Py_DECREF(made);                             // (it is kept where it was made)
    return p;
}
// One of two sizes: few buffers, whatever the calls'.
int64_t of(const int64_t (&sizes)[2], int64_t bytes) { return bytes <= sizes[0] ? sizes[0] : bytes <= sizes[1] ? sizes[1] : bytes; }
// gemm_workspace's buffer, or one that is enough for any call of this kind.  Other calls on the stream use it too, so
// its first bytes are counters and stay zero.
void* gemm_workspace(int64_t bytes, const at::Tensor& t, PyObject* stream, mcv_stream_t h) {
    return workspace(g_gemm, of(g_gemm_sizes, bytes), t, stream, h);
}
void* delta_workspace(int64_t bytes, const at::Tensor& t, PyObject* stream, mcv_stream_t h) {
    return workspace(g_delta, of(g_delta_sizes, bytes), t, stream, h);
}

// (who, q, k, v, g, beta, state, cu, step, scale, normalize, state_index, out, state_out, stream) -> (out, state_out)
PyObject* delta(PyObject* const* a) {
    const char* who = PyUnicode_AsUTF8(a[0]);
    const at::Tensor &q = tensor(who, "q", a[1]), &k = tensor(who, "k", a[2]), &v = tensor(who, "v", a[3]);
    const at::Tensor &g = tensor(who, "g", a[4]), &beta = tensor(who, "beta", a[5]);
    const at::Tensor *state = maybe(who, "state", a[6]), *cu = maybe(who, "cu_seqlens", a[7]);
    const bool step = truth(a[8]);
    const at::Tensor* index = maybe(who, "state_index", a[11]);
    const at::Tensor* given = maybe(who, "out", a[12]);
    const at::Tensor* state_given = maybe(who, "state_out", a[13]);
    if (q.dim() != 3 || v.dim() != 3) refuse("%s: q, k and v must be [T, heads, D]", who);
    const int64_t T = q.size(0), Hk = q.size(1), Dk = q.size(2), Hv = v.size(1), Dv = v.size(2);
    int64_t B = step ? T : 1;
    if (cu) {
        if (cu->scalar_type() != at::kInt || cu->dim() != 1 || cu->numel() < 2 || !cu->is_contiguous())
            refuse("%s: cu_seqlens must be contiguous int32 [B + 1]", who);
        B = cu->numel() - 1;
    }
    if (k.sizes() != q.sizes()) refuse("%s: q %s and k %s must have one shape", who, shape(q).c_str(), shape(k).c_str());
    const Heads qa = heads(who, "q", q, T), ka = heads(who, "k", k, T), va = heads(who, "v", v, T);
    for (const at::Tensor* t : {&g, &beta})
        if (t->scalar_type() != at::kFloat || !is_shape(*t, {T, Hv}) || (Hv > 1 && t->stride(1) != 1))
            refuse("%s: %s must be fp32 [%lld, %lld] with contiguous rows", who, t == &g ? "g" : "beta", (long long)T, (long long)Hv);
    int64_t n_states = B;
    at::Tensor out, state_out;
    if (index) {
        if (index->scalar_type() != at::kInt || !is_shape(*index, {B}) || !index->is_contiguous())
            refuse("%s: state_index must be contiguous int32 [%lld]", who, (long long)B);
        const at::Tensor* pool = state_given ? state_given : state;
        if (!pool) refuse("%s: state_index needs a state or state_out to index", who);
        if (pool->dim() > 0) n_states = pool->size(0);
        if (!state_given) state_given = state;   // a pool is updated in place
    }
    for (const at::Tensor* t : {state, state_given})
        if (t && (t->scalar_type() != at::kFloat || !is_shape(*t, {n_states, Hv, Dk, Dv}) || !t->is_contiguous()))
            refuse("%s: %s must be contiguous fp32 [%lld, %lld, %lld, %lld]", who, t == state ? "state" : "state_out", (long long)n_states,
                   (long long)Hv, (long long)Dk, (long long)Dv);
    if (given && (given->scalar_type() != at::kHalf || given->sizes() != v.sizes() || !given->is_contiguous()))
        refuse("%s: out must be contiguous fp16 %s", who, shape(v).c_str());
    same_device(who, q, {&k, &v, &g, &beta, state, state_given, index, cu, given});
    const auto device = on_gpu(who, q);
    const mcv_stream_t h = handle(a[14]);
    out = given ? *given : fresh(v.sizes(), at::kHalf, q, a[14], h);
    state_out = state_given ? *state_given : fresh({B, Hv, Dk, Dv}, at::kFloat, q, a[14], h);
    if (B == 0) {                                // nothing to launch, of shapes that a batch would be taken of
        if (Hk == 0 || Hv == 0 || Hv % Hk != 0 || (Dk != 64 && Dk != 128) || Dv == 0 || Dv % 16 != 0 || Dv > 256)
            refuse("%s: bad shape q %s, v %s", who, shape(q).c_str(), shape(v).c_str());
        return Py_BuildValue("(NN)", wrapped(out), wrapped(state_out));
    }
    const int64_t bytes = mcv_delta_rule_workspace_bytes(B, T, Hk, Hv, Dk, Dv);
    void* ws = bytes ? delta_workspace(bytes, q, a[14], h) : nullptr;
    check(mcv_delta_rule(qa.p, qa.row, qa.head, ka.p, ka.row, ka.head, va.p, va.row, va.head, g.data_ptr(), stride_of(g, 0), beta.data_ptr(),
                         stride_of(beta, 0), ptr(state), state_out.data_ptr(), ptr(index), n_states, ptr(cu), B, T, Hk, Hv, Dk, Dv,
                         number(a[9], 1.0 / std::sqrt(static_cast<double>(Dk))), truth(a[10]), out.data_ptr(),
                         ws, ws ? bytes : 0, h),
          who);
    return Py_BuildValue("(NN)", wrapped(out), wrapped(state_out));
}

// (q, k_cache, v_cache, block_table, seq_lens, scale, max_seq_len, out, stream) -> out
PyObject* paged(PyObject* const* a) {
    const char* who = "paged_attention_decode";
    const at::Tensor &q = tensor(who, "q", a[0]), &kc = tensor(who, "k_cache", a[1]), &vc = tensor(who, "v_cache", a[2]);
    const at::Tensor &table = tensor(who, "block_table", a[3]), &lens = tensor(who, "seq_lens", a[4]);
    const at::Tensor* given = maybe(who, "out", a[7]);
    if (q.dim() != 3 || kc.dim() != 4) refuse("%s: q must be [B, Hq, D] and the caches [pages, page_size, Hkv, D]", who);
    const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), pages = kc.size(0), page = kc.size(1), Hkv = kc.size(2);
    const Heads qa = heads(who, "q", q, B);
    const Cache ka = cache(who, "k_cache", kc, kc, Hkv, D), va = cache(who, "v_cache", vc, kc, Hkv, D);
    if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != B || (table.size(1) > 1 && table.stride(1) != 1))
        refuse("%s: block_table must be int32 [%lld, width] with contiguous rows", who, (long long)B);
    if (lens.scalar_type() != at::kInt || !is_shape(lens, {B}) || !lens.is_contiguous())
        refuse("%s: seq_lens must be contiguous int32 [%lld]", who, (long long)B);
    if (given && (given->scalar_type() != at::kHalf || given->sizes() != q.sizes() || !given->is_contiguous()))
        refuse("%s: out must be contiguous fp16 %s", who, shape(q).c_str());
    same_device(who, q, {&kc, &vc, &table, &lens, given});
    int64_t most = table.size(1) * page;
    if (a[6] != Py_None) {
        most = PyLong_AsLongLong(a[6]);
        if (most == -1 && PyErr_Occurred()) throw Failed{};
    }
    const auto device = on_gpu(who, q);
    const mcv_stream_t h = handle(a[8]);
    const at::Tensor out = given ? *given : fresh(q.sizes(), at::kHalf, q, a[8], h);
    if (B == 0) {
        if (Hq == 0 || Hkv == 0 || Hq % Hkv != 0 || (D != 64 && D != 128 && D != 256) || page == 0 || page % 16 != 0)
            refuse("%s: bad shape q %s, caches %s", who, shape(q).c_str(), shape(kc).c_str());
        return wrapped(out);
    }
    const int64_t bytes = mcv_paged_attention_workspace_bytes(B, Hq, Hkv, D, most);
    void* ws = bytes ? gemm_workspace(bytes, q, a[8], h) : nullptr;
    check(mcv_paged_attention(qa.p, qa.row, qa.head, ka.p, ka.page, ka.token, ka.head, va.p, va.page, va.token, va.head, pages, page,
                              table.data_ptr(), stride_of(table, 0), table.size(1), lens.data_ptr(), most, B, Hq, Hkv, D,
                              number(a[5], 1.0 / std::sqrt(static_cast<double>(D))), out.data_ptr(), ws, ws ? bytes : 0, h),
          who);
    return wrapped(out);
}

// (q, k, positions, freq, axis, q_out, k_out, stream) -> (q_out, k_out), or
// (q, k, positions, freq, axis, q_out, v, k_cache, v_cache, slots, stream) -> q_out
PyObject* rotary(PyObject* const* a, bool cached) {
    const char* who = cached ? "rotary_axes_cached" : "rotary_axes";
    const at::Tensor &q = tensor(who, "q", a[0]), &k = tensor(who, "k", a[1]), &pos = tensor(who, "positions", a[2]);
    const at::Tensor &freq = tensor(who, "freq", a[3]), &axis = tensor(who, "axis", a[4]);
    const at::Tensor* given = maybe(who, "q_out", a[5]);
    if (q.dim() != 3 || k.dim() != 3 || k.size(0) != q.size(0) || k.size(2) != q.size(2))
        refuse("%s: q and k must be [T, heads, D], got %s and %s", who, shape(q).c_str(), shape(k).c_str());
    const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = k.size(1), half = freq.numel();
    if (pos.scalar_type() != at::kLong || pos.dim() != 2 || pos.size(1) != T) refuse("%s: positions must be int64 [axes, %lld]", who, (long long)T);
    if (freq.scalar_type() != at::kDouble || !freq.is_contiguous() || axis.scalar_type() != at::kInt || axis.numel() != half || !axis.is_contiguous())
        refuse("%s: freq must be contiguous fp64 [rot / 2] and axis contiguous int32 of its length", who);
    if (given && given->sizes() != q.sizes()) refuse("%s: q_out must be %s", who, shape(q).c_str());
    same_device(who, q, {&k, &pos, &freq, &axis, given});
    const Heads qa = heads(who, "q", q, T), ka = heads(who, "k", k, T);
    if (!cached) {
        const at::Tensor* k_given = maybe(who, "k_out", a[6]);
        if (k_given && k_given->sizes() != k.sizes()) refuse("%s: k_out must be %s", who, shape(k).c_str());
        same_device(who, q, {k_given});
        for (const at::Tensor* t : {given, k_given})
            if (t) heads(who, t == given ? "q_out" : "k_out", *t, T);
        const auto device = on_gpu(who, q);
        const mcv_stream_t h = handle(a[7]);
        const at::Tensor q_out = given ? *given : fresh(q.sizes(), at::kHalf, q, a[7], h);
        const at::Tensor k_out = k_given ? *k_given : fresh(k.sizes(), at::kHalf, q, a[7], h);
        const Heads qo = heads(who, "q_out", q_out, T), ko = heads(who, "k_out", k_out, T);
        if (T)
            check(mcv_rotary_axes(qa.p, qa.row, qa.head, ka.p, ka.row, ka.head, pos.data_ptr(), stride_of(pos, 0), stride_of(pos, 1), pos.size(0),
                                  freq.data_ptr(), axis.data_ptr(), T, Hq, Hkv, D, 2 * half, qo.p, qo.row, qo.head, ko.p, ko.row, ko.head,
                                  h),
                  who);
        return Py_BuildValue("(NN)", wrapped(q_out), wrapped(k_out));
    }
    const at::Tensor &v = tensor(who, "v", a[6]), &kc = tensor(who, "k_cache", a[7]), &vc = tensor(who, "v_cache", a[8]);
    const at::Tensor& slots = tensor(who, "slots", a[9]);
    if (kc.dim() != 4 || v.sizes() != k.sizes())
        refuse("%s: v must be %s and the caches [pages, page_size, %lld, %lld]", who, shape(k).c_str(), (long long)Hkv, (long long)D);
    if (slots.scalar_type() != at::kLong || !is_shape(slots, {T}) || !slots.is_contiguous())
        refuse("%s: slots must be contiguous int64 [%lld]", who, (long long)T);
    const Cache kca = cache(who, "k_cache", kc, kc, Hkv, D), vca = cache(who, "v_cache", vc, kc, Hkv, D);
    same_device(who, q, {&v, &kc, &vc, &slots});
    const Heads va = heads(who, "v", v, T);
    if (given) heads(who, "q_out", *given, T);
    const auto device = on_gpu(who, q);
    const mcv_stream_t h = handle(a[10]);
    const at::Tensor q_out = given ? *given : fresh(q.sizes(), at::kHalf, q, a[10], h);
    const Heads qo = heads(who, "q_out", q_out, T);
    if (T)
        check(mcv_rotary_axes_cached(qa.p, qa.row, qa.head, ka.p, ka.row, ka.head, va.p, va.row, va.head, pos.data_ptr(), stride_of(pos, 0),
                                     stride_of(pos, 1), pos.size(0), freq.data_ptr(), axis.data_ptr(), T, Hq, Hkv, D, 2 * half, qo.p, qo.row,
                                     qo.head, kca.p, kca.page, kca.token, kca.head, vca.p, vca.page, vca.token, vca.head, kc.size(0),
                                     kc.size(1), slots.data_ptr(), h),
              who);
    return wrapped(q_out);
}

// C++ exceptions end here.
template <class F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
    if (got != want) return PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", got, want);
    try {
        return f();
    } catch (const Failed&) {
    } catch (const std::exception& e) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject* py_delta(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 15, [&] { return delta(a); }); }
PyObject* py_paged(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 9, [&] { return paged(a); }); }
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 8, [&] { return rotary(a, false); }); }
PyObject* py_rotary_cached(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 11, [&] { return rotary(a, true); }); }

// (McvError, _empty_on, gemm_workspace, the buffers it keeps, two sizes of them, delta_workspace, its, two of them)
PyObject* py_bind(PyObject*, PyObject* args) {
    PyObject *error, *empty_on;
    Workspaces gemm, delta;
    long long sizes[4];
    if (!PyArg_ParseTuple(args, "OOOO!LLOO!LL", &error, &empty_on, &gemm.make, &PyDict_Type, &gemm.held, &sizes[0], &sizes[1], &delta.make, &PyDict_Type,
                          &delta.held, &sizes[2], &sizes[3]))
        return nullptr;
    for (PyObject* o : {error, empty_on, gemm.make, gemm.held, delta.make, delta.held}) Py_INCREF(o);
    g_error = error;
    g_empty_on = empty_on;
    g_gemm = gemm;
    g_delta = delta;
    for (int i = 0; i < 2; ++i) {
        g_gemm_sizes[i] = sizes[i];
        g_delta_sizes[i] = sizes[2 + i];
    }
    Py_RETURN_NONE;
}

template <class F>
PyCFunction method(F* f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {{"bind", py_bind, METH_VARARGS, nullptr},
                         {"delta", method(py_delta), METH_FASTCALL, nullptr},
                         {"paged", method(py_paged), METH_FASTCALL, nullptr},
                         {"rotary", method(py_rotary), METH_FASTCALL, nullptr},
                         {"rotary_cached", method(py_rotary_cached), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mcv_mixers", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mcv_mixers() { return PyModule_Create(&module); }
