// The short way from tensors to the quantised K/V history's entry points: otter_amd/ops.py asks here first.
//
// A call whose kernel takes 3 to 12 us spends as long again in the interpreter when its operands' shapes, strides and addresses are
// read one attribute at a time.  These functions read them from the tensors themselves, allocate the results and launch.  They
// take the calls that are as they should be and return None for every other one -- wrong shapes and types, subclasses, another device
// than the current one, a refusal of the entry point -- without having done anything: ops.py then takes its own way, which names the fault.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <algorithm>
#include <array>
#include <cmath>

#include "otter_hip.h"

namespace {

struct Entries {
    decltype(&otter_kv_cache_write) write;
    decltype(&otter_kv_cache_read) read;
    decltype(&otter_attn_cache) attend;
    decltype(&otter_attn_cache_workspace_floats) workspace;
    PyObject* stream;                              // torch's (device) -> raw handle of its current stream
} entries;

// the tensor behind an object, null if it is not exactly a torch.Tensor
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? OTTER_DT_F32 : t == at::kBFloat16 ? OTTER_DT_BF16 : t == at::kHalf ? OTTER_DT_F16 : -1;
}
at::ScalarType dtype_of(long code) { return code == OTTER_DT_F32 ? at::kFloat : code == OTTER_DT_BF16 ? at::kBFloat16 : at::kHalf; }

bool whole(PyObject* o, long least, long most, long& v) {
    if (!PyLong_Check(o)) return false;
    int over = 0;
    v = PyLong_AsLongAndOverflow(o, &over);
    return !over && v >= least && v <= most;
}

struct Call {
    otter_kv_cache cache{};
    otter_kv_rows rows{};
    c10::Device device{c10::kCPU};
    long heads = 0, episodes = 0, capacity = 0;
    void* stream = nullptr;

    bool take_cache(PyObject* pc, PyObject* ps, long head_dim) {
        const at::Tensor *c = tensor(pc), *s = tensor(ps);
        if (!c || !s || c->scalar_type() != at::kByte || s->scalar_type() != at::kByte || c->dim() != 5 || s->dim() != 5 || !c->is_cuda()) return false;
        device = c->device();
        if (s->device() != device || (head_dim != 32 && head_dim != 64 && head_dim != 96 && head_dim != 128)) return false;
        const auto z = c->sizes(), zs = s->sizes(), st = c->strides(), ss = s->strides();
        const long row = z[4];
        const int bits = row * 2 == head_dim ? 4 : row == head_dim ? 8 : 0;
        constexpr long most = (1L << 31) - 1;
        if (!bits || z[0] != 2 || zs[0] != 2 || zs[1] != z[1] || zs[2] != z[2] || zs[3] != z[3] || zs[4] != 4) return false;
        if (z[1] > most || z[2] < 1 || z[2] > most || z[3] < 1 || z[3] > most) return false;
        if ((z[3] > 1 && (st[3] != row || ss[3] != 4)) || st[4] != 1 || ss[4] != 1) return false;
        episodes = z[1]; heads = z[2]; capacity = z[3];
        cache.codes = (unsigned char*)c->data_ptr();
        cache.scales = (unsigned char*)s->data_ptr();
        cache.code_kv = st[0];
        cache.scale_kv = ss[0];
        cache.code_episode = episodes > 1 ? st[1] : 0;
        cache.scale_episode = episodes > 1 ? ss[1] : 0;
        cache.code_head = heads > 1 ? st[2] : 0;
        cache.scale_head = heads > 1 ? ss[2] : 0;
        cache.bits = bits;
        cache.episodes = (int)episodes;
        cache.heads = (int)heads;
        cache.capacity = (int)capacity;
        cache.head_dim = (int)head_dim;
        return true;
    }
    bool take_index(PyObject* o, long length, const int*& p) {
        p = nullptr;
        if (o == Py_None) return true;
        const at::Tensor* t = tensor(o);
        if (!t || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != length || t->device() != device || !t->is_contiguous()) return false;
        p = (const int*)t->data_ptr();
        return true;
    }
    bool take_rows(long n, long steps, PyObject* pos, PyObject* idx, PyObject* count) {
        if (n < 1 || n >= (1L << 31) || steps < 1 || steps > (1L << 30) || (idx == Py_None && n > episodes)) return false;
        rows.n_rows = (int)n;
        rows.steps = (int)steps;
        return take_index(idx, n, rows.idx) && take_index(pos, episodes, rows.pos) && take_index(count, n, rows.count);
    }
    // (row, step, head, dim), or without steps
    bool take_operand(const at::Tensor* t, at::ScalarType type, at::IntArrayRef shape, otter_kv_operand& o) const {
        if (!t || t->scalar_type() != type || t->sizes() != shape || t->device() != device) return false;
        const auto st = t->strides();
        const size_t last = shape.size() - 1;
        if (st[last] != 1) return false;
        o = {t->data_ptr(), shape[0] > 1 ? st[0] : 0, last == 3 && shape[1] > 1 ? st[1] : 0, shape[last - 1] > 1 ? st[last - 1] : 0};
        return true;
    }
    // the current device's current stream; false if the cache is on another one
    bool on_current_device() {
        const c10::impl::VirtualGuardImpl guard(device.type());
        if (guard.getDevice() != device) return false;
        PyObject* index = PyLong_FromLong(device.index());
        PyObject* raw = index ? PyObject_CallOneArg(entries.stream, index) : nullptr;
        Py_XDECREF(index);
        if (!raw) return false;
        stream = PyLong_AsVoidPtr(raw);
        Py_DECREF(raw);
        return !PyErr_Occurred();
    }
    at::Tensor make(at::IntArrayRef shape, at::ScalarType type) const { return at::empty(shape, at::TensorOptions().dtype(type).device(device)); }
};

PyObject* not_taken() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

// (an exception -- a tensor without strides or storage, no memory -- ends here too: ops.py asks again and raises torch's own error)
typedef PyObject* Function(PyObject* const* a, Py_ssize_t na);
template <Function* F> PyObject* guarded(PyObject*, PyObject* const* a, Py_ssize_t na) {
    try {
        return F(a, na);
    } catch (...) {
        return not_taken();
    }
}
template <Function* F> constexpr PyMethodDef method(const char* name) { return {name, (PyCFunction)(void (*)(void))guarded<F>, METH_FASTCALL, nullptr}; }

// write(k, v, codes, scales, pos, idx, count) -> True
PyObject* kv_write(PyObject* const* a, Py_ssize_t na) {
    Call c;
    const at::Tensor *k = na == 7 ? tensor(a[0]) : nullptr, *v = k ? tensor(a[1]) : nullptr;
    if (!v || k->dim() != 4) return not_taken();
    const auto z = k->sizes();
    const int dt = dtype_code(k->scalar_type());
    otter_kv_operand ko, vo;
    if (dt < 0 || !c.take_cache(a[2], a[3], z[3]) || z[2] != c.heads || !c.take_rows(z[0], z[1], a[4], a[5], a[6]) ||
        !c.take_operand(k, k->scalar_type(), z, ko) || !c.take_operand(v, k->scalar_type(), z, vo) || !c.on_current_device())
        return not_taken();
    if (entries.write(&c.cache, &c.rows, dt, &ko, &vo, c.stream) != 0) return not_taken();
    Py_RETURN_TRUE;
}

// read(codes, scales, head_dim, steps, pos, idx, count, n_rows, dtype) -> (k, v); n_rows counts without idx, None: every episode
PyObject* kv_read(PyObject* const* a, Py_ssize_t na) {
    Call c;
    long d, steps, n, dt;
    if (na != 9 || !whole(a[2], 1, 128, d) || !whole(a[3], 1, 1L << 30, steps) || !whole(a[8], 0, 2, dt) || !c.take_cache(a[0], a[1], d)) return not_taken();
    if (const at::Tensor* idx = tensor(a[5])) n = idx->dim() == 1 ? idx->size(0) : 0;
    else if (a[7] == Py_None) n = c.episodes;
    else if (!whole(a[7], 1, (1L << 31) - 1, n)) return not_taken();
    if (!c.take_rows(n, steps, a[4], a[5], a[6]) || !c.on_current_device()) return not_taken();
    const std::array<int64_t, 4> shape = {n, steps, c.heads, d};
    at::Tensor k = c.make(shape, dtype_of(dt)), v = c.make(shape, dtype_of(dt));
    const long step = c.heads * d;
    const otter_kv_operand ko = {k.data_ptr(), steps * step, step, d}, vo = {v.data_ptr(), steps * step, step, d};
    if (entries.read(&c.cache, &c.rows, (int)dt, &ko, &vo, c.stream) != 0) return not_taken();
    PyObject* pk = THPVariable_Wrap(std::move(k));
    PyObject* pv = pk ? THPVariable_Wrap(std::move(v)) : nullptr;
    PyObject* both = pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return both;
}

// attend(q, k, v, codes, scales, pos, idx, count, causal, window, scale, max_len) -> out; k, v: both None or the step's own rows
PyObject* kv_attend(PyObject* const* a, Py_ssize_t na) {
    Call c;
    const at::Tensor* q = na == 12 ? tensor(a[0]) : nullptr;
    if (!q || q->dim() != (a[1] == Py_None ? 4 : 3)) return not_taken();
    const auto z = q->sizes();
    const long n = z[0], steps = z.size() == 4 ? z[1] : 1, hq = z[z.size() - 2], d = z[z.size() - 1];
    const at::ScalarType type = q->scalar_type();
    const int dt = dtype_code(type);
    long window, max_len;
    otter_kv_operand qo, ko, vo;
    const bool append = a[1] != Py_None;
    if (dt < 0 || !c.take_cache(a[3], a[4], d) || hq < 1 || hq >= (1L << 31) || hq % c.heads != 0 || !c.take_rows(n, steps, a[5], a[6], a[7]) ||
        !c.take_operand(q, type, z, qo) || c.episodes < 1 || !whole(a[9], 0, (1L << 31) - 1, window))
        return not_taken();
    max_len = c.capacity;
    if (a[11] != Py_None && !whole(a[11], 1, (1L << 31) - 1, max_len)) return not_taken();
    max_len = std::min(max_len, c.capacity);
    window = std::min(window, 1L << 30);
    if (append) {
        const std::array<int64_t, 3> shape = {n, c.heads, d};
        if (!c.take_operand(tensor(a[1]), type, shape, ko) || !c.take_operand(tensor(a[2]), type, shape, vo)) return not_taken();
    }
    double scale = a[10] == Py_None ? std::pow((double)d, -0.5) : PyFloat_AsDouble(a[10]);
    const int causal = PyObject_IsTrue(a[8]);
    if (PyErr_Occurred() || causal < 0 || !(scale > 0.0 && scale < 1.0e38) || !c.on_current_device()) return not_taken();
    at::Tensor out = c.make(z, type), ws;
    const long need = entries.workspace(dt, (int)n, (int)steps, (int)hq, (int)c.heads, (int)d, (int)window, (int)max_len);
    if (need) ws = c.make({need}, at::kFloat);                      // the call's own, from the allocator of the stream it runs on
    const otter_kv_operand oo = {out.data_ptr(), steps * hq * d, hq * d, d};
    if (entries.attend(&c.cache, &c.rows, dt, &qo, (int)hq, append ? &ko : nullptr, append ? &vo : nullptr, &oo, causal, (int)window, (int)max_len,
                       (float)scale, need ? (float*)ws.data_ptr() : nullptr, need, c.stream) != 0)
        return not_taken();
    return THPVariable_Wrap(std::move(out));
}

// bind(write, read, attend, workspace, stream): addresses of the library's entry points and torch's look-up of the current stream
PyObject* bind(PyObject* const* a, Py_ssize_t na) {
    if (na != 5) {
        PyErr_SetString(PyExc_TypeError, "bind takes four addresses and a function");
        return nullptr;
    }
    void* p[4];
    for (int i = 0; i < 4; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_INCREF(a[4]);
    Py_XDECREF(entries.stream);
    entries = {(decltype(entries.write))p[0], (decltype(entries.read))p[1], (decltype(entries.attend))p[2], (decltype(entries.workspace))p[3], a[4]};
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {method<bind>("bind"), method<kv_write>("write"), method<kv_read>("read"), method<kv_attend>("attend"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (the structs' layouts and the entry points' signatures are compiled in: _lib.py compares their version before it binds)
PyMODINIT_FUNC PyInit__kv_binding(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddIntConstant(m, "ABI_VERSION", OTTER_HIP_ABI_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
