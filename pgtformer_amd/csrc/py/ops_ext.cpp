// Launches of the cached-attention operators without the interpreter between the arguments and the launch: what ops.py checks, allocates and passes on
// in some 8 us of Python (of 11 to 12 for a call of a few tokens) takes 2 here.  A serving step is made of such calls.
//
// Every function takes the current device and its stream, then the operator's arguments, and returns the operator's result - or None, with nothing
// launched, for ANY call that is not plainly right (another device or type, odd strides, a missing tensor, no memory ...): ops.py then goes its own
// way, which does the rest of the work or says what is wrong.  A status that the library returns comes back as an int.
#include <ATen/ops/empty.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <limits>

#include "pgt_hip.h"

namespace {

struct Entries {
    decltype(&pgt_qk_norm_rope) rope;
    decltype(&pgt_qk_norm_rope_backward) rope_bwd;
    decltype(&pgt_qk_norm_rope_backward_workspace_bytes) rope_bwd_bytes;
    decltype(&pgt_kv_append) append;
    decltype(&pgt_kv_read) read;
    decltype(&pgt_kv_attention) attention;
    decltype(&pgt_kv_attention_workspace_bytes) attention_bytes;
} go = {};

struct No {};      // not a call for here

long long integer(PyObject* o) {
    if (!PyLong_Check(o)) throw No();
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    if (over) throw No();
    return v;
}
int32_t int32(long long v) {
    if (v < std::numeric_limits<int32_t>::min() || v > std::numeric_limits<int32_t>::max()) throw No();
    return (int32_t)v;
}
int32_t int32(PyObject* o) { return int32(integer(o)); }
float real(PyObject* o) {
    if (PyFloat_Check(o)) return (float)PyFloat_AS_DOUBLE(o);
    return (float)integer(o);
}
struct Call {
    int dev;
    pgt_stream_t stream;
    Call(PyObject* const* a) : dev((int)int32(a[0])), stream((pgt_stream_t)(uintptr_t)integer(a[1])) {}
    const at::Tensor& tensor(PyObject* o) const {
        if (!THPVariable_Check(o)) throw No();
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.get_device() != dev || t.layout() != at::kStrided) throw No();
        return t;
    }
    // (n) contiguous of one type; None: null if `or_none`
    template <typename T> T* vec(PyObject* o, at::ScalarType type, int64_t n, bool or_none = false) const {
        if (or_none && o == Py_None) return nullptr;
        const at::Tensor& t = tensor(o);
        if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) throw No();
        return (T*)t.data_ptr();
    }
    // (rows, cols), elements of a row adjacent, rows not overlapping; its row stride
    int32_t rows(const at::Tensor& t, int64_t rows, int64_t cols) const {
        if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || t.stride(1) != 1) throw No();
        if (rows <= 1) return int32(cols);
        if (t.stride(0) < cols) throw No();
        return int32(t.stride(0));
    }
};
int32_t dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PGT_F32;
        case at::kBFloat16: return PGT_BF16;
        case at::kHalf: return PGT_F16;
        default: throw No();
    }
}
PyObject* result(int rc, std::initializer_list<at::Tensor> ts) {
    if (rc) return PyLong_FromLong(rc);
    if (ts.size() == 1) return THPVariable_Wrap(*ts.begin());
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
    return r;
}

// the norm + rotation's common arguments: q, k, positions, freqs, q_gain, k_gain, heads, kv_heads
struct Rope {
    const at::Tensor &q, &k;
    int32_t dtype, rows, heads, kv, hd, rot, ldq, ldk;
    const int32_t* pos;
    const double* freqs;
    const float *qg, *kg;
    Rope(const Call& c, PyObject* const* a) : q(c.tensor(a[0])), k(c.tensor(a[1])) {
        heads = int32(a[6]);
        kv = int32(a[7]);
        if (heads <= 0 || kv <= 0 || q.dim() != 2 || q.size(1) % heads || k.scalar_type() != q.scalar_type()) throw No();
        dtype = dtype_of(q);
        rows = int32(q.size(0));
        hd = int32(q.size(1) / heads);
        ldq = c.rows(q, rows, q.size(1));
        ldk = c.rows(k, rows, (int64_t)kv * hd);
        rot = 0;
        pos = nullptr;
        freqs = nullptr;
        if (a[3] != Py_None) {
            const at::Tensor& f = c.tensor(a[3]);
            rot = int32(2 * f.numel());
            if (f.scalar_type() != at::kDouble || !f.is_contiguous()) throw No();
            if (rot) {
                freqs = (const double*)f.data_ptr();
                pos = c.vec<int32_t>(a[2], at::kInt, rows);
            }
        }
        qg = c.vec<float>(a[4], at::kFloat, hd, true);
        kg = c.vec<float>(a[5], at::kFloat, hd, true);
    }
    at::Tensor out_q() const { return at::empty({rows, (int64_t)heads * hd}, q.options().requires_grad(false)); }
    at::Tensor out_k() const { return at::empty({rows, (int64_t)kv * hd}, q.options().requires_grad(false)); }
};

// (dev, stream, q, k, positions, freqs, q_gain, k_gain, heads, kv_heads, eps, interleaved)
PyObject* qk_norm_rope(PyObject* const* a) {
    const Call c(a);
    const Rope r(c, a + 2);
    const float eps = real(a[10]);
    const int32_t inter = a[11] == Py_True;
    const at::Tensor qo = r.out_q(), ko = r.out_k();
    return result(go.rope(r.dtype, r.q.data_ptr(), r.ldq, r.k.data_ptr(), r.ldk, r.rows, r.heads, r.kv, r.hd, r.pos, r.freqs, r.rot, inter, r.qg, r.kg, eps,
                          qo.data_ptr(), r.heads * r.hd, ko.data_ptr(), r.kv * r.hd, c.stream), {qo, ko});
}
// (dev, stream, q, k, positions, freqs, q_gain, k_gain, heads, kv_heads, eps, interleaved, dq, dk)
PyObject* qk_norm_rope_backward(PyObject* const* a) {
    const Call c(a);
    const Rope r(c, a + 2);
    const float eps = real(a[10]);
    const int32_t inter = a[11] == Py_True;
    const at::Tensor &dq = c.tensor(a[12]), &dk = c.tensor(a[13]);
    if (dq.scalar_type() != r.q.scalar_type() || dk.scalar_type() != r.q.scalar_type()) throw No();
    const int32_t lddq = c.rows(dq, r.rows, (int64_t)r.heads * r.hd), lddk = c.rows(dk, r.rows, (int64_t)r.kv * r.hd);
    const at::Tensor qo = r.out_q(), ko = r.out_k();
    const auto f32 = r.q.options().dtype(at::kFloat).requires_grad(false);
    const at::Tensor gq = at::empty({r.hd}, f32), gk = at::empty({r.hd}, f32);
    const size_t bytes = go.rope_bwd_bytes(r.rows, r.hd);
    const at::Tensor ws = at::empty({(int64_t)(bytes / 4)}, f32);
    return result(go.rope_bwd(r.dtype, dq.data_ptr(), lddq, dk.data_ptr(), lddk, r.q.data_ptr(), r.ldq, r.k.data_ptr(), r.ldk, r.rows, r.heads, r.kv, r.hd,
                              r.pos, r.freqs, r.rot, inter, r.qg, r.kg, eps, qo.data_ptr(), r.heads * r.hd, ko.data_ptr(), r.kv * r.hd,
                              (float*)gq.data_ptr(), (float*)gk.data_ptr(), ws.data_ptr(), bytes, c.stream), {qo, ko, gq, gk});
}

// a cache, a table and the sequences: k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, hd, table, lens, cu
struct Kv {
    uint8_t *kp, *vp;
    float *ks, *vs;
    int32_t pages, page, kv, hd, B, width, ldt, most;
    const int32_t *table, *lens, *cu;
    Kv(const Call& c, PyObject* const* a, int64_t rows, PyObject* limit) {
        const at::Tensor &k = c.tensor(a[0]), &v = c.tensor(a[1]), &sk = c.tensor(a[2]), &sv = c.tensor(a[3]), &t = c.tensor(a[8]);
        kp = (uint8_t*)k.data_ptr(), vp = (uint8_t*)v.data_ptr();
        ks = (float*)sk.data_ptr(), vs = (float*)sv.data_ptr();
        pages = int32(a[4]), page = int32(a[5]), kv = int32(a[6]), hd = int32(a[7]);
        // (the cache checked its tensors against each other; these are the sizes that the kernels go by)
        if (k.scalar_type() != at::kByte || v.scalar_type() != at::kByte || sk.scalar_type() != at::kFloat || sv.scalar_type() != at::kFloat ||
            k.numel() != (int64_t)pages * page * kv * hd || v.numel() != k.numel() || sk.numel() != (int64_t)pages * kv || sv.numel() != sk.numel())
            throw No();
        if (t.scalar_type() != at::kInt || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) throw No();
        B = int32(t.size(0)), width = int32(t.size(1)), ldt = B > 1 ? int32(t.stride(0)) : width;
        table = (const int32_t*)t.data_ptr();
        lens = c.vec<int32_t>(a[9], at::kInt, B);
        cu = c.vec<int32_t>(a[10], at::kInt, (int64_t)B + 1, true);
        int64_t m = limit == Py_None ? -1 : integer(limit);
        if (limit != Py_None && m < 0) throw No();
        if (!cu) {
            if (B <= 0 || rows % B || (m >= 0 && m != rows / B)) throw No();
            m = rows / B;
        } else {
            if (m > rows) throw No();
            if (m < 0) m = rows;
        }
        most = int32(m);
    }
};

// (dev, stream, cache, table, lens, cu: see Kv, k, v, max_new)
PyObject* kv_append(PyObject* const* a) {
    const Call c(a);
    const at::Tensor &k = c.tensor(a[13]), &v = c.tensor(a[14]);
    if (k.dim() != 2 || k.scalar_type() != v.scalar_type()) throw No();
    const int32_t rows = int32(k.size(0));
    const Kv p(c, a + 2, rows, a[15]);
    const int32_t dtype = dtype_of(k), ldk = c.rows(k, rows, (int64_t)p.kv * p.hd), ldv = c.rows(v, rows, (int64_t)p.kv * p.hd);
    const int rc = go.append(dtype, k.data_ptr(), ldk, v.data_ptr(), ldv, p.kp, p.vp, p.ks, p.vs, p.pages, p.page, p.kv, p.hd, p.table, p.ldt, p.width, p.lens,
                             p.cu, p.B, rows, p.most, c.stream);
    return PyLong_FromLong(rc);
}
// (dev, stream, cache, table, start, cu, rows, max_rows, type)
PyObject* kv_read(PyObject* const* a) {
    const Call c(a);
    const int32_t rows = int32(a[13]);
    if (rows < 0) throw No();
    const Kv p(c, a + 2, rows, a[14]);
    if (!THPDtype_Check(a[15])) throw No();
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[15])->scalar_type;
    if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) throw No();
    const auto opt = c.tensor(a[2]).options().dtype(type).requires_grad(false);
    const int32_t n = int32((int64_t)p.kv * p.hd);
    const at::Tensor ko = at::empty({rows, n}, opt), vo = at::empty({rows, n}, opt);
    return result(go.read(dtype_of(ko), ko.data_ptr(), n, vo.data_ptr(), n, p.kp, p.vp, p.ks, p.vs, p.pages, p.page, p.kv, p.hd, p.table, p.ldt, p.width, p.lens,
                          p.cu, p.B, rows, p.most, c.stream), {ko, vo});
}
// (dev, stream, cache, table, lens, cu, q, heads, max_new, causal, window, scale or None)
PyObject* kv_attention(PyObject* const* a) {
    const Call c(a);
    const at::Tensor& q = c.tensor(a[13]);
    if (q.dim() != 2) throw No();
    const int32_t rows = int32(q.size(0)), heads = int32(a[14]), causal = int32(a[16]), window = int32(a[17]);
    const Kv p(c, a + 2, rows, a[15]);
    const int32_t dtype = dtype_of(q), n = int32((int64_t)heads * p.hd), ldq = c.rows(q, rows, n);
    const float scale = a[18] == Py_None ? (float)(1.0 / std::sqrt((double)p.hd)) : real(a[18]);
    const at::Tensor out = at::empty({rows, n}, q.options().requires_grad(false));
    const size_t bytes = go.attention_bytes(dtype, p.B, p.most, heads, p.kv, p.hd, p.width, p.page, causal, window);
    at::Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte).requires_grad(false));
    return result(go.attention(dtype, q.data_ptr(), ldq, p.kp, p.vp, p.ks, p.vs, p.pages, p.page, p.kv, p.hd, p.table, p.ldt, p.width, p.lens, p.cu, p.B, rows,
                               p.most, heads, scale, causal, window, out.data_ptr(), n, bytes ? ws.data_ptr() : nullptr, bytes, c.stream), {out});
}

template <PyObject* (*F)(PyObject* const*), int N> PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != N) return PyErr_Format(PyExc_TypeError, "%d arguments wanted, got %zd", N, n);
    try {
        return F(a);
    } catch (...) {      // No; or no memory: the other way says so in its own words
    }
    if (PyErr_Occurred()) PyErr_Clear();
    Py_RETURN_NONE;
}

// addresses of the library's entry points, in the order of Entries
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7) return PyErr_Format(PyExc_TypeError, "7 addresses wanted, got %zd", n);
    uintptr_t f[7];
    for (int i = 0; i < 7; ++i) {
        f[i] = (uintptr_t)PyLong_AsUnsignedLongLong(a[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    go.rope = (decltype(go.rope))f[0];
    go.rope_bwd = (decltype(go.rope_bwd))f[1];
    go.rope_bwd_bytes = (decltype(go.rope_bwd_bytes))f[2];
    go.append = (decltype(go.append))f[3];
    go.read = (decltype(go.read))f[4];
    go.attention = (decltype(go.attention))f[5];
    go.attention_bytes = (decltype(go.attention_bytes))f[6];
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void*)entry<qk_norm_rope, 12>, METH_FASTCALL, nullptr},
    {"qk_norm_rope_backward", (PyCFunction)(void*)entry<qk_norm_rope_backward, 14>, METH_FASTCALL, nullptr},
    {"kv_append", (PyCFunction)(void*)entry<kv_append, 16>, METH_FASTCALL, nullptr},
    {"kv_read", (PyCFunction)(void*)entry<kv_read, 16>, METH_FASTCALL, nullptr},
    {"kv_attention", (PyCFunction)(void*)entry<kv_attention, 19>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pgt_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pgt_ops() { return PyModule_Create(&module); }
