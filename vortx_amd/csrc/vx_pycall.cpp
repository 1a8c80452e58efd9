// vx_pycall.cpp — the Python binding's calls with torch tensors, as a CPython
// extension (vortx_amd/_pycall.<Python's tag>.so).
//
// Building the views of a call with ctypes structures took about 9 us of
// host time a call; reading the tensors' attributes through the C API instead
// takes 1 to 2. Calls whose kernel is shorter than that ran at the host's pace
// (a Q4_0 product at batch 1, 4096 x 4096: 11.4 us a call, now 5.6; a 64 x 64
// x 64 GEMM 13.0, now 7.0). These functions know only the plain case: exact
// torch.Tensor objects on the GPU of the expected element type, at most rank
// 4, streams by their cuda_stream attribute. For anything else (layout pairs,
// subclasses, wrong types, an exception on the way) they return None and the
// caller takes the ctypes path, which handles it or raises.
// Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <initializer_list>

#include "vortx_hip.h"

namespace {

PyObject *g_qweight, *g_tensor, *g_f32, *g_i32, *g_raw_stream, *g_get_device;  // setup()
PyObject *s_dtype, *s_is_cuda, *s_shape, *s_stride, *s_data_ptr, *s_element_size, *s_cuda_stream, *s_data, *s_qtype, *s_rows,
    *s_cols, *s_row_stride, *s_is_contiguous, *s_nbytes;

struct Ref {  // owned reference
    PyObject* o;
    explicit Ref(PyObject* p) : o(p) {}
    ~Ref() { Py_XDECREF(o); }
    Ref(const Ref&) = delete;
    Ref& operator=(const Ref&) = delete;
};

bool as_u64(PyObject* o, uint64_t max, uint64_t* out) {
    if (!o || !PyLong_CheckExact(o)) return false;
    const unsigned long long v = PyLong_AsUnsignedLongLong(o);
    if (v == (unsigned long long)-1 && PyErr_Occurred()) return false;
    *out = v;
    return v <= max;
}

bool attr_u64(PyObject* o, PyObject* name, uint64_t max, uint64_t* out) {
    Ref a(PyObject_GetAttr(o, name));
    return as_u64(a.o, max, out);
}

bool call_u64(PyObject* o, PyObject* name, uint64_t max, uint64_t* out) {
    Ref a(PyObject_CallMethodNoArgs(o, name));
    return as_u64(a.o, max, out);
}

bool is_gpu_tensor(PyObject* v) {
    if ((PyObject*)Py_TYPE(v) != g_tensor) return false;
    Ref c(PyObject_GetAttr(v, s_is_cuda));
    return c.o == Py_True;
}

// any4: any element type of four bytes, else float32
template <class View>
bool view_of(PyObject* v, bool any4, View* out) {
    if (!is_gpu_tensor(v)) return false;
    {
        Ref d(PyObject_GetAttr(v, s_dtype));
        uint64_t es = 0;
        if (d.o != g_f32 && !(any4 && d.o && call_u64(v, s_element_size, 4, &es) && es == 4)) return false;
    }
    Ref shape(PyObject_GetAttr(v, s_shape)), stride(PyObject_CallMethodNoArgs(v, s_stride));
    if (!shape.o || !stride.o || !PyTuple_Check(shape.o) || !PyTuple_Check(stride.o)) return false;
    const Py_ssize_t n = PyTuple_GET_SIZE(shape.o);
    if (n > 4 || PyTuple_GET_SIZE(stride.o) != n) return false;
    vx_layout& l = out->layout;
    for (int i = 0; i < 4; ++i) {
        uint64_t sz = 1, st = 1;
        if (i < n && (!as_u64(PyTuple_GET_ITEM(shape.o, i), UINT32_MAX, &sz) ||
                      !as_u64(PyTuple_GET_ITEM(stride.o, i), UINT32_MAX, &st)))
            return false;
        l.size[i] = (uint32_t)sz;
        l.stride[i] = (uint32_t)st;
    }
    l.rank = (uint32_t)n;
    l.offset = 0;  // in the pointer
    uint64_t p = 0;
    if (!call_u64(v, s_data_ptr, UINT64_MAX, &p) || !p) return false;  // (0: torch's for any empty view)
    out->base = (decltype(out->base))(uintptr_t)p;
    return true;
}

// A [tokens, heads, dim] view of f32.
template <class View>
bool rows_of(PyObject* v, View* out) {
    return view_of(v, false, out) && out->layout.rank == 3;
}

// An int32 GPU tensor of n x cols elements, rows in order: [n] with cols 0, else [n, cols] of any row stride.
bool ints_of(PyObject* v, uint32_t n, bool matrix, const int32_t** at, uint32_t* cols, uint32_t* row_stride) {
    if (!is_gpu_tensor(v)) return false;
    Ref d(PyObject_GetAttr(v, s_dtype)), shape(PyObject_GetAttr(v, s_shape)), stride(PyObject_CallMethodNoArgs(v, s_stride));
    const Py_ssize_t rank = matrix ? 2 : 1;
    if (d.o != g_i32 || !shape.o || !stride.o || !PyTuple_Check(shape.o) || !PyTuple_Check(stride.o) ||
        PyTuple_GET_SIZE(shape.o) != rank || PyTuple_GET_SIZE(stride.o) != rank)
        return false;
    uint64_t sz[2] = {0, 0}, st[2] = {0, 0}, p = 0;
    for (Py_ssize_t i = 0; i < rank; ++i)
        if (!as_u64(PyTuple_GET_ITEM(shape.o, i), UINT32_MAX, &sz[i]) || !as_u64(PyTuple_GET_ITEM(stride.o, i), UINT32_MAX, &st[i]))
            return false;
    if (sz[0] != n || st[rank - 1] != 1 || (matrix && n > 1 && st[0] < sz[1])) return false;
    if (!call_u64(v, s_data_ptr, UINT64_MAX, &p) || !p) return false;
    *at = (const int32_t*)(uintptr_t)p;
    if (matrix) *cols = (uint32_t)sz[1], *row_stride = n > 1 ? (uint32_t)st[0] : (uint32_t)sz[1];
    return true;
}

bool weight_of(PyObject* w, vx_qweight* out) {
    if ((PyObject*)Py_TYPE(w) != g_qweight) return false;
    Ref data(PyObject_GetAttr(w, s_data));
    uint64_t p = 0, q = 0, r = 0, c = 0, rs = 0;
    if (!data.o || !call_u64(data.o, s_data_ptr, UINT64_MAX, &p) || !attr_u64(w, s_qtype, UINT32_MAX, &q) ||
        !attr_u64(w, s_rows, UINT32_MAX, &r) || !attr_u64(w, s_cols, UINT32_MAX, &c) ||
        !attr_u64(w, s_row_stride, UINT64_MAX, &rs))
        return false;
    *out = vx_qweight{(const void*)(uintptr_t)p, (uint32_t)q, (uint32_t)r, (uint32_t)c, 0u, rs};
    return true;
}

// torch.cuda.current_stream().cuda_stream, or the attribute of the given one
bool stream_of(PyObject* s, vx_stream* out) {
    uint64_t v = 0;
    if (s == Py_None) {
        if (g_raw_stream == Py_None || g_get_device == Py_None) return false;
        Ref dev(PyObject_CallNoArgs(g_get_device));
        if (!dev.o) return false;
        Ref raw(PyObject_CallOneArg(g_raw_stream, dev.o));
        if (!as_u64(raw.o, UINT64_MAX, &v)) return false;
    } else if (!attr_u64(s, s_cuda_stream, UINT64_MAX, &v)) {
        return false;
    }
    *out = (vx_stream)(uintptr_t)v;
    return true;
}

void* addr(PyObject* o) {
    uint64_t v = 0;
    return as_u64(o, UINT64_MAX, &v) ? (void*)(uintptr_t)v : nullptr;
}

PyObject* other_path() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

template <class F>
PyObject* run(F f) {
    int s;
    Py_BEGIN_ALLOW_THREADS
    s = f();
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(s);
}

// setup(QWeight, torch.Tensor, torch.float32, raw stream of a device | None, current device | None, torch.int32)
PyObject* py_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    PyObject** g[] = {&g_qweight, &g_tensor, &g_f32, &g_raw_stream, &g_get_device, &g_i32};
    if (n != 6) return PyErr_Format(PyExc_TypeError, "setup takes 6 arguments");
    for (int i = 0; i < 6; ++i) {
        Py_INCREF(a[i]);
        Py_XSETREF(*g[i], a[i]);
    }
    Py_RETURN_NONE;
}

// gemm(fn, ctx, stream, out, lhs, rhs[, alpha, beta, flags]): fn a vx_gemm_f32 or, with the options, vx_gemm_f32_ex
PyObject* py_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 6 && n != 9) return other_path();
    void* fn = addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    vx_stream st;
    vx_mview o;
    vx_cview l, r;
    if (!fn || PyErr_Occurred() || !view_of(a[3], false, &o) || !view_of(a[4], false, &l) || !view_of(a[5], false, &r) ||
        !stream_of(a[2], &st))
        return other_path();
    if (n == 6) {
        auto f = (int (*)(vx_ctx, vx_stream, const vx_mview*, const vx_cview*, const vx_cview*))fn;
        return run([&] { return f(ctx, st, &o, &l, &r); });
    }
    uint64_t flags = 0;
    const double al = PyFloat_AsDouble(a[6]), be = PyFloat_AsDouble(a[7]);
    if (PyErr_Occurred() || !as_u64(a[8], UINT32_MAX, &flags)) return other_path();
    const vx_gemm_opts opts{(float)al, (float)be, (uint32_t)flags, 0u};
    auto f = (int (*)(vx_ctx, vx_stream, const vx_mview*, const vx_cview*, const vx_cview*, const vx_gemm_opts*))fn;
    return run([&] { return f(ctx, st, &o, &l, &r, &opts); });
}

// gemv(vx_gemv_q_ex, vx_gemv_q_ws, ctx, stream, y, w, x, flags, workspace | None)
PyObject* py_gemv(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 9) return other_path();
    void *fex = addr(a[0]), *fws = addr(a[1]);
    vx_ctx ctx = (vx_ctx)addr(a[2]);
    vx_stream st;
    vx_mview y;
    vx_cview x;
    vx_qweight w;
    uint64_t flags = 0, wp = 0, wn = 0;
    if (!fex || !fws || PyErr_Occurred() || !view_of(a[4], false, &y) || !view_of(a[6], false, &x) || !weight_of(a[5], &w) ||
        !as_u64(a[7], UINT32_MAX, &flags) || !stream_of(a[3], &st))
        return other_path();
    if (a[8] == Py_None) {
        auto f = (int (*)(vx_ctx, vx_stream, const vx_mview*, const vx_qweight*, const vx_cview*, uint32_t))fex;
        return run([&] { return f(ctx, st, &y, &w, &x, (uint32_t)flags); });
    }
    if (!is_gpu_tensor(a[8])) return other_path();
    Ref c(PyObject_CallMethodNoArgs(a[8], s_is_contiguous));
    if (c.o != Py_True || !call_u64(a[8], s_data_ptr, UINT64_MAX, &wp) || !attr_u64(a[8], s_nbytes, UINT64_MAX, &wn))
        return other_path();
    auto f = (int (*)(vx_ctx, vx_stream, const vx_mview*, const vx_qweight*, const vx_cview*, uint32_t, void*, uint64_t))fws;
    return run([&] { return f(ctx, st, &y, &w, &x, (uint32_t)flags, (void*)(uintptr_t)wp, wn); });
}

// dequantize(fn, ctx, stream, out, w)
PyObject* py_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 5) return other_path();
    auto f = (int (*)(vx_ctx, vx_stream, const vx_mview*, const vx_qweight*))addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    vx_stream st;
    vx_mview o;
    vx_qweight w;
    if (!f || PyErr_Occurred() || !view_of(a[3], false, &o) || !weight_of(a[4], &w) || !stream_of(a[2], &st)) return other_path();
    return run([&] { return f(ctx, st, &o, &w); });
}

// quantize(fn, ctx, stream, w, x)
PyObject* py_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 5) return other_path();
    auto f = (int (*)(vx_ctx, vx_stream, const vx_qweight*, const vx_cview*))addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    vx_stream st;
    vx_cview x;
    vx_qweight w;
    if (!f || PyErr_Occurred() || !weight_of(a[3], &w) || !view_of(a[4], false, &x) || !stream_of(a[2], &st)) return other_path();
    return run([&] { return f(ctx, st, &w, &x); });
}

// contiguous(fn, ctx, stream, out, src)
PyObject* py_contiguous(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 5) return other_path();
    auto f = (int (*)(vx_ctx, vx_stream, const vx_mview*, const vx_cview*, const uint32_t*))addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    vx_stream st;
    vx_mview o;
    vx_cview v;
    if (!f || PyErr_Occurred() || !view_of(a[3], true, &o) || !view_of(a[4], true, &v) || !stream_of(a[2], &st)) return other_path();
    return run([&] { return f(ctx, st, &o, &v, nullptr); });
}

// kv_write(fn, ctx, stream, cache, k, v, slots), cache the address of a vx_kv_cache; kv_read the same
template <class View, class F>
PyObject* kv_rows(PyObject* const* a, Py_ssize_t n, F call) {
    if (n != 7) return other_path();
    void* fn = addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    const vx_kv_cache* cache = (const vx_kv_cache*)addr(a[3]);
    vx_stream st;
    View k, v;
    const int32_t* slots = nullptr;
    if (!fn || !cache || PyErr_Occurred() || !rows_of(a[4], &k) || !rows_of(a[5], &v) ||
        !ints_of(a[6], k.layout.size[0], false, &slots, nullptr, nullptr) || !stream_of(a[2], &st))
        return other_path();
    return run([&] { return call(fn, ctx, st, cache, &k, &v, slots); });
}
PyObject* py_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return kv_rows<vx_cview>(a, n, [](void* fn, vx_ctx ctx, vx_stream st, const vx_kv_cache* c, const vx_cview* k, const vx_cview* v,
                                      const int32_t* slots) { return ((decltype(&vx_kv_write))fn)(ctx, st, c, k, v, slots); });
}
PyObject* py_kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return kv_rows<vx_mview>(a, n, [](void* fn, vx_ctx ctx, vx_stream st, const vx_kv_cache* c, const vx_mview* k, const vx_mview* v,
                                      const int32_t* slots) { return ((decltype(&vx_kv_read))fn)(ctx, st, k, v, c, slots); });
}

// What a vortx_amd.attention.Rotation says of itself: the address of its
// vx_rotation, the dim and heads that its weights are for (0: any) and the
// rotated dims, from a[0]; positions an int32 tensor or None.
struct Turn {
    const vx_rotation* how = nullptr;
    const int32_t* positions = nullptr;
    uint64_t dim = 0, q_heads = 0, k_heads = 0, rotated = 0;
    bool read(PyObject* const* a, PyObject* pos, uint32_t tokens) {
        how = (const vx_rotation*)addr(a[0]);
        if (!how || !as_u64(a[1], UINT32_MAX, &dim) || !as_u64(a[2], UINT32_MAX, &q_heads) || !as_u64(a[3], UINT32_MAX, &k_heads) ||
            !as_u64(a[4], UINT32_MAX, &rotated))
            return false;
        return pos == Py_None ? !rotated : ints_of(pos, tokens, false, &positions, nullptr, nullptr);
    }
    bool fits(const vx_layout& l, uint64_t heads) const {
        return (!dim || l.size[2] == dim) && (!heads || l.size[1] == heads);
    }
};

// rotate(fn, ctx, stream, q_out, q, k_out | None, k | None, positions | None, *Rotation's)
PyObject* py_rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 13) return other_path();
    auto f = (decltype(&vx_rotate))addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    vx_stream st;
    vx_mview qo, ko;
    vx_cview q, k;
    Turn t;
    const bool keys = a[5] != Py_None || a[6] != Py_None;
    if (!f || PyErr_Occurred() || !rows_of(a[3], &qo) || !rows_of(a[4], &q) || (keys && (!rows_of(a[5], &ko) || !rows_of(a[6], &k))) ||
        !t.read(a + 8, a[7], q.layout.size[0]) || !t.fits(q.layout, t.q_heads) || (keys && !t.fits(k.layout, t.k_heads)) ||
        !stream_of(a[2], &st))
        return other_path();
    return run([&] { return f(ctx, st, &qo, &q, keys ? &ko : nullptr, keys ? &k : nullptr, t.positions, t.how); });
}

// kv_write_rotated(fn, ctx, stream, cache, q_out | None, q | None, k, v, positions | None, slots, *Rotation's)
PyObject* py_kv_write_rotated(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 15) return other_path();
    auto f = (decltype(&vx_kv_write_rotated))addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    const vx_kv_cache* cache = (const vx_kv_cache*)addr(a[3]);
    vx_stream st;
    vx_mview qo;
    vx_cview q, k, v;
    Turn t;
    const int32_t* slots = nullptr;
    const bool queries = a[4] != Py_None || a[5] != Py_None;
    if (!f || !cache || PyErr_Occurred() || (queries && (!rows_of(a[4], &qo) || !rows_of(a[5], &q))) || !rows_of(a[6], &k) ||
        !rows_of(a[7], &v) || !ints_of(a[9], k.layout.size[0], false, &slots, nullptr, nullptr) ||
        !t.read(a + 10, a[8], k.layout.size[0]) || (queries && !t.fits(q.layout, t.q_heads)) || !t.fits(k.layout, t.k_heads) ||
        !stream_of(a[2], &st))
        return other_path();
    return run([&] { return f(ctx, st, cache, queries ? &qo : nullptr, queries ? &q : nullptr, &k, &v, t.positions, slots, t.how); });
}

// kv_resize(fn, ctx, stream, pages, seqs, want, starts, slots, positions, tokens): a vx_kv_pages and the outputs by their addresses
PyObject* py_kv_resize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 10) return other_path();
    auto f = (decltype(&vx_kv_resize))addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    const vx_kv_pages* pages = (const vx_kv_pages*)addr(a[3]);
    vx_stream st;
    uint64_t seqs = 0, starts = 0, slots = 0, positions = 0, tokens = 0;
    const int32_t* want = nullptr;
    if (!f || !pages || PyErr_Occurred() || !as_u64(a[4], UINT32_MAX, &seqs) || !ints_of(a[5], (uint32_t)seqs, false, &want, nullptr, nullptr) ||
        !as_u64(a[6], UINT64_MAX, &starts) || !as_u64(a[7], UINT64_MAX, &slots) || !as_u64(a[8], UINT64_MAX, &positions) ||
        !as_u64(a[9], UINT32_MAX, &tokens) || !stream_of(a[2], &st))
        return other_path();
    return run([&] {
        return f(ctx, st, pages, want, (int32_t*)(uintptr_t)starts, (int32_t*)(uintptr_t)slots, (int32_t*)(uintptr_t)positions, (uint32_t)tokens);
    });
}

// i8_quantize(fn, ctx, stream, rows, x), rows the address of a vx_i8_rows
PyObject* py_i8_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 5) return other_path();
    auto f = (decltype(&vx_i8_quantize))addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    const vx_i8_rows* rows = (const vx_i8_rows*)addr(a[3]);
    vx_stream st;
    vx_cview x;
    if (!f || !rows || PyErr_Occurred() || !view_of(a[4], false, &x) || !stream_of(a[2], &st)) return other_path();
    return run([&] { return f(ctx, st, rows, &x); });
}

// gemm_i8(fn, ctx, stream, out, rows | None, x, w, up | None, act, workspace | None): fn a vx_gemm_i8 or vx_gemm_i8_gated
// of rows, the address of a vx_i8_rows, or without them their _x forms of x, a tensor (whatever x is otherwise); w and up addresses
PyObject* py_gemm_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 10) return other_path();
    void* fn = addr(a[0]);
    vx_ctx ctx = (vx_ctx)addr(a[1]);
    const vx_i8_rows *w = (const vx_i8_rows*)addr(a[6]), *u = nullptr;
    const bool rows = a[4] != Py_None, gated = a[7] != Py_None;
    if (gated && !(u = (const vx_i8_rows*)addr(a[7]))) return other_path();
    vx_stream st;
    vx_mview o;
    vx_cview x;
    uint64_t act = 0, wp = 0, wn = 0;
    const vx_i8_rows* xq = rows ? (const vx_i8_rows*)addr(a[4]) : nullptr;
    if (!fn || !w || (rows && !xq) || PyErr_Occurred() || !view_of(a[3], false, &o) || (!rows && !view_of(a[5], false, &x)) ||
        !as_u64(a[8], UINT32_MAX, &act) || !stream_of(a[2], &st))
        return other_path();
    if (rows)
        return run([&] {
            return gated ? ((decltype(&vx_gemm_i8_gated))fn)(ctx, st, &o, xq, w, u, (uint32_t)act) : ((decltype(&vx_gemm_i8))fn)(ctx, st, &o, xq, w);
        });
    if (a[9] != Py_None) {
        if (!is_gpu_tensor(a[9])) return other_path();
        Ref c(PyObject_CallMethodNoArgs(a[9], s_is_contiguous));
        if (c.o != Py_True || !call_u64(a[9], s_data_ptr, UINT64_MAX, &wp) || !attr_u64(a[9], s_nbytes, UINT64_MAX, &wn)) return other_path();
    }
    void* ws = (void*)(uintptr_t)wp;
    return run([&] {
        return gated ? ((decltype(&vx_gemm_i8_gated_x))fn)(ctx, st, &o, &x, w, u, (uint32_t)act, ws, wn)
                     : ((decltype(&vx_gemm_i8_x))fn)(ctx, st, &o, &x, w, ws, wn);
    });
}

// attend(vx_attention, vx_attention_tree, ctx, stream, out, q, tree | None, cache, batch, opts, workspace, its bytes,
//        query heads, tokens at most), the plan's structs by their addresses
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 14) return other_path();
    void *fn = addr(a[0]), *ft = addr(a[1]);
    vx_ctx ctx = (vx_ctx)addr(a[2]);
    const vx_kv_cache* cache = (const vx_kv_cache*)addr(a[7]);
    const vx_attn_batch* batch = (const vx_attn_batch*)addr(a[8]);
    const vx_attn_opts* opts = (const vx_attn_opts*)addr(a[9]);
    vx_stream st;
    vx_mview o;
    vx_cview q;
    uint64_t ws = 0, bytes = 0, heads = 0, most = 0;
    if (!fn || !ft || !cache || !batch || !opts || PyErr_Occurred() || !rows_of(a[4], &o) || !rows_of(a[5], &q) ||
        !as_u64(a[10], UINT64_MAX, &ws) || !as_u64(a[11], UINT64_MAX, &bytes) || !as_u64(a[12], UINT32_MAX, &heads) ||
        !as_u64(a[13], UINT32_MAX, &most) || q.layout.size[1] != heads || q.layout.size[0] > most || !stream_of(a[3], &st))
        return other_path();
    if (a[6] == Py_None)
        return run([&] { return ((decltype(&vx_attention))fn)(ctx, st, &o, &q, cache, batch, opts, (void*)(uintptr_t)ws, bytes); });
    const int32_t* tree = nullptr;
    uint32_t words = 0, stride = 0;
    if (!ints_of(a[6], q.layout.size[0], true, &tree, &words, &stride)) return other_path();
    return run([&] {
        return ((decltype(&vx_attention_tree))ft)(ctx, st, &o, &q, cache, batch, opts, (const uint32_t*)tree, words, stride,
                                                  (void*)(uintptr_t)ws, bytes);
    });
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"setup", FAST(py_setup)},           {"gemm", FAST(py_gemm)},
                         {"gemv", FAST(py_gemv)},             {"dequantize", FAST(py_dequantize)},
                         {"quantize", FAST(py_quantize)},     {"contiguous", FAST(py_contiguous)},
                         {"kv_write", FAST(py_kv_write)},     {"kv_read", FAST(py_kv_read)},
                         {"attend", FAST(py_attend)},         {"rotate", FAST(py_rotate)},
                         {"kv_write_rotated", FAST(py_kv_write_rotated)}, {"kv_resize", FAST(py_kv_resize)},
                         {"i8_quantize", FAST(py_i8_quantize)}, {"gemm_i8", FAST(py_gemm_i8)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pycall(void) {
    struct {
        PyObject** s;
        const char* n;
    } names[] = {{&s_dtype, "dtype"},       {&s_is_cuda, "is_cuda"},           {&s_shape, "shape"},
                 {&s_stride, "stride"},     {&s_data_ptr, "data_ptr"},         {&s_element_size, "element_size"},
                 {&s_cuda_stream, "cuda_stream"}, {&s_data, "data"},           {&s_qtype, "qtype"},
                 {&s_rows, "rows"},         {&s_cols, "cols"},                 {&s_row_stride, "row_stride"},
                 {&s_is_contiguous, "is_contiguous"}, {&s_nbytes, "nbytes"}};
    for (auto& e : names)
        if (!(*e.s = PyUnicode_InternFromString(e.n))) return nullptr;
    for (PyObject** g : {&g_qweight, &g_tensor, &g_f32, &g_i32, &g_raw_stream, &g_get_device}) {  // nothing matches before setup()
        Py_INCREF(Py_None);
        *g = Py_None;
    }
    return PyModule_Create(&module);
}
