/*
 * binding.cpp -- the per-step calls of Hy3Attn (attn.py) as native functions: batch_set, append, decode_step, prefill; and the operators
 * beside the attention (layer.py): route, experts, adapters, quantize4, linear4, logprobs.
 *
 * A decode step of a short context takes 6 to 9 us on the GPU; the same call through ctypes cost the host 6.6 us (four to seven
 * tensors asked for their strides, types and addresses one attribute at a time, 11 to 15 arguments converted one by one).  Here the
 * checks are the same and made on every call, on the tensors themselves.  The C ABI stays the way in: the functions' addresses come
 * from the library that _lib.py loaded (bind()).
 */
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/hy3_attn.h"

namespace {

decltype(&hy3a_batch_set) f_batch_set;
decltype(&hy3a_append) f_append;
decltype(&hy3a_decode_step) f_decode_step;
decltype(&hy3a_prefill) f_prefill;
decltype(&hy3a_route) f_route;
decltype(&hy3a_experts_workspace) f_experts_workspace;
decltype(&hy3a_experts) f_experts;
decltype(&hy3a_adapters_workspace) f_adapters_workspace;
decltype(&hy3a_adapters) f_adapters;
decltype(&hy3a_quantize4) f_quantize4;
decltype(&hy3a_linear4) f_linear4;
decltype(&hy3a_logprobs) f_logprobs;

constexpr int64_t kH = HY3A_N_HEAD, kD = HY3A_HEAD_DIM;

PyObject *refuse(const char *what) {
    PyErr_SetString(PyExc_AssertionError, what);
    return nullptr;
}
/* a tensor argument: nullptr for None */
bool tensor(PyObject *o, const at::Tensor *&t) {
    t = nullptr;
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) { PyErr_SetString(PyExc_TypeError, "expected a torch.Tensor or None"); return false; }
    t = &THPVariable_Unpack(o);
    return true;
}
template <class T> T *ptr(const at::Tensor *t) { return t ? static_cast<T *>(t->data_ptr()) : nullptr; }
/* fp32 rows of dense heads: n of them, row stride free */
bool rows(const at::Tensor *t, int64_t n) {
    if (!t) return true;
    const int64_t d = t->dim();
    return d >= 2 && t->size(0) == n && t->scalar_type() == at::kFloat && t->stride(d - 1) == 1 && t->stride(d - 2) == kD;
}
size_t stride0(const at::Tensor *t) { return t ? (size_t)t->stride(0) : 0; }

/* a C-contiguous host buffer */
struct buffer {
    Py_buffer b;
    bool held = false;
    ~buffer() { if (held) PyBuffer_Release(&b); }
    bool get(PyObject *o) {
        if (PyObject_GetBuffer(o, &b, PyBUF_C_CONTIGUOUS)) return false;
        held = true;
        return true;
    }
};

/* C++ exceptions (a tensor without storage, without strides) become Python's */
template <PyObject *(*F)(PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *, PyObject *const *a, Py_ssize_t na) {
    try {
        return F(a, na);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

int as_int(PyObject *o) {
    const long v = PyLong_AsLong(o);
    if (v != (int)v) PyErr_SetString(PyExc_OverflowError, "value does not fit an int");
    return (int)v;
}
/* the leading arguments of the per-layer calls: ctx, layer */
bool head(PyObject *const *a, hy3a_ctx *&h, int &layer) {
    h = (hy3a_ctx *)PyLong_AsVoidPtr(a[0]);
    if (!h && PyErr_Occurred()) return false;
    layer = as_int(a[1]);
    return !PyErr_Occurred();
}

/* batch_set(ctx, seq, slot, pos): int32 arrays of the same length */
PyObject *batch_set(PyObject *const *a, Py_ssize_t na) {
    if (na != 4) return refuse("batch_set: 4 arguments");
    hy3a_ctx *h = (hy3a_ctx *)PyLong_AsVoidPtr(a[0]);
    if (!h && PyErr_Occurred()) return nullptr;
    buffer v[3];
    for (int i = 0; i < 3; i++) if (!v[i].get(a[1 + i])) return nullptr;
    if (v[0].b.itemsize != 4 || v[1].b.itemsize != 4 || v[2].b.itemsize != 4 || v[0].b.len != v[1].b.len || v[0].b.len != v[2].b.len)
        return refuse("batch_set: int32 arrays of one length");
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_batch_set(h, (int)(v[0].b.len / 4), (const int *)v[0].b.buf, (const int *)v[1].b.buf, (const int *)v[2].b.buf);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* append(ctx, layer, n, q, k, v, q_out, q_out16) */
PyObject *append(PyObject *const *a, Py_ssize_t na) {
    if (na != 8) return refuse("append: 8 arguments");
    hy3a_ctx *h;
    int layer;
    if (!head(a, h, layer)) return nullptr;
    const int64_t n = PyLong_AsLongLong(a[2]);
    const at::Tensor *q, *k, *v, *qo, *q16;
    if (PyErr_Occurred() || !tensor(a[3], q) || !tensor(a[4], k) || !tensor(a[5], v) || !tensor(a[6], qo) || !tensor(a[7], q16)) return nullptr;
    if (!q || !k != !v) return refuse("append: q, and k with v");
    if (!rows(q, n) || !rows(k, n) || !rows(v, n)) return refuse("append: q, k, v are fp32 with n rows of dense heads");
    if (q16 && (q16->scalar_type() != at::kHalf || !q16->is_contiguous() || q16->numel() != n * kH * kD)) return refuse("append: q_out16 is contiguous fp16 [n, 64, 128]");
    const float *qp = ptr<const float>(q), *kp = ptr<const float>(k), *vp = ptr<const float>(v);
    float *qop = ptr<float>(qo);
    void *q16p = ptr<void>(q16);
    const size_t sq = stride0(q), sk = stride0(k), sv = stride0(v), so = stride0(qo);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_append(h, layer, qp, sq, kp, sk, vp, sv, qop, so, q16p);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* decode_step(ctx, layer, n, q, k, v, q_out, out, partials) */
PyObject *decode_step(PyObject *const *a, Py_ssize_t na) {
    if (na != 9) return refuse("decode_step: 9 arguments");
    hy3a_ctx *h;
    int layer;
    if (!head(a, h, layer)) return nullptr;
    const int64_t n = PyLong_AsLongLong(a[2]);
    const at::Tensor *q, *k, *v, *qo, *out, *part;
    if (PyErr_Occurred() || !tensor(a[3], q) || !tensor(a[4], k) || !tensor(a[5], v) || !tensor(a[6], qo) || !tensor(a[7], out) || !tensor(a[8], part)) return nullptr;
    if (!q || !k != !v) return refuse("decode_step: q, and k with v");
    if (!rows(q, n) || !rows(k, n) || !rows(v, n)) return refuse("decode_step: q, k, v are fp32 with n rows of dense heads");
    const float *qp = ptr<const float>(q), *kp = ptr<const float>(k), *vp = ptr<const float>(v);
    float *qop = ptr<float>(qo), *op = ptr<float>(out), *pp = ptr<float>(part);
    const size_t sq = stride0(q), sk = stride0(k), sv = stride0(v), sqo = stride0(qo), so = stride0(out);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_decode_step(h, layer, qp, sq, kp, sk, vp, sv, qop, sqo, op, so, pp);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* prefill(ctx, layer, seq, base_slot, q16, out) */
PyObject *prefill(PyObject *const *a, Py_ssize_t na) {
    if (na != 6) return refuse("prefill: 6 arguments");
    hy3a_ctx *h;
    int layer;
    if (!head(a, h, layer)) return nullptr;
    const int seq = as_int(a[2]), base = PyErr_Occurred() ? 0 : as_int(a[3]);
    const at::Tensor *q16, *out;
    if (PyErr_Occurred() || !tensor(a[4], q16) || !tensor(a[5], out)) return nullptr;
    if (!q16 || !out || q16->dim() < 1 || q16->scalar_type() != at::kHalf || !q16->is_contiguous()) return refuse("prefill: q16 is contiguous fp16, out a tensor");
    const int nq = (int)q16->size(0);
    const void *qp = ptr<const void>(q16);
    float *op = ptr<float>(out);
    const size_t so = stride0(out);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_prefill(h, layer, seq, base, nq, qp, op, so);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* ---- operators beside the attention: tensors on one GPU, checked here; outputs and workspaces from torch's allocator ---- */
int dtype_code(const at::Tensor *t) {
    switch (t->scalar_type()) {
        case at::kFloat: return HY3A_F32;
        case at::kHalf: return HY3A_F16;
        case at::kBFloat16: return HY3A_BF16;
        default: return -1;
    }
}
bool on_gpu_with(const at::Tensor *t, const at::Tensor &x) { return t->is_cuda() && t->device() == x.device(); }
/* a matrix with dense rows; its row stride (of a single row: its length) */
bool matrix(const at::Tensor *t) { return t->dim() == 2 && (t->stride(1) == 1 || t->size(1) <= 1); }
size_t row_stride(const at::Tensor *t) { return (size_t)(t->size(0) > 1 ? t->stride(0) : t->size(1)); }
bool dense(const at::Tensor *t, at::ScalarType type, const at::Tensor &x) { return t->scalar_type() == type && t->is_contiguous() && on_gpu_with(t, x); }
/* sizes are ints in the C ABI */
bool fits(std::initializer_list<int64_t> v) { for (int64_t n : v) if (n < 0 || n > 0x7fffffff) return false; return true; }
at::Tensor workspace(size_t bytes, const at::Tensor &x) { return at::empty({(int64_t)(bytes ? bytes : 1)}, x.options().dtype(at::kByte)); }
void *as_stream(PyObject *o) { return PyLong_AsVoidPtr(o); }

/* Whether autograd would look for a gradient here: there is none, and an output without one would end it unseen. */
bool wants_grad(std::initializer_list<const at::Tensor *> v) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor *t : v) if (t && t->requires_grad()) return true;
    return false;
}
/* what was written into has changed, for those that keep it for a backward pass */
void changed(const at::Tensor *t) { if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version(); }

/* route(stream, logits, bias, top_k, score, groups, top_groups, renormalize, scale) -> (ids, weights) */
PyObject *route(PyObject *const *a, Py_ssize_t na) {
    if (na != 9) return refuse("route: 9 arguments");
    void *stream = as_stream(a[0]);
    const at::Tensor *l, *bias;
    if (PyErr_Occurred() || !tensor(a[1], l) || !tensor(a[2], bias)) return nullptr;
    int v[4];
    for (int i = 0; i < 4; i++) { v[i] = as_int(a[3 + i]); if (PyErr_Occurred()) return nullptr; }
    const int renorm = PyObject_IsTrue(a[7]);
    const double scale = PyFloat_AsDouble(a[8]);
    if (PyErr_Occurred()) return nullptr;
    if (!l || !l->is_cuda() || !matrix(l) || dtype_code(l) < 0) return refuse("route: logits are a CUDA matrix of fp32, fp16 or bf16 with dense rows");
    const int64_t rows = l->size(0), n = l->size(1);
    if (bias && (!dense(bias, at::kFloat, *l) || bias->numel() != n)) return refuse("route: bias is fp32 [experts] on the logits' device");
    if (wants_grad({l, bias})) return refuse("route: computes no gradients: call it under torch.no_grad()");
    if (!fits({rows, n})) return refuse("route: sizes do not fit an int");
    const int64_t k = v[0] < 0 ? 0 : v[0];
    c10::DeviceGuard guard(l->device());
    at::Tensor ids = at::empty({rows, k}, l->options().dtype(at::kInt)), w = at::empty({rows, k}, l->options().dtype(at::kFloat));
    const void *lp = l->data_ptr();
    const float *bp = ptr<const float>(bias);
    int *ip = (int *)ids.data_ptr();
    float *wp = (float *)w.data_ptr();
    const size_t stride = row_stride(l);
    const int dt = dtype_code(l);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_route(stream, dt, (int)rows, (int)n, lp, stride, bp, v[0], v[1], v[2], v[3], renorm, (float)scale, ip, wp);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    PyObject *pi = THPVariable_Wrap(ids), *pw = THPVariable_Wrap(w), *r = pi && pw ? PyTuple_Pack(2, pi, pw) : nullptr;
    Py_XDECREF(pi);
    Py_XDECREF(pw);
    return r;
}
/* experts(stream, x, ids, weights, gate, up, down, first_expert, out) -> out */
PyObject *experts(PyObject *const *a, Py_ssize_t na) {
    if (na != 9) return refuse("experts: 9 arguments");
    void *stream = as_stream(a[0]);
    const at::Tensor *x, *ids, *w, *gate, *up, *down, *given;
    if (PyErr_Occurred() || !tensor(a[1], x) || !tensor(a[2], ids) || !tensor(a[3], w) || !tensor(a[4], gate) || !tensor(a[5], up) || !tensor(a[6], down) || !tensor(a[8], given)) return nullptr;
    const int first = as_int(a[7]);
    if (PyErr_Occurred()) return nullptr;
    if (!x || !ids || !w || !gate || !up || !down) return refuse("experts: tensors, and out or None");
    const at::ScalarType type = x->scalar_type();
    if (!x->is_cuda() || !matrix(x) || (type != at::kHalf && type != at::kBFloat16)) return refuse("experts: x is a CUDA matrix of fp16 or bf16 with dense rows");
    const int64_t rows = x->size(0), hidden = x->size(1);
    if (ids->dim() != 2 || ids->size(0) != rows || !dense(ids, at::kInt, *x) || w->sizes() != ids->sizes() || !dense(w, at::kFloat, *x))
        return refuse("experts: ids and weights are contiguous int32 and fp32 [rows, top_k] on x's device");
    if (gate->dim() != 3 || gate->size(2) != hidden || up->sizes() != gate->sizes() || down->dim() != 3 || down->size(0) != gate->size(0) || down->size(1) != hidden ||
        down->size(2) != gate->size(1) || !dense(gate, type, *x) || !dense(up, type, *x) || !dense(down, type, *x))
        return refuse("experts: gate and up [held, inter, hidden] and down [held, hidden, inter] are contiguous, of x's type and on its device");
    const int64_t held = gate->size(0), inter = gate->size(1), k = ids->size(1);
    if (given && (!on_gpu_with(given, *x) || given->scalar_type() != type || !matrix(given) || given->sizes() != x->sizes())) return refuse("experts: out is like x");
    if (wants_grad({x, w, gate, up, down, given})) return refuse("experts: computes no gradients: call it under torch.no_grad()");
    if (!fits({rows, hidden, held, inter, k})) return refuse("experts: sizes do not fit an int");
    c10::DeviceGuard guard(x->device());
    at::Tensor out = given ? *given : at::empty({rows, hidden}, x->options());
    const size_t bytes = f_experts_workspace((int)rows, (int)k, (int)hidden, (int)inter, (int)held);
    at::Tensor work = workspace(bytes, *x);
    const int dt = dtype_code(x);
    const void *xp = x->data_ptr(), *gp = gate->data_ptr(), *up_ = up->data_ptr(), *dp = down->data_ptr();
    const int *ip = (const int *)ids->data_ptr();
    const float *wp = (const float *)w->data_ptr();
    void *op = out.data_ptr(), *kp = work.data_ptr();
    const size_t sx = row_stride(x), so = row_stride(&out);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_experts(stream, dt, (int)rows, (int)k, (int)hidden, (int)inter, (int)held, first, xp, sx, ip, wp, gp, up_, dp, op, so, kp, bytes);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    changed(given);
    return THPVariable_Wrap(out);
}
/* adapters(stream, x, base, a, b, ids, scales, out) -> out */
PyObject *adapters(PyObject *const *a, Py_ssize_t na) {
    if (na != 8) return refuse("adapters: 8 arguments");
    void *stream = as_stream(a[0]);
    const at::Tensor *x, *base, *la, *lb, *ids, *sc, *given;
    if (PyErr_Occurred() || !tensor(a[1], x) || !tensor(a[2], base) || !tensor(a[3], la) || !tensor(a[4], lb) || !tensor(a[5], ids) || !tensor(a[6], sc) || !tensor(a[7], given)) return nullptr;
    if (!x || !base || !la || !lb || !ids || !sc) return refuse("adapters: tensors, and out or None");
    const at::ScalarType type = x->scalar_type();
    if (!x->is_cuda() || !matrix(x) || (type != at::kHalf && type != at::kBFloat16)) return refuse("adapters: x is a CUDA matrix of fp16 or bf16 with dense rows");
    const int64_t rows = x->size(0), width = x->size(1);
    if (!matrix(base) || base->size(0) != rows || !on_gpu_with(base, *x) || (base->scalar_type() != type && base->scalar_type() != at::kFloat))
        return refuse("adapters: base is a matrix of x's rows, of x's type or fp32, on its device");
    const int64_t wide = base->size(1);
    if (la->dim() != 3 || la->size(2) != width || lb->dim() != 3 || lb->size(0) != la->size(0) || lb->size(1) != wide || lb->size(2) != la->size(1) || !dense(la, type, *x) || !dense(lb, type, *x))
        return refuse("adapters: a [adapters, rank, width] and b [adapters, out_width, rank] are contiguous, of x's type and on its device");
    const int64_t n = la->size(0), rank = la->size(1);
    if (!dense(ids, at::kInt, *x) || ids->dim() != 1 || ids->size(0) != rows || !dense(sc, at::kFloat, *x) || sc->numel() != n)
        return refuse("adapters: ids are int32 [rows], scales fp32 [adapters], on x's device");
    if (given && (!on_gpu_with(given, *x) || given->scalar_type() != base->scalar_type() || !matrix(given) || given->sizes() != base->sizes())) return refuse("adapters: out is like base");
    if (wants_grad({x, base, la, lb, sc, given})) return refuse("adapters: computes no gradients: call it under torch.no_grad()");
    if (!fits({rows, width, wide, n, rank})) return refuse("adapters: sizes do not fit an int");
    c10::DeviceGuard guard(x->device());
    at::Tensor out = given ? *given : at::empty({rows, wide}, base->options());
    const size_t bytes = f_adapters_workspace((int)rows, (int)width, (int)rank);
    at::Tensor work = workspace(bytes, *x);
    const int dt = dtype_code(x), bt = dtype_code(base);
    const void *xp = x->data_ptr(), *bp = base->data_ptr(), *ap = la->data_ptr(), *b2 = lb->data_ptr();
    const int *ip = (const int *)ids->data_ptr();
    const float *sp = (const float *)sc->data_ptr();
    void *op = out.data_ptr(), *kp = work.data_ptr();
    const size_t sx = row_stride(x), sb = row_stride(base), so = row_stride(&out);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_adapters(stream, dt, (int)rows, (int)width, (int)wide, (int)n, (int)rank, xp, sx, bt, bp, sb, ap, b2, ip, sp, op, so, kp, bytes);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    changed(given);
    return THPVariable_Wrap(out);
}
/* a torch.dtype, `fallback` for None */
bool scalar_type(PyObject *o, at::ScalarType fallback, at::ScalarType &t) {
    t = fallback;
    if (o == Py_None) return true;
    if (!THPDtype_Check(o)) { PyErr_SetString(PyExc_TypeError, "expected a torch.dtype or None"); return false; }
    t = reinterpret_cast<THPDtype *>(o)->scalar_type;
    return true;
}
int code_of(at::ScalarType t) { return t == at::kFloat ? HY3A_F32 : (t == at::kHalf ? HY3A_F16 : (t == at::kBFloat16 ? HY3A_BF16 : -1)); }

/* quantize4(stream, w, group, dtype) -> (codes, scales) */
PyObject *quantize4(PyObject *const *a, Py_ssize_t na) {
    if (na != 4) return refuse("quantize4: 4 arguments");
    void *stream = as_stream(a[0]);
    const at::Tensor *w;
    if (PyErr_Occurred() || !tensor(a[1], w)) return nullptr;
    const int group = as_int(a[2]);
    if (PyErr_Occurred()) return nullptr;
    if (!w || !w->is_cuda() || !matrix(w) || dtype_code(w) < 0) return refuse("quantize4: w is a CUDA matrix of fp32, fp16 or bf16 with dense rows");
    at::ScalarType type;
    if (!scalar_type(a[3], w->scalar_type() == at::kHalf ? at::kHalf : at::kBFloat16, type)) return nullptr;
    if (type != at::kHalf && type != at::kBFloat16) return refuse("quantize4: dtype is fp16 or bf16");
    if (wants_grad({w})) return refuse("quantize4: computes no gradients: call it under torch.no_grad()");
    const int64_t out = w->size(0), width = w->size(1);
    if (!fits({out, width})) return refuse("quantize4: sizes do not fit an int");
    const int64_t groups = group > 0 ? (width + group - 1) / group : 0;
    c10::DeviceGuard guard(w->device());
    at::Tensor codes = at::empty({out, width / 2}, w->options().dtype(at::kByte)), scales = at::empty({out, groups}, w->options().dtype(type));
    const void *wp = w->data_ptr();
    void *cp = codes.data_ptr(), *sp = scales.data_ptr();
    const size_t stride = row_stride(w);
    const int wt = dtype_code(w), st = code_of(type);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_quantize4(stream, wt, (int)out, (int)width, group, wp, stride, st, cp, sp);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    PyObject *pc = THPVariable_Wrap(codes), *ps = THPVariable_Wrap(scales), *r = pc && ps ? PyTuple_Pack(2, pc, ps) : nullptr;
    Py_XDECREF(pc);
    Py_XDECREF(ps);
    return r;
}
/* linear4(stream, x, codes, scales, out_dtype, out) -> out */
PyObject *linear4(PyObject *const *a, Py_ssize_t na) {
    if (na != 6) return refuse("linear4: 6 arguments");
    void *stream = as_stream(a[0]);
    const at::Tensor *x, *codes, *scales, *given;
    if (PyErr_Occurred() || !tensor(a[1], x) || !tensor(a[2], codes) || !tensor(a[3], scales) || !tensor(a[5], given)) return nullptr;
    if (!x || !codes || !scales) return refuse("linear4: tensors, and out or None");
    const at::ScalarType type = x->scalar_type();
    if (!x->is_cuda() || !matrix(x) || (type != at::kHalf && type != at::kBFloat16)) return refuse("linear4: x is a CUDA matrix of fp16 or bf16 with dense rows");
    const int64_t rows = x->size(0), width = x->size(1);
    if (codes->dim() != 2 || codes->size(1) * 2 != width || !dense(codes, at::kByte, *x) || scales->dim() != 2 || scales->size(0) != codes->size(0) || !dense(scales, type, *x))
        return refuse("linear4: codes are contiguous uint8 [out_width, width / 2], scales [out_width, groups] of x's type, on its device");
    const int64_t wide = codes->size(0), groups = scales->size(1);
    /* (two sizes that make as many groups make one of them: it does not matter which is meant) */
    int group = 0;
    for (int g = 32; g <= 128 && !group; g *= 2) if ((width + g - 1) / g == groups) group = g;
    if (!group) return refuse("linear4: scales are one for each 32, 64 or 128 neighbours in a row");
    at::ScalarType result;
    if (!scalar_type(a[4], given ? given->scalar_type() : type, result)) return nullptr;
    if (result != type && result != at::kFloat) return refuse("linear4: the result is of x's type or fp32");
    if (given && (!on_gpu_with(given, *x) || given->scalar_type() != result || !matrix(given) || given->size(0) != rows || given->size(1) != wide)) return refuse("linear4: out is a matrix [rows, out_width] of the result's type on x's device");
    if (wants_grad({x, scales, given})) return refuse("linear4: computes no gradients: call it under torch.no_grad()");
    if (!fits({rows, width, wide})) return refuse("linear4: sizes do not fit an int");
    c10::DeviceGuard guard(x->device());
    at::Tensor out = given ? *given : at::empty({rows, wide}, x->options().dtype(result));
    const int dt = dtype_code(x), ot = code_of(result);
    const void *xp = x->data_ptr(), *cp = codes->data_ptr(), *sp = scales->data_ptr();
    void *op = out.data_ptr();
    const size_t sx = row_stride(x), so = row_stride(&out);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_linear4(stream, dt, (int)rows, (int)width, (int)wide, group, xp, sx, cp, sp, ot, op, so);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    changed(given);
    return THPVariable_Wrap(out);
}
/* logprobs(stream, logits, tokens, top_k) -> (log probabilities or None, entropy, ids, their log probabilities) */
PyObject *logprobs(PyObject *const *a, Py_ssize_t na) {
    if (na != 4) return refuse("logprobs: 4 arguments");
    void *stream = as_stream(a[0]);
    const at::Tensor *l, *tokens;
    if (PyErr_Occurred() || !tensor(a[1], l) || !tensor(a[2], tokens)) return nullptr;
    const int top_k = as_int(a[3]);
    if (PyErr_Occurred()) return nullptr;
    if (!l || !l->is_cuda() || !matrix(l) || dtype_code(l) < 0) return refuse("logprobs: logits are a CUDA matrix of fp32, fp16 or bf16 with dense rows");
    const int64_t rows = l->size(0), vocab = l->size(1);
    if (tokens && (tokens->dim() < 1 || tokens->dim() > 2 || tokens->size(0) != rows || !dense(tokens, at::kInt, *l))) return refuse("logprobs: tokens are contiguous int32 [rows] or [rows, asked] on the logits' device");
    const int64_t asked = !tokens ? 0 : (tokens->dim() == 1 ? 1 : tokens->size(1));
    if (wants_grad({l})) return refuse("logprobs: computes no gradients: call it under torch.no_grad()");
    if (!fits({rows, vocab, asked})) return refuse("logprobs: sizes do not fit an int");
    const int64_t k = top_k < 0 ? 0 : top_k;
    c10::DeviceGuard guard(l->device());
    const at::TensorOptions f32 = l->options().dtype(at::kFloat);
    at::Tensor logp = tokens ? at::empty(tokens->sizes(), f32) : at::Tensor(), entropy = at::empty({rows}, f32), ids = at::empty({rows, k}, l->options().dtype(at::kInt)), top = at::empty({rows, k}, f32);
    const void *lp = l->data_ptr();
    const int *tp = ptr<const int>(tokens);
    float *ap = tokens ? (float *)logp.data_ptr() : nullptr, *ep = (float *)entropy.data_ptr(), *pp = (float *)top.data_ptr();
    int *ip = (int *)ids.data_ptr();
    const size_t stride = row_stride(l);
    const int dt = dtype_code(l);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_logprobs(stream, dt, (int)rows, (int)vocab, lp, stride, tp, (int)asked, top_k, ap, ep, ip, pp);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    PyObject *v[4] = {tokens ? THPVariable_Wrap(logp) : Py_NewRef(Py_None), THPVariable_Wrap(entropy), THPVariable_Wrap(ids), THPVariable_Wrap(top)};
    PyObject *r = v[0] && v[1] && v[2] && v[3] ? PyTuple_Pack(4, v[0], v[1], v[2], v[3]) : nullptr;
    for (PyObject *o : v) Py_XDECREF(o);
    return r;
}
/* bind(addresses of hy3a_batch_set, _append, _decode_step, _prefill, _route, _experts_workspace, _experts, _adapters_workspace, _adapters, _quantize4, _linear4, _logprobs) */
PyObject *bind(PyObject *const *a, Py_ssize_t na) {
    if (na != 12) return refuse("bind: 12 addresses");
    void *f[12];
    for (int i = 0; i < 12; i++) {
        f[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    f_batch_set = (decltype(f_batch_set))f[0]; f_append = (decltype(f_append))f[1]; f_decode_step = (decltype(f_decode_step))f[2]; f_prefill = (decltype(f_prefill))f[3];
    f_route = (decltype(f_route))f[4]; f_experts_workspace = (decltype(f_experts_workspace))f[5]; f_experts = (decltype(f_experts))f[6];
    f_adapters_workspace = (decltype(f_adapters_workspace))f[7]; f_adapters = (decltype(f_adapters))f[8];
    f_quantize4 = (decltype(f_quantize4))f[9]; f_linear4 = (decltype(f_linear4))f[10]; f_logprobs = (decltype(f_logprobs))f[11];
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))guarded<name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(batch_set), METHOD(append), METHOD(decode_step), METHOD(prefill),
                         METHOD(route), METHOD(experts), METHOD(adapters), METHOD(quantize4), METHOD(linear4), METHOD(logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods};

} /* namespace */

/* `torch_key`: the torch it was built for; the loader compares */
PyMODINIT_FUNC PyInit__native(void) {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_key", HY3A_TORCH_KEY)) Py_CLEAR(m);
    return m;
}
