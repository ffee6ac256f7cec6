// w4a8_native.cpp -- a short way from Python to the C entry points of the operators
// that decode steps call most: norm, cache write and read, attention, 8-bit linears, rotary
// positions, pages.
//
// The Python wrappers (ops.py, kvcache.py) read some thirty tensor attributes a call
// to check their arguments, which costs more than such a call's kernels run.  These
// functions do the same checks on the tensors themselves, allocate the outputs and
// call the C ABI.  They take the well-formed common case only -- exact torch tensors on
// the current GPU, dense, 16-byte aligned -- and return NotImplemented for everything else, a refusal
// by the C entry point included; the wrapper then goes the long way, with its
// messages, copies and strided forms.  Results are the same either way.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "w4a8_b200.h"

namespace {

// Entry points of the library that the package loaded (bind()).
struct Table {
    decltype(&w4a8_rms_norm) rms_norm;
    decltype(&w4a8_rms_norm_quant) rms_norm_quant;
    decltype(&w4a8_kv_write) kv_write;
    decltype(&w4a8_kv_read) kv_read;
    decltype(&w4a8_attention) attention;
    decltype(&w4a8_int8_linear) int8_linear;
    decltype(&w4a8_int8_linear_rms_norm) int8_linear_rms_norm;
    decltype(&w4a8_rotary) rotary;
    decltype(&w4a8_pages_plan) pages_plan;
    decltype(&w4a8_pages_shrink) pages_shrink;
} g{};

PyObject* later()
{
    Py_INCREF(Py_NotImplemented);
    return Py_NotImplemented;
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool is(const at::Tensor* t, at::ScalarType type, int dev, int64_t dims)
{
    return t && t->is_cuda() && t->scalar_type() == type && t->get_device() == dev && t->dim() == dims;
}

// The library launches on the current GPU; the long way makes the tensors' one current.
bool current(int dev) { return c10::cuda::current_device() == dev; }

bool dense(const at::Tensor* t, at::ScalarType type, int dev, int64_t dims) { return is(t, type, dev, dims) && t->is_contiguous(); }

at::Tensor make(at::IntArrayRef size, at::ScalarType type, int dev)
{
    return at::detail::empty_cuda(size, type, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt);
}

void* stream(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

PyObject* pair(PyObject* a, PyObject* b)
{
    if (!a || !b) {
        Py_XDECREF(a);
        Py_XDECREF(b);
        return nullptr;
    }
    PyObject* r = PyTuple_Pack(2, a, b);
    Py_DECREF(a);
    Py_DECREF(b);
    return r;
}

// Rows of a norm call: x, weight and (unless None) residual, dense, of one shape.
struct Rows {
    const at::Tensor *x, *w, *r;
    int64_t M, K;
    int dev, wd;
};

bool rows(PyObject* const* a, Rows& n)
{
    n.x = tensor(a[0]);
    n.w = tensor(a[1]);
    if (!n.x || !n.w || !n.x->is_cuda() || n.x->dim() < 1 || n.x->scalar_type() != at::kBFloat16 || !n.x->is_contiguous())
        return false;
    n.dev = n.x->get_device();
    n.K = n.x->size(-1);
    if (n.K < 1 || !n.w->is_cuda() || n.w->get_device() != n.dev || n.w->dim() != 1 || n.w->size(0) != n.K ||
        !n.w->is_contiguous())
        return false;
    if (n.w->scalar_type() == at::kBFloat16) n.wd = W4A8_DTYPE_BF16;
    else if (n.w->scalar_type() == at::kFloat) n.wd = W4A8_DTYPE_F32;
    else return false;
    n.r = nullptr;
    if (a[2] != Py_None) {
        n.r = tensor(a[2]);
        if (!dense(n.r, at::kBFloat16, n.dev, n.x->dim()) || n.r->sizes() != n.x->sizes()) return false;
    }
    n.M = n.x->numel() / n.K;
    return current(n.dev);
}

const void* ptr(const at::Tensor* t) { return t ? t->const_data_ptr() : nullptr; }

// rms_norm(x, weight, residual or None, eps)
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    Rows t;
    if (n != 4 || !PyFloat_Check(a[3]) || !g.rms_norm || !rows(a, t)) return later();
    at::Tensor y = make(t.x->sizes(), at::kBFloat16, t.dev), ro;
    if (t.r) ro = make(t.x->sizes(), at::kBFloat16, t.dev);
    const int rc = g.rms_norm(ptr(t.x), t.M, t.K, t.K, ptr(t.r), t.r ? t.K : 0, t.r ? ro.data_ptr() : nullptr, t.r ? t.K : 0,
                              ptr(t.w), t.wd, static_cast<float>(PyFloat_AS_DOUBLE(a[3])), y.data_ptr(), t.K, stream(t.dev));
    if (rc != W4A8_OK) return later();
    return t.r ? pair(wrap(y), wrap(ro)) : wrap(y);
}

// rms_norm_quant(x, weight, residual or None, eps, group_size, scale dtype)
PyObject* rms_norm_quant(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    Rows t;
    if (n != 6 || !PyFloat_Check(a[3]) || !PyLong_Check(a[4]) || !g.rms_norm_quant || !rows(a, t) || t.x->dim() != 2) return later();
    const long gk = PyLong_AsLong(a[4]);
    if (gk <= 0 || gk > 65536) {
        PyErr_Clear();
        return later();
    }
    if (!THPDtype_Check(a[5])) return later();
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    if (type != at::kFloat && type != at::kBFloat16) return later();
    at::Tensor q = make({t.M, t.K}, at::kChar, t.dev), ro;
    at::Tensor s = make({(t.K + gk - 1) / gk, t.M}, type, t.dev);
    if (t.r) ro = make(t.x->sizes(), at::kBFloat16, t.dev);
    const int rc = g.rms_norm_quant(ptr(t.x), t.M, t.K, t.K, ptr(t.r), t.r ? t.K : 0, t.r ? ro.data_ptr() : nullptr,
                                    t.r ? t.K : 0, ptr(t.w), t.wd, static_cast<float>(PyFloat_AS_DOUBLE(a[3])),
                                    static_cast<int32_t>(gk), static_cast<int8_t*>(q.data_ptr()), s.data_ptr(),
                                    type == at::kFloat ? W4A8_DTYPE_F32 : W4A8_DTYPE_BF16, stream(t.dev));
    if (rc != W4A8_OK) return later();
    PyObject* pq = wrap(q);
    PyObject* ps = wrap(s);
    PyObject* pr = t.r ? wrap(ro) : Py_NewRef(Py_None);
    if (!pq || !ps || !pr) {
        Py_XDECREF(pq);
        Py_XDECREF(ps);
        Py_XDECREF(pr);
        return nullptr;
    }
    PyObject* r = PyTuple_Pack(3, pq, ps, pr);
    Py_DECREF(pq);
    Py_DECREF(ps);
    Py_DECREF(pr);
    return r;
}

// The cache's descriptor and device, and the batch tensors, from four arguments on.
struct Batch {
    const w4a8_kv_cache* cache;
    int dev;
    const at::Tensor *table, *lens, *cu;
    int64_t B, cols;
};

bool batch(PyObject* const* a, Batch& b)
{
    if (!PyLong_Check(a[0]) || !PyLong_Check(a[1])) return false;
    b.cache = static_cast<const w4a8_kv_cache*>(PyLong_AsVoidPtr(a[0]));
    b.dev = static_cast<int>(PyLong_AsLong(a[1]));
    b.table = tensor(a[2]);
    b.lens = tensor(a[3]);
    b.cu = tensor(a[4]);
    if (!b.cache || !dense(b.table, at::kInt, b.dev, 2) || !dense(b.lens, at::kInt, b.dev, 1) || !dense(b.cu, at::kInt, b.dev, 1))
        return false;
    b.B = b.lens->size(0);
    b.cols = b.table->size(1);
    return b.B > 0 && b.table->size(0) == b.B && b.cu->size(0) == b.B + 1 && current(b.dev);
}

// bf16 [tokens, heads, head_dim] with dense heads and 16-byte rows; its row stride.
bool heads(const at::Tensor* t, const Batch& b, int64_t& ld)
{
    if (!is(t, at::kBFloat16, b.dev, 3) || t->size(2) != b.cache->head_dim || t->size(0) == 0 || t->size(1) == 0) return false;
    ld = t->stride(0);
    return t->stride(2) == 1 && (t->stride(1) == b.cache->head_dim || t->size(1) == 1) && ld % 8 == 0 &&
           ld >= t->size(1) * t->size(2) && reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0;
}

const int32_t* ints(const at::Tensor* t) { return static_cast<const int32_t*>(t->const_data_ptr()); }

// kv_write(cache, device, page_table, kv_lens, cu, k, v, q or None, cos_sin or None, interleaved)
PyObject* kv_write(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    Batch b;
    if (n != 10 || !g.kv_write || !batch(a, b)) return later();
    const at::Tensor *k = tensor(a[5]), *v = tensor(a[6]), *q = nullptr, *cs = nullptr;
    int64_t ldk = 0, ldv = 0, ldq = 0;
    if (!heads(k, b, ldk) || !heads(v, b, ldv) || k->size(1) != b.cache->kv_heads || v->sizes() != k->sizes()) return later();
    at::Tensor out;
    if (a[7] != Py_None) {
        q = tensor(a[7]);
        if (!heads(q, b, ldq) || q->size(0) != k->size(0)) return later();
        out = make(q->sizes(), at::kBFloat16, b.dev);
    }
    if (a[8] != Py_None) {
        cs = tensor(a[8]);
        // (an empty table's null pointer would mean "no rotary" to the C call)
        if (!dense(cs, at::kFloat, b.dev, 2) || cs->numel() == 0) return later();
    }
    const int interleaved = PyObject_IsTrue(a[9]);
    if (interleaved < 0) {
        PyErr_Clear();
        return later();
    }
    const int rc = g.kv_write(b.cache, ints(b.table), b.cols, b.cols, ints(b.lens), ints(b.cu), b.B, k->size(0), ptr(k), ldk,
                              ptr(v), ldv, ptr(q), ldq, q ? static_cast<int32_t>(q->size(1)) : 0, q ? out.data_ptr() : nullptr,
                              q ? q->size(1) * q->size(2) : 0, static_cast<const float*>(ptr(cs)), cs ? cs->size(0) : 0,
                              cs ? static_cast<int32_t>(cs->size(1)) : 0, interleaved, stream(b.dev));
    if (rc != W4A8_OK) return later();
    return q ? wrap(out) : Py_NewRef(Py_None);
}

// kv_read(cache, device, page_table, kv_lens, cu, tokens)
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    Batch b;
    if (n != 6 || !g.kv_read || !batch(a, b) || !PyLong_Check(a[5])) return later();
    const int64_t tokens = PyLong_AsLongLong(a[5]);
    if (tokens <= 0) {
        PyErr_Clear();
        return later();
    }
    at::Tensor k = make({tokens, b.cache->kv_heads, b.cache->head_dim}, at::kBFloat16, b.dev);
    at::Tensor v = make({tokens, b.cache->kv_heads, b.cache->head_dim}, at::kBFloat16, b.dev);
    const int rc = g.kv_read(b.cache, ints(b.table), b.cols, b.cols, ints(b.lens), ints(b.cu), b.B, tokens, k.data_ptr(),
                             v.data_ptr(), stream(b.dev));
    return rc == W4A8_OK ? pair(wrap(k), wrap(v)) : later();
}

// attention(cache, device, page_table, kv_lens, cu, q, max_q_len, scale, workspace, workspace bytes)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    Batch b;
    if (n != 10 || !g.attention || !batch(a, b) || !PyLong_Check(a[6]) || !PyFloat_Check(a[7]) || !PyLong_Check(a[8]) ||
        !PyLong_Check(a[9]))
        return later();
    const at::Tensor* q = tensor(a[5]);
    int64_t ldq = 0;
    const long mq = PyLong_AsLong(a[6]);
    if (mq <= 0 || mq > 0x7FFFFFFF || !heads(q, b, ldq)) {
        PyErr_Clear();
        return later();
    }
    at::Tensor out = make(q->sizes(), at::kBFloat16, b.dev);
    const int rc = g.attention(b.cache, ints(b.table), b.cols, b.cols, ints(b.lens), ints(b.cu), b.B, q->size(0), ptr(q), ldq,
                               static_cast<int32_t>(q->size(1)), static_cast<int32_t>(mq),
                               static_cast<float>(PyFloat_AS_DOUBLE(a[7])), out.data_ptr(), q->size(1) * q->size(2),
                               PyLong_AsVoidPtr(a[8]), static_cast<size_t>(PyLong_AsUnsignedLongLong(a[9])), stream(b.dev));
    return rc == W4A8_OK ? wrap(out) : later();
}

// An 8-bit layer (_lib.Int8LayerDesc).
struct Layer {
    const int8_t* w;
    const float *scale, *bias;
    int64_t N, K, ldw;
};

const Layer* layer_of(PyObject* o) { return PyLong_Check(o) ? static_cast<const Layer*>(PyLong_AsVoidPtr(o)) : nullptr; }

at::Tensor outputs(const at::Tensor* x, int64_t N, int dev)
{
    if (x->dim() == 2) return make({x->size(0), N}, at::kBFloat16, dev);
    std::vector<int64_t> size(x->sizes().begin(), x->sizes().end());
    size.back() = N;
    return make(size, at::kBFloat16, dev);
}

// linear_int8(layer, device, x, act, workspace, workspace bytes)
PyObject* linear_int8(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (n != 6 || !g.int8_linear || !PyLong_Check(a[1]) || !PyLong_Check(a[3]) || !PyLong_Check(a[4]) || !PyLong_Check(a[5])) return later();
    const Layer* L = layer_of(a[0]);
    const int dev = static_cast<int>(PyLong_AsLong(a[1])), act = static_cast<int>(PyLong_AsLong(a[3]));
    const at::Tensor* x = tensor(a[2]);
    if (!L || !x || x->dim() < 1 || !dense(x, at::kBFloat16, dev, x->dim()) || !current(dev)) return later();
    const int64_t wide = act == W4A8_ACT_SWIGLU ? 2 * L->K : L->K;
    if (x->size(-1) != wide || x->numel() == 0) return later();
    at::Tensor y = outputs(x, L->N, dev);
    const int rc = g.int8_linear(ptr(x), x->numel() / wide, L->K, wide, act, L->w, L->ldw, L->scale, L->bias, L->N, y.data_ptr(), L->N,
                                 PyLong_AsVoidPtr(a[4]), static_cast<size_t>(PyLong_AsUnsignedLongLong(a[5])), stream(dev));
    return rc == W4A8_OK ? wrap(y) : later();
}

// linear_int8_rms_norm(x, weight, residual or None, eps, layer, workspace, workspace bytes)
PyObject* linear_int8_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    Rows t;
    if (n != 7 || !PyFloat_Check(a[3]) || !PyLong_Check(a[5]) || !PyLong_Check(a[6]) || !g.int8_linear_rms_norm || !rows(a, t)) return later();
    const Layer* L = layer_of(a[4]);
    if (!L || L->K != t.K || t.M == 0) return later();
    at::Tensor y = outputs(t.x, L->N, t.dev), ro;
    if (t.r) ro = make(t.x->sizes(), at::kBFloat16, t.dev);
    const int rc = g.int8_linear_rms_norm(ptr(t.x), t.M, t.K, t.K, ptr(t.r), t.r ? t.K : 0, t.r ? ro.data_ptr() : nullptr,
                                          t.r ? t.K : 0, ptr(t.w), t.wd, static_cast<float>(PyFloat_AS_DOUBLE(a[3])), L->w, L->ldw,
                                          L->scale, L->bias, L->N, y.data_ptr(), L->N, PyLong_AsVoidPtr(a[5]),
                                          static_cast<size_t>(PyLong_AsUnsignedLongLong(a[6])), stream(t.dev));
    if (rc != W4A8_OK) return later();
    return t.r ? pair(wrap(y), wrap(ro)) : wrap(y);
}

// [tokens, heads, D] with dense heads and 16-byte rows; its row stride.
bool plain_heads(const at::Tensor* t, int dev, int64_t D, int64_t& ld)
{
    if (!is(t, at::kBFloat16, dev, 3) || t->size(2) != D || t->size(0) == 0 || t->size(1) == 0) return false;
    ld = t->stride(0);
    return t->stride(2) == 1 && (t->stride(1) == D || t->size(1) == 1) && ld % 8 == 0 && ld >= t->size(1) * D &&
           reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0;
}

// rotary(q, k or None, cos_sin, positions, axes, pairs, axis of each pair or 0, interleaved)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (n != 8 || !g.rotary || !PyLong_Check(a[4]) || !PyLong_Check(a[5]) || !PyLong_Check(a[6])) return later();
    const at::Tensor *q = tensor(a[0]), *k = nullptr, *cs = tensor(a[2]), *pos = tensor(a[3]);
    if (!q || !q->is_cuda() || q->dim() != 3) return later();
    const int dev = q->get_device(), axes = static_cast<int>(PyLong_AsLong(a[4]));
    const int64_t D = q->size(2), T = q->size(0);
    int64_t ldq = 0, ldk = 0;
    if (!plain_heads(q, dev, D, ldq) || !current(dev)) return later();
    if (a[1] != Py_None) {
        k = tensor(a[1]);
        if (!plain_heads(k, dev, D, ldk) || k->size(0) != T) return later();
    }
    if (!dense(cs, at::kFloat, dev, 2) || cs->numel() == 0 || cs->size(1) != 2 * PyLong_AsLong(a[5])) return later();
    if (!dense(pos, at::kInt, dev, 2) || pos->size(0) != axes || pos->size(1) != T) return later();
    const int interleaved = PyObject_IsTrue(a[7]);
    if (interleaved < 0) {
        PyErr_Clear();
        return later();
    }
    at::Tensor qo = make(q->sizes(), at::kBFloat16, dev), ko;
    if (k) ko = make(k->sizes(), at::kBFloat16, dev);
    const int rc = g.rotary(ptr(q), ldq, static_cast<int32_t>(q->size(1)), qo.data_ptr(), q->size(1) * D, ptr(k), ldk,
                            k ? static_cast<int32_t>(k->size(1)) : 0, k ? ko.data_ptr() : nullptr, k ? k->size(1) * D : 0, T,
                            static_cast<int32_t>(D), static_cast<const float*>(ptr(cs)), cs->size(0),
                            static_cast<int32_t>(cs->size(1)), interleaved, ints(pos), T, axes,
                            static_cast<const uint8_t*>(PyLong_AsVoidPtr(a[6])), stream(dev));
    if (rc != W4A8_OK) return later();
    return pair(wrap(qo), k ? wrap(ko) : Py_NewRef(Py_None));
}

// pages_plan(state, device, rows, counts, tokens, axes, seg_cu or None, segs or None)
PyObject* pages_plan(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (n != 8 || !g.pages_plan || !PyLong_Check(a[0]) || !PyLong_Check(a[1]) || !PyLong_Check(a[4]) || !PyLong_Check(a[5])) return later();
    const w4a8_page_state* st = static_cast<const w4a8_page_state*>(PyLong_AsVoidPtr(a[0]));
    const int dev = static_cast<int>(PyLong_AsLong(a[1]));
    const int64_t tokens = PyLong_AsLongLong(a[4]), axes = PyLong_AsLongLong(a[5]);
    const at::Tensor *rows = tensor(a[2]), *counts = tensor(a[3]), *cu = nullptr, *segs = nullptr;
    if (!st || tokens < 0 || axes < 1 || axes > 4 || !dense(rows, at::kInt, dev, 1) || !dense(counts, at::kInt, dev, 1) || !current(dev)) {
        PyErr_Clear();
        return later();
    }
    const int64_t B = rows->size(0);
    if (counts->size(0) != B || B > W4A8_PLAN_MAX_BATCH) return later();
    if (a[6] != Py_None) {
        cu = tensor(a[6]);
        segs = tensor(a[7]);
        if (axes != 3 || !dense(cu, at::kInt, dev, 1) || !dense(segs, at::kInt, dev, 2) || cu->size(0) != B + 1 || segs->size(1) != 4)
            return later();
    }
    // the outputs are parts of one allocation, each from a multiple of 16 bytes on
    const int64_t wide[5] = {B * st->columns, B, B + 1, tokens, axes * tokens};
    int64_t at_[5], total = 0;
    for (int i = 0; i < 5; ++i) {
        at_[i] = total;
        total += (wide[i] + 3) / 4 * 4;
    }
    const at::Tensor whole = make({total}, at::kInt, dev);
    const auto part = [&](int i, at::IntArrayRef size) {
        auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
        impl->set_storage_offset(at_[i]);
        impl->set_sizes_contiguous(size);
        return at::Tensor(std::move(impl));
    };
    const at::Tensor out[5] = {part(0, {B, st->columns}), part(1, {B}), part(2, {B + 1}), part(3, {tokens}), part(4, {axes, tokens})};
    int32_t* p[5];
    for (int i = 0; i < 5; ++i) p[i] = static_cast<int32_t*>(whole.data_ptr()) + at_[i];
    const int rc = g.pages_plan(st, ints(rows), ints(counts), B, tokens, static_cast<int32_t>(axes), cu ? ints(cu) : nullptr,
                                segs ? ints(segs) : nullptr, segs ? segs->size(0) : 0, p[0], p[1], p[2], p[3], p[4], stream(dev));
    if (rc != W4A8_OK) return later();
    PyObject* r = PyTuple_New(5);
    for (int i = 0; r && i < 5; ++i) {
        PyObject* o = wrap(out[i]);
        if (!o) {
            Py_DECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, i, o);
    }
    return r;
}

// pages_shrink(state, device, rows, keep or None): True
PyObject* pages_shrink(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (n != 4 || !g.pages_shrink || !PyLong_Check(a[0]) || !PyLong_Check(a[1])) return later();
    const int dev = static_cast<int>(PyLong_AsLong(a[1]));
    const at::Tensor *rows = tensor(a[2]), *keep = nullptr;
    if (!dense(rows, at::kInt, dev, 1) || !current(dev)) return later();
    if (a[3] != Py_None) {
        keep = tensor(a[3]);
        if (!dense(keep, at::kInt, dev, 1) || keep->size(0) != rows->size(0)) return later();
    }
    const int rc = g.pages_shrink(static_cast<const w4a8_page_state*>(PyLong_AsVoidPtr(a[0])), ints(rows), keep ? ints(keep) : nullptr,
                                  rows->size(0), stream(dev));
    return rc == W4A8_OK ? Py_NewRef(Py_True) : later();
}

// C++ exceptions (an allocation that fails) become Python ones.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    try {
        return F(self, a, n);
    } catch (const c10::OutOfMemoryError&) {
        return later();                              // the long way raises torch's own error
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// Addresses of entry points, in order.
bool addresses(PyObject* const* a, Py_ssize_t n, void* (&p)[5])
{
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "bind: five addresses");
        return false;
    }
    for (int i = 0; i < 5; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
            return false;
        }
    }
    return true;
}

// bind(rms_norm, rms_norm_quant, kv_write, kv_read, attention)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    void* p[5];
    if (!addresses(a, n, p)) return nullptr;
    g.rms_norm = reinterpret_cast<decltype(g.rms_norm)>(p[0]);
    g.rms_norm_quant = reinterpret_cast<decltype(g.rms_norm_quant)>(p[1]);
    g.kv_write = reinterpret_cast<decltype(g.kv_write)>(p[2]);
    g.kv_read = reinterpret_cast<decltype(g.kv_read)>(p[3]);
    g.attention = reinterpret_cast<decltype(g.attention)>(p[4]);
    Py_RETURN_NONE;
}

// bind_more(int8_linear, int8_linear_rms_norm, rotary, pages_plan, pages_shrink)
PyObject* bind_more(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    void* p[5];
    if (!addresses(a, n, p)) return nullptr;
    g.int8_linear = reinterpret_cast<decltype(g.int8_linear)>(p[0]);
    g.int8_linear_rms_norm = reinterpret_cast<decltype(g.int8_linear_rms_norm)>(p[1]);
    g.rotary = reinterpret_cast<decltype(g.rotary)>(p[2]);
    g.pages_plan = reinterpret_cast<decltype(g.pages_plan)>(p[3]);
    g.pages_shrink = reinterpret_cast<decltype(g.pages_shrink)>(p[4]);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction entry()
{
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<F>));
}

PyMethodDef methods[] = {{"bind", entry<bind>(), METH_FASTCALL, nullptr},
                         {"bind_more", entry<bind_more>(), METH_FASTCALL, nullptr},
                         {"rms_norm", entry<rms_norm>(), METH_FASTCALL, nullptr},
                         {"rms_norm_quant", entry<rms_norm_quant>(), METH_FASTCALL, nullptr},
                         {"kv_write", entry<kv_write>(), METH_FASTCALL, nullptr},
                         {"kv_read", entry<kv_read>(), METH_FASTCALL, nullptr},
                         {"attention", entry<attention>(), METH_FASTCALL, nullptr},
                         {"linear_int8", entry<linear_int8>(), METH_FASTCALL, nullptr},
                         {"linear_int8_rms_norm", entry<linear_int8_rms_norm>(), METH_FASTCALL, nullptr},
                         {"rotary", entry<rotary>(), METH_FASTCALL, nullptr},
                         {"pages_plan", entry<pages_plan>(), METH_FASTCALL, nullptr},
                         {"pages_shrink", entry<pages_shrink>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__native() { return PyModule_Create(&module); }
