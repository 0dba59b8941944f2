// Python binding of the sequence operators (include/aie_seq.h) on torch
// tensors: argument checks, outputs and scratch from torch's allocator, one C
// call.  The documented functions are ai_engine_b200/attention.py and pages.py;
// these take their arguments by position.  A call through ctypes with the
// checks in Python took 11 us of host time around the 4 us of the C call; this
// takes about 2.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <optional>

#include "../../include/aie_seq.h"

namespace {

PyObject *g_check = nullptr;  // ai_engine_b200._lib.check: raises AieError

[[noreturn]] void refuse(PyObject *type, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw python_error();
}

void check(int status, const char *where)
{
    if (status == AIE_OK) return;
    Py_XDECREF(PyObject_CallFunction(g_check, "is", status, where));
    throw python_error();
}

const at::Tensor &tensor(PyObject *o, const char *name)
{
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", name);
    return THPVariable_Unpack(o);
}

const at::Tensor *optional(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }

long long integer(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

double real(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

bool truth(PyObject *o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}

uint32_t u32(int64_t v, const char *what)
{
    if (v < 0 || v > 0xffffffffll) refuse(PyExc_ValueError, "%s is %lld", what, (long long)v);
    return (uint32_t)v;
}

int dtype_id(const at::Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return AIE_DT_F32;
    case at::kHalf: return AIE_DT_F16;
    case at::kBFloat16: return AIE_DT_BF16;
    default: return -1;
    }
}

// The operators have no backward pass; dropping a gradient without a word would
// give wrong ones.
const at::Tensor &no_grad(const at::Tensor &t, const char *name)
{
    if (t.requires_grad() && at::GradMode::is_enabled())
        refuse(PyExc_ValueError, "%s requires a gradient, which this call does not pass on: detach it, or call under "
                                 "torch.no_grad()", name);
    return t;
}

// To autograd, a tensor that a call has written is another one than it saved.
void written(const at::Tensor &t)
{
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// What the other tensors of a call have to match.
struct Like {
    at::ScalarType type;
    int device;
    int32_t dtype;
};

Like first_heads(const at::Tensor &t, const char *name)
{
    const int dt = dtype_id(t);
    if (dt < 0 || !t.is_cuda() || t.dim() != 3)
        refuse(PyExc_TypeError, "%s must be a float16, bfloat16 or float32 CUDA tensor [tokens, heads, head_dim]", name);
    return {t.scalar_type(), (int)t.get_device(), dt};
}

void same_kind(const at::Tensor &t, const char *name, const Like &l, int64_t dims)
{
    if (t.scalar_type() != l.type || !t.is_cuda() || t.get_device() != l.device || t.dim() != dims)
        refuse(PyExc_TypeError, "%s must be a %lld-D %s tensor on cuda:%d", name, (long long)dims, c10::toString(l.type),
                               l.device);
}

aie_heads heads(const at::Tensor &t, const char *name, const Like &l)
{
    same_kind(no_grad(t, name), name, l, 3);
    if (t.stride(2) != 1 && t.size(2) != 1)
        refuse(PyExc_ValueError, "%s's heads must be contiguous (stride 1 in the last dimension)", name);
    return {t.data_ptr(), t.stride(0), t.stride(1)};
}

void *vector(const at::Tensor &t, const char *name, at::ScalarType type, int device, int64_t dims = 1)
{
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != device || t.dim() != dims || !t.is_contiguous())
        refuse(PyExc_TypeError, "%s must be a contiguous %lld-D %s tensor on cuda:%d", name, (long long)dims,
                               c10::toString(type), device);
    return no_grad(t, name).data_ptr();
}

void same_shape(const at::Tensor &t, const char *name, const at::Tensor &want, const char *what)
{
    if (t.sizes() != want.sizes()) refuse(PyExc_ValueError, "%s and %s differ in shape", name, what);
}

aie_kv_pages cache(const at::Tensor &k, const at::Tensor &v, const Like &l, int64_t kv_heads, int64_t dim)
{
    same_kind(no_grad(k, "k_pages"), "k_pages", l, 4);
    same_kind(no_grad(v, "v_pages"), "v_pages", l, 4);
    if (k.sizes() != v.sizes() || k.strides() != v.strides())
        refuse(PyExc_ValueError, "k_pages and v_pages must have the same shape and strides");
    if (k.size(2) != kv_heads || k.size(3) != dim)
        refuse(PyExc_ValueError, "the cache holds %lld heads of %lld, not %lld of %lld", (long long)k.size(2),
                                (long long)k.size(3), (long long)kv_heads, (long long)dim);
    if (k.stride(3) != 1 && dim != 1) refuse(PyExc_ValueError, "a cached head must be contiguous (stride 1 in the last dimension)");
    return {k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), u32(k.size(0), "pages"), u32(k.size(1), "page_size")};
}

// The stream of a call: the given one (a torch stream or a handle) or the
// current one of the tensors' device, which becomes the current device.  Memory
// taken while this lives belongs to that stream's pool, so it is not a block
// that work queued elsewhere may still use.
class OnStream {
public:
    OnStream(PyObject *o, int device) : guard_(device), stream_(c10::cuda::getCurrentCUDAStream(device))
    {
        if (o == Py_None) return;
        PyObject *h = PyObject_HasAttrString(o, "cuda_stream") ? PyObject_GetAttrString(o, "cuda_stream") : Py_NewRef(o);
        const long long v = h ? PyLong_AsLongLong(h) : -1;
        Py_XDECREF(h);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        stream_ = c10::cuda::getStreamFromExternal((cudaStream_t)v, (c10::DeviceIndex)device);
        on_.emplace(stream_);
    }
    void *get() const { return (void *)stream_.stream(); }

private:
    c10::cuda::CUDAGuard guard_;
    c10::cuda::CUDAStream stream_;
    std::optional<c10::cuda::CUDAStreamGuard> on_;
};

// Contiguous memory straight from torch's allocator (by way of the dispatcher
// every tensor costs about 0.5 us more).
at::Tensor fresh_like(const at::Tensor &t)
{
    return at::detail::empty_cuda(t.sizes(), t.scalar_type(), t.device(), std::nullopt);
}

at::Tensor scratch(int64_t n, at::ScalarType type, int device)
{
    return at::detail::empty_cuda({n}, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

void arguments(Py_ssize_t got, Py_ssize_t want)
{
    if (got != want) refuse(PyExc_TypeError, "%lld arguments, not %lld", (long long)want, (long long)got);
}

// q, k, positions, cos_sin, q_weight, k_weight, eps, interleaved, v, k_pages, v_pages, slots, q_out, k_out, stream
PyObject *qk_norm_rope(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 15);
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &pos = tensor(a[2], "positions"), &cs = tensor(a[3], "cos_sin");
    const Like l = first_heads(q, "q");
    aie_qk_rope p = {};
    p.q = heads(q, "q", l);
    p.k = heads(k, "k", l);
    const int64_t tokens = q.size(0), d = q.size(2);
    if (k.size(0) != tokens || k.size(2) != d) refuse(PyExc_ValueError, "q and k differ in tokens or head_dim");
    p.positions = (const int32_t *)vector(pos, "positions", at::kInt, l.device);
    p.cos_sin = (const float *)vector(cs, "cos_sin", at::kFloat, l.device, 2);
    if (pos.size(0) != tokens) refuse(PyExc_ValueError, "%lld positions for %lld tokens", (long long)pos.size(0), (long long)tokens);
    for (int i = 0; i < 2; i++)
        if (const at::Tensor *w = optional(a[4 + i], "a weight")) {
            (i ? p.k_weight : p.q_weight) = (const float *)vector(*w, "a weight", at::kFloat, l.device);
            if (w->size(0) != d) refuse(PyExc_ValueError, "a weight of %lld for heads of %lld", (long long)w->size(0), (long long)d);
        }
    const at::Tensor *v = optional(a[8], "v"), *kp = optional(a[9], "k_pages"), *vp = optional(a[10], "v_pages"),
                     *slots = optional(a[11], "slots");
    const bool keep_k = a[13] != Py_False;
    if (kp) {
        if (!v || !vp || !slots) refuse(PyExc_ValueError, "filing into the cache takes v, v_pages and slots");
        p.v = heads(*v, "v", l);
        same_shape(*v, "v", k, "k");
        p.pages = cache(*kp, *vp, l, k.size(1), d);
        p.slots = (const int64_t *)vector(*slots, "slots", at::kLong, l.device);
        if (slots->size(0) != tokens) refuse(PyExc_ValueError, "%lld slots for %lld tokens", (long long)slots->size(0), (long long)tokens);
    } else if (v || vp || slots || !keep_k)
        refuse(PyExc_ValueError, "v, v_pages, slots and k_out=False go with a cache (k_pages)");
    const at::Tensor *qo = optional(a[12], "q_out"), *ko = keep_k ? optional(a[13], "k_out") : nullptr;
    OnStream on(a[14], l.device);
    const at::Tensor q_out = qo ? *qo : fresh_like(q);
    const at::Tensor k_out = ko ? *ko : keep_k ? fresh_like(k) : at::Tensor();
    same_shape(q_out, "q_out", q, "q");
    p.q_out = heads(q_out, "q_out", l);
    if (keep_k) {
        same_shape(k_out, "k_out", k, "k");
        p.k_out = heads(k_out, "k_out", l);
    }
    p.tokens = u32(tokens, "tokens");
    p.q_heads = u32(q.size(1), "q's heads");
    p.kv_heads = u32(k.size(1), "k's heads");
    p.head_dim = u32(d, "head_dim");
    p.rot_dim = u32(cs.size(1), "rot_dim");
    p.max_pos = u32(cs.size(0), "positions");
    p.dtype = l.dtype;
    p.interleaved = truth(a[7]);
    p.eps = (float)real(a[6]);
    check(aie_qk_norm_rope(&p, on.get()), "aie_qk_norm_rope");
    if (qo) written(*qo);
    if (ko) written(*ko);
    if (kp) {
        written(*kp);
        written(*vp);
    }
    PyObject *r0 = qo ? Py_NewRef(a[12]) : THPVariable_Wrap(q_out);
    PyObject *r1 = ko ? Py_NewRef(a[13]) : keep_k ? THPVariable_Wrap(k_out) : Py_NewRef(Py_None);
    return Py_BuildValue("(NN)", r0, r1);
    END_HANDLE_TH_ERRORS
}

// q, k, v, cu, causal, scale, out, stream
PyObject *prompt_attention(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 8);
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &cu = tensor(a[3], "cu");
    const Like l = first_heads(q, "q");
    aie_prompt p = {};
    p.q = heads(q, "q", l);
    p.k = heads(k, "k", l);
    p.v = heads(v, "v", l);
    if (k.size(0) != q.size(0) || k.size(2) != q.size(2)) refuse(PyExc_ValueError, "q and k differ in tokens or head_dim");
    same_shape(v, "v", k, "k");
    p.cu = (const int32_t *)vector(cu, "cu", at::kInt, l.device);
    if (cu.size(0) < 1) refuse(PyExc_ValueError, "cu holds at least one entry");
    const at::Tensor *o = optional(a[6], "out");
    OnStream on(a[7], l.device);
    const at::Tensor out = o ? *o : fresh_like(q);
    same_shape(out, "out", q, "q");
    p.out = heads(out, "out", l);
    p.tokens = u32(q.size(0), "tokens");
    p.seqs = u32(cu.size(0) - 1, "sequences");
    p.q_heads = u32(q.size(1), "q's heads");
    p.kv_heads = u32(k.size(1), "k's heads");
    p.head_dim = u32(q.size(2), "head_dim");
    p.dtype = l.dtype;
    p.causal = truth(a[4]);
    p.scale = a[5] == Py_None ? 1.f / std::sqrt((float)q.size(2)) : (float)real(a[5]);
    check(aie_prompt_attn(&p, on.get()), "aie_prompt_attn");
    if (o) written(*o);
    return o ? Py_NewRef(a[6]) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// q, k_pages, v_pages, prefix, prefix_len, table, lens, max_len, scale, out, stream
PyObject *prefix_attention(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 11);
    const at::Tensor &q = tensor(a[0], "q"), &kp = tensor(a[1], "k_pages"), &vp = tensor(a[2], "v_pages"),
                     &table = tensor(a[5], "table"), &lens = tensor(a[6], "lens");
    const Like l = first_heads(q, "q");
    aie_prefix p = {};
    p.q = heads(q, "q", l);
    p.pages = cache(kp, vp, l, kp.dim() == 4 ? kp.size(2) : 0, q.size(2));
    p.table = (const int32_t *)vector(table, "table", at::kInt, l.device, 2);
    p.lens = (const int32_t *)vector(lens, "lens", at::kInt, l.device);
    const int64_t b = q.size(0), size = p.pages.page_size, shared = integer(a[4]);
    if (table.size(0) != b || lens.size(0) != b)
        refuse(PyExc_ValueError, "%lld streams, but %lld table rows and %lld lengths", (long long)b, (long long)table.size(0),
                                (long long)lens.size(0));
    if (shared < 0) refuse(PyExc_ValueError, "prefix_len is %lld", (long long)shared);
    if (shared) {
        const at::Tensor &prefix = tensor(a[3], "prefix");
        p.prefix = (const int32_t *)vector(prefix, "prefix", at::kInt, l.device);
        if (prefix.size(0) * size < shared)
            refuse(PyExc_ValueError, "%lld pages of %lld do not hold a prefix of %lld", (long long)prefix.size(0), (long long)size,
                                    (long long)shared);
    }
    const int64_t top = a[7] == Py_None ? std::max(table.size(1) * size, shared) : integer(a[7]);
    const at::Tensor *o = optional(a[9], "out");
    OnStream on(a[10], l.device);
    const at::Tensor out = o ? *o : fresh_like(q);
    same_shape(out, "out", q, "q");
    p.out = heads(out, "out", l);
    p.batch = u32(b, "the batch");
    p.q_heads = u32(q.size(1), "q's heads");
    p.kv_heads = u32(kp.size(2), "the cache's heads");
    p.head_dim = u32(q.size(2), "head_dim");
    p.prefix_len = u32(shared, "prefix_len");
    p.max_len = u32(top, "max_len");
    p.table_stride = u32(table.size(1), "the table's width");
    p.dtype = l.dtype;
    p.scale = a[8] == Py_None ? 1.f / std::sqrt((float)q.size(2)) : (float)real(a[8]);
    p.workspace_bytes = std::max<uint64_t>(aie_prefix_attn_workspace(&p), 16);
    const at::Tensor ws = scratch((int64_t)p.workspace_bytes, at::kByte, l.device);
    p.workspace = ws.data_ptr();
    check(aie_prefix_attn(&p, on.get()), "aie_prefix_attn");
    if (o) written(*o);
    return o ? Py_NewRef(a[9]) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// ---- pages

// kv into p; its device
int pack_kv(PyObject *o, aie_pages &p)
{
    const at::Tensor &kv = no_grad(tensor(o, "kv"), "kv");
    if (dtype_id(kv) < 0 || !kv.is_cuda() || kv.dim() != 6 || kv.size(1) != 2 || !kv.is_contiguous())
        refuse(PyExc_TypeError, "kv must be a contiguous float16, bfloat16 or float32 CUDA tensor "
                               "[layers, 2, pages, page_size, kv_heads, head_dim]");
    p.kv = kv.data_ptr();
    p.layers = u32(kv.size(0), "layers");
    p.pages = u32(kv.size(2), "pages");
    p.page_size = u32(kv.size(3), "page_size");
    p.page_bytes = (uint64_t)(kv.size(3) * kv.size(4) * kv.size(5) * kv.element_size());
    return (int)kv.get_device();
}

// the state (refs, lens, table, status) into p; its device
int pack_state(PyObject *o, aie_pages &p)
{
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse(PyExc_TypeError, "the state is a PageState");
    const at::Tensor &refs = tensor(PyTuple_GET_ITEM(o, 0), "refs"), &lens = tensor(PyTuple_GET_ITEM(o, 1), "lens"),
                     &table = tensor(PyTuple_GET_ITEM(o, 2), "table"), &status = tensor(PyTuple_GET_ITEM(o, 3), "status");
    const int device = refs.is_cuda() ? (int)refs.get_device() : -1;
    p.refs = (int32_t *)vector(refs, "refs", at::kInt, device);
    p.lens = (int32_t *)vector(lens, "lens", at::kInt, device);
    p.table = (int32_t *)vector(table, "table", at::kInt, device, 2);
    p.status = (int32_t *)vector(status, "status", at::kInt, device);
    if (table.size(0) != lens.size(0) || status.size(0) != 1)
        refuse(PyExc_ValueError, "the state is refs [pages], lens [rows], table [rows, width] and status [1]");
    if (p.kv && (int64_t)p.pages != refs.size(0))
        refuse(PyExc_ValueError, "kv has %u pages, the state %lld", p.pages, (long long)refs.size(0));
    p.pages = u32(refs.size(0), "pages");
    p.rows = u32(lens.size(0), "rows");
    p.width = u32(table.size(1), "a table row");
    return device;
}

void written_state(PyObject *o)
{
    for (int i = 0; i < 4; i++) written(THPVariable_Unpack(PyTuple_GET_ITEM(o, i)));
}

uint32_t lists(PyObject *a, PyObject *b, const char *what, int device, const int32_t **x, const int32_t **y)
{
    const at::Tensor &s = tensor(a, what), &t = tensor(b, what);
    *x = (const int32_t *)vector(s, what, at::kInt, device);
    *y = (const int32_t *)vector(t, what, at::kInt, device);
    if (s.size(0) != t.size(0)) refuse(PyExc_ValueError, "%s differ in length: %lld and %lld", what, (long long)s.size(0), (long long)t.size(0));
    return u32(s.size(0), what);
}

at::Tensor page_scratch(aie_pages &p, uint32_t n, int device)
{
    const at::Tensor ws = scratch((int64_t)aie_pages_workspace(p.pages, n) / 4, at::kInt, device);
    p.workspace = (int32_t *)ws.data_ptr();
    return ws;
}

// state, page_size, rows, counts, tokens, stream
PyObject *pages_grow(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 6);
    aie_pages p = {};
    const int device = pack_state(a[0], p);
    p.page_size = u32(integer(a[1]), "page_size");
    const int32_t *rows, *counts;
    const uint32_t count = lists(a[2], a[3], "rows and counts", device, &rows, &counts), tokens = u32(integer(a[4]), "tokens");
    OnStream on(a[5], device);
    const at::Tensor ws = page_scratch(p, count, device), slots = scratch(tokens, at::kLong, device);
    check(aie_pages_grow(&p, rows, counts, count, (int64_t *)slots.data_ptr(), tokens, on.get()), "aie_pages_grow");
    written_state(a[0]);
    return THPVariable_Wrap(slots);
    END_HANDLE_TH_ERRORS
}

// kv, state, src, dst, stream
PyObject *pages_fork(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 5);
    aie_pages p = {};
    const int device = pack_kv(a[0], p);
    if (pack_state(a[1], p) != device) refuse(PyExc_ValueError, "kv and the state are on different devices");
    const int32_t *src, *dst;
    const uint32_t count = lists(a[2], a[3], "src and dst", device, &src, &dst);
    OnStream on(a[4], device);
    const at::Tensor ws = page_scratch(p, count, device);
    check(aie_pages_fork(&p, src, dst, count, on.get()), "aie_pages_fork");
    written(THPVariable_Unpack(a[0]));
    written_state(a[1]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// kv, src, dst, stream
PyObject *pages_copy(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 4);
    aie_pages p = {};
    const int device = pack_kv(a[0], p);
    const int32_t *src, *dst;
    const uint32_t count = lists(a[1], a[2], "src and dst", device, &src, &dst);
    OnStream on(a[3], device);
    check(aie_pages_copy(&p, src, dst, count, on.get()), "aie_pages_copy");
    written(THPVariable_Unpack(a[0]));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// state, rows, stream
PyObject *pages_free(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 3);
    aie_pages p = {};
    const int device = pack_state(a[0], p);
    const at::Tensor &rows = tensor(a[1], "rows");
    const int32_t *list = (const int32_t *)vector(rows, "rows", at::kInt, device);
    OnStream on(a[2], device);
    check(aie_pages_free(&p, list, u32(rows.size(0), "rows"), on.get()), "aie_pages_free");
    written_state(a[0]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// kv, state, stream
PyObject *pages_compact(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    arguments(n, 3);
    aie_pages p = {};
    const int device = pack_kv(a[0], p);
    if (pack_state(a[1], p) != device) refuse(PyExc_ValueError, "kv and the state are on different devices");
    OnStream on(a[2], device);
    const at::Tensor ws = page_scratch(p, 0, device), remap = scratch(p.pages, at::kInt, device);
    check(aie_pages_compact(&p, (int32_t *)remap.data_ptr(), on.get()), "aie_pages_compact");
    written(THPVariable_Unpack(a[0]));
    written_state(a[1]);
    return THPVariable_Wrap(remap);
    END_HANDLE_TH_ERRORS
}

#define FN(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FN(qk_norm_rope), FN(prompt_attention), FN(prefix_attention), FN(pages_grow), FN(pages_fork),
                         FN(pages_copy),   FN(pages_free),       FN(pages_compact),    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_seqcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__seqcall(void)
{
    PyObject *lib = PyImport_ImportModule("ai_engine_b200._lib");
    if (!lib) return nullptr;
    g_check = PyObject_GetAttrString(lib, "check");
    Py_DECREF(lib);
    return g_check ? PyModule_Create(&module) : nullptr;
}
