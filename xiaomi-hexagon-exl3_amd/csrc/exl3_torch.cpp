// exl3_torch.cpp -- the C-ABI of the attention and linear-attention blocks for torch tensors, as a CPython module.
//
// Through ctypes, with views, checks and allocations in Python, the host time of a call is several
// times its kernel's at decode sizes: one token's qk_norm_rope took 16.8 us a call, here 5.2; a cache
// write and read of eight tokens 24.3, here 9.2.  The module
// holds no state and no kernels: every function ends in one exl3_hip_* call.  A refused
// argument raises AssertionError; a status other than EXL3_OK is returned as an int.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <stdexcept>

#include "exl3_hip.h"

namespace {

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void need(bool ok, const char *what) {
    if (!ok) throw Refused(what);
}

bool given(PyObject *o) { return o && o != Py_None; }

// One call: its device is that of its first tensor, which all others share.  on() makes that device and the call's
// stream current until the call ends, so that outputs come from the memory pool of the stream that writes them: from
// another stream's pool they could be memory that this stream's earlier work still reads, or that a later
// allocation gets while this call's kernel still writes it.
struct Call {
    c10::DeviceIndex device = -1;
    std::optional<c10::hip::HIPGuard> on_device;
    std::optional<c10::hip::HIPStreamGuard> on_stream;
    hipStream_t stream = nullptr;

    const at::Tensor &tensor(PyObject *o, const char *what) {
        need(THPVariable_Check(o), what);
        const at::Tensor &t = THPVariable_Unpack(o);
        need(t.is_cuda(), "tensors must be on a HIP device");
        if (device < 0) device = t.get_device();
        need(t.get_device() == device, "tensors are on different devices");
        return t;
    }

    // stream: a torch.cuda.Stream (or what has its cuda_stream), None: the device's current one
    void on(PyObject *o) {
        if (!given(o)) {
            if (c10::hip::current_device() != device) on_device.emplace(device);
            stream = c10::hip::getCurrentHIPStream(device).stream();
            return;
        }
        PyObject *raw = PyObject_GetAttrString(o, "cuda_stream");
        if (!raw) throw python_error();
        void *p = PyLong_AsVoidPtr(raw);
        Py_DECREF(raw);
        if (!p && PyErr_Occurred()) throw python_error();
        if (PyObject *index = PyObject_GetAttrString(o, "device_index")) {
            const long i = PyLong_AsLong(index);
            Py_DECREF(index);
            if (i == -1 && PyErr_Occurred()) throw python_error();
            need(i == device, "the stream is of another device than the tensors");
        } else {
            PyErr_Clear();
        }
        stream = (hipStream_t)p;
        on_stream.emplace(p ? c10::hip::getStreamFromExternal(stream, device) : c10::hip::getDefaultHIPStream(device));
    }

    // a dense vector (or matrix) of `count` elements of one type; NULL where it may be left out
    void *dense(PyObject *o, at::ScalarType type, int64_t count, const char *what, bool optional = false) {
        if (optional && !given(o)) return nullptr;
        const at::Tensor &t = tensor(o, what);
        need(t.scalar_type() == type && t.is_contiguous() && (count < 0 || t.numel() == count), what);
        return t.data_ptr();
    }

    at::Tensor output(PyObject *o, at::IntArrayRef shape, at::ScalarType type) {
        if (given(o)) {
            const at::Tensor &t = tensor(o, "out is a tensor");
            need(t.sizes() == shape, "out has another shape");
            return t;
        }
        // at::empty without its dispatch
        return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, device), std::nullopt);
    }

    void *workspace(PyObject *o, size_t *bytes) {  // None: the library's own
        *bytes = 0;
        if (!given(o)) return nullptr;
        const at::Tensor &t = tensor(o, "workspace is a tensor");
        *bytes = t.nbytes();
        return t.data_ptr();
    }
};

// rows of heads [tokens, heads, head_dim], F16 or F32, a head's elements dense (of no elements, any strides)
exl3_head_view heads(const at::Tensor &t) {
    need(t.dim() == 3, "rows of heads are [tokens, heads, head_dim]");
    need(t.size(2) <= 1 || t.stride(2) == 1 || !t.numel(), "the elements of a head must be dense");
    need(t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat, "heads are float16 or float32");
    return {t.data_ptr(), (size_t)t.size(1), (size_t)t.stride(0), (size_t)t.stride(1)};
}
exl3_dtype type_of(const at::Tensor &t) { return t.scalar_type() == at::kHalf ? EXL3_F16 : EXL3_F32; }
bool same_shape(const at::Tensor &a, const at::Tensor &b) { return a.sizes() == b.sizes(); }

at::ScalarType dtype_or(PyObject *o, at::ScalarType otherwise) {
    if (!given(o)) return otherwise;
    need(THPDtype_Check(o), "out_dtype is a torch.dtype");
    return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

size_t count_of(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    need(v >= 0, "sizes are not negative");
    return (size_t)v;
}
float real_of(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)v;
}

PyObject *one(exl3_status st, const at::Tensor &t) {
    return st == EXL3_OK ? THPVariable_Wrap(t) : PyLong_FromLong(st);
}
PyObject *two(exl3_status st, const at::Tensor &a, const at::Tensor *b) {
    if (st != EXL3_OK) return PyLong_FromLong(st);
    PyObject *x = THPVariable_Wrap(a), *y = b ? THPVariable_Wrap(*b) : Py_NewRef(Py_None);
    PyObject *r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
}

// (q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, rope_scale, out_dtype, q_out, k_out, stream)
PyObject *qk_norm_rope(PyObject *const *a) {
    Call c;
    const at::Tensor &q = c.tensor(a[0], "q is a tensor");
    c.on(a[12]);
    exl3_head_view qv = heads(q), kv{}, ko{};
    const at::Tensor qo = c.output(a[10], q.sizes(), dtype_or(a[9], q.scalar_type()));
    const exl3_head_view qov = heads(qo);
    at::Tensor k_out;
    const bool keys = given(a[1]);
    if (keys) {
        const at::Tensor &k = c.tensor(a[1], "k is a tensor");
        kv = heads(k);
        need(k.size(0) == q.size(0) && k.size(2) == q.size(2) && k.scalar_type() == q.scalar_type(),
             "q and k differ in tokens, head_dim or type");
        k_out = c.output(a[11], k.sizes(), qo.scalar_type());
        ko = heads(k_out);
        need(k_out.scalar_type() == qo.scalar_type(), "q_out and k_out differ in type");
    }
    const int64_t tokens = q.size(0), d = q.size(2);
    const bool turned = given(a[3]);
    const void *freq = c.dense(a[3], at::kFloat, -1, "inv_freq: dense float32", true);
    const void *pos = turned ? c.dense(a[2], at::kInt, tokens, "positions: dense int32, one per token") : nullptr;
    const size_t rot = turned ? 2 * (size_t)THPVariable_Unpack(a[3]).numel() : 0;
    const void *qw = c.dense(a[4], at::kFloat, d, "q_weight: dense float32 [head_dim]", true);
    const void *kw = c.dense(a[5], at::kFloat, d, "k_weight: dense float32 [head_dim]", true);
    const int pairs = PyObject_IsTrue(a[7]);
    if (pairs < 0) throw python_error();
    const exl3_status st = exl3_hip_qk_norm_rope(
        &qv, keys ? &kv : nullptr, type_of(q), (size_t)tokens, (size_t)d, (const float *)qw, (const float *)kw,
        real_of(a[6]), (const int32_t *)pos, (const float *)freq, rot, pairs, real_of(a[8]), &qov,
        keys ? &ko : nullptr, type_of(qo), c.stream);
    return two(st, qo, keys ? &k_out : nullptr);
}

// pages uint8 [page_count, page bytes]
struct Pages {
    void *data;
    size_t count, tokens;
    unsigned bits;
};
Pages pages_of(Call &c, PyObject *o, PyObject *bits, PyObject *page_tokens, size_t kv_heads, size_t head_dim) {
    const at::Tensor &t = c.tensor(o, "pages is a tensor");
    need(t.scalar_type() == at::kByte && t.dim() == 2 && t.is_contiguous(), "pages: dense uint8 [pages, page bytes]");
    const size_t b = count_of(bits);
    need(b == 4 || b == 8, "bits: 4 or 8");
    Pages p{t.data_ptr(), (size_t)t.size(0), count_of(page_tokens), (unsigned)b};
    need((size_t)t.size(1) == exl3_hip_kv_page_bytes(p.bits, kv_heads, head_dim, p.tokens), "page bytes");
    return p;
}

// (pages, k, v, slots, bits, page_tokens, bad_slots, stream)
PyObject *kv_cache_write(PyObject *const *a) {
    Call c;
    const at::Tensor &k = c.tensor(a[1], "k is a tensor"), &v = c.tensor(a[2], "v is a tensor");
    c.on(a[7]);
    const exl3_head_view kv = heads(k), vv = heads(v);
    need(same_shape(k, v) && k.scalar_type() == v.scalar_type(), "k and v differ in shape or type");
    const Pages p = pages_of(c, a[0], a[4], a[5], kv.heads, (size_t)k.size(2));
    const void *slots = c.dense(a[3], at::kLong, k.size(0), "slots: dense int64, one per token");
    void *bad = c.dense(a[6], at::kInt, 1, "bad_slots: int32, one element", true);
    return PyLong_FromLong(exl3_hip_kv_cache_write(p.data, p.count, p.bits, p.tokens, (size_t)k.size(2), &kv, &vv,
                                                   type_of(k), (size_t)k.size(0), (const int64_t *)slots, (int *)bad,
                                                   c.stream));
}

// (pages, slots, kv_heads, head_dim, bits, page_tokens, out_dtype, k, v, bad_slots, stream)
PyObject *kv_cache_read(PyObject *const *a) {
    Call c;
    const size_t h = count_of(a[2]), d = count_of(a[3]);
    const Pages p = pages_of(c, a[0], a[4], a[5], h, d);
    c.on(a[10]);
    const void *slots = c.dense(a[1], at::kLong, -1, "slots: dense int64");
    const int64_t n = THPVariable_Unpack(a[1]).numel(), shape[3] = {n, (int64_t)h, (int64_t)d};
    const at::Tensor k = c.output(a[7], shape, dtype_or(a[6], at::kHalf));
    const at::Tensor v = c.output(a[8], shape, k.scalar_type());
    const exl3_head_view kv = heads(k), vv = heads(v);
    need(v.scalar_type() == k.scalar_type(), "k and v differ in type");
    void *bad = c.dense(a[9], at::kInt, 1, "bad_slots: int32, one element", true);
    const exl3_status st =
        exl3_hip_kv_cache_read(p.data, p.count, p.bits, p.tokens, d, (const int64_t *)slots, (size_t)n, &kv, &vv,
                               type_of(k), (int *)bad, c.stream);
    return two(st, k, &v);
}

float scale_of(PyObject *o, int64_t head_dim) { return given(o) ? real_of(o) : 1.0f / std::sqrt((float)head_dim); }

// (q, pages, page_table, kv_lens, kv_heads, bits, page_tokens, q_len, scale, out, workspace, stream)
PyObject *attention_cached(PyObject *const *a) {
    Call c;
    const at::Tensor &q = c.tensor(a[0], "q is a tensor");
    c.on(a[11]);
    const exl3_head_view qv = heads(q);
    const size_t d = (size_t)q.size(2), h = count_of(a[4]), q_len = count_of(a[7]);
    const Pages p = pages_of(c, a[1], a[5], a[6], h, d);
    const at::Tensor &table = c.tensor(a[2], "page_table is a tensor");
    need(table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous(),
         "page_table: dense int32 [sequences, pages]");
    const size_t n = (size_t)table.size(0);
    const void *lens = c.dense(a[3], at::kInt, (int64_t)n, "kv_lens: dense int32, one per sequence");
    need(q.scalar_type() == at::kHalf && (size_t)q.size(0) == n * q_len, "q: float16 [sequences * q_len, heads, head_dim]");
    const at::Tensor out = c.output(a[9], q.sizes(), at::kHalf);
    const exl3_head_view ov = heads(out);
    need(out.scalar_type() == at::kHalf, "out: float16");
    size_t ws_bytes;
    void *const ws = c.workspace(a[10], &ws_bytes);
    return one(exl3_hip_attention_cached(&qv, &ov, d, p.data, p.count, p.bits, p.tokens, h,
                                         (const int32_t *)table.data_ptr(), (size_t)table.size(1), (const int32_t *)lens,
                                         n, q_len, scale_of(a[8], (int64_t)d), ws, ws_bytes, c.stream),
               out);
}

// (q, k, v, q_starts, kv_starts, causal, scale, out, workspace, stream)
PyObject *attention_prompt(PyObject *const *a) {
    Call c;
    const at::Tensor &q = c.tensor(a[0], "q is a tensor"), &k = c.tensor(a[1], "k is a tensor"),
                     &v = c.tensor(a[2], "v is a tensor");
    c.on(a[9]);
    const exl3_head_view qv = heads(q), kv = heads(k), vv = heads(v);
    need(q.scalar_type() == at::kHalf && k.scalar_type() == at::kHalf && v.scalar_type() == at::kHalf,
         "q, k and v are float16");
    need(same_shape(k, v) && k.size(2) == q.size(2), "q, k and v differ in shape");
    const void *qs = c.dense(a[3], at::kInt, -1, "q_starts: dense int32");
    const int64_t starts = THPVariable_Unpack(a[3]).numel();
    need(starts >= 1, "q_starts: sequences + 1 elements");
    const void *kst = given(a[4]) ? c.dense(a[4], at::kInt, starts, "kv_starts: dense int32, as many as q_starts") : qs;
    const int causal = PyObject_IsTrue(a[5]);
    if (causal < 0) throw python_error();
    const at::Tensor out = c.output(a[7], q.sizes(), at::kHalf);
    const exl3_head_view ov = heads(out);
    need(out.scalar_type() == at::kHalf, "out: float16");
    size_t ws_bytes;
    void *const ws = c.workspace(a[8], &ws_bytes);
    return one(exl3_hip_attention_prompt(&qv, &kv, &vv, &ov, (size_t)q.size(2), (const int32_t *)qs,
                                         (const int32_t *)kst, (size_t)starts - 1, (size_t)q.size(0),
                                         (size_t)k.size(0), scale_of(a[6], q.size(2)), causal, ws, ws_bytes, c.stream),
               out);
}

// rows [tokens, heads, width], or [tokens, width] as one head each
exl3_head_view rows_or_heads(const at::Tensor &t) {
    if (t.dim() == 3) return heads(t);
    need(t.dim() == 2, "rows are [tokens, width] or [tokens, heads, width]");
    need(t.size(1) <= 1 || t.stride(1) == 1 || !t.numel(), "the elements of a row must be dense");
    need(t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat, "rows are float16 or float32");
    return {t.data_ptr(), 1, (size_t)t.stride(0), 0};
}

// (x, weight, residual, gate, eps, out_dtype, out, residual_out, stream)
PyObject *rms_norm(PyObject *const *a) {
    Call c;
    const at::Tensor &x = c.tensor(a[0], "x is a tensor");
    c.on(a[8]);
    const exl3_head_view xv = rows_or_heads(x);
    const int64_t width = x.size(x.dim() - 1);
    const void *w = c.dense(a[1], at::kFloat, width, "weight: dense float32, one per element of a row", true);
    exl3_head_view rv{}, zv{}, rov{};
    at::Tensor kept;
    const bool res = given(a[2]), gated = given(a[3]);
    exl3_dtype rt = EXL3_F32;
    need(res || !given(a[7]), "residual_out without a residual");
    if (res) {
        const at::Tensor &r = c.tensor(a[2], "residual is a tensor");
        need(same_shape(x, r), "x and residual differ in shape");
        rv = rows_or_heads(r);
        rt = type_of(r);
        kept = c.output(a[7], r.sizes(), r.scalar_type());
        need(kept.scalar_type() == r.scalar_type(), "residual and residual_out differ in type");
        rov = rows_or_heads(kept);
    }
    if (gated) {
        const at::Tensor &z = c.tensor(a[3], "gate is a tensor");
        need(same_shape(x, z) && z.scalar_type() == x.scalar_type(), "x and gate differ in shape or type");
        zv = rows_or_heads(z);
    }
    const at::Tensor out = c.output(a[6], x.sizes(), dtype_or(a[5], x.scalar_type()));
    const exl3_head_view ov = rows_or_heads(out);
    const exl3_status st = exl3_hip_rms_norm(&xv, gated ? &zv : nullptr, type_of(x), res ? &rv : nullptr,
                                             res ? &rov : nullptr, rt, (size_t)x.size(0), (size_t)width,
                                             (const float *)w, real_of(a[4]), &ov, type_of(out), c.stream);
    if (st == EXL3_OK && res) return two(st, out, &kept);
    return one(st, out);
}

// starts int32 [sequences + 1], or None and the sequences' number; the pool's slots of the sequences
struct Packed {
    const int32_t *starts, *in, *out;
    size_t sequences, slots;
    void *states;
};
Packed packed(Call &c, PyObject *starts, PyObject *sequences, PyObject *states, PyObject *in, PyObject *out,
              at::ScalarType type, at::IntArrayRef shape) {
    Packed p{};
    if (given(starts)) {
        p.starts = (const int32_t *)c.dense(starts, at::kInt, -1, "starts: dense int32");
        const int64_t n = THPVariable_Unpack(starts).numel();
        need(n >= 1, "starts: sequences + 1 elements");
        p.sequences = (size_t)n - 1;
    } else {
        p.sequences = count_of(sequences);
    }
    if (given(states)) {
        const at::Tensor &t = c.tensor(states, "states is a tensor");
        need(t.scalar_type() == type && t.is_contiguous() && t.dim() == (int64_t)shape.size() + 1 &&
                 t.sizes().slice(1) == shape,
             "states: dense, of the operator's state shape and type");
        p.slots = (size_t)t.size(0);
        p.states = t.data_ptr();
    }
    p.in = (const int32_t *)c.dense(in, at::kInt, (int64_t)p.sequences, "slots_in: dense int32, one per sequence", true);
    p.out = (const int32_t *)c.dense(out, at::kInt, (int64_t)p.sequences, "slots_out: dense int32, one per sequence", true);
    return p;
}
// the row stride of a matrix whose rows are dense; one of a single row may have any
size_t row_stride(const at::Tensor &t) {
    return (size_t)(t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)));
}

// (x, weight, bias, silu, starts, sequences, states, slots_in, slots_out, out_dtype, out, stream)
PyObject *short_conv(PyObject *const *a) {
    Call c;
    const at::Tensor &x = c.tensor(a[0], "x is a tensor");
    c.on(a[11]);
    need(x.dim() == 2, "x: [tokens, channels]");
    rows_or_heads(x);
    const int64_t n = x.size(0), ch = x.size(1);
    const at::Tensor &w = c.tensor(a[1], "weight is a tensor");
    need(w.scalar_type() == at::kFloat && w.is_contiguous() && w.dim() == 2 && w.size(0) == ch,
         "weight: dense float32 [channels, width]");
    const int64_t state[2] = {w.size(1) - 1, ch};
    const Packed p = packed(c, a[4], a[5], a[6], a[7], a[8], x.scalar_type(), state);
    const void *bias = c.dense(a[2], at::kFloat, ch, "bias: dense float32, one per channel", true);
    const int act = PyObject_IsTrue(a[3]);
    if (act < 0) throw python_error();
    const at::Tensor out = c.output(a[10], x.sizes(), dtype_or(a[9], x.scalar_type()));
    rows_or_heads(out);
    return one(exl3_hip_short_conv(x.data_ptr(), type_of(x), row_stride(x), (size_t)n, (size_t)ch,
                                   (const float *)w.data_ptr(), (size_t)w.size(1), (const float *)bias, act, p.starts,
                                   p.sequences, p.states, p.slots, p.in, p.out, out.data_ptr(), type_of(out),
                                   row_stride(out), c.stream),
               out);
}

// (q, k, v, g, beta, a_log, dt_bias, starts, sequences, states, slots_in, slots_out, scale, qk_eps, out, workspace,
//  stream)
PyObject *delta_rule(PyObject *const *a) {
    Call c;
    const at::Tensor &q = c.tensor(a[0], "q is a tensor"), &k = c.tensor(a[1], "k is a tensor"),
                     &v = c.tensor(a[2], "v is a tensor");
    c.on(a[16]);
    const exl3_head_view qv = heads(q), kv = heads(k), vv = heads(v);
    need(q.scalar_type() == at::kHalf && k.scalar_type() == at::kHalf && v.scalar_type() == at::kHalf,
         "q, k and v are float16");
    need(same_shape(q, k) && v.size(0) == q.size(0), "q, k and v differ in shape");
    const int64_t n = q.size(0), h = v.size(1), dk = q.size(2), dv = v.size(2);
    const at::Tensor &g = c.tensor(a[3], "g is a tensor"), &beta = c.tensor(a[4], "beta is a tensor");
    need(g.scalar_type() == at::kFloat && beta.scalar_type() == at::kFloat && g.dim() == 2 && g.size(0) == n &&
             g.size(1) == h && same_shape(g, beta) && (h == 1 || !n || (g.stride(1) == 1 && beta.stride(1) == 1)) &&
             (n <= 1 || row_stride(g) == row_stride(beta)),
         "g and beta: float32 [tokens, v heads] with the same row stride, dense rows");
    const void *al = c.dense(a[5], at::kFloat, h, "a_log: dense float32 [v heads]", true);
    const void *dt = c.dense(a[6], at::kFloat, h, "dt_bias: dense float32 [v heads]", true);
    const int64_t state[3] = {h, dk, dv};
    const Packed p = packed(c, a[7], a[8], a[9], a[10], a[11], at::kFloat, state);
    const at::Tensor out = c.output(a[14], v.sizes(), at::kHalf);
    const exl3_head_view ov = heads(out);
    need(out.scalar_type() == at::kHalf, "out: float16");
    size_t ws_bytes;
    void *const ws = c.workspace(a[15], &ws_bytes);
    return one(exl3_hip_delta_rule(&qv, &kv, &vv, (const float *)g.data_ptr(), (const float *)beta.data_ptr(),
                                   std::max(row_stride(g), row_stride(beta)), (const float *)al, (const float *)dt, &ov, (size_t)dk, (size_t)dv,
                                   p.starts, p.sequences, (size_t)n, (float *)p.states, p.slots, p.in, p.out,
                                   scale_of(a[12], dk), given(a[13]) ? real_of(a[13]) : -1.f, ws, ws_bytes, c.stream),
               out);
}

// a METH_FASTCALL entry of N positional arguments around F
template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused &e) {
        PyErr_SetString(PyExc_AssertionError, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

#define EXL3_ENTRY(name, n) \
    { #name, (PyCFunction)(void (*)(void))entry<name, n>, METH_FASTCALL, nullptr }
PyMethodDef methods[] = {EXL3_ENTRY(qk_norm_rope, 13),     EXL3_ENTRY(kv_cache_write, 8),
                         EXL3_ENTRY(kv_cache_read, 11),    EXL3_ENTRY(attention_cached, 12),
                         EXL3_ENTRY(attention_prompt, 10), EXL3_ENTRY(rms_norm, 9),
                         EXL3_ENTRY(short_conv, 12),       EXL3_ENTRY(delta_rule, 17),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "exl3_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_exl3_torch() { return PyModule_Create(&module_def); }
