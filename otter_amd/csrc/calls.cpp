// The host side of a training operator's call: checks of the arguments, the outputs and the workspace, and the call of the
// library's entry point (include/otter_hip.h), as the Python module otter_amd._calls.
//
// Small batches are bound by what a call costs on the host, not by their kernels (16 questions of 70 tokens: 8 us of attention
// kernel).  The same checks in Python took most of a call.  Us a call, Python -> here, of which launches are 2 to 6:
// attention 12.7 -> 5.1 and backward 17.0 -> 6.5, layer norm 12.9 -> 5.8 and 17.5 -> 9.9, dropout 6.2 -> 4.1, loss 16.7 -> 9.5
// and 10.9 -> 5.7.
//
// The GIL is held while arguments are read and released around allocations and launches.  Exceptions leave as Python ones.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>

#include "../../include/otter_hip.h"

namespace {

using at::Tensor;

// ------------------------------------------------------------------ the library, bound once
struct Library {
#define OTTER_CALLS(X)                                                                                               \
    X(otter_dropout) X(otter_layernorm_forward) X(otter_layernorm_backward) X(otter_layernorm_backward_workspace)    \
    X(otter_attention_forward) X(otter_attention_backward) X(otter_attention_backward_workspace)                     \
    X(otter_inbatch_loss_forward) X(otter_inbatch_loss_backward) X(otter_inbatch_loss_workspace)                     \
    X(otter_inbatch_loss_backward_workspace)
#define OTTER_MEMBER(name) decltype(&::name) name = nullptr;
    OTTER_CALLS(OTTER_MEMBER)
    PyObject* check = nullptr;      // _lib.check(rc, name): raises for rc != 0
    PyObject* stream = nullptr;     // a device's current stream
} lib;

struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};

// a Python exception is set: unwind to the entry
PyObject* checked(int64_t rc, const char* name) {
    PyObject* r = PyObject_CallFunction(lib.check, "Ls", (long long)rc, name);
    if (!r) throw python_error();
    return r;
}
void check(int64_t rc, const char* name) {
    if (rc) Py_DECREF(checked(rc, name));
}

void* stream_of(int device) {
    PyObject* r = PyObject_CallFunction(lib.stream, "i", device);
    if (!r) throw python_error();
    void* s = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    if (PyErr_Occurred()) throw python_error();
    return s;
}

// ------------------------------------------------------------------ arguments
const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

double number(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw python_error();
    return x;
}

int dtype_code(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? OTTER_F32 : t.scalar_type() == at::kBFloat16 ? OTTER_BF16 : -1;
}

// the first operand: on a GPU, of a supported dtype
const Tensor& first(const char* what, const char* name, PyObject* o) {
    const Tensor* t = tensor(o);
    TORCH_CHECK_VALUE(t && t->is_cuda(), what, ": ", name, " must be a tensor on a GPU (the HIP path has no CPU fallback)");
    TORCH_CHECK_VALUE(dtype_code(*t) >= 0, what, ": ", name, " must be float32 or bfloat16, got ", t->scalar_type());
    return *t;
}

// the first one's shape, dtype and device
const Tensor& like(const char* what, const char* name, PyObject* o, const Tensor& a) {
    const Tensor* t = tensor(o);
    TORCH_CHECK_VALUE(t && t->scalar_type() == a.scalar_type() && t->sizes() == a.sizes() && t->device() == a.device(), what, ": ",
                      name, " must be like the first operand: expected ", a.scalar_type(), " ", a.sizes(), " on ", a.device());
    return *t;
}

// a float32 tensor that a forward call returned
const float* kept(const char* what, const char* name, PyObject* o, at::IntArrayRef shape, const Tensor& a) {
    const Tensor* t = tensor(o);
    TORCH_CHECK_VALUE(t && t->scalar_type() == at::kFloat && t->device() == a.device() && t->sizes() == shape && t->is_contiguous(),
                      what, ": ", name, " must be what the forward call returned");
    return t->const_data_ptr<float>();
}

struct Drop {
    double p;
    const int64_t* seed = nullptr;
    uint32_t call = 0;
    Drop(const char* what, PyObject* op, PyObject* oseed, PyObject* ocall, const Tensor& a) : p(number(op)) {
        TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0, what, ": dropout probability ", p, " is not in [0, 1)");
        if (p != 0.0) {
            const Tensor* s = tensor(oseed);
            TORCH_CHECK_VALUE(s && s->scalar_type() == at::kLong && s->numel() == 1 && s->device() == a.device(), what,
                              ": dropout needs seed, an int64 tensor with one element on ", a.device(), " (training.new_seed)");
            seed = s->const_data_ptr<int64_t>();
        }
        PyObject* n = PyNumber_Index(ocall);
        if (!n) throw python_error();
        int over = 0;
        const long long c = PyLong_AsLongLongAndOverflow(n, &over);
        Py_DECREF(n);
        TORCH_CHECK_VALUE(!over && c >= 0 && c < (1ll << 32), what, ": call is not in [0, 2^32)");
        call = (uint32_t)c;
    }
};

// ------------------------------------------------------------------ results
Tensor make(at::IntArrayRef shape, const Tensor& a, at::ScalarType t) { return at::empty(shape, a.options().dtype(t)); }
Tensor make(at::IntArrayRef shape, const Tensor& a) { return at::empty(shape, a.options()); }

PyObject* wrap(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    PyObject* r = THPVariable_Wrap(t);
    if (!r) throw python_error();
    return r;
}
template <typename... Ts>
PyObject* results(const Ts&... ts) {
    PyObject* out = PyTuple_New(sizeof...(ts));
    if (!out) throw python_error();
    Py_ssize_t i = 0;
    try {
        (PyTuple_SET_ITEM(out, i++, wrap(ts)), ...);
    } catch (...) {
        Py_DECREF(out);
        throw;
    }
    return out;
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
// a caller's tensor is written: whoever saved it for a backward pass is to find out
void written(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

// ------------------------------------------------------------------ dropout
PyObject* dropout(const char* what, PyObject* ox, PyObject* op, PyObject* oseed, PyObject* ocall, PyObject* oout) {
    const Tensor& x = first(what, "x", ox);
    const Drop d(what, op, oseed, ocall, x);
    const Tensor* to = oout == Py_None ? nullptr : tensor(oout);
    TORCH_CHECK_VALUE(oout == Py_None || (to && to->sizes() == x.sizes() && to->scalar_type() == x.scalar_type() &&
                                          to->device() == x.device() && to->is_contiguous()),
                      what, ": out must be a contiguous ", x.scalar_type(), " tensor of shape ", x.sizes(), " on ", x.device());
    if (to && x.is_contiguous()) {         // otherwise a copy of x is read
        const char *a = (const char*)x.const_data_ptr(), *b = (const char*)to->const_data_ptr();
        const int64_t bytes = x.numel() * (int64_t)x.element_size();
        TORCH_CHECK_VALUE(a == b || a >= b + bytes || b >= a + bytes, what, ": out overlaps x (it may be x itself)");
    }
    void* const stream = stream_of(x.device().index());
    int rc = 0;
    Tensor out;
    {
        NoGil no_gil;
        if (d.p == 0.0) {
            if (to) to->copy_(x.contiguous());      // copied first where out is another view of it
            else out = x.clone();
        } else {
            const Tensor in = x.contiguous();
            out = to ? *to : at::empty_like(in);
            if (to) written(out);
            const int64_t cols = in.dim() ? in.sizes().back() : 1;
            rc = lib.otter_dropout(x.device().index(), dtype_code(x), ptr(in), out_ptr(out), cols ? in.numel() / cols : 0, cols,
                                   (float)d.p, d.seed, d.call, stream);
        }
    }
    check(rc, "otter_dropout");
    if (!to) return wrap(out);
    Py_INCREF(oout);
    return oout;
}

// ------------------------------------------------------------------ layer norm
struct Norm {
    Tensor x, residual, weight;
    int64_t rows, cols;
    int device, dt, wdt;
    Norm(const char* what, PyObject* ox, PyObject* ow, PyObject* ores) : x(first(what, "x", ox)) {
        TORCH_CHECK_VALUE(x.dim() >= 1, what, ": x has no dimension to normalise over");
        if (ores != Py_None) residual = like(what, "residual", ores, x);
        cols = x.sizes().back();
        const Tensor* w = tensor(ow);
        wdt = w ? dtype_code(*w) : -1;
        TORCH_CHECK_VALUE(wdt >= 0 && w->device() == x.device() && w->dim() == 1 && w->size(0) == cols, what,
                          ": weight must be a float32 or bfloat16 tensor [", cols, "] on ", x.device());
        TORCH_CHECK_VALUE(cols <= INT32_MAX, what, ": cols=", cols, " is too large");
        weight = *w;
        rows = cols ? x.numel() / cols : 0;
        device = x.device().index();
        dt = dtype_code(x);
    }
    void dense() {
        x = x.contiguous();
        weight = weight.contiguous();
        if (residual.defined()) residual = residual.contiguous();
    }
};

PyObject* layer_norm_forward(PyObject* const* a) {
    const char* what = "layer_norm";
    Norm n(what, a[0], a[1], a[4]);
    Tensor bias = like(what, "bias", a[2], n.weight);
    const double eps = number(a[3]);
    const Drop d(what, a[5], a[6], a[7], n.x);
    void* const stream = stream_of(n.device);
    Tensor y, mean, rstd;
    int rc;
    {
        NoGil no_gil;
        n.dense();
        bias = bias.contiguous();
        y = at::empty_like(n.x);
        const at::IntArrayRef lead = n.x.sizes().slice(0, n.x.dim() - 1);
        mean = make(lead, n.x, at::kFloat);
        rstd = make(lead, n.x, at::kFloat);
        rc = lib.otter_layernorm_forward(n.device, n.dt, n.wdt, ptr(n.x), ptr(n.residual), ptr(n.weight), ptr(bias), n.rows,
                                         (int)n.cols, (float)eps, (float)d.p, d.seed, d.call, out_ptr(y),
                                         mean.mutable_data_ptr<float>(), rstd.mutable_data_ptr<float>(), stream);
    }
    check(rc, "otter_layernorm_forward");
    return results(y, mean, rstd);
}

PyObject* layer_norm_backward(PyObject* const* a) {
    const char* what = "layer_norm_backward";
    Norm n(what, a[1], a[2], a[5]);
    Tensor dy = like(what, "dy", a[0], n.x);
    const at::IntArrayRef lead = n.x.sizes().slice(0, n.x.dim() - 1);
    const float *mean = kept(what, "mean", a[3], lead, n.x), *rstd = kept(what, "rstd", a[4], lead, n.x);
    const Drop d(what, a[6], a[7], a[8], n.x);
    const int64_t bytes = lib.otter_layernorm_backward_workspace(n.rows, (int)n.cols);
    if (bytes < 0) check(bytes, "otter_layernorm_backward_workspace");
    void* const stream = stream_of(n.device);
    Tensor dx, dres, dw, db;
    int rc;
    {
        NoGil no_gil;
        n.dense();
        dy = dy.contiguous();
        dx = at::empty_like(n.x);
        if (n.residual.defined() && d.p > 0.0) dres = at::empty_like(n.x);
        dw = make(n.weight.sizes(), n.weight);
        db = make(n.weight.sizes(), n.weight);
        const Tensor ws = make(bytes, n.x, at::kByte);
        rc = lib.otter_layernorm_backward(n.device, n.dt, n.wdt, ptr(dy), ptr(n.x), ptr(n.residual), ptr(n.weight), mean, rstd,
                                          n.rows, (int)n.cols, (float)d.p, d.seed, d.call, out_ptr(dx), out_ptr(dres),
                                          out_ptr(dw), out_ptr(db), out_ptr(ws), bytes, stream);
    }
    check(rc, "otter_layernorm_backward");
    if (n.residual.defined() && !dres.defined()) dres = dx;
    return results(dx, dres, dw, db);
}

// ------------------------------------------------------------------ attention
// The kernels read a tensor in place if its heads are 64 contiguous elements and data and strides multiples of 16 bytes.
bool in_place(const Tensor& t) {
    const int64_t n = t.dim(), mask = 16 / (int64_t)t.element_size() - 1;
    int64_t s = 0;
    for (int64_t i = 0; i < n - 1; ++i) s |= t.stride(i);
    return t.stride(n - 1) == 1 && (s & mask) == 0 && ((uintptr_t)t.const_data_ptr() & 15) == 0;
}

otter_view view(const Tensor& t) {
    const int64_t n = t.dim();
    return {const_cast<void*>(t.const_data_ptr()), n == 4 ? t.stride(0) : 0, t.stride(n - 3), t.stride(n - 2)};
}

struct Attention {
    Tensor q, k, v, mask, cu;
    otter_attention_args args{};
    int64_t lse_shape[3], lse_dims;
    at::IntArrayRef lse() const { return {lse_shape, (size_t)lse_dims}; }
    // a: q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed, call, scale
    Attention(const char* what, PyObject* const* a) : q(first(what, "q", a[0])) {
        const bool packed = a[4] != Py_None;
        const Tensor *tk = tensor(a[1]), *tv = tensor(a[2]);
        TORCH_CHECK_VALUE(tk && tv && q.dim() == (packed ? 3 : 4) && tk->sizes() == q.sizes() && tv->sizes() == q.sizes(), what,
                          ": q, k and v must all be [", packed ? "total" : "batch, tokens", ", heads, 64]; got ", q.sizes(), " ",
                          tk ? tk->sizes() : at::IntArrayRef(), " ", tv ? tv->sizes() : at::IntArrayRef());
        k = like(what, "k", a[1], q);
        v = like(what, "v", a[2], q);
        const at::IntArrayRef shape = q.sizes();
        const int64_t heads = shape[shape.size() - 2], dim = shape.back();
        TORCH_CHECK_VALUE(heads >= 1, what, ": no heads");
        for (const int64_t n : shape) TORCH_CHECK_VALUE(n <= INT32_MAX, what, ": q is too large");
        TORCH_CHECK_VALUE(!packed || a[3] == Py_None, what, ": a key mask and packed sequences exclude each other");
        const Drop d(what, a[6], a[7], a[8], q);
        args.dtype = dtype_code(q);
        args.heads = (int32_t)heads;
        args.head_dim = (int32_t)dim;
        args.call = d.call;
        args.scale = (float)(a[9] == Py_None ? 1.0 / std::sqrt((double)std::max<int64_t>(1, dim)) : number(a[9]));
        args.dropout_p = (float)d.p;
        args.seed = d.seed;
        if (packed) {
            const Tensor* c = tensor(a[4]);
            TORCH_CHECK_VALUE(c && c->scalar_type() == at::kInt && c->dim() == 1 && c->numel() >= 1 && c->numel() <= INT32_MAX &&
                                  c->device() == q.device(),
                              what, ": cu_seqlens must be int32 [batch + 1] on ", q.device());
            cu = *c;
            const double longest = number(a[5]);
            TORCH_CHECK_VALUE(longest <= INT32_MAX, what, ": max_seqlen=", longest, " is too large");
            args.batch = (int32_t)(cu.numel() - 1);
            args.tokens = longest > 0 ? (int32_t)longest : 0;
            args.total = shape[0];
            lse_shape[0] = heads, lse_shape[1] = shape[0], lse_dims = 2;
            return;
        }
        args.batch = (int32_t)shape[0];
        args.tokens = (int32_t)shape[1];
        lse_shape[0] = shape[0], lse_shape[1] = heads, lse_shape[2] = shape[1], lse_dims = 3;
        if (a[3] != Py_None) {
            const Tensor* m = tensor(a[3]);
            TORCH_CHECK_VALUE(m && m->dim() == 2 && m->sizes() == shape.slice(0, 2) && m->device() == q.device(), what,
                              ": mask must be [", shape[0], ", ", shape[1], "] on ", q.device());
            mask = *m;
        }
    }
    // the tensors as the kernels read them, copied where they cannot; without the GIL
    void operands() {
        for (Tensor* t : {&q, &k, &v}) place(*t);
        args.q = view(q), args.k = view(k), args.v = view(v);
        if (cu.defined()) args.cu_seqlens = (cu = cu.contiguous()).const_data_ptr<int32_t>();
        if (mask.defined()) {
            if (mask.scalar_type() != at::kLong) mask = mask.ne(0).to(at::kLong);
            args.mask = (mask = mask.contiguous()).const_data_ptr<int64_t>();
        }
    }
    // not contiguous(), which hands an unaligned but contiguous tensor back
    static void place(Tensor& t) {
        if (!in_place(t)) t = t.clone(at::MemoryFormat::Contiguous);
    }
};

PyObject* attention_forward(PyObject* const* a) {
    Attention s("attention", a);
    const int device = s.q.device().index();
    void* const stream = stream_of(device);
    Tensor out, lse;
    int rc;
    {
        NoGil no_gil;
        s.operands();
        out = make(s.q.sizes(), s.q);
        lse = make(s.lse(), s.q, at::kFloat);
        s.args.out = view(out);
        s.args.lse = lse.mutable_data_ptr<float>();
        rc = lib.otter_attention_forward(device, &s.args, stream);
    }
    check(rc, "otter_attention_forward");
    return results(out, lse);
}

// a: dout, out, lse, grads (None or three tensors), then those of Attention
PyObject* attention_backward(PyObject* const* a) {
    const char* what = "attention_backward";
    Attention s(what, a + 4);
    Tensor dout = like(what, "dout", a[0], s.q), out = like(what, "out", a[1], s.q);
    s.args.lse = const_cast<float*>(kept(what, "lse", a[2], s.lse(), s.q));
    Tensor g[3];
    if (a[3] != Py_None) {
        PyObject* seq = PySequence_Fast(a[3], "attention_backward: grads must be three tensors");
        if (!seq) throw python_error();
        bool good = PySequence_Fast_GET_SIZE(seq) == 3;
        for (int i = 0; i < 3 && good; ++i) {
            const Tensor* t = tensor(PySequence_Fast_GET_ITEM(seq, i));
            good = t && t->sizes() == s.q.sizes() && t->scalar_type() == s.q.scalar_type() && t->device() == s.q.device() && in_place(*t);
            for (int64_t n = 0; n < 4 && good && n < t->dim(); ++n) good = t->size(n) <= 1 || t->stride(n) != 0;   // no expanded ones
            if (good) g[i] = *t;
        }
        Py_DECREF(seq);
        TORCH_CHECK_VALUE(good, what, ": grads must be like q, their heads contiguous, data and strides multiples of 16 bytes, not expanded");
        const Tensor* const all[] = {&g[0], &g[1], &g[2], &s.q, &s.k, &s.v, &dout, &out};
        for (int i = 0; i < 3; ++i)
            for (int j = i + 1; j < 8; ++j)
                TORCH_CHECK_VALUE(s.q.numel() == 0 || g[i].const_data_ptr() != all[j]->const_data_ptr(), what,
                                  ": grads may not be one another or an operand");
    }
    const int device = s.q.device().index();
    void* const stream = stream_of(device);
    int64_t bytes;
    int rc = 0;
    {
        NoGil no_gil;
        s.operands();
        Attention::place(dout);
        Attention::place(out);
        for (Tensor& t : g) {
            if (t.defined()) written(t);
            else t = make(s.q.sizes(), s.q);
        }
        s.args.out = view(out), s.args.dout = view(dout);
        s.args.dq = view(g[0]), s.args.dk = view(g[1]), s.args.dv = view(g[2]);
        bytes = lib.otter_attention_backward_workspace(&s.args);
        if (bytes >= 0) {
            const Tensor ws = make(bytes, s.q, at::kByte);
            s.args.workspace = out_ptr(ws);
            s.args.workspace_bytes = bytes;
            rc = lib.otter_attention_backward(device, &s.args, stream);
        }
    }
    if (bytes < 0) check(bytes, "otter_attention_backward_workspace");
    check(rc, "otter_attention_backward");
    return results(g[0], g[1], g[2]);
}

// ------------------------------------------------------------------ in-batch loss
struct Loss {
    Tensor q, c, neg;
    int B, d, ncol, device;
    Loss(const char* what, PyObject* const* a) {
        const Tensor *tq = tensor(a[0]), *tc = tensor(a[1]), *tn = a[2] == Py_None ? nullptr : tensor(a[2]);
        TORCH_CHECK_VALUE(tq && tq->is_cuda(), what, ": q must be a tensor on a GPU (the HIP path has no CPU fallback)");
        TORCH_CHECK_VALUE(tq->dim() == 2 && tc && tc->sizes() == tq->sizes() && (a[2] == Py_None || (tn && tn->sizes() == tq->sizes())),
                          what, ": q, c and neg_c must all be [B, d]; got ", tq->sizes(), " ", tc ? tc->sizes() : at::IntArrayRef(),
                          " ", tn ? tn->sizes() : at::IntArrayRef());
        TORCH_CHECK_VALUE(tc->device() == tq->device() && (!tn || tn->device() == tq->device()), what,
                          ": q, c and neg_c must be on one GPU");
        TORCH_CHECK_VALUE(tq->size(0) < INT32_MAX && tq->size(1) <= INT32_MAX, what, ": q is too large");
        q = *tq, c = *tc;
        if (tn) neg = *tn;
        B = (int)q.size(0), d = (int)q.size(1), ncol = B + (tn != nullptr);
        device = q.device().index();
    }
    void operands() {
        for (Tensor* t : {&q, &c, &neg})
            if (t->defined()) *t = t->to(at::kFloat).contiguous();
    }
};

PyObject* inbatch_loss_forward(PyObject* const* a) {
    Loss s("inbatch_loss", a);
    const int64_t bytes = lib.otter_inbatch_loss_workspace(s.B, s.d);
    if (bytes < 0) check(bytes, "otter_inbatch_loss_workspace");
    void* const stream = stream_of(s.device);
    Tensor loss, buf, product, stats;
    int rc;
    {
        NoGil no_gil;
        s.operands();
        const int64_t ld = (s.ncol + 3ll) / 4 * 4;         // rows of whole 16-byte pieces
        buf = make({s.B, ld}, s.q);
        stats = make({2, s.B}, s.q);
        loss = make({}, s.q);
        const Tensor ws = make(bytes, s.q, at::kByte);
        rc = lib.otter_inbatch_loss_forward(s.device, s.q.const_data_ptr<float>(), s.c.const_data_ptr<float>(), (const float*)ptr(s.neg),
                                            s.B, s.d, buf.mutable_data_ptr<float>(), (int)ld, stats.mutable_data_ptr<float>(),
                                            loss.mutable_data_ptr<float>(), out_ptr(ws), bytes, stream);
        product = buf.narrow(1, 0, s.ncol);
    }
    check(rc, "otter_inbatch_loss_forward");
    return results(loss, product, stats);
}

// a: dloss, q, c, neg_c, product, stats
PyObject* inbatch_loss_backward(PyObject* const* a) {
    const char* what = "inbatch_loss_backward";
    Loss s(what, a + 1);
    const Tensor *product = tensor(a[4]), *stats = tensor(a[5]), *dloss = tensor(a[0]);
    TORCH_CHECK_VALUE(product && product->dim() == 2 && product->size(0) == s.B && product->size(1) == s.ncol &&
                          product->scalar_type() == at::kFloat && product->device() == s.q.device() &&
                          (s.ncol <= 1 || product->stride(1) == 1) && product->stride(0) <= INT32_MAX && stats && stats->dim() == 2 &&
                          stats->size(0) == 2 && stats->size(1) == s.B && stats->scalar_type() == at::kFloat &&
                          stats->device() == s.q.device() && stats->is_contiguous(),
                      what, ": product and stats must be what inbatch_loss_forward returned");
    TORCH_CHECK_VALUE(dloss && dloss->numel() == 1 && dloss->scalar_type() == at::kFloat && dloss->device() == s.q.device(), what,
                      ": dloss must be one float32 element on ", s.q.device());
    const int64_t bytes = lib.otter_inbatch_loss_backward_workspace(s.B, s.d);
    if (bytes < 0) check(bytes, "otter_inbatch_loss_backward_workspace");
    void* const stream = stream_of(s.device);
    Tensor dq, dc, dneg;
    int rc;
    {
        NoGil no_gil;
        s.operands();
        dq = make(s.q.sizes(), s.q);
        dc = make(s.q.sizes(), s.q);
        if (s.neg.defined()) dneg = make(s.q.sizes(), s.q);
        Tensor ws;
        if (bytes) ws = make(bytes, s.q, at::kByte);
        rc = lib.otter_inbatch_loss_backward(s.device, dloss->const_data_ptr<float>(), s.q.const_data_ptr<float>(),
                                             s.c.const_data_ptr<float>(), (const float*)ptr(s.neg), s.B, s.d,
                                             product->const_data_ptr<float>(), s.B > 1 ? (int)product->stride(0) : s.ncol,
                                             stats->const_data_ptr<float>(), dq.mutable_data_ptr<float>(), dc.mutable_data_ptr<float>(),
                                             (float*)out_ptr(dneg), out_ptr(ws), bytes, stream);
    }
    check(rc, "otter_inbatch_loss_backward");
    return results(dq, dc, dneg);
}

// ------------------------------------------------------------------ the module
PyObject* load(PyObject* const* a) {
    const char* path = PyUnicode_AsUTF8(a[0]);
    if (!path) throw python_error();
    void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(h, dlerror());
#define OTTER_BIND(name)                                                     \
    lib.name = reinterpret_cast<decltype(&::name)>(dlsym(h, #name));         \
    TORCH_CHECK(lib.name, #name, " is not in ", path);
    OTTER_CALLS(OTTER_BIND)
    Py_INCREF(a[1]);
    Py_INCREF(a[2]);
    Py_XSETREF(lib.check, a[1]);
    Py_XSETREF(lib.stream, a[2]);
    Py_RETURN_NONE;
}

PyObject* dropout_forward(PyObject* const* a) { return dropout("dropout", a[0], a[1], a[2], a[3], a[4]); }
PyObject* dropout_backward(PyObject* const* a) { return dropout("dropout_backward", a[0], a[1], a[2], a[3], a[4]); }

// one entry: N positional arguments, C++ exceptions turned into Python's
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == N, "expected ", N, " arguments, got ", n);
    if (F != load) TORCH_CHECK(lib.check, "otter_amd._calls.load() has not been called");
    at::NoGradGuard no_grad;               // copies and casts made here are no part of a caller's graph
    return F(a);
    END_HANDLE_TH_ERRORS
}

#define OTTER_ENTRY(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {OTTER_ENTRY(load, 3),
                         OTTER_ENTRY(dropout_forward, 5),
                         OTTER_ENTRY(dropout_backward, 5),
                         OTTER_ENTRY(layer_norm_forward, 8),
                         OTTER_ENTRY(layer_norm_backward, 9),
                         OTTER_ENTRY(attention_forward, 10),
                         OTTER_ENTRY(attention_backward, 14),
                         OTTER_ENTRY(inbatch_loss_forward, 3),
                         OTTER_ENTRY(inbatch_loss_backward, 6),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Host side of the training operators' calls", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
