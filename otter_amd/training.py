"""Layer operators of a fine-tuning step on MI355X: attention, layer norm of a sum and dropout, each with its gradient.

The reference trains its encoders with torch autograd through HF's BERT/RoBERTa layers (retrieval/models/tb_retriever.py,
scripts/train_1hop_tb_retrieval.py:196-262); these are the operators of such a layer that are not plain matrix products, as
HIP kernels of libotter_hip.so (include/otter_hip.h).  The loss of the same step is otter_amd.inbatch.inbatch_loss.

Each operator comes in two forms:
  * attention / layer_norm / dropout            one differentiable call (torch autograd, first order)
  * *_forward / *_backward                      the two halves as plain calls, for loops that keep their own tape and for
                                                captured graphs
Activations are float32 or bfloat16; sums, softmax statistics and probabilities are float32.  There is no CPU path.

Dropout stores no mask.  Its random numbers are drawn from `seed`, an int64 tensor with one element ON THE GPU (a captured
graph reads the value it holds at replay), and `call`, a number that tells apart the calls sharing that seed: give every
dropout of a step its own `call`, every step a new seed, and a backward call those of its forward call.

Under graph capture use the *_forward / *_backward calls.  (torch's own autograd engine ends the process when a backward
pass is captured while an eager graph over the same leaves is alive; that is not particular to these operators.)
"""
import math
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.OTTER_F32, torch.bfloat16: _lib.OTTER_BF16}


def new_seed(device=None, generator=None):
    """A random seed for the dropout of one step: int64 [1] on the GPU, drawn there."""
    dev = torch.device("cuda") if device is None else device
    return torch.randint(0, 2 ** 62, (1,), dtype=torch.int64, device=dev, generator=generator)


def _on_gpu(what, name, t):
    """The tensor is on a GPU and of a supported dtype; returns (device, dtype code)."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError("%s: %s must be a tensor on a GPU (the HIP path has no CPU fallback)" % (what, name))
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError("%s: %s must be float32 or bfloat16, got %s" % (what, name, t.dtype))
    return t.device, code


def _like(what, name, t, first):
    """t has the first tensor's shape, dtype and device."""
    if not isinstance(t, torch.Tensor) or t.dtype is not first.dtype or t.shape != first.shape or t.device != first.device:
        raise ValueError("%s: %s must be like the first operand: expected %s %r on %s" % (
            what, name, first.dtype, tuple(first.shape), first.device))


def _seed_ptr(what, seed, dropout_p, dev):
    if not 0.0 <= dropout_p < 1.0:
        raise ValueError("%s: dropout probability %r is not in [0, 1)" % (what, dropout_p))
    if dropout_p == 0.0:
        return None
    if not (torch.is_tensor(seed) and seed.dtype == torch.int64 and seed.numel() == 1 and seed.device == dev):
        raise ValueError("%s: dropout needs seed, an int64 tensor with one element on %s (training.new_seed)" % (what, dev))
    return seed.data_ptr()


def _call_id(what, call):
    call = int(call)
    if not 0 <= call < 2 ** 32:
        raise ValueError("%s: call=%d is not in [0, 2^32)" % (what, call))
    return call


# The handle of a device's current stream; torch.cuda.current_stream() builds an object around it, which takes as long as a
# small kernel.
_stream = torch._C._cuda_getCurrentRawStream


# ------------------------------------------------------------------------------------------------------------ dropout
def _dropout(what, x, p, seed, call, out=None):
    lib = _lib.load()
    dev, dt = _on_gpu(what, "x", x)
    ptr = _seed_ptr(what, seed, p, dev)
    if p == 0.0:
        return x.clone() if out is None else out.copy_(x)
    if not x.is_contiguous():
        x = x.contiguous()
    cols = x.shape[-1] if x.dim() else 1
    rows = x.numel() // cols if cols else 0
    if out is None:
        out = torch.empty_like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("%s: out must be a contiguous %s tensor of shape %r on %s" % (what, x.dtype, tuple(x.shape), dev))
    _lib.check(lib.otter_dropout(dev.index, dt, x.data_ptr(), out.data_ptr(), rows, cols, p, ptr, _call_id(what, call),
                                 _stream(dev.index)), "otter_dropout")
    return out


def dropout_forward(x, p, seed, call=0, out=None):
    """y = x * keep / (1 - p); the draws are counted along x's last dimension, the others together are its rows.
    A dropped value is zero whatever it was.  out may be x itself."""
    return _dropout("dropout", x, p, seed, call, out)


def dropout_backward(dy, p, seed, call=0, out=None):
    """dx = dy * keep / (1 - p), with the draws of the forward call of the same seed and `call`."""
    return _dropout("dropout_backward", dy, p, seed, call, out)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, call):
        ctx.save_for_backward(seed)
        ctx.p, ctx.call = p, call
        return dropout_forward(x, p, seed, call)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return dropout_backward(dy, ctx.p, ctx.saved_tensors[0], ctx.call), None, None, None


def dropout(x, p, seed, call=0):
    """Differentiable dropout (dropout_forward)."""
    return _Dropout.apply(x, p, seed, call)


# --------------------------------------------------------------------------------------------------------- layer norm
def _norm_args(what, x, weight, residual, dropout_p, seed, call):
    dev, dt = _on_gpu(what, "x", x)
    if x.dim() < 1:
        raise ValueError("%s: x has no dimension to normalise over" % what)
    if residual is not None:
        _like(what, "residual", residual, x)
    cols = x.shape[-1]
    wdt = _DTYPES.get(weight.dtype) if isinstance(weight, torch.Tensor) else None
    if wdt is None or weight.device != dev or weight.shape != (cols,):
        raise ValueError("%s: weight must be a float32 or bfloat16 tensor [%d] on %s" % (what, cols, dev))
    rows = x.numel() // cols if cols else 0
    return dev, dt, wdt, rows, cols, _seed_ptr(what, seed, dropout_p, dev), _call_id(what, call)


def layer_norm_forward(x, weight, bias, eps=1e-5, residual=None, dropout_p=0.0, seed=None, call=0):
    """y = LayerNorm(dropout(x) + residual) over the last dimension (<= 8192); returns (y, mean, rstd), the last two float32
    of x's leading shape.  weight and bias share one dtype, float32 or bfloat16, whatever x's is."""
    lib = _lib.load()
    what = "layer_norm"
    dev, dt, wdt, rows, cols, ptr, call = _norm_args(what, x, weight, residual, dropout_p, seed, call)
    _like(what, "bias", bias, weight)
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    y = torch.empty_like(x)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    _lib.check(lib.otter_layernorm_forward(
        dev.index, dt, wdt, x.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(),
        bias.data_ptr(), rows, cols, eps, dropout_p, ptr, call, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _stream(dev.index)),
        "otter_layernorm_forward")
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, residual=None, dropout_p=0.0, seed=None, call=0):
    """Gradients of layer_norm_forward: (dx, dresidual, dweight, dbias).  dresidual is None without a residual and dx itself
    without dropout (the two are equal then)."""
    lib = _lib.load()
    what = "layer_norm_backward"
    dev, dt, wdt, rows, cols, ptr, call = _norm_args(what, x, weight, residual, dropout_p, seed, call)
    _like(what, "dy", dy, x)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.device != dev or t.numel() != rows or not t.is_contiguous():
            raise ValueError("%s: %s must be what layer_norm_forward returned for x" % (what, name))
    dy, x, weight = dy.contiguous(), x.contiguous(), weight.contiguous()
    residual = None if residual is None else residual.contiguous()
    dx = torch.empty_like(x)
    dres = torch.empty_like(x) if residual is not None and dropout_p > 0.0 else None
    dw, db = torch.empty((2, cols), dtype=weight.dtype, device=dev).unbind(0)
    nbytes = lib.otter_layernorm_backward_workspace(rows, cols)
    if nbytes < 0:
        _lib.check(int(nbytes), "otter_layernorm_backward_workspace")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _lib.check(lib.otter_layernorm_backward(
        dev.index, dt, wdt, dy.data_ptr(), x.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(),
        mean.data_ptr(), rstd.data_ptr(), rows, cols, dropout_p, ptr, call, dx.data_ptr(),
        None if dres is None else dres.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), nbytes, _stream(dev.index)),
        "otter_layernorm_backward")
    return dx, (dx if dres is None and residual is not None else dres), dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, dropout_p, seed, call):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps, residual, dropout_p, seed, call)
        ctx.save_for_backward(x, weight, mean, rstd, residual, seed)
        ctx.dropout_p, ctx.call = dropout_p, call
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd, residual, seed = ctx.saved_tensors
        dx, dres, dw, db = layer_norm_backward(dy, x, weight, mean, rstd, residual, ctx.dropout_p, seed, ctx.call)
        return dx, dw, db, None, dres, None, None, None


def layer_norm(x, weight, bias, eps=1e-5, residual=None, dropout_p=0.0, seed=None, call=0):
    """Differentiable LayerNorm(dropout(x) + residual) (layer_norm_forward)."""
    return _LayerNorm.apply(x, weight, bias, eps, residual, dropout_p, seed, call)


# ---------------------------------------------------------------------------------------------------------- attention
# otter_attention_args of include/otter_hip.h: the head, q k v out, lse, dout dq dk dv, workspace and its size
_HEAD = struct.Struct("=5iI2fqQQQ")
_VIEWS = struct.Struct("=16q")
_TAIL = struct.Struct("=Qq")
_NO_VIEWS = _VIEWS.pack(*(0,) * 16)


def _operand(t, mask):
    """(t, its pointer and strides) if the kernels can read it in place -- heads of 64 contiguous elements, 16-byte aligned data
    and strides (mask: elements of 16 bytes, less one) -- otherwise of a contiguous copy."""
    s, p = t.stride(), t.data_ptr()
    if len(s) == 4:
        sb, st, sh, inner = s
    else:
        sb, (st, sh, inner) = 0, s
    if inner != 1 or p & 15 or (sb | st | sh) & mask:
        return _operand(t.clone(memory_format=torch.contiguous_format), mask)
    return t, (p, sb, st, sh)


def _dense(p, shape):
    """Pointer and strides of a contiguous tensor."""
    row = shape[-2] * shape[-1]
    return (p, shape[1] * row if len(shape) == 4 else 0, row, shape[-1])


def _attention_args(what, q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed, call, scale):
    """(packed head of the arguments, the views of q, k and v, tensors to keep alive, device, lse shape, alignment mask)."""
    dev, dt = _on_gpu(what, "q", q)
    packed = cu_seqlens is not None
    shape = q.shape
    if len(shape) != (3 if packed else 4) or k.shape != shape or v.shape != shape:
        raise ValueError("%s: q, k and v must all be [%s, heads, 64]; got %r %r %r" % (
            what, "total" if packed else "batch, tokens", tuple(shape), tuple(k.shape), tuple(v.shape)))
    _like(what, "k", k, q)
    _like(what, "v", v, q)
    heads, dim = shape[-2], shape[-1]
    if heads < 1:
        raise ValueError("%s: no heads" % what)
    if packed and mask is not None:
        raise ValueError("%s: a key mask and packed sequences exclude each other" % what)
    align = 16 // q.element_size() - 1
    q, vq = _operand(q, align)
    k, vk = _operand(k, align)
    v, vv = _operand(v, align)
    views = vq + vk + vv
    seed_ptr, call = _seed_ptr(what, seed, dropout_p, dev) or 0, _call_id(what, call)
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, dim))
    if packed:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.device != dev:
            raise ValueError("%s: cu_seqlens must be int32 [batch + 1] on %s" % (what, dev))
        cu_seqlens = cu_seqlens.contiguous()
        if max_seqlen is None:
            max_seqlen = int(cu_seqlens.diff().max()) if cu_seqlens.numel() > 1 else 0
        head = _HEAD.pack(dt, cu_seqlens.numel() - 1, max(0, int(max_seqlen)), heads, dim, call, scale, dropout_p, shape[0], 0,
                          cu_seqlens.data_ptr(), seed_ptr)
        return head, views, (q, k, v, cu_seqlens), dev, (heads, shape[0]), align
    mask_ptr = 0
    if mask is not None:
        if not torch.is_tensor(mask) or mask.shape != shape[:2] or mask.device != dev:
            raise ValueError("%s: mask must be [%d, %d] on %s" % (what, shape[0], shape[1], dev))
        mask = (mask if mask.dtype == torch.int64 else (mask != 0).to(torch.int64)).contiguous()
        mask_ptr = mask.data_ptr()
    head = _HEAD.pack(dt, shape[0], shape[1], heads, dim, call, scale, dropout_p, 0, mask_ptr, 0, seed_ptr)
    return head, views, (q, k, v, mask), dev, (shape[0], heads, shape[1]), align


def attention_forward(q, k, v, mask=None, cu_seqlens=None, max_seqlen=None, dropout_p=0.0, seed=None, call=0, scale=None):
    """out = dropout(softmax(scale q k^T)) v, every token attending to every key that counts; returns (out, lse).

    Dense: q, k, v [batch, tokens, heads, 64], mask [batch, tokens] (non-zero = the key counts; as input_mask of the encoder)
    or None.  Keys left out reach nothing, whatever they hold; a sequence whose mask leaves nothing attends to all its keys
    evenly.  Packed: [total, heads, 64] with cu_seqlens int32 [batch + 1] (non-decreasing) and max_seqlen, the longest
    sequence (None: read back from the GPU); rows of no sequence come out as zeros.
    Views of a fused projection, qkv.unbind(-3), are read in place.  scale: 1 / 8 by default.
    lse (float32 [batch, heads, tokens] / [heads, total]) is what the backward pass needs."""
    lib = _lib.load()
    head, views, keep, dev, lse_shape, _ = _attention_args("attention", q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed,
                                                           call, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(lse_shape, dtype=torch.float32, device=dev)
    args = b"".join((head, _VIEWS.pack(*views, *_dense(out.data_ptr(), out.shape)), lse.data_ptr().to_bytes(8, "little"),
                     _NO_VIEWS, _TAIL.pack(0, 0)))
    _lib.check(lib.otter_attention_forward(dev.index, args, _stream(dev.index)), "otter_attention_forward")
    return out, lse


def attention_backward(dout, q, k, v, out, lse, mask=None, cu_seqlens=None, max_seqlen=None, dropout_p=0.0, seed=None, call=0,
                       scale=None, grads=None):
    """Gradients (dq, dk, dv) of attention_forward, whose other arguments must be given again.  grads: three tensors to
    write them to, for instance the views dqkv.unbind(-3) of one buffer."""
    lib = _lib.load()
    what = "attention_backward"
    head, views, keep, dev, lse_shape, align = _attention_args(what, q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed,
                                                               call, scale)
    _like(what, "dout", dout, q)
    _like(what, "out", out, q)
    if lse.shape != lse_shape or lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous():
        raise ValueError("%s: lse must be what attention_forward returned" % what)
    dout, v_dout = _operand(dout, align)
    out, v_out = _operand(out, align)
    if grads is None:
        buf = torch.empty((3,) + q.shape, dtype=q.dtype, device=dev)
        p, step = buf.data_ptr(), q.numel() * q.element_size()
        to = _dense(p, q.shape) + _dense(p + step, q.shape) + _dense(p + 2 * step, q.shape)
        grads = buf.unbind(0)
    else:
        to = ()
        for t in grads:
            if t.shape != q.shape or t.dtype != q.dtype or t.device != dev or _operand(t, align)[0] is not t:
                raise ValueError("%s: grads must be like q, their heads contiguous, data and strides multiples of 16 bytes" % what)
            to += _operand(t, align)[1]
    views = _VIEWS.pack(*views, *v_out)
    lse_ptr = lse.data_ptr().to_bytes(8, "little")
    nbytes = lib.otter_attention_backward_workspace(b"".join((head, views, lse_ptr, _NO_VIEWS, _TAIL.pack(0, 0))))
    if nbytes < 0:
        _lib.check(int(nbytes), "otter_attention_backward_workspace")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args = b"".join((head, views, lse_ptr, _VIEWS.pack(*v_dout, *to), _TAIL.pack(ws.data_ptr(), nbytes)))
    _lib.check(lib.otter_attention_backward(dev.index, args, _stream(dev.index)), "otter_attention_backward")
    dq, dk, dv = grads
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed, call, scale):
        if cu_seqlens is not None and max_seqlen is None:
            max_seqlen = int(cu_seqlens.diff().max()) if cu_seqlens.numel() > 1 else 0
        out, lse = attention_forward(q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed, call, scale)
        ctx.save_for_backward(q, k, v, out, lse, mask, cu_seqlens, seed)
        ctx.rest = (max_seqlen, dropout_p, call, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, mask, cu_seqlens, seed = ctx.saved_tensors
        max_seqlen, dropout_p, call, scale = ctx.rest
        dq, dk, dv = attention_backward(dout, q, k, v, out, lse, mask, cu_seqlens, max_seqlen, dropout_p, seed, call, scale)
        return dq, dk, dv, None, None, None, None, None, None, None


def attention(q, k, v, mask=None, cu_seqlens=None, max_seqlen=None, dropout_p=0.0, seed=None, call=0, scale=None):
    """Differentiable attention (attention_forward)."""
    return _Attention.apply(q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed, call, scale)
