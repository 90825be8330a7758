"""Layer operators of a fine-tuning step on MI355X: attention, layer norm of a sum and dropout, each with its gradient.

The reference trains its encoders with torch autograd through HF's BERT/RoBERTa layers (retrieval/models/tb_retriever.py,
scripts/train_1hop_tb_retrieval.py:196-262); these are the operators of such a layer that are not plain matrix products, as
HIP kernels of libotter_hip.so (include/otter_hip.h).  The loss of the same step is otter_amd.inbatch.inbatch_loss.

Each operator comes in two forms:
  * attention / layer_norm / dropout            one differentiable call (torch autograd, first order)
  * *_forward / *_backward                      the two halves as plain calls, for loops that keep their own tape and for
                                                captured graphs
Activations are float32 or bfloat16; sums, softmax statistics and norms are float32.  bfloat16 attention rounds the dropped-out
probabilities and the scores' gradients to bfloat16 in front of the matrix products that take them.  There is no CPU path.

Dropout stores no mask.  Its random numbers are drawn from `seed`, an int64 tensor with one element ON THE GPU (a captured
graph reads the value it holds at replay), and `call`, a number that tells apart the calls sharing that seed: give every
dropout of a step its own `call`, every step a new seed, and a backward call those of its forward call.

Under graph capture use the *_forward / *_backward calls.  (torch's own autograd engine ends the process when a backward
pass is captured while an eager graph over the same leaves is alive; that is not particular to these operators.)
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib


def new_seed(device=None, generator=None):
    """A random seed for the dropout of one step: int64 [1] on the GPU, drawn there."""
    dev = torch.device("cuda") if device is None else device
    return torch.randint(0, 2 ** 62, (1,), dtype=torch.int64, device=dev, generator=generator)


# ------------------------------------------------------------------------------------------------------------ dropout
def dropout_forward(x, p, seed, call=0, out=None):
    """y = x * keep / (1 - p); the draws are counted along x's last dimension, the others together are its rows.
    A dropped value is zero whatever it was.  out may be x itself but not overlap it otherwise."""
    return _lib.calls().dropout_forward(x, p, seed, call, out)


def dropout_backward(dy, p, seed, call=0, out=None):
    """dx = dy * keep / (1 - p), with the draws of the forward call of the same seed and `call`."""
    return _lib.calls().dropout_backward(dy, p, seed, call, out)


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
def layer_norm_forward(x, weight, bias, eps=1e-5, residual=None, dropout_p=0.0, seed=None, call=0):
    """y = LayerNorm(dropout(x) + residual) over the last dimension (<= 8192); returns (y, mean, rstd), the last two float32
    of x's leading shape.  weight and bias share one dtype, float32 or bfloat16, whatever x's is."""
    return _lib.calls().layer_norm_forward(x, weight, bias, eps, residual, dropout_p, seed, call)


def layer_norm_backward(dy, x, weight, mean, rstd, residual=None, dropout_p=0.0, seed=None, call=0):
    """Gradients of layer_norm_forward: (dx, dresidual, dweight, dbias).  dresidual is None without a residual and dx itself
    without dropout (the two are equal then)."""
    return _lib.calls().layer_norm_backward(dy, x, weight, mean, rstd, residual, dropout_p, seed, call)


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
def _longest(cu_seqlens, max_seqlen):
    """max_seqlen, read back from the GPU if it is not given."""
    if cu_seqlens is not None and max_seqlen is None:
        max_seqlen = int(cu_seqlens.diff().max()) if cu_seqlens.numel() > 1 else 0
    return max_seqlen


def attention_forward(q, k, v, mask=None, cu_seqlens=None, max_seqlen=None, dropout_p=0.0, seed=None, call=0, scale=None):
    """out = dropout(softmax(scale q k^T)) v, every token attending to every key that counts; returns (out, lse).

    Dense: q, k, v [batch, tokens, heads, 64], mask [batch, tokens] (non-zero = the key counts; as input_mask of the encoder)
    or None.  Keys left out reach nothing, whatever they hold; a sequence whose mask leaves nothing attends to all its keys
    evenly.  Packed: [total, heads, 64] with cu_seqlens int32 [batch + 1] (non-decreasing) and max_seqlen, the longest
    sequence (None: read back from the GPU); rows of no sequence come out as zeros.
    Views of a fused projection, qkv.unbind(-3), are read in place.  scale: 1 / 8 by default.
    lse (float32 [batch, heads, tokens] / [heads, total]) is what the backward pass needs."""
    return _lib.calls().attention_forward(q, k, v, mask, cu_seqlens, _longest(cu_seqlens, max_seqlen), dropout_p, seed, call,
                                          scale)


def attention_backward(dout, q, k, v, out, lse, mask=None, cu_seqlens=None, max_seqlen=None, dropout_p=0.0, seed=None, call=0,
                       scale=None, grads=None):
    """Gradients (dq, dk, dv) of attention_forward, whose other arguments must be given again.  grads: three tensors to
    write them to, for instance the views dqkv.unbind(-3) of one buffer; they may not overlap each other or an operand."""
    return _lib.calls().attention_backward(dout, out, lse, grads, q, k, v, mask, cu_seqlens, _longest(cu_seqlens, max_seqlen),
                                           dropout_p, seed, call, scale)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, cu_seqlens, max_seqlen, dropout_p, seed, call, scale):
        max_seqlen = _longest(cu_seqlens, max_seqlen)
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
