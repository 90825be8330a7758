"""The 64-bit restatement of the training operators (oracle/training_ref.py) on the CPU: the generator against the published
vectors, every gradient against differences, and the refusals of the entry points, which come before any GPU work."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import training_ref as R
from otter_amd import _lib


def _rand(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64)


def test_philox_known_answers():
    """Vectors of the authors' Random123 distribution for 7 and 10 rounds."""
    assert [hex(int(x)) for x in R.philox(0, 0, 0, 0, 0, 7)] == ["0x5f6fb709", "0xd893f64", "0x4f121f81", "0x4f730a48"]
    assert [hex(int(x)) for x in R.philox(0, 0, 0, 0, 0, 10)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    m = 0xFFFFFFFF
    assert [hex(int(x)) for x in R.philox(m, m, m, m, (m << 32) | m, 10)] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


def test_draws_are_fair_and_differ():
    n = 512
    keep = [(R.score_factor(b, 2, n, 0.1, seed, call) > 0).double() for b, seed, call in ((0, 7, 0), (1, 7, 0), (0, 8, 0), (0, 7, 1))]
    keep.append((R.row_factor(n, 2 * n, 0.1, 7, 0) > 0).double().reshape(2, n, n))
    q = 1 - R.threshold(0.1) / 65536
    sd = (q * (1 - q)) ** 0.5
    for i, a in enumerate(keep):
        assert abs(a.mean() - q) < 5 * sd / a.numel() ** 0.5
        for b in keep[i + 1:]:
            assert abs(((a - q) * (b - q)).mean()) < 5 * sd * sd / a.numel() ** 0.5
    a = keep[0][0] - q                                        # neighbours in both directions and across a call's words
    for di, dj in ((0, 1), (1, 0), (1, 1), (0, 4), (2, 0)):
        x, y = a[:n - di, :n - dj], a[di:, dj:]
        assert abs((x * y).mean()) < 5 * sd * sd / x.numel() ** 0.5


def _differences(fn, inputs, grads, h=1e-6):
    """sum over one random direction of every input: <grad, dir> against the central difference of the scalar fn."""
    for i, (x, g) in enumerate(zip(inputs, grads)):
        if x is None:
            continue
        d = _rand(100 + i, *x.shape)
        hi, lo = (fn(*[t + s * h * d if j == i else t for j, t in enumerate(inputs)]) for s in (1, -1))
        num, ana = float(hi - lo) / (2 * h), float((g * d).sum())
        assert abs(num - ana) < 1e-6 * (1 + abs(ana)), (i, num, ana)


@pytest.mark.parametrize("p,residual", [(0.0, False), (0.3, True), (0.3, False)])
def test_layer_norm_gradients_match_differences(p, residual):
    x, r, dy = _rand(1, 5, 12), (_rand(2, 5, 12) if residual else None), _rand(3, 5, 12)
    w, b = 1 + 0.1 * _rand(4, 12), _rand(5, 12)

    def run(x, w, b, r):
        return R.layer_norm(x, w, b, 1e-5, r, p, 11, 3, dy, torch.float32, torch.float32)

    o = run(x, w, b, r)
    _differences(lambda *t: (run(*t)["y"][0] * dy).sum(), (x, w, b, r),
                 (o["dx"][0], o["dweight"][0], o["dbias"][0], o["dresidual"][0]))


@pytest.mark.parametrize("p,keys", [(0.0, "all"), (0.3, "all"), (0.3, "some"), (0.3, "none")])
def test_attention_gradients_match_differences(p, keys):
    H, n = 2, 9
    q, k, v, do = (_rand(i, H, n, 64) for i in range(4))
    key = torch.ones(n, dtype=torch.bool)
    if keys == "some":
        key[[0, 4, 8]] = False
    elif keys == "none":
        key[:] = False

    def run(q, k, v):
        return R.attention_sequence(q, k, v, key, p, 5, 2, 1, do, 0.125, torch.float32)

    o = run(q, k, v)
    _differences(lambda *t: (run(*t)["out"][0] * do).sum(), (q, k, v), (o["dq"][0], o["dk"][0], o["dv"][0]))
    if keys == "some":
        assert (o["dk"][0][:, ~key] == 0).all() and (o["dv"][0][:, ~key] == 0).all()


@pytest.mark.parametrize("B,neg", [(1, True), (6, False), (6, True)])
def test_inbatch_loss_gradients_match_differences(B, neg):
    q, c, n = _rand(1, B, 7), _rand(2, B, 7), (_rand(3, B, 7) if neg else None)
    o = R.inbatch_loss(q, c, n, 1.7)
    _differences(lambda *t: 1.7 * R.inbatch_loss(*t)["loss"][0], (q, c, n),
                 (o["dq"][0], o["dc"][0], o["dneg"][0] if neg else None))


def test_inbatch_loss_matches_the_reference_golden():
    """The number the reference's loss_single returned for the golden batches (oracle/gen_inbatch_golden.py)."""
    import os
    g = np.load(os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "inbatch.npz"))
    for n in ("a", "b"):
        o = R.inbatch_loss(*(torch.from_numpy(g[n + s]).double() for s in ("_q", "_c", "_neg")))
        # the golden was computed in float32: d + B + a few half steps of the largest scores
        tol = 2.0 ** -24 * (g[n + "_q"].shape[1] + 64) * float(o["product"][0].abs().max())
        assert abs(float(o["loss"][0]) - float(g[n + "_loss"])) <= tol


# ----------------------------------------------------------------------------------------------- refusals (no GPU needed)
def _fails(rc, text):
    assert rc == _lib.OTTER_EINVAL or rc == _lib.OTTER_ENOTIMPL, rc
    assert text in _lib.load().otter_last_error().decode(), _lib.load().otter_last_error()


def test_row_entry_points_refuse_bad_calls():
    lib = _lib.load()
    P = ctypes.c_void_p(4096)                                  # never followed: every call below is refused first
    _fails(lib.otter_dropout(0, 7, P, P, 1, 8, 0.1, P, 0, None), "dtype")
    _fails(lib.otter_dropout(0, 0, P, P, -1, 8, 0.1, P, 0, None), "rows")
    _fails(lib.otter_dropout(0, 0, P, P, 1 << 32, 8, 0.1, P, 0, None), "rows")
    for p in (1.0, -0.1, float("nan"), 0.999999):
        _fails(lib.otter_dropout(0, 0, P, P, 1, 8, p, P, 0, None), "probability")
    _fails(lib.otter_dropout(0, 0, P, P, 1, 8, 0.1, None, 0, None), "seed")
    _fails(lib.otter_dropout(0, 0, None, P, 1, 8, 0.1, P, 0, None), "NULL")
    assert lib.otter_dropout(0, 0, None, None, 0, 8, 0.1, P, 0, None) == 0

    def fwd(dtype=0, wdtype=0, x=P, rows=1, cols=8, eps=1e-5, p=0.0, seed=None):
        return lib.otter_layernorm_forward(0, dtype, wdtype, x, None, P, P, rows, cols, eps, p, seed, 0, P, P, P, None)

    _fails(fwd(dtype=2), "dtype")
    _fails(fwd(wdtype=3), "dtype")
    _fails(fwd(cols=0), "cols")
    _fails(fwd(cols=8193), "8192")
    _fails(fwd(eps=-1.0), "eps")
    _fails(fwd(eps=float("nan")), "eps")
    _fails(fwd(p=0.5), "seed")
    _fails(fwd(x=None), "NULL")
    assert fwd(rows=0) == 0
    need = lib.otter_layernorm_backward_workspace(100, 768)
    assert need > 0 and lib.otter_layernorm_backward_workspace(0, 768) == 0
    _fails(lib.otter_layernorm_backward_workspace(1, 0), "cols")

    def bwd(dres=None, res=None, ws=need, dw=P):
        return lib.otter_layernorm_backward(0, 0, 0, P, P, res, P, P, P, 100, 768, 0.0, None, 0, P, dres, dw, P, P, ws, None)

    _fails(bwd(ws=need - 1), "workspace")
    _fails(bwd(dres=P), "residual")
    _fails(bwd(dw=None), "NULL")


def test_attention_entry_points_refuse_bad_calls():
    lib = _lib.load()

    def args(**kw):
        a = _lib.AttentionArgs()
        a.dtype, a.batch, a.tokens, a.heads, a.head_dim, a.scale = 0, 1, 4, 2, 64, 0.125
        for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
            setattr(a, n, _lib.View(4096, 512, 128, 64))
        a.lse = a.workspace = 4096
        a.workspace_bytes = 1 << 20
        for n, x in kw.items():
            setattr(a, n, x)
        return ctypes.byref(a)

    for fn in (lib.otter_attention_forward, lib.otter_attention_backward):
        _fails(fn(0, None, None), "NULL")
        _fails(fn(0, args(dtype=2), None), "dtype")
        _fails(fn(0, args(head_dim=32), None), "head dimension")
        _fails(fn(0, args(batch=-1), None), "batch")
        _fails(fn(0, args(heads=0), None), "heads")
        _fails(fn(0, args(mask=4096, cu_seqlens=4096, total=4), None), "exclude")
        _fails(fn(0, args(cu_seqlens=4096, total=1 << 31), None), "total")
        _fails(fn(0, args(dropout_p=0.5), None), "seed")
        _fails(fn(0, args(dropout_p=1.0, seed=4096), None), "probability")
        _fails(fn(0, args(scale=float("nan")), None), "scale")
        _fails(fn(0, args(batch=1 << 20, heads=1 << 12), None), "too large")
        _fails(fn(0, args(v=_lib.View(None, 512, 128, 64)), None), "v must be")
        _fails(fn(0, args(q=_lib.View(4100, 512, 128, 64)), None), "16-byte")
        _fails(fn(0, args(k=_lib.View(4096, 512, 129, 64)), None), "16 bytes")
        _fails(fn(0, args(lse=None), None), "lse")
        assert fn(0, args(tokens=0), None) == 0 and fn(0, args(batch=0), None) == 0
    _fails(lib.otter_attention_backward(0, args(workspace_bytes=4 * 2 * 4 - 1), None), "workspace")
    _fails(lib.otter_attention_backward(0, args(dv=_lib.View(None, 0, 0, 0)), None), "dv must be")
    assert lib.otter_attention_backward_workspace(args()) >= 4 * 2 * 4


def test_inbatch_loss_entry_points_refuse_bad_calls():
    lib = _lib.load()
    P = ctypes.c_void_p(4096)
    need = lib.otter_inbatch_loss_workspace(4, 8)
    assert need >= 16
    _fails(lib.otter_inbatch_loss_workspace(0, 8), "B=0")

    def fwd(q=P, neg=None, B=4, d=8, ld=4, ws=need):
        return lib.otter_inbatch_loss_forward(0, q, P, neg, B, d, P, ld, P, P, P, ws, None)

    _fails(fwd(B=0), "mean over no rows")
    _fails(fwd(d=0), "d=0")
    _fails(fwd(B=65537, ld=65537), "65536")
    _fails(fwd(ld=3), "ld=3")
    _fails(fwd(neg=P), "ld=4")
    _fails(fwd(q=None), "NULL")
    _fails(fwd(ws=need - 1), "workspace")

    def bwd(dl=P, neg=None, dneg=None, ld=8):
        return lib.otter_inbatch_loss_backward(0, dl, P, P, neg, 4, 8, P, ld, P, P, P, dneg, None, 0, None)

    _fails(bwd(dl=None), "NULL")
    _fails(bwd(neg=P), "NULL")
    _fails(bwd(ld=2), "ld=2")
    need = lib.otter_inbatch_loss_backward_workspace(600, 64)
    assert need > 0 and lib.otter_inbatch_loss_backward_workspace(4, 8) == 0
    _fails(lib.otter_inbatch_loss_backward(0, P, P, P, None, 600, 64, P, 600, P, P, P, None, P, need - 1, None), "workspace")
    _fails(lib.otter_inbatch_loss_backward(0, P, P, P, None, 600, 64, P, 600, P, P, P, None, ctypes.c_void_p(4104), need, None), "aligned")


def test_python_entry_points_refuse_cpu_tensors():
    from otter_amd import inbatch, training as T
    x = torch.zeros(2, 8)
    q = torch.zeros(1, 2, 1, 64)
    for call in (lambda: T.dropout(x, 0.1, torch.zeros(1, dtype=torch.int64)),
                 lambda: T.layer_norm(x, torch.ones(8), torch.zeros(8)),
                 lambda: T.attention(q, q, q),
                 lambda: inbatch.inbatch_loss(x, x)):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()


def test_call_module_is_bound_to_the_library():
    """otter_amd._calls: wrong argument counts and errors of the library's own checks come out as Python exceptions."""
    m = _lib.calls()
    assert m is _lib.calls()
    with pytest.raises(TypeError, match="arguments"):
        m.dropout_forward(1)
    with pytest.raises(RuntimeError, match="no_such_library"):
        m.load("/no_such_library.so", _lib.check, None)
    with pytest.raises(ValueError, match="no CPU fallback"):
        m.dropout_forward(torch.zeros(2, 8), 0.1, None, 0, None)
