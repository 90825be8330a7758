"""The training operators on the GPU against their 64-bit restatement (oracle/training_ref.py), each output element within the
bound that is derived there from the operator's documented roundings."""
import numpy as np
import pytest
import torch

from oracle import training_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
SEED = 0x1234_5678_9ABC_DEF


def _dev():
    return torch.device("cuda:0")


def _seed(value=SEED):
    return torch.tensor([value], dtype=torch.int64, device=_dev())


def _rand(seed, *shape, dtype=F32, scale=1.0):
    """Values of the type itself (rounded before any computation), on the CPU in float64 and on the GPU."""
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype)
    return t.double(), t.to(_dev())


def _close(name, got, ref, where=None):
    val, bound = ref
    err = (got.detach().double().cpu() - val).abs()
    assert got.shape == val.shape, (name, got.shape, val.shape)
    ok = err <= bound
    if where is not None:
        ok = ok | ~where
    assert bool(ok.all()), "%s: %d of %d outside, worst error %g where %g is allowed" % (
        name, int((~ok).sum()), ok.numel(), float(err[~ok].max()), float(bound[~ok].min()))


def _same(a, b):
    for x, y in zip(a, b):
        if x is not None:
            assert torch.equal(x.reshape(-1).view(torch.uint8), y.reshape(-1).view(torch.uint8))


# ------------------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,p", [((1, 1), 0.5), ((3, 7), 0.1), ((5, 8), 0.9), ((64, 768), 0.1), ((17, 771), 0.3),
                                     ((1000,), 0.1), ((2, 3, 40), 0.25), ((4, 0), 0.1), ((0, 8), 0.1), ((), 0.5),
                                     ((70000, 16), 0.1), ((3, 100003), 0.1), ((9, 8), 1e-6)])
def test_dropout_is_exact(dtype, shape, p):
    from otter_amd import training as T
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    cols = shape[-1] if shape else 1
    rows = x.numel() // cols if cols else 0
    f = R.row_factor(rows, cols, p, SEED, 9).reshape(shape) if x.numel() else torch.zeros(shape, dtype=torch.float64)
    # one float32 product with the scale rounded to float32, one rounding to the type
    exp = (x.float() * f.float()).to(dtype)
    y = T.dropout_forward(x.to(_dev()), p, _seed(), 9)
    assert y.dtype == dtype and torch.equal(y.cpu(), exp)
    assert torch.equal(T.dropout_backward(x.to(_dev()), p, _seed(), 9).cpu(), exp)


def test_dropout_unaligned_strided_in_place_and_special_values():
    from otter_amd import training as T
    dev = _dev()
    base = torch.randn(8 * 16 + 1, device=dev, dtype=BF16)
    x = base[1:].view(8, 16)                                    # 2-byte aligned
    f = R.row_factor(8, 16, 0.3, SEED, 0).float().to(dev)
    assert torch.equal(T.dropout_forward(x, 0.3, _seed()), (x.float() * f).to(BF16))
    t = torch.randn(16, 8, device=dev).t()                      # not contiguous
    assert torch.equal(T.dropout_forward(t, 0.3, _seed()), t * f)
    z = torch.randn(8, 16, device=dev)
    exp = z * f
    assert T.dropout_forward(z, 0.3, _seed(), out=z) is z and torch.equal(z, exp)
    bad = torch.full((8, 16), float("nan"), device=dev)
    y = T.dropout_forward(bad, 0.3, _seed())
    assert (y[f == 0] == 0).all() and torch.isnan(y[f != 0]).all()
    assert torch.equal(T.dropout_forward(z, 0.0, None), z)
    seeds = [T.dropout_forward(torch.ones(64, 64, device=dev), 0.5, _seed(s), c) for s, c in ((1, 0), (2, 0), (1, 1), (-1, 0))]
    assert all(not torch.equal(seeds[0], o) for o in seeds[1:])
    assert torch.equal(seeds[3].cpu() > 0, R.row_factor(64, 64, 0.5, -1 & (2 ** 64 - 1), 0) > 0)


def test_dropout_autograd():
    from otter_amd import training as T
    x = torch.randn(6, 24, device=_dev(), requires_grad=True)
    s = _seed()
    y = T.dropout(x, 0.4, s, call=2)
    g = torch.randn_like(y)
    dx, = torch.autograd.grad(y, x, g)
    assert torch.equal(dx, T.dropout_backward(g, 0.4, s, call=2))
    y = T.dropout(x, 0.4, s, call=2)
    s.add_(1)                                                   # the seed of a pass must live until its backward pass
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = T.dropout(x, 0.4, s, call=2).sum()
    dx, = torch.autograd.grad(y, x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()                                     # first order only


# --------------------------------------------------------------------------------------------------------- layer norm
NORM = [(1, 1, 0.0, False), (1, 8, 0.0, True), (3, 7, 0.3, True), (5, 255, 0.1, False), (9, 256, 0.1, True), (70, 512, 0.1, True),
        (33, 768, 0.1, True), (1, 768, 0.0, False), (40, 771, 0.0, False), (17, 1000, 0.5, True), (16, 1024, 0.1, True),
        (5, 1025, 0.1, True), (7, 2048, 0.0, True), (3, 4099, 0.1, True), (2, 8192, 0.1, True), (9000, 64, 0.1, True),
        (2600, 1032, 0.1, False)]


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("rows,cols,p,residual", NORM)
def test_layer_norm(rows, cols, p, residual, dtype, wdtype):
    from otter_amd import training as T
    x64, x = _rand(1, rows, cols, dtype=dtype)
    r64, r = _rand(2, rows, cols, dtype=dtype) if residual else (None, None)
    dy64, dy = _rand(3, rows, cols, dtype=dtype)
    w64, w = _rand(4, cols, dtype=wdtype)
    b64, b = _rand(5, cols, dtype=wdtype)
    kw = dict(residual=r, dropout_p=p, seed=_seed() if p else None, call=3)
    ref = R.layer_norm(x64, w64, b64, 1e-5, r64, p, SEED, 3, dy64, dtype, wdtype)
    y, mean, rstd = T.layer_norm_forward(x, w, b, eps=1e-5, **kw)
    dx, dres, dw, db = T.layer_norm_backward(dy, x, w, mean, rstd, **kw)
    got = {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dweight": dw, "dbias": db}
    if residual:
        got["dresidual"] = dres
    assert y.dtype == dx.dtype == dtype and dw.dtype == db.dtype == wdtype
    for name, t in got.items():
        _close(name, t, ref[name])
    _same(T.layer_norm_backward(dy, x, w, mean, rstd, **kw), (dx, dres, dw, db))


def test_layer_norm_shapes_strides_and_empty():
    from otter_amd import training as T
    dev = _dev()
    x = torch.randn(4, 6, 40, device=dev)
    w, b = torch.randn(40, device=dev), torch.randn(40, device=dev)
    y, mean, rstd = T.layer_norm_forward(x.transpose(0, 1), w, b)
    z, *_ = T.layer_norm_forward(x, w, b)
    assert y.shape == (6, 4, 40) and mean.shape == (6, 4) and torch.equal(y, z.transpose(0, 1))
    u = torch.randn(4 * 40 + 1, device=dev)[1:].view(4, 40)     # 4-byte aligned
    assert torch.equal(T.layer_norm_forward(u, w, b)[0], T.layer_norm_forward(u.clone(), w, b)[0])
    # the bits of a row do not depend on its alignment, with everything switched on either
    for dt in (F32, BF16):
        g = torch.Generator(device=dev).manual_seed(7)
        big = [torch.randn(300 * 768 + 1, generator=g, device=dev).to(dt) for _ in range(3)]
        w2, b2 = torch.randn(768, generator=g, device=dev), torch.randn(768, generator=g, device=dev)
        res = []
        for o in (0, 1):
            x2, r2, d2 = (t[1:].view(300, 768) if o else t[1:].clone().view(300, 768) for t in big)
            kw = dict(residual=r2, dropout_p=0.2, seed=_seed(), call=4)
            f = T.layer_norm_forward(x2, w2, b2, **kw)
            res.append((*f, *T.layer_norm_backward(d2, x2, w2, f[1], f[2], **kw)))
        _same(res[0], res[1])
    y, mean, rstd = T.layer_norm_forward(x[:0], w, b)
    dx, dres, dw, db = T.layer_norm_backward(x[:0], x[:0], w, mean, rstd)
    assert y.shape == dx.shape == (0, 6, 40) and dres is None and (dw == 0).all() and (db == 0).all()
    # fused dropout and residual = the separate calls
    s, r = _seed(), torch.randn(4, 6, 40, device=dev)
    a = T.layer_norm_forward(x, w, b, residual=r, dropout_p=0.2, seed=s, call=4)[0]
    assert torch.allclose(a, T.layer_norm_forward(T.dropout_forward(x, 0.2, s, 4) + r, w, b)[0], rtol=0, atol=1e-5)
    # a constant row: no variance, y = bias
    one = T.layer_norm_forward(torch.full((2, 40), 3.0, device=dev), w, b)[0]
    assert torch.equal(one, b.expand(2, 40))


def test_layer_norm_autograd():
    from otter_amd import training as T
    dev = _dev()
    x, r = torch.randn(5, 64, device=dev, requires_grad=True), torch.randn(5, 64, device=dev, requires_grad=True)
    w, b = torch.randn(64, device=dev, requires_grad=True), torch.randn(64, device=dev, requires_grad=True)
    g, s = torch.randn(5, 64, device=dev), _seed()
    for p in (0.0, 0.25):
        y = T.layer_norm(x, w, b, 1e-5, r, p, s, 1)
        got = torch.autograd.grad(y, (x, r, w, b), g)
        ref = R.layer_norm(*(t.detach().double().cpu() for t in (x, w, b)), 1e-5, r.detach().double().cpu(), p, SEED, 1,
                           g.double().cpu(), F32, F32)
        for name, t in zip(("dx", "dresidual", "dweight", "dbias"), got):
            _close(name, t, ref[name])
    # one tensor as input and residual: its gradient is the sum
    y = T.layer_norm(x, w, b, 1e-5, x, 0.0)
    dx, = torch.autograd.grad(y, x, g)
    ref = R.layer_norm(*(t.detach().double().cpu() for t in (x, w, b)), 1e-5, x.detach().double().cpu(), 0.0, SEED, 1,
                       g.double().cpu(), F32, F32)
    v, e = ref["dx"]
    _close("dx", dx, (2 * v, 2 * e + 4 * R.E32 * v.abs()))


# ---------------------------------------------------------------------------------------------------------- attention
def _check_attention(q, k, v, do, kw, mask=None, cu=None, p=0.0, call=6, scale=0.125):
    """q, k, v, do: (float64 on the CPU, GPU tensor) pairs."""
    from otter_amd import training as T
    dtype = q[1].dtype
    ref = R.attention(q[0], k[0], v[0], mask, cu, p, SEED, call, do[0], scale, dtype)
    out, lse = T.attention_forward(q[1], k[1], v[1], **kw)
    assert out.dtype == dtype and out.is_contiguous() and lse.dtype == F32
    grads = T.attention_backward(do[1], q[1], k[1], v[1], out, lse, **kw)
    for name, t in (("out", out), ("lse", lse), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        _close(name, t, ref[name])
    out2, lse2 = T.attention_forward(q[1], k[1], v[1], **kw)
    _same((out2, lse2, *T.attention_backward(do[1], q[1], k[1], v[1], out, lse, **kw)), (out, lse, *grads))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H,p", [(40, 33, 8, 0.1), (40, 70, 8, 0.1), (300, 3, 1, 0.1), (1, 1, 1, 0.0), (1, 1, 1, 0.5), (2, 2, 3, 0.1), (1, 31, 2, 0.1), (2, 32, 1, 0.1), (1, 33, 2, 0.0),
                                     (2, 63, 1, 0.1), (1, 64, 2, 0.1), (3, 65, 2, 0.1), (2, 70, 12, 0.1), (1, 127, 2, 0.1),
                                     (1, 129, 1, 0.3), (1, 255, 2, 0.1), (1, 257, 2, 0.1), (1, 512, 2, 0.1), (1, 513, 1, 0.1),
                                     (2, 300, 2, 0.0), (1, 1100, 1, 0.1)])
def test_attention_dense(B, L, H, p, dtype):
    x = [_rand(10 + i, B, L, H, 64, dtype=dtype) for i in range(4)]
    _check_attention(*x, dict(dropout_p=p, seed=_seed() if p else None, call=6), p=p)


MASKS = ["prefix", "holes", "first", "last", "tile", "none", "alternate"]


def _mask(kind, B, L):
    m = torch.zeros((B, L), dtype=torch.int64)
    for b in range(B):
        if kind == "prefix":
            m[b, :max(1, L - 37 * (b % 9))] = 1
        elif kind == "holes":
            m[b] = (torch.rand(L, generator=torch.Generator().manual_seed(b)) < 0.5).long()
        elif kind == "first":
            m[b, 0] = 1
        elif kind == "last":
            m[b, L - 1] = 1
        elif kind == "tile":                                    # a whole tile of 64 keys left out in the middle
            m[b] = 1
            m[b, 64:128] = 0
        elif kind == "alternate":                               # sequences that leave nothing beside ones that do
            m[b, :L // 2] = b % 2
    return m


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("B,L", [(3, 70), (130, 70), (3, 200), (3, 530)])
def test_attention_masks(kind, B, L, dtype):
    H, p = 2, 0.1
    m = _mask(kind, B, L)
    x = [_rand(20 + i, B, L, H, 64, dtype=dtype) for i in range(4)]
    _check_attention(*x, dict(mask=m.to(_dev()), dropout_p=p, seed=_seed(), call=6), mask=m, p=p)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_keys_reach_nothing_whatever_they_hold(dtype):
    from otter_amd import training as T
    B, L, H = 2, 150, 2
    m = _mask("holes", B, L)
    x = [_rand(30 + i, B, L, H, 64, dtype=dtype) for i in range(4)]
    kw = dict(mask=m.to(_dev()), dropout_p=0.1, seed=_seed(), call=6)
    q, k, v, do = (t[1] for t in x)
    out, lse = T.attention_forward(q, k, v, **kw)
    grads = T.attention_backward(do, q, k, v, out, lse, **kw)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        k2, v2 = k.clone(), v.clone()
        k2[m.to(_dev()) == 0] = bad
        v2[m.to(_dev()) == 0] = bad
        out2, lse2 = T.attention_forward(q, k2, v2, **kw)
        _same((out2, lse2, *T.attention_backward(do, q, k2, v2, out2, lse2, **kw)), (out, lse, *grads))
    # bool and int32 masks mean the same
    for mm in (m.bool(), m.int(), 5 * m):
        _same(T.attention_forward(q, k, v, **dict(kw, mask=mm.to(_dev()))), (out, lse))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,lead,tail,hint", [([5], 0, 0, None), ([1, 0, 3, 64, 65, 0], 0, 7, None), ([200, 130, 1], 0, 0, 200),
                                                 ([300, 20], 3, 100, 300), ([0, 0], 0, 4, 0), ([150, 40], 0, 0, 40),
                                                 ([512, 530, 600], 0, 5, 600)])
def test_attention_packed(lens, lead, tail, hint, dtype):
    """lead / tail: rows of no sequence in front and behind (zeros in every output); hint: max_seqlen, once too small."""
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    total, H, p = cu[-1] + tail, 2, 0.1
    x = [_rand(40 + i, total, H, 64, dtype=dtype) for i in range(4)]
    for t64, t in x:                                            # what those rows hold reaches nothing
        for rows in (slice(0, lead), slice(cu[-1], total)):
            t64[rows] = 0
            t[rows] = float("nan")
    cut = torch.tensor(cu, dtype=torch.int32, device=_dev())
    _check_attention(*x, dict(cu_seqlens=cut, max_seqlen=hint, dropout_p=p, seed=_seed(), call=6), cu=cu, p=p)


# Many heads and sequences of more than 128: the backward pass in one pass over the scores, keys 256 at a time
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("L,kind", [(129, None), (256, "prefix"), (257, "holes"), (290, "tile"), (300, "first"), (300, "last"),
                                    (300, "alternate"), (260, "none"), (520, "prefix"), (545, None)])
def test_attention_one_pass_dense(L, kind, p):
    B, H = 4, 64
    m = None if kind is None else _mask(kind, B, L)
    x = [_rand(100 + i, B, L, H, 64, dtype=BF16) for i in range(4)]
    kw = dict(dropout_p=p, seed=_seed() if p else None, call=6)
    if m is not None:
        kw["mask"] = m.to(_dev())
    _check_attention(*x, kw, mask=m, p=p)


@pytest.mark.parametrize("lens,lead,tail,hint", [([300, 20, 1, 256], 0, 0, 300), ([0, 257, 130, 5], 3, 70, None), ([150, 520, 40, 33], 0, 2, 150)])
def test_attention_one_pass_packed(lens, lead, tail, hint):
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    total, H, p = cu[-1] + tail, 64, 0.1
    x = [_rand(110 + i, total, H, 64, dtype=BF16) for i in range(4)]
    for t64, t in x:
        for rows in (slice(0, lead), slice(cu[-1], total)):
            t64[rows] = 0
            t[rows] = float("nan")
    cut = torch.tensor(cu, dtype=torch.int32, device=_dev())
    _check_attention(*x, dict(cu_seqlens=cut, max_seqlen=hint, dropout_p=p, seed=_seed(), call=6), cu=cu, p=p)


def test_one_pass_masked_keys_reach_nothing_whatever_they_hold():
    from otter_amd import training as T
    B, L, H = 4, 270, 64
    m = _mask("holes", B, L).to(_dev())
    m[3] = 0
    x = [torch.randn(B, L, H, 64, device=_dev()).to(BF16) for _ in range(4)]
    q, k, v, do = x
    kw = dict(mask=m, dropout_p=0.1, seed=_seed(), call=6)
    out, lse = T.attention_forward(q, k, v, **kw)
    grads = T.attention_backward(do, q, k, v, out, lse, **kw)
    for bad in (float("nan"), float("inf"), torch.finfo(BF16).min):
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        live = m.any(1, keepdim=True).expand_as(m)
        k2[m == 0] = bad                                        # of the sequence that leaves nothing: k and q, not v
        v2[(m == 0) & live] = bad
        q2[3] = bad
        out2, lse2 = T.attention_forward(q2, k2, v2, **kw)
        _same((out2, lse2, *T.attention_backward(do, q2, k2, v2, out2, lse2, **kw)), (out, lse, *grads))


def test_packed_and_dense_agree_bit_for_bit():
    from otter_amd import training as T
    dev, H = _dev(), 3
    lens = [70, 1, 33, 128]
    L = max(lens)
    qkv = torch.randn(len(lens), L, 3, H, 64, device=dev, dtype=BF16)
    m = (torch.arange(L)[None, :] < torch.tensor(lens)[:, None]).to(dev)
    packed = qkv[m]
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=dev)
    kw = dict(dropout_p=0.1, seed=_seed(), call=1)
    out, lse = T.attention_forward(*packed.unbind(-3), cu_seqlens=cu, max_seqlen=L, **kw)
    d_out, d_lse = T.attention_forward(*qkv.unbind(-3), mask=m, **kw)
    assert torch.equal(out, d_out[m]) and torch.equal(lse, d_lse.transpose(1, 2)[m].t())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_strides_and_gradient_buffers(dtype):
    from otter_amd import training as T
    dev, B, L, H = _dev(), 2, 90, 3
    kw = dict(dropout_p=0.1, seed=_seed(), call=1)
    qkv = torch.randn(B, L, 3, H, 64, device=dev).to(dtype)
    do = torch.randn(B, L, H, 64, device=dev).to(dtype)
    q, k, v = (t.contiguous() for t in qkv.unbind(-3))
    out, lse = T.attention_forward(q, k, v, **kw)
    grads = T.attention_backward(do, q, k, v, out, lse, **kw)
    # views of one buffer, in and out
    buf = torch.full((B, L, 3, H, 64), 7.0, device=dev, dtype=dtype)
    got = T.attention_backward(do, *qkv.unbind(-3), out, lse, grads=buf.unbind(-3), **kw)
    _same(got, grads)
    _same(buf.unbind(-3), grads)
    # heads in front of tokens, head dimension not contiguous, 2- / 4-byte aligned data, broadcast batch
    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def odd(t):
        s = torch.empty(t.numel() + 1, device=dev, dtype=dtype)[1:].view(t.shape)
        return s.copy_(t)

    for f in (heads_first, odd, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        o2, l2 = T.attention_forward(f(q), f(k), f(v), **kw)
        _same((o2, l2, *T.attention_backward(f(do), f(q), f(k), f(v), f(out), lse, **kw)), (out, lse, *grads))
    ke = k[:1].expand(B, L, H, 64)
    _same(T.attention_forward(q, ke, v, **kw), T.attention_forward(q, ke.contiguous(), v, **kw))


def test_attention_large_scores_and_scale():
    """Scores of several hundred, a scale of one's own; one key far above the others."""
    q, k, v, do = (_rand(50 + i, 1, 100, 2, 64, scale=s) for i, s in enumerate((6.0, 6.0, 1.0, 1.0)))
    _check_attention(q, k, v, do, dict(scale=0.3), scale=0.3)
    _check_attention(q, k, v, do, dict(scale=-0.01), scale=-0.01)
    _check_attention(q, k, v, do, dict(scale=0.0), scale=0.0)
    m = _mask("holes", 1, 100)
    for scale in (0.0, -0.3, 0.3):
        _check_attention(q, k, v, do, dict(scale=scale, mask=m.to(_dev())), mask=m, scale=scale)
    # scores far below zero throughout
    low = (q[0].abs(), q[1].abs()), (-k[0].abs(), -k[1].abs())
    _check_attention(*low, v, do, dict(mask=m.to(_dev())), mask=m)
    low = [tuple(t[0].to(BF16).double() if i == 0 else t[1].to(BF16) for i in range(2)) for t in (*low, v, do)]
    _check_attention(*low, dict(mask=m.to(_dev())), mask=m)


def test_attention_autograd_and_broadcast_inputs():
    from otter_amd import training as T
    dev = _dev()
    q64, q = _rand(60, 2, 40, 2, 64)
    k64, k = _rand(61, 1, 40, 2, 64)
    v64, v = _rand(62, 2, 40, 2, 64)
    d64, do = _rand(63, 2, 40, 2, 64)
    q, k, v = q.requires_grad_(), k.requires_grad_(), v.requires_grad_()
    out = T.attention(q, k.expand(2, 40, 2, 64), v, dropout_p=0.2, seed=_seed(), call=2)
    got = torch.autograd.grad(out, (q, k, v), do)
    ref = R.attention(q64, k64.expand(2, 40, 2, 64), v64, None, None, 0.2, SEED, 2, d64, 0.125, F32)
    _close("dq", got[0], ref["dq"])
    _close("dv", got[2], ref["dv"])
    val, bound = ref["dk"]
    total = val.sum(0, keepdim=True)
    _close("dk", got[1], (total, bound.sum(0, keepdim=True) + 2 * R.E32 * total.abs()))
    # packed, length read back
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=dev)
    x = q.detach()[0].requires_grad_()
    o = T.attention(x, x, x, cu_seqlens=cu)
    g, = torch.autograd.grad(o, x, do[0])
    ref = R.attention(q64[0], q64[0], q64[0], None, [0, 30, 40], 0.0, SEED, 0, d64[0], 0.125, F32)
    val = sum(ref[n][0] for n in ("dq", "dk", "dv"))
    _close("dx", g, (val, sum(ref[n][1] for n in ("dq", "dk", "dv")) + 4 * R.E32 * sum(ref[n][0].abs() for n in ("dq", "dk", "dv"))))


def test_attention_refusals():
    from otter_amd import training as T
    dev = _dev()
    q = torch.zeros(2, 8, 2, 64, device=dev)
    with pytest.raises(ValueError, match="must all be"):
        T.attention(q, q[:, :4], q)
    with pytest.raises(ValueError, match="must all be"):
        T.attention(q[0], q[0], q[0])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        T.attention(q.half(), q.half(), q.half())
    with pytest.raises(ValueError, match="expected"):
        T.attention(q, q.bfloat16(), q)
    with pytest.raises(NotImplementedError, match="head dimension"):
        T.attention(*(torch.zeros(2, 8, 2, 32, device=dev),) * 3)
    with pytest.raises(ValueError, match="mask must be"):
        T.attention(q, q, q, mask=torch.ones(2, 7, device=dev))
    with pytest.raises(ValueError, match="needs seed"):
        T.attention(q, q, q, dropout_p=0.1)
    with pytest.raises(ValueError, match="needs seed"):
        T.attention(q, q, q, dropout_p=0.1, seed=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="not in"):
        T.attention(q, q, q, dropout_p=1.0, seed=_seed())
    with pytest.raises(ValueError, match="call"):
        T.attention(q, q, q, call=-1)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="exclude"):
        T.attention(q[0], q[0], q[0], cu_seqlens=cu, mask=torch.ones(1, 8, device=dev))
    with pytest.raises(ValueError, match="int32"):
        T.attention(q[0], q[0], q[0], cu_seqlens=cu.long())
    out, lse = T.attention_forward(q, q, q)
    with pytest.raises(ValueError, match="lse"):
        T.attention_backward(out, q, q, q, out, lse[:1])
    with pytest.raises(ValueError, match="grads"):
        T.attention_backward(out, q, q, q, out, lse, grads=(q[..., :32],) * 3)
    for shape in ((0, 8, 2, 64), (2, 0, 2, 64)):
        e = torch.zeros(shape, device=dev)
        o, l = T.attention_forward(e, e, e)
        assert o.shape == shape and all(g.shape == shape for g in T.attention_backward(e, e, e, e, o, l))


def test_attention_offsets_past_32_bits():
    """Rows more than 2^32 bytes (2^31 elements and more) apart."""
    from otter_amd import training as T
    dev, L = _dev(), 5
    step = (1 << 29) + 8                                        # elements between tokens
    buf = torch.empty(L * step, device=dev, dtype=BF16)
    x = torch.randn(1, L, 1, 64, device=dev).to(BF16)
    far = torch.as_strided(buf, (1, L, 1, 64), (L * step, step, 64, 1))
    far.copy_(x)
    out, lse = T.attention_forward(x, x, x)
    grads = T.attention_backward(x, x, x, x, out, lse)
    o2, l2 = T.attention_forward(far, far, far)
    g2 = T.attention_backward(far, far, far, far, out, lse, grads=tuple(
        torch.as_strided(buf, (1, L, 1, 64), (L * step, step, 64, 1), 64 * (i + 1)) for i in range(3)))
    _same((o2, l2, *g2), (out, lse, *grads))


# --------------------------------------------------------------------------------------------------------------- loss
@pytest.mark.parametrize("B,d,neg", [(1, 1, True), (1, 768, True), (2, 3, False), (7, 100, True), (16, 2304, True), (63, 64, False),
                                     (64, 768, True), (65, 770, True), (130, 257, True), (200, 2304, False), (513, 100, True),
                                     (700, 33, True), (1030, 96, False)])
def test_inbatch_loss(B, d, neg):
    from otter_amd import inbatch as IB
    q64, q = _rand(70, B, d, scale=d ** -0.25)
    c64, c = _rand(71, B, d, scale=d ** -0.25)
    n64, n = _rand(72, B, d, scale=d ** -0.25) if neg else (None, None)
    dloss = torch.tensor(1.7, device=_dev())
    ref = R.inbatch_loss(q64, c64, n64, float(dloss.double()))
    loss, product, stats = IB.inbatch_loss_forward(q, c, n)
    dq, dc, dneg = IB.inbatch_loss_backward(dloss, q, c, n, product, stats)
    got = {"loss": loss, "product": product, "lse": stats[0], "rest": stats[1], "dq": dq, "dc": dc}
    if neg:
        got["dneg"] = dneg
    for name, t in got.items():
        _close(name, t, ref[name])
    again = IB.inbatch_loss_forward(q, c, n)
    _same(again, (loss, product, stats))
    _same(IB.inbatch_loss_backward(dloss, q, c, n, product, stats), (dq, dc, dneg))
    # a contiguous copy of the scores does as well (rows that are not whole 16-byte pieces)
    _same(IB.inbatch_loss_backward(dloss, q, c, n, product.contiguous(), stats), (dq, dc, dneg))
    if B <= 513:                                                # the matrix of the dev-set evaluation, in the same order
        P, _ = IB.inbatch_scores(q, c, n)
        assert (P - product).abs().max().item() <= 2 * float(ref["product"][1].max())


@pytest.mark.parametrize("B", [2, 40, 640])
@pytest.mark.parametrize("margin", [5.0, 16.0, 40.0])
def test_inbatch_loss_of_confident_rows(B, margin):
    """Targets far above the other columns: a loss of e^-margin and gradients as small keep their relative precision."""
    from otter_amd import inbatch as IB
    c64 = torch.nn.functional.normalize(_rand(94, B, 128)[0], dim=1).float().double()
    q64 = (margin * c64).float().double()
    ref = R.inbatch_loss(q64, c64, None, 1.0)
    q, c = q64.float().to(_dev()), c64.float().to(_dev())
    loss, product, stats = IB.inbatch_loss_forward(q, c)
    dq, dc, _ = IB.inbatch_loss_backward(torch.ones((), device=_dev()), q, c, None, product, stats)
    for name, t in (("loss", loss), ("rest", stats[1]), ("dq", dq), ("dc", dc)):
        _close(name, t, ref[name])
    assert float(loss) > 0


@pytest.mark.parametrize("B", [40, 640])
@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e4])
def test_inbatch_loss_of_small_and_large_embeddings(B, scale):
    """q scaled down or up and c the other way round: the scores stay, the float16 planes have to follow the sizes."""
    from otter_amd import inbatch as IB
    q64, q = _rand(90, B, 128, scale=scale * 128 ** -0.25)
    c64, c = _rand(91, B, 128, scale=128 ** -0.25 / scale)
    ref = R.inbatch_loss(q64, c64, None, 1.0)
    loss, product, stats = IB.inbatch_loss_forward(q, c)
    dq, dc, _ = IB.inbatch_loss_backward(torch.ones((), device=_dev()), q, c, None, product, stats)
    for name, t in (("loss", loss), ("product", product), ("lse", stats[0]), ("dq", dq), ("dc", dc)):
        _close(name, t, ref[name])
    # rows of very different sizes
    row = torch.logspace(-3, 3, B, dtype=torch.float64)[:, None]
    q64, q = _rand(92, B, 128, scale=128 ** -0.25)
    q64 = (q64 * row).float().double()
    c64, c = _rand(93, B, 128, scale=1e-3)
    ref = R.inbatch_loss(q64, c64, None, 1.0)
    q = q64.float().to(_dev())
    loss, product, stats = IB.inbatch_loss_forward(q, c)
    dq, dc, _ = IB.inbatch_loss_backward(torch.ones((), device=_dev()), q, c, None, product, stats)
    for name, t in (("loss", loss), ("product", product), ("lse", stats[0]), ("dq", dq), ("dc", dc)):
        _close(name, t, ref[name])


def test_inbatch_loss_at_its_limit():
    """B = 65536: offsets past 32 bits; rows and columns here and there against 64 bits."""
    from otter_amd import inbatch as IB
    B, d, dev = 65536, 64, _dev()
    g = torch.Generator(device=dev).manual_seed(5)
    q, c = (torch.randn(B, d, generator=g, device=dev) * d ** -0.25 for _ in range(2))
    loss, product, stats = IB.inbatch_loss_forward(q, c)
    dq, dc, _ = IB.inbatch_loss_backward(torch.ones((), device=dev), q, c, None, product, stats)
    lse = stats[0]
    pick = torch.tensor([0, 1, 32767, 32768, 50001, 65535], device=dev)
    qd, cd = q.double(), c.double()
    S = qd[pick] @ cd.t()
    tol = (d + 8) * R.E32 * float(qd.abs().sum(1).max() * cd.abs().max())     # of a score, and of what follows from it
    assert (product[pick].double() - S).abs().max() <= tol
    assert (lse[pick].double() - torch.logsumexp(S, 1)).abs().max() <= tol + (B / 256 + 64) * R.E32
    rows = torch.logsumexp(qd[:4096] @ cd.t(), 1) - (qd[:4096] * cd[:4096]).sum(1)
    every = lse.double() - (qd * cd).sum(1)
    assert (every[:4096] - rows).abs().max() <= 2 * tol + (B / 256 + 64) * R.E32
    assert abs(loss.double() - every.mean()) <= tol
    G = torch.exp(S - lse[pick].double()[:, None])
    G[torch.arange(len(pick), device=dev), pick] -= 1
    Gc = torch.exp(qd @ cd[pick].t() - lse.double()[:, None])
    Gc[pick, torch.arange(len(pick), device=dev)] -= 1
    # a gradient's error: its G's relative one (a score's, twice) over all terms, and the sum's own over B of them
    rel = 4 * tol + (B / 64 + 64) * R.E32
    for got, ref, mag in ((dq[pick], G @ cd, G.abs() @ cd.abs()), (dc[pick], Gc.t() @ qd, Gc.abs().t() @ qd.abs())):
        assert ((got.double() * B - ref).abs() <= rel * mag).all()


def test_inbatch_loss_autograd_and_edges():
    from otter_amd import inbatch as IB
    dev = _dev()
    q64, q = _rand(80, 12, 40)
    c64, c = _rand(81, 12, 40)
    q, c = q.requires_grad_(), c.requires_grad_()
    loss = IB.inbatch_loss(q, c)
    dq, dc = torch.autograd.grad(3.0 * loss, (q, c))
    ref = R.inbatch_loss(q64, c64, None, 3.0)
    _close("dq", dq, ref["dq"])
    _close("dc", dc, ref["dc"])
    # bfloat16 embeddings: computed in float32, gradients in their own type
    qb, cb = q.detach().bfloat16().requires_grad_(), c.detach().bfloat16().requires_grad_()
    gb = torch.autograd.grad(IB.inbatch_loss(qb, cb), (qb, cb))
    ref = R.inbatch_loss(qb.detach().double().cpu(), cb.detach().double().cpu(), None, 1.0)
    for name, t in zip(("dq", "dc"), gb):
        assert t.dtype == BF16
        _close(name, t, (ref[name][0], ref[name][1] + R.half_step(BF16) * ref[name][0].abs()))
    # scores of thousands: the softmax is one-hot, the gradient exactly so
    big = torch.eye(8, device=dev) * 100.0
    loss, product, stats = IB.inbatch_loss_forward(big, big)
    assert loss.item() == 0.0 and all((g == 0).all() for g in IB.inbatch_loss_backward(torch.ones((), device=dev), big, big, None, product, stats)[:2])
    with pytest.raises(ValueError, match="mean over no rows"):
        IB.inbatch_loss(torch.zeros((0, 8), device=dev), torch.zeros((0, 8), device=dev))
    with pytest.raises(ValueError, match="B, d"):
        IB.inbatch_loss(torch.zeros((3, 8), device=dev), torch.zeros((4, 8), device=dev))
    with pytest.raises(ValueError, match="returned"):
        IB.inbatch_loss_backward(torch.ones((), device=dev), big, big, big, product, stats)


# ------------------------------------------------------------------------------------ streams, graphs and a whole layer
def _step(T, IB, W, x, mask, dy, seed):
    """One post-norm layer forward and backward with explicit calls; returns its output and all gradients."""
    B, L, D = x.shape
    H = D // 64
    p = 0.1
    e = T.dropout_forward(x, p, seed, call=0)
    qkv = (e @ W["qkv"]).view(B, L, 3, H, 64)
    ctx, lse = T.attention_forward(*qkv.unbind(2), mask=mask, dropout_p=p, seed=seed, call=1)
    a = ctx.view(B, L, D) @ W["o"]
    y, mean, rstd = T.layer_norm_forward(a, W["g"], W["b"], 1e-5, e, p, seed, 2)
    emb = y[:, 0].float()
    n = B // 2
    loss, product, stats = IB.inbatch_loss_forward(emb[:n], emb[n:])
    dq, dc, _ = IB.inbatch_loss_backward(torch.ones_like(loss), emb[:n], emb[n:], None, product, stats)
    dyy = dy.clone()
    dyy[:, 0] += torch.cat((dq, dc)).to(dy.dtype)
    da, de, dg, db = T.layer_norm_backward(dyy, a, W["g"], mean, rstd, e, p, seed, 2)
    dctx = (da @ W["o"].t().contiguous()).view(B, L, H, 64)
    dqkv = torch.empty_like(qkv)
    T.attention_backward(dctx, *qkv.unbind(2), ctx, lse, mask=mask, dropout_p=p, seed=seed, call=1, grads=dqkv.unbind(2))
    de = de + dqkv.view(B, L, 3 * D) @ W["qkv"].t().contiguous()
    dx = T.dropout_backward(de, p, seed, call=0)
    dWo = ctx.view(B * L, D).t().contiguous() @ da.view(B * L, D)
    return [y, loss, dx, dg, db, dWo]


def _layer(dtype, B=6, L=70, H=4):
    dev, D = _dev(), H * 64
    g = torch.Generator(device=dev).manual_seed(3)
    W = {"qkv": (torch.randn(D, 3 * D, generator=g, device=dev) * D ** -0.5).to(dtype),
         "o": (torch.randn(D, D, generator=g, device=dev) * D ** -0.5).to(dtype),
         "g": 1 + 0.1 * torch.randn(D, generator=g, device=dev), "b": 0.1 * torch.randn(D, generator=g, device=dev)}
    x = torch.randn(B, L, D, generator=g, device=dev).to(dtype)
    dy = torch.randn(B, L, D, generator=g, device=dev).to(dtype)
    mask = (torch.arange(L, device=dev)[None, :] < torch.tensor([L - 9 * b for b in range(B)], device=dev)[:, None]).long()
    return W, x, mask, dy


def test_a_layers_step_matches_64_bits_and_autograd():
    """Embedding dropout, attention, output projection, residual norm and the loss, forward and backward, in float32."""
    from otter_amd import inbatch as IB, training as T
    W, x, mask, dy = _layer(F32)
    B, L, D = x.shape
    H, p, seed = D // 64, 0.1, _seed()
    got = _step(T, IB, W, x, mask, dy, seed)
    # the same through autograd
    xa, wo = x.clone().requires_grad_(), W["o"].clone().requires_grad_()
    ga, ba = W["g"].clone().requires_grad_(), W["b"].clone().requires_grad_()
    e = T.dropout(xa, p, seed, 0)
    qkv = (e @ W["qkv"]).view(B, L, 3, H, 64)
    ctx = T.attention(*qkv.unbind(2), mask=mask, dropout_p=p, seed=seed, call=1)
    y = T.layer_norm(ctx.reshape(B, L, D) @ wo, ga, ba, 1e-5, e, p, seed, 2)
    loss = IB.inbatch_loss(y[:B // 2, 0], y[B // 2:, 0])
    auto = torch.autograd.grad((y * dy).sum() + loss, (xa, ga, ba, wo))
    # and in 64 bits by torch's own differentiation of the plain formulas
    x6, o6 = x.double().cpu().requires_grad_(), W["o"].double().cpu().requires_grad_()
    g6, b6 = W["g"].double().cpu().requires_grad_(), W["b"].double().cpu().requires_grad_()
    e6 = x6 * R.row_factor(B * L, D, p, SEED, 0).view(B, L, D)
    q6, k6, v6 = (t.transpose(1, 2) for t in (e6 @ W["qkv"].double().cpu()).view(B, L, 3, H, 64).unbind(2))
    f6 = torch.stack([R.score_factor(b, H, L, p, SEED, 1) for b in range(B)])
    s6 = (q6 @ k6.transpose(2, 3) / 8).masked_fill((mask == 0).cpu()[:, None, None, :], -1e300)
    c6 = ((torch.softmax(s6, -1) * f6) @ v6).transpose(1, 2).reshape(B, L, D)
    z6 = (c6 @ o6) * R.row_factor(B * L, D, p, SEED, 2).view(B, L, D) + e6
    y6 = torch.nn.functional.layer_norm(z6, (D,), g6, b6, 1e-5)
    pr = y6[:B // 2, 0] @ y6[B // 2:, 0].t()
    l6 = torch.nn.functional.cross_entropy(pr, torch.arange(B // 2))
    ref = torch.autograd.grad((y6 * dy.double().cpu()).sum() + l6, (x6, g6, b6, o6))
    # tolerance, relative to each output's largest value: the longest chain is 6 products whose rows are scaled to norm 1 and
    # whose sums run over at most 768 terms, (768 + 64) e each, and the normalisations keep the scale: 6 * 832 e = 3e-4
    tol = 6 * 832 * R.E32
    for name, a, b in zip(("y", "loss", "dx", "dg", "db", "dWo"), got, (y6.detach(), l6.detach(), *ref)):
        assert (a.double().cpu() - b).abs().max() <= tol * b.abs().max(), name
    for name, a, b in zip(("dx", "dg", "db", "dWo"), auto, ref):
        assert (a.double().cpu() - b).abs().max() <= tol * b.abs().max(), name


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_step_follows_new_inputs_and_seeds(dtype):
    """Forward and backward in one graph, replayed with eager work and synchronizations between the replays."""
    from otter_amd import inbatch as IB, training as T
    W, x, mask, dy = _layer(dtype)
    seed = _seed(1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(T, IB, W, x, mask, dy, seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(T, IB, W, x, mask, dy, seed)
    seen = []
    for i in range(4):
        seed.fill_(100 + i)
        x.copy_(torch.randn_like(x))
        mask[:, 1:] = (torch.rand(mask.shape, device=mask.device) < 0.7)[:, 1:].long()
        eager = [t.clone() for t in _step(T, IB, W, x, mask, dy, seed)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _same(outs, eager)
        seen.append(outs[0].clone())
    assert not torch.equal(seen[0], seen[1])


def test_another_stream_and_two_at_once():
    from otter_amd import inbatch as IB, training as T
    W, x, mask, dy = _layer(BF16)
    exp = _step(T, IB, W, x, mask, dy, _seed(5))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    seeds = [_seed(5), _seed(6)]
    torch.cuda.synchronize()
    res = []
    for s, seed in zip(streams, seeds):
        with torch.cuda.stream(s):
            res.append(_step(T, IB, W, x, mask, dy, seed))
    torch.cuda.synchronize()
    _same(res[0], exp)
    _same(res[1], _step(T, IB, W, x, mask, dy, seeds[1]))


def test_two_threads_at_once():
    """The calls let other threads run while they allocate and launch."""
    import threading
    from otter_amd import inbatch as IB, training as T
    W, x, mask, dy = _layer(BF16)
    seeds = [_seed(5), _seed(6)]
    exp = [_step(T, IB, W, x, mask, dy, s) for s in seeds]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = _step(T, IB, W, x, mask, dy, seeds[i])
                    torch.cuda.current_stream().synchronize()
                    _same(got, exp[i])
        except BaseException as e:                              # noqa: B902 -- reported below
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_calls_refuse_what_is_no_tensor():
    from otter_amd import inbatch as IB, training as T
    dev = _dev()
    q = torch.zeros(2, 8, 2, 64, device=dev)
    x, w = torch.zeros(4, 8, device=dev), torch.ones(8, device=dev)
    cu = torch.tensor([0, 8, 16], dtype=torch.int32, device=dev)
    for bad in (None, 3.0, "q", [1, 2]):
        for call in (lambda: T.attention_forward(bad, q, q), lambda: T.attention_forward(q, q, bad),
                     lambda: T.layer_norm_forward(bad, w, w), lambda: T.layer_norm_forward(x, bad, w),
                     lambda: T.layer_norm_forward(x, w, bad), lambda: T.dropout_forward(bad, 0.1, _seed()),
                     lambda: T.dropout_forward(x, 0.1, bad), lambda: IB.inbatch_loss_forward(bad, x),
                     lambda: IB.inbatch_loss_forward(x, bad), lambda: T.attention_backward(bad, q, q, q, q, q)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(TypeError):
        T.dropout_forward(x, "0.1", _seed())
    with pytest.raises(ValueError, match="probability"):
        T.dropout_forward(x, float("nan"), _seed())
    with pytest.raises(TypeError):
        T.dropout_forward(x, 0.1, _seed(), call="a")
    for call in (2 ** 32, 2 ** 70, -1):
        with pytest.raises(ValueError, match="call"):
            T.dropout_forward(x, 0.1, _seed(), call=call)
    with pytest.raises(ValueError, match="max_seqlen"):
        T.attention_forward(q[0].repeat(2, 1, 1), *(q[0].repeat(2, 1, 1),) * 2, cu_seqlens=cu, max_seqlen=2 ** 40)
    out, lse = T.attention_forward(q, q, q)
    for grads in ((q, q), (q, q, None), q[..., 1:], 5):
        with pytest.raises((ValueError, TypeError), match="grads"):
            T.attention_backward(out, q, q, q, out, lse, grads=grads)
    with pytest.raises(ValueError, match="out must be"):
        T.dropout_forward(x, 0.1, _seed(), out=x.t())
    y, mean, rstd = T.layer_norm_forward(x, w, w)
    with pytest.raises(ValueError, match="mean"):
        T.layer_norm_backward(x, x, w, mean[:2], rstd)


@pytest.mark.parametrize("B,d,neg", [(513, 2304, True), (260, 6400, False), (900, 768, True), (1500, 200, True), (1100, 330, False),
                                     (2100, 60, True), (2050, 65, False), (300, 40, True), (200, 768, True), (129, 1, True)])
def test_inbatch_loss_in_pieces_and_planes(B, d, neg):
    """Both sides of the choices by work and by tiles: float16 planes or float32, sums in one piece or several."""
    test_inbatch_loss(B, d, neg)


@pytest.mark.parametrize("margin", [3.0, 20.0])
def test_inbatch_loss_of_confident_rows_in_planes(margin):
    test_inbatch_loss_of_confident_rows(2000, margin)


@pytest.mark.parametrize("scale", [1e-6, 1e6])
def test_inbatch_loss_of_small_and_large_embeddings_in_planes(scale):
    test_inbatch_loss_of_small_and_large_embeddings(2000, scale)


@pytest.mark.parametrize("B,d", [(300, 64), (700, 100), (1600, 256)])
def test_inbatch_loss_repeats_its_bits(B, d):
    from otter_amd import inbatch as IB
    q, c, n = (_rand(95 + i, B, d, scale=d ** -0.25)[1] for i in range(3))
    one = torch.ones((), device=_dev())

    def run():
        loss, product, stats = IB.inbatch_loss_forward(q, c, n)
        return (loss, product, stats, *IB.inbatch_loss_backward(one, q, c, n, product, stats))

    first = run()
    for _ in range(3):
        _same(run(), first)


# Many workgroups: a wave to 32 rows (where there are few, two waves share them), the backward pass in two passes
@pytest.mark.parametrize("dtype,L,kind,p", [(F32, 129, None, 0.1), (F32, 200, "tile", 0.0), (F32, 260, "alternate", 0.1), (F32, 150, "holes", 0.1),
                                            (BF16, 257, "holes", 0.1), (BF16, 300, "alternate", 0.0), (BF16, 320, "none", 0.1)])
def test_attention_many_workgroups_dense(dtype, L, kind, p):
    B, H = 5, 64
    m = None if kind is None else _mask(kind, B, L)
    x = [_rand(130 + i, B, L, H, 64, dtype=dtype) for i in range(4)]
    kw = dict(dropout_p=p, seed=_seed() if p else None, call=6)
    if m is not None:
        kw["mask"] = m.to(_dev())
    _check_attention(*x, kw, mask=m, p=p)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_many_workgroups_packed(dtype):
    lens, H, p = [300, 20, 1, 256, 65], 64, 0.1
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x = [_rand(140 + i, cu[-1] + 9, H, 64, dtype=dtype) for i in range(4)]
    for t64, t in x:
        t64[cu[-1]:] = 0
        t[cu[-1]:] = float("nan")
    cut = torch.tensor(cu, dtype=torch.int32, device=_dev())
    _check_attention(*x, dict(cu_seqlens=cut, max_seqlen=300, dropout_p=p, seed=_seed(), call=6), cu=cu, p=p)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0])
def test_attention_scales(dtype, scale):
    """Also scores of hundreds, where a wave's half of the keys holds none of a row's weight."""
    m = _mask("holes", 2, 150)
    x = [_rand(150 + i, 2, 150, 2, 64, dtype=dtype) for i in range(4)]
    _check_attention(*x, dict(mask=m.to(_dev()), dropout_p=0.1, seed=_seed(), call=6, scale=scale), mask=m, p=0.1, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H,how", [(3, 1, 2, "dense"), (300, 1, 4, "dense"), (4, 40, 2, "mask"), (3, 300, 2, "mask"), (5, 200, 64, "mask"),
                                       (70, 1, 4, "packed"), (3, 1, 1, "packed")])
def test_one_key_leaves_no_gradient(B, L, H, how, dtype):
    """With one key the probabilities are 1 whatever q and k are: their gradients are zero and not a rounding's rest."""
    from otter_amd import training as T
    dev = _dev()
    q, k, v, do = (_rand(160 + i, B, L, H, 64, dtype=dtype)[1] * 3 for i in range(4))
    kw = dict(dropout_p=0.1, seed=_seed(), call=6)
    if how == "mask":
        kw["mask"] = torch.zeros(B, L, dtype=torch.int64, device=dev)
        kw["mask"][:, 0] = 1
    elif how == "packed":
        q, k, v, do = (t[:, 0] for t in (q, k, v, do))
        kw.update(cu_seqlens=torch.arange(B + 1, dtype=torch.int32, device=dev), max_seqlen=1)
    out, lse = T.attention_forward(q, k, v, **kw)
    dq, dk, dv = T.attention_backward(do, q, k, v, out, lse, **kw)
    assert (dq == 0).all() and (dk == 0).all() and (dv != 0).any()


def test_expanded_gradient_buffers_are_refused():
    from otter_amd import training as T
    q = torch.randn(2, 8, 2, 64, device=_dev())
    out, lse = T.attention_forward(q, q, q)
    g = torch.zeros_like(q)
    with pytest.raises(ValueError, match="grads"):
        T.attention_backward(out, q, q, q, out, lse, grads=(g, g.clone(), g[:1].expand(2, 8, 2, 64)))
    one = q[:1]                                                 # a dimension of one may have any stride
    out, lse = T.attention_forward(one, one, one)
    T.attention_backward(out, one, one, one, out, lse, grads=tuple(torch.zeros(8, 2, 64, device=_dev())[None] for _ in range(3)))


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("cols", list(range(1, 18)) + [249, 250, 255, 257, 263, 505, 511, 513, 519, 1023, 1025, 1031, 2041, 2049, 4097, 8185, 8191])
def test_layer_norm_rows_cut_anywhere(cols, dtype, wdtype):
    """Rows whose last group of eight holds one to eight elements, in the first and the last group of a lane."""
    from otter_amd import training as T
    rows, p, dev = 5, 0.2, _dev()
    x64, x = _rand(170, rows, cols, dtype=dtype)
    r64, r = _rand(171, rows, cols, dtype=dtype)
    d64, dy = _rand(172, rows, cols, dtype=dtype)
    w64, w = _rand(173, cols, dtype=wdtype)
    b64, b = _rand(174, cols, dtype=wdtype)
    kw = dict(residual=r, dropout_p=p, seed=_seed(), call=3)
    y, mean, rstd = T.layer_norm_forward(x, w, b, 1e-5, **kw)
    dx, dres, dw, db = T.layer_norm_backward(dy, x, w, mean, rstd, **kw)
    ref = R.layer_norm(x64, w64, b64, 1e-5, r64, p, SEED, 3, d64, dtype, wdtype)
    for name, t in (("y", y), ("dx", dx), ("dresidual", dres), ("dweight", dw), ("dbias", db)):
        _close(name, t, ref[name])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [1, 3, 7, 9, 257, 771, 1029])
def test_layer_norm_writes_nothing_behind_its_rows(cols, dtype):
    from otter_amd import _lib
    lib, dev, rows = _lib.load(), _dev(), 9
    n, code = rows * cols, _lib.OTTER_F32 if dtype == F32 else _lib.OTTER_BF16
    x, r, dy = (_rand(180 + i, rows, cols, dtype=dtype)[1] for i in range(3))
    w, b = torch.ones(cols, device=dev), torch.zeros(cols, device=dev)
    bufs = [torch.full((n + 64,), 7.0, device=dev, dtype=dtype) for _ in range(3)]
    small = [torch.full((m + 64,), 7.0, device=dev) for m in (rows, rows, cols, cols)]
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.otter_layernorm_forward(0, code, 0, x.data_ptr(), r.data_ptr(), w.data_ptr(), b.data_ptr(), rows, cols, 1e-5, 0.1,
                                           _seed().data_ptr(), 0, bufs[0].data_ptr(), small[0].data_ptr(), small[1].data_ptr(), stream))
    need = lib.otter_layernorm_backward_workspace(rows, cols)
    ws = torch.full((need + 64,), 9, dtype=torch.uint8, device=dev)
    seed = _seed()
    _lib.check(lib.otter_layernorm_backward(0, code, 0, dy.data_ptr(), x.data_ptr(), r.data_ptr(), w.data_ptr(), small[0].data_ptr(),
                                            small[1].data_ptr(), rows, cols, 0.1, seed.data_ptr(), 0, bufs[1].data_ptr(),
                                            bufs[2].data_ptr(), small[2].data_ptr(), small[3].data_ptr(), ws.data_ptr(), need, stream))
    for t, m in list(zip(bufs, (n,) * 3)) + list(zip(small, (rows, rows, cols, cols))):
        assert (t[m:] == 7).all() and torch.isfinite(t).all()
    assert (ws[need:] == 9).all()


def test_attention_one_pass_three_key_blocks():
    """Many pairs of more than 512 keys: the carried dQ is written, read and added to, and read and finished."""
    B, H, L, p = 10, 64, 520, 0.1
    m = _mask("prefix", B, L)
    x = [_rand(190 + i, B, L, H, 64, dtype=BF16) for i in range(4)]
    _check_attention(*x, dict(mask=m.to(_dev()), dropout_p=p, seed=_seed(), call=6), mask=m, p=p)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H", [(1, 700, 3), (3, 300, 5), (9, 130, 9), (17, 257, 7)])
def test_every_pair_is_dealt_out(B, L, H, dtype):
    """Numbers of (sequence, head) pairs that are no multiples of anything: every row of every pair, dense and packed."""
    m = _mask("prefix", B, L)
    x = [_rand(200 + i, B, L, H, 64, dtype=dtype) for i in range(4)]
    _check_attention(*x, dict(mask=m.to(_dev()), dropout_p=0.0, seed=None, call=6), mask=m)
    cu = [L * b for b in range(B + 1)]
    y = [(t64.flatten(0, 1), t.flatten(0, 1)) for t64, t in x]
    _check_attention(*y, dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=_dev()), max_seqlen=L), cu=cu)
