"""Calls of the training operators at the edges of what they allow: values that are not finite, rows of very different weight in
one batch, masks that leave one key, each against the 64-bit restatement (oracle/training_ref.py) or the formula's own limit."""
import pytest
import torch

from oracle import training_ref as R
from tests.test_training_gpu import BF16, F32, _check_attention, _close, _dev, _mask, _rand, _same, _seed
from tests.test_training_paths import takes_one_pass

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


# --------------------------------------------------------------------------------------------------------------- loss
def _loss_step(q, c, neg):
    from otter_amd import inbatch as IB
    loss, product, stats = IB.inbatch_loss_forward(q, c, neg)
    return loss, product, stats, *IB.inbatch_loss_backward(torch.ones((), device=_dev()), q, c, neg, product, stats)


# one row; few rows in one piece of d and in several; one and several pieces of many rows; float16 planes
LOSS_SIZES = [(1, 8), (2, 3), (40, 40), (64, 768), (64, 2304), (200, 33), (200, 768), (700, 768), (1000, 100)]


@pytest.mark.parametrize("B,d", LOSS_SIZES)
def test_a_hard_negative_that_is_not_finite(B, d):
    """A NaN or +inf score makes its own row's loss and gradients NaN and no other's; a score of -inf has no weight."""
    q, c, neg = (_rand(300 + i, B, d, scale=d ** -0.25)[1] for i in range(3))
    i = B // 2
    q[i, 0] = 1.0
    clean = _loss_step(q, c, neg)
    others = torch.arange(B, device=_dev()) != i
    for bad in (NAN, INF):
        n = neg.clone()
        n[i, 0] = bad
        loss, product, stats, dq, dc, dneg = _loss_step(q, c, n)
        assert torch.isnan(loss) and torch.isnan(stats[:, i]).all(), (float(loss), stats[:, i])
        assert torch.isnan(dq[i]).all() and torch.isnan(dneg[i]).all() and torch.isnan(dc).all()
        _same((stats[:, others], product[others]), (clean[2][:, others], clean[1][others]))
        assert torch.isfinite(dq[others]).all() and torch.isfinite(dneg[others]).all()
    n = neg.clone()
    n[i, 0] = -INF
    loss, product, stats, dq, dc, dneg = _loss_step(q, c, n)
    alone = _loss_step(q, c, None)
    # one column more or less at the end of the sum: a few half steps of the numbers that are formed
    tol = 16 * R.E32 * (1 + alone[2][0, i].abs())
    assert torch.isfinite(loss) and (stats[:, i] - alone[2][:, i]).abs().max() <= tol
    assert (dneg[i] == 0).all() and torch.isfinite(dc).all() and torch.isnan(dq[i, 0])      # 0 * -inf


@pytest.mark.parametrize("B,d", LOSS_SIZES)
def test_a_nan_in_a_block_reaches_every_row(B, d):
    q, c, neg = (_rand(310 + i, B, d, scale=d ** -0.25)[1] for i in range(3))
    c[B // 2, 0] = NAN
    for n in (None, neg):
        loss, product, stats, dq, dc, dneg = _loss_step(q, c, n)
        assert torch.isnan(loss) and torch.isnan(product[:, B // 2]).all() and torch.isnan(stats).all()
        assert torch.isnan(dq).all() and torch.isnan(dc).all()


@pytest.mark.parametrize("B,d", LOSS_SIZES)
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinity_in_a_block_is_not_hidden(B, d, sign):
    """A target's score of +inf is inf - inf, one of -inf an infinite loss: neither comes out as a finite number."""
    q, c, neg = (_rand(320 + i, B, d, scale=d ** -0.25)[1] for i in range(3))
    i = B // 2
    q[i, 0] = 1.0
    c[i, 0] = sign * INF
    for n in (None, neg):
        loss, _, stats, *_ = _loss_step(q, c, n)
        assert not torch.isfinite(loss), float(loss)
        if sign > 0:
            assert torch.isnan(loss) and torch.isnan(stats[1, i])


def _margins(B, d, seed, margin):
    """float32 inputs: row i's target lies margin[i] above the others, whose scores are a few margins / sqrt(d)."""
    c = torch.nn.functional.normalize(_rand(seed, B, d)[0], dim=1).float().double()
    return (margin[:, None] * c).float().double(), c


def _close_loss(q64, c64, names=("loss", "rest", "dq", "dc")):
    ref = R.inbatch_loss(q64, c64, None, 1.0)
    loss, _, stats, dq, dc, _ = _loss_step(q64.float().to(_dev()), c64.float().to(_dev()), None)
    got = {"loss": loss, "rest": stats[1], "lse": stats[0], "dq": dq, "dc": dc}
    for name in names:
        _close(name, got[name], ref[name])


# float32 products, float16 planes in one and in several pieces
MIXED = [(200, 128), (640, 768), (700, 768), (2000, 128), (1100, 300), (4096, 64), (600, 2304)]


@pytest.mark.parametrize("B,d", MIXED)
@pytest.mark.parametrize("margin", [12.0, 25.0, 60.0])
@pytest.mark.parametrize("hard", ["spread", "confused"])
def test_loss_of_confident_rows_beside_one_that_is_not(B, d, margin, hard):
    """The other rows' gradients are e^-margin of the hard one's and as exact; a confused row has its weight on one wrong column,
    so that the other columns' gradients are as small."""
    m = torch.full((B,), margin, dtype=torch.float64)
    q, c = _margins(B, d, 330, m)
    i = B // 3
    q[i] = 0.01 * c[i] if hard == "spread" else margin * c[(i + 7) % B]
    _close_loss(q.float().double(), c)


@pytest.mark.parametrize("B,d", MIXED)
def test_loss_of_rows_of_every_confidence(B, d):
    m = torch.linspace(0.0, 40.0, B, dtype=torch.float64)[torch.randperm(B, generator=torch.Generator().manual_seed(7))]
    _close_loss(*_margins(B, d, 340, m))


@pytest.mark.parametrize("B,d", MIXED)
def test_loss_of_blocks_of_very_different_sizes(B, d):
    """Blocks whose sizes span twelve decades, met by questions that point away from the large ones."""
    size = torch.logspace(-6, 6, B, dtype=torch.float64)[torch.randperm(B, generator=torch.Generator().manual_seed(8))][:, None]
    u = torch.nn.functional.normalize(_rand(350, B, d)[0].abs(), dim=1)
    c = (size * u).float().double()
    q = _rand(351, B, d)[0].abs() * torch.where(torch.arange(B)[:, None] % 2 == 0, -1e-3, 1e-9)
    _close_loss(q.float().double(), c, ("loss", "lse", "dq", "dc"))


# ---------------------------------------------------------------------------------------------------------- attention
# one pass over the scores (bfloat16) with rows of one, two and three blocks of 256 keys; two passes, with one and two waves to 32 rows
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H", [(4, 40, 2), (3, 70, 2), (130, 70, 2), (3, 128, 3), (5, 200, 64), (4, 300, 64), (13, 520, 64), (3, 530, 2), (5, 150, 64)])
@pytest.mark.parametrize("at", ["middle", "last", "each"])
def test_one_key_anywhere_leaves_no_gradient(B, L, H, at, dtype):
    """With one key the probabilities are 1 whatever q and k are, wherever the key stands."""
    from otter_amd import training as T
    q, k, v, do = (_rand(360 + i, B, L, H, 64, dtype=dtype)[1] * 3 for i in range(4))
    where = torch.tensor([L // 2 if at == "middle" else L - 1 if at == "last" else (37 * b + 1) % L for b in range(B)], device=_dev())
    mask = (torch.arange(L, device=_dev())[None, :] == where[:, None]).long()
    kw = dict(mask=mask, dropout_p=0.1, seed=_seed(), call=6)
    out, lse = T.attention_forward(q, k, v, **kw)
    dq, dk, dv = T.attention_backward(do, q, k, v, out, lse, **kw)
    assert (dq == 0).all() and (dk == 0).all(), (float(dq.abs().max()), float(dk.abs().max()))
    assert (dv[mask == 0] == 0).all() and (dv[mask != 0] != 0).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L,keys", [(70, (0, 69)), (70, (3, 4)), (200, (0, 199)), (300, (63, 64)), (600, (0, 599)), (600, (1, 320))])
def test_two_keys_far_apart(L, keys, dtype):
    """Two keys that count, in one chunk of the mask's 64 and in chunks that are looked at one after the other."""
    B, H = 3, 2
    m = torch.zeros(B, L, dtype=torch.int64)
    m[:, list(keys)] = 1
    m[1, keys[0]] = 0                                           # and a sequence with one beside them
    x = [_rand(370 + i, B, L, H, 64, dtype=dtype) for i in range(4)]
    _check_attention(*x, dict(mask=m.to(_dev()), dropout_p=0.1, seed=_seed(), call=6), mask=m, p=0.1)


# The backward pass in one pass and in two on either side of the rules that choose; the path is asserted, so that a rule that
# moves does not leave one of them untested
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("lens,lead,tail,H,one", [([300, 20, 1, 256, 400, 0, 130], 3, 70, 64, True), ([512, 257, 33, 290, 511, 64, 500], 0, 0, 64, True),
                                                  ([520] * 4, 0, 0, 64, True), ([520, 500, 516, 513], 2, 30, 64, True), ([600, 450, 500, 1, 530], 0, 5, 150, True),
                                                  ([600, 20, 130, 0, 257], 0, 5, 150, False), ([300, 20, 1, 256], 0, 9, 64, False)])
def test_attention_packed_either_way(lens, lead, tail, H, one, p):
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    total = cu[-1] + tail
    assert takes_one_pass(len(lens), max(lens), H, total=total) == one
    x = [_rand(380 + i, total, H, 64, dtype=BF16) for i in range(4)]
    for t64, t in x:
        for rows in (slice(0, lead), slice(cu[-1], total)):
            t64[rows] = 0
            t[rows] = NAN
    cut = torch.tensor(cu, dtype=torch.int32, device=_dev())
    _check_attention(*x, dict(cu_seqlens=cut, max_seqlen=max(lens), dropout_p=p, seed=_seed(), call=6), cu=cu, p=p)


@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("B,L,H,kind,one", [(4, 520, 64, None, True), (4, 777, 60, None, True), (3, 300, 60, None, True), (3, 300, 64, "holes", True),
                                            (2, 300, 64, None, False), (4, 520, 64, "prefix", False), (11, 530, 64, "alternate", True), (3, 260, 40, "tile", False)])
def test_attention_dense_either_way(B, L, H, kind, one, p):
    assert takes_one_pass(B, L, H, mask=kind is not None) == one
    m = None if kind is None else _mask(kind, B, L)
    x = [_rand(390 + i, B, L, H, 64, dtype=BF16) for i in range(4)]
    kw = dict(dropout_p=p, seed=_seed() if p else None, call=6)
    if m is not None:
        kw["mask"] = m.to(_dev())
    _check_attention(*x, kw, mask=m, p=p)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H", [(13, 140, 9), (5, 400, 7), (3, 512, 11), (7, 260, 3)])
def test_every_pair_of_several_workgroups(B, L, H, dtype):
    """Pairs dealt out one by one and eight at a time, whole eights and a rest: every row of every pair, dense and packed."""
    m = _mask("prefix", B, L)
    x = [_rand(400 + i, B, L, H, 64, dtype=dtype) for i in range(4)]
    _check_attention(*x, dict(mask=m.to(_dev()), dropout_p=0.1, seed=_seed(), call=6), mask=m, p=0.1)
    cu = [0]
    for n in m.sum(1).tolist():
        cu.append(cu[-1] + n)
    y = [(t64[m != 0], t[m.to(_dev()) != 0]) for t64, t in x]
    _check_attention(*y, dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=_dev()), max_seqlen=L), cu=cu)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,lead,tail,H", [([30, 0, 5], 900, 6000, 12), ([300], 0, 3001, 1), ([70] * 6, 1, 2000, 40), ([], 0, 500, 3), ([129, 1], 5000, 0, 5)])
def test_packed_buffers_with_many_unused_rows(lens, lead, tail, H, dtype):
    """A buffer of a fixed size: rows of no sequence come out as zeros, whatever the outputs' views, and nothing else of them is written."""
    from otter_amd import training as T
    n, dev = sum(lens), _dev()
    total = lead + n + tail
    cu = torch.tensor([lead] + [lead + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device=dev)
    q, k, v, do = (_rand(410 + i, total, H, 64, dtype=dtype)[1] for i in range(4))
    kw = dict(max_seqlen=max(lens, default=0), dropout_p=0.1, seed=_seed(), call=6)
    used = slice(lead, lead + n)
    out, lse = T.attention_forward(q, k, v, cu_seqlens=cu, **kw)
    buf = torch.full((total + 8, 5, H, 64), 7.0, device=dev, dtype=dtype)       # three of its five columns are the gradients
    grads = buf[4:4 + total, 1:4].unbind(1)
    T.attention_backward(do, q, k, v, out, lse, cu_seqlens=cu, grads=grads, **kw)
    if n:
        tight = tuple(t[used].contiguous() for t in (q, k, v))
        out2, lse2 = T.attention_forward(*tight, cu_seqlens=cu - lead, **kw)
        g2 = T.attention_backward(do[used].contiguous(), *tight, out2, lse2, cu_seqlens=cu - lead, **kw)
        _same((out[used], lse[:, used]), (out2, lse2))
        for a, b in zip(grads, g2):                             # the way may be another one: a half step of each
            assert ((a[used].double() - b.double()).abs() <= 4 * R.half_step(dtype) * b.double().abs().amax()).all()
    for t in (out, lse.t(), *grads):
        assert (t[:lead] == 0).all() and (t[lead + n:] == 0).all()
    assert (buf[:4] == 7).all() and (buf[4 + total:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 4] == 7).all()


# ------------------------------------------------------------------------------------------------- autograd's own records
def test_explicit_halves_have_no_history():
    """Whatever p is and whatever has to be copied or cast on the way."""
    from otter_amd import inbatch as IB, training as T
    x = torch.randn(6, 8, device=_dev(), requires_grad=True)
    w = torch.ones(8, device=_dev(), requires_grad=True)
    for p in (0.0, 0.3):
        for t in (x, x.t(), x * 1.0):
            assert not T.dropout_forward(t, p, _seed()).requires_grad
        out = torch.empty(6, 8, device=_dev())
        assert T.dropout_forward(x, p, _seed(), out=out) is out and not out.requires_grad
        assert not any(t.requires_grad for t in T.layer_norm_forward(x.bfloat16(), w, w, dropout_p=p, seed=_seed()))
    assert not any(t.requires_grad for t in IB.inbatch_loss_forward(x.bfloat16(), x * 2.0))
    # the differentiable call keeps it
    g, = torch.autograd.grad(T.dropout(x, 0.0, None).sum(), x)
    assert (g == 1).all()


def test_tensors_that_are_written_say_so():
    """A tensor saved for a backward pass and then written by a call: the backward pass refuses instead of using the new values."""
    from otter_amd import training as T
    for p in (0.0, 0.3):
        x = torch.randn(6, 8, device=_dev(), requires_grad=True)
        y = x.exp()                                             # its backward pass needs y
        T.dropout_forward(y.detach(), p, _seed(), out=y.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    q = torch.randn(2, 8, 2, 64, device=_dev())
    out, lse = T.attention_forward(q, q, q)
    buf = torch.randn(2, 8, 3, 2, 64, device=_dev(), requires_grad=True)
    y = buf.exp()
    T.attention_backward(out, q, q, q, out, lse, grads=y.detach().unbind(2))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# -------------------------------------------------------------------------------------------------------- shared memory
def test_overlapping_outputs_are_refused():
    from otter_amd import training as T
    buf = torch.randn(100, device=_dev())
    for p in (0.0, 0.3):
        for x, out in ((buf[:64], buf[1:65]), (buf[32:96], buf[:64]), (buf[:64].view(8, 8), buf[8:72].view(8, 8))):
            with pytest.raises(ValueError, match="overlaps"):
                T.dropout_forward(x, p, _seed(), out=out)
        x = torch.randn(8, 8, device=_dev())                    # a view that has to be copied first may be overwritten
        exp = T.dropout_forward(x.t(), p, _seed())
        assert torch.equal(T.dropout_forward(x.t(), p, _seed(), out=x), exp)
        T.dropout_forward(buf[:32], p, _seed(), out=buf[32:64])
    q, k, v, do = (torch.randn(2, 8, 2, 64, device=_dev()) for _ in range(4))
    out, lse = T.attention_forward(q, k, v)
    a, b, c = (torch.empty_like(q) for _ in range(3))
    for grads in ((a, a, c), (a, b, a), (a, b, b), (q, b, c), (a, k, c), (a, b, v), (do, b, c), (a, out, c), (k, b, c)):
        with pytest.raises(ValueError, match="one another or an operand"):
            T.attention_backward(do, q, k, v, out, lse, grads=grads)
    ref = T.attention_backward(do, q, k, v, out, lse)
    _same(T.attention_backward(do, q, k, v, out, lse, grads=(a, b, c)), ref)
    empty = torch.empty(0, 8, 2, 64, device=_dev())
    T.attention_backward(empty, empty, empty, empty, empty, torch.empty(0, 2, 8, device=_dev()), grads=(empty,) * 3)


def test_mixed_types_are_refused():
    """What autocast makes of a layer: a product in bfloat16 beside a residual in float32."""
    from otter_amd import training as T
    x = torch.randn(4, 8, device=_dev())
    w = torch.ones(8, device=_dev())
    with pytest.raises(ValueError, match="residual must be like"):
        T.layer_norm(x.bfloat16(), w, w, residual=x)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        T.layer_norm(x.half(), w, w)
    assert T.layer_norm(x.bfloat16(), w, w, residual=x.bfloat16()).dtype == BF16


# ------------------------------------------------------------------------------------------------------ graphs and streams
@pytest.mark.parametrize("dtype,total,longest", [(F32, 700, 300), (BF16, 700, 300), (BF16, 3000, 512)])
def test_captured_packed_step_follows_its_lengths(dtype, total, longest):
    """A buffer of a fixed size in a graph: every replay has other sequences in it, and other rows of no sequence."""
    from otter_amd import training as T
    H, B, dev = 12, 8, _dev()
    q, k, v, do = (_rand(420 + i, total, H, 64, dtype=dtype)[1] for i in range(4))
    cu, seed = torch.zeros(B + 1, dtype=torch.int32, device=dev), _seed(1)

    def step():
        kw = dict(cu_seqlens=cu, max_seqlen=longest, dropout_p=0.1, seed=seed, call=2)
        out, lse = T.attention_forward(q, k, v, **kw)
        return (out, lse, *T.attention_backward(do, q, k, v, out, lse, **kw))

    with torch.cuda.stream(torch.cuda.Stream()):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    g = torch.Generator().manual_seed(9)
    for i in range(5):
        lens = torch.randint(0, min(longest, total // B) + 1, (B,), generator=g)
        lead = int(torch.randint(0, total - int(lens.sum()) + 1, (1,), generator=g))
        cu.copy_(lead + torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0))).int())
        seed.fill_(50 + i)
        q.copy_(torch.randn_like(q))
        exp = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _same(got, exp)
        n = int(lens.sum())
        assert all((t[:lead] == 0).all() and (t[lead + n:] == 0).all() for t in (got[0], *got[2:]))


@pytest.mark.parametrize("B,d", [(40, 768), (64, 2304), (300, 100), (700, 768), (1300, 256)])
def test_captured_loss_follows_its_inputs(B, d):
    q, c, n = (_rand(430 + i, B, d, scale=d ** -0.25)[1] for i in range(3))
    with torch.cuda.stream(torch.cuda.Stream()):
        _loss_step(q, c, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    one = torch.ones((), device=_dev())
    from otter_amd import inbatch as IB
    with torch.cuda.graph(graph):
        loss, product, stats = IB.inbatch_loss_forward(q, c, n)
        got = (loss, product, stats, *IB.inbatch_loss_backward(one, q, c, n, product, stats))
    for i in range(4):
        for t in (q, c, n):
            t.copy_(torch.randn_like(t) * (0.5 + i) * d ** -0.25)
        exp = [t.clone() for t in _loss_step(q, c, n)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _same(got, exp)


def test_two_losses_at_once_on_two_streams():
    x = [[_rand(440 + 3 * s + i, 900, 768, scale=768 ** -0.25)[1] for i in range(3)] for s in range(2)]
    exp = [_loss_step(*t) for t in x]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for t in x:
            with torch.cuda.stream(torch.cuda.Stream()):
                got.append(_loss_step(*t))
        torch.cuda.synchronize()
        for a, b in zip(got, exp):
            _same(a, b)


@pytest.mark.parametrize("B,d", [(40, 96), (700, 640)])
def test_loss_of_strided_and_mixed_inputs(B, d):
    """Transposed, sliced and half-width inputs give what their float32 copies give."""
    q, c, n = (_rand(450 + i, B, d, scale=d ** -0.25)[1] for i in range(3))
    exp = _loss_step(q, c.bfloat16().float(), n)
    wide = torch.zeros(B, 2 * d + 1, device=_dev())
    wide[:, 1:d + 1] = n
    _same(_loss_step(q.t().contiguous().t(), c.bfloat16(), wide[:, 1:d + 1]), exp)
