"""Calls of the training operators at the edges of what they allow: values that are not finite, rows of very different weight in
one batch, masks that leave one key, each against the 64-bit restatement (oracle/training_ref.py) or the formula's own limit."""
import pytest
import torch

from oracle import training_ref as R
from tests.test_training_gpu import _dev, _rand, _same

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
