"""Which way attention's backward pass takes, as its workspace tells (no GPU needed): D of every row and head for two passes over the
scores; in one pass nothing up to 256 tokens of a dense batch and a float32 dQ otherwise."""
import ctypes

import pytest

from otter_amd import _lib


def takes_one_pass(batch, tokens, heads, dtype=_lib.OTTER_BF16, mask=False, total=None):
    """total: rows of a packed batch."""
    a = _lib.AttentionArgs()
    a.dtype, a.batch, a.tokens, a.heads, a.head_dim, a.scale = dtype, batch, tokens, heads, 64, 0.125
    if mask:
        a.mask = 4096
    if total is not None:
        a.cu_seqlens, a.total = 4096, total
    rows = batch * tokens if total is None else total
    need = _lib.load().otter_attention_backward_workspace(ctypes.byref(a))
    assert need in (0, 4 * rows * heads, 256 * rows * heads), need
    return need != 4 * rows * heads


@pytest.mark.parametrize("batch,tokens", [(40, 1500), (21, 700), (64, 2000), (20, 512), (12, 512), (16, 300), (40, 700)])
def test_full_batches_take_one_pass_where_it_is_faster(batch, tokens):
    assert takes_one_pass(batch, tokens, 12)
    assert takes_one_pass(batch, tokens, 12, total=batch * tokens)


@pytest.mark.parametrize("batch,tokens", [(10, 512), (14, 300), (16, 1500), (22, 512), (64, 3000), (42, 8192)])
def test_full_batches_take_two_passes_where_those_are_faster(batch, tokens):
    assert not takes_one_pass(batch, tokens, 12)


def test_ragged_batches():
    for batch, tokens, one in ((40, 1500, False), (40, 700, False), (64, 700, True), (64, 1500, True), (64, 2000, False), (16, 512, True),
                               (12, 512, False), (42, 512, True)):
        assert takes_one_pass(batch, tokens, 12, mask=True) == one, (batch, tokens)
    for batch, tokens, fill, one in ((64, 1500, 0.56, False), (64, 1500, 0.8, True), (64, 1000, 0.56, False), (64, 1000, 0.7, True),
                                     (40, 700, 0.7, False), (40, 700, 0.9, True), (16, 512, 0.56, False), (128, 512, 0.56, True),
                                     (42, 512, 0.56, True)):
        assert takes_one_pass(batch, tokens, 12, total=int(fill * batch * tokens)) == one, (batch, tokens, fill)


def test_short_batches_and_float32():
    assert takes_one_pass(16, 70, 12, total=600) and not takes_one_pass(64, 70, 12, total=2000)
    assert takes_one_pass(16, 200, 12, total=2000) and not takes_one_pass(4, 200, 12, total=800)
    assert not takes_one_pass(128, 512, 12, dtype=_lib.OTTER_F32) and not takes_one_pass(16, 200, 12, dtype=_lib.OTTER_F32)
    assert not takes_one_pass(0, 700, 12, dtype=_lib.OTTER_F32, total=0)
