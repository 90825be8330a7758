"""Sizes that no launch of the training operators can take are refused before anything is allocated or enqueued (no GPU needed)."""
import ctypes

import pytest

from otter_amd import _lib


def _refused(rc):
    assert rc == _lib.OTTER_EINVAL, rc
    assert "too large for one launch" in _lib.load().otter_last_error().decode()


@pytest.mark.parametrize("B,d", [(1, 2 ** 31 - 1), (1, 2 ** 31 - 64), (1, 2 ** 30), (1, 2 ** 29 + 1), (64, 2 ** 29), (65, 2 ** 28 + 1), (65536, 2 ** 20)])
def test_inbatch_loss_refuses_grids_past_32_bits(B, d):
    lib = _lib.load()
    P, ld = ctypes.c_void_p(4096), B
    _refused(lib.otter_inbatch_loss_workspace(B, d))
    _refused(lib.otter_inbatch_loss_backward_workspace(B, d))
    _refused(lib.otter_inbatch_loss_forward(0, P, P, None, B, d, P, ld, P, P, P, 1 << 60, None))
    _refused(lib.otter_inbatch_loss_backward(0, P, P, P, None, B, d, P, ld, P, P, P, None, P, 1 << 60, None))


@pytest.mark.parametrize("B,d", [(1, 2 ** 29 - 64), (65, 2 ** 28 - 128), (65536, 2 ** 18)])
def test_inbatch_loss_has_a_workspace_for_the_largest(B, d):
    lib = _lib.load()
    assert lib.otter_inbatch_loss_workspace(B, d) > 0 and lib.otter_inbatch_loss_backward_workspace(B, d) >= 0


@pytest.mark.parametrize("batch,tokens,heads,packed", [(1 << 24, 1, 1, False), (1 << 22, 1, 4, False), ((1 << 24) // 12 + 1, 70, 12, True),
                                                       (1 << 16, 4096, 8, False), (1 << 20, 256, 8, True), (2 ** 31 - 1, 1, 2, False)])
def test_attention_refuses_grids_past_32_bits(batch, tokens, heads, packed):
    lib = _lib.load()
    a = _lib.AttentionArgs()
    a.dtype, a.batch, a.tokens, a.heads, a.head_dim, a.scale = _lib.OTTER_BF16, batch, tokens, heads, 64, 0.125
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, n, _lib.View(4096, 64 * heads * tokens, 64 * heads, 64))
    a.lse = a.workspace = 4096
    a.workspace_bytes = 1 << 60
    if packed:
        a.cu_seqlens, a.total = 4096, 2 ** 31 - 1
    for rc in (lib.otter_attention_forward(0, ctypes.byref(a), None), lib.otter_attention_backward(0, ctypes.byref(a), None),
               lib.otter_attention_backward_workspace(ctypes.byref(a))):
        _refused(rc)


def test_attention_has_a_workspace_for_the_largest():
    a = _lib.AttentionArgs()
    a.dtype, a.batch, a.tokens, a.heads, a.head_dim, a.scale = _lib.OTTER_F32, (1 << 24) // 12 - 3, 100, 12, 64, 0.125
    assert _lib.load().otter_attention_backward_workspace(ctypes.byref(a)) == a.batch * 100 * 12 * 4
