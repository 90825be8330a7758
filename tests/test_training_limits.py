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
