"""Arguments of the norms that are refused by their own checks, with the error that says why."""

import numpy as np
import pytest
import torch

import flaggems_vllm_b200 as fg


@pytest.mark.parametrize("value", [3e38, 3.5e38, 1e39, 1e300, 10 ** 60])
def test_eps_beyond_fp32(value):
    x, w = torch.zeros(4, 64), torch.ones(64)
    for call in (lambda: fg.rms_norm(x, w, value), lambda: fg.rms_norm_quant(x, w, value), lambda: fg.fused_add_rms_norm(x, x.clone(), w, value)):
        with pytest.raises(ValueError, match="eps"):
            call()
    with pytest.raises(ValueError, match="quant_eps"):
        fg.rms_norm_quant(x, w, quant_eps=value)


@pytest.mark.parametrize("group", [0.5, 2.5, 64 / 3])
def test_group_sizes_that_are_no_whole_number(group):
    """The row may well be a multiple of them: they used to be cut to whole numbers, 0.5 to the whole row."""
    x, w = torch.zeros(4, 64 if group != 2.5 else 10), torch.ones(64 if group != 2.5 else 10)
    with pytest.raises(ValueError, match="whole number"):
        fg.rms_norm_quant(x, w, group_size=group)


@pytest.mark.parametrize("group", [32, 32.0, np.int64(32)])
def test_group_sizes_that_are_one(group):
    with pytest.raises(RuntimeError, match="no CPU path"):  # past every other check
        fg.rms_norm_quant(torch.zeros(4, 64), torch.ones(64), group_size=group)


def test_c_gradient_over_its_inputs():
    """Rows of more than 64 KB are read again for the weight's gradient when dx has been written.  No call gets as far as a launch."""
    from flaggems_vllm_b200 import _lib

    P, before = 1 << 20, _lib.LAUNCHES
    for dy, dh, h, dx in ((P, None, 2 * P, P), (P, None, 2 * P, 2 * P), (P, 3 * P, 2 * P, 3 * P)):
        rc = _lib.lib().moe_rms_norm_grad(dy, dh, h, 64, 4 * P, 0, 0, 4, 64, 1e-6, dx, 5 * P, 6 * P, 1 << 30, None)
        assert rc == -1 and b"apart" in _lib.lib().moe_last_error()
    assert _lib.LAUNCHES == before


@pytest.mark.parametrize("cols", [64, 8192, 1 << 16, 1 << 20, 1 << 22, 1 << 24])
def test_workspace_of_the_gradient_does_not_outgrow_its_rows(cols):
    """256 MB of partial sums, or those of 16 rows, and a number per row."""
    import ctypes

    from flaggems_vllm_b200 import _lib

    need = ctypes.c_int64()
    for rows in (1, 16, 300, 5000):
        _lib.check(_lib.lib().moe_rms_norm_grad_workspace(rows, cols, ctypes.addressof(need)))
        assert need.value <= 4 * rows + max(256 << 20, 4 * 16 * cols)
