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
