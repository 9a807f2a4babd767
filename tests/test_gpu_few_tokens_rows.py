"""fused_moe_few_tokens: tokens in rows of a wider buffer, where they fit in shared memory and where they do not."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from test_gpu_few_tokens import call, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def in_wider_rows(x, ld, offset=8):
    M, H = x.shape
    flat = torch.empty((M - 1) * ld + offset + H, dtype=x.dtype, device=DEV)
    if ld < 1 << 20:
        flat.fill_(float("nan"))
    rows = flat.as_strided((M, H), (ld, 1), offset)
    rows.copy_(x)
    return rows


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,H", [(2, 512), (8, 4096), (8, 7168), (3, 16384), (8, 16384)])  # the last three: read where they lie
@pytest.mark.parametrize("gap", [16, 1000])
def test_rows_of_a_wider_buffer(M, H, gap, dtype):
    d = make(M, 8, H, 128, 64, dtype)
    want = call(d, 3)
    d["x"] = in_wider_rows(d["x"], H + gap)
    assert all(torch.equal(p, q) for p, q in zip(call(d, 3), want)) and fg.read_status() == 0


@pytest.mark.parametrize("M,H,fp8", [(3, 16384, False), (3, 512, False), (3, 8192, True)])
def test_rows_far_apart(M, H, fp8):
    """2^30 elements: the distance in bytes passes 31 bits."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("not enough free memory")
    d = make(M, 4, H, 128, 0, BF, fp8)
    want = call(d, 2)
    d["x"] = in_wider_rows(d["x"], 1 << 30)
    assert all(torch.equal(p, q) for p, q in zip(call(d, 2), want)) and fg.read_status() == 0
