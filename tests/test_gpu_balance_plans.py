"""How moe_balance_loss shares out its rows: either side of one and of four turns of a block, with and without sequences."""

import ctypes

import pytest
import torch

from flaggems_vllm_b200 import _lib
from test_gpu_balance import check, make

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("E,k,turn", [(8, 2, 512), (256, 8, 32), (128, 8, 64), (1000, 4, 8), (60, 4, 128)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_either_side_of_the_lines(E, k, turn, scoring):
    for T in (turn - 1, turn, turn + 1, 2 * turn + 3, 4 * turn - 1, 4 * turn, 4 * turn + 1, 9 * turn):
        logits, ids = make(T, E, k, seed=T)
        check(logits, ids, scoring, dloss=float(T))
        for edges in ([0, T], [0, 1, T // 2, T // 2, T - 1], [0] + [T // 2] * 40 + [T], list(range(0, T + 1, max(1, T // 50)))):
            check(logits, ids, scoring, torch.tensor(edges, dtype=torch.int32, device=DEV), dloss=float(T))


@pytest.mark.parametrize("T,E,turn", [(2000, 8, 512), (128, 256, 32)])
def test_a_call_with_sequences_is_shared_out(T, E, turn):
    """One block for all rows saves the second launch where there are no sequences; with them it only walks them alone.  Every part
    of a sequence that a block holds leaves E sums, E counts and its tokens in the workspace: blocks + sequences - 1 parts here."""
    S, k = 8, 2
    logits, ids = make(T, E, k)
    cu = torch.linspace(0, T, S + 1, device=DEV).int()
    cu[1:-1] += 3  # no edge of a sequence is one of a block
    two = (ctypes.c_int64 * 2)()
    _lib.check(_lib.lib().moe_balance_loss_workspace(T, E, k, S, ctypes.addressof(two)))
    ws = torch.full((two[0] // 4,), -1, dtype=torch.int32, device=DEV)
    saved, counts = (torch.empty(n // 4, dtype=torch.int32, device=DEV) for n in (two[1], 4 * S * E))
    loss = torch.empty((), device=DEV)
    _lib.check(_lib.lib().moe_balance_loss(logits.data_ptr(), E, _lib.MOE_F32, T, E, ids.data_ptr(), 0, k, 0, cu.data_ptr(), S, None,
                                           loss.data_ptr(), counts.data_ptr(), saved.data_ptr(), ws.data_ptr(), two[0], None,
                                           torch.cuda.current_stream().cuda_stream))
    blocks = -(-T // turn)
    assert (ws != -1).sum().item() >= (blocks + S - 1) * (2 * E + 1)
