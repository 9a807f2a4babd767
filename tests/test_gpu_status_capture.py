"""The status word of a process whose first call is captured into a graph."""

import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib

logits = torch.randn(64, 16, device="cuda")
ids = torch.randint(0, 16, (64, 2), device="cuda", dtype=torch.int32)
bad = ids.clone()
bad[3, 1] = 16
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    loss, counts = fg.moe_balance_loss(logits, ids)
assert _lib.read_status() == 0                        # before the first replay too
want = fg.moe_balance_loss(logits, bad)[1]
graph.replay()                                        # a replay is no reset
assert _lib.read_status() == _lib.ST_BAD_EXPERT_ID
assert torch.equal(counts, torch.bincount(ids.flatten().long(), minlength=16).int())
ids.copy_(bad)
graph.replay()
assert _lib.read_status() == _lib.ST_BAD_EXPERT_ID and torch.equal(counts, want)
del graph, loss, counts
torch.cuda.empty_cache()
assert _lib.read_status() == 0
print("done")
"""


def test_a_first_call_that_is_captured():
    run = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "done" in run.stdout, run.stderr[-2000:]
