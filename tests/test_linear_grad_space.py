"""What moe_fused_linear_grad_workspace_of says, and refuses (no device is needed)."""

import ctypes

import pytest

from flaggems_vllm_b200 import _lib

P = 1 << 20


def say(dy=P, x=P, x_ld=64, w=P, w_ld=64, dtype=_lib.MOE_BF16, M=100, N=32, K=64, act=0, dx=1, dw=1, db=0, out=True):
    need = ctypes.c_int64(-1)
    rc = _lib.lib().moe_fused_linear_grad_workspace_of(dy, x, x_ld, w, w_ld, dtype, M, N, K, act, dx, dw, db, ctypes.addressof(need) if out else None)
    return need.value if rc == 0 else rc


@pytest.mark.parametrize("dtype,size", [(_lib.MOE_BF16, 2), (_lib.MOE_F16, 2), (_lib.MOE_F32, 4)])
def test_parts(dtype, size):
    half = size == 2
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    assert say(dtype=dtype) == 0
    assert say(dtype=dtype, db=1) == up(4 * 32 * 4)  # four blocks of rows
    assert say(dtype=dtype, M=10**6, db=1) == 512 * 32 * 4
    assert say(dtype=dtype, act=1) == up(100 * 32 * size) and say(dtype=dtype, act=5) == up(100 * 64 * size)
    assert say(dtype=dtype, act=1, dx=0, dw=0, db=1) == up(4 * 32 * 4)
    assert say(dtype=dtype, act=1, dx=0, dw=0) == 0
    assert say(dtype=dtype, dy=P + size) == say(dtype=dtype, dy=None) == (up(100 * 32 * 2) if half else 0)
    assert say(dtype=dtype, dy=P + size, dx=0, dw=0, db=1) == up(4 * 32 * 4)
    for change, at in ((dict(x=P + size), "dw"), (dict(w=P + size), "dx")):
        copy = up((100 if at == "dw" else 32) * 64 * 2) if half else 0
        assert say(dtype=dtype, **change) == copy and say(dtype=dtype, **change, **{at: 0}) == 0
    need = ctypes.c_int64()
    for act in range(6):  # never more than is said for any dy and any results
        assert _lib.lib().moe_fused_linear_grad_workspace(P + size, 65, P, 64, dtype, 100, 31, 64, act, ctypes.addressof(need)) == 0
        for which in range(8):
            assert say(dy=P + size, x=P + size, x_ld=65, dtype=dtype, N=31, act=act, dx=which & 1, dw=which & 2, db=which & 4) <= need.value


def test_refusals():
    for bad, code in ((dict(out=False), -1), (dict(M=-1), -1), (dict(N=0), -1), (dict(K=0), -1), (dict(act=6), -1), (dict(dtype=3), -2),
                      (dict(M=1 << 30), -5), (dict(N=1 << 29), -5), (dict(K=1 << 30), -5)):
        assert say(**bad) == code, bad
