"""Norms and balance loss through the C entry points on memory of the test's own: every byte around the outputs, workspaces and
saved buffers keeps its pattern, and what they held before changes nothing.  Threads of one process beside one another."""

import ctypes
import threading

import pytest
import torch

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
BAND = 4096
CODE = {torch.float32: _lib.MOE_F32, torch.float16: _lib.MOE_F16, torch.bfloat16: _lib.MOE_BF16}


class Guarded:
    """Buffers in one allocation, each between two bands of a pattern."""

    def __init__(self, fill, **sizes):
        self.at, end = {}, BAND
        for name, size in sizes.items():
            self.at[name] = (end, size)
            end = (end + size + 255) // 256 * 256 + BAND
        self.buf = torch.full((end,), fill, dtype=torch.uint8, device=DEV)
        self.fill = fill

    def ptr(self, name):
        return self.buf.data_ptr() + self.at[name][0]

    def view(self, name, dtype, *shape):
        start, size = self.at[name]
        return self.buf[start:start + size].view(dtype).view(*shape)

    def intact(self):
        outside = torch.ones_like(self.buf, dtype=torch.bool)
        for start, size in self.at.values():
            outside[start:start + size] = False
        return bool((self.buf[outside] == self.fill).all())


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 1000), (301, 1032), (7, 2056), (4, 5001), (9, 7168), (3, 16392), (2, 20001)])
def test_norm_writes_its_outputs_only(dtype, rows, cols):
    size = dtype.itemsize
    x, r, dy, dh = (torch.randn(rows, cols, device=DEV).to(dtype) for _ in range(4))
    w = torch.randn(cols, device=DEV).to(dtype)
    group = next(g for g in (128, 8, 7, 1) if cols % g == 0)
    need = ctypes.c_int64()
    _lib.check(_lib.lib().moe_rms_norm_grad_workspace(rows, cols, ctypes.addressof(need)))
    seen = []
    for fill in (0xFF, 0x5A):  # NaN among them
        g = Guarded(fill, y=rows * cols * size, h=rows * cols * size, q=rows * cols, s=4 * rows * (cols // group), st=4 * (rows + 3) * (cols // group),
                    dx=rows * cols * size, dw=cols * size, ws=need.value)
        lib, c = _lib.lib(), CODE[dtype]
        _lib.check(lib.moe_rms_norm(x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), c, c, rows, cols, 1e-6, g.ptr("y"), cols, g.ptr("h"),
                                    cols, stream()))
        _lib.check(lib.moe_rms_norm_quant(x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), c, c, rows, cols, 1e-6, 0, group, 1e-10, 0,
                                          g.ptr("q"), g.ptr("s"), 0, None, g.ptr("h"), stream()))
        _lib.check(lib.moe_rms_norm_quant(x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), c, c, rows, cols, 1e-6, 0, group, 1e-10, 1,
                                          g.ptr("q"), g.ptr("st"), rows + 3, None, g.ptr("h"), stream()))
        _lib.check(lib.moe_rms_norm_grad(dy.data_ptr(), dh.data_ptr(), g.ptr("h"), cols, w.data_ptr(), c, c, rows, cols, 1e-6, g.ptr("dx"),
                                         g.ptr("dw"), g.ptr("ws"), need.value, stream()))
        assert g.intact()
        st = g.view("st", torch.float32, cols // group, rows + 3)
        assert (st[:, rows:].contiguous().view(torch.uint8) == fill).all()  # columns behind the last row
        assert torch.equal(st[:, :rows].t(), g.view("s", torch.float32, rows, cols // group))
        seen.append([g.view(n, dtype, -1).clone() for n in ("y", "h", "dx", "dw")] + [g.view("q", torch.uint8, -1).clone()])
    assert all(torch.equal(a, b) for a, b in zip(*seen))
    xl, wl, rl = (t.clone().requires_grad_() for t in (x, w, r))
    y, h = fg.rms_norm(xl, wl, 1e-6, rl)
    dx, dw = torch.autograd.grad([y, h], [xl, wl], [dy, dh])
    for a, b in zip(seen[0], (y, h, dx, dw)):
        assert torch.equal(a, b.detach().flatten())


@pytest.mark.parametrize("T,E,k,S", [(1, 1, 1, 1), (5, 8, 2, 1), (129, 256, 8, 1), (700, 60, 4, 1), (700, 60, 4, 9), (3000, 128, 8, 700), (50, 1024, 32, 3),
                                     (40, 1021, 3, 1)])
def test_balance_writes_its_outputs_only(T, E, k, S):
    logits = torch.randn(T, E, device=DEV)
    ids = torch.randint(-1, E, (T, k), device=DEV, dtype=torch.int32)
    cu = None if S == 1 else torch.sort(torch.randint(0, T + 1, (S + 1,), device=DEV)).values.int()
    need = (ctypes.c_int64 * 2)()
    _lib.check(_lib.lib().moe_balance_loss_workspace(T, E, k, S, ctypes.addressof(need)))
    one = torch.ones((), device=DEV)
    seen = []
    for fill in (0xFF, 0x5A):
        g = Guarded(fill, loss=4, counts=4 * S * E, saved=need[1], ws=need[0], d=4 * T * E)
        _lib.check(_lib.lib().moe_balance_loss(logits.data_ptr(), E, _lib.MOE_F32, T, E, ids.data_ptr(), 0, k, 1, _lib.ptr(cu), S, None,
                                               g.ptr("loss"), g.ptr("counts"), g.ptr("saved"), g.ptr("ws"), need[0], None, stream()))
        _lib.check(_lib.lib().moe_balance_loss_grad(logits.data_ptr(), E, _lib.MOE_F32, T, E, k, 1, _lib.ptr(cu), S, None, g.ptr("saved"),
                                                    one.data_ptr(), g.ptr("d"), stream()))
        assert g.intact()
        seen.append((g.view("loss", torch.float32, 1).clone(), g.view("counts", torch.int32, -1).clone(), g.view("d", torch.float32, T, E).clone()))
    assert all(torch.equal(a, b) for a, b in zip(*seen))
    leaf = logits.clone().requires_grad_()
    loss, counts = fg.moe_balance_loss(leaf, ids, "sigmoid", cu)
    (d,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(seen[0][0], loss.detach().view(1)) and torch.equal(seen[0][1], counts.flatten()) and torch.equal(seen[0][2], d)


def test_threads_beside_one_another():
    """Four threads, each with its own stream and sizes, forward and backward at once."""
    work, wrong = [], []
    for i in range(4):
        g = torch.Generator(device=DEV)
        g.manual_seed(i)
        M, H, E, k = 300 + 97 * i, 512 * (i + 1), 32 * (i + 1), 4
        x, r, dy = (torch.randn((M, H), generator=g, device=DEV).bfloat16() for _ in range(3))
        w = torch.randn((H,), generator=g, device=DEV).bfloat16()
        logits = torch.randn((M, E), generator=g, device=DEV)
        ids = torch.randint(0, E, (M, k), generator=g, device=DEV)
        work.append((x, r, w, dy, logits, ids))

    def step(x, r, w, dy, logits, ids):
        leaves = [t.clone().requires_grad_() for t in (x, r, w, logits)]
        y, h = fg.rms_norm(leaves[0], leaves[2], 1e-6, leaves[1])
        q = fg.rms_norm_quant(x, w, 1e-6, r, group_size=128)
        loss, counts = fg.moe_balance_loss(leaves[3], ids)
        grads = torch.autograd.grad([y, loss], leaves, [dy, torch.ones_like(loss)])
        return [y.detach(), h.detach(), q[0].view(torch.uint8), q[1], loss.detach(), counts, *grads]

    want = [step(*w) for w in work]
    torch.cuda.synchronize()

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(30):
                    got = step(*work[i])
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
                s.synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
