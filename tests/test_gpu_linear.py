"""fused_linear against 64 bits: value and gradients, layouts, sizes, refusals.

Tolerances, element by element, with u = eps / 2 of the type and S = |x| |W|^T (+ |b|) in 64 bits:

* a sum of K products in fp32 is off by at most K 2^-23 S (any order, each step rounded or cut), called dz below;
* the activations have slopes of at most 1.13 (gelu) and 1.1 (silu), and are evaluated to 2^-20 of |z| + 1; the gate's product is
  off by |up| 1.1 dgate + |silu(gate)| dup + 2^-19 |y|;
* y is rounded once: u |y|, and half of the smallest subnormal of f16 below 2^-14;
* z is kept rounded (for the gated activation in fp32; below 2^-14 in f16 by half of the smallest subnormal, which takes a z of less
  than 2^-25 to the zero at relu's step), which moves act' by at most u |z| max|act''| (0.8 gelu, 0.5 silu; relu's step only where z is
  within its own error of zero, and those elements are given the whole of |dy|); dz itself is rounded, u |dz|.  Both reach dx and dW
  through the products of absolute values."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "silu_and_mul"]
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 0.0, torch.float32: 0.0}


def _act64(z, act):
    F = torch.nn.functional
    if act == "silu_and_mul":
        h = z.shape[-1] // 2
        return F.silu(z[..., :h]) * z[..., h:]
    return {None: lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[act](z)


def make(M, K, N, dtype, act=None, bias=None, residual=False, gap=0, offset=0, seed=0, std=0.05):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    W = 2 * N if act == "silu_and_mul" else N

    def rows(r, c, s=1.0):
        t = (s * torch.randn((r * (c + gap) + offset,), generator=g, device=DEV)).to(dtype)
        return t[offset:].view(r, c + gap)[:, :c]

    b = None if bias is None else torch.randn((W,), generator=g, device=DEV).to(dtype if bias == "same" else torch.float32)
    return rows(M, K), rows(W, K, std), b, rows(M, N) if residual else None


def reference(x, w, b, r, act, dy=None):
    """y, gradients and the bounds of the header, in 64 bits."""
    dtype = x.dtype
    u = torch.finfo(dtype).eps / 2
    K, M = x.shape[1], x.shape[0]
    leaves = [t.detach().double().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    X, W, B, R = leaves
    z = X @ W.t()
    if B is not None:
        z = z + B
    z.retain_grad()
    y = _act64(z, act)
    out = y if R is None else y + R
    S = X.abs() @ W.abs().t() + (0 if B is None else B.abs())
    dz_err = (K + 2) * 2.0**-23 * S
    if act == "silu_and_mul":
        h = z.shape[1] // 2
        gate, up = z[:, :h], z[:, h:]
        s = torch.nn.functional.silu(gate)
        y_err = up.abs() * 1.1 * dz_err[:, :h] + s.abs() * dz_err[:, h:] + 1.1 * dz_err[:, :h] * dz_err[:, h:] + 2.0**-19 * y.abs()
    else:
        y_err = 1.13 * dz_err + (0 if act is None else 2.0**-20 * (z.abs() + 1))
    bounds = {"y": (y_err + 2.0**-23 * out.abs() + u * (out.abs() + y_err) + TINY[dtype]).detach()}
    got = {"y": out.detach()}
    if dy is not None:
        out.backward(dy.double())
        D, dZ = dy.double().abs(), z.grad
        e = dz_err if act == "silu_and_mul" else u * z.abs() + TINY[dtype] + dz_err  # of the z that the backward pass sees
        if act == "silu_and_mul":
            eg, eu = e[:, :h], e[:, h:]
            err = torch.cat([D * ((up.abs() + eu) * 0.5 * eg + 1.1 * eu), D * 1.1 * eg], 1)
            err = err + 2.0**-19 * torch.cat([D * (up.abs() + eu), D * (gate.abs() + 1)], 1)
        elif act == "relu":
            err = D * (z.abs() <= e)
        else:
            err = D * e * {None: 0.0, "silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.85}[act]
        if act not in (None, "silu_and_mul"):
            err = err + 2.0**-19 * D
        db_err = err.sum(0) + (M + 16) * 2.0**-23 * dZ.abs().sum(0)
        err = (err + (0 if act is None else u * (dZ.abs() + err) + TINY[dtype])).detach()
        A = dZ.detach().abs() + err

        def product(p, q, pe, k):  # sum over k of p q with p off by pe
            return pe @ q + (k + 2) * 2.0**-23 * (p @ q)

        got |= {"dx": X.grad, "dw": W.grad}
        ex, ew = product(A, W.abs().detach(), err, W.shape[0]), product(A.t(), X.abs().detach(), err.t(), M)
        bounds |= {"dx": ex + u * (X.grad.abs() + ex) + TINY[dtype], "dw": ew + u * (W.grad.abs() + ew) + TINY[dtype]}
        if b is not None:
            got["db"] = B.grad
            ub = torch.finfo(b.dtype).eps / 2
            bounds["db"] = (db_err + ub * (B.grad.abs() + db_err) + TINY[b.dtype]).detach()
        if r is not None:
            got["dr"], bounds["dr"] = R.grad, torch.zeros_like(R.grad)
    return got, bounds


def close(name, got, want, bound):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), name
    bad = off > bound
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} beyond, worst {float((off / bound.clamp(min=1e-300)).max()):.3g} times"


def check(M, K, N, dtype, act=None, bias=None, residual=False, train=False, **kw):
    import flaggems_vllm_b200 as fg

    x, w, b, r = make(M, K, N, dtype, act, bias, residual, **kw)
    dy = torch.randn((M, N), device=DEV, generator=torch.Generator(device=DEV).manual_seed(9)).to(dtype) if train else None
    want, bound = reference(x, w, b, r, act, dy)
    if not train:
        y = fg.fused_linear(x, w, b, act, r)
        assert y.shape == (M, N) and y.dtype == dtype and y.is_contiguous()
        close("y", y, want["y"], bound["y"])
        assert torch.equal(y, fg.fused_linear(x, w, b, act, r)), "two runs differ"
        return
    names = [n for n, t in (("dx", x), ("dw", w), ("db", b), ("dr", r)) if t is not None]
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    y = fg.fused_linear(x, w, b, act, r)
    grads = torch.autograd.grad(y, leaves, dy)
    close("y", y.detach(), want["y"], bound["y"])
    for n, g, leaf in zip(names, grads, leaves):
        assert g.shape == leaf.shape and g.dtype == leaf.dtype
        close(n, g, want[n], bound[n])
    assert fg.read_status() == 0


HALF = [torch.bfloat16, torch.float16]
# one token to some thousand; tile edges (64, 128, 256) and one beside them; K of less than a step and of many
SIZES = [(1, 64, 16), (1, 2048, 512), (1, 7168, 256), (2, 136, 128), (7, 512, 1000), (16, 1024, 64), (17, 64, 4096), (33, 4096, 264),
         (64, 2048, 2048), (65, 256, 136), (128, 128, 128), (129, 320, 384), (200, 7168, 72), (255, 512, 512), (257, 1024, 520),
         (512, 2048, 768), (1000, 512, 1032), (1500, 256, 2048), (2049, 192, 1288), (4096, 64, 4096)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_values(M, K, N, dtype):
    check(M, K, N, dtype)
    check(M, K, N, dtype, "silu_and_mul", residual=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", [(1, 256, 200), (40, 520, 96), (300, 256, 384), (2100, 128, 2056)])
def test_epilogues(M, K, N, act):
    check(M, K, N, torch.bfloat16, act, bias="same", residual=True)
    check(M, K, N, torch.float16, act, bias="f32")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", [(1, 128, 64), (24, 264, 80), (300, 512, 256), (1111, 200, 328), (2304, 512, 1024)])
def test_gradients(M, K, N, act):
    check(M, K, N, torch.bfloat16, act, bias="f32", residual=True, train=True)
    check(M, K, N, torch.float16, act, bias="same", train=True)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 7, 3), (3, 65, 17), (50, 1023, 129), (501, 333, 767), (2000, 37, 1201)])
def test_odd_sizes(M, K, N, train):
    for act in (None, "gelu", "silu_and_mul"):
        check(M, K, N, torch.float16, act, bias="same", residual=True, train=train)
        check(M, K, N, torch.bfloat16, act, train=train)


@pytest.mark.parametrize("gap,offset", [(8, 0), (1, 0), (0, 1), (8, 8), (3, 5)])
@pytest.mark.parametrize("M", [1, 30, 300])
def test_layouts(M, gap, offset):
    for act in (None, "silu_and_mul"):
        check(M, 256, 192, torch.bfloat16, act, residual=True, train=True, gap=gap, offset=offset)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 500, 300), (70, 33, 129), (300, 501, 333), (129, 256, 64)])
def test_fp32(M, K, N, act):
    check(M, K, N, torch.float32, act, bias="same", residual=True, train=True)
    check(M, K, N, torch.float32, act, gap=3)
