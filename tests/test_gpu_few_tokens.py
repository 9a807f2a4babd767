"""fused_moe_few_tokens against 64 bits and against the operators that it stands for.

Tolerances, element by element, with u = eps / 2 of the activations' type: a sum of n products in fp32 is off by at most n 2^-23 of
the sum of absolute products; h is rounded to u |h| (half of the smallest subnormal of f16 below 2^-14) behind a gate that is off by
what its two sums are (slopes of at most 1.1) and 2^-19 of itself; a routing weight by 2^-20 of itself; both reach the output
through |W2|, which is rounded once.  In e4m3 a value that the two computations put on either side of a border moves by a whole step,
so the layer's own tolerance holds there: relative L2 1e-2, cosine 0.9999."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import testing

pytestmark = pytest.mark.gpu
DEV = "cuda"
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 0.0}


def make(M, E, H, I, Is=0, dtype=torch.bfloat16, fp8=False, router=None, bias=True, residual=False, seed=0, gap=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    d = {"x": n(M, H + gap).to(dtype)[:, :H], "router": (n(E, H) / H**0.5).to(router or dtype), "bias": 0.1 * n(E) if bias else None,
         "residual": n(M, H).to(dtype) if residual else None, "w1_scale": None, "w2_scale": None, "shared_w1": None, "shared_w2": None,
         "shared_w1_scale": None, "shared_w2_scale": None}
    if fp8:
        d["w1"], d["w1_scale"] = testing.make_fp8_block_weights(E, 2 * I, H, DEV, seed=seed + 1, std=0.05)
        d["w2"], d["w2_scale"] = testing.make_fp8_block_weights(E, H, I, DEV, seed=seed + 2, std=0.05)
        if Is:
            a, b = testing.make_fp8_block_weights(1, 2 * Is, H, DEV, seed=seed + 3, std=0.05)
            c, e = testing.make_fp8_block_weights(1, H, Is, DEV, seed=seed + 4, std=0.05)
            d |= {"shared_w1": a[0], "shared_w1_scale": b[0], "shared_w2": c[0], "shared_w2_scale": e[0]}
    else:
        d["w1"], d["w2"] = (0.05 * n(E, 2 * I, H)).to(dtype), (0.05 * n(E, H, I)).to(dtype)
        if Is:
            d["shared_w1"], d["shared_w2"] = (0.05 * n(2 * Is, H)).to(dtype), (0.05 * n(H, Is)).to(dtype)
    return d


def call(d, topk, scoring="sigmoid", groups=1, kept=1, factor=1.0, renormalize=True, routing=True):
    rest = {k: d[k] for k in ("w1_scale", "w2_scale", "shared_w1", "shared_w2", "shared_w1_scale", "shared_w2_scale", "residual")}
    return fg.fused_moe_few_tokens(d["x"], d["router"], d["w1"], d["w2"], topk, renormalize, scoring, groups, kept, factor, d["bias"],
                                   return_routing=routing, **rest)


def route64(d, topk, scoring, groups, kept, factor, renormalize):
    logits = d["x"].double() @ d["router"].double().t()
    u = logits.sigmoid() if scoring == "sigmoid" else logits.softmax(-1)
    r = u if d["bias"] is None else u + d["bias"].double()
    M, E = r.shape
    per = E // groups
    if groups > 1:
        score = r.view(M, groups, per).topk(min(2, per), -1).values.sum(-1)
        keep = torch.zeros_like(score, dtype=torch.bool).scatter_(1, score.topk(kept, -1).indices, True)
        r = r.masked_fill(~keep.repeat_interleave(per, 1), float("-inf"))
    ids = r.topk(topk, -1).indices
    w = u.gather(1, ids)
    return (w / w.sum(-1, keepdim=True) if renormalize else w) * factor, ids


def widened(w, s):
    return w.double() if s is None else w.double() * s.double().repeat_interleave(128, -2).repeat_interleave(128, -1)


def held(v):
    g = v.unflatten(-1, (-1, 128))
    s = g.abs().amax(-1, keepdim=True).float().clamp(min=1e-10) * torch.tensor(1 / 448, device=v.device)
    return ((g.float() / s).clamp(-448, 448).to(torch.float8_e4m3fn).double() * s.double()).flatten(-2)


def expert64(x, w1, w2, dtype, fp8):
    """Output of one expert for a token and the bound on what the kernel may be off, before the last rounding."""
    u = torch.finfo(dtype).eps / 2
    if fp8:
        x = held(x)
    H, I = w1.shape[1], w2.shape[1]
    z, S = w1 @ x, w1.abs() @ x.abs()
    e = (H + 2) * 2.0**-23 * S
    s, up = torch.nn.functional.silu(z[:I]), z[I:]
    h = s * up
    eh = up.abs() * 1.1 * e[:I] + s.abs() * e[I:] + 1.1 * e[:I] * e[I:] + 2.0**-19 * h.abs()
    eh = eh + u * (h.abs() + eh) + TINY[dtype]
    if fp8:
        h = held(h.to(dtype).double())
    return w2 @ h, w2.abs() @ eh + (I + 2) * 2.0**-23 * (w2.abs() @ (h.abs() + eh))


def check(d, topk, scoring="sigmoid", groups=1, kept=1, factor=1.0, renormalize=True, tokens=None):
    """``tokens``: those whose results are looked at, all by default."""
    out, tw, ti = call(d, topk, scoring, groups, kept, factor, renormalize)
    x, dtype, fp8 = d["x"], d["x"].dtype, d["w1_scale"] is not None
    M, H = x.shape
    tokens = list(range(M)) if tokens is None else tokens
    assert out.shape == (M, H) and out.dtype == dtype and tw.dtype == torch.float32 and ti.dtype == torch.int32
    w64, i64 = route64(d, topk, scoring, groups, kept, factor, renormalize)
    assert torch.equal(ti[tokens].long(), i64[tokens]), "routed elsewhere"
    torch.testing.assert_close(tw[tokens].double(), w64[tokens], rtol=2e-5, atol=1e-7)
    u = torch.finfo(dtype).eps / 2
    want, bound = [], []
    for t in tokens:
        y = torch.zeros(H, dtype=torch.float64, device=DEV) if d["residual"] is None else d["residual"][t].double()
        e, mag = torch.zeros_like(y), y.abs()
        for j in range(topk):
            q = int(ti[t, j])
            a, b = expert64(x[t].double(), widened(d["w1"][q], None if not fp8 else d["w1_scale"][q]),
                            widened(d["w2"][q], None if not fp8 else d["w2_scale"][q]), dtype, fp8)
            w = float(tw[t, j])
            y, e, mag = y + w * a, e + abs(w) * (b + 2.0**-20 * a.abs()), mag + abs(w) * a.abs()
        if d["shared_w1"] is not None:
            a, b = expert64(x[t].double(), widened(d["shared_w1"], d["shared_w1_scale"]), widened(d["shared_w2"], d["shared_w2_scale"]), dtype, fp8)
            y, e, mag = y + a, e + b, mag + a.abs()
        e = e + (topk + 16) * 2.0**-23 * mag
        want.append(y)
        bound.append(e + u * (y.abs() + e) + TINY[dtype])
    want, bound = torch.stack(want), torch.stack(bound)
    off = (out[tokens].double() - want).abs()
    if fp8:
        assert off.norm() <= 1e-2 * want.norm()
        assert torch.nn.functional.cosine_similarity(out[tokens].double().flatten(), want.flatten(), dim=0) >= 0.9999
    else:
        assert (off <= bound).all(), f"{float((off / bound).max()):.3g} times the bound"
    again = call(d, topk, scoring, groups, kept, factor, renormalize)
    assert all(torch.equal(p[tokens], q[tokens]) for p, q in zip((out, tw, ti), again)), "two runs differ"
    assert fg.read_status() == 0


HALF = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("E,topk,H,I,Is", [(1, 1, 64, 64, 0), (8, 2, 256, 128, 0), (16, 4, 512, 192, 64), (60, 4, 1408, 704, 128), (64, 32, 320, 64, 448)])
def test_half(E, topk, H, I, Is, M, dtype):
    check(make(M, E, H, I, Is, dtype, residual=M % 2 == 1), topk)
    check(make(M, E, H, I, Is, dtype, bias=False, seed=7), topk, "softmax")


@pytest.mark.parametrize("M", [1, 3, 8])
@pytest.mark.parametrize("E,topk,H,I,Is", [(8, 2, 256, 128, 0), (16, 4, 512, 384, 128), (32, 8, 2048, 768, 0), (16, 8, 7168, 256, 256), (2, 1, 4736, 128, 128)])
def test_fp8(E, topk, H, I, Is, M):
    check(make(M, E, H, I, Is, fp8=True, residual=M == 3), topk)
    check(make(M, E, H, I, Is, torch.float16, fp8=True, seed=5), topk, "softmax", factor=2.5)


@pytest.mark.parametrize("M", [1, 8])
def test_full_sizes(M):
    check(make(M, 128, 2048, 768, 768, residual=True), 8, "softmax")
    check(make(M, 8, 4096, 14336), 2, "softmax")
    check(make(M, 24, 7168, 2048, 2048, fp8=True, residual=True), 8, "sigmoid", 8, 4, 2.5)


@pytest.mark.parametrize("E,groups,kept,topk", [(256, 8, 4, 8), (64, 4, 1, 6), (60, 3, 2, 5), (32, 32, 4, 4), (1024, 32, 2, 32), (300, 1, 1, 7)])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_groups(E, groups, kept, topk, scoring):
    check(make(8, E, 128, 64), topk, scoring, groups, kept, 1.5, renormalize=False)


@pytest.mark.parametrize("M", [1, 2, 4])
def test_routing_is_the_routers(M):
    d = make(M, 256, 7168, 64, seed=3)
    _, tw, ti = call(d, 8, "sigmoid", 8, 4, 2.5)
    w, i = fg.router_gemm_grouped_topk(d["x"], d["router"], 8, 4, 8, True, 2.5, d["bias"], 1)
    assert torch.equal(ti, i)
    torch.testing.assert_close(tw, w, rtol=1e-6, atol=0)


@pytest.mark.parametrize("gap", [8, 1, 3])
def test_layouts(gap):
    check(make(4, 16, 256, 128, 64, gap=gap, residual=True), 4)
    d = make(4, 16, 256, 128, 64, router=torch.float32, residual=True)
    d["residual"] = d["residual"].t().contiguous().t()
    d["bias"] = d["bias"].view(1, -1)
    d["bias"] = d["bias"][0]
    check(d, 4)
    flat = torch.empty(16 * 256 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:]
    d["w1"] = flat.view(16, 256, 256).copy_(d["w1"])  # begins at an odd address
    check(d, 4)


@pytest.mark.parametrize("M", [1, 8])
def test_wide_rows_beyond_shared_memory(M):
    check(make(M, 4, 16384, 64, 64), 2)
