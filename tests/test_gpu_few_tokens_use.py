"""fused_moe_few_tokens in use: graphs, streams, threads, guard bands, bad values, long offsets; together with the operators around it."""

import ctypes
import subprocess
import sys
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwad

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib
from flaggems_vllm_b200.router_gemm import ROW_STREAM_MAX
from test_gpu_few_tokens import call, check, make
from test_gpu_norm_balance_bounds import CODE, Guarded, stream

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16
FORMATS = [(BF, False), (HF, False), (BF, True)]


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype,fp8", FORMATS)
def test_captured_and_replayed(dtype, fp8):
    """Two graphs of one layer, replayed in turn with other tokens in place."""
    d = make(5, 32, 512, 256, 128, dtype, fp8, residual=True)
    call(d, 4)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(d, 4)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(d, 4))
    for seed in (5, 6, 7):
        n = make(5, 32, 512, 256, 128, dtype, fp8, residual=True, seed=seed)
        d["x"].copy_(n["x"])
        d["residual"].copy_(n["residual"])
        want = call(d, 4)
        for graph, out in zip(graphs, outs):
            for t in out:
                t.zero_()
            graph.replay()
            assert same(out, want)
    assert fg.read_status() == 0


@pytest.mark.parametrize("dtype,fp8", FORMATS)
def test_two_streams_at_once(dtype, fp8):
    """Each call takes the whole GPU if it can get it; two of them share it and both end."""
    ds = [make(3 + i, 64, 1024, 512, 256, dtype, fp8, seed=10 * i) for i in range(2)]
    want = [call(d, 6) for d in ds]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(ds[i], 6))
    torch.cuda.synchronize()
    assert all(same(g, want[i]) for i in range(2) for g in got[i])
    assert fg.read_status() == 0


def test_threads_beside_one_another():
    ds = [make(1 + 2 * i, 16 * (i + 1), 256 * (i + 1), 128 * (i + 1), 128, (BF, HF, BF)[i], i == 2, seed=i, residual=True) for i in range(3)]
    want = [call(d, 3) for d in ds]
    torch.cuda.synchronize()
    wrong = []

    def body(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = call(ds[i], 3)
                torch.cuda.current_stream().synchronize()
                if not same(got, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and fg.read_status() == 0


@pytest.mark.parametrize("dtype,fp8", FORMATS)
def test_behind_the_kernels_that_make_its_operands(dtype, fp8):
    """Called right behind kernels of this library and torch's that write its tokens, residual and weights."""
    d = make(4, 16, 512, 256, 128, dtype, fp8, residual=True)
    eye = torch.eye(512, device=DEV, dtype=dtype)
    want = call(d, 4)
    held = {k: d[k].clone() for k in ("x", "residual", "w1", "w2", "router")}
    for _ in range(5):
        for k in held:
            d[k].zero_()
        for k in ("w1", "w2", "residual", "router"):
            d[k].copy_(held[k])
        d["x"] = fg.fused_linear(held["x"], eye)  # the same bits: one product of each sum is not zero
        assert same(call(d, 4), want)


@pytest.mark.parametrize("dtype,fp8", FORMATS)
def test_bad_values_stay_in_their_token(dtype, fp8):
    """NaN and Inf in a token, and weights of NaN, reach no token that has nothing to do with them.  A token of other values chooses
    other experts, and with the experts of a call its work is shared out anew: the others' sums may be added in another order, so they
    are held to the bounds of any call.  Their routing keeps its bits."""
    d = make(6, 32, 512, 256, 128, dtype, fp8)
    out, tw, ti = call(d, 4)
    for value in (float("nan"), float("inf"), torch.finfo(dtype).max):
        b = dict(d)
        b["x"] = d["x"].clone()
        b["x"][2, 7] = value
        got, gw, gi = call(b, 4)
        keep = [0, 1, 3, 4, 5]
        assert torch.equal(gw[keep], tw[keep]) and torch.equal(gi[keep], ti[keep])
        check(b, 4, tokens=keep)
        assert ((gi >= 0) & (gi < 32)).all() and all(len(set(r.tolist())) == 4 for r in gi)
        if value != value:
            assert got[2].isnan().all()
    e = int(ti[0, 0])
    b = dict(d)
    for k in ("w1", "w2"):
        b[k] = d[k].clone()
        b[k].view(torch.uint8)[e] = 0x7F  # NaN in e4m3; in the wider types finite in f16's case or NaN, so written as such
        if not fp8:
            b[k][e] = float("nan")
    got, gw, gi = call(b, 4)
    has = (ti == e).any(1)
    assert torch.equal(gi, ti) and torch.equal(got[~has], out[~has]) and got[has].isnan().all()
    b = dict(d)
    for bad in (float("nan"), float("inf"), -float("inf")):  # any logits, any choice: experts that exist, each once
        b["router"] = d["router"].clone()
        b["router"][::3] = bad
        for scoring in ("sigmoid", "softmax"):
            _, _, gi = call(b, 4, scoring, 4, 2)
            assert ((gi >= 0) & (gi < 32)).all() and all(len(set(r.tolist())) == 4 for r in gi)
    assert fg.read_status() == 0


@pytest.mark.parametrize("dtype,fp8", FORMATS)
@pytest.mark.parametrize("M,E,H,I,Is,topk", [(1, 1, 128, 128, 0, 1), (8, 8, 128, 128, 128, 8), (3, 60, 1408, 384, 0, 4), (2, 64, 2048, 768, 512, 32)])
def test_writes_its_outputs_only(M, E, H, I, Is, topk, dtype, fp8):
    d = make(M, E, H, I, Is, dtype, fp8, residual=True)
    lib, need = _lib.lib(), ctypes.c_int64()
    _lib.check(lib.moe_few_tokens_workspace(M, E, I, Is, topk, int(fp8), ctypes.addressof(need)))
    p, seen = _lib.ptr, []
    for fill in (0xFF, 0x5A):
        g = Guarded(fill, out=M * H * 2, w=M * topk * 4, ids=M * topk * 4, ws=need.value)
        _lib.check(lib.moe_few_tokens(p(d["x"]), H, CODE[dtype], p(d["router"]), CODE[dtype], p(d["bias"]), p(d["w1"]), p(d["w2"]), p(d["w1_scale"]),
                                      p(d["w2_scale"]), p(d["shared_w1"]), p(d["shared_w2"]), p(d["shared_w1_scale"]), p(d["shared_w2_scale"]),
                                      p(d["residual"]), H, M, E, H, I, Is, topk, 1, 1, 1, 1.0, 1, g.ptr("out"), g.ptr("w"), g.ptr("ids"), g.ptr("ws"),
                                      need.value, _lib.status_word(d["x"].device).data_ptr(), stream()))
        assert g.intact()
        seen.append((g.view("out", dtype, M, H).clone(), g.view("w", torch.float32, M, topk).clone(), g.view("ids", torch.int32, M, topk).clone()))
    assert same(*seen) and same(seen[0], call(d, topk)) and fg.read_status() == 0


@pytest.mark.parametrize("dtype,fp8", [(BF, False), (BF, True)])
def test_offsets_beyond_32_bits_of_weights(dtype, fp8):
    """Experts that begin more than 2^31 elements into w1 and w2; the first and the last are routed to."""
    E, H, I = 1024, 2048, 1152  # w1: 4.8 10^9 elements, w2: 2.4 10^9
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough free memory")
    small = make(3, 4, H, I, 0, dtype, fp8, bias=False)
    spots = [0, 511, 1000, 1023]
    d = dict(small)
    for k in ("w1", "w2", "w1_scale", "w2_scale"):
        if small[k] is None:
            continue
        d[k] = torch.zeros((E, *small[k].shape[1:]), dtype=torch.uint8 if small[k].dtype.itemsize == 1 else small[k].dtype, device=DEV)
        if d[k].dtype == torch.uint8:
            d[k][spots] = small[k].view(torch.uint8)
            d[k] = d[k].view(torch.float8_e4m3fn)
        else:
            d[k][spots] = small[k]
    d["router"] = torch.zeros((E, H), dtype=dtype, device=DEV)
    d["router"][spots] = small["router"]
    d["bias"] = torch.full((E,), -10.0, device=DEV)
    d["bias"][spots] = 0.0
    out, tw, ti = call(d, 4)
    want, ww, wi = call(small, 4)
    assert torch.equal(ti, torch.tensor(spots, device=DEV, dtype=torch.int32)[wi.long()]) and torch.equal(tw, ww)
    assert torch.equal(out, want)


def test_layouts_that_are_copied_first():
    d = make(4, 16, 256, 128, 64, BF, residual=True)
    want = call(d, 4)
    odd = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    apart = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731
    for change in (odd, apart):
        for k in ("x", "router", "w1", "w2", "shared_w1", "shared_w2", "residual", "bias"):
            assert same(call({**d, k: change(d[k])}, 4), want), k
    assert same(call({**d, "bias": d["bias"].double().view(4, 4)}, 4), want)
    assert same(call({**d, "w1": d["w1"].transpose(1, 2).contiguous().transpose(1, 2)}, 4), want)


def test_no_tokens_and_no_gradient():
    d = make(0, 16, 256, 128, 64, BF)
    out, tw, ti = call(d, 4)
    assert out.shape == (0, 256) and tw.shape == ti.shape == (0, 4) and ti.dtype == torch.int32
    d = make(2, 16, 256, 128, 64, BF)
    want = call(d, 4)
    d["w1"].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        call(d, 4)
    with torch.no_grad():
        assert same(call(d, 4), want)
    with torch.inference_mode():
        assert same(call(d, 4), want)
    with fwad.dual_level(), torch.no_grad():
        for k in ("x", "router", "w2", "shared_w1", "bias"):
            with pytest.raises(RuntimeError, match="forward mode"):
                call({**d, k: fwad.make_dual(d[k], torch.ones_like(d[k]))}, 4)


def test_arguments_of_other_types():
    """Numbers that are not Python's own are taken by their value."""
    import numpy as np

    d = make(2, 16, 256, 128, 0, BF)
    want = call(d, 4, "softmax", 4, 2, 2.5, True)
    got = fg.fused_moe_few_tokens(d["x"], d["router"], d["w1"], d["w2"], np.int64(4), np.bool_(True), "softmax", np.int32(4), torch.tensor(2), np.float32(2.5),
                                  d["bias"], return_routing=True)
    assert same(got, want)


def test_launches_are_counted():
    d = make(2, 16, 256, 128, 0, BF)
    before = _lib.LAUNCHES
    call(d, 4)
    assert _lib.LAUNCHES == before + 2


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M", [1, 6])
def test_a_layer_in_one_call_and_in_parts(M, dtype):
    """norm -> (router, experts, shared expert, residual) in one call, against the operators one behind another.  The parts round the
    routed sum and the shared expert's output to the type on the way: twice more than the one call, so the two are apart by at most
    three roundings of what passes through, beside the bounds that both keep (both take at most that again)."""
    E, H, I, Is, topk = 32, 512, 256, 128, 4
    d = make(M, E, H, I, Is, dtype, residual=True)
    gamma = torch.rand(H, device=DEV).to(dtype) + 0.5
    d["x"], stream_out = fg.rms_norm(d["x"], gamma, 1e-6, d["residual"])
    d["residual"] = stream_out
    out, tw, ti = call(d, topk)
    logits = fg.router_gemm(d["x"], d["router"])
    pw, pi = fg.grouped_topk(logits, 1, 1, topk, True, 1.0, d["bias"], 1)
    assert torch.equal(pi.int(), ti)
    if M <= ROW_STREAM_MAX:  # one order of the logits' sums
        assert torch.equal(pw, tw)
    # each logit is off by H 2^-23 of its absolute products in either order; a score by that much of itself at most, and so is the sum
    # of the scores: twice that for a weight, in each of the two
    S = (d["x"].double().abs() @ d["router"].double().abs().t()).max()
    assert ((pw - tw).abs() <= (4 * H * 2.0**-23 * float(S) + 2.0**-20) * tw).all()
    routed = fg.fused_experts_impl(d["x"], d["w1"], d["w2"], pw, pi)
    base = routed + d["residual"]
    h = fg.fused_linear(d["x"], d["shared_w1"], activation="silu_and_mul")
    parts = fg.fused_linear(h, d["shared_w2"], residual=base)
    u = torch.finfo(dtype).eps / 2
    through = routed.double().abs() + base.double().abs() + parts.double().abs() + (parts.double() - base.double()).abs()
    # sums of absolute products, of which both forms round the same factors (h to u, twice over in the routed part: value and weight)
    hw = (h.double().abs() @ d["shared_w2"].double().abs().t())
    slack = torch.zeros_like(hw)
    for t in range(M):
        for j in range(topk):
            q = int(ti[t, j])
            z = d["w1"][q].double() @ d["x"][t].double()
            slack[t] += float(tw[t, j]) * (d["w2"][q].double().abs() @ (torch.nn.functional.silu(z[:I]) * z[I:]).abs())
    assert ((out.double() - parts.double()).abs() <= 4 * u * through + 4 * u * (hw + slack)).all()
    assert fg.read_status() == 0


def test_decode_steps_of_three_layers_in_a_graph():
    """Norm, projection, norm, layer of experts, three deep, captured once and replayed for several steps, against the eager calls."""
    H, E, I, Is, M = 512, 16, 256, 128, 2
    g = torch.Generator(device=DEV).manual_seed(1)
    layers = []
    for i in range(3):
        proj = (0.05 * torch.randn((H, H), generator=g, device=DEV)).to(BF)
        layers.append((torch.ones(H, device=DEV, dtype=BF), proj, torch.ones(H, device=DEV, dtype=BF), make(M, E, H, I, Is, BF, fp8=i == 1, seed=i)))

    def step(x):
        for n1, proj, n2, d in layers:
            x = fg.fused_linear(fg.rms_norm(x, n1), proj, activation="gelu", residual=x)
            y = fg.rms_norm(x, n2)
            rest = {k: d[k] for k in ("w1_scale", "w2_scale", "shared_w1", "shared_w2", "shared_w1_scale", "shared_w2_scale")}
            x = fg.fused_moe_few_tokens(y, d["router"], d["w1"], d["w2"], 4, scoring="sigmoid", e_score_correction_bias=d["bias"], residual=x, **rest)
        return x

    x = torch.randn((M, H), generator=g, device=DEV).to(BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph, buf = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = step(buf)
    eager = x
    for _ in range(4):
        graph.replay()
        eager = step(eager)
        assert torch.equal(out, eager) and torch.isfinite(out).all()
        buf.copy_(out)
    assert fg.read_status() == 0


def test_training_step_of_a_shared_expert_beside_the_router():
    """Norm, shared expert, balance loss: gradients through all of them against torch's.  Sums of up to n = 512 products in fp32 are
    off by n 2^-23 of their absolute sum, which is about sqrt(n) = 22 times a typical one: 2^-9.5 of the largest."""
    M, H, I, E = 100, 256, 128, 16
    g = torch.Generator(device=DEV).manual_seed(2)
    leaves = [torch.randn(s, generator=g, device=DEV) * f for s, f in (((M, H), 1.0), ((H,), 1.0), ((2 * I, H), 0.06), ((H, I), 0.09), ((E, H), 0.06), ((E,), 1.0))]

    def own(x, gamma, w1, w2, router, b):
        y = fg.rms_norm(x, gamma)
        out = fg.fused_linear(fg.fused_linear(y, w1, activation="silu_and_mul"), w2, residual=x)
        logits = fg.fused_linear(y, router, b)
        loss, _ = fg.moe_balance_loss(logits, logits.topk(2).indices)
        return out.square().mean() + loss

    def plain(x, gamma, w1, w2, router, b):
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gamma
        a, u = (y @ w1.t()).chunk(2, -1)
        out = (torch.nn.functional.silu(a) * u) @ w2.t() + x
        logits = y @ router.t() + b
        p = logits.softmax(-1)
        counts = torch.bincount(logits.topk(2).indices.flatten(), minlength=E)
        return out.square().mean() + (counts * p.mean(0)).sum() * E / (2 * M)

    a = [t.clone().requires_grad_() for t in leaves]
    b = [t.double().requires_grad_() for t in leaves]
    for p, q in zip(torch.autograd.grad(own(*a), a), torch.autograd.grad(plain(*b), b)):
        assert (p.double() - q).abs().max() <= 2.0**-9.5 * q.abs().max()


@pytest.mark.parametrize("dtype,fp8", [(BF, False), (BF, True)])
def test_more_work_than_one_run_for_a_block(dtype, fp8):
    """8.4 million outputs of W1: more than a block takes at once, more groups of 128 than its list holds."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("not enough free memory")
    check(make(1, 8, 128 if fp8 else 64, 1 << 20, 0, dtype, fp8), 8)


PROGRAM = """
import torch
import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib

g = torch.Generator(device="cuda").manual_seed(0)
rand = lambda *s: (0.1 * torch.randn(s, generator=g, device="cuda")).bfloat16()
x, w, router, w1, w2 = rand(3, 256), rand(64, 256), rand(16, 256), rand(16, 256, 256), rand(16, 256, 128)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph), torch.no_grad():
    y = fg.fused_linear(x, w, activation="silu")
    out = fg.fused_moe_few_tokens(x, router, w1, w2, 4)
    z = fg.fused_linear(out.float(), w.float())
assert _lib.read_status() == 0
graph.replay()
held = [t.clone() for t in (y, out, z)]
with torch.no_grad():
    want = [fg.fused_linear(x, w, activation="silu"), fg.fused_moe_few_tokens(x, router, w1, w2, 4)]
    want.append(fg.fused_linear(want[1].float(), w.float()))
assert all(torch.equal(a, b) for a, b in zip(held, want)) and _lib.read_status() == 0
print("done")
"""


def test_a_first_call_that_is_captured():
    run = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "done" in run.stdout, run.stderr[-2000:]
