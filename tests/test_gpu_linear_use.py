"""fused_linear in use: graphs, streams, threads, differentiation, guard bands, long offsets, bad values."""

import ctypes
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwad
import torch.utils.checkpoint

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib
from test_gpu_linear import ACTS, TINY, _act64, make, reference
from test_gpu_norm_balance_autograd import hooks
from test_gpu_norm_balance_bounds import CODE, Guarded, stream

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
NUMBER = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "silu_and_mul": 5}


def leaves_of(*ts):
    return [t.detach().clone().requires_grad_() for t in ts if t is not None]


def grads(leaves, act, dy, bias=True, residual=True):
    x, w = leaves[:2]
    b = leaves[2] if bias else None
    r = leaves[-1] if residual else None
    y = fg.fused_linear(x, w, b, act, r)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


# ------------------------------------------------------------------ differences
@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh", "silu_and_mul"])
@pytest.mark.parametrize("which", ["x", "w", "b", "r"])
def test_gradient_against_differences(act, which):
    """Central differences along a direction v, in fp32: step h = 2^-6; operands are multiples of 2^-8 below 4 and v of 2^-4, so
    that x + h v is exact.  Off by the third derivative (at most 1 for every activation; the gate's product: |g'|^3 |u| + 3 g'^2 |u'|),
    h^2 / 6 of it, by the value's bound over h, and by the gradient's own bound."""
    M, K, N = 9, 20, 12
    g = torch.Generator(device=DEV).manual_seed(3)
    W = 2 * N if act == "silu_and_mul" else N

    def grid(*s, by=8, std=1.0):
        return (std * torch.randn(s, generator=g, device=DEV) * 2**by).round().clamp(-(4 * 2**by), 4 * 2**by) / 2**by

    t = {"x": grid(M, K), "w": grid(W, K, std=0.25), "b": grid(W), "r": grid(M, N)}
    dy, v, h = grid(M, N), grid(*t[which].shape, by=4), 2.0**-6
    leaves = leaves_of(*t.values())
    y = fg.fused_linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
    got = dict(zip(t, torch.autograd.grad(y, leaves, dy)))[which].double()
    value = {}
    for s in (1, -1):
        m = dict(t)
        m[which] = t[which] + s * h * v
        value[s] = (fg.fused_linear(m["x"], m["w"], m["b"], act, m["r"]).double() * dy.double()).sum()
    want, bound = reference(t["x"], t["w"], t["b"], t["r"], act, dy)
    own = (bound["d" + which] * v.double().abs()).sum()
    c, X, Wt, V = dy.double().abs(), t["x"].double(), t["w"].double(), v.double()
    d = {"x": V @ Wt.t() if which == "x" else None, "w": X @ V.t() if which == "w" else None, "b": V.expand(M, W) if which == "b" else None}.get(which)
    third = 0.0
    if d is not None and act == "silu_and_mul":
        z = X @ Wt.t() + t["b"].double()
        third = (c * (d[:, :N].abs() ** 3 * (z[:, N:].abs() + h * d[:, N:].abs()) + 3 * d[:, :N] ** 2 * d[:, N:].abs())).sum()
    elif d is not None and act is not None:
        third = (c * d.abs() ** 3).sum()
    off = ((value[1] - value[-1]) / (2 * h) - (got * v.double()).sum()).abs()
    # the value's bound where the operand has been moved: its terms grow by at most the same again
    assert off <= h * h / 6 * third + 2 * (c * bound["y"]).sum() / h + own


# ------------------------------------------------------------------ graphs, streams, threads
@pytest.mark.parametrize("dtype,M,K,N", [(BF, 300, 520, 96), (HF, 17, 1024, 64), (BF, 2304, 512, 1024), (F32, 130, 200, 72), (BF, 40, 333, 65)])
def test_training_step_captured_and_replayed(dtype, M, K, N):
    act = "silu_and_mul"
    sets = [make(M, K, N, dtype, act, "f32", True, seed=s) for s in range(3)]
    dy = torch.randn(M, N, device=DEV).to(dtype)
    leaves = leaves_of(*sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(leaves, act, dy)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same step, replayed in turn
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(grads(leaves, act, dy))
    for s in (1, 2):
        with torch.no_grad():
            for leaf, new in zip(leaves, sets[s]):
                leaf.copy_(new)
        want = grads(leaves_of(*sets[s]), act, dy)
        for graph, out in zip(graphs, outs):
            for t in out[:-1]:
                t.zero_()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert fg.read_status() == 0


def test_two_streams_at_once():
    sets = [make(200 + 300 * i, 1024, 520, BF, "gelu", "same", seed=i) for i in range(2)]
    small = [make(3, 4096, 1024, HF, "silu_and_mul", seed=i) for i in range(2)]  # K over a cluster
    run = lambda i: (fg.fused_linear(*sets[i][:3], "gelu"), fg.fused_linear(small[i][0], small[i][1], None, "silu_and_mul"))  # noqa: E731
    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for pair in got[i] for a, b in zip(pair, want[i]))


def test_threads_beside_one_another():
    work = [(make(100 + 90 * i, 256 * (i + 1), 128 + 8 * i, (BF, HF, F32, BF)[i], ACTS[2 + i], "same", True, seed=i)) for i in range(4)]
    dys = [torch.randn_like(w[3]) for w in work]
    want = [grads(leaves_of(*work[i]), ACTS[2 + i], dys[i]) for i in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def body(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = grads(leaves_of(*work[i]), ACTS[2 + i], dys[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------ the rest of torch's differentiation
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("mode", ["plain", "no_grad", "strided"])
def test_forward_mode_is_refused(which, mode):
    args = make(5, 24, 16, F32, None, "same", True)
    with fwad.dual_level(), torch.set_grad_enabled(mode != "no_grad"):
        duals = list(args)
        if mode == "strided":
            duals[which] = torch.stack([duals[which]] * 2, -1)[..., 0]
        duals[which] = fwad.make_dual(duals[which], torch.ones_like(duals[which]))
        with pytest.raises(RuntimeError, match="forward mode"):
            fg.fused_linear(duals[0], duals[1], duals[2], None, duals[3])


def test_second_derivative_is_refused_where_it_is_asked_for():
    x, w, b, r = leaves_of(*make(5, 24, 16, F32, "silu", "same", True))
    y = fg.fused_linear(x, w, b, "silu", r)
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


@pytest.mark.parametrize("act", [None, "gelu", "silu_and_mul"])
@pytest.mark.parametrize("change", [lambda t: t.cpu().cuda(), lambda t: torch.stack([t, t], -1)[..., 0], lambda t: t.clone(),
                                    lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)], ids=["moved", "strided", "copied", "odd address"])
def test_saved_tensors_in_another_layout(act, change):
    for dtype in (BF, F32):
        args = make(33, 72, 40, dtype, act, "same")
        dy = torch.randn(33, 40, device=DEV).to(dtype)
        want = grads(leaves_of(*args), act, dy, residual=False)
        leaves = leaves_of(*args)
        with hooks(change):
            y = fg.fused_linear(*leaves, act)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want[1:]))


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t[:-1], lambda t: torch.cat([t, t]), lambda t: t.to(torch.float64), lambda t: t[..., :-1]],
                         ids=["on the host", "shorter", "longer", "another type", "narrower"])
def test_saved_tensors_that_changed_are_refused(which, change):
    leaves = leaves_of(*make(33, 72, 40, BF, "silu", "same"))
    with hooks(change, which):
        y = fg.fused_linear(*leaves, "silu")
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, torch.ones_like(y))


def test_gradients_of_some_inputs():
    """Each of the sixteen sets of inputs that want one gets the bits that all together get."""
    args = make(70, 96, 48, BF, "gelu_tanh", "f32", True)
    dy = torch.randn(70, 48, device=DEV).to(BF)
    want = grads(leaves_of(*args), "gelu_tanh", dy)[1:]
    for mask in range(1, 16):
        ts = [t.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args)]
        y = fg.fused_linear(ts[0], ts[1], ts[2], "gelu_tanh", ts[3])
        y.backward(dy)
        for i in range(4):
            assert (ts[i].grad is None) if not mask >> i & 1 else torch.equal(ts[i].grad, want[i])


def test_gradients_of_shared_and_broadcast_inputs():
    """A tensor that is two operands, operands broadcast from fewer elements, leaves that accumulate: torch's own sums of the same parts."""
    x, _, _, _ = make(48, 48, 48, F32)
    dy = torch.randn(48, 48, device=DEV)
    parts = grads(leaves_of(x, x, x), None, dy, bias=False)[1:]
    (t,) = leaves_of(x)
    (g,) = torch.autograd.grad(fg.fused_linear(t, t, None, None, t), t, dy)
    torch.testing.assert_close(g, sum(parts), rtol=0, atol=float(3 * 2.0**-23 * sum(p.abs().max() for p in parts)))
    row, one = leaves_of(x[:1], x[0, :1])
    y = fg.fused_linear(row.expand(48, 48), x, one.expand(48), "silu", row.expand(48, 48))
    wide = leaves_of(x[:1].expand(48, 48), x[0, :1].expand(48), x[:1].expand(48, 48))
    gx, gb, gr = torch.autograd.grad(fg.fused_linear(wide[0], x, wide[1], "silu", wide[2]), wide, dy)
    got = torch.autograd.grad(y, (row, one), dy)
    torch.testing.assert_close(got[1], gb.sum(0, keepdim=True), rtol=0, atol=float(50 * 2.0**-23 * gb.abs().sum()))
    torch.testing.assert_close(got[0], gx.sum(0, keepdim=True) + gr.sum(0, keepdim=True), rtol=0, atol=float(50 * 2.0**-23 * (gx.abs() + gr.abs()).sum(0).max()))
    (w,) = leaves_of(x)
    for _ in range(2):
        fg.fused_linear(x, w).backward(dy)
    once = torch.autograd.grad(fg.fused_linear(x, w), w, dy)[0]
    assert torch.equal(w.grad, once + once)
    # a gradient that arrives expanded, and one that arrives transposed
    (w2,) = leaves_of(x)
    fg.fused_linear(x, w2).sum().backward()
    assert torch.equal(w2.grad, torch.autograd.grad(fg.fused_linear(x, w), w, torch.ones(48, 48, device=DEV))[0])
    assert torch.equal(torch.autograd.grad(fg.fused_linear(x, w), w, dy.t())[0], torch.autograd.grad(fg.fused_linear(x, w), w, dy.t().contiguous())[0])


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint_computes_the_same_again(reentrant):
    args = make(40, 64, 64, BF, "silu_and_mul", "same", True)
    dy = torch.randn(40, 64, device=DEV).to(BF)
    want = grads(leaves_of(*args), "silu_and_mul", dy)[1:]
    x, w, b, r = leaves_of(*args)
    y = torch.utils.checkpoint.checkpoint(lambda x, w, b, r: fg.fused_linear(x, w, b, "silu_and_mul", r), x, w, b, r, use_reentrant=reentrant)
    y.backward(dy)
    assert all(torch.equal(t.grad, g) for t, g in zip((x, w, b, r), want))


def test_a_graph_that_is_kept_and_values_that_change():
    """A second backward pass through one forward; y may be changed afterwards, an operand that the gradient needs may not."""
    leaves = leaves_of(*make(33, 72, 40, BF, "silu", "same", True))
    dy = torch.randn(33, 40, device=DEV).to(BF)
    y = fg.fused_linear(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    z = y.add_(1.0)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(z, leaves, dy, retain_graph=True)))
    with torch.no_grad():
        leaves[1].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z, leaves, dy)


def test_inference_mode_and_no_grad():
    x, w, b, r = make(20, 64, 40, BF, "relu", "same", True)
    want = fg.fused_linear(x, w, b, "relu", r)
    with torch.inference_mode():
        y = fg.fused_linear(x, w.requires_grad_(), b, "relu", r)
        assert y.is_inference() and torch.equal(y, want)
    with torch.no_grad():
        assert not fg.fused_linear(x, w, b, "relu", r).requires_grad
    assert torch.equal(fg.fused_linear(x, w, b, "relu", r).detach(), want)


# ------------------------------------------------------------------ shapes and layouts
def test_no_rows():
    for dtype in (BF, F32):
        x, w, b, r = leaves_of(torch.zeros(0, 3, 64, device=DEV, dtype=dtype), torch.ones(32, 64, device=DEV, dtype=dtype),
                               torch.ones(32, device=DEV), torch.zeros(0, 3, 32, device=DEV, dtype=dtype))
        y = fg.fused_linear(x, w, b, "silu", r)
        assert y.shape == (0, 3, 32)
        got = torch.autograd.grad(y, (x, w, b, r), torch.zeros_like(y))
        assert got[0].shape == x.shape and not got[1].any() and not got[2].any() and got[3].shape == r.shape


def test_every_rank_and_stride():
    x, w, b, r = make(2 * 3 * 4, 40, 24, BF, "silu", "same", True)
    want = fg.fused_linear(x, w, b, "silu", r)
    assert torch.equal(fg.fused_linear(x.view(2, 3, 4, 40), w, b, "silu", r.view(2, 3, 4, 24)), want.view(2, 3, 4, 24))
    assert torch.equal(fg.fused_linear(x[5], w, b, "silu", r[5]), fg.fused_linear(x[5:6], w, b, "silu", r[5:6])[0])
    t = x.view(2, 3, 4, 40).transpose(0, 2)  # rows without a single distance
    assert torch.equal(fg.fused_linear(t, w, b, "silu", r.view(2, 3, 4, 24).transpose(0, 2)), want.view(2, 3, 4, 24).transpose(0, 2))
    columns = x.t().contiguous().t()  # [K, M] in memory, and weights likewise
    assert torch.equal(fg.fused_linear(columns, w.t().contiguous().t(), b, "silu", r.t().contiguous().t()), want)
    assert torch.equal(fg.fused_linear(x, w, torch.stack([b, b], 1)[:, 0], "silu", r), want)
    assert torch.equal(fg.fused_linear(x[::2], w, b, "silu", r[::2]), fg.fused_linear(x[::2].contiguous(), w, b, "silu", r[::2].contiguous()))
    one = x[:1].expand(24, 40)
    assert torch.equal(fg.fused_linear(one, w, b, "silu", r), fg.fused_linear(one.contiguous(), w, b, "silu", r))
    windows = x.view(-1)[: 20 * 40].as_strided((20, 40), (24, 1))  # rows that overlap
    assert torch.equal(fg.fused_linear(windows, w), fg.fused_linear(windows.contiguous(), w))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,K,N", [(4, 2048, 256), (100, 264, 130), (2304, 64, 1024)])
def test_bad_values_stay_in_their_row(dtype, M, K, N):
    """Inf and NaN in rows of x reach their rows of y only; in the weights, their columns only; in the gradients, the other way about."""
    x, w, b, r = make(M, K, N, dtype, "silu", "same", True)
    clean = grads(leaves_of(x, w, b, r), "silu", r)
    bad = x.clone()
    bad[1, 3], bad[M - 1, K - 1] = float("nan"), float("inf")
    got = grads(leaves_of(bad, w, b, r), "silu", r)
    rows = torch.ones(M, dtype=torch.bool, device=DEV)
    rows[1] = rows[M - 1] = False
    assert torch.equal(got[0][rows], clean[0][rows]) and torch.equal(got[1][rows], clean[1][rows]) and got[0][1].isnan().all()
    wb = w.clone()
    wb[N - 2, 5] = float("nan")
    got = grads(leaves_of(x, wb, b, r), "silu", r)
    cols = torch.ones(N, dtype=torch.bool, device=DEV)
    cols[N - 2] = False
    assert torch.equal(got[0][:, cols], clean[0][:, cols]) and got[0][:, N - 2].isnan().all()
    assert torch.equal(got[2][cols], clean[2][cols]) and torch.equal(got[3][cols], clean[3][cols]) and got[2][N - 2].isnan().all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh", "silu_and_mul"])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_extreme_sums(act, dtype):
    """Activations far out: exact zeros and identities, no NaN, infinities where the formula has them."""
    z = torch.tensor([-float("inf"), -3e4, -500.0, -90.0, -0.0, 0.0, 90.0, 500.0, 3e4, float("inf")], device=DEV, dtype=F32)
    N = z.numel()
    x, w = torch.zeros(3, 8, device=DEV, dtype=dtype), torch.zeros(2 * N if act == "silu_and_mul" else N, 8, device=DEV, dtype=dtype)
    bias = torch.cat([z, torch.ones_like(z)]) if act == "silu_and_mul" else z
    y = fg.fused_linear(x, w, bias, act).double()
    want = _act64(bias.double(), act)
    want = torch.where(z == -float("inf"), torch.zeros_like(want), want)  # the limit, where 64 bits multiply 0 by infinity
    got = torch.where(z == -float("inf"), torch.where(y.isnan(), torch.zeros_like(y), y), y)
    assert torch.equal(got.isinf(), want.to(dtype).double().expand_as(got).isinf())
    fin = want.isfinite().expand_as(got) & ~got.isinf()
    u = torch.finfo(dtype).eps / 2
    off = (got - want).abs()
    assert (off[fin] <= ((u + 2.0**-18) * want.abs() + 2.0**-20 + TINY[dtype]).expand_as(got)[fin]).all()


# ------------------------------------------------------------------ memory
@pytest.mark.parametrize("act", [None, "gelu", "silu_and_mul"])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 4096, 40), (9, 65, 33), (70, 136, 200), (300, 333, 129), (2304, 72, 1032), (2100, 64, 1025)])
def test_writes_its_outputs_only(M, K, N, dtype, act):
    x, w, b, r = make(M, K, N, dtype, act, "f32", True)
    W, s, c, lib = w.shape[0], dtype.itemsize, CODE[dtype], _lib.lib()
    dy = torch.randn(M, N, device=DEV).to(dtype)
    zt = F32 if act == "silu_and_mul" else dtype
    need, grad_need = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(lib.moe_fused_linear_workspace(x.data_ptr(), K, w.data_ptr(), K, c, M, N, K, NUMBER[act], ctypes.addressof(need)))
    _lib.check(lib.moe_fused_linear_grad_workspace(x.data_ptr(), K, w.data_ptr(), K, c, M, N, K, NUMBER[act], ctypes.addressof(grad_need)))
    ld = N + 3
    seen = []
    for fill in (0xFF, 0x5A):
        g = Guarded(fill, y=((M - 1) * ld + N) * s, z=M * W * zt.itemsize, ws=need.value, gws=grad_need.value, dx=M * K * s, dw=W * K * s, db=W * 4)
        _lib.check(lib.moe_fused_linear(x.data_ptr(), K, w.data_ptr(), K, b.data_ptr(), _lib.MOE_F32, r.data_ptr(), N, c, M, N, K, NUMBER[act], g.ptr("y"),
                                        ld, g.ptr("z"), W, g.ptr("ws"), need.value, _lib.status_word(x.device).data_ptr(), stream()))
        _lib.check(lib.moe_fused_linear_grad(dy.data_ptr(), g.ptr("z"), W, x.data_ptr(), K, w.data_ptr(), K, c, M, N, K, NUMBER[act], g.ptr("dx"), g.ptr("dw"),
                                             g.ptr("db"), _lib.MOE_F32, g.ptr("gws"), grad_need.value, _lib.status_word(x.device).data_ptr(), stream()))
        assert g.intact()
        flat = g.view("y", dtype, -1)
        y = flat.as_strided((M, N), (ld, 1)).clone()
        if M > 1:
            assert (flat.as_strided((M - 1, 3), (ld, 1), flat.storage_offset() + N).contiguous().view(torch.uint8) == fill).all()  # behind the rows
        seen.append([y] + [g.view(n, t, -1).clone() for n, t in (("dx", dtype), ("dw", dtype), ("db", F32))])
    assert all(torch.equal(p, q) for p, q in zip(*seen))
    want = grads(leaves_of(x, w, b, r), act, dy)
    assert all(torch.equal(p.flatten(), q.flatten()) for p, q in zip(seen[0], want))
    assert fg.read_status() == 0


@pytest.mark.parametrize("M", [4, 300])
def test_offsets_beyond_32_bits_of_operands(M):
    """Rows that begin more than 2^31 elements into their buffer."""
    ld = 1 << 30 if M == 4 else (1 << 32) // 299 // 64 * 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough free memory")
    buf = torch.empty(M * ld + 64, dtype=BF, device=DEV)
    x = buf[: M * ld].view(M, ld)[:, 64:64 + 512]
    x.copy_(torch.randn(M, 512, device=DEV))
    _, w, b, r = make(M, 512, 256, BF, "silu", "same", True)
    dy = torch.randn(M, 256, device=DEV).to(BF)
    far = x.detach().requires_grad_()
    got = grads([far, *leaves_of(w, b, r)], "silu", dy)
    want = grads(leaves_of(x.contiguous(), w, b, r), "silu", dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype,K", [(BF, 64), (F32, 8)])
def test_offsets_beyond_32_bits_of_results(dtype, K):
    M, N = 66_000, 33_000  # 2.2 10^9 results, more than 2^31
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("not enough free memory")
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w = (torch.randn(n, K, generator=g, device=DEV).to(dtype) for n in (M, N))
    y = fg.fused_linear(x, w, None, "relu")
    rows = torch.cat([torch.arange(0, M, 997), torch.arange(M - 300, M)]).to(DEV)
    want = torch.relu(x[rows].double() @ w.double().t())
    S = x[rows].double().abs() @ w.double().abs().t()
    bound = (K + 2) * 2.0**-23 * S + torch.finfo(dtype).eps / 2 * want + 2.0**-19
    assert ((y[rows].double() - want).abs() <= bound).all()


def test_many_rows_of_weights():
    """More tiles of rows than a grid's second dimension has."""
    for dtype, rows, K in ((BF, 65536 * 128 + 300, 8), (F32, 65536 * 128 + 300, 4)):
        g = torch.Generator(device=DEV).manual_seed(0)
        x, w = torch.randn(rows, K, generator=g, device=DEV).to(dtype), torch.randn(16, K, generator=g, device=DEV).to(dtype)
        y = fg.fused_linear(x, w)
        at = torch.cat([torch.arange(0, rows, 99_991), torch.arange(rows - 400, rows)]).to(DEV)
        want, S = x[at].double() @ w.double().t(), x[at].double().abs() @ w.double().abs().t()
        assert ((y[at].double() - want).abs() <= (K + 2) * 2.0**-23 * S + torch.finfo(dtype).eps / 2 * want.abs()).all()


def test_launches_are_counted():
    x, w, b, _ = make(4, 64, 32, BF, None, "same")
    before = _lib.LAUNCHES
    fg.fused_linear(x, w, b)
    assert _lib.LAUNCHES == before + 1
