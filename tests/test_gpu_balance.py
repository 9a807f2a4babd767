"""moe_balance_loss against its definition in 64 bits, and the run from a layer's output to the experts.

Tolerances: a score is exp2((u - max) log2 e) over its sum.  The argument is off by 3 roundings of itself, u of the sigmoid
form by some 4 of its own and 4 of one, exp2 by 2, the sum over a row and the quotient by 40 roundings at most; a mean over tokens by one
for each addition."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32 = 2.0 ** -24


def make(T, E, k, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    logits = (torch.randn((T, E), generator=g, device=DEV) * scale + 0.3 * torch.randn((E,), generator=g, device=DEV)).to(dtype)
    ids = (torch.rand((T, E), generator=g, device=DEV) + 0.1 * logits.float()).topk(k, -1).indices.int() if T else \
        torch.empty((0, k), dtype=torch.int32, device=DEV)
    return logits, ids


def definition(logits, ids, scoring, cu=None, pad=None, dloss=1.0):
    """loss, counts [S, E], dlogits, and the bound of each element's fp32 error in dlogits and of the loss."""
    T, E = logits.shape
    k = ids.shape[1]
    edges = [0, T] if cu is None else cu.tolist()
    l = logits.detach().double()
    counts = torch.zeros((len(edges) - 1, E), dtype=torch.int64, device=DEV)
    dlogits, slack = torch.zeros_like(l), torch.zeros_like(l)
    parts = []
    for s, (a, b) in enumerate(zip(edges[:-1], edges[1:])):
        rows = torch.arange(a, b, device=DEV)
        if pad is not None:
            rows = rows[~pad[a:b]]
        if rows.numel():
            parts.append((s, rows))
    loss, off = 0.0, 0.0
    for s, rows in parts:
        part = l[rows]
        u = part if scoring == "softmax" else torch.nn.functional.logsigmoid(part)
        dead = (u == -float("inf")).all(-1, keepdim=True)
        p = torch.where(dead, 0.0, torch.softmax(u, -1))
        flat = ids[rows].long().flatten()
        counts[s] = torch.bincount(flat[(flat >= 0) & (flat < E)], minlength=E)
        n = rows.numel()
        f = E * counts[s].double() / (k * n)
        one = (f * p.mean(0)).sum()
        loss += one.item() / len(parts)
        a = dloss * f / (n * len(parts))
        d = p * (a - (p * a).sum(-1, keepdim=True))
        size = p * (a.abs() + (p * a.abs()).sum(-1, keepdim=True) + dloss / (n * len(parts)))
        if scoring == "sigmoid":
            d, size = d * torch.sigmoid(-part), size * torch.sigmoid(-part)
        finite = torch.where(u.isfinite(), u, 0.0)
        # arguments beyond 160 give scores below the smallest number: their error is that number, not a share of themselves
        reach = (finite.amax(-1, keepdim=True) - finite).clamp(max=160.0) * 3 + (0 if scoring == "softmax" else finite.abs().clamp(max=160.0) * 4)
        rel = (reach.amax(-1, keepdim=True) * 1.5 + 64) * F32
        dlogits[rows], slack[rows] = d, size * 3 * rel
        off += float((f * (p * rel).mean(0)).sum()) / len(parts) + one.item() * 256 * F32 / len(parts)
    return loss, counts if cu is not None else counts[0], dlogits, slack, off


def check(logits, ids, scoring, cu=None, pad=None, dloss=1.0):
    want, counts, dwant, slack, off = definition(logits, ids, scoring, cu, pad, dloss)
    leaf = logits.detach().clone().as_strided(logits.size(), logits.stride()) if logits.is_contiguous() else logits.detach()
    leaf.requires_grad_()
    loss, got = fg.moe_balance_loss(leaf, ids, scoring, cu, pad)
    assert loss.dtype == torch.float32 and loss.shape == () and got.dtype == torch.int32
    assert torch.equal(got.long(), counts)
    assert abs(loss.item() - want) <= off + 1e-30
    (d,) = torch.autograd.grad(loss, leaf, torch.tensor(dloss, device=DEV))
    assert d.dtype == logits.dtype and d.shape == logits.shape
    info = torch.finfo(logits.dtype)
    tol = dwant.abs() * info.eps / 2 + slack + info.smallest_normal * info.eps / 2
    assert ((d.double() - dwant).abs() <= tol).all()
    with torch.no_grad():
        plain, same = fg.moe_balance_loss(logits, ids, scoring, cu, pad)
    assert torch.equal(plain, loss.detach()) and torch.equal(same, got)
    return loss, got, d


@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (3, 2), (8, 2), (60, 4), (64, 6), (100, 8), (128, 8), (160, 6), (256, 8), (257, 8),
                                 (384, 8), (511, 4), (512, 10), (516, 4), (520, 4), (1000, 8), (1023, 7), (1024, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_every_number_of_experts(E, k, scoring):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for T in (1, 3, 130, 1111):
            logits, ids = make(T, E, k, dtype, seed=T)
            check(logits, ids, scoring, dloss=float(T))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_sequences(scoring):
    T, E, k = 700, 64, 6
    logits, ids = make(T, E, k)
    for edges in ([0, 700], [0, 0, 1, 3, 3, 300, 699], [5, 40, 40, 41, 600], [0] * 6 + [700], [0, 0], [700, 700], [350, 350, 350],
                  list(range(0, 701, 1)), list(range(0, 701, 7))):
        cu = torch.tensor(edges, dtype=torch.int32, device=DEV)
        loss, counts, d = check(logits, ids, scoring, cu)
        assert not d[:edges[0]].any() and not d[edges[-1]:].any()
        if edges[0] == edges[-1]:
            assert loss.item() == 0.0 and not counts.any()
    assert _lib.read_status() == 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [33, 5000])
def test_padding_holds_anything(scoring, T):
    E, k = 128, 8
    logits, ids = make(T, E, k)
    pad = torch.rand(T, device=DEV) < 0.4
    cu = torch.tensor([0, T // 3, T // 3, T - 2], dtype=torch.int32, device=DEV)
    pad[: T // 3] = True  # a sequence of nothing else
    clean = check(logits, ids, scoring, cu, pad)
    for value in (float("nan"), float("inf"), -float("inf")):
        dirty = logits.clone()
        dirty[pad] = value
        dirty[T - 2:] = value  # behind the last sequence
        bad = ids.clone()
        bad[pad] = -1
        loss, counts, d = check(dirty, bad, scoring, cu, pad)
        assert torch.equal(loss, clean[0]) and torch.equal(counts, clean[1]) and torch.equal(d, clean[2])
    everything = torch.ones(T, dtype=torch.bool, device=DEV)
    loss, counts, d = check(logits, ids, scoring, None, everything)
    assert loss.item() == 0.0 and not counts.any() and not d.any()


@pytest.mark.parametrize("E", [8, 100, 256])
def test_masked_experts_and_extreme_logits(E):
    T, k = 50, 2
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        low = torch.finfo(dtype).min
        for scoring in ("softmax", "sigmoid"):
            for mask in (-float("inf"), low):
                logits, ids = make(T, E, k, dtype)
                logits[:, E // 2:] = mask            # experts that nobody may use
                logits[7] = mask                     # a row that may use none
                check(logits, ids, scoring)
            logits, ids = make(T, E, k, dtype)
            logits[3] = -200.0                       # every sigmoid underflows in fp32, their shares do not
            logits[4] = 200.0
            logits[5, 1] = 300.0
            check(logits, ids, scoring)
        logits, ids = make(T, E, k, dtype)
        logits[9, 2] = float("nan")
        leaf = logits.clone().requires_grad_()
        loss, counts = fg.moe_balance_loss(leaf, ids)
        (d,) = torch.autograd.grad(loss, leaf)
        assert loss.isnan() and d[9].isnan().all()
        assert d[[i for i in range(T) if i != 9]].isfinite().all()
        logits[9] = float("nan")                     # a row of nothing else
        assert fg.moe_balance_loss(logits, ids)[0].isnan()
        assert fg.moe_balance_loss(logits, ids, "sigmoid")[0].isnan()


def test_ids_of_every_kind():
    T, E, k = 300, 32, 4
    logits, ids = make(T, E, k)
    base = check(logits, ids, "softmax")
    for other in (ids.long(), ids.view(torch.uint32), torch.cat([ids, ids], 1)[:, :k]):
        loss, counts = fg.moe_balance_loss(logits, other)
        assert torch.equal(loss, base[0].detach()) and torch.equal(counts, base[1])
    same = ids.clone()
    same[:] = ids[:, :1]  # the same expert in every place counts every time
    check(logits, same, "softmax")
    none = torch.full_like(ids, -1)
    loss, counts, d = check(logits, none, "softmax")
    assert loss.item() == 0.0 and not counts.any()
    assert _lib.read_status() == 0
    bad = ids.clone()
    bad[5, 2], bad[6, 0] = E, 1 << 30
    check(logits, bad, "softmax")
    assert _lib.read_status() == _lib.ST_BAD_EXPERT_ID
    wide = ids.long()
    wide[0, 0] = 1 << 40
    check(logits, wide, "softmax")
    assert _lib.read_status() == _lib.ST_BAD_EXPERT_ID


def test_sequences_out_of_order_are_reported():
    logits, ids = make(64, 16, 2)
    for edges in ([0, 40, 30, 64], [0, 65], [-1, 64], [0, 1 << 30], [64, 0]):
        cu = torch.tensor(edges, dtype=torch.int32, device=DEV)
        leaf = logits.clone().requires_grad_()
        loss, counts = fg.moe_balance_loss(leaf, ids, "softmax", cu)
        (d,) = torch.autograd.grad(loss, leaf)
        assert loss.isnan() and not counts.any() and d.shape == logits.shape
        assert _lib.read_status() == _lib.ST_BAD_ROW


def test_layouts():
    T, E, k = 200, 64, 4
    logits, ids = make(T, E, k)
    base = fg.moe_balance_loss(logits, ids)
    wide = torch.zeros(T, E + 3, device=DEV)
    wide[:, :E] = logits
    check(wide[:, :E], ids, "softmax")            # rows apart, not in 16-byte pieces
    wide = torch.zeros(T, E + 4, device=DEV)
    wide[:, 4:] = logits
    strided = wide[:, 4:]
    check(strided, ids, "sigmoid")
    for other in (logits.t().contiguous().t(), torch.stack([logits, logits], 1)[:, 0]):
        loss, counts = fg.moe_balance_loss(other, ids)
        assert torch.equal(loss, base[0]) and torch.equal(counts, base[1])
    one = logits[:1].expand(T, E)
    loss, _ = fg.moe_balance_loss(one, ids)
    assert torch.equal(loss, fg.moe_balance_loss(one.contiguous(), ids)[0])
    leaf = logits[:1].clone().requires_grad_()
    (d,) = torch.autograd.grad(fg.moe_balance_loss(leaf.expand(T, E), ids)[0], leaf)
    full = one.contiguous().requires_grad_()
    (dfull,) = torch.autograd.grad(fg.moe_balance_loss(full, ids)[0], full)
    assert torch.allclose(d, dfull.sum(0, keepdim=True), rtol=0, atol=T * F32 * float(dfull.abs().sum(0).max()))


def test_no_tokens():
    logits, ids = make(0, 16, 2)
    leaf = logits.requires_grad_()
    loss, counts = fg.moe_balance_loss(leaf, ids)
    assert loss.item() == 0.0 and counts.shape == (16,) and not counts.any()
    assert torch.autograd.grad(loss, leaf)[0].shape == (0, 16)
    loss, counts = fg.moe_balance_loss(logits.detach(), ids, "sigmoid", torch.zeros(4, dtype=torch.int32, device=DEV))
    assert loss.item() == 0.0 and counts.shape == (3, 16) and not counts.any()


def test_even_use_is_one():
    E, k = 16, 4
    ids = torch.stack([torch.arange(4 * i, 4 * i + 4) % E for i in range(64)]).int().to(DEV)
    for scoring in ("softmax", "sigmoid"):
        loss, counts = fg.moe_balance_loss(torch.zeros(64, E, device=DEV), ids, scoring)
        assert abs(loss.item() - 1.0) <= 64 * F32 and torch.equal(counts, torch.full_like(counts, 16))
        leaf = torch.randn(64, E, device=DEV, requires_grad=True)
        (d,) = torch.autograd.grad(fg.moe_balance_loss(leaf, ids, scoring)[0], leaf)
        assert not d.any()  # what is left of equal counts is exactly zero


def test_gradient_against_differences():
    for scoring in ("softmax", "sigmoid"):
        logits, ids = make(40, 24, 3, seed=4)
        leaf = logits.clone().requires_grad_()
        (d,) = torch.autograd.grad(fg.moe_balance_loss(leaf, ids, scoring)[0], leaf)
        direction = torch.randn(40, 24, device=DEV, dtype=torch.float64)
        step = 1e-4
        hi = definition(logits.double() + step * direction, ids, scoring)[0]
        lo = definition(logits.double() - step * direction, ids, scoring)[0]
        # third derivatives of a mean of 40 rows' scores, at most 24 / 3 times 6 per row, times step^2
        tol = (d.double() * direction).abs().sum().item() * 512 * F32 + 48 * step ** 2 * direction.abs().max().item() ** 3
        assert abs((hi - lo) / (2 * step) - (d.double() * direction).sum().item()) <= tol


def test_large_and_repeatable():
    for T, E, k, dtype in ((65536, 256, 8, torch.float32), (70001, 8, 2, torch.float32), (30011, 160, 6, torch.bfloat16)):
        logits, ids = make(T, E, k, dtype)
        one = check(logits, ids, "softmax", dloss=float(T))
        two = check(logits, ids, "softmax", dloss=float(T))
        assert all(torch.equal(a, b) for a, b in zip(one, two))
    T, E, k = 20000, 64, 6
    logits, ids = make(T, E, k)
    cu = torch.sort(torch.randint(0, T + 1, (4001,), device=DEV)).values.int()
    check(logits, ids, "sigmoid", cu, torch.rand(T, device=DEV) < 0.2)


def test_offsets_beyond_32_bits():
    """Rows that begin more than 2^31 elements into their buffer."""
    ld, E = 1 << 28, 96
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("not enough free memory")
    buf = torch.empty(9 * ld, dtype=torch.bfloat16, device=DEV).view(9, ld)
    logits, ids = make(9, E, 4, torch.bfloat16)
    far = buf[:, 64:64 + E]
    far.copy_(logits)
    for scoring in ("softmax", "sigmoid"):
        near = check(logits, ids, scoring)
        leaf = far.detach().requires_grad_()
        loss, counts = fg.moe_balance_loss(leaf, ids, scoring)
        assert torch.equal(loss, near[0]) and torch.equal(counts, near[1])
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], near[2])


def test_counts_are_the_callers():
    logits, ids = make(100, 16, 2)
    leaf = logits.clone().requires_grad_()
    loss, counts = fg.moe_balance_loss(leaf, ids)
    want = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
    assert not counts.requires_grad
    counts.zero_()  # as an all-reduce over ranks might write it
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)


def test_second_derivative_is_refused_where_it_is_asked_for():
    logits, ids = make(10, 16, 2)
    leaf = logits.clone().requires_grad_()
    (d,) = torch.autograd.grad(fg.moe_balance_loss(leaf, ids)[0], leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.square().sum().backward()


def test_captured_and_replayed_twice_over():
    T, E, k = 3000, 128, 8
    logits, ids = make(T, E, k)
    cu = torch.tensor([0, 100, 2000, 3000], dtype=torch.int32, device=DEV)
    leaf = logits.clone().requires_grad_()

    def step():
        loss, counts = fg.moe_balance_loss(leaf, ids, "sigmoid", cu)
        return loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of one pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            out = step()
        graphs.append((graph, out))
    for seed in (1, 2):
        nl, ni = make(T, E, k, seed=seed)
        with torch.no_grad():
            leaf.copy_(nl)
            ids.copy_(ni)
        want = [t.clone() for t in step()]
        for graph, out in graphs:
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    sets = [make(9000, 256, 8, seed=i) for i in range(2)]
    want = [fg.moe_balance_loss(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(fg.moe_balance_loss(*s))
    torch.cuda.synchronize()
    for i in range(2):
        for loss, counts in got[i]:
            assert torch.equal(loss, want[i][0]) and torch.equal(counts, want[i][1])


# ---- together --------------------------------------------------------------------------------------------------------


def test_a_serving_step_from_norm_to_experts():
    from oracle import moe_oracle as O
    from flaggems_vllm_b200 import testing as TT

    M, E, H, I, k = 96, 32, 512, 256, 8
    x, residual = TT.make_activations(M, H, DEV, seed=1), TT.make_activations(M, H, DEV, seed=2)
    gate = TT.make_half_weights(1, E, H, DEV, seed=3)[0]
    w1, s1 = TT.make_fp8_block_weights(E, 2 * I, H, DEV, seed=4)
    w2, s2 = TT.make_fp8_block_weights(E, H, I, DEV, seed=5)
    weight = torch.rand(H, device=DEV).bfloat16() + 0.5
    bias = 0.1 * torch.randn(E, device=DEV)
    bx, br = x.clone(), residual.clone()

    def step():
        fg.fused_add_rms_norm(bx, br, weight)
        logits = fg.router_gemm(bx, gate)
        tw, ti = fg.grouped_topk(logits, 4, 2, k, True, 2.5, bias, 1)
        loss, counts = fg.moe_balance_loss(logits, ti, "sigmoid")
        out = fg.fused_experts_impl(bx, w1, w2, tw, ti, use_fp8_w8a8=True, w1_scale=s1, w2_scale=s2, block_shape=[128, 128])
        return logits, ti, tw, loss, counts, out

    logits, ti, tw, loss, counts, out = step()
    y, h = fg.rms_norm(x, weight, residual=residual)
    assert torch.equal(bx, y) and torch.equal(br, h)
    assert torch.equal(counts, torch.bincount(ti.flatten().long(), minlength=E).int())
    want = definition(logits, ti, "sigmoid")
    assert abs(loss.item() - want[0]) <= want[4]
    ref = O.fused_moe_fp8_block_oracle(y, w1, w2, s1, s2, tw, ti)
    assert O.rel_l2(out.float(), ref) <= 1e-2
    # the same step as a graph
    bx.copy_(x)
    br.copy_(residual)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    bx.copy_(x)
    br.copy_(residual)
    graph.replay()
    for a, b in zip(got, (logits, ti, tw, loss, counts, out)):
        assert torch.equal(a, b)
    assert _lib.read_status() == 0


def test_a_training_step_of_a_router():
    """Norm, gate, choice and loss, with gradients down to the stream, the norm's weight and the gate."""
    M, E, H, k = 200, 16, 256, 4
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    x, residual = (torch.randn((M, H), generator=g, device=DEV) for _ in range(2))
    weight = 1.0 + 0.1 * torch.randn((H,), generator=g, device=DEV)
    gate = torch.randn((E, H), generator=g, device=DEV) / H ** 0.5
    leaves = [t.clone().requires_grad_() for t in (x, residual, weight, gate)]
    y, h = fg.rms_norm(leaves[0], leaves[2], 1e-6, leaves[1])
    logits = (y.unsqueeze(1) * leaves[3]).sum(-1)  # fp32, whatever the settings of library products
    tw, ti, rows = (torch.empty((M, k), device=DEV, dtype=t) for t in (torch.float32, torch.int32, torch.int32))
    fg.topk_softmax(tw, ti, rows, logits.detach(), True)
    loss, counts = fg.moe_balance_loss(logits, ti)
    grads = torch.autograd.grad(100.0 * loss + h.square().mean(), leaves)

    xd, rd, wd, gd = (t.double().requires_grad_() for t in (x, residual, weight, gate))
    hd = xd + rd
    ld = (hd / (hd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wd) @ gd.t()
    f = E * counts.double() / (k * M)
    want = torch.autograd.grad(100.0 * (f * torch.softmax(ld, -1).mean(0)).sum() + hd.square().mean(), (xd, rd, wd, gd))
    for a, b in zip(grads, want):
        # every step is fp32: some hundred roundings of sums of H or M terms, relative to the largest entries
        assert (a.double() - b).abs().max() <= 2000 * F32 * b.abs().max()
