"""What the norms and the balance loss do with the rest of torch's differentiation: forward mode is refused, not lost, and hooks on
saved tensors may hand back another layout, nothing else."""

import pytest
import torch
import torch.autograd.forward_ad as fwad
import torch.utils.checkpoint

import flaggems_vllm_b200 as fg

pytestmark = pytest.mark.gpu

DEV = "cuda"


def rows(dtype=torch.float32, M=6, H=64):
    g = torch.Generator(device=DEV)
    g.manual_seed(0)
    return [torch.randn(shape, generator=g, device=DEV).to(dtype) for shape in ((M, H), (H,), (M, H))]


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("mode", ["plain", "no_grad", "strided"])
def test_forward_mode_of_the_norms_is_refused(which, mode):
    args = rows()
    with fwad.dual_level(), torch.set_grad_enabled(mode != "no_grad"):
        duals = list(args)
        if mode == "strided":
            duals[which] = torch.stack([duals[which]] * 2, -1)[..., 0]
        duals[which] = fwad.make_dual(duals[which], torch.ones_like(duals[which]))
        x, w, r = duals
        for call in (lambda: fg.rms_norm(x, w, 1e-6, r), lambda: fg.rms_norm_quant(x, w, 1e-6, r), lambda: fg.fused_add_rms_norm(x, r, w)):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
        if which < 2:
            with pytest.raises(RuntimeError, match="forward mode"):
                fg.rms_norm(x, w)
        for before, now in zip(rows(), args):
            assert torch.equal(before, now)  # nothing was written
        primal = [fwad.unpack_dual(t).primal for t in duals]
        y, h = fg.rms_norm(primal[0], primal[1], 1e-6, primal[2])  # what has no tangent is served beside it
    want = fg.rms_norm(*args[:2], 1e-6, args[2])
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])


@pytest.mark.parametrize("strided", [False, True])
def test_forward_mode_of_the_balance_loss_is_refused(strided):
    logits = torch.randn(20, 8, device=DEV)
    ids = torch.randint(0, 8, (20, 2), device=DEV)
    with fwad.dual_level():
        l = logits.t().contiguous().t() if strided else logits
        with pytest.raises(RuntimeError, match="forward mode"):
            fg.moe_balance_loss(fwad.make_dual(l, torch.ones_like(l)), ids)
        inside = fg.moe_balance_loss(logits, ids)
    assert torch.equal(inside[0], fg.moe_balance_loss(logits, ids)[0])


def hooks(change, which=None):
    """Saved tensors come back changed, all of them or the one that was saved as the `which`-th."""
    saved = []

    def pack(t):
        saved.append(t)
        return len(saved) - 1, t

    def unpack(item):
        return change(item[1]) if which is None or item[0] == which else item[1]

    return torch.autograd.graph.saved_tensors_hooks(pack, unpack)


def apart(t):
    return torch.stack([t, t], -1)[..., 0]


def norm_grads(residual=True):
    x, w, r = (t.requires_grad_() for t in rows(torch.bfloat16))
    out = fg.rms_norm(x, w, 1e-6, r if residual else None)
    leaves = (x, w, r) if residual else (x, w)
    return lambda: torch.autograd.grad([t.float().square().sum() for t in (out if residual else [out])], leaves)


def balance_grads():
    g = torch.Generator(device=DEV)
    g.manual_seed(0)
    l = torch.randn((50, 16), generator=g, device=DEV).requires_grad_()
    ids = torch.randint(0, 16, (50, 2), generator=g, device=DEV)
    cu = torch.tensor([0, 20, 45], dtype=torch.int32, device=DEV)
    loss, _ = fg.moe_balance_loss(l, ids, "softmax", cu, torch.rand((50,), generator=g, device=DEV) < 0.2)
    return lambda: torch.autograd.grad(loss, l)


@pytest.mark.parametrize("make", [norm_grads, lambda: norm_grads(False), balance_grads], ids=["norm", "norm alone", "balance"])
@pytest.mark.parametrize("change", [lambda t: t.cpu().cuda(), apart, lambda t: t.clone()], ids=["moved", "strided", "copied"])
def test_saved_tensors_in_another_layout(make, change):
    want = make()()
    with hooks(change):
        grads = make()
    assert all(torch.equal(a, b) for a, b in zip(grads(), want))


@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t[:-1], lambda t: torch.cat([t, t]), lambda t: t.to(torch.float64)],
                         ids=["on the host", "shorter", "longer", "another type"])
def test_saved_tensors_that_changed_are_refused(which, change):
    for make in (norm_grads, balance_grads):
        if make is norm_grads and which > 1:
            continue
        with hooks(change, which):
            grads = make()
        with pytest.raises((RuntimeError, ValueError)):  # a row more or less without sequences or padding is the engine's to refuse
            grads()


def test_a_stream_of_another_type_is_refused():
    with hooks(lambda t: t.float()):  # the norm's own types, but not those of the gradient that comes in
        grads = norm_grads()
    with pytest.raises(RuntimeError, match="came back"):
        grads()


def test_inference_mode():
    x, w, r = rows(torch.bfloat16)
    want = fg.rms_norm(x, w, 1e-6, r)
    with torch.inference_mode():
        y, h = fg.rms_norm(x, w.requires_grad_(), 1e-6, r)
        assert y.is_inference() and torch.equal(y, want[0]) and torch.equal(h, want[1])
        q = fg.rms_norm_quant(y, w, 1e-6, h)
        assert torch.equal(q[2], (y.float() + h.float()).bfloat16())
        bx, br = x.clone(), r.clone()
        fg.fused_add_rms_norm(bx, br, w)
        assert torch.equal(bx, y) and torch.equal(br, h)
        loss, counts = fg.moe_balance_loss(torch.zeros(4, 8, device=DEV), torch.zeros(4, 1, device=DEV, dtype=torch.int32))
        assert counts[0].item() == 4 and abs(loss.item() - 1.0) <= 64 * 2.0 ** -24
    w.requires_grad_(False)
    fg.fused_add_rms_norm(x, r, w)
    assert torch.equal(x, want[0]) and torch.equal(r, want[1])


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint_computes_the_same_again(reentrant):
    x, w, r = (t.requires_grad_() for t in rows())
    gate = torch.randn(8, 64, device=DEV, requires_grad=True)
    ids = torch.randint(0, 8, (6, 2), device=DEV)

    def block(x, w, r, gate):
        y, h = fg.rms_norm(x, w, 1e-6, r)
        loss, _ = fg.moe_balance_loss((y.unsqueeze(1) * gate).sum(-1), ids)
        return y, h, loss

    leaves = (x, w, r, gate)

    def grads(outs):
        for t in leaves:
            t.grad = None
        sum(t.square().sum() for t in outs).backward()
        return [t.grad.clone() for t in leaves]

    want = grads(block(*leaves))
    got = grads(torch.utils.checkpoint.checkpoint(block, *leaves, use_reentrant=reentrant))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
