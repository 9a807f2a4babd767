"""What the norms and the balance loss do with the rest of torch's differentiation: forward mode is refused, not lost."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

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
