"""Norms of rows that lie in wider buffers, with any number of dimensions in front, and weights between the rows."""

import pytest
import torch

import flaggems_vllm_b200 as fg

pytestmark = pytest.mark.gpu

DEV = "cuda"
SHAPES = [(8,), (2, 4), (2, 1, 4), (1, 8), (8, 1), (1, 2, 2, 2), (1, 1), ()]


def window(front, H, gap, dtype, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    buf = torch.randn((*front, H + gap), generator=g, device=DEV).to(dtype)
    return buf, buf[..., gap // 2:gap // 2 + H]


@pytest.mark.parametrize("front", SHAPES)
@pytest.mark.parametrize("H,gap", [(64, 16), (64, 6), (65, 3), (1, 4), (2056, 8)])
def test_windows_of_any_rank(front, H, gap):
    for dtype in (torch.bfloat16, torch.float32):
        bx, x = window(front, H, gap, dtype, 1)
        br, r = window(front, H, gap + 2, dtype, 2)
        w = torch.randn(H, device=DEV).to(dtype)
        # the same memory as a plain table of rows: the kernel, and so every bit, is the same (a copy of the rows may lie in
        # longer pieces, whose sums are joined in another order)
        fx, fr = (b.view(-1, b.shape[-1])[:, g // 2:g // 2 + H] for b, g in ((bx, gap), (br, gap + 2)))
        want = [t.view(x.shape) for t in fg.rms_norm(fx, w, 1e-6, fr)]
        h = (x.double() + r.double()).to(dtype)
        exact = h.double() / (h.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        got = fg.rms_norm(x, w, 1e-6, r)
        assert all(a.shape == x.shape and a.is_contiguous() and torch.equal(a, b) for a, b in zip(got, want))
        # a row's sum has at most H / 256 + 69 additions behind one another, its root half of their error, and six roundings follow
        tol = exact.abs() * (torch.finfo(dtype).eps / 2 + ((H // 256 + 69) / 2 + 6) * 2.0 ** -24) + 1e-38
        assert torch.equal(got[1], h) and ((got[0].double() - exact).abs() <= tol).all()
        q, s = fg.rms_norm_quant(x, w)
        q2, s2 = fg.rms_norm_quant(fx, w)
        assert torch.equal(q.view(torch.uint8).view(-1, H), q2.view(torch.uint8)) and torch.equal(s.view(-1, 1), s2) and q.shape == x.shape
        xl, wl = x.detach().requires_grad_(), w.clone().requires_grad_()
        dl, vl = fx.detach().requires_grad_(), w.clone().requires_grad_()
        for a, b in zip(torch.autograd.grad(fg.rms_norm(xl, wl).sum(), (xl, wl)), torch.autograd.grad(fg.rms_norm(dl, vl).sum(), (dl, vl))):
            assert torch.equal(a.view(b.shape), b)
        keep, dense = (bx.clone(), br.clone()), (x.detach().clone(), r.clone())
        fg.fused_add_rms_norm(x.detach(), r, w)
        assert torch.equal(x.detach(), want[0]) and torch.equal(r, want[1])
        x.detach().copy_(dense[0])
        r.copy_(dense[1])
        assert torch.equal(bx, keep[0]) and torch.equal(br, keep[1])  # what lies between the rows stays


def test_rows_without_a_single_distance():
    base = torch.randn(3, 4, 70, device=DEV)
    w = torch.randn(64, device=DEV)
    for x in (base[:, :3, :64], base[:, ::2, :64], base[::2, :, :64].transpose(0, 1), base[:, :1, :64].expand(3, 4, 64),
              base[:1, :, :64].expand(3, 4, 64)):
        keep = base.clone()
        copied = fg.rms_norm(x.contiguous(), w)
        # two orders of a sum of 64 squares: each off by its additions at most, the root by half of that
        assert ((fg.rms_norm(x, w) - copied).abs() <= copied.abs() * (69 + 6) * 2.0 ** -24).all()
        if x.stride(0) == x.shape[1] * x.stride(1) > 0:
            continue  # every other row of all: that is one distance
        with pytest.raises(ValueError, match="rows of contiguous elements"):
            fg.fused_add_rms_norm(x, torch.randn(x.shape, device=DEV), w)
        assert torch.equal(base, keep)


def test_a_weight_between_the_rows():
    for dtype, off in ((torch.bfloat16, 64), (torch.bfloat16, 70), (torch.float32, 64)):
        buf = torch.randn(4, 160, device=DEV).to(dtype)
        x, w = buf[:, :64], buf[2, off:off + 64]
        r = torch.randn(4, 64, device=DEV).to(dtype)
        want = fg.rms_norm(x, w, 1e-6, r)
        fg.fused_add_rms_norm(x, r, w)
        assert torch.equal(x, want[0]) and torch.equal(r, want[1])
        for meets in (buf[2, 63:127], buf.view(-1)[160 + 97:160 + 161], buf.view(-1)[160 + 120:160 + 184]):
            with pytest.raises(ValueError, match="share no memory"):
                fg.fused_add_rms_norm(x, r, meets)
