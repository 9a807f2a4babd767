"""rms_norm, fused_add_rms_norm and rms_norm_quant against plain implementations in 64 bits.

Tolerances are counted, not tuned.  With n additions in a row, a sum of squares is off by n 2^-24 of itself, its root by half
of that; each fp32 product, quotient or root adds 2^-24, and the rounding to the output type half a step of it."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32 = 2.0 ** -24
EPS = 1e-6


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance of subnormals: what a rounding loses at least."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def adds(cols):
    """Additions behind one another in a row's sum: a thread's own, its warp's, the warps of the block."""
    return cols // 256 + 32 + 5 + 32


def make(M, H, dtype, residual=True, weight_dtype=None, seed=0, gap=0, offset=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def rows(scale):
        flat = torch.randn((M * (H + gap) + offset,), generator=g, device=DEV) * scale
        return flat.to(dtype)[offset:].view(M, H + gap)[:, :H]

    w = (1.0 + 0.5 * torch.randn((H,), generator=g, device=DEV)).to(weight_dtype or dtype)
    return rows(1.0), (rows(3.0) if residual else None), w, g


def plain(x, w, residual, eps=EPS):
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    hd = h.double()
    inv = 1.0 / (hd.square().mean(-1, keepdim=True) + eps).sqrt()
    return hd * inv * w.double(), h, inv


def check_norm(y, want, cols, dtype):
    tol = want.abs() * (half_step(dtype) + (adds(cols) / 2 + 6) * F32) + smallest(dtype)
    assert ((y.double() - want).abs() <= tol).all()


ROWS = [1, 2, 5, 37, 300]
COLS = [1, 7, 8, 33, 64, 100, 128, 256, 1000, 1023, 1024, 1032, 1999, 2048, 2056, 4096, 4104, 5001, 7168, 8191, 8192, 8200, 16384,
        16392, 20001, 20480, 33000]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_of_every_row_length(cols, dtype):
    for M in (1, 37):
        for residual in (False, True):
            for wt in {dtype, torch.float32}:
                x, r, w, _ = make(M, cols, dtype, residual, wt, seed=cols)
                want, h, _ = plain(x, w, r)
                out = fg.rms_norm(x, w, EPS, r)
                y, got_h = out if residual else (out, None)
                assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
                check_norm(y, want, cols, dtype)
                if residual:
                    assert torch.equal(got_h, h)


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("gap,offset", [(0, 0), (8, 0), (1, 0), (0, 1), (64, 8), (3, 5)])
def test_rows_in_wider_buffers_and_at_odd_addresses(M, gap, offset):
    for cols, dtype in ((768, torch.bfloat16), (2048, torch.float16), (516, torch.float32), (333, torch.bfloat16)):
        x, r, w, _ = make(M, cols, dtype, gap=gap, offset=offset, seed=M)
        want, h, _ = plain(x, w, r)
        y, got = fg.rms_norm(x, w, EPS, r)
        assert torch.equal(got, h)
        check_norm(y, want, cols, dtype)


def test_layouts_that_are_copied_first():
    x, r, w, _ = make(24, 128, torch.bfloat16)
    want, h, _ = plain(x, w, r)
    y3, h3 = fg.rms_norm(x.view(2, 3, 4, 128), w, EPS, r.view(2, 3, 4, 128))
    assert y3.shape == (2, 3, 4, 128) and torch.equal(h3.view(24, 128), h)
    check_norm(y3.view(24, 128), want, 128, torch.bfloat16)
    yt = fg.rms_norm(x.t().contiguous().t(), w, EPS)  # columns apart
    assert torch.equal(yt, fg.rms_norm(x, w, EPS))
    one = x[:1].expand(24, 128)                       # the same row for all
    assert torch.equal(fg.rms_norm(one, w, EPS), fg.rms_norm(one.contiguous(), w, EPS))
    wide = torch.stack([w, w], 1).flatten()[::2]      # a weight with a stride
    assert torch.equal(fg.rms_norm(x, wide, EPS), fg.rms_norm(x, w, EPS))
    assert torch.equal(fg.rms_norm(x[0], w, EPS), fg.rms_norm(x, w, EPS)[0])  # one dimension


def test_no_rows():
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    x = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16)
    y, h = fg.rms_norm(x, w, EPS, x)
    assert y.shape == h.shape == (0, 64)
    q, s = fg.rms_norm_quant(x, w, group_size=32, column_major_scales=True)
    assert q.shape == (0, 64) and s.shape == (0, 2)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(fg.rms_norm(xg, wg), (xg, wg), x)
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("cols", [64, 1023, 2048, 7168, 16392])
def test_bad_values_stay_in_their_row(cols):
    for dtype in (torch.bfloat16, torch.float32):
        x, r, w, _ = make(6, cols, dtype, seed=1)
        x[1, cols // 2] = float("nan")
        x[3, 0] = float("inf")
        x[4] = 0.0
        r[4] = 0.0
        want, h, _ = plain(x, w, r)
        y, got = fg.rms_norm(x, w, EPS, r)
        assert torch.equal(got.isnan(), h.isnan()) and torch.equal(got[[0, 2, 4, 5]], h[[0, 2, 4, 5]])
        check_norm(y[[0, 2, 4, 5]], want[[0, 2, 4, 5]], cols, dtype)
        assert torch.equal(y.isnan(), want.isnan())  # inf / inf is no number, the rest of its row is zero
        assert (y[4] == 0).all() and (y[3, 1:] == 0).all() and y[1].isnan().all()
        q, s, _ = fg.rms_norm_quant(x, w, EPS, r)
        assert s[1].isnan().all() and s[3].isnan().all() and torch.isfinite(s[[0, 2, 4, 5]]).all()
        assert (q[4].float() == 0).all() and s[4].item() == pytest.approx(1e-10 / 448, rel=1e-6)


def test_in_place():
    for cols, dtype, gap in ((64, torch.bfloat16, 0), (7168, torch.bfloat16, 0), (2048, torch.float16, 16), (1023, torch.float32, 3),
                             (16392, torch.bfloat16, 0), (20001, torch.float32, 1),
                             (33000, torch.bfloat16, 0)):
        for M in (1, 5, 200):
            bx = torch.randn(M, cols + gap, device=DEV).to(dtype)
            br = torch.randn(M, cols + gap, device=DEV).to(dtype)
            w = torch.randn(cols, device=DEV).to(dtype)
            x, r = bx[:, :cols], br[:, :cols]
            y, h = fg.rms_norm(x, w, EPS, r)
            keep = bx[:, cols:].clone(), br[:, cols:].clone()
            versions = bx._version, br._version
            got = fg.fused_add_rms_norm(x, r, w, EPS)
            assert got[0] is x and got[1] is r
            assert torch.equal(x, y) and torch.equal(r, h)
            assert torch.equal(bx[:, cols:], keep[0]) and torch.equal(br[:, cols:], keep[1])
            assert bx._version > versions[0] and br._version > versions[1]


def test_in_place_in_two_windows_of_one_buffer():
    for H in (64, 65):
        both = torch.randn(8, 2 * H + 6, device=DEV).bfloat16()
        w = torch.randn(H, device=DEV).bfloat16()
        x, r, rest = both[:, :H], both[:, H + 6:], both[:, H:H + 6].clone()
        y, h = fg.rms_norm(x, w, EPS, r)
        fg.fused_add_rms_norm(x, r, w, EPS)
        assert torch.equal(x, y) and torch.equal(r, h) and torch.equal(both[:, H:H + 6], rest)
        y, h = fg.rms_norm(r, w, EPS, x)
        fg.fused_add_rms_norm(r, x, w, EPS)
        assert torch.equal(r, y) and torch.equal(x, h)


def test_in_place_refusals():
    x, r, w, _ = make(8, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="share no memory"):
        fg.fused_add_rms_norm(x, x, w)
    buf = torch.zeros(9, 64, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share no memory"):
        fg.fused_add_rms_norm(buf[:8], buf[1:], w)
    with pytest.raises(ValueError, match="share no memory"):
        fg.fused_add_rms_norm(x[:1].expand(8, 64), r, w)  # every row is the same memory
    with pytest.raises(ValueError, match="share no memory"):
        fg.fused_add_rms_norm(x, r, x[3])
    with pytest.raises(ValueError, match="share no memory"):
        fg.fused_add_rms_norm(x, r, r[0])
    both = torch.randn(8, 130, device=DEV).bfloat16()
    with pytest.raises(ValueError, match="share no memory"):
        fg.fused_add_rms_norm(both[:, :66], both[:, 64:], torch.ones(66, device=DEV).bfloat16())
    with pytest.raises(ValueError, match="rows of contiguous elements"):
        fg.fused_add_rms_norm(x.t().contiguous().t(), r, w)
    with pytest.raises(RuntimeError, match="no gradient"):
        fg.fused_add_rms_norm(x, r, w.clone().requires_grad_())
    with torch.no_grad():
        fg.fused_add_rms_norm(x, r, w.clone().requires_grad_())


# ---- gradients -------------------------------------------------------------------------------------------------------


def check_grads(x, r, w, dy, dh, dx, dw, eps=EPS):
    """Against the formula in 64 bits; the bounds are those of its terms."""
    M, H = x.shape
    _, h, inv = plain(x, w, r, eps)
    hd, wd, dyd = h.double(), w.double(), dy.double()
    mean = (wd * dyd * hd).mean(-1, keepdim=True)
    want = inv * (wd * dyd - hd * inv * inv * mean)
    n = adds(H)
    slack = (inv * wd * dyd).abs() * (n / 2 + 6) + (hd * inv ** 3 * mean).abs() * (1.5 * n + 12)
    slack = slack + (hd * inv ** 3).abs() * (wd * dyd * hd).abs().mean(-1, keepdim=True) * (n + 3)
    if dh is not None:
        want = want + dh.double()
        slack = slack + want.abs() + dh.double().abs()
    if dx is not None:
        tol = want.abs() * half_step(x.dtype) + slack * F32 + smallest(x.dtype)
        assert ((dx.double() - want).abs() <= tol).all()
    if dw is not None:
        terms = dyd * hd * inv
        sms = torch.cuda.get_device_properties(x.device).multi_processor_count
        behind = M // sms + 64  # a block's rows, its warps, the blocks' sums
        tol = terms.sum(0).abs() * half_step(w.dtype) + terms.abs().sum(0) * (behind + n / 2 + 8) * F32 + smallest(w.dtype)
        assert ((dw.double() - terms.sum(0)).abs() <= tol).all()


@pytest.mark.parametrize("cols", [1, 7, 64, 100, 128, 1000, 1023, 1024, 1032, 1999, 2048, 2056, 4096, 4104, 7168, 8200, 16384, 16392,
                                  20001, 20480, 33000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradients(cols, dtype):
    for M in (1, 3, 333):
        for residual in (False, True):
            for wt in {dtype, torch.float32}:
                x, r, w, g = make(M, cols, dtype, residual, wt, seed=M + cols)
                dy = torch.randn((M, cols), generator=g, device=DEV).to(dtype)
                dh = torch.randn((M, cols), generator=g, device=DEV).to(dtype) if residual else None
                leaves = [t.clone().requires_grad_() for t in (x, w, r) if t is not None]
                out = fg.rms_norm(leaves[0], leaves[1], EPS, leaves[2] if residual else None)
                outs, gs = (list(out), [dy, dh]) if residual else ([out], [dy])
                grads = torch.autograd.grad(outs, leaves, gs)
                check_grads(x, r, w, dy, dh, grads[0], grads[1])
                if residual:
                    assert torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("M", [1, 296, 297, 2000])
def test_gradient_rows_are_dealt_out_whole(M):
    for cols, dtype in ((64, torch.bfloat16), (1024, torch.float32), (4096, torch.float16), (777, torch.bfloat16)):
        x, r, w, g = make(M, cols, dtype, seed=3)
        dy = torch.randn((M, cols), generator=g, device=DEV).to(dtype)
        xl, wl, rl = (t.clone().requires_grad_() for t in (x, w, r))
        y, _ = fg.rms_norm(xl, wl, EPS, rl)
        one = torch.autograd.grad(y, (xl, wl, rl), dy, retain_graph=True)
        check_grads(x, r, w, dy, None, one[0], one[1])
        two = torch.autograd.grad(y, (xl, wl, rl), dy)
        assert all(torch.equal(a, b) for a, b in zip(one, two))  # the order of the sums is fixed


def test_gradient_against_differences():
    torch.manual_seed(0)
    x, r, w, g = make(9, 200, torch.float32, seed=5)
    dy, dh = torch.randn_like(x), torch.randn_like(x)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    grads = torch.autograd.grad(list(fg.rms_norm(leaves[0], leaves[1], EPS, leaves[2])), leaves, [dy, dh])

    def value(x, w, r):  # without the rounding of the stream, which has no derivative
        h = x + r
        y = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        return (y * dy.double()).sum() + (h * dh.double()).sum()

    step = 1e-4
    for i in range(3):
        at = [t.double() for t in (x, w, r)]
        direction = torch.randn_like(at[i])
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - step * direction, at[i] + step * direction
        want = (value(*hi) - value(*lo)) / (2 * step)
        got = (grads[i].double() * direction).sum()
        # third derivatives times step^2; the stream's rounding shifts h by 2^-24 of itself; the gradient's own roundings
        tol = (grads[i].double() * direction).abs().sum() * (adds(200) + 40) * F32 + 20 * step ** 2 * direction.norm() * dy.norm()
        assert abs(got - want) <= tol


def test_gradient_of_one_output_and_of_some_inputs():
    x, r, w, g = make(40, 512, torch.bfloat16)
    dy = torch.randn((40, 512), generator=g, device=DEV).bfloat16()
    xl, wl, rl = (t.clone().requires_grad_() for t in (x, w, r))
    y, h = fg.rms_norm(xl, wl, EPS, rl)
    only_h = torch.autograd.grad(h, (xl, wl, rl), dy, retain_graph=True)
    assert torch.equal(only_h[0], dy) and torch.equal(only_h[2], dy) and torch.equal(only_h[1], torch.zeros_like(w))
    (dw,) = torch.autograd.grad(y, (wl,), dy, retain_graph=True)
    check_grads(x, r, w, dy, None, None, dw)
    (dr,) = torch.autograd.grad(y, (rl,), dy)
    check_grads(x, r, w, dy, None, dr, None)
    y, h = fg.rms_norm(x, w, EPS, rl)  # only the residual wants one
    (dr2,) = torch.autograd.grad(y, (rl,), dy)
    assert torch.equal(dr, dr2)


def test_gradient_of_shared_and_broadcast_inputs():
    x, _, w, g = make(16, 256, torch.float32, residual=False)
    dy = torch.randn((16, 256), generator=g, device=DEV)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, _ = fg.rms_norm(xl, wl, EPS, xl)  # x is its own residual: h = 2 x
    (dx,) = torch.autograd.grad(y, (xl,), dy)
    a, b, c = (t.clone().requires_grad_() for t in (x, x, w))
    da, db = torch.autograd.grad(fg.rms_norm(a, c, EPS, b)[0], (a, b), dy)
    assert torch.equal(dx, da + db)
    row = x[:1].clone().requires_grad_()
    (drow,) = torch.autograd.grad(fg.rms_norm(row.expand(16, 256), wl, EPS), (row,), dy)
    full = x[:1].expand(16, 256).contiguous().requires_grad_()
    (dfull,) = torch.autograd.grad(fg.rms_norm(full, wl, EPS), (full,), dy)
    assert torch.allclose(drow, dfull.sum(0, keepdim=True), rtol=0, atol=16 * F32 * float(dfull.abs().sum(0).max()))
    # a gradient that is one number for all
    (ds,) = torch.autograd.grad(fg.rms_norm(xl, wl, EPS).sum(), (xl,))
    check_grads(x, None, w, torch.ones_like(x), None, ds, None)


def test_leaves_accumulate():
    x, r, w, g = make(8, 128, torch.float32)
    xl, wl, rl = (t.clone().requires_grad_() for t in (x, w, r))
    for _ in range(2):
        y, h = fg.rms_norm(xl, wl, EPS, rl)
        (y.sum() + h.sum()).backward()
    dx, dw, dr = torch.autograd.grad([t.sum() for t in fg.rms_norm(xl, wl, EPS, rl)], (xl, wl, rl))
    for leaf, d in ((xl, dx), (wl, dw), (rl, dr)):
        assert torch.equal(leaf.grad, d + d)
    xl.grad.zero_()
    assert torch.equal(rl.grad, dr + dr)  # the two share no memory


def test_second_derivative_is_refused_where_it_is_asked_for():
    x, _, w, _ = make(4, 64, torch.float32, residual=False)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    (dx,) = torch.autograd.grad(fg.rms_norm(xl, wl).square().sum(), (xl,), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


def test_a_changed_stream_is_noticed():
    x, r, w, _ = make(4, 64, torch.float32)
    y, h = fg.rms_norm(x.clone().requires_grad_(), w, EPS, r)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- 8 bits ----------------------------------------------------------------------------------------------------------

QMAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0, torch.int8: 127.0}


def check_quant(q, s, want, group, dtype, quant_eps, ue8m0, cols):
    M = want.shape[0]
    blocks = want.view(M, -1, group)
    delta = (adds(cols) / 2 + 10) * F32
    raw = blocks.abs().amax(-1).clamp(min=quant_eps) / QMAX[dtype]
    if ue8m0:
        raw = raw.clamp(min=1e-10)
        assert (torch.frexp(s)[0] == 0.5).all()
        assert (s.double() >= raw * (1 - delta)).all() and (s.double() / 2 < raw * (1 + delta)).all()
    else:
        assert ((s.double() - raw).abs() <= raw * delta).all()
    sd = s.double().unsqueeze(-1)
    back = (q.to(torch.float64) if dtype == torch.int8 else q.float().double()).view(M, -1, group) * sd
    if dtype == torch.int8:
        tol = sd * (0.5 + 127 * 2 * delta)
    else:
        # half a step relative to the value, half a step of the subnormals below
        step, sub = (2.0 ** -4, 2.0 ** -10) if dtype == torch.float8_e4m3fn else (2.0 ** -3, 2.0 ** -17)
        tol = torch.maximum(blocks.abs() * step, sd * sub) + blocks.abs() * 2 * delta
    assert ((back - blocks).abs() <= tol + 1e-300).all()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.int8])
@pytest.mark.parametrize("cols,groups", [(128, (None, 128, 64, 8)), (512, (None, 256, 512, 1)), (1000, (None, 8, 40, 125)),
                                         (2048, (None, 128)), (7168, (None, 128, 64)), (16384, (None, 128)), (16896, (None, 128, 96)), (1032, (None, 8, 24)), (5000, (None, 8)), (1040, (None, 16)), (20480, (None, 128)), (33024, (None, 128)),
                                         (777, (None, 7))])
def test_quant(dtype, cols, groups):
    for in_dtype in (torch.bfloat16, torch.float32):
        for M in (1, 50):
            x, r, w, _ = make(M, cols, in_dtype, seed=cols)
            want, h, _ = plain(x, w, r)
            for group in groups:
                for ue8m0 in (False, True) if dtype != torch.int8 else (False,):
                    q, s, got_h, got_y = fg.rms_norm_quant(x, w, EPS, r, group_size=group, dtype=dtype, scale_ue8m0=ue8m0,
                                                           return_norm=True)
                    assert q.dtype == dtype and s.dtype == torch.float32 and s.shape == (M, cols // (group or cols))
                    assert torch.equal(got_h, h)
                    check_norm(got_y, want, cols, in_dtype)  # a group that no warp holds is normed by another kernel: other sums
                    check_quant(q, s, want, group or cols, dtype, 1e-10, ue8m0, cols)


@pytest.mark.parametrize("in_dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("group", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_quant_is_the_two_steps_in_fp32(in_dtype, group, dtype):
    """Bit for bit: an fp32 norm holds the value that the 8 bits are made of."""
    x, _, w, _ = make(333, 2048, in_dtype, residual=False, weight_dtype=torch.float32)
    for cm in (False, True):
        q, s = fg.rms_norm_quant(x, w, EPS, group_size=group, dtype=dtype, column_major_scales=cm)
        y = fg.rms_norm(x.float(), w, EPS)
        q2, s2 = fg.per_token_group_quant_fp8(y, group, dtype=dtype, column_major_scales=cm)
        if in_dtype == torch.float32:
            assert torch.equal(s, s2) and s.stride() == s2.stride()
            assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
        else:  # the row's sum is added up in another order from fp16's pieces
            assert s.stride() == s2.stride() and ((s - s2).abs() <= s2 * adds(2048) * F32).all()


def test_quant_options():
    x, r, w, _ = make(6, 256, torch.bfloat16)
    a = fg.rms_norm_quant(x, w, EPS)
    assert len(a) == 2 and a[0].dtype == torch.float8_e4m3fn and a[1].shape == (6, 1)
    b = fg.rms_norm_quant(x, w, EPS, r, return_norm=True)
    assert len(b) == 4
    c = fg.rms_norm_quant(x.view(2, 3, 256), w, EPS, group_size=128)
    assert c[0].shape == (2, 3, 256) and c[1].shape == (2, 3, 2)
    d = fg.rms_norm_quant(x, w, EPS, group_size=128, column_major_scales=True)
    assert d[1].shape == (6, 2) and d[1].stride() == (1, 6) and torch.equal(d[1], c[1].view(6, 2))
    big = fg.rms_norm_quant(x, w, EPS, group_size=128, quant_eps=1e4)
    assert torch.equal(big[1], torch.full_like(big[1], 1e4) * torch.tensor(1 / 448, dtype=torch.float32, device=DEV))
    for cols in (256, 250):  # nothing to scale and no floor under it
        for dtype in QMAX:
            for group in (None, 2, cols):
                q, s = fg.rms_norm_quant(x[:, :cols] * 0, w[:cols], EPS, quant_eps=0.0, dtype=dtype, group_size=group)
                assert (s == 0).all() and (q.float() == 0).all()
    with pytest.raises(RuntimeError, match="no gradient"):
        fg.rms_norm_quant(x.clone().requires_grad_(), w)


# ---- streams, graphs, sizes ------------------------------------------------------------------------------------------


def test_captured_and_replayed():
    x, r, w, _ = make(300, 2048, torch.bfloat16)
    bx, br = x.clone(), r.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fg.rms_norm_quant(bx, w, EPS, br, group_size=128)
        fg.rms_norm(bx, w, EPS, br)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = fg.rms_norm(bx, w, EPS, br)
        q, s, h2 = fg.rms_norm_quant(bx, w, EPS, br, group_size=128)
        fg.fused_add_rms_norm(bx, br, w, EPS)
    for seed in (1, 2):
        nx, nr, _, _ = make(300, 2048, torch.bfloat16, seed=seed)
        bx.copy_(nx)
        br.copy_(nr)
        graph.replay()
        wy, wh = fg.rms_norm(nx, w, EPS, nr)
        wq = fg.rms_norm_quant(nx, w, EPS, nr, group_size=128)
        assert torch.equal(y, wy) and torch.equal(h, wh) and torch.equal(h2, wh)
        assert torch.equal(q.view(torch.uint8), wq[0].view(torch.uint8)) and torch.equal(s, wq[1])
        assert torch.equal(bx, wy) and torch.equal(br, wh)


def test_training_step_captured_and_replayed():
    def step(x, r, w, dy, dh):
        return torch.autograd.grad(list(fg.rms_norm(x, w, EPS, r)), (x, w, r), (dy, dh))

    x, r, w, g = make(500, 1024, torch.float16, weight_dtype=torch.float32)
    for t in (x, r, w):
        t.requires_grad_()
    dy = torch.randn((500, 1024), generator=g, device=DEV).half()
    dh = torch.randn((500, 1024), generator=g, device=DEV).half()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, r, w, dy, dh)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, r, w, dy, dh)
    for seed in (1, 2):
        nx, nr, _, _ = make(500, 1024, torch.float16, seed=seed)
        with torch.no_grad():
            x.copy_(nx)
            r.copy_(nr)
        graph.replay()
        held = [t.clone() for t in got]
        want = step(x, r, w, dy, dh)
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_two_streams_at_once():
    sets = [make(700, 4096, torch.bfloat16, seed=i) for i in range(2)]
    want = [fg.rms_norm(x, w, EPS, r) for x, r, w, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, (x, r, w, _) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(fg.rms_norm(x, w, EPS, r))
    torch.cuda.synchronize()
    for i in range(2):
        for y, h in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(h, want[i][1])


def test_offsets_beyond_32_bits():
    """Rows that begin more than 2^31 elements into their buffer."""
    ld = 1 << 28
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("not enough free memory")
    buf = torch.empty(9 * ld, dtype=torch.bfloat16, device=DEV).view(9, ld)
    x = buf[:, 128:128 + 512]
    x.copy_(torch.randn(9, 512, device=DEV))
    w = torch.ones(512, device=DEV, dtype=torch.bfloat16)
    dense = x.contiguous()
    assert torch.equal(fg.rms_norm(x, w), fg.rms_norm(dense, w))
    xl, dl = x.requires_grad_(), dense.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fg.rms_norm(xl, w).sum(), xl)[0], torch.autograd.grad(fg.rms_norm(dl, w).sum(), dl)[0])


def test_many_rows():
    x, r, w, _ = make(200_003, 64, torch.bfloat16)
    want, h, _ = plain(x, w, r)
    y, got = fg.rms_norm(x, w, EPS, r)
    assert torch.equal(got, h)
    check_norm(y, want, 64, torch.bfloat16)


def test_launches_are_counted():
    x, r, w, _ = make(4, 64, torch.bfloat16)
    before = _lib.LAUNCHES
    fg.rms_norm(x, w, EPS, r)
    assert _lib.LAUNCHES == before + 1
