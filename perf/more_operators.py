"""Performance cases of the dense products around the experts, and of the whole layer for a few tokens.

Two operators, each in a plain form (elementary torch operations in 32 bits) and, where ``own`` is true, through the calls
that a user makes:

``linear``  ``fused_linear``: matrix product with bias, activation and residual in its epilogue, as the shared expert beside
            the routed ones, a dense layer between layers of experts and the projections need it; with gradients where
            the case trains.
``few``     ``fused_moe_few_tokens``: router, routed experts, shared expert and residual of one layer for the tokens of a
            decode step or of one speculative draft.

Experts, hidden sizes, weight formats and value distributions are those of ``bench.py`` and ``perf/cases.py``: activations
~N(0, 1), weights ~N(0, 0.02), routing bias ~N(0, 0.1)."""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_FP8 = torch.float8_e4m3fn
_FP8_MAX, _FP8_EPS = 448.0, 1e-10

# experts, experts per token, hidden size, intermediate size; scoring and groups of the router; the factor of its weights
_SHAPES = {
    "dsv3": {"E": 256, "topk": 8, "H": 7168, "I": 2048, "scoring": "sigmoid", "groups": 8, "kept": 4, "scaling": 2.5},
    "mixtral": {"E": 8, "topk": 2, "H": 4096, "I": 14336, "scoring": "softmax", "groups": 1, "kept": 1, "scaling": 1.0},
    "qwen3": {"E": 128, "topk": 8, "H": 2048, "I": 768, "scoring": "softmax", "groups": 1, "kept": 1, "scaling": 1.0},
    "small": {"E": 8, "topk": 2, "H": 1024, "I": 2048, "scoring": "softmax", "groups": 1, "kept": 1, "scaling": 1.0},
    "odd": {"E": 60, "topk": 4, "H": 1408, "I": 704, "scoring": "sigmoid", "groups": 3, "kept": 2, "scaling": 1.0},
}


def _linear(tokens, k, n, act="none", dtype="bf16", bias=False, residual=False, train=False, gap=0):
    """n: columns of the result; a gated activation has twice as many rows of weights."""
    return {"op": "linear", "tokens": tokens, "k": k, "n": n, "act": act, "dtype": dtype, "bias": bias, "residual": residual,
            "train": train, "gap": gap}


def _few(shape, tokens, fmt="half", dtype="bf16", shared=0, residual=False, topk=0):
    """shared: intermediate size of the shared expert, 0 for none; topk: experts per token, 0 for the shape's own."""
    return {"op": "few", "shape": shape, "tokens": tokens, "format": fmt, "dtype": dtype, "shared": shared, "residual": residual,
            "topk": topk or _SHAPES[shape]["topk"]}


def listed():
    return [
        # gate and up projection of a shared expert, one sequence being decoded
        {"name": "linear_up_decode_1", **_linear(1, 7168, 2048, "silu_and_mul")},
        # down projection of a dense layer onto the residual stream, a decode batch
        {"name": "linear_down_decode_33", **_linear(33, 14336, 4096, residual=True)},
        # a short prompt through sizes that no vector width divides
        {"name": "linear_odd_501", **_linear(501, 1023, 767, "gelu", "f16", bias=True)},
        # gate and up projection of a dense layer, a prefill chunk
        {"name": "linear_up_prefill_4096", **_linear(4096, 4096, 14336, "silu_and_mul")},
        # one micro-batch of training, forward and backward: a dense layer's first product
        {"name": "linear_train_4096", **_linear(4096, 2048, 4096, "gelu_tanh", bias=True, train=True)},
        # the shared expert's gate and up projection in training
        {"name": "linear_train_gated_8192", **_linear(8192, 2048, 768, "silu_and_mul", "f16", train=True)},
        # 32 bits, as a probe's head or a test of gradients has it
        {"name": "linear_train_f32_300", **_linear(300, 501, 333, "relu", "f32", bias=True, residual=True, train=True)},
        # one sequence being decoded, experts in 8 bits with block scales, a shared expert beside them
        {"name": "few_dsv3_fp8_1", **_few("dsv3", 1, "fp8_block", shared=2048, residual=True)},
        # a small decode batch of the same
        {"name": "few_dsv3_fp8_6", **_few("dsv3", 6, "fp8_block", shared=2048)},
        # few large experts
        {"name": "few_mixtral_bf16_2", **_few("mixtral", 2)},
        # many small experts: latency and launches
        {"name": "few_qwen3_bf16_1", **_few("qwen3", 1, residual=True)},
        # a draft of eight tokens
        {"name": "few_qwen3_f16_8", **_few("qwen3", 8, dtype="f16", shared=768)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.4:
        shape = rng.choice(("dsv3", "mixtral", "qwen3", "small", "odd"))
        return _few(shape, rng.randint(1, 8), "fp8_block" if shape == "dsv3" else "half",
                    "bf16" if shape == "dsv3" else rng.choice(("bf16", "f16")),
                    shared=rng.choice((0, 128 * rng.randint(1, 20), 128 * rng.randint(1, 20))), residual=rng.random() < 0.5,
                    topk=rng.choice((0, rng.randint(1, 8))))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f16", "f16", "f32"))
    most = 2048 if dtype == "f32" else 8192
    size = lambda: rng.choice((_log_int(rng, 16, most), 8 * _log_int(rng, 2, most // 8), rng.choice((1024, 2048, 4096, most))))  # noqa: E731
    k, n, train = size(), size(), rng.random() < 0.4
    act = rng.choice(("none", "none", "relu", "silu", "gelu", "gelu_tanh", "silu_and_mul", "silu_and_mul"))
    # no more than the largest listed case multiplies
    room = (1 << 31 if dtype == "f32" else 1 << 38) // (k * n * (3 if train else 1) * (2 if act == "silu_and_mul" else 1))
    return _linear(_log_int(rng, 1, max(1, min(8192, room))), k, n, act, dtype, rng.random() < 0.5, rng.random() < 0.5, train,
                   rng.choice((0, 0, 8, 1)))


def _prepare_linear(case, g):
    M, K, N, dtype = case["tokens"], case["k"], case["n"], _DTYPES[case["dtype"]]
    dev, rows = g.device, case["n"] * (2 if case["act"] == "silu_and_mul" else 1)
    s = {"case": case, "x": torch.randn((M, K + case["gap"]), generator=g, device=dev).to(dtype)[:, :K],
         "weight": (0.02 * torch.randn((rows, K), generator=g, device=dev)).to(dtype), "bias": None, "residual": None}
    if case["bias"]:
        s["bias"] = (0.1 * torch.randn((rows,), generator=g, device=dev)).to(dtype)
    if case["residual"]:
        s["residual"] = torch.randn((M, N), generator=g, device=dev).to(dtype)
    if case["train"]:
        s["dy"] = torch.randn((M, N), generator=g, device=dev).to(dtype)
        s["leaves"] = [t for t in (s["x"], s["weight"], s["bias"], s["residual"]) if t is not None]
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


def _expert_weights(case, experts, n, k, g):
    """(weights [experts, n, k], their scales or None), a few experts at a time."""
    fp8 = case["format"] == "fp8_block"
    w = torch.empty((experts, n, k), dtype=_FP8 if fp8 else _DTYPES[case["dtype"]], device=g.device)
    scale = torch.empty((experts, n // 128, k // 128), device=g.device) if fp8 else None
    step = max(1, (1 << 28) // (n * k))
    for e in range(0, experts, step):
        part = 0.02 * torch.randn((min(step, experts - e), n, k), generator=g, device=g.device)
        if fp8:
            blocks = part.view(-1, n // 128, 128, k // 128, 128)
            scale[e:e + step] = blocks.abs().amax((2, 4)).clamp(min=_FP8_EPS) / _FP8_MAX
            part = blocks.div_(scale[e:e + step, :, None, :, None]).clamp_(-_FP8_MAX, _FP8_MAX).view_as(part)
        w[e:e + step] = part.to(w.dtype)
    return w, scale


def _prepare_few(case, g):
    c, M, dtype, dev = _SHAPES[case["shape"]], case["tokens"], _DTYPES[case["dtype"]], g.device
    E, H, I = c["E"], c["H"], c["I"]
    s = {"case": case, "x": torch.randn((M, H), generator=g, device=dev).to(dtype),
         "router": (0.02 * torch.randn((E, H), generator=g, device=dev)).to(dtype),
         "bias": 0.1 * torch.randn((E,), generator=g, device=dev) if c["scoring"] == "sigmoid" else None,
         "residual": torch.randn((M, H), generator=g, device=dev).to(dtype) if case["residual"] else None}
    s["w1"], s["s1"] = _expert_weights(case, E, 2 * I, H, g)
    s["w2"], s["s2"] = _expert_weights(case, E, H, I, g)
    s["shared_w1"] = s["shared_s1"] = s["shared_w2"] = s["shared_s2"] = None
    if case["shared"]:
        w1, s1 = _expert_weights(case, 1, 2 * case["shared"], H, g)
        w2, s2 = _expert_weights(case, 1, H, case["shared"], g)
        s["shared_w1"], s["shared_w2"] = w1[0], w2[0]
        if s1 is not None:
            s["shared_s1"], s["shared_s2"] = s1[0], s2[0]
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return _prepare_few(case, g) if case["op"] == "few" else _prepare_linear(case, g)


# ---- the framework's calls -------------------------------------------------------------------------------------------


def _own_linear(s):
    import flaggems_vllm_b200 as fg

    act = s["case"]["act"]
    y = fg.fused_linear(s["x"], s["weight"], s["bias"], None if act == "none" else act, s["residual"])
    if not s["case"]["train"]:
        return {"y": y}
    return {"y": y, "grads": list(torch.autograd.grad(y, s["leaves"], s["dy"]))}


def _own_few(s):
    import flaggems_vllm_b200 as fg

    c = _SHAPES[s["case"]["shape"]]
    out, weights, ids = fg.fused_moe_few_tokens(
        s["x"], s["router"], s["w1"], s["w2"], s["case"]["topk"], renormalize=True, scoring=c["scoring"], num_expert_group=c["groups"],
        topk_group=c["kept"], routed_scaling_factor=c["scaling"], e_score_correction_bias=s["bias"], w1_scale=s["s1"],
        w2_scale=s["s2"], shared_w1=s["shared_w1"], shared_w2=s["shared_w2"], shared_w1_scale=s["shared_s1"],
        shared_w2_scale=s["shared_s2"], residual=s["residual"], return_routing=True)
    return {"out": out, "weights": weights, "ids": ids}


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _act(z, act):
    """The activation of z and, as a function of the gradient of its result, the gradient of z; both in z's type."""
    if act == "none":
        return z, lambda d: d
    if act == "relu":
        return z.clamp(min=0.0), lambda d: d * (z > 0)
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, lambda d: d * (sig * (1.0 + z * (1.0 - sig)))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, lambda d: d * (cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), lambda d: d * (0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z))
    gate, up = z.chunk(2, -1)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    return gate * sig * up, lambda d: torch.cat([d * up * (sig * (1.0 + gate * (1.0 - sig))), d * (gate * sig)], -1)


def _plain_linear(s):
    c, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, back = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if c["train"]:
        dz = back(s["dy"].float())
        out["grads"] = [(dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
        if s["bias"] is not None:
            out["grads"].append(dz.sum(0, dtype=torch.float64).to(dtype))
        if s["residual"] is not None:
            out["grads"].append(s["dy"])
    return out


def _plain_route(s):
    """(weights fp32 [M, topk], ids [M, topk]) of the tokens; ties go to the lowest index."""
    c = _SHAPES[s["case"]["shape"]]
    logits = (s["x"].float() @ s["router"].float().t()).double()
    M, E = logits.shape
    if c["scoring"] == "sigmoid":
        u = 1.0 / (1.0 + torch.exp(-logits))
    else:
        u = torch.exp(logits - logits.amax(-1, keepdim=True))
        u = u / u.sum(-1, keepdim=True)
    u = u.float()
    rank = u if s["bias"] is None else u + s["bias"]
    if c["groups"] > 1:
        best = rank.view(M, c["groups"], -1).sort(-1, descending=True).values[..., :2].sum(-1)
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, best.sort(dim=-1, descending=True, stable=True).indices[:, :c["kept"]], True)
        rank = torch.where(keep[:, :, None], rank.view(M, c["groups"], -1), float("-inf")).view(M, E)
    ids = rank.sort(dim=-1, descending=True, stable=True).indices[:, :s["case"]["topk"]]
    w = u.gather(1, ids)
    return w / (w.sum(-1, keepdim=True) + 1e-20) * c["scaling"], ids


def _plain_quantised(v):
    """v as groups of 128 in e4m3 hold it."""
    groups = v.view(v.shape[0], -1, 128)
    scale = groups.abs().amax(-1, keepdim=True).clamp(min=_FP8_EPS) * (1.0 / _FP8_MAX)
    return ((groups / scale).clamp(-_FP8_MAX, _FP8_MAX).to(_FP8).float() * scale).view_as(v)


def _widened(w, scale):
    if scale is None:
        return w.float()
    n, k = w.shape[-2:]
    return (w.float().view(-1, n // 128, 128, k // 128, 128) * scale.view(-1, n // 128, 1, k // 128, 1)).view(w.shape)


def _rows(w, ids):
    """w[ids]; 8-bit floats are picked as bytes."""
    return None if w is None else w.view(torch.uint8)[ids].view(w.dtype) if w.dtype == _FP8 else w[ids]


def _plain_expert(x, w1, s1, w2, s2, dtype):
    """silu(gate) * up through the down projection; w1 [n, 2I, H] takes row i of x [n, H]."""
    if s1 is not None:
        x = _plain_quantised(x)
    gate, up = torch.bmm(_widened(w1, s1), x.unsqueeze(-1)).squeeze(-1).chunk(2, -1)
    h = gate / (1.0 + torch.exp(-gate)) * up
    if s2 is not None:
        h = _plain_quantised(h.to(dtype).float())  # 8 bits are made of what the activations' type holds
    return torch.bmm(_widened(w2, s2), h.unsqueeze(-1)).squeeze(-1)


def _plain_few(s):
    x, dtype = s["x"].float(), s["x"].dtype
    M, H = x.shape
    weights, ids = _plain_route(s)
    flat = ids.flatten()
    y = _plain_expert(x.repeat_interleave(ids.shape[1], 0), _rows(s["w1"], flat), _rows(s["s1"], flat), _rows(s["w2"], flat),
                      _rows(s["s2"], flat), dtype)
    out = (y.view(M, -1, H) * weights[..., None]).sum(1)
    if s["shared_w1"] is not None:
        each = [None if t is None else t[None].expand(M, *t.shape) for t in (s["shared_w1"], s["shared_s1"], s["shared_w2"], s["shared_s2"])]
        out = out + _plain_expert(x, each[0], None if each[1] is None else each[1].reshape(M, -1), each[2],
                                  None if each[3] is None else each[3].reshape(M, -1), dtype)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return {"out": out.to(dtype), "weights": weights, "ids": ids.int()}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "few": _own_few}[op](state)
    with torch.no_grad():
        return {"linear": _plain_linear, "few": _plain_few}[op](state)


# ---- in 64 bits, from the definitions --------------------------------------------------------------------------------


def _exact_linear(case, s):
    leaf = {n: s[n].detach().double().requires_grad_(case["train"]) for n in ("x", "weight", "bias", "residual") if s[n] is not None}
    z = torch.nn.functional.linear(leaf["x"], leaf["weight"], leaf.get("bias"))
    act, F = case["act"], torch.nn.functional
    if act == "silu_and_mul":
        half = z.shape[-1] // 2
        y = F.silu(z[:, :half]) * z[:, half:]
    else:
        y = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
             "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[act](z)
    if "residual" in leaf:
        y = y + leaf["residual"]
    out = {"y": y.detach()}
    if case["train"]:
        out["grads"] = list(torch.autograd.grad(y, list(leaf.values()), s["dy"].double()))
    return out


def _exact_few(case, s):
    c = _SHAPES[case["shape"]]
    E, k, per = c["E"], case["topk"], c["E"] // c["groups"]
    fp8 = case["format"] == "fp8_block"

    def held(v):  # in groups of 128, in 8 bits: scale and quotient are 32-bit numbers, as per_token_group_quant_fp8 defines them
        if not fp8:
            return v
        scale = v.unflatten(-1, (-1, 128)).abs().amax(-1).float().clamp(min=_FP8_EPS).mul(torch.tensor(1.0 / _FP8_MAX, device=v.device))
        scale = scale.repeat_interleave(128, -1)
        return (v.float() / scale).clamp(-_FP8_MAX, _FP8_MAX).to(_FP8).double() * scale.double()

    def matrix(w, scale):
        w = w.double()
        return w if scale is None else w * scale.double().repeat_interleave(128, 0).repeat_interleave(128, 1)

    def expert(v, w1, s1, w2, s2):
        gate, up = (matrix(w1, s1) @ held(v)).tensor_split(2)
        h = torch.nn.functional.silu(gate) * up
        if fp8:
            h = held(h.to(s["x"].dtype).double())
        return matrix(w2, s2) @ h

    out, weights = [], []
    for t in range(case["tokens"]):
        v = s["x"][t].double()
        logits = s["router"].double() @ v
        score = torch.sigmoid(logits) if c["scoring"] == "sigmoid" else torch.softmax(logits, 0)
        liked = score if s["bias"] is None else score + s["bias"].double()
        groups = sorted(range(c["groups"]), key=lambda q: -float(liked[q * per:(q + 1) * per].topk(min(2, per)).values.sum()))[:c["kept"]]
        chosen = sorted((e for q in groups for e in range(q * per, (q + 1) * per)), key=lambda e: -float(liked[e]))[:k]
        w = score[chosen]
        w = w / w.sum() * c["scaling"]
        y = torch.zeros_like(v) if s["residual"] is None else s["residual"][t].double()
        for e, we in zip(chosen, w):
            y = y + we * expert(v, s["w1"][e], None if s["s1"] is None else s["s1"][e], s["w2"][e], None if s["s2"] is None else s["s2"][e])
        if case["shared"]:
            y = y + expert(v, s["shared_w1"], s["shared_s1"], s["shared_w2"], s["shared_s2"])
        out.append(y)
        weights.append(w)
    return {"out": torch.stack(out), "weights": torch.stack(weights), "ids": None}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_few(case, s) if case["op"] == "few" else _exact_linear(case, s)


def work(case):
    if case["op"] == "few":
        c, M, width = _SHAPES[case["shape"]], case["tokens"], 1 if case["format"] == "fp8_block" else 2
        used = c["E"] * (1.0 - (1.0 - case["topk"] / c["E"]) ** M)  # different experts of M tokens, on average
        rows = used * c["I"] + case["shared"]
        scales = rows * c["H"] * 3 / 16384 * 4 if width == 1 else 0
        return {"bytes": int(rows * c["H"] * 3 * width + scales + c["E"] * c["H"] * 2 + M * c["H"] * (6 if case["residual"] else 4)),
                "flops": int(2 * M * c["H"] * (c["E"] + 3 * (case["topk"] * c["I"] + case["shared"])))}
    M, K, N, width = case["tokens"], case["k"], case["n"], 4 if case["dtype"] == "f32" else 2
    rows = N * (2 if case["act"] == "silu_and_mul" else 1)
    once = M * K + rows * K + M * N * (2 if case["residual"] else 1) + (rows if case["bias"] else 0)
    more = M * N * (2 if case["residual"] else 1) + M * K + rows * K + (rows if case["bias"] else 0)
    return {"bytes": width * (once + (more if case["train"] else 0)), "flops": 2 * M * K * rows * (3 if case["train"] else 1)}
