"""Performance cases of the operators between two layers of experts.

Three operators, each in a plain form (elementary torch operations in 32 bits) and, where ``own`` is true, through the
calls that a user makes:

``norm``     ``rms_norm``: the residual's addition and the root-mean-square norm in front of a layer; with gradients
             where the case trains.
``quant``    ``rms_norm_quant``: the same with an 8-bit output and its scales, for projections that take 8 bits.
``balance``  ``moe_balance_loss``: the loss that keeps a router's experts evenly used, the tokens that each expert got,
             and the gradient of the router's logits.

Hidden sizes, experts and value distributions are those of ``bench.py`` and ``perf/cases.py``: activations and logits
~N(0, 1), routing bias ~N(0, 0.1)."""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6
_QUANT_EPS = 1e-10
_QMAX = {"e4m3": 448.0, "int8": 127.0}


def _norm(tokens, hidden, dtype="bf16", weight="same", residual=True, train=False, gap=0):
    return {"op": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "weight": weight, "residual": residual,
            "train": train, "gap": gap}


def _quant(tokens, hidden, group, out="e4m3", dtype="bf16", residual=True, also_norm=False, column_major=False, gap=0):
    return {"op": "quant", "tokens": tokens, "hidden": hidden, "group": group, "out": out, "dtype": dtype,
            "residual": residual, "also_norm": also_norm, "column_major": column_major, "gap": gap}


def _balance(tokens, experts, topk, scoring="softmax", dtype="f32", sequences=0, padded=False, train=True):
    return {"op": "balance", "tokens": tokens, "experts": experts, "topk": topk, "scoring": scoring, "dtype": dtype,
            "sequences": sequences, "padded": padded, "train": train}


def listed():
    return [
        # one sequence being decoded: latency and launches
        {"name": "norm_decode_1", **_norm(1, 7168)},
        # a full prefill chunk
        {"name": "norm_prefill_8192", **_norm(8192, 7168)},
        # one micro-batch of training, forward and backward
        {"name": "norm_train_4096", **_norm(4096, 4096, train=True)},
        # a hidden size that no vector width divides, no residual, 32 bits
        {"name": "norm_train_odd_1000", **_norm(1000, 1023, "f32", residual=False, train=True)},
        # mixed precision training: activations in f16, the weight and its gradient in f32
        {"name": "norm_train_16384", **_norm(16384, 4096, "f16", weight="f32", train=True)},
        # a decode batch in front of a projection with block scales
        {"name": "quant_fp8_decode_61", **_quant(61, 7168, 128)},
        # a prefill chunk: the 8 bits for the projections, the norm itself for the router
        {"name": "quant_fp8_prefill_8192", **_quant(8192, 7168, 128, also_norm=True, column_major=True)},
        # a mixed batch in front of int8 with a scale per token; the rows lie in a wider buffer
        {"name": "quant_int8_mixed_500", **_quant(500, 2048, 0, out="int8", gap=64)},
        # the smallest router
        {"name": "balance_64", **_balance(64, 8, 2)},
        # logits in bf16, one micro-batch as a whole
        {"name": "balance_4096", **_balance(4096, 128, 8, dtype="bf16")},
        # packed sequences of uneven length, each balanced by itself, with padding in them
        {"name": "balance_packed_8192", **_balance(8192, 256, 8, "sigmoid", sequences=23, padded=True)},
        # a global batch
        {"name": "balance_65536", **_balance(65536, 256, 8)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "norm", "quant", "quant", "balance", "balance"))
    if op == "balance":
        experts = rng.choice((8, 16, 60, 64, 128, 160, 256))
        tokens = _log_int(rng, 16, 65536)
        return _balance(tokens, experts, rng.randint(1, min(8, experts)), rng.choice(("softmax", "sigmoid")),
                        rng.choice(("f32", "f32", "bf16")), sequences=rng.choice((0, 1, _log_int(rng, 2, 64))),
                        padded=rng.random() < 0.5, train=rng.random() < 0.75)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    tokens = _log_int(rng, 1, 8192)
    if op == "norm":
        hidden = rng.choice((7168, 4096, 2048, 1024, _log_int(rng, 64, 8192), 8 * _log_int(rng, 8, 1024)))
        return _norm(tokens, hidden, dtype if hidden * tokens < 1 << 25 else "bf16", rng.choice(("same", "f32")),
                     rng.random() < 0.75, rng.random() < 0.5, rng.choice((0, 0, 8, 1)))
    group = rng.choice((128, 128, 64, 0))
    hidden = rng.choice((7168, 4096, 2048, 1024, 128 * _log_int(rng, 1, 64), 64 * _log_int(rng, 1, 96)))
    group = group if group and hidden % group == 0 else 0
    return _quant(tokens, hidden, group, rng.choice(("e4m3", "e4m3", "int8")), dtype if hidden * tokens < 1 << 25 else "bf16",
                  rng.random() < 0.75, rng.random() < 0.5, bool(group) and rng.random() < 0.5, rng.choice((0, 0, 8)))


def _rows(tokens, hidden, gap, dtype, g):
    """[tokens, hidden] ~N(0, 1), the rows ``hidden + gap`` elements apart."""
    return torch.randn((tokens, hidden + gap), generator=g, device=g.device).to(dtype)[:, :hidden]


def _prepare_norm(case, g):
    M, H, dtype = case["tokens"], case["hidden"], _DTYPES[case["dtype"]]
    weight = 1.0 + 0.1 * torch.randn((H,), generator=g, device=g.device)
    if case.get("weight") != "f32":
        weight = weight.to(dtype)
    state = {"case": case, "x": _rows(M, H, case["gap"], dtype, g), "residual": None, "weight": weight}
    if case["residual"]:
        state["residual"] = 2.0 * _rows(M, H, 0, dtype, g)  # the stream is larger than what a layer adds to it
    if case.get("train"):
        state["dy"] = _rows(M, H, 0, dtype, g)
        state["dh"] = _rows(M, H, 0, dtype, g)
        state["leaves"] = [t for t in (state["x"], state["residual"], weight) if t is not None]
        for t in state["leaves"]:
            t.requires_grad_(True)
    return state


def _prepare_balance(case, g):
    T, E, k = case["tokens"], case["experts"], case["topk"]
    dev = g.device
    bias = 0.1 * torch.randn((E,), generator=g, device=dev)
    logits = torch.randn((T, E), generator=g, device=dev) + 2.0 * bias  # some experts are liked more
    logits = logits.to(_DTYPES[case["dtype"]])
    scores = logits.float().sigmoid() if case["scoring"] == "sigmoid" else logits.float().softmax(-1)
    ids = (scores + (bias if case["scoring"] == "sigmoid" else 0.0)).topk(k, dim=-1).indices.int()
    state = {"case": case, "logits": logits, "ids": ids, "cu_seqlens": None, "is_padding": None}
    if case["sequences"]:
        # uneven lengths, some of them zero; what the last sequence leaves of the buffer belongs to none
        cuts = (torch.rand((case["sequences"],), generator=g, device=dev) * (T + 1)).long().clamp_(max=T)
        cu = torch.cat([cuts.new_zeros(1), cuts]).sort().values
        state["cu_seqlens"] = cu.int()
    if case["padded"]:
        pad = torch.rand((T,), generator=g, device=dev) < 0.15
        logits[pad] = float("nan")  # rows that nobody wrote
        ids[pad] = -1               # what the routers give for them
        state["is_padding"] = pad
    # the factor of the loss in the objective, times a scale that keeps 16-bit gradients out of the subnormals
    state["dloss"] = torch.full((), 1e-3 * (T if case["dtype"] != "f32" else 1.0), device=dev)
    if case["train"]:
        logits.requires_grad_(True)
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return _prepare_balance(case, g) if case["op"] == "balance" else _prepare_norm(case, g)


# ---- the framework's calls -------------------------------------------------------------------------------------------


def _own_norm(s):
    import flaggems_vllm_b200 as fg

    out = fg.rms_norm(s["x"], s["weight"], _EPS, residual=s["residual"])
    y, h = out if s["residual"] is not None else (out, None)
    if not s["case"]["train"]:
        return {"y": y, "h": h}
    outs, grads = ([y], [s["dy"]]) if h is None else ([y, h], [s["dy"], s["dh"]])
    return {"y": y, "h": h, "grads": list(torch.autograd.grad(outs, s["leaves"], grads))}


def _own_quant(s):
    import flaggems_vllm_b200 as fg

    c = s["case"]
    out = fg.rms_norm_quant(s["x"], s["weight"], _EPS, residual=s["residual"], group_size=c["group"] or None,
                            dtype=torch.int8 if c["out"] == "int8" else torch.float8_e4m3fn,
                            column_major_scales=c["column_major"], return_norm=c["also_norm"])
    q, scale = out[0], out[1]
    return {"q": q.to(s["x"].dtype) if c["out"] == "int8" else q, "scale": scale, "rest": list(out[2:])}


def _own_balance(s):
    import flaggems_vllm_b200 as fg

    loss, counts = fg.moe_balance_loss(s["logits"], s["ids"], s["case"]["scoring"], cu_seqlens=s["cu_seqlens"],
                                       is_padding=s["is_padding"])
    out = {"loss": loss, "counts": counts}
    if s["case"]["train"]:
        (out["dlogits"],) = torch.autograd.grad(loss, s["logits"], s["dloss"])
    return out


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _plain_stream(s):
    """The residual stream behind the addition, as it is stored, and in 32 bits."""
    if s["residual"] is None:
        return None, s["x"].float()
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    return h, h.float()


def _plain_norm(s):
    h, hf = _plain_stream(s)
    w = s["weight"].float()
    H = hf.shape[1]
    inv = 1.0 / torch.sqrt((hf * hf).sum(-1, keepdim=True) / H + _EPS)
    out = {"y": (hf * inv * w).to(s["x"].dtype), "h": h}
    if not s["case"]["train"]:
        return out
    # y_j = w_j h_j r, r = (mean(h^2) + eps)^-1/2:  dh_i = r (w_i dy_i - h_i r^2 mean(w dy h)),  dw_j = sum over rows of dy_j h_j r
    dy = s["dy"].float()
    wdy = w * dy
    dx = inv * (wdy - hf * (inv * inv * ((wdy * hf).sum(-1, keepdim=True) / H)))
    if h is not None:
        dx = dx + s["dh"].float()
    dx = dx.to(s["x"].dtype)
    dw = (dy * (hf * inv)).sum(0).to(s["weight"].dtype)
    out["grads"] = [dx, dw] if h is None else [dx, dx, dw]
    return out


def _plain_quant(s):
    c = s["case"]
    h, hf = _plain_stream(s)
    M, H = hf.shape
    inv = 1.0 / torch.sqrt((hf * hf).sum(-1, keepdim=True) / H + _EPS)
    y = hf * inv * s["weight"].float()
    groups = y.view(M, -1, c["group"] or H)
    scale = groups.abs().amax(-1).clamp(min=_QUANT_EPS) * (1.0 / _QMAX[c["out"]])
    q = groups / scale.unsqueeze(-1)
    if c["out"] == "int8":
        q = q.round().clamp(-128.0, 127.0).to(s["x"].dtype)
    else:
        q = q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    if c["column_major"]:
        scale = scale.t().contiguous().t()
    return {"q": q.view(M, H), "scale": scale,
            "rest": ([h] if h is not None else []) + ([y.to(s["x"].dtype)] if c["also_norm"] else [])}


def _plain_balance(s):
    c, logits, ids, cu, pad = s["case"], s["logits"].float(), s["ids"].long(), s["cu_seqlens"], s["is_padding"]
    (T, E), k = logits.shape, ids.shape[1]
    dev = logits.device
    live = torch.ones((T,), dtype=torch.bool, device=dev) if pad is None else ~pad
    seq = torch.zeros((T,), dtype=torch.long, device=dev)
    S = 1
    if cu is not None:
        S = cu.numel() - 1
        seq = torch.searchsorted(cu[1:].contiguous(), torch.arange(T, device=dev, dtype=cu.dtype), right=True)
        live = live & (seq < S)
        seq = seq.clamp(max=S - 1)
    logits = torch.where(live[:, None], logits, 0.0)
    u = -torch.log1p(torch.exp(-logits.abs())) + logits.clamp(max=0.0) if c["scoring"] == "sigmoid" else logits
    p = torch.exp(u - u.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    p = torch.where(live[:, None], p, 0.0)
    tokens = torch.zeros((S,), dtype=torch.float64, device=dev).index_add_(0, seq, live.double())
    used = (ids >= 0) & (ids < E) & live[:, None]
    counts = torch.zeros((S * E,), dtype=torch.int32, device=dev)
    counts.index_add_(0, (seq[:, None] * E + ids.clamp(0, E - 1)).flatten(), used.int().flatten())
    counts = counts.view(S, E)
    if S == 1:
        mass = p.sum(0, dtype=torch.float64)[None]
    else:
        mass = torch.zeros((S, E), dtype=torch.float64, device=dev).index_add_(0, seq, p.double())
    share = tokens.clamp(min=1.0)
    filled = (tokens > 0).double().sum().clamp(min=1.0)
    each = E * (counts.double() * mass).sum(-1) / (k * share * share)
    out = {"loss": (each.sum() / filled).float(), "counts": counts if cu is not None else counts[0]}
    if c["train"]:
        # each = sum_e f_e P_e with the fractions f held: dP_e = f_e, and the softmax's (log-sigmoid's) own derivative behind it
        f = (s["dloss"].double() * E * counts.double() / (k * share * share * filled)[:, None]).float()[seq]
        d = p * (f - (p * f).sum(-1, keepdim=True))
        if c["scoring"] == "sigmoid":
            d = d / (1.0 + torch.exp(logits))
        out["dlogits"] = torch.where(live[:, None], d, 0.0).to(s["logits"].dtype)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "quant": _own_quant, "balance": _own_balance}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "quant": _plain_quant, "balance": _plain_balance}[op](state)


# ---- in 64 bits, from the definitions --------------------------------------------------------------------------------


def _exact_norm(case, s):
    x = s["x"].detach().double()
    total = x if s["residual"] is None else x + s["residual"].detach().double()
    stream = total.to(s["x"].dtype).double().requires_grad_(True)  # the norm is that of the stream as it is stored
    weight = s["weight"].detach().double().requires_grad_(True)
    y = stream / (stream.square().mean(-1, keepdim=True) + _EPS).sqrt() * weight
    if case["op"] == "quant":
        y = y.detach()
        blocks = y.unflatten(-1, (-1, case["group"] or case["hidden"]))
        scale = blocks.abs().amax(-1).clamp(min=_QUANT_EPS) / _QMAX[case["out"]]
        rest = ([] if s["residual"] is None else [total]) + ([y] if case["also_norm"] else [])
        q = (blocks / scale.unsqueeze(-1)).flatten(-2)
        # int8 values are whole numbers; an 8-bit float is held against the value before its rounding
        return {"q": q.round() if case["out"] == "int8" else q, "scale": scale, "rest": rest}
    out = {"y": y.detach(), "h": None if s["residual"] is None else total}
    if case["train"]:
        dstream, dweight = torch.autograd.grad(y, (stream, weight), s["dy"].double())
        if s["residual"] is None:
            out["grads"] = [dstream, dweight]
        else:
            dstream = dstream + s["dh"].double()
            out["grads"] = [dstream, dstream, dweight]
    return out


def _exact_balance(case, s):
    logits = s["logits"].detach().double()
    E, k = case["experts"], case["topk"]
    cu = [0, case["tokens"]] if s["cu_seqlens"] is None else s["cu_seqlens"].tolist()
    loss, grads, filled = 0.0, torch.zeros_like(logits), 0
    pieces = []
    for a, b in zip(cu[:-1], cu[1:]):
        rows = torch.arange(a, b, device=logits.device)
        if s["is_padding"] is not None:
            rows = rows[~s["is_padding"][a:b]]
        if rows.numel():
            filled += 1
            pieces.append(rows)
    for rows in pieces:
        part = logits[rows].requires_grad_(True)
        if case["scoring"] == "sigmoid":
            affinity = torch.sigmoid(part)
            prob = affinity / affinity.sum(-1, keepdim=True)
        else:
            prob = torch.softmax(part, -1)
        chosen = torch.bincount(s["ids"][rows].long().flatten(), minlength=E).double()
        fraction = chosen * E / (k * rows.numel())
        one = (fraction * prob.mean(0)).sum() / filled
        loss += one.item()
        if case["train"]:
            (grads[rows],) = torch.autograd.grad(one, part, s["dloss"].double())
    out = {"loss": torch.tensor(loss, dtype=torch.float64), "counts": None}
    if case["train"]:
        out["dlogits"] = grads
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_balance(case, s) if case["op"] == "balance" else _exact_norm(case, s)


def work(case):
    if case["op"] == "balance":
        T, E, k, width = case["tokens"], case["experts"], case["topk"], 4 if case["dtype"] == "f32" else 2
        read = T * E * width + T * k * 4 + (T if case["padded"] else 0) + 4 * case["sequences"]
        return {"bytes": read + 4 * E * max(1, case["sequences"]) + (T * E * width if case["train"] else 0),
                "flops": T * E * (13 if case["train"] else 6)}
    n, width = case["tokens"] * case["hidden"], 4 if case["dtype"] == "f32" else 2
    tensors = 4 if case["residual"] else 2  # x, residual, stream, norm
    if case["op"] == "quant":
        groups = case["tokens"] * (case["hidden"] // case["group"] if case["group"] else 1)
        return {"bytes": n * width * (tensors - 1 + case["also_norm"]) + n + 4 * groups + 4 * case["hidden"], "flops": 8 * n}
    if case["train"]:
        tensors += 3 if case["residual"] else 2  # the gradients that come in, the one that goes out
    return {"bytes": n * width * tensors + 4 * case["hidden"] * (2 if case["train"] else 1),
            "flops": (16 if case["train"] else 5) * n}
