"""
The operators of a routed mixture-of-experts model and of its dense projections with block scales, as measurable cases.

* ``route``    from router logits to expert weights, expert ids and tokens per expert
               (``olmo_core_amd.ops.moe.route``), in training with the gradient of the logits
* ``linear``   ``y = q(x) q(W)^T`` in float8 e4m3 with one power-of-two scale for each block: 1 x 128 of activations and
               gradients, 128 x 128 of weights (``olmo_core_amd.float8.blockwise_linear``); in training with the gradients
               ``gx = q(g) q(W)`` and ``gW = q(g^T) q(x^T)^T``, whose operands have their blocks along the tokens
* ``experts``  the same product for rows sorted by expert, each group of rows with a weight of its own
               (``olmo_core_amd.float8.blockwise_grouped_linear``)

A block's scale is the largest power of two that keeps the block's largest magnitude times the scale within 448, at most 2^120.

:func:`listed` names twelve cases, :func:`draw` gives others of the same ranges.
"""

import math

import torch

own = False

_MOST_SCALE = 120
# (in, out) of single projections: generic ones, one whose sizes are multiples of 16 and of nothing larger, the 7B shapes
_LINEAR_DIMS = [(768, 2048), (1024, 1024), (1024, 2816), (1040, 2768), (2048, 8192), (4096, 4096), (4096, 11008), (11008, 4096)]
# (d_model, expert hidden, experts, top_k) of expert layers; the up projection (d_model -> hidden) is what is measured
_EXPERT_DIMS = [(512, 256, 8, 2), (1024, 512, 32, 4), (1040, 336, 12, 3), (1024, 1792, 8, 2), (2048, 1024, 64, 8)]
# (experts, top_k, groups, groups kept)
_ROUTES = [(8, 2, 1, 1), (12, 3, 1, 1), (32, 4, 1, 1), (60, 4, 1, 1), (64, 8, 1, 1), (64, 6, 8, 3), (128, 8, 1, 1), (256, 8, 8, 4)]
# no drawn case has more arithmetic than the largest listed one
_MOST_FLOPS = 6.0 * 16384 * 4096 * 11008


def listed():
    return [
        # a small batch of sequences generating: latency alone
        {"name": "route_decode_48", "kind": "route", "tokens": 48, "experts": 64, "top_k": 8, "groups": 1, "kept": 1,
         "gating": "softmax", "bias": False, "normalize": False, "half": True, "train": False},
        # the router of the 64-expert layer in training
        {"name": "route_train_64", "kind": "route", "tokens": 16384, "experts": 64, "top_k": 8, "groups": 1, "kept": 1,
         "gating": "softmax", "bias": False, "normalize": True, "half": True, "train": True},
        # many experts in groups, sigmoid scores and a balancing bias, float32 logits
        {"name": "route_train_256_groups", "kind": "route", "tokens": 16384, "experts": 256, "top_k": 8, "groups": 8, "kept": 4,
         "gating": "sigmoid", "bias": True, "normalize": True, "half": False, "train": True},
        # one sequence generating, the float8 weight kept between calls
        {"name": "linear_decode_1", "kind": "linear", "mode": "kept", "tokens": 1, "d": 4096, "n": 11008},
        # an odd number of sequences in flight
        {"name": "linear_decode_23", "kind": "linear", "mode": "kept", "tokens": 23, "d": 4096, "n": 11008},
        # a prompt of ordinary length
        {"name": "linear_prefill_777", "kind": "linear", "mode": "kept", "tokens": 777, "d": 4096, "n": 11008},
        # a small model in training, the token count of a packed batch
        {"name": "linear_train_small", "kind": "linear", "mode": "train", "tokens": 1999, "d": 1024, "n": 2816},
        # sizes that are multiples of 16 only
        {"name": "linear_train_odd", "kind": "linear", "mode": "train", "tokens": 1537, "d": 1040, "n": 2768},
        # the 7B projection at batch 4 x 4096: the largest case
        {"name": "linear_train_7b", "kind": "linear", "mode": "train", "tokens": 16384, "d": 4096, "n": 11008},
        # an expert layer's projection generating for a small batch
        {"name": "experts_decode_48", "kind": "experts", "mode": "kept", "tokens": 48, "d": 2048, "n": 1024, "experts": 64, "top_k": 8},
        # a small expert layer in training
        {"name": "experts_train_small", "kind": "experts", "mode": "train", "tokens": 1002, "d": 1024, "n": 512, "experts": 32, "top_k": 4},
        # 64 experts of skewed popularity, some of them empty
        {"name": "experts_train", "kind": "experts", "mode": "train", "tokens": 16384, "d": 2048, "n": 1024, "experts": 64, "top_k": 8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["route", "route", "linear", "linear", "linear", "experts", "experts"])
        if kind == "route":
            experts, top_k, groups, kept = rng.choice(_ROUTES)
            case = {"kind": kind, "tokens": _log_int(rng, 1, 16384), "experts": experts, "top_k": top_k, "groups": groups, "kept": kept,
                    "gating": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "normalize": rng.random() < 0.5,
                    "half": rng.random() < 0.5, "train": rng.random() < 0.6}
        elif kind == "linear":
            d, n = rng.choice(_LINEAR_DIMS)
            mode = rng.choice(["kept", "forward", "train", "train"])
            case = {"kind": kind, "mode": mode, "tokens": _log_int(rng, 200 if mode == "train" else 1, 16384), "d": d, "n": n}
        else:
            d, n, experts, top_k = rng.choice(_EXPERT_DIMS)
            mode = rng.choice(["kept", "train"])
            case = {"kind": kind, "mode": mode, "tokens": _log_int(rng, 200 if mode == "train" else 1, 16384), "d": d, "n": n,
                    "experts": experts, "top_k": top_k}
        if work(case)["flops"] <= _MOST_FLOPS:
            return case


# ---- inputs ----------------------------------------------------------------------------------------------------


def _activations(g, rows, cols):
    """What reaches a projection: features of unlike size, 0.1 % of the entries twenty times larger."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    x *= torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 1e-3, 20.0, 1.0)
    return x.to(torch.bfloat16)


def _tensors(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = case["tokens"]
    if case["kind"] == "route":
        experts = case["experts"]
        # popularity falls off with the rank of the expert, as a router's scores do before they are balanced
        rank = torch.arange(1, experts + 1, device="cuda", dtype=torch.float32)
        logits = torch.randn(tokens, experts, generator=g, device="cuda") - 0.5 * torch.log(rank)
        state = {"logits": logits.to(torch.bfloat16) if case["half"] else logits, "bias": None}
        if case["bias"]:
            state["bias"] = torch.randn(experts, generator=g, device="cuda").mul_(0.05)
        if case["train"]:
            state["grad"] = torch.randn(tokens, case["top_k"], generator=g, device="cuda").mul_(1e-3)
        return state
    rows, experts = tokens, case.get("experts", 1)
    state = {}
    if case["kind"] == "experts":
        rows = tokens * case["top_k"]
        # skewed popularity (Zipf s = 1.1), so that with many experts some get no token
        rank = torch.arange(1, experts + 1, device="cuda", dtype=torch.float32)
        scores = torch.randn(tokens, experts, generator=g, device="cuda") - 1.75 * 1.1 * torch.log(rank)
        state["sizes"] = torch.bincount(scores.topk(case["top_k"], dim=-1).indices.flatten(), minlength=experts)
    state["x"] = _activations(g, rows, case["d"])
    state["weight"] = torch.randn(experts * case["n"], case["d"], generator=g, device="cuda").mul_(0.02).to(torch.bfloat16)
    if case["mode"] == "train":
        state["grad"] = torch.randn(rows, case["n"], generator=g, device="cuda").mul_(1e-3).to(torch.bfloat16)
    return state


def prepare(case, seed):
    state = _tensors(case, seed)
    state["case"] = case
    train = case["train"] if case["kind"] == "route" else case["mode"] == "train"
    if train:
        for name in ("logits", "x", "weight"):
            if name in state:
                state[name].requires_grad_(True)
    if case["kind"] == "experts":
        state["groups"] = state["sizes"].tolist()  # (the plain form's loop over the experts)
    if case.get("mode") == "kept":
        # a server quantises its weights once
        if own:
            from olmo_core_amd.float8 import blockwise_weight

            state["kept"] = blockwise_weight(state["weight"], experts=case.get("experts", 1))
        else:
            state["kept"] = [_weight_values(w) for w in state["weight"].split(case["n"])]
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------


def _step(amax):
    """Exponent k of the scale 2^k of blocks with these largest magnitudes."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa 2^exponent, 0.5 <= mantissa < 1; 448 = 0.875 2^9
    return (9 - exponent - (mantissa > 0.875).to(exponent.dtype)).clamp(max=_MOST_SCALE)


def _power(k):
    """2^k in float32, by its exponent field (``torch.ldexp`` goes through ``pow``, which is off in the last bits)."""
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, dims):
    """float32 values that blocks ``x`` (the axes ``dims`` inside a block) have in float8."""
    k = _step(x.abs().amax(dim=dims, keepdim=True))
    return (x * _power(k)).to(torch.float8_e4m3fn).float() * _power(-k)


def _row_values(x):
    """``x [rows, K]`` with a scale for each 128 of K."""
    rows, K = x.shape
    pad = -K % 128
    blocks = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, 128)
    return _quantise(blocks, (2,)).view(rows, K + pad)[:, :K]


def _weight_values(w):
    """``w [N, K]`` with a scale for each 128 x 128."""
    N, K = w.shape
    blocks = torch.nn.functional.pad(w.float(), (0, -K % 128, 0, -N % 128))
    blocks = blocks.view(blocks.shape[0] // 128, 128, blocks.shape[1] // 128, 128)
    return _quantise(blocks, (1, 3)).view(blocks.shape[0] * 128, -1)[:N, :K]


def _plain_linear(x, w_values):
    return (_row_values(x) @ w_values.t()).to(x.dtype)


def _plain_backward(x, w_values, grad, w_dtype):
    gx = (_row_values(grad) @ w_values).to(x.dtype)
    gw = (_row_values(grad.t()) @ _row_values(x.t()).t()).to(w_dtype)
    return gx, gw


def _plain_products(state):
    case, x, n = state["case"], state["x"].detach(), state["case"]["n"]
    groups = state["groups"] if case["kind"] == "experts" else [x.shape[0]]
    weights = state["weight"].detach().split(n)
    train = case["mode"] == "train"
    ys, gxs, gws = [], [], []
    first = 0
    for e, rows in enumerate(groups):
        w = state["kept"][e] if case["mode"] == "kept" else _weight_values(weights[e]) if rows else None
        here = slice(first, first + rows)
        first += rows
        if rows:
            ys.append(_plain_linear(x[here], w))
        if train:
            if rows:
                gx, gw = _plain_backward(x[here], w, state["grad"][here], weights[e].dtype)
                gxs.append(gx)
            else:
                gw = torch.zeros_like(weights[e])
            gws.append(gw)
    out = {"y": torch.cat(ys)}
    if train:
        out.update(x_grad=torch.cat(gxs), weight_grad=torch.cat(gws))
    return out


def _plain_route(state):
    case, logits, bias = state["case"], state["logits"].detach(), state["bias"]
    tokens, experts, top_k, groups = case["tokens"], case["experts"], case["top_k"], case["groups"]
    softmax = case["gating"] == "softmax"
    # the choice in 64 bits: scores next to one another change places in 32
    choice = torch.softmax(logits.double(), -1) if softmax else torch.sigmoid(logits.double())
    if bias is not None:
        choice = choice + bias.double()
    if groups > 1:
        grouped = choice.view(tokens, groups, experts // groups)
        best = torch.sort(grouped, dim=-1, descending=True, stable=True).values[..., :2].sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :case["kept"]]
        mask = torch.zeros(tokens, groups, dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
        choice = grouped.masked_fill(~mask.unsqueeze(-1), -math.inf).view(tokens, experts)
    indices = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :top_k].contiguous()
    scores = torch.softmax(logits.float(), -1) if softmax else torch.sigmoid(logits.float())
    chosen = scores.gather(1, indices)
    total = chosen.sum(-1, keepdim=True) if case["normalize"] else torch.ones_like(chosen[:, :1])
    weights = chosen / total
    out = {"weights": weights, "indices": indices, "batch_size_per_expert": torch.bincount(indices.flatten(), minlength=experts)}
    if case["train"]:
        grad = state["grad"]
        g = (grad - (grad * weights).sum(-1, keepdim=True)) / total if case["normalize"] else grad
        g = torch.zeros_like(scores).scatter_(1, indices, g)
        g = scores * (g - (g * scores).sum(-1, keepdim=True)) if softmax else g * scores * (1 - scores)
        out["logits_grad"] = g.to(logits.dtype)
    return out


# ---- one pass --------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if not own:
        return _plain_route(state) if case["kind"] == "route" else _plain_products(state)
    if case["kind"] == "route":
        from olmo_core_amd.ops.moe import route

        logits = state["logits"]
        logits.grad = None
        weights, indices, sizes = route(logits, case["top_k"], gating=case["gating"], bias=state["bias"], groups=case["groups"],
                                        groups_kept=case["kept"], normalize=case["normalize"])
        out = {"weights": weights.detach(), "indices": indices, "batch_size_per_expert": sizes}
        if case["train"]:
            weights.backward(state["grad"])
            out["logits_grad"] = logits.grad
        return out
    from olmo_core_amd.float8 import blockwise_grouped_linear, blockwise_linear

    x, weight = state["x"], state["weight"]
    x.grad = weight.grad = None
    if case["kind"] == "linear":
        y = blockwise_linear(x, weight, kept=state.get("kept"))
    else:
        y = blockwise_grouped_linear(x, weight, state["sizes"], kept=state.get("kept"))
    if case["mode"] != "train":
        return {"y": y}
    y.backward(state["grad"])
    return {"y": y.detach(), "x_grad": x.grad, "weight_grad": weight.grad}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def _float8(v):
    """64-bit ``v`` rounded to the nearest multiple of the e4m3 spacing at its size (ties to even), at most 448."""
    size = v.abs()
    _, e = torch.frexp(size.clamp(min=2.0 ** -6))  # 2^(e - 1) <= size < 2^e
    spacing = torch.ones_like(size).view(torch.int64).add_((e.long() - 4) << 52).view(torch.float64)
    return torch.copysign((torch.round(size / spacing) * spacing).clamp(max=448.0), v)


def _scaled(x, amax):
    _, e = torch.frexp(448.0 / amax.clamp(min=2.0 ** -200))  # 2^(e - 1) <= 448 / amax < 2^e
    scale = ((e.long() - 1).clamp(max=_MOST_SCALE) + 1023 << 52).view(torch.float64)
    return _float8(x * scale) / scale


def _exact_rows(x):
    """Scales along the last axis, piece by piece (the last piece may be shorter)."""
    return torch.cat([_scaled(p, p.abs().amax(-1, keepdim=True)) for p in x.double().split(128, dim=-1)], -1)


def _exact_weight(w):
    return torch.cat([torch.cat([_scaled(b, b.abs().max()) for b in strip.split(128, dim=1)], 1) for strip in w.double().split(128)])


def exact(case, seed):
    t = _tensors(case, seed)
    if case["kind"] != "route":
        groups = t["sizes"].tolist() if case["kind"] == "experts" else [t["x"].shape[0]]
        xs = t["x"].split(groups)
        ws = t["weight"].split(case["n"])
        out = {"y": torch.cat([_exact_rows(x) @ _exact_weight(w).t() for x, w in zip(xs, ws)])}
        if case["mode"] == "train":
            gs = t["grad"].split(groups)
            out["x_grad"] = torch.cat([_exact_rows(g) @ _exact_weight(w) for g, w in zip(gs, ws)])
            out["weight_grad"] = torch.cat([_exact_rows(g.t()) @ _exact_rows(x.t()).t() if g.shape[0] else torch.zeros_like(w.double())
                                            for g, x, w in zip(gs, xs, ws)])
        return out
    logits, top_k = t["logits"].double(), case["top_k"]
    rows = torch.arange(case["tokens"], device=logits.device)
    if case["gating"] == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-logits))
    c = s.clone() if t["bias"] is None else s + t["bias"].double()
    if case["groups"] > 1:
        per = case["experts"] // case["groups"]
        first = torch.stack([p.amax(-1) for p in c.split(per, -1)], -1)
        second = torch.stack([p.scatter(-1, p.argmax(-1, keepdim=True), -math.inf).amax(-1) for p in c.split(per, -1)], -1)
        left = first + second
        allowed = torch.zeros_like(left)
        for _ in range(case["kept"]):
            g = left.argmax(-1)
            allowed[rows, g] = 1
            left[rows, g] = -math.inf
        c = torch.where(allowed.repeat_interleave(per, -1) > 0, c, -math.inf)
    # one expert after the other, the lowest id of equal scores
    ids = []
    number = torch.arange(case["experts"], device=logits.device)
    for _ in range(top_k):
        best = torch.where(c == c.amax(-1, keepdim=True), number, case["experts"]).amin(-1)
        ids.append(best)
        c[rows, best] = -math.inf
    indices = torch.stack(ids, -1)
    chosen = torch.stack([s[rows, i] for i in ids], -1)
    total = chosen.sum(-1, keepdim=True) if case["normalize"] else torch.ones_like(chosen[:, :1])
    out = {"weights": chosen / total, "indices": indices,
           "batch_size_per_expert": (indices.unsqueeze(-1) == number).sum((0, 1))}
    if case["train"]:
        # dL/ds_i of the chosen experts, then through the scores' own derivative
        grad = t["grad"].double()
        ds = torch.zeros_like(s)
        share = (grad * chosen).sum(-1) / total[:, 0] ** 2 if case["normalize"] else torch.zeros_like(total[:, 0])
        for j, i in enumerate(ids):
            ds[rows, i] = grad[:, j] / total[:, 0] - share
        if case["gating"] == "softmax":
            out["logits_grad"] = s * ds - s * (s * ds).sum(-1, keepdim=True)
        else:
            out["logits_grad"] = ds * s * (1 - s)
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    tokens = case["tokens"]
    if case["kind"] == "route":
        experts, top_k, size = case["experts"], case["top_k"], 2 if case["half"] else 4
        data = tokens * (experts * size + top_k * 12) + experts * 8 + (4 * experts if case["bias"] else 0)
        if case["train"]:  # the gradient of the weights in, that of the logits out
            data += tokens * (experts * size + top_k * 4)
        return {"bytes": float(data), "flops": float(tokens * experts * (16 if case["train"] else 8))}
    d, n, experts = case["d"], case["n"], case.get("experts", 1)
    rows = tokens * case.get("top_k", 1)
    if case["mode"] == "train":  # x, grad, W in; y, gx, gW out
        return {"bytes": 4.0 * rows * (d + n) + 4.0 * experts * n * d, "flops": 6.0 * rows * d * n}
    used = experts * (1.0 - (1.0 - 1.0 / experts) ** rows) if experts > 1 else 1.0  # experts that have a row
    size = 1 if case["mode"] == "kept" else 2
    return {"bytes": 2.0 * rows * (d + n) + used * size * n * d, "flops": 2.0 * rows * d * n}
