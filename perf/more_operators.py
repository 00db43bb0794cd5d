"""
What a transformer block runs beside its float8 layers, in the model's own type, as measurable cases.

* ``linear``   ``y = residual + act(x W^T + bias)`` (``olmo_core_amd.ops.linear.linear``), in training with all gradients
* ``experts``  the same product without an epilogue for rows sorted by expert, each group of rows with a weight of its own
               (``olmo_core_amd.ops.linear.grouped_linear``), in training with both gradients
* ``norm``     a block's output on its way into the residual stream and the norm in front of the next block
               (``olmo_core_amd.ops.norm.residual_norm``):
               ``h = residual_scale residual + scale gate drop(norm(branch) post)``, ``n = norm(h) pre``, where
               ``norm(v) = v / sqrt(mean(v^2) + eps)``; every part may be absent
* ``dropout``  ``y = x / (1 - p)`` where the element is kept, else 0 (``olmo_core_amd.ops.dropout.dropout``)

Which elements are kept: element ``i`` of a tensor in the order of its rows takes the 16 bits ``i % 8`` (the lowest of the first word first) of
what Philox-4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with 7 rounds makes of the
counter ``(i / 8, offset)`` and the key ``seed``, 64 bits each, low word first.  It is kept where they are at least ``t = round(65536 p)``, and kept
values are multiplied with ``65536 / (65536 - t)``.

:func:`listed` names twelve cases, :func:`draw` gives others of the same ranges.
"""

import math

import torch

own = False

_EPS = 1e-6
_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
# (in, out) of single projections: generic ones, some whose sizes are no multiples of anything, the 7B shapes
_LINEAR_DIMS = [(768, 2048), (1001, 1000), (1024, 1024), (1024, 2816), (1031, 2771), (1040, 2768), (2048, 8192), (4096, 4096), (4096, 11008),
                (11008, 4096)]
_ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
# (in, out, experts, top_k) of expert layers
_EXPERT_DIMS = [(512, 256, 8, 2), (1024, 512, 32, 4), (1031, 517, 12, 3), (1040, 336, 12, 3), (1024, 1792, 8, 2), (2048, 1024, 64, 8)]
# a head's features, models' features, odd ones, those of the widest layers
_NORM_DIMS = [64, 128, 768, 1000, 1024, 1031, 2048, 2500, 4096, 5120, 8192, 11008]
# no drawn case has more work than the largest listed one
_MOST_FLOPS = 6.0 * 16384 * 4096 * 11008
_MOST_ELEMENTS = 16384 * 4096


def listed():
    return [
        # one sequence generating: the weight is read once
        {"name": "linear_decode_1", "kind": "linear", "train": False, "tokens": 1, "d": 4096, "n": 11008, "bias": False,
         "activation": "silu", "residual": False, "type": "bfloat16"},
        # a prompt of ordinary length
        {"name": "linear_prefill_777", "kind": "linear", "train": False, "tokens": 777, "d": 4096, "n": 11008, "bias": True,
         "activation": "gelu", "residual": False, "type": "bfloat16"},
        # a small model in training; no size is a multiple of 16 bytes
        {"name": "linear_train_odd", "kind": "linear", "train": True, "tokens": 1537, "d": 1031, "n": 2771, "bias": True,
         "activation": "gelu_tanh", "residual": True, "type": "float16"},
        # the 7B down projection at batch 4 x 4096, joined with the residual stream: the largest case
        {"name": "linear_train_7b", "kind": "linear", "train": True, "tokens": 16384, "d": 11008, "n": 4096, "bias": True,
         "activation": "none", "residual": True, "type": "bfloat16"},
        # an expert layer's projection generating for a small batch
        {"name": "experts_decode_48", "kind": "experts", "train": False, "tokens": 48, "d": 2048, "n": 1024, "experts": 64, "top_k": 8,
         "transposed": False, "type": "bfloat16"},
        # a small expert layer's projection back to the model's features, in training
        {"name": "experts_train_small", "kind": "experts", "train": True, "tokens": 1002, "d": 512, "n": 1024, "experts": 32, "top_k": 4,
         "transposed": True, "type": "bfloat16"},
        # 64 experts of skewed popularity, some of them empty
        {"name": "experts_train", "kind": "experts", "train": True, "tokens": 16384, "d": 2048, "n": 1024, "experts": 64, "top_k": 8,
         "transposed": False, "type": "bfloat16"},
        # a few sequences generating in a model with norms on both sides of its blocks: latency alone
        {"name": "norm_decode_5", "kind": "norm", "train": False, "tokens": 5, "d": 4096, "post": True, "pre": True, "gate": False,
         "residual": True, "wide": False, "p": 0.0, "scale": 1.0, "residual_scale": 1.0, "type": "bfloat16", "wide_weights": False},
        # the 7B model in training, every part of the operator
        {"name": "norm_train_7b", "kind": "norm", "train": True, "tokens": 16384, "d": 4096, "post": True, "pre": True, "gate": True,
         "residual": True, "wide": False, "p": 0.1, "scale": 1.0, "residual_scale": 1.0, "type": "bfloat16", "wide_weights": False},
        # a packed batch of odd sizes, the residual stream in float32, depth scaled
        {"name": "norm_train_odd", "kind": "norm", "train": True, "tokens": 1999, "d": 1031, "post": False, "pre": True, "gate": True,
         "residual": True, "wide": True, "p": 0.0, "scale": 0.25, "residual_scale": 1.0, "type": "bfloat16", "wide_weights": True},
        # a small model's activations, float32, an odd number of them
        {"name": "dropout_train_odd", "kind": "dropout", "train": True, "tokens": 777, "d": 1031, "p": 0.25, "type": "float32"},
        # the 7B model's residual branch
        {"name": "dropout_train_7b", "kind": "dropout", "train": True, "tokens": 16384, "d": 4096, "p": 0.1, "type": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["linear", "linear", "experts", "experts", "norm", "norm", "dropout"])
        train = rng.random() < 0.6
        tokens = _log_int(rng, 200 if train else 1, 16384)
        case = {"kind": kind, "train": train, "tokens": tokens, "type": rng.choice(["bfloat16", "bfloat16", "float16"])}
        if kind == "linear":
            d, n = rng.choice(_LINEAR_DIMS)
            case.update(d=d, n=n, bias=rng.random() < 0.5, activation=rng.choice(_ACTIVATIONS), residual=rng.random() < 0.5)
        elif kind == "experts":
            d, n, experts, top_k = rng.choice(_EXPERT_DIMS)
            case.update(d=d, n=n, experts=experts, top_k=top_k, transposed=rng.random() < 0.5)
        elif kind == "norm":
            post, pre = rng.choice([(True, True), (True, False), (False, True), (False, True)])
            case.update(d=rng.choice(_NORM_DIMS), post=post, pre=pre, gate=rng.random() < 0.4, residual=rng.random() < 0.8,
                        wide=rng.random() < 0.3, p=rng.choice([0.0, 0.0, 0.1]), scale=rng.choice([1.0, 0.22]),
                        residual_scale=rng.choice([1.0, 1.0, 1.5]), type=rng.choice(["bfloat16", "float16", "float32"]),
                        wide_weights=rng.random() < 0.5)
        else:
            case.update(d=rng.choice(_NORM_DIMS), p=rng.choice([0.05, 0.1, 0.25, 0.5]), type=rng.choice(["bfloat16", "float16", "float32"]))
        if kind in ("norm", "dropout"):
            if tokens * case["d"] <= _MOST_ELEMENTS:
                return case
        elif work(case)["flops"] <= _MOST_FLOPS:
            return case


# ---- inputs ----------------------------------------------------------------------------------------------------


def _activations(g, rows, cols, dtype):
    """What reaches a projection: features of unlike size, 0.1 % of the entries twenty times larger."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    x *= torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 1e-3, 20.0, 1.0)
    return x.to(dtype)


def _tensors(case, seed):
    """Everything that :func:`prepare` and :func:`exact` start from, by name; ``None`` for what the case has not."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, tokens, d = _TYPES[case["type"]], case["tokens"], case["d"]

    def normal(*shape, size=1.0, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda").mul_(size).to(dtype)

    if case["kind"] == "linear":
        n = case["n"]
        return {"x": _activations(g, tokens, d, dtype), "weight": normal(n, d, size=0.02), "bias": normal(n, size=0.1) if case["bias"] else None,
                "residual": normal(tokens, n) if case["residual"] else None, "grad": normal(tokens, n, size=1e-3) if case["train"] else None}
    if case["kind"] == "experts":
        n, experts, top_k = case["n"], case["experts"], case["top_k"]
        # skewed popularity (Zipf s = 1.1), so that with many experts some get no token
        rank = torch.arange(1, experts + 1, device="cuda", dtype=torch.float32)
        scores = torch.randn(tokens, experts, generator=g, device="cuda") - 1.75 * 1.1 * torch.log(rank)
        sizes = torch.bincount(scores.topk(top_k, dim=-1).indices.flatten(), minlength=experts)
        shape = (experts * d, n) if case["transposed"] else (experts * n, d)
        return {"x": _activations(g, tokens * top_k, d, dtype), "weight": normal(*shape, size=0.02), "sizes": sizes,
                "grad": normal(tokens * top_k, n, size=1e-3) if case["train"] else None}
    # a generator's state, as a program draws one for each call
    numbers = {"seed": (seed * 0x9E3779B97F4A7C15 + 0x1234567) % 2 ** 63, "offset": (seed * 0x100000001) % 2 ** 40}
    if case["kind"] == "dropout":
        return {"x": _activations(g, tokens, d, dtype), "grad": normal(tokens, d, size=1e-3) if case["train"] else None, **numbers}
    stream = torch.float32 if case["wide"] else dtype
    weights = torch.float32 if case["wide_weights"] else dtype
    out_type = stream if case["residual"] else dtype
    return {"branch": _activations(g, tokens, d, dtype),
            "residual": _activations(g, tokens, d, stream) if case["residual"] else None,
            "post": normal(d, size=0.1, dtype=torch.float32).add_(1).to(weights) if case["post"] else None,
            "pre": normal(d, size=0.1, dtype=torch.float32).add_(1).to(weights) if case["pre"] else None,
            "gate": normal(d, size=0.5, dtype=weights) if case["gate"] else None,
            "stream_grad": normal(tokens, d, size=1e-3, dtype=out_type) if case["train"] else None,
            "normed_grad": normal(tokens, d, size=1e-3) if case["train"] and case["pre"] else None, **numbers}


_DIFFERENTIABLE = {"linear": ("x", "weight", "bias", "residual"), "experts": ("x", "weight"), "dropout": ("x",),
                   "norm": ("branch", "residual", "post", "pre", "gate")}


def _inputs(case, state):
    """Names of the inputs that have a gradient."""
    return [k for k in _DIFFERENTIABLE[case["kind"]] if state[k] is not None]


def prepare(case, seed):
    state = _tensors(case, seed)
    state["case"] = case
    if case["train"]:
        for name in _inputs(case, state):
            state[name].requires_grad_(True)
    if case["kind"] == "experts":
        state["groups"] = state["sizes"].tolist()  # (the plain form's loop over the experts)
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------


def _f(t):
    return None if t is None else t.detach().float()


def _plain_activation(name, z):
    """``(act(z), act'(z))``."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).float()
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _plain_linear(state):
    case, dtype = state["case"], state["x"].dtype
    x, w, bias, residual = _f(state["x"]), _f(state["weight"]), _f(state["bias"]), _f(state["residual"])
    z = x @ w.t()
    if bias is not None:
        z = z + bias
    y, slope = _plain_activation(case["activation"], z)
    if residual is not None:
        y = y + residual
    out = {"y": y.to(dtype)}
    if case["train"]:
        dz = state["grad"].float() * slope
        out.update(x_grad=(dz @ w).to(dtype), weight_grad=(dz.t() @ x).to(dtype))
        if bias is not None:
            out["bias_grad"] = dz.sum(0).to(dtype)
        if residual is not None:
            out["residual_grad"] = state["grad"]
    return out


def _plain_experts(state):
    case, x, dtype = state["case"], state["x"].detach(), state["x"].dtype
    weights = state["weight"].detach().chunk(case["experts"])
    ys, gxs, gws = [], [], []
    first = 0
    for w, rows in zip(weights, state["groups"]):
        here = slice(first, first + rows)
        first += rows
        w = w.float() if case["transposed"] else w.float().t()  # [in, out]
        xs = x[here].float()
        ys.append((xs @ w).to(dtype))
        if case["train"]:
            gs = state["grad"][here].float()
            gxs.append((gs @ w.t()).to(dtype))
            gws.append((xs.t() @ gs if case["transposed"] else gs.t() @ xs).to(dtype))
    out = {"y": torch.cat(ys)}
    if case["train"]:
        out.update(x_grad=torch.cat(gxs), weight_grad=torch.cat(gws))
    return out


def _plain_kept(shape, p, seed, offset):
    """Truth values: the element is kept."""
    elements = math.prod(shape)
    low = 0xFFFFFFFF
    i = torch.arange((elements + 7) // 8, device="cuda")
    c = [i & low, i >> 32, torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)]
    key = [seed & low, seed >> 32]
    for _ in range(7):
        # (the low 64 bits of a product are the same with and without a sign)
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32 & low) ^ c[1] ^ key[0], b & low, (a >> 32 & low) ^ c[3] ^ key[1], a & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    words = torch.stack(c, -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).flatten()[:elements]
    return (bits >= round(65536 * p)).view(shape)


def _kept_factor(p):
    t = round(65536 * p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def _plain_dropout(state):
    case, x, dtype = state["case"], state["x"].detach(), state["x"].dtype
    kept, factor = _plain_kept(x.shape, case["p"], state["seed"], state["offset"]), _kept_factor(case["p"])
    out = {"y": torch.where(kept, x.float() * factor, 0).to(dtype)}
    if case["train"]:
        out["x_grad"] = torch.where(kept, state["grad"].float() * factor, 0).to(dtype)
    return out


def _plain_norm(state):
    case, dtype = state["case"], state["branch"].dtype
    u, residual = _f(state["branch"]), _f(state["residual"])
    post, pre, gate = _f(state["post"]), _f(state["pre"]), _f(state["gate"])
    scale, residual_scale, p = case["scale"], case["residual_scale"], case["p"]
    out_type = dtype if residual is None else state["residual"].dtype
    v = u
    if post is not None:
        ru = torch.rsqrt((u * u).mean(-1, keepdim=True) + _EPS)
        v = u * ru * post
    if p > 0:
        kept, factor = _plain_kept(u.shape, p, state["seed"], state["offset"]), _kept_factor(p)
        v = torch.where(kept, v * factor, 0)
    h = scale * (v if gate is None else gate * v)
    if residual is not None:
        h = h + residual_scale * residual
    out = {"stream": h.to(out_type)}
    if pre is not None:
        rh = torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)
        out["normed"] = (h * rh * pre).to(dtype)
    if not case["train"]:
        return out
    dh = state["stream_grad"].float()
    if pre is not None:
        dn, hat = state["normed_grad"].float(), h * rh
        out["pre_grad"] = (dn * hat).sum(0).to(state["pre"].dtype)
        dhat = dn * pre
        dh = dh + rh * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))
    if residual is not None:
        out["residual_grad"] = (residual_scale * dh).to(out_type)
    dv = scale * dh
    if gate is not None:
        out["gate_grad"] = (dv * v).sum(0).to(state["gate"].dtype)
        dv = dv * gate
    if p > 0:
        dv = torch.where(kept, dv * factor, 0)
    if post is not None:
        hat = u * ru
        out["post_grad"] = (dv * hat).sum(0).to(state["post"].dtype)
        dhat = dv * post
        dv = ru * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))
    out["branch_grad"] = dv.to(dtype)
    return out


_PLAIN = {"linear": _plain_linear, "experts": _plain_experts, "norm": _plain_norm, "dropout": _plain_dropout}


# ---- one pass --------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if not own:
        return _PLAIN[case["kind"]](state)
    if case["kind"] == "linear":
        from olmo_core_amd.ops.linear import linear

        activation = None if case["activation"] == "none" else case["activation"]
        outs = {"y": linear(state["x"], state["weight"], state["bias"], activation=activation, residual=state["residual"])}
        grads = [state["grad"]]
    elif case["kind"] == "experts":
        from olmo_core_amd.ops.linear import grouped_linear

        outs = {"y": grouped_linear(state["x"], state["weight"], state["sizes"], transposed=case["transposed"])}
        grads = [state["grad"]]
    elif case["kind"] == "dropout":
        from olmo_core_amd.ops.dropout import dropout

        outs = {"y": dropout(state["x"], case["p"], seed=state["seed"], offset=state["offset"])}
        grads = [state["grad"]]
    else:
        from olmo_core_amd.ops.norm import residual_norm

        stream, normed = residual_norm(state["branch"], state["residual"], post_weight=state["post"], pre_weight=state["pre"],
                                       gate=state["gate"], scale=case["scale"], residual_scale=case["residual_scale"], eps=_EPS,
                                       p=case["p"], seed=state["seed"], offset=state["offset"])
        outs, grads = {"stream": stream}, [state["stream_grad"]]
        if normed is not None:
            outs["normed"] = normed
            grads.append(state["normed_grad"])
    if not case["train"]:
        return outs
    names = _inputs(case, state)
    made = torch.autograd.grad(list(outs.values()), [state[k] for k in names], grads)
    result = {k: v.detach() for k, v in outs.items()}
    result.update((k + "_grad", v) for k, v in zip(names, made))
    return result


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def _exact_kept(shape, p, seed, offset):
    """The generator on words of 32 bits whose products are made from halves of 16."""
    elements = math.prod(shape)
    blocks = torch.arange(-(-elements // 8), device="cuda")

    def product(word, constant):  # (high, low) words
        a, b = word // 65536, word % 65536
        c, d = divmod(constant, 65536)
        middle = a * d + b * c
        low = b * d + (middle % 65536) * 65536
        return a * c + middle // 65536 + low // 2 ** 32, low % 2 ** 32

    x0, x1 = blocks % 2 ** 32, blocks // 2 ** 32
    x2, x3 = torch.full_like(blocks, offset % 2 ** 32), torch.full_like(blocks, offset // 2 ** 32)
    for r in range(7):
        k0 = (seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32
        k1 = (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32
        h0, l0 = product(x0, 0xD2511F53)
        h1, l1 = product(x2, 0xCD9E8D57)
        x0, x1, x2, x3 = h1 ^ x1 ^ k0, l1, h0 ^ x3 ^ k1, l0
    kept = torch.empty(blocks.numel(), 8, dtype=torch.bool, device="cuda")
    for j, word in enumerate((x0, x1, x2, x3)):
        kept[:, 2 * j] = word % 65536 >= round(65536 * p)
        kept[:, 2 * j + 1] = word // 65536 >= round(65536 * p)
    return kept.view(-1)[:elements].view(shape)


def _exact_outputs(case, t):
    """The outputs of the forward as 64-bit functions of the 64-bit inputs ``t``, for autograd to differentiate."""
    if case["kind"] == "linear":
        y = torch.matmul(t["x"], t["weight"].transpose(0, 1))
        if t["bias"] is not None:
            y = y + t["bias"]
        act = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
               "gelu": lambda z: 0.5 * z * torch.erfc(-z / math.sqrt(2.0)),
               "gelu_tanh": lambda z: z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z * z * z))}[case["activation"]]
        y = act(y)
        return {"y": y if t["residual"] is None else t["residual"] + y}
    if case["kind"] == "experts":
        ws = t["weight"].chunk(case["experts"])
        rows = t["x"].split(t["sizes"].tolist())
        return {"y": torch.cat([x.matmul(w if case["transposed"] else w.transpose(0, 1)) for x, w in zip(rows, ws)])}
    if case["kind"] == "dropout":
        kept = _exact_kept(t["x"].shape, case["p"], t["seed"], t["offset"])
        return {"y": t["x"] * kept * (1 / (1 - round(65536 * case["p"]) / 65536))}

    def norm(v):
        return v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / v.shape[-1] + _EPS)

    branch = t["branch"] if t["post"] is None else t["post"] * norm(t["branch"])
    if case["p"] > 0:
        kept = _exact_kept(branch.shape, case["p"], t["seed"], t["offset"])
        branch = branch * kept * (1 / (1 - round(65536 * case["p"]) / 65536))
    if t["gate"] is not None:
        branch = branch * t["gate"]
    out = {"stream": branch * case["scale"]}
    if t["residual"] is not None:
        out["stream"] = t["residual"] * case["residual_scale"] + out["stream"]
    if t["pre"] is not None:
        out["normed"] = t["pre"] * norm(out["stream"])
    return out


def exact(case, seed):
    t = _tensors(case, seed)
    names = _inputs(case, t)
    grads = [t[k].double() for k in ("grad", "stream_grad", "normed_grad") if t.get(k) is not None]
    wide = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in t.items()}
    for name in names:
        wide[name].requires_grad_(case["train"])
    with torch.set_grad_enabled(case["train"]):
        outs = _exact_outputs(case, wide)
    if not case["train"]:
        return outs
    made = torch.autograd.grad(list(outs.values()), [wide[k] for k in names], grads)
    result = {k: v.detach() for k, v in outs.items()}
    result.update((k + "_grad", v) for k, v in zip(names, made))
    return result


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    tokens, d, train = case["tokens"], case["d"], case["train"]
    size = _TYPES[case["type"]].itemsize
    if case["kind"] == "dropout":
        return {"bytes": float(tokens * d * size * (4 if train else 2)), "flops": float(tokens * d * (2 if train else 1))}
    if case["kind"] == "norm":
        stream = 4 if case["residual"] and case["wide"] else size
        once = size + stream + (stream if case["residual"] else 0) + (size if case["pre"] else 0)  # branch, stream, residual, normed
        parts = 4 * (case["post"] + case["pre"]) + case["gate"] + 2 * (case["p"] > 0) + 2
        # in training a gradient comes or goes for each of them
        return {"bytes": float(tokens * d * once * (2 if train else 1)), "flops": float(tokens * d * parts * (3 if train else 1))}
    n, experts = case["n"], case.get("experts", 1)
    rows = tokens * case.get("top_k", 1)
    extra = rows * n * case.get("residual", False) + n * case.get("bias", False)
    if train:  # x, weight, grad, residual in; y, the gradients of x, weight and residual out
        return {"bytes": float(size * (2 * rows * (d + n) + 2 * experts * n * d + 2 * extra)), "flops": 6.0 * rows * d * n}
    used = experts * (1.0 - (1.0 - 1.0 / experts) ** rows) if experts > 1 else 1.0  # experts that have a row
    return {"bytes": float(size * (rows * (d + n) + used * n * d + extra)), "flops": 2.0 * rows * d * n}
