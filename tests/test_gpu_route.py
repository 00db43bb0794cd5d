"""Routing to experts against the 64-bit oracle, its gradient, and routers with their experts."""

import math

import pytest
import torch

from olmo_core_amd.nn import DroplessMoE, DroplessMoEMLP, MoERouter, ParallelDroplessMLP
from olmo_core_amd.ops.moe import route
from oracle import route_oracle as R

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# float32 of a score: the difference to the largest logit is off by 2^-24 of itself (at most 40 here), exp, division and multiplications
# by a unit in the last place or two each, a sum of positive terms over 16 lanes by their number of additions (at most 36)
REL = (40 + 36 + 8) * 2.0 ** -24


def make(tokens, experts, seed, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, experts, generator=g) * std).to(dtype)


def check(dev, logits, top_k, grad=True, **kw):
    want_w, want_i, want_n = R.route(logits, top_k, **kw)
    d = dict(kw)
    if d.get("bias") is not None:
        d["bias"] = d["bias"].to(dev)
    l = logits.to(dev).requires_grad_(grad)
    w, i, n = route(l, top_k, **d)
    assert w.dtype == F32 and i.dtype == n.dtype == torch.int64
    assert torch.equal(i.cpu(), want_i) and torch.equal(n.cpu(), want_n)
    err = (w.detach().cpu().double() - want_w).abs()
    assert bool((err <= want_w.abs() * REL + 1e-38).all()), float((err / want_w.abs().clamp(min=1e-30)).max())
    if not grad:
        return
    g = make(logits.shape[0], top_k, 99)
    w.backward(g.to(dev))
    args = {k: kw[k] for k in ("gating", "normalize", "scale") if k in kw}
    want = R.grad(logits, want_i, g, **args)
    # a gradient is a difference of products of weights: off by their errors and one rounding of the logits' type
    bound = want.abs() * (torch.finfo(logits.dtype).eps / 2) * 1.01 + 4 * REL * (want_w * g.abs().double()).sum(-1, keepdim=True) + torch.finfo(logits.dtype).tiny
    assert l.grad.dtype == logits.dtype
    err = (l.grad.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 12, 3), (48, 64, 8), (130, 60, 4), (300, 33, 5), (129, 128, 8), (200, 256, 8), (70, 257, 20), (40, 512, 64)]


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,experts,top_k", SHAPES)
def test_route(dev, tokens, experts, top_k, dtype, gating, normalize):
    check(dev, make(tokens, experts, 1, dtype, 2.0), top_k, gating=gating, normalize=normalize, scale=2.5 if normalize else 1.0)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,experts,top_k", SHAPES)
def test_bias(dev, tokens, experts, top_k, dtype, gating):
    bias = make(1, experts, 2, std=0.05)[0]
    check(dev, make(tokens, experts, 3, dtype), top_k, gating=gating, bias=bias, normalize=True)


GROUPS = [(64, 8, 8, 3), (256, 8, 8, 4), (64, 6, 4, 1), (60, 4, 5, 2), (24, 3, 8, 4), (96, 8, 32, 20), (512, 10, 16, 2), (48, 2, 3, 3), (16, 1, 16, 5)]


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("experts,top_k,groups,kept", GROUPS)
def test_groups(dev, experts, top_k, groups, kept, dtype, gating, biased):
    bias = make(1, experts, 4, std=0.05)[0] if biased else None
    check(dev, make(150, experts, 5, dtype), top_k, gating=gating, bias=bias, groups=groups, groups_kept=kept, normalize=True, scale=1.5)


def test_ties_go_to_the_lowest_index(dev):
    for gating in ("softmax", "sigmoid"):
        for kw in (dict(), dict(bias=torch.full((64,), 0.25)), dict(groups=8, groups_kept=3)):
            check(dev, torch.zeros(140, 64), 8, gating=gating, **kw)
            check(dev, make(140, 64, 6).sign(), 8, gating=gating, **kw)
            check(dev, make(140, 64, 6).mul(2).round(), 8, gating=gating, **kw)


def test_neighbours_closer_than_float32(dev):
    """Scores that float32 cannot order: logits and biases whose sums agree in 30 bits and more."""
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(256, 64, generator=g) * 0.5
    s = torch.sigmoid(logits.double())
    # the bias (float32) brings every expert of the first row near the same value
    bias = (0.75 - s[0]).float()
    logits[1:128] = logits[0]
    check(dev, logits, 8, gating="sigmoid", bias=bias)
    check(dev, logits, 8, gating="sigmoid", bias=bias, groups=8, groups_kept=4)
    check(dev, logits, 8, gating="softmax", bias=(0.5 - R.scores(logits[:1], "softmax")[0]).float())


@pytest.mark.parametrize("experts", [64, 128, 256, 257, 512])
def test_long_sums_beside_a_bias(dev, experts):
    """One expert that has almost everything, others of less than half a unit in the last place of its score, which a sum in one go loses one by one, and
    a bias that brings another expert next to it.  The float32 scores may be off by some thirty 2^-24 here; the ids are those of 64 bits."""
    u = 2.0 ** -24
    few = -(-experts // 16)  # experts of a lane
    for some in (few, experts):
        for at in {1, few, experts - 1}:
            rows = torch.full((33, experts), -40.0)
            rows[:, 1:some] = math.log(0.98 * u)
            rows[:, 0] = torch.arange(33) * 2.0 ** -9
            s = R.scores(rows, "softmax")
            for lead in (-40, -20, -8, -3, -1, 1, 3, 8, 20, 40):
                bias = torch.zeros(experts)
                bias[at] = float(s[0, 0] - s[0, at] + lead * u)
                check(dev, rows, 1, grad=False, bias=bias)
                check(dev, rows, min(8, experts), grad=False, bias=bias, normalize=True)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_infinite_logits(dev, gating, groups):
    kept = 2 if groups > 1 else 1
    l = make(20, 32, 8)
    l[0] = -math.inf
    l[1, 3:] = -math.inf
    l[2, ::2] = -math.inf
    l[3, 5] = torch.finfo(F32).min
    l[4] = torch.finfo(F32).min
    check(dev, l, 6, grad=False, gating=gating, normalize=True, groups=groups, groups_kept=kept)
    check(dev, l, 6, grad=False, gating=gating, bias=make(1, 32, 9)[0], groups=groups, groups_kept=kept)
    bias = make(1, 32, 9)[0]
    bias[7] = -math.inf
    check(dev, l[5:], 6, gating=gating, bias=bias)


def test_scores_below_the_normal_range(dev):
    """Chosen scores of less than 2^-126 (sigmoid of -88 and less, a softmax of which only the far end is chosen) still have weights that add up to one, and a
    gradient; where all of them are below 2^-1024 the weights are zero."""
    g = torch.Generator().manual_seed(30)
    l = torch.full((6, 40), -300.0)
    l[0, [3, 7, 30]] = torch.tensor([-90.0, -95.0, -91.5])
    l[1, [0, 39, 20]] = torch.tensor([-87.0, -88.5, -60.0])
    l[2] = -100 - 20 * torch.rand(40, generator=g)
    l[3] = -300 - 2 * torch.rand(40, generator=g)
    l[4, [1, 2, 3]] = torch.tensor([-20.0, -45.0, -55.0])
    l[5, [1, 2, 3]] = torch.tensor([5.0, 4.0, -20.0])
    for top_k in (2, 3):
        check(dev, l, top_k, gating="sigmoid", normalize=True, scale=2.5)
    check(dev, l[2:4], 20, gating="sigmoid", normalize=True)
    check(dev, l[2:4], 8, gating="sigmoid", normalize=True, groups=4, groups_kept=2)
    check(dev, l[2:4].to(BF16), 8, gating="sigmoid", normalize=True)
    # the chosen experts are those of the bias, far below the largest logit
    l = torch.randn(5, 64, generator=g) - 95.0
    l[:, 0] = 0.0
    l[1, :32] = -600.0
    l[1, 0] = 0.0
    bias = torch.zeros(64)
    bias[40:60] = 2.0 + torch.arange(20) * 0.125
    check(dev, l, 4, gating="softmax", bias=bias, normalize=True)
    check(dev, l, 18, gating="softmax", bias=bias, normalize=True)
    low = torch.full((2, 40), -715.0)
    low[1] = -800.0
    w = route(low.to(dev).requires_grad_(True), 3, gating="sigmoid", normalize=True)[0]
    assert not w.any()
    check(dev, torch.full((1, 40), -700.0), 3, grad=False, gating="sigmoid", normalize=True)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
def test_nan_logits_leave_the_others_alone(dev, gating):
    l = make(40, 64, 10)
    clean = l.clone()
    l[7, 3], l[9] = math.nan, math.nan
    l[11, 20] = math.inf
    for kw in (dict(), dict(bias=make(1, 64, 11)[0].to(dev)), dict(groups=8, groups_kept=2)):
        w, i, n = route(l.to(dev), 8, gating=gating, normalize=True, **kw)
        w2, i2, _ = route(clean.to(dev), 8, gating=gating, normalize=True, **kw)
        rest = torch.ones(40, dtype=torch.bool, device=dev)
        rest[[7, 9, 11]] = False
        assert torch.equal(w[rest], w2[rest]) and torch.equal(i[rest], i2[rest])
        assert int(n.sum()) == 320 and bool((i >= 0).all()) and bool((i < 64).all())
        assert all(len(set(row)) == 8 for row in i.tolist())


def test_gradient_against_differences(dev):
    """Central differences of the float32 weights along a direction: with h = 2^-7 the second-order term of functions whose derivatives up to the
    third are at most 1 is h^2 / 6 of the direction's size, the rounding of the weights 2^-24 / h."""
    for gating in ("softmax", "sigmoid"):
        for normalize in (False, True):
            l = make(64, 32, 12).to(dev).requires_grad_(True)
            g, d = make(64, 4, 13).to(dev), make(64, 32, 14).to(dev)
            w, i, _ = route(l, 4, gating=gating, normalize=normalize)
            w.backward(g)
            h = 2.0 ** -7

            def weights(at):  # of the experts chosen at l
                s = torch.softmax(at, -1) if gating == "softmax" else torch.sigmoid(at)
                s = s.gather(1, i)
                return s / s.sum(-1, keepdim=True) if normalize else s

            at = l.detach().double()
            diff = ((weights(at + h * d) - weights(at - h * d)) * g.double()).sum(-1) / (2 * h)
            along = (l.grad.double() * d.double()).sum(-1)
            size = (g.abs().sum(-1) * d.abs().amax(-1) ** 3).double()
            assert bool(((diff - along).abs() <= size * (h * h + 2.0 ** -16)).all())


def test_shapes_and_empty(dev):
    l = make(24, 16, 15).to(dev)
    w, i, n = route(l, 2)
    w3, i3, n3 = route(l.view(2, 3, 4, 16), 2)
    assert w3.shape == (2, 3, 4, 2) and torch.equal(w3.view(24, 2), w) and torch.equal(i3.view(24, 2), i) and torch.equal(n, n3)
    wt, it, _ = route(l.t().contiguous().t(), 2)
    assert torch.equal(w, wt) and torch.equal(i, it)
    w, i, n = route(l[:0].requires_grad_(True), 2)
    w.sum().backward()
    assert w.shape == (0, 2) and not n.any()


def test_captured_and_replayed(dev):
    for tokens in (48, 700):
        l = make(tokens, 64, 16).to(dev).requires_grad_(True)
        g = make(tokens, 8, 17).to(dev)
        bias = make(1, 64, 18, std=0.1)[0].to(dev)

        def work():
            w, i, n = route(l, 8, gating="sigmoid", bias=bias, groups=8, groups_kept=4, normalize=True)
            return w.detach(), i, n, *torch.autograd.grad(w, l, g)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
        for seed in (19, 20, 21):
            with torch.no_grad():
                l.copy_(make(tokens, 64, seed))
            eager = work()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals(dev):
    l = make(4, 64, 22).to(dev)
    for bad in (dict(top_k=0), dict(top_k=65), dict(groups=7), dict(groups=0), dict(groups=8, groups_kept=9), dict(groups=8, groups_kept=0),
                dict(top_k=9, groups=8, groups_kept=1), dict(gating="relu"), dict(bias=torch.zeros(63, device=dev)),
                dict(bias=torch.zeros(64)), dict(bias=torch.zeros(64, dtype=torch.int32, device=dev))):
        with pytest.raises(ValueError):
            route(l, **{"top_k": 8, **bad})
    with pytest.raises(ValueError):
        route(make(1, 513, 1).to(dev), 8)
    with pytest.raises(TypeError):
        route(l.int(), 8)


# ---- routers with their experts ------------------------------------------------------------------------------------------


def layer(dev, scaling, d=256, h=144, experts=8, top_k=2, **kw):
    torch.manual_seed(3)
    mlp = DroplessMoEMLP(d_model=d, hidden_size=h, num_experts=experts, dtype=BF16, init_device=dev, scaling=scaling)
    router = MoERouter(d_model=d, num_experts=experts, top_k=top_k, dtype=BF16, init_device=dev, **kw)
    with torch.no_grad():
        router.weight.mul_(5)
    return DroplessMoE(router=router, experts=ParallelDroplessMLP(mlp=mlp, top_k=top_k))


@pytest.mark.parametrize("scaling", ["rowwise", "blockwise"])
@pytest.mark.parametrize("tokens", [1, 70, 300])
def test_routed_layer(dev, scaling, tokens):
    """The layer against its formula in float64 on the same routing: activations and weights rounded to float8 (2^-4 of a value at most, about
    0.03 of it on average) three times in a row, so the norm of the error is below a tenth.  The router's gradient is another matter: with p_j = g . z_j
    for the outputs z_1, z_2 of a token's experts, dl_1 = w_1 w_2 (1 - s_1) (p_1 - p_2), a difference in which p_j is off by up to a tenth of |g| |z_j|
    however small it is itself; so dl_1 is off by w_1 w_2 (1 - s_1) |g| (|z_1| + |z_2|) / 10, and likewise dl_2."""
    moe = layer(dev, scaling, gating="sigmoid", normalize=True, groups=4, groups_kept=2, bias_gamma=0.01)
    x = make(tokens, 256, 23, BF16).to(dev).requires_grad_(True)
    y = moe(x)
    g = make(tokens, 256, 24, BF16).to(dev)
    y.backward(g)
    grads = [x.grad, *(p.grad for p in moe.parameters())]
    assert all(t is not None and bool(torch.isfinite(t.float()).all()) for t in grads)

    xd = x.detach().double().requires_grad_(True)
    ps = [p.detach().double().requires_grad_(True) for p in moe.parameters()]
    names = dict(zip((n for n, _ in moe.named_parameters()), ps))
    with torch.no_grad():
        _, idx, sizes = moe.router(x.detach())
    assert int(sizes.sum()) == 2 * tokens
    s = torch.sigmoid(xd @ names["router.weight"].t()).gather(1, idx)
    w = s / s.sum(-1, keepdim=True)
    w1, w2, w3 = (names[f"experts.mlp.w{i}"].view(8, 144, 256) for i in (1, 2, 3))
    parts = []
    for j in range(2):
        e = idx[:, j]
        a = torch.matmul(w1[e].float().double(), xd.unsqueeze(-1)).squeeze(-1)
        b = torch.matmul(w3[e].float().double(), xd.unsqueeze(-1)).squeeze(-1)
        h = torch.nn.functional.silu(a) * b
        parts.append(torch.matmul(h.unsqueeze(1), w2[e]).squeeze(1))
    ref = w[:, :1] * parts[0] + w[:, 1:] * parts[1]
    with torch.no_grad():
        off = 0.1 * w.prod(-1, keepdim=True) * (1 - s) * g.double().norm(dim=-1, keepdim=True) * sum(z.norm(dim=-1, keepdim=True) for z in parts)
        off = off.norm(dim=-1)  # of a token's two logits
        extra = {"router.weight": float((off * xd.norm(dim=-1)).sum()), "x": float(off.norm() * names["router.weight"].norm())}
    ref.backward(g.double())
    for got, want, what in zip([y.detach(), *grads], [ref.detach(), xd.grad, *(p.grad for p in ps)], ["y", "x", *(n for n, _ in moe.named_parameters())]):
        err = float((got.double() - want).norm())
        assert err < 0.1 * float(want.norm()) + extra.get(what, 0.0), (what, err, float(want.norm()))


def test_blockwise_layer_is_its_parts(dev):
    """Kept weights, gathered and scattered slots: the bits of the operators called one by one."""
    from olmo_core_amd.float8 import blockwise_grouped_linear
    from olmo_core_amd.nn import swiglu
    from olmo_core_amd.ops import moe as moe_ops

    moe = layer(dev, "blockwise")
    x = make(90, 256, 25, BF16).to(dev)
    with torch.no_grad():
        w, idx, sizes = moe.router(x)
        y = moe(x)
        moe.experts.mlp.keep_float8_weights = True
        assert torch.equal(moe(x), y) and moe.experts.mlp.weight_operands() is moe.experts.mlp.weight_operands()
        indices, bin_ids, bins = moe_ops._sort_slots(idx.flatten(), sizes)
        xs = moe_ops.gather(x, indices, bin_ids, bins, 2)
        m = moe.experts.mlp
        h = swiglu(blockwise_grouped_linear(xs, m.w1, sizes), blockwise_grouped_linear(xs, m.w3, sizes))
        z = blockwise_grouped_linear(h, m.w2, sizes, transposed=True)
        assert torch.equal(y, moe_ops.scatter(z, indices, bin_ids, w.flatten(), bins, 2))
    with pytest.raises(NotImplementedError):
        m.forward_gathered(x, indices, 2, sizes)


@pytest.mark.parametrize("scaling", ["blockwise"])
def test_layer_of_no_tokens(dev, scaling):
    moe = layer(dev, scaling)
    x = torch.empty(0, 256, dtype=BF16, device=dev, requires_grad=True)
    y = moe(x)
    assert y.shape == (0, 256)
    y.sum().backward()
    assert x.grad.shape == (0, 256) and all(not p.grad.any() for p in moe.experts.parameters())


def test_compiled_router_breaks_the_graph(dev):
    router = MoERouter(d_model=64, num_experts=8, top_k=2, init_device=dev)
    x = make(30, 64, 27).to(dev)
    for a, b in zip(torch.compile(router, backend="eager")(x), router(x)):
        assert torch.equal(a, b)


def test_bias_evens_out_the_load(dev):
    router = MoERouter(d_model=64, num_experts=8, top_k=2, gating="sigmoid", bias_gamma=0.05, init_device=dev)
    x = make(512, 64, 26).to(dev)
    before = router.score_bias.clone()
    sizes = router(x)[2]
    router.post_batch()
    load = sizes.float()
    assert torch.allclose(router.score_bias - before, 0.05 * torch.sign(load.mean() - load))
    assert not router.slots_since.any()
    router.eval()
    router(x)
    assert not router.slots_since.any()

@pytest.mark.parametrize("scaling", ["rowwise", "blockwise"])
def test_layer_of_strided_tokens(dev, scaling):
    """Tokens of any leading shape, also one that cannot be flattened without a copy."""
    moe = layer(dev, scaling)
    x = make(35, 256, 28, BF16).view(5, 7, 256).to(dev)
    g = make(35, 256, 29, BF16).view(7, 5, 256).to(dev)
    a, b = x.transpose(0, 1).requires_grad_(True), x.transpose(0, 1).contiguous().requires_grad_(True)
    ya, yb = moe(a), moe(b)
    assert ya.shape == (7, 5, 256) and torch.equal(ya, yb)
    assert torch.equal(torch.autograd.grad(ya, a, g)[0], torch.autograd.grad(yb, b, g)[0])
