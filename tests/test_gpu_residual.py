"""
Products, norms and dropout of a model's own type as they are used together: blocks on a residual stream.

The values of a chain are compared with the same chain in 64 bits, which is computed twice: exactly, and with every output and every gradient rounded where the
operators round theirs.  The errors of the rounded chain and of the kernels are sums of as many independent roundings of the same sizes, so their norms over
thousands of elements are about the same; twice the rounded chain's error is the bound.
"""

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
import torch.utils.checkpoint

from olmo_core_amd.nn import DroplessMoE, DroplessMoEMLP, FeedForward, MoERouter, ParallelDroplessMLP, ResidualBlocks, ResidualNorm, swiglu
from olmo_core_amd.ops import moe as moe_ops
from olmo_core_amd.ops.dropout import dropout
from olmo_core_amd.ops.linear import grouped_linear, linear
from olmo_core_amd.ops.norm import residual_norm

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Dense(nn.Module):
    """Two linears, an activation between them."""

    def __init__(self, d, h, dtype, activation):
        super().__init__()
        self.activation = activation
        self.w1, self.b1 = nn.Parameter(torch.randn(h, d, dtype=dtype) / d ** 0.5), nn.Parameter(torch.randn(h, dtype=dtype) / 4)
        self.w2, self.b2 = nn.Parameter(torch.randn(d, h, dtype=dtype) / h ** 0.5), nn.Parameter(torch.randn(d, dtype=F32) / 4)

    def forward(self, x):
        return linear(linear(x, self.w1, self.b1, activation=self.activation), self.w2, self.b2)


class Sorted(nn.Module):
    """Experts on rows that are sorted already."""

    def __init__(self, d, h, sizes, dtype):
        super().__init__()
        self.mlp = DroplessMoEMLP(d_model=d, hidden_size=h, num_experts=len(sizes), dtype=dtype, scaling="none")
        self.register_buffer("sizes", torch.tensor(sizes))

    def forward(self, x):
        return self.mlp(x, self.sizes)


class Round(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dtype):
        ctx.dtype = dtype
        return x.to(dtype).double()

    @staticmethod
    def backward(ctx, g):
        return g.to(ctx.dtype).double(), None


def _plain(model, head, x, p, seed, norm, dtype, stream_dtype, rounded):
    """The chain in 64 bits."""
    r = (lambda t, dt=dtype: Round.apply(t, dt)) if rounded else (lambda t, dt=dtype: t)
    params = {n: v.detach().double().requires_grad_(True) for n, v in list(model.named_parameters()) + [("head", head)]}

    def normed(a, w):
        return a * torch.rsqrt((a * a).mean(-1, keepdim=True) + 1e-6) * w if w is not None else a

    def mask(like, offset):
        return dropout(torch.ones(like.shape, device="cuda"), p, seed=seed, offset=offset).double()

    x = x.detach().double().requires_grad_(True)
    stream = r(x * mask(x, 99), stream_dtype)
    get = lambda i, name: params.get(f"joins.{i}.{name}")  # noqa: E731
    into = r(r(normed(stream, get(0, "pre_weight")), stream_dtype)) if norm != "after" else r(stream)
    for i, block in enumerate(model.blocks):
        w = {n.split(".")[-1]: v for n, v in params.items() if n.startswith(f"blocks.{i}.")}
        if isinstance(block, Dense):
            act = {"silu": F.silu, "gelu": F.gelu}[block.activation]
            y = r(r(act(into @ w["w1"].t() + w["b1"])) @ w["w2"].t() + w["b2"])
        else:
            sizes, parts = block.sizes.tolist(), []
            e_w = [w[k].view(len(sizes), -1, into.shape[1]) for k in ("w1", "w2", "w3")]
            for e, rows in enumerate(into.split(sizes)):
                w1, w2, w3 = (v[e] for v in e_w)
                a, b = r(rows @ w1.t()), r(rows @ w3.t())
                h = r(F.silu(a)) * b if dtype == F16 else F.silu(a) * b
                parts.append(r(r(h) @ w2))
            y = torch.cat(parts)
        stream = stream + get(i + 1, "gate") * mask(stream, i) * normed(y, get(i + 1, "post_weight"))
        n = normed(stream, get(i + 1, "pre_weight"))
        stream = r(stream, stream_dtype)
        last = i == len(model.blocks) - 1
        into = r(n) if get(i + 1, "pre_weight") is not None else stream if last else r(stream)
    out = r(r(into, dtype) @ params["head"].t())
    return x, params, out


CASES = [("before", BF16, F32, 0.0), ("before", BF16, BF16, 0.1), ("after", BF16, F32, 0.1), ("both", F16, F16, 0.2), ("both", F16, F32, 0.0)]


def _chain(norm, dtype, stream_dtype, p, d=136, rows=307):
    torch.manual_seed(5)
    sizes = [100, 0, 7, rows - 107]
    model = ResidualBlocks(
        [Dense(d, 333, dtype, "silu"), Sorted(d, 72, sizes, dtype), Dense(d, 256, dtype, "gelu")], d_model=d, norm=norm, gate=0.5, dropout=p, block_dtype=dtype)
    with torch.no_grad():
        for w in model.joins.parameters():
            w.add_(torch.randn_like(w) / 8)
    head = nn.Parameter((torch.randn(91, d) / d ** 0.5).to(dtype).cuda())
    return model.cuda(), head, torch.randn(rows, d).to(stream_dtype).cuda(), torch.randn(rows, 91).to(dtype).cuda()


def _run(model, head, x, p, seed):
    return linear(model(dropout(x, p, seed=seed, offset=99), seed=seed).to(head.dtype), head)


@pytest.mark.parametrize("norm,dtype,stream_dtype,p", CASES, ids=lambda v: str(v).removeprefix("torch."))
def test_chain_of_blocks(norm, dtype, stream_dtype, p):
    model, head, x, g = _chain(norm, dtype, stream_dtype, p)
    x.requires_grad_(True)
    out = _run(model, head, x, p, 17)
    names, params = zip(*model.named_parameters())
    made = [out, *torch.autograd.grad(out, [x, head, *params], g)]
    want = {}
    for rounded in (False, True):
        px, ps, po = _plain(model, head, x, p, 17, norm, dtype, stream_dtype, rounded)
        want[rounded] = [po, *torch.autograd.grad(po, [px, ps["head"], *(ps[n] for n in names)], g.double())]
        assert set(ps) == {*names, "head"}
    for name, got, exact, rounded in zip(("out", "x", "head", *names), made, want[False], want[True]):
        assert got.dtype == (dtype if name in ("out", "head") or "blocks" in name and not name.endswith("b2") else stream_dtype if name == "x" else F32)
        ours, allowed = (got.double() - exact).norm(), (rounded - exact).norm() + torch.finfo(got.dtype).eps / 2 * exact.norm()
        assert ours <= 2 * allowed, f"{name}: {float(ours)} for {float(allowed)}"
        assert allowed < 0.1 * exact.norm(), name  # (the bound says something)


@pytest.mark.parametrize("norm,dtype,stream_dtype,p", CASES[:3], ids=lambda v: str(v).removeprefix("torch."))
def test_chain_is_its_calls(norm, dtype, stream_dtype, p):
    """The modules add nothing to the operators' bits; without gradients the same, in evaluation no dropout."""
    model, head, x, g = _chain(norm, dtype, stream_dtype, p)
    with torch.no_grad():
        got = model(x, seed=3)
        assert torch.equal(got, model(x, seed=3))
        joins = model.joins
        stream, normed = residual_norm(x, pre_weight=joins[0].pre_weight) if joins[0].pre_weight is not None else (x, None)
        for i, block in enumerate(model.blocks):
            y = block((stream if normed is None else normed).to(dtype))
            j = joins[i + 1]
            stream, normed = residual_norm(y, stream, post_weight=j.post_weight, pre_weight=j.pre_weight, gate=j.gate, p=p, seed=3, offset=i)
        assert torch.equal(got, normed)
        model.eval()
        assert torch.equal(model(x), model(x, seed=9))
        model.train()
        torch.manual_seed(1)
        a = model(x)
        torch.manual_seed(1)
        assert torch.equal(a, model(x)) and (p == 0 or not torch.equal(a, model(x)))
    assert torch.equal(_run(model, head, x, p, 4).detach(), _run(model, head, x.requires_grad_(True), p, 4).detach())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_captured_and_replayed(dtype):
    """Forward and backward of the whole chain in one graph, on a seed and inputs that change between the replays."""
    model, head, x, g = _chain("both", dtype, F32, 0.1)
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    x.requires_grad_(True)
    leaves = [x, head, *model.parameters()]

    def step():
        out = _run(model, head, x, 0.1, seed)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(warm, step()):
        assert torch.equal(a, b)
    del warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        seed.fill_(i)
        with torch.no_grad():
            x.mul_(1.25)
            head.mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want)


def test_drawn_seed_is_refused_in_a_graph():
    join = ResidualNorm(d_model=64, pre_norm=True, dropout=0.1).cuda()
    x = torch.randn(8, 64, device="cuda")
    with torch.no_grad():
        join(x, x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="seed on the GPU"):
                join(x, x)
            y = join(x, x, seed=torch.ones(1, dtype=torch.int64, device="cuda"))[1]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, join(x, x, seed=1)[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,d,h", [(1, 256, 144), (70, 136, 72), (300, 96, 40)])
def test_routed_experts_without_scaling(dtype, tokens, d, h):
    """The layer is its router, the permutation and the experts, bit for bit; against 64 bits on the same routing its roundings (of x1, x3, h, the product and its
    weighted sum, at most half a step each, the first three through one or two products) stay below five steps of the type in norm."""
    torch.manual_seed(3)
    mlp = DroplessMoEMLP(d_model=d, hidden_size=h, num_experts=8, dtype=dtype, init_device="cuda", scaling="none")
    router = MoERouter(d_model=d, num_experts=8, top_k=2, dtype=dtype, init_device="cuda", normalize=True)
    moe = DroplessMoE(router=router, experts=ParallelDroplessMLP(mlp=mlp, top_k=2))
    x = torch.randn(tokens, d, device="cuda").to(dtype).requires_grad_(True)
    y = moe(x)
    assert y.dtype == dtype
    grads = torch.autograd.grad(y, [x, *moe.parameters()], torch.randn_like(y))
    assert all(bool(torch.isfinite(t.float()).all()) for t in grads)
    with torch.no_grad():
        weights, idx, sizes = moe.router(x)
        indices, bin_ids, bins = moe.experts.indices_and_bins(idx.flatten(), sizes)
        rows = moe_ops.gather(x, indices, bin_ids, bins, 2)
        a, b = grouped_linear(rows, mlp.w1, sizes), grouped_linear(rows, mlp.w3, sizes)
        z = grouped_linear(swiglu(a, b) if dtype == BF16 else F.silu(a) * b, mlp.w2, sizes, transposed=True)
        assert torch.equal(y, moe_ops.scatter(z, indices, bin_ids, weights.flatten(), bins, 2))
        w1, w2, w3 = (w.double().view(8, h, d) for w in (mlp.w1, mlp.w2, mlp.w3))
        want = torch.zeros(tokens, d, dtype=torch.float64, device="cuda")
        for j in range(2):
            for t in range(tokens):
                e = int(idx[t, j])
                xt = x[t].double()
                want[t] += weights[t, j].double() * ((F.silu(w1[e] @ xt) * (w3[e] @ xt)) @ w2[e])
        assert (y.double() - want).norm() <= 5 * torch.finfo(dtype).eps * want.norm()


def test_experts_of_any_size_and_master_weights():
    """Sizes that are no multiples of anything, float32 weights and inputs, no rows."""
    torch.manual_seed(2)
    mlp = DroplessMoEMLP(d_model=37, hidden_size=21, num_experts=3, init_device="cuda", scaling="none")
    sizes = torch.tensor([4, 0, 5], device="cuda")
    x = torch.randn(9, 37, device="cuda", requires_grad=True)
    y = mlp(x, sizes)
    assert y.dtype == F32 and y.shape == x.shape
    y.sum().backward()
    assert all(w.grad.dtype == F32 and bool(torch.isfinite(w.grad).all()) for w in mlp.parameters())
    assert not mlp.w1.grad[21:42].any() and mlp.w1.grad[:21].any()
    half = DroplessMoEMLP(d_model=37, hidden_size=21, num_experts=3, dtype=BF16, init_device="cuda", scaling="none")
    half.load_state_dict(mlp.state_dict())
    assert torch.equal(half(x.detach().to(BF16), sizes).float(), y.detach())
    empty = mlp(x.detach()[:0], torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert empty.shape == (0, 37)


def test_feed_forward_on_the_stream():
    """The blocks that the framework has already stand on the stream as they are."""
    torch.manual_seed(4)
    model = ResidualBlocks([FeedForward(d_model=64, hidden_size=128, bias=False, dtype=BF16) for _ in range(2)], d_model=64, block_dtype=BF16).cuda()
    x = torch.randn(2, 33, 64, device="cuda", requires_grad=True)
    y = model(x)
    assert y.shape == x.shape and y.dtype == BF16
    y.float().square().sum().backward()
    assert x.grad is not None and bool(torch.isfinite(x.grad).all())
    assert all(p.grad is not None for p in model.parameters())


def _calls():
    x = torch.randn(12, 24, device="cuda").to(BF16).requires_grad_(True)
    w = torch.randn(40, 24, device="cuda").to(BF16).requires_grad_(True)
    sizes = torch.tensor([5, 7], device="cuda")
    return x, {
        "linear": lambda t: linear(t, w, activation="silu"),
        "grouped_linear": lambda t: grouped_linear(t, w, sizes),
        "residual_norm": lambda t: residual_norm(t, t, post_norm=True, pre_norm=True)[1],
        "dropout": lambda t: dropout(t, 0.5, seed=1),
    }


@pytest.mark.parametrize("name", ["linear", "grouped_linear", "residual_norm", "dropout"])
def test_only_first_derivatives_in_reverse(name):
    """A second derivative, forward mode and a transform are refused, and not taken for zero."""
    x, calls = _calls()
    y = calls[name](x)
    torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    # a graph that is recomputed runs in a mode where gradients are on
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    again = torch.utils.checkpoint.checkpoint(calls[name], x, use_reentrant=True)
    again.backward(torch.ones_like(again))
    assert torch.equal(x.grad, g)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            calls[name](dual)
    with pytest.raises(RuntimeError):
        torch.func.vmap(calls[name])(x.detach().expand(3, 12, 24))


def test_under_torch_compile():
    """The calls are breaks of the traced graph: the same bits as without, forward and backward, and a mask that is drawn anew on every call."""
    torch.manual_seed(6)
    model = ResidualBlocks([Dense(64, 96, BF16, "silu"), Sorted(64, 40, [20, 0, 13], BF16)], d_model=64, norm="both", gate=0.5, dropout=0.2, block_dtype=BF16).cuda()
    x, g = torch.randn(33, 64, device="cuda", requires_grad=True), torch.randn(33, 64, device="cuda").to(BF16)
    traced = torch.compile(model, backend="eager")
    for seed in (3, torch.tensor([4], device="cuda")):
        want, got = model(x, seed=seed), traced(x, seed=seed)
        assert torch.equal(got, want)
        for a, b in zip(*(torch.autograd.grad(y, [x, *model.parameters()], g) for y in (got, want))):
            assert torch.equal(a, b)
    with torch.no_grad():
        drawn = [traced(x) for _ in range(4)]
        assert all(not torch.equal(drawn[i], drawn[j]) for i in range(4) for j in range(i))
        torch.manual_seed(9)
        a = model(x)
        torch.manual_seed(9)
        assert torch.equal(traced(x), a)


def test_chains_that_share_a_seed():
    """Two chains on one seed tensor take different masks where their offsets differ by at least a chain's number of blocks, which is how many offsets it uses."""
    torch.manual_seed(8)
    a = ResidualBlocks([nn.Identity() for _ in range(3)], d_model=64, final_norm=False, dropout=0.5, init_device="cuda")
    x = torch.randn(40, 64, device="cuda")
    seed = torch.tensor([77], device="cuda")
    with torch.no_grad():
        stream, normed = a.joins[0](x)
        for i in range(3):
            stream, normed = a.joins[i + 1](normed, stream, seed=seed, offset=5 + i)
        assert torch.equal(a(x, seed=seed, offset=5), stream)
        assert torch.equal(a(x, seed=seed), a(x, seed=seed, offset=0))
        masks = []

        class Ones(nn.Module):  # (what is dropped of it is what the mask drops)
            def forward(self, into):
                return torch.ones_like(into)

        for offset in (0, 2, 4):
            chain = ResidualBlocks([Ones(), Ones()], d_model=64, norm="after", final_norm=False, dropout=0.5, init_device="cuda")
            zero = torch.zeros(40, 64, device="cuda")
            for i in range(2):
                masks.append(residual_norm(zero + 1, p=0.5, seed=seed, offset=offset + i)[0] != 0)
            assert torch.equal(chain(zero, seed=seed, offset=offset) != 0, masks[-2] | masks[-1])
        assert all(not torch.equal(p, q) for i, p in enumerate(masks) for q in masks[:i])
