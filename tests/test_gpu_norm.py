"""
``ops.norm.residual_norm`` and ``ops.dropout.dropout`` against the formulas in 64 bits.

Bounds (:func:`_want`) are carried along with the values: a float32 operation is off by 2^-24 of its result, a sum over n by n 2^-24 of the sum of magnitudes, the
reciprocal square root by 2^-22, and the backward's normed stream by half a step of the type that the stream is stored in.  Outputs are rounded once, by half a
step of their type.
"""

import math

import pytest
import torch

from olmo_core_amd import _C
from olmo_core_amd.ops.dropout import dropout
from olmo_core_amd.ops.norm import MOST_FEATURES, residual_norm

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5


def philox_kept(count, p, seed, offset):
    """Truth values of ``count`` elements, the generator written with Python's integers (and numpy for many of them)."""
    import numpy as np

    u64 = np.uint64
    low = u64(0xFFFFFFFF)
    i = np.arange((count + 7) // 8, dtype=u64)
    c = [i & low, i >> u64(32), np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(7):
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(b >> u64(32)) ^ c[1] ^ u64(k[0]), b & low, (a >> u64(32)) ^ c[3] ^ u64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack([h for w in c for h in (w & u64(0xFFFF), w >> u64(16))], -1).reshape(-1)[:count]
    return torch.from_numpy(halves >= round(65536 * p)).cuda()


def factor(p):
    t = round(65536 * p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- dropout -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7,), 0.3), ((8,), 0.3), ((3, 5, 11), 0.1), ((1000, 8), 0.25), ((777, 1031), 0.9), ((600, 4096), 0.1), ((40,), 0.0), ((40,), 1.0)])
def test_dropout(dtype, shape, p):
    g = _gen(math.prod(shape))
    seed, offset = 0x123456789ABCDEF0, 0xFEDCBA987
    x = torch.randn(shape, generator=g).to(dtype).cuda().requires_grad_(True)
    gy = torch.randn(shape, generator=g).to(dtype).cuda()
    y = dropout(x, p, seed=seed, offset=offset)
    gx = torch.autograd.grad(y, x, gy)[0]
    kept = philox_kept(x.numel(), p, seed, offset).view(shape)
    f = torch.tensor(factor(p), dtype=F32).item()
    for got, of in ((y, x.detach()), (gx, gy)):
        assert torch.equal(got, torch.where(kept, (of.float() * f), 0).to(dtype))


def test_dropout_masks_differ_by_seed_and_offset_and_keep_the_mean():
    x = torch.ones(1 << 20, device="cuda")
    masks = [dropout(x, 0.3, seed=s, offset=o) != 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 << 32, 0), (1, 1 << 32))]
    n, q = x.numel(), 1 - round(65536 * 0.3) / 65536
    for m in masks:
        assert abs(m.sum().item() - n * q) < 6 * math.sqrt(n * q * (1 - q))
    for i in range(len(masks)):
        for j in range(i):
            agree = (masks[i] == masks[j]).sum().item()
            expected = q * q + (1 - q) ** 2
            assert abs(agree - n * expected) < 6 * math.sqrt(n * expected * (1 - expected))
    # neighbours, and the elements of one call, are independent
    m = masks[0].float() - q
    for lag in (1, 2, 3, 4, 7, 8, 16):
        assert abs((m[lag:] * m[:-lag]).sum().item()) < 6 * math.sqrt(n) * q * (1 - q)
    per = masks[0].view(-1, 8).sum(0).float()
    assert ((per - n / 8 * q).abs() < 6 * math.sqrt(n / 8 * q * (1 - q))).all()


def test_dropout_of_views_and_not_finite_values():
    g = _gen(1)
    x = torch.randn(30, 50, generator=g).to(BF16).cuda()
    want = dropout(x, 0.5, seed=3)
    odd = torch.empty(30 * 50 + 1, dtype=BF16, device="cuda")[1:].view(30, 50).copy_(x)
    assert torch.equal(dropout(odd, 0.5, seed=3), want)
    assert torch.equal(dropout(x.t().contiguous().t(), 0.5, seed=3), want)
    assert dropout(x[:0], 0.5, seed=3).shape == (0, 50)
    kept = philox_kept(1500, 0.5, 3, 0).view(30, 50)
    bad = torch.where(kept, x, math.nan)
    assert torch.equal(dropout(bad, 0.5, seed=3), want)


def test_seed_on_the_gpu_and_captured():
    g = _gen(2)
    x = torch.randn(100, 72, generator=g).cuda().requires_grad_(True)
    gy = torch.randn(100, 72, generator=g).cuda()
    place = torch.tensor([5], device="cuda")
    want = {s: dropout(x.detach(), 0.4, seed=s, offset=9) for s in (5, 6, 7, 1 << 40)}
    assert torch.equal(dropout(x.detach(), 0.4, seed=place, offset=9), want[5])

    def step():
        y = dropout(x, 0.4, seed=place, offset=9)
        return y.detach(), torch.autograd.grad(y, x, gy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = step()
    for s in (5, 6, 7, 1 << 40):
        place.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[s])
        assert torch.equal(gx, dropout(gy, 0.4, seed=s, offset=9))
        assert torch.equal(step()[1], gx)
    # the backward needs the seed that the forward read
    y = dropout(x, 0.4, seed=place)
    place.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- the residual stream and its norms -----------------------------------------------------------------------------


def _norm_back(rstd, hat, hat_err, dy, dy_err, w):
    """Gradient of norm(a) w for the gradient dy: ``(da, its error, dw's terms, their errors)``; errors are absolute, ``hat_err`` relative."""
    n = hat.shape[-1]
    a, a_err = dy * w, dy_err * w.abs() + 2.0 ** -24 * (dy * w).abs()
    mean = (a * hat).mean(-1, keepdim=True)
    size = (a * hat).abs().mean(-1, keepdim=True)
    mean_err = (a_err * hat.abs()).mean(-1, keepdim=True) + (hat_err + n * 2.0 ** -24) * size
    da = rstd * (a - hat * mean)
    da_err = rstd * (a_err + hat.abs() * (mean_err + hat_err * mean.abs())) + 8 * 2.0 ** -24 * rstd * (a.abs() + (hat * mean).abs()) + 2.0 ** -21 * da.abs()
    return da, da_err * (1 + 2.0 ** -10), dy * hat, dy_err * hat.abs() + hat_err * (dy * hat).abs()


def _want(t, o, grads):
    """Outputs and gradients with their errors before they are rounded: ``{name: (value, error)}``."""
    w = {k: (None if v is None else v.detach().double()) for k, v in t.items()}
    u = w["branch"]
    n = u.shape[-1]
    one = torch.ones(n, dtype=torch.float64, device="cuda")
    post, pre, gate = (w[k] if w[k] is not None else one for k in ("post", "pre", "gate"))
    stat = (n + 8) * 2.0 ** -24 + 2.0 ** -22  # relative, of a norm's reciprocal root
    v, v_err = u, torch.zeros_like(u)
    if o["post_norm"]:
        ru = 1 / torch.sqrt((u * u).mean(-1, keepdim=True) + EPS)
        v = u * ru * post
        v_err = v.abs() * (stat + 2.0 ** -22)
    kept = torch.ones_like(u, dtype=torch.bool)
    f = 1.0
    if o["p"]:
        kept, f = philox_kept(u.numel(), o["p"], 11, 13).view(u.shape), factor(o["p"])
    d, d_err = torch.where(kept, v * f, 0), torch.where(kept, (v_err + v.abs() * 2.0 ** -23) * f, 0)
    h = o["scale"] * gate * d
    h_err = (o["scale"] * gate).abs() * d_err + h.abs() * 2.0 ** -22
    if w["residual"] is not None:
        h_err = h_err + 2.0 ** -23 * (h.abs() + (o["residual_scale"] * w["residual"]).abs())
        h = h + o["residual_scale"] * w["residual"]
    out = {"stream": (h, h_err)}
    dh, dh_err = grads["stream"].double() if "stream" in grads else torch.zeros_like(h), torch.zeros_like(h)
    if o["pre_norm"]:
        rh = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        hat = h * rh
        # the statistic moves with the stream's error as well
        moved = rh * rh * (h.abs() * h_err).mean(-1, keepdim=True)
        out["normed"] = (hat * pre, (rh * h_err + hat.abs() * (stat + moved + 2.0 ** -22)) * pre.abs())
        if "normed" in grads:
            stored = _half_step(o["stream_dtype"])
            hat_err = stored + stat + moved + (h_err / h.abs().clamp(min=1e-30)).clamp(max=1)
            da, da_err, dw, dw_err = _norm_back(rh, hat, hat_err, grads["normed"].double(), torch.zeros_like(h), pre)
            dh, dh_err = dh + da, da_err + 2.0 ** -23 * (dh.abs() + da.abs())
            out["pre_grad"] = (dw.sum(0), (dw_err + 2.0 ** -22 * dw.abs()).sum(0) + (dw.shape[0] + 8) * 2.0 ** -24 * dw.abs().sum(0))
    out["residual_grad"] = (o["residual_scale"] * dh, abs(o["residual_scale"]) * dh_err + 2.0 ** -23 * (o["residual_scale"] * dh).abs())
    g = torch.where(kept, o["scale"] * f * dh, 0)
    g_err = torch.where(kept, abs(o["scale"]) * f * dh_err + 2.0 ** -22 * g.abs(), 0)
    terms = g * v
    out["gate_grad"] = (terms.sum(0), (g_err * v.abs() + g.abs() * v_err + 2.0 ** -22 * terms.abs()).sum(0) + (g.shape[0] + 8) * 2.0 ** -24 * terms.abs().sum(0))
    g, g_err = g * gate, g_err * gate.abs() + 2.0 ** -23 * (g * gate).abs()
    if o["post_norm"]:
        g, g_err, dw, dw_err = _norm_back(ru, u * ru, stat + torch.zeros_like(u), g, g_err, post)
        out["post_grad"] = (dw.sum(0), (dw_err + 2.0 ** -22 * dw.abs()).sum(0) + (dw.shape[0] + 8) * 2.0 ** -24 * dw.abs().sum(0))
    out["branch_grad"] = (g, g_err)
    return out


def _tensors(rows, n, dtype, stream_dtype, weight_dtype, residual, post, pre, gate, seed=0):
    g = _gen(seed + rows + n)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {
        "branch": (rand(rows, n) * torch.exp(rand(n) * 0.5)).to(dtype).cuda(),
        "residual": rand(rows, n).to(stream_dtype).cuda() if residual else None,
        "post": (1 + 0.2 * rand(n)).to(weight_dtype).cuda() if post else None,
        "pre": (1 + 0.2 * rand(n)).to(weight_dtype).cuda() if pre else None,
        "gate": rand(n).to(weight_dtype).cuda() if gate else None,
    }


def _check(t, o, also=()):
    """Runs the operator and its gradients and compares all of them."""
    names = [k for k, v in t.items() if v is not None]
    for k in names:
        t[k].requires_grad_(True)
    kw = {"p": o["p"], "seed": 11, "offset": 13} if o["p"] else {}
    stream, normed = residual_norm(t["branch"], t["residual"], post_norm=o["post_norm"], post_weight=t["post"], pre_norm=o["pre_norm"], pre_weight=t["pre"],
                                   gate=t["gate"], scale=o["scale"], residual_scale=o["residual_scale"], eps=EPS, **kw)
    assert (normed is not None) == o["pre_norm"]
    dtype = t["branch"].dtype
    assert stream.dtype == o["stream_dtype"] and (normed is None or normed.dtype == dtype)
    g = _gen(77)
    grads = {"stream": torch.randn(stream.shape, generator=g).to(stream.dtype).cuda()}
    outs = [stream]
    if normed is not None:
        grads["normed"] = torch.randn(normed.shape, generator=g).to(dtype).cuda()
        outs.append(normed)
    for drop in also:
        i = list(grads).index(drop)
        del grads[drop], outs[i]
    made = dict(zip((k + "_grad" for k in names), torch.autograd.grad(outs, [t[k] for k in names], list(grads.values()), allow_unused=True)))
    want = _want(t, o, grads)
    made.update(stream=stream, normed=normed)
    for name, got in made.items():
        if got is None or name not in want:
            assert name not in want or name == "normed" or "stream" in also or "normed" in also, name
            continue
        value, err = want[name]
        assert got.shape == value.shape
        bound = err * (1 + 2.0 ** -6) + _half_step(got.dtype) * (value.abs() + err) + torch.finfo(got.dtype).smallest_normal
        worst = ((got.double() - value).abs() / bound).max().item()
        assert worst <= 1, f"{name}: {worst} times the bound"


def _options(stream_dtype, post=True, pre=True, scale=1.0, residual_scale=1.0, p=0.0):
    return {"post_norm": post, "pre_norm": pre, "scale": scale, "residual_scale": residual_scale, "p": p, "stream_dtype": stream_dtype}


# every number of lanes and chunks, lengths at their borders, odd ones; one row, fewer rows than a workgroup has, more than the grid
LENGTHS = [(1, 1), (5, 7), (3, 64), (300, 128), (33, 129), (9, 512), (17, 513), (130, 1024), (5, 1031), (40, 2048), (7, 2049), (70, 4096), (3, 4100), (11, 8192),
           (4, 8200), (3, 11008), (2, MOST_FEATURES)]
# every length of a row's last chunk, for each number of lanes
LENGTHS += [(3, n) for first in (129, 513, 1025, 4097, 8193) for n in range(first, first + 7)] + [(530, 8195), (2, MOST_FEATURES - 1)]


@pytest.mark.parametrize("types", [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16), (F32, F32, F32)],
                         ids=["bf16", "bf16-f32", "f16", "f16-f32", "f32"])
@pytest.mark.parametrize("rows,n", LENGTHS)
def test_every_part(types, rows, n):
    dtype, stream_dtype, weight_dtype = types
    _check(_tensors(rows, n, dtype, stream_dtype, weight_dtype, True, True, True, True), _options(stream_dtype, scale=0.7, residual_scale=1.25, p=0.2))


@pytest.mark.parametrize("n", [96, 333, 2560])
@pytest.mark.parametrize("parts", range(32))
def test_parts_alone(parts, n):
    """Each of residual, norms with and without weights, gate."""
    residual, post, pre, gate, weights = (bool(parts >> i & 1) for i in range(5))
    if not (post or pre or gate or residual):
        pytest.skip("nothing to do")
    t = _tensors(19, n, BF16, F32 if parts % 3 == 0 and residual else BF16, BF16, residual, post and weights, pre and weights, gate)
    stream_dtype = t["residual"].dtype if residual else BF16
    # (a norm in front alone: the stream is the branch itself, and autograd adds its gradient to the operator's rounded one)
    alone = not (residual or post or gate or parts % 2)
    _check(t, _options(stream_dtype, post=post, pre=pre, p=0.3 if parts % 2 else 0.0), also=("stream",) if alone else ())


@pytest.mark.parametrize("absent", ["stream", "normed"])
def test_only_one_gradient_arrives(absent):
    t = _tensors(50, 200, BF16, BF16, BF16, True, True, True, True)
    _check(t, _options(BF16), also=(absent,))


def test_rows_of_more_than_the_grid():
    _check(_tensors(9000, 64, BF16, BF16, F32, True, True, True, True), _options(BF16))
    _check(_tensors(5000, 264, F16, F32, F32, True, False, True, False), _options(F32, post=False))
    _check(_tensors(2500, 1000, BF16, BF16, F32, True, True, False, True), _options(BF16, pre=False, p=0.1))


def test_the_mask_is_that_of_dropout():
    for n in (64, 99):
        x = torch.randn(30, n, generator=_gen(n)).cuda()
        stream, _ = residual_norm(x, p=0.3, seed=21, offset=4)
        assert torch.equal(stream, dropout(x, 0.3, seed=21, offset=4))


def test_nothing_to_do_returns_the_branch():
    x = torch.randn(4, 6, 32, generator=_gen(3)).cuda().requires_grad_(True)
    stream, normed = residual_norm(x)
    assert stream is x and normed is None
    stream, normed = residual_norm(x, pre_norm=True, eps=EPS)
    assert stream is x
    want = x.detach() / torch.sqrt((x.detach() ** 2).mean(-1, keepdim=True) + EPS)
    assert (normed - want).abs().max() < 1e-5
    both = torch.autograd.grad([stream.sum(), normed.sum()], x)[0]
    alone = torch.autograd.grad(residual_norm(x, pre_norm=True, eps=EPS)[1].sum(), x)[0]
    assert (both - (1 + alone)).abs().max() < 1e-5


def test_shapes_strides_and_empty():
    g = _gen(4)
    big = torch.randn(3, 10, 80, generator=g).to(BF16).cuda()
    w = torch.randn(40, generator=g).cuda()
    base = residual_norm(big[..., 8:48].contiguous(), big[..., 40:].contiguous(), post_weight=w, pre_weight=w)
    for b, r in ((big[..., 8:48], big[..., 40:]), (big[..., 8:48].transpose(0, 1).contiguous().transpose(0, 1), big[..., 40:]),
                 (big.flip(2).flip(2)[..., 8:48], big[..., 40:].clone())):
        for got, want in zip(residual_norm(b, r, post_weight=w, pre_weight=w), base):
            assert torch.equal(got, want)
    for got, want in zip(residual_norm(big[0, 0, 8:48], big[0, 0, 40:], post_weight=w, pre_weight=w), base):
        assert torch.equal(got, want[0, 0])
    odd = big[..., 3:43]  # (6 bytes off a 16-byte border)
    for got, want in zip(residual_norm(odd, big[..., 40:], post_weight=w, pre_weight=w),
                         residual_norm(odd.contiguous(), big[..., 40:].contiguous(), post_weight=w, pre_weight=w)):
        assert torch.equal(got, want)
    e = torch.empty(0, 40, dtype=BF16, device="cuda", requires_grad=True)
    we = w.clone().requires_grad_(True)
    stream, normed = residual_norm(e, e, post_weight=we, pre_weight=w, gate=w)
    assert stream.shape == normed.shape == (0, 40)
    ge, gw = torch.autograd.grad([stream, normed], [e, we], [stream, normed])
    assert ge.shape == (0, 40) and gw.shape == (40,) and not gw.any()
    # gradients that are views, and the same value everywhere
    b = big[..., 8:48].clone().requires_grad_(True)
    y = residual_norm(b, post_weight=w)[0]
    one = torch.autograd.grad(y, b, torch.ones_like(y), retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y.sum(), b)[0], one)


def test_zero_rows_and_not_finite_values_stay_in_their_row():
    x = torch.randn(40, 130, generator=_gen(5)).to(BF16).cuda()
    x[3] = 0
    want = residual_norm(x, post_norm=True, pre_norm=True)
    assert not want[0][3].any() and not want[1][3].any()
    bad = x.clone()
    bad[7, 5], bad[9, 0] = math.nan, math.inf
    got = residual_norm(bad, post_norm=True, pre_norm=True)
    rows = torch.ones(40, dtype=torch.bool)
    rows[[7, 9]] = False
    for a, b in zip(got, want):
        assert torch.equal(a[rows], b[rows])
    assert got[0][7].isnan().all() and got[0][9, 0].isnan()


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_captured_and_replayed(p):
    t = _tensors(300, 136, BF16, F32, BF16, True, True, True, True)
    for v in t.values():
        v.requires_grad_(True)
    place = torch.tensor([1], device="cuda")
    gs, gn = torch.randn(300, 136, device="cuda"), torch.randn(300, 136, device="cuda").to(BF16)

    def step():
        outs = residual_norm(t["branch"], t["residual"], post_weight=t["post"], pre_weight=t["pre"], gate=t["gate"], p=p, seed=place)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(t.values()), [gs, gn]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        place.fill_(i)
        with torch.no_grad():
            t["branch"].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want)


def test_gradient_agrees_with_differences():
    t = _tensors(6, 48, F32, F32, F32, True, True, True, True)
    for v in t.values():
        v.requires_grad_(True)
    g = _gen(9)
    gs, gn = torch.randn(6, 48, generator=g).cuda(), torch.randn(6, 48, generator=g).cuda()
    outs = residual_norm(t["branch"], t["residual"], post_weight=t["post"], pre_weight=t["pre"], gate=t["gate"], eps=EPS)
    made = torch.autograd.grad(outs, list(t.values()), [gs, gn])
    d = {k: v.detach().double() for k, v in t.items()}

    def loss(d):
        norm = lambda a: a / torch.sqrt((a * a).mean(-1, keepdim=True) + EPS)  # noqa: E731
        h = d["residual"] + d["gate"] * norm(d["branch"]) * d["post"]
        return (gs.double() * h).sum() + (gn.double() * norm(h) * d["pre"]).sum()

    for (name, value), grad in zip(d.items(), made):
        for at in ((0,) if value.dim() == 1 else (2, 5), (47,) if value.dim() == 1 else (0, 47)):
            step = torch.zeros_like(value)
            step[at] = 1e-5
            slope = (loss({**d, name: value + step}) - loss({**d, name: value - step})) / 2e-5
            # (six rows' terms of size about 10, float32: differences and the gradient's rounding are far below)
            assert abs(grad[at].item() - slope.item()) < 1e-3, name


def test_library_refuses():
    a = _C.ResidualNorm(rows=2, features=8, branch_dtype=_C.MI8_BF16, stream_dtype=_C.MI8_BF16)
    x = torch.zeros(2, 8, dtype=BF16, device="cuda")
    a.branch = a.stream = x.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    assert _C.lib().mi8_residual_norm_forward(a, stream) == 0
    for name, value in (("features", MOST_FEATURES + 1), ("rows", -1), ("stream_dtype", _C.MI8_F16), ("threshold", 65537), ("branch", None), ("pre_norm", 1),
                        ("post", x.data_ptr())):
        bad = _C.ResidualNorm.from_buffer_copy(a)
        setattr(bad, name, value)
        assert _C.lib().mi8_residual_norm_forward(bad, stream) < 0, name
        assert _C.last_error()
    assert _C.lib().mi8_dropout(x.data_ptr(), _C.MI8_BF16, 16, 65537, 1.0, 0, None, 0, x.data_ptr(), stream) < 0
    assert _C.lib().mi8_dropout(x.data_ptr(), 7, 16, 0, 1.0, 0, None, 0, x.data_ptr(), stream) < 0


def test_offsets_past_32_bits():
    """More than 2^31 elements: the mask of the last ones is the generator's, the last rows are what they are alone, forward and backward."""
    rows, n = (1 << 19) + 131, 4104
    x = torch.ones(rows, n, dtype=BF16, device="cuda")
    y = dropout(x, 0.5, seed=9)
    first = rows * n - 4096
    import numpy as np

    i = np.arange(first // 8, rows * n // 8, dtype=np.uint64)
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    c, k = [i & low, i >> u64(32), np.zeros_like(i), np.zeros_like(i)], [9, 0]
    for _ in range(7):
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(b >> u64(32)) ^ c[1] ^ u64(k[0]), b & low, (a >> u64(32)) ^ c[3] ^ u64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    kept = np.stack([h for w in c for h in (w & u64(0xFFFF), w >> u64(16))], -1).reshape(-1) >= 32768
    assert torch.equal(y.view(-1)[first:], 2 * torch.from_numpy(kept).cuda().to(BF16))
    del y
    tail = torch.randn(300, n, generator=_gen(4)).cuda().to(BF16)
    x[-300:] = tail
    w, g = torch.rand(n, device="cuda").requires_grad_(True), torch.zeros(rows, n, dtype=BF16, device="cuda")
    g[-300:] = torch.randn(300, n, generator=_gen(5)).cuda().to(BF16)
    outs = residual_norm(x.requires_grad_(True), post_weight=w, pre_weight=w)
    gx = torch.autograd.grad(outs, x, [g, g])[0]
    alone = tail.clone().requires_grad_(True)
    few = residual_norm(alone, post_weight=w, pre_weight=w)
    assert torch.equal(outs[0][-300:], few[0]) and torch.equal(outs[1][-300:], few[1])
    assert torch.equal(gx[-300:], torch.autograd.grad(few, alone, [g[-300:], g[-300:]])[0]) and not gx[:-300].any()


def test_rows_that_lie_over_one_another():
    """Expanded branches, residuals and gradients."""
    b, r, g = (torch.randn(1, 72, generator=_gen(i)).cuda().to(BF16) for i in range(3))
    w = torch.rand(72, generator=_gen(3)).cuda().requires_grad_(True)
    many = residual_norm(b.expand(50, 72), r.expand(50, 72), post_weight=w, pre_weight=w)
    whole = residual_norm(b.expand(50, 72).contiguous(), r.expand(50, 72).contiguous(), post_weight=w, pre_weight=w)
    assert all(torch.equal(a, c) for a, c in zip(many, whole))
    made = [torch.autograd.grad(o, w, [g.expand(50, 72)] * 2)[0] for o in (many, whole)]
    assert torch.equal(*made)


@pytest.mark.parametrize("types", [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32)], ids=["bf16", "bf16-f32", "f16"])
@pytest.mark.parametrize("post,gate,residual,p", [(True, False, True, 0.0), (False, True, True, 0.0), (True, True, True, 0.2), (True, False, False, 0.0), (False, True, False, 0.2)])
@pytest.mark.parametrize("rows,n", [(40, 96), (19, 333), (12, 2560), (5, 5000), (4, 8195)])
def test_gradient_at_the_unrounded_stream(types, post, gate, residual, p, rows, n):
    """Where the branch is normed or gated, the backward's normed stream is that of the unrounded one: its error is float32's alone, without the half step of the
    stored stream that :func:`_want` grants."""
    dtype, stream_dtype, weight_dtype = types
    t = _tensors(rows, n, dtype, stream_dtype, weight_dtype, residual, post, True, gate)
    o = _options(stream_dtype, post=post, scale=0.7, residual_scale=1.25, p=p)
    names = [k for k, v in t.items() if v is not None]
    for k in names:
        t[k].requires_grad_(True)
    kw = {"p": p, "seed": 11, "offset": 13} if p else {}
    outs = residual_norm(t["branch"], t["residual"], post_weight=t["post"], pre_weight=t["pre"], gate=t["gate"], scale=0.7, residual_scale=1.25, eps=EPS, **kw)
    grads = {k: torch.randn(v.shape, generator=_gen(i)).to(v.dtype).cuda() for i, (k, v) in enumerate(zip(("stream", "normed"), outs))}
    made = torch.autograd.grad(outs, [t[k] for k in names], list(grads.values()))
    want = _want(t, {**o, "stream_dtype": torch.float64}, grads)
    for name, got in zip(names, made):
        value, err = want[name + "_grad"]
        bound = err * (1 + 2.0 ** -6) + _half_step(got.dtype) * (value.abs() + err) + torch.finfo(got.dtype).smallest_normal
        worst = ((got.double() - value).abs() / bound).max().item()
        assert worst <= 1, f"{name}: {worst} times the bound"


@pytest.mark.parametrize("form", ["all", "in_front", "behind", "alone"])
def test_gradients_only_of_what_is_asked(form):
    """Whichever inputs want a gradient, each gets the bits that it gets together with all others."""
    parts = {"all": (True, True, True, True), "in_front": (True, False, True, False), "behind": (True, True, False, False), "alone": (False, False, True, False)}[form]
    t = {k: v for k, v in _tensors(23, 333, BF16, F32 if form == "all" else BF16, F32, *parts).items() if v is not None}
    names = list(t)
    kw = {"p": 0.2, "seed": 5} if form == "all" else {}
    gs, gn = torch.randn(23, 333, generator=_gen(1)).cuda(), torch.randn(23, 333, generator=_gen(2)).cuda()

    def grads(wanted):
        ins = {k: v.detach().clone().requires_grad_(k in wanted) for k, v in t.items()}
        outs = residual_norm(ins["branch"], ins.get("residual"), post_weight=ins.get("post"), pre_weight=ins.get("pre"), gate=ins.get("gate"), **kw)
        pairs = [(o, g.to(o.dtype)) for o, g in zip(outs, (gs, gn)) if o is not None and o.requires_grad and o is not ins["branch"]]
        return dict(zip(wanted, torch.autograd.grad([o for o, _ in pairs], [ins[k] for k in wanted], [g for _, g in pairs])))

    every = grads(names)
    for bits in range(1, 1 << len(names)):
        wanted = [k for i, k in enumerate(names) if bits >> i & 1]
        got = grads(wanted)
        for k in wanted:
            assert torch.equal(got[k], every[k]), (k, wanted)


@pytest.mark.parametrize("residual", [True, False])
def test_a_gate_that_is_not_learnt(residual):
    """The gradient of the stream's norm is that at the unrounded stream wherever there is a gate, whether its own gradient is wanted or not: the same bits."""
    t = {k: v for k, v in _tensors(23, 333, BF16, BF16, F32, residual, False, True, True).items() if v is not None}
    g = torch.randn(23, 333, generator=_gen(2)).to(BF16).cuda()
    made = []
    for learnt in (True, False):
        ins = {k: v.detach().clone().requires_grad_(k != "gate" or learnt) for k, v in t.items()}
        normed = residual_norm(ins["branch"], ins.get("residual"), pre_weight=ins["pre"], gate=ins["gate"])[1]
        made.append(torch.autograd.grad(normed, [v for k, v in ins.items() if k != "gate"], g))
    assert all(torch.equal(a, b) for a, b in zip(*made))


@pytest.mark.parametrize("weight", [None, BF16, F32], ids=["no_weight", "bf16", "f32"])
@pytest.mark.parametrize("residual,p,scale", [(True, 0.0, 1.0), (True, 0.2, 0.7), (False, 0.2, 1.0), (False, 0.0, 0.3)])
@pytest.mark.parametrize("rows,n", [(300, 136), (40, 333), (12, 2560), (5, 5000), (4, 8195)])
def test_gradient_at_the_unrounded_stream_of_a_plain_join(weight, residual, p, scale, rows, n):
    """The same where the branch has neither norm nor gate: a 16-bit stream that was stored is not what the backward starts from.  A float32 weight's gradient shows
    it, whose own rounding is small."""
    t = _tensors(rows, n, BF16, BF16, weight or F32, residual, False, weight is not None, False)
    o = {**_options(torch.float64, post=False, scale=scale, residual_scale=1.25, p=p)}
    names = [k for k, v in t.items() if v is not None]
    for k in names:
        t[k].requires_grad_(True)
    kw = {"p": p, "seed": 11, "offset": 13} if p else {}
    outs = residual_norm(t["branch"], t["residual"], pre_norm=True, pre_weight=t["pre"], scale=scale, residual_scale=1.25, eps=EPS, **kw)
    assert outs[0].dtype == BF16
    grads = {k: torch.randn(v.shape, generator=_gen(i)).to(v.dtype).cuda() for i, (k, v) in enumerate(zip(("stream", "normed"), outs))}
    made = torch.autograd.grad(outs, [t[k] for k in names], list(grads.values()))
    want = _want(t, o, grads)
    for name, got in zip(names, made):
        value, err = want[name + "_grad"]
        bound = err * (1 + 2.0 ** -6) + _half_step(got.dtype) * (value.abs() + err) + torch.finfo(got.dtype).smallest_normal
        worst = ((got.double() - value).abs() / bound).max().item()
        assert worst <= 1, f"{name}: {worst} times the bound"
