"""Block-scaled float8 casts, products and layers against the 64-bit oracle (oracle/block_oracle.py)."""

import pytest
import torch

from olmo_core_amd.float8 import (
    AOFloat8LinearRecipe,
    Float8Config,
    blockwise_grouped_linear,
    blockwise_linear,
    blockwise_weight,
    ops,
)
from olmo_core_amd.float8.linear import Float8Linear, float8_projections
from olmo_core_amd.float8.native_config import Float8LinearConfig
from oracle import block_oracle as B

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32

# v_mfma_f32_16x16x128_f8f6f4 adds its 128 products in groups of eight consecutive ones, each aligned to the group's largest exponent sum and
# cut toward zero at 2^-13 of it (found with one product of 2^16 beside one of 2^(16 - j): kept up to j = 13 in the same eight, up to
# 23 elsewhere); the largest itself, a product of two four-bit mantissas, is whole.  So a group loses at most 7 * 2^-13 of its largest product, and a sum
# at most that share of the sum of its magnitudes; what the groups and the accumulator lose among themselves, 2^-23 of the
# largest for each of 17 terms and block, is 2^-18 of it.
SUM_ERROR = 7 * 2.0 ** -13 + 2.0 ** -18
# The cuts of unlike products point in unlike directions: for n products of size s the error's norm is at most
# sqrt(n) * 0.29 * 2^-13 * 4 s where the sum's is sqrt(n) s.
NORM_ERROR = 2.0 ** -12


def make(shape, seed, std=1.0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    x = x * torch.where(torch.rand(shape, generator=g) < 0.01, 20.0, 1.0)
    return x.to(dtype)


def close(got, exact, magnitude, what):
    """One rounding of the output type on top of the error of the sum."""
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    err = (got.detach().double().cpu() - exact).abs()
    bound = exact.abs() * (torch.finfo(got.dtype).eps / 2) * (1 + 2.0 ** -10) + magnitude * SUM_ERROR
    worst = (err - bound).max()
    assert bool((err <= bound).all()), f"{what}: {int((err > bound).sum())} of {err.numel()} off, worst by {float(worst):.3e}"
    if magnitude.numel() >= 256:
        share = float(err.norm() / exact.norm())
        assert share <= torch.finfo(got.dtype).eps / 2 + NORM_ERROR, f"{what}: off by {share:.2e} of the norm"


def codes(t):
    return t.cpu().float().double()


def same_codes(got, want):
    g = codes(got)
    assert bool(((g == want) | (torch.isnan(g) & torch.isnan(want))).all())


def same_bytes(got, k, rows):
    """got: stored exponents of one operand; k [rows, blocks]."""
    want = B.scale_bytes(k, rows)
    g = got.cpu().view(torch.uint8).to(torch.int64)
    assert g.shape == want.shape
    assert bool(((g == want) | (want < 0)).all())


# ---- casts -----------------------------------------------------------------------------------------------------------

SHAPES = [(1, 16), (5, 48), (128, 128), (129, 144), (300, 1040), (64, 2048), (1000, 112)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_cast_of_rows_and_columns(dev, shape, dtype):
    x = make(shape, 1, dtype=dtype)
    q, s, q_t, s_t = ops.cast_blockwise(x.to(dev), want_transposed=True)
    rows, cols = shape
    want, k, _ = B.quantise(x, 1, 128)
    same_codes(q, want)
    same_bytes(s, k, rows)
    want, k, _ = B.quantise(x.t(), 1, 128)
    same_codes(q_t, want)
    same_bytes(s_t, k, cols)
    for kw in (dict(want_rowmajor=True), dict(want_rowmajor=False, want_transposed=True)):
        one = ops.cast_blockwise(x.to(dev), **kw)
        for a, b in zip(one, (q, s, q_t, s_t)):
            assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("matrices", [1, 3])
@pytest.mark.parametrize("shape", [(16, 16), (128, 128), (208, 336), (1040, 144)])
def test_cast_of_weights(dev, shape, matrices, dtype):
    rows, cols = shape
    w = make((matrices * rows, cols), 2, std=0.02, dtype=dtype)
    w[: rows // 2] *= 2.0 ** -9
    q, s, q_t, s_t = ops.cast_blockwise(w.to(dev), square=True, matrices=matrices, want_transposed=True)
    q, s = q.view(matrices, rows, -1), s.view(matrices, *s.shape[-2:])
    q_t, s_t = q_t.view(matrices, cols, -1), s_t.view(matrices, *s_t.shape[-2:])
    for e in range(matrices):
        want, k, _ = B.quantise(w[e * rows:(e + 1) * rows], 128, 128)
        same_codes(q[e], want[:rows])
        same_codes(q_t[e], want.t()[:cols])
        same_bytes(s[e], k.repeat_interleave(128, 0), rows)
        same_bytes(s_t[e], k.t().repeat_interleave(128, 0), cols)


def test_cast_of_border_magnitudes(dev):
    """Blocks whose largest magnitude sits at a border of the scale, at the ends of the exponent's range, zero, not finite."""
    tops = [448.0, 449.0, 447.0, 1.75, 1.7578125, 1.0, 0.0, 2.0 ** -126, 2.0 ** -133, 2.0 ** -112, 1.75 * 2.0 ** -112, 2.0 ** -113, 3.3e38, 2.0 ** 127,
            float("inf"), float("nan"), float("-inf"), 1e-12]
    x = make((len(tops), 384), 3, std=0.1).float().clamp(-0.9, 0.9)
    for i, t in enumerate(tops):
        finite = t if abs(t) < float("inf") else 1.0
        x[i, 128:256] *= finite
        x[i, 200] = t
    for dtype in (BF16, F32):
        xd = x.to(dtype)
        q, s, q_t, s_t = ops.cast_blockwise(xd.to(dev), want_transposed=True)
        want, k, _ = B.quantise(xd, 1, 128)
        same_codes(q, want)
        same_bytes(s, k, len(tops))
        want, k, _ = B.quantise(xd.t(), 1, 128)
        same_codes(q_t, want)
        q, _, q_t, _ = ops.cast_blockwise(xd[:, 128:256].contiguous().to(dev), square=True, want_transposed=True)
        want, _, _ = B.quantise(xd[:, 128:256], 128, 128)
        same_codes(q, want[: len(tops)])
        same_codes(q_t, want.t()[:128])


def spread(T, E, kind, seed=5):
    g = torch.Generator().manual_seed(seed)
    if kind == "skew":
        ids = (torch.rand(T, generator=g) ** 3 * E).long().clamp(max=E - 1)
        return torch.bincount(ids, minlength=E)
    if kind == "one":
        sizes = torch.zeros(E, dtype=torch.long)
        sizes[E // 2] = T
        return sizes
    if kind == "short":  # rows behind the last group
        sizes = torch.bincount(torch.randint(0, E, (max(T - 37, 0),), generator=g), minlength=E)
        return sizes
    return torch.zeros(E, dtype=torch.long)  # "none"


GROUPS = [(1, 1, "one"), (300, 4, "skew"), (1000, 7, "short"), (513, 70, "skew"), (200, 3, "one"), (90, 5, "none")]


@pytest.mark.parametrize("T,E,kind", GROUPS)
def test_grouped_cast(dev, T, E, kind):
    cols = 208
    x, sizes = make((T, cols), 6), spread(T, E, kind)
    q, s, q_t, s_t = ops.grouped_cast_blockwise(x.to(dev), sizes.to(dev), want_transposed=True)
    first = unit = 0
    sb, stb = s.cpu().view(torch.uint8).long(), s_t.cpu().view(torch.uint8).long()
    for m in sizes.tolist():
        if m:
            part = x[first:first + m]
            want, k, _ = B.quantise(part, 1, 128)
            same_codes(q[first:first + m], want)
            rows = B.scale_bytes(k, m)
            here = sb[:, 128 * unit:128 * unit + rows.shape[1]]
            assert bool(((here == rows) | (rows < 0)).all())
            want, k, _ = B.quantise(part.t(), 1, 128)
            same_codes(q_t[:, 128 * unit:128 * unit + want.shape[1]], want)
            for u in range(k.shape[1]):
                cb = B.scale_bytes(k[:, u:u + 1], cols)[0]
                assert bool(((stb[unit + u] == cb) | (cb < 0)).all())
        first += m
        unit += -(-m // 128)


# ---- products --------------------------------------------------------------------------------------------------------

PRODUCTS = [(1, 16, 16), (7, 48, 144), (64, 128, 128), (65, 144, 1040), (200, 336, 256), (300, 2768, 400), (1000, 1024, 2064), (2100, 2176, 640)]


@pytest.mark.parametrize("dtype,w_dtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear_and_gradients(dev, M, N, K, dtype, w_dtype):
    x, w, g = make((M, K), 7, dtype=dtype), make((N, K), 8, std=0.05, dtype=w_dtype), make((M, N), 9, std=1e-3, dtype=dtype)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = blockwise_linear(xd, wd)
    y.backward(g.to(dev))
    assert y.dtype == xd.grad.dtype == dtype and wd.grad.dtype == w_dtype
    for got, want, size, what in zip((y, xd.grad, wd.grad), B.linear(x, w, g), B.magnitudes(x, w, g), ("y", "gx", "gw")):
        close(got, want, size, what)


@pytest.mark.parametrize("M,N,K", [(3300, 3600, 400), (3585, 3584, 128), (300, 43024, 272), (49000, 272, 144)])
def test_large_products(dev, M, N, K):
    """Enough tiles for the persistent kernel, ragged in either direction."""
    x, w = make((M, K), 50), make((N, K), 51, std=0.05)
    y = blockwise_linear(x.to(dev), w.to(dev))
    close(y, B.linear(x, w), B.magnitudes(x, w), "y")


@pytest.mark.parametrize("M,N,K", [(1, 16, 48), (65, 144, 128), (300, 272, 400), (513, 528, 1040), (40, 1040, 2064), (129, 264, 640)])
def test_kernels_agree(dev, M, N, K):
    """Every tile shape on every size: the bits of one another, within the bound of the oracle."""
    x, w = make((M, K), 56), make((N, K), 57, std=0.05)
    a, sa, _, _ = ops.cast_blockwise(x.to(dev))
    b, sb, _, _ = ops.cast_blockwise(w.to(dev), square=True) if N % 16 == 0 else ops.cast_blockwise(w.to(dev))
    ys = [ops.gemm_fp8_blockwise(a, sa, b, sb, k=K, variant=v) for v in range(4)]
    close(ys[0], B.rows_values(x) @ (B.square_values(w) if N % 16 == 0 else B.rows_values(w)).t(), B.magnitudes(x, w), "y")
    assert all(torch.equal(ys[0], y) for y in ys[1:])
    fs = [ops.gemm_fp8_blockwise(a, sa, b, sb, k=K, variant=v, out_dtype=F32) for v in range(3)]
    assert all(torch.equal(fs[0], f) for f in fs[1:]) and torch.equal(fs[0].to(BF16), ys[0])


@pytest.mark.parametrize("T,E,kind", [(6001, 7, "skew"), (6001, 70, "skew"), (5990, 9, "short"), (6001, 5, "one"), (6001, 4, "none")])
def test_large_grouped_products(dev, T, E, kind):
    """The same for groups, also empty ones and rows behind the last."""
    N, K = 2064, 272
    x, w = make((T, K), 52), make((E * N, K), 53, std=0.05)
    sizes = spread(T, E, kind)
    y = blockwise_grouped_linear(x.to(dev), w.to(dev), sizes.to(dev))
    first = 0
    for e, m in enumerate(sizes.tolist()):
        if m:
            rows, we = slice(first, first + m), w[e * N:(e + 1) * N]
            close(y[rows], B.linear(x[rows], we), B.magnitudes(x[rows], we), f"y {e}")
        first += m
    assert not y[first:].any()


@pytest.mark.parametrize("T,E,kind", [(2500, 9, "skew"), (900, 70, "skew"), (2490, 11, "short"), (2500, 8, "one"), (1, 8, "one"), (100, 8, "none")])
def test_large_grouped_weight_gradients(dev, T, E, kind):
    N, K = (1040, 1296) if E < 20 else (528, 272)
    x, g = make((T, K), 54), make((T, N), 55, std=1e-3)
    sizes = spread(T, E, kind)
    w = torch.zeros(E * N, K, dtype=BF16, device=dev, requires_grad=True)
    blockwise_grouped_linear(x.to(dev), w, sizes.to(dev)).backward(g.to(dev))
    first = 0
    for e, m in enumerate(sizes.tolist()):
        gw = w.grad[e * N:(e + 1) * N]
        if m:
            xv, gv = B.rows_values(x[first:first + m].t()), B.rows_values(g[first:first + m].t())
            close(gw, gv @ xv.t(), gv.abs() @ xv.abs().t(), f"gw {e}")
        else:
            assert not gw.any()
        first += m


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 96, 130])
@pytest.mark.parametrize("N,K", [(16, 48), (1040, 2064), (528, 8192)])
def test_linear_with_kept_weight(dev, M, N, K):
    x, w = make((M, K), 10), make((N, K), 11, std=0.05)
    kept = blockwise_weight(w.to(dev))
    with torch.no_grad():
        y = blockwise_linear(x.to(dev), w.to(dev), kept=kept)
    close(y, B.linear(x, w), B.magnitudes(x, w), "y")
    x3 = x.to(dev).unsqueeze(0).expand(2, M, K)
    assert torch.equal(blockwise_linear(x3, w.to(dev), kept=kept), y.expand(2, M, N))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,E,kind", [(8, 1, "one"), (60, 8, "skew"), (512, 64, "skew"), (500, 70, "short"), (100, 16, "one"), (40, 5, "none")])
@pytest.mark.parametrize("N,K", [(48, 144), (1040, 2064)])
def test_few_rows_of_groups(dev, T, E, kind, N, K, dtype):
    """Rows that the product quantises itself, in groups longer than its tiles and empty ones."""
    x, w = make((T, K), 60, dtype=dtype), make((E * N, K), 61, std=0.05)
    sizes = spread(T, E, kind)
    with torch.no_grad():
        y = blockwise_grouped_linear(x.to(dev), w.to(dev), sizes.to(dev), kept=blockwise_weight(w.to(dev), experts=E))
    assert y.dtype == dtype
    first = 0
    for e, m in enumerate(sizes.tolist()):
        if m:
            rows, we = slice(first, first + m), w[e * N:(e + 1) * N]
            close(y[rows], B.linear(x[rows], we), B.magnitudes(x[rows], we), f"y {e}")
        first += m
    assert not y[first:].any()


@pytest.mark.parametrize("M", [5, 100])
def test_recorded_calls(dev, M):
    """From the third call on the launches of a linear are replayed: other data, same sizes, the bits of the calls one by one."""
    from olmo_core_amd.float8 import blockwise

    w = make((272, 400), 62, std=0.05).to(dev).requires_grad_(True)
    we = make((4 * 48, 400), 63, std=0.05).to(dev).requires_grad_(True)
    sizes = spread(M, 4, "skew").to(dev)

    def step(seed):
        x = make((M, 400), seed).to(dev).requires_grad_(True)
        g, ge = make((M, 272), seed + 1).to(dev), make((M, 48), seed + 2).to(dev)
        y, z = blockwise_linear(x, w), blockwise_grouped_linear(x, we, sizes)
        with torch.no_grad():
            y2 = blockwise_linear(x, w)
        return (y.detach(), y2, z.detach(), *torch.autograd.grad(y, (x, w), g), *torch.autograd.grad(z, (x, we), ge))

    replayed = [step(s) for s in range(70, 76)]
    planned = blockwise.plan.call
    blockwise.plan.call = lambda *a, **k: None
    try:
        single = [step(s) for s in range(70, 76)]
    finally:
        blockwise.plan.call = planned
    for a, b in zip(replayed, single):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_checkpointed(dev):
    from torch.utils.checkpoint import checkpoint

    w = make((144, 256), 64, std=0.05).to(dev).requires_grad_(True)
    x = make((50, 256), 65).to(dev).requires_grad_(True)
    g = make((50, 144), 66).to(dev)
    want = torch.autograd.grad(blockwise_linear(x, w), (x, w), g)
    for _ in range(4):
        got = torch.autograd.grad(checkpoint(blockwise_linear, x, w, use_reentrant=False), (x, w), g)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_outliers_stay_in_their_block(dev):
    """A block with one huge value costs its own 127 neighbours, nobody else."""
    x, w = make((40, 512), 12), make((64, 512), 13, std=0.05)
    x2 = x.clone()
    x2[3, 130] = 3e30
    y, y2 = (blockwise_linear(t.to(dev), w.to(dev)).cpu() for t in (x, x2))
    assert torch.equal(y[:3], y2[:3]) and torch.equal(y[4:], y2[4:])
    close(y2, B.linear(x2, w), B.magnitudes(x2, w), "y")


def test_not_finite(dev):
    x, w = make((40, 512), 14), make((160, 512), 15, std=0.05)
    x[3, 130], x[7, 5] = float("nan"), float("inf")
    y = blockwise_linear(x.to(dev), w.to(dev)).cpu()
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[3, 7]] = True
    assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all())
    w[130, 0] = float("nan")  # its block of 128 x 128 covers the rows from 128 on
    y = blockwise_linear(make((40, 512), 14).to(dev), w.to(dev)).cpu()
    assert bool(torch.isnan(y[:, 128:]).all()) and bool(torch.isfinite(y[:, :128]).all())


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("N,K", [(48, 144), (256, 128), (1040, 336)])
@pytest.mark.parametrize("T,E,kind", GROUPS)
def test_grouped_linear_and_gradients(dev, T, E, kind, N, K, transposed):
    n_in, n_out = (N, K) if transposed else (K, N)
    x, w, g = make((T, n_in), 16), make((E * N, K), 17, std=0.05), make((T, n_out), 18, std=1e-3)
    sizes = spread(T, E, kind)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = blockwise_grouped_linear(xd, wd, sizes.to(dev), transposed=transposed)
    y.backward(g.to(dev))
    kept = blockwise_weight(w.to(dev), experts=E)
    with torch.no_grad():
        y2 = blockwise_grouped_linear(x.to(dev), w.to(dev), sizes.to(dev), transposed=transposed, kept=kept)
    first = 0
    for e, m in enumerate(sizes.tolist()):
        we = w[e * N:(e + 1) * N]
        we = we.t() if transposed else we
        gw = wd.grad[e * N:(e + 1) * N]
        gw = gw.t() if transposed else gw
        rows = slice(first, first + m)
        if m:
            want, size = B.linear(x[rows], we, g[rows]), B.magnitudes(x[rows], we, g[rows])
            close(y[rows], want[0], size[0], f"y {e}")
            close(y2[rows], want[0], size[0], f"y kept {e}")
            close(xd.grad[rows], want[1], size[1], f"gx {e}")
            close(gw, want[2], size[2], f"gw {e}")
        else:
            assert not gw.any()
        first += m
    assert not y[first:].any() and not y2[first:].any() and not xd.grad[first:].any()


def test_gradient_against_differences(dev):
    """The loss is linear in x and in W: its difference along a direction against the gradients, both through float8.  Every value is
    rounded by at most 2^-4 of itself, independently, so a sum of n products is off by about 2^-4 sqrt(3 / n) of its norm: with 512 x 384
    and more of them 1 % would be twenty deviations."""
    x, w, g = make((512, 384), 19), make((256, 384), 20), make((512, 256), 21)
    dx, dw = make((512, 384), 22), make((256, 384), 23)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    blockwise_linear(xd, wd).backward(g.to(dev))
    loss = lambda a, b: float((blockwise_linear(a.to(dev), b.to(dev)).double() * g.to(dev).double()).sum())  # noqa: E731
    for grad, d, diff in ((xd.grad, dx, loss(x + dx, w) - loss(x - dx, w)), (wd.grad, dw, loss(x, w + dw) - loss(x, w - dw))):
        along = float((grad.double().cpu() * d.double()).sum())
        norm = float(grad.double().norm().cpu() * d.double().norm())
        assert abs(diff / 2 - along) <= 0.01 * norm


def test_empty_and_partial_gradients(dev):
    w = make((48, 144), 24).to(dev).requires_grad_(True)
    x = torch.empty(0, 144, dtype=BF16, device=dev, requires_grad=True)
    y = blockwise_linear(x, w)
    assert y.shape == (0, 48)
    y.sum().backward()
    assert not w.grad.any() and x.grad.shape == x.shape
    sizes = torch.zeros(3, dtype=torch.long, device=dev)
    we = make((48, 144), 24).to(dev).requires_grad_(True)
    y = blockwise_grouped_linear(torch.empty(0, 144, dtype=BF16, device=dev), we, sizes)
    y.sum().backward()
    assert y.shape == (0, 16) and not we.grad.any()
    x = make((20, 144), 25).to(dev)
    blockwise_linear(x, w).float().sum().backward()  # only the weight's
    x.requires_grad_(True)
    w2 = w.detach()
    blockwise_linear(x, w2).float().sum().backward()
    assert x.grad is not None and w2.grad is None
    assert torch.equal(w.grad, torch.autograd.grad(blockwise_linear(x, w).float().sum(), w)[0])


# ---- layers ----------------------------------------------------------------------------------------------------------


def test_recipe_converts_linears(dev):
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(256, 144, dtype=BF16), torch.nn.Linear(144, 32, bias=False, dtype=BF16)).to(dev)
    ref = [m.weight.detach().clone() for m in model]
    Float8Config(ao_recipe=AOFloat8LinearRecipe.blockwise).apply_float8_linear(model)
    assert all(isinstance(m, Float8Linear) for m in model) and "blk_e4m3" in repr(model[0])
    x = make((3, 50, 256), 26).to(dev).requires_grad_(True)
    y = model[0](x)
    assert torch.equal(y, blockwise_linear(x, ref[0]) + model[0].bias)
    y = model(x)
    y.float().sum().backward()
    assert x.grad.shape == x.shape and model[0].weight.grad.dtype == BF16 and model[0].bias.grad is not None


def test_gradients_with_a_kept_weight(dev):
    """The gradients with kept copies are those without, also where only the weight, or only the input, has one."""
    x, w, g = make((40, 400), 43).to(dev), make((144, 400), 44, std=0.05).to(dev), make((40, 144), 45).to(dev)
    kept = blockwise_weight(w)
    for need_x, need_w in ((True, True), (True, False), (False, True)):
        for _ in range(4):
            got, want = [], []
            for k, out in ((kept, got), (None, want)):
                a, b = x.clone().requires_grad_(need_x), w.clone().requires_grad_(need_w)
                blockwise_linear(a, b, kept=k).backward(g)
                out += [a.grad, b.grad]
            for s, t in zip(got, want):
                assert (s is None) == (t is None) and (s is None or torch.equal(s, t))


def test_module_keeps_float8_weights(dev):
    config = Float8LinearConfig.from_recipe_name("blockwise")
    config.enable_fsdp_float8_all_gather = True
    m = Float8Linear(256, 64, bias=False, dtype=BF16, device=dev, config=config)
    x = make((9, 256), 27).to(dev)
    with torch.no_grad():
        y = m(x)
        kept = m.weight_operands()
        assert m.weight_operands() is kept and torch.equal(y, blockwise_linear(x, m.weight))
        m.weight.mul_(2)
        assert m.weight_operands() is not kept and torch.equal(m(x), 2 * y)


def test_projections_share_the_input(dev):
    torch.manual_seed(1)
    mods = [torch.nn.Linear(256, n, bias=n == 64, dtype=BF16, device=dev) for n in (256, 64, 64)]
    holder = torch.nn.ModuleList(mods)
    Float8Config(ao_recipe=AOFloat8LinearRecipe.blockwise).apply_float8_linear(holder)
    x1 = make((70, 256), 28).to(dev).requires_grad_(True)
    x2 = x1.detach().clone().requires_grad_(True)
    gs = [make((70, m.out_features), 29 + i, std=1e-3).to(dev) for i, m in enumerate(holder)]
    ys = float8_projections(x1, *holder)
    torch.autograd.backward(ys, gs)
    grads = [m.weight.grad.clone() for m in holder]
    holder.zero_grad()
    zs = [m(x2) for m in holder]
    torch.autograd.backward(zs, gs)
    assert all(torch.equal(a, b) for a, b in zip(ys, zs)) and torch.equal(x1.grad, x2.grad)
    assert all(torch.equal(a, m.weight.grad) for a, m in zip(grads, holder))


def test_autocast_with_float32_parameters(dev):
    m = torch.nn.Linear(256, 48, bias=False, device=dev)
    holder = torch.nn.ModuleList([m])
    Float8Config(ao_recipe=AOFloat8LinearRecipe.blockwise).apply_float8_linear(holder)
    x = make((33, 256), 30, dtype=F32).to(dev).requires_grad_(True)
    with torch.autocast("cuda", dtype=BF16):
        y = holder[0](x)
    assert y.dtype == BF16
    y.float().sum().backward()
    assert x.grad.dtype == F32 and holder[0].weight.grad.dtype == F32
    assert torch.equal(y, blockwise_linear(x.detach().to(BF16), holder[0].weight.detach()))


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------------


def test_captured_and_replayed(dev):
    """A forward and a backward in graphs of their own inputs, replayed between eager calls."""
    w = make((272, 400), 31, std=0.05).to(dev)
    kept = blockwise_weight(w)
    sizes = spread(150, 4, "skew").to(dev)
    we = make((4 * 48, 400), 32, std=0.05).to(dev).requires_grad_(True)
    x, g = make((150, 400), 33).to(dev).requires_grad_(True), make((150, 48), 34).to(dev)

    def work():
        with torch.no_grad():
            y = blockwise_linear(x, w, kept=kept)
        z = blockwise_grouped_linear(x, we, sizes)
        return (y, z.detach(), *torch.autograd.grad(z, (x, we), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (35, 36, 37):
        with torch.no_grad():
            x.copy_(make((150, 400), seed))
        sizes.copy_(spread(150, 4, "skew", seed))
        eager = work()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_on_a_stream_of_its_own(dev):
    x, w = make((100, 400), 38).to(dev), make((272, 400), 39).to(dev)
    torch.cuda.synchronize()
    want = blockwise_linear(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = blockwise_linear(x, w)
    s.synchronize()
    assert torch.equal(got, want)


def test_compiled_module_breaks_the_graph(dev):
    holder = torch.nn.Sequential(torch.nn.Linear(256, 64, bias=False, dtype=BF16, device=dev))
    Float8Config(ao_recipe=AOFloat8LinearRecipe.blockwise).apply_float8_linear(holder)
    x = make((20, 256), 67).to(dev)
    want = holder(x)
    assert torch.equal(torch.compile(holder, backend="eager")(x), want)


def test_one_weight_twice_and_views(dev):
    """The same module twice in one call; inputs that are views of other tensors; a vector."""
    holder = torch.nn.ModuleList([torch.nn.Linear(256, 64, bias=False, dtype=BF16, device=dev)])
    Float8Config(ao_recipe=AOFloat8LinearRecipe.blockwise).apply_float8_linear(holder)
    m = holder[0]
    x = make((20, 256), 68).to(dev)
    a, b = float8_projections(x, m, m)
    (a + 2 * b).float().sum().backward()
    (w3,) = torch.autograd.grad((3 * blockwise_linear(x, m.weight)).float().sum(), m.weight)
    assert torch.equal(a, b) and float((m.weight.grad.float() - w3.float()).norm()) <= 2.0 ** -6 * float(w3.float().norm())
    big = make((60, 600), 69).to(dev)
    view = big[1:41:2, 7:263]
    assert torch.equal(blockwise_linear(view, m.weight), blockwise_linear(view.contiguous(), m.weight))
    assert torch.equal(blockwise_linear(x[3], m.weight), blockwise_linear(x, m.weight)[3])
    assert torch.equal(blockwise_linear(x.t().contiguous().t(), m.weight), blockwise_linear(x, m.weight))


def test_refusals(dev):
    x, w = make((8, 144), 40).to(dev), make((48, 144), 41).to(dev)
    with pytest.raises(ValueError, match="input features"):
        blockwise_linear(x[:, :128], w)
    with pytest.raises(ValueError, match="multiples of 16"):
        blockwise_linear(x, w[:40])
    with pytest.raises(TypeError, match="input type"):
        blockwise_linear(x.half(), w)
    with pytest.raises(TypeError, match="weight type"):
        blockwise_linear(x, w.half())
    with pytest.raises(ValueError, match="kept"):
        blockwise_linear(x, w, kept=blockwise_weight(w[:32]))
    with pytest.raises(ValueError, match="no transposed copy"):
        blockwise_linear(x.clone().requires_grad_(True), w, kept=blockwise_weight(w, transposed=False))
    for grads in (False, True):
        with pytest.raises(ValueError, match="no transposed copy"):
            blockwise_grouped_linear(make((8, 48), 42).to(dev), w.clone().requires_grad_(grads), torch.tensor([8], device=dev), transposed=True,
                                     kept=blockwise_weight(w, transposed=False))
    with pytest.raises(ValueError, match="0 matrices"):
        blockwise_weight(w, experts=0)
    with pytest.raises(ValueError, match="weight on cpu"):
        blockwise_linear(x, w.cpu())
    with pytest.raises(ValueError, match="vector of integers"):
        blockwise_grouped_linear(x, w, torch.tensor([4.0, 4.0, 0.0], device=dev))
    with pytest.raises(ValueError, match="not 5 matrices"):
        blockwise_grouped_linear(x, w, torch.tensor([4, 1, 1, 1, 1], device=dev))
    q, s, _, _ = ops.cast_blockwise(x)
    with pytest.raises(ValueError, match="scales"):
        ops.gemm_fp8_blockwise(q, s, q, s[:1].contiguous(), k=144)
    with pytest.raises(TypeError, match="float8_e8m0fnu"):
        ops.gemm_fp8_blockwise(q, s.float(), q, s, k=144)
    with pytest.raises(RuntimeError):  # no second derivative
        z = x.clone().requires_grad_(True)
        (gz,) = torch.autograd.grad(blockwise_linear(z, w).float().sum(), z, create_graph=True)
        gz.float().sum().backward()


def test_casts_together(dev):
    """One launch for weights, rows, rows in groups and several matrices gives what the calls one by one give."""
    sizes = torch.tensor([130, 0, 1, 169], device=dev)
    for dtype in (BF16, F32):
        items = [
            (make((208, 336), 1, dtype=dtype).to(dev), dict(square=True, want_transposed=True)),
            (make((300, 144), 2, dtype=dtype).to(dev), dict(group_sizes=sizes, want_transposed=True)),
            (make((1, 16), 3, dtype=dtype).to(dev), dict(want_rowmajor=False, want_transposed=True)),
            (make((390, 272), 4, dtype=dtype).to(dev), dict(square=True, matrices=3, want_transposed=True)),
            (make((0, 144), 5, dtype=dtype).to(dev), dict(want_transposed=True)),
            (make((513, 1040), 6, dtype=BF16).to(dev), dict()),
            (make((256, 272), 7, dtype=dtype).to(dev), dict(matrices=2, want_transposed=True)),
        ]
        for (x, kw), got in zip(items, ops.cast_blockwise_batch(items)):
            alone = ops.grouped_cast_blockwise if "group_sizes" in kw else ops.cast_blockwise
            want = alone(x, **kw)
            if "group_sizes" in kw:  # (2 + 0 + 1 + 2 tiles of rows; the rest of the axis is not touched)
                got, want = [(q, s[:, :640], q_t[:, :640], s_t[:5]) for q, s, q_t, s_t in (got, want)]
            for a, b in zip(got, want):
                assert (a is None) == (b is None)
                assert a is None or (a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)))
    with pytest.raises(ValueError):
        ops.cast_blockwise_batch([(torch.zeros(16, 24, device=dev), {})] * 2)


@pytest.mark.parametrize("shapes", [[(1, 16, 48), (65, 144, 128)], [(300, 272, 400), (513, 528, 1040), (40, 1040, 2064), (300, 272, 400)],
                                    [(129, 264, 640), (3585, 3584, 128)], [(5, 16, 16)], [(16, 32, 48)] * 8])
def test_products_together(dev, shapes):
    """Small ones in one launch, a large one beside them on its own kernel, with outputs of either type."""
    products = []
    for i, (M, N, K) in enumerate(shapes):
        a, b = make((M, K), 2 * i).to(dev), make((N, K), 2 * i + 1).to(dev)
        products.append((*ops.cast_blockwise(a)[:2], *ops.cast_blockwise(b, square=True)[:2], K, (BF16, F32)[i % 2]))
    for (a, sa, b, sb, k, dtype), got in zip(products, ops.gemm_fp8_blockwise_batch(products)):
        assert got.dtype == dtype and torch.equal(got, ops.gemm_fp8_blockwise(a, sa, b, sb, k=k, out_dtype=dtype))
    with pytest.raises(TypeError):
        ops.gemm_fp8_blockwise_batch([(*p[:5], torch.float16) for p in products * 2][:2])


@pytest.mark.parametrize("widths,frozen,unused", [((256, 64, 64), (), ()), ((48, 272, 144, 16, 1040), (), ()), ((256, 64, 64), (1,), ()),
                                                  ((256, 64, 64), (), (2,)), ((64, 64), (0, 1), ())])
def test_recorded_calls_of_several_weights(dev, widths, frozen, unused):
    """The replayed backward of several weights makes the terms of the input's gradient apart and adds them in the order of the calls one by one."""
    from olmo_core_amd.float8 import blockwise

    ws = [make((n, 256), 90 + i, std=0.05).to(dev).requires_grad_(i not in frozen) for i, n in enumerate(widths)]
    es = [make((3 * 48, 256), 100 + i, std=0.05).to(dev).requires_grad_(i not in frozen) for i in range(len(widths))]
    sizes = torch.tensor([60, 0, 37], device=dev)

    def step(seed):
        x = make((97, 256), seed).to(dev).requires_grad_(True)
        out = []
        for weights, ys in ((ws, blockwise._linears(x, ws, [None] * len(ws))),
                            (es, blockwise._grouped_linears(x, es, sizes, [None] * len(es), False))):
            used = [i for i in range(len(ys)) if i not in unused]
            gs = [make(ys[i].shape, seed + 1 + i).to(dev) for i in used]
            asked = [x] + [weights[i] for i in used if i not in frozen]
            out += [y.detach() for y in ys] + list(torch.autograd.grad([ys[i] for i in used], asked, gs))
        return out

    before = sum(type(q) is blockwise.plan.Plan for p in blockwise.plan._plans.values() if type(p) is blockwise.plan.Plan for q in p.then.values())
    replayed = [step(s) for s in range(120, 180, 12)]
    after = sum(type(q) is blockwise.plan.Plan for p in blockwise.plan._plans.values() if type(p) is blockwise.plan.Plan for q in p.then.values())
    assert after >= before + 2
    planned = blockwise.plan.call
    blockwise.plan.call = lambda *a, **k: None
    try:
        single = [step(s) for s in range(120, 180, 12)]
    finally:
        blockwise.plan.call = planned
    for a, b in zip(replayed, single):
        assert len(a) == len(b) and all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("warm", [2, 4])
def test_several_weights_captured_and_replayed(dev, warm):
    """Casts and products that share launches, in a graph: captured call by call (2 calls before) and as recorded sequences (4)."""
    from olmo_core_amd.float8 import blockwise

    T = 140 + warm  # (sizes of its own)
    ws = [make((n, 256), 190 + n, std=0.05).to(dev).requires_grad_(True) for n in (272, 64, 48)]
    x = make((T, 256), 191).to(dev).requires_grad_(True)
    gs = [make((T, w.shape[0]), 192 + i).to(dev) for i, w in enumerate(ws)]

    def work():
        ys = blockwise._linears(x, ws, [None] * 3)
        return [y.detach() for y in ys] + list(torch.autograd.grad(ys, [x, *ws], gs))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(warm):
            work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (195, 205, 215, 225):
        with torch.no_grad():
            x.copy_(make((T, 256), seed))
            for i, (w, g) in enumerate(zip(ws, gs)):
                w.copy_(make(w.shape, seed + 1 + i, std=0.05))
                g.copy_(make(g.shape, seed + 5 + i))
        eager = work()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.parametrize("rows", [1, 4, 20, 200])
def test_no_input_features(dev, rows):
    """A sum of no terms is zero for any number of rows."""
    w = torch.empty(48, 0, dtype=BF16, device=dev, requires_grad=True)
    x = torch.empty(rows, 0, dtype=BF16, device=dev, requires_grad=True)
    y = blockwise_linear(x, w)
    assert y.shape == (rows, 48) and not y.any()
    y.sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    sizes = torch.tensor([rows, 0, 0], device=dev)
    with torch.no_grad():
        assert not blockwise_linear(x, w).any() and not blockwise_linear(x, w, kept=blockwise_weight(w)).any()
        z = blockwise_grouped_linear(x, w, sizes)
        assert z.shape == (rows, 16) and not z.any()



def test_compiled_module_keeps_float8_weights(dev, monkeypatch):
    """A compiled module uses the copies that it keeps: its weight is quantised once, in training as in generation, and again after it changed."""
    from olmo_core_amd.float8 import blockwise

    config = Float8LinearConfig.from_recipe_name("blockwise")
    config.enable_fsdp_float8_all_gather = True
    m = Float8Linear(256, 64, bias=False, dtype=BF16, device=dev, config=config)
    compiled = torch.compile(m, backend="eager")
    casts = []
    batch = ops.cast_blockwise_batch
    monkeypatch.setattr(ops, "cast_blockwise_batch", lambda items: casts.extend(kw for _, kw in items if kw.get("square")) or batch(items))
    x, g = make((40, 256), 300).to(dev), make((40, 64), 301).to(dev)
    with torch.no_grad():
        for _ in range(3):
            assert torch.equal(compiled(x), blockwise.blockwise_linear(x, m.weight, kept=blockwise_weight(m.weight)))
        casts.clear()
        compiled(x)
        assert not casts
    a = x.clone().requires_grad_(True)
    compiled(a).backward(g)
    assert not casts
    want = torch.autograd.grad(blockwise_linear(a, m.weight), (a, m.weight), g)
    assert torch.equal(a.grad, want[0]) and torch.equal(m.weight.grad, want[1])
    with torch.no_grad():
        m.weight.mul_(2)
        casts.clear()
        y = compiled(x)
        assert len(casts) == 1 and torch.equal(y, blockwise_linear(x, m.weight))


def _sizes_of(T, E, kind):
    if kind == "comb":  # single rows and nothing in turn around two large groups
        sizes = torch.arange(E) % 2
        sizes[0] = (T - int(sizes.sum())) // 3
        sizes[E - 2] += T - int(sizes.sum())
        return sizes
    return spread(T, E, kind)


def _poison(dev, n, dtype):
    torch.full((n,), float("nan"), dtype=dtype, device=dev)  # (what an output that is not written is likely to hold)


@pytest.mark.parametrize("T,E,N,K", [(6001, 7, 2064, 272), (5001, 16, 2064, 528), (16001, 70, 1040, 528)])
@pytest.mark.parametrize("kind", ["skew", "short", "one", "comb", "none"])
def test_persistent_groups_are_their_products(dev, T, E, N, K, kind):
    """The 256 x 256 kernel on several groups that have rows, also more than a wave's 64: the bits of the ring tiles on each group alone."""
    assert ops._C.lib().mi8_grouped_gemm_fp8_block_variant(T, N, K, E, ops._HP_CODE[BF16]) == 3
    x, w = make((T, K), 400).to(dev), make((E * N, K), 401, std=0.05).to(dev)
    sizes = _sizes_of(T, E, kind)
    on_gpu = sizes.to(dev)
    a, sa, _, _ = ops.grouped_cast_blockwise(x, on_gpu)
    b, sb, _, _ = ops.cast_blockwise(w, square=True, matrices=E)
    _poison(dev, T * N, BF16)
    y = ops.grouped_gemm_fp8_blockwise(a, sa, b, sb, on_gpu, n=N, k=K)
    first = unit = 0
    for e, m in enumerate(sizes.tolist()):
        if m:
            rows, tiles = slice(first, first + m), -(-m // 128)
            want = ops.gemm_fp8_blockwise(a[rows], sa[:, 128 * unit:128 * (unit + tiles)].contiguous(), b[e * N:(e + 1) * N], sb[e], k=K, variant=0)
            assert torch.equal(y[rows], want), (e, m)
            first, unit = first + m, unit + tiles
    assert first <= T and not y[first:].any()
    assert torch.equal(blockwise_grouped_linear(x, w, on_gpu), y)


@pytest.mark.parametrize("T,E,N,K", [(3001, 9, 784, 1296), (3001, 16, 2064, 1040), (12001, 70, 1296, 1296), (12001, 100, 256, 512)])
@pytest.mark.parametrize("kind", ["skew", "short", "one", "comb", "none"])
def test_persistent_weight_gradients_are_their_products(dev, T, E, N, K, kind):
    """The same for the products over the tokens of groups."""
    assert ops._C.lib().mi8_grouped_wgrad_fp8_block_variant(T, N, K, E, ops._HP_CODE[BF16]) == 3
    g, x = make((T, N), 402, std=1e-3).to(dev), make((T, K), 403).to(dev)
    sizes = _sizes_of(T, E, kind)
    on_gpu = sizes.to(dev)
    _, _, a, sa = ops.grouped_cast_blockwise(g, on_gpu, want_rowmajor=False, want_transposed=True)
    _, _, b, sb = ops.grouped_cast_blockwise(x, on_gpu, want_rowmajor=False, want_transposed=True)
    _poison(dev, E * N * K, BF16)
    gw = ops.grouped_wgrad_fp8_blockwise(a, sa, b, sb, on_gpu, tokens=T)
    unit = 0
    for e, m in enumerate(sizes.tolist()):
        tiles = -(-m // 128)
        if m:
            here = slice(unit, unit + tiles)
            cols = slice(128 * unit, 128 * (unit + tiles))
            want = ops.gemm_fp8_blockwise(a[:, cols], sa[here], b[:, cols], sb[here], k=128 * tiles, variant=0)
            assert torch.equal(gw[e], want), (e, m)
            unit += tiles
        else:
            assert not gw[e].any(), e



def _recorded(plan):
    """How many sequences of this package's block-scaled calls are in the tables, forward and backward."""
    ours = [p for k, p in plan._plans.items() if k[0][0] == "blockwise"]
    return sum(type(p) is plan.Plan for p in ours), sum(type(q) is plan.Plan for p in ours if type(p) is plan.Plan for q in p.then.values())


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("M", [5, 100])
def test_calls_that_are_replayed_were_recorded(dev, monkeypatch, M, captured):
    """One linear, three on one input and one of experts, on tables of their own: from the third call on each is a recorded sequence, forward and
    backward, also where it is captured into a graph, and gives the bits of the calls one by one."""
    from olmo_core_amd.float8 import blockwise

    plan = blockwise.plan
    monkeypatch.setattr(plan, "_plans", {})
    monkeypatch.setattr(plan, "_seen", {})
    w = make((272, 400), 410, std=0.05).to(dev).requires_grad_(True)
    ws = [make((n, 400), 411 + n, std=0.05).to(dev).requires_grad_(True) for n in (48, 64, 16)]
    we = make((4 * 48, 400), 412, std=0.05).to(dev).requires_grad_(True)
    sizes = spread(M, 4, "skew").to(dev)
    x = make((M, 400), 413).to(dev).requires_grad_(True)
    gs = [make((M, n), 414 + n).to(dev) for n in (272, 48, 64, 16, 48)]

    def work():
        ys = [blockwise_linear(x, w), *blockwise._linears(x, ws, [None] * 3), blockwise_grouped_linear(x, we, sizes)]
        with torch.no_grad():
            alone = blockwise_linear(x, w)
        grads = []
        for part, leaves, g in ((ys[:1], (x, w), gs[:1]), (ys[1:4], (x, *ws), gs[1:4]), (ys[4:], (x, we), gs[4:])):
            grads += torch.autograd.grad(part, leaves, g)
        return [y.detach() for y in ys] + [alone] + grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            work()
    torch.cuda.current_stream().wait_stream(side)
    assert _recorded(plan) == (4, 3)
    assert all(type(p) is plan.Plan for p in plan._plans.values())
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
    for seed in (420, 421, 422):
        with torch.no_grad():
            x.copy_(make((M, 400), seed))
            w.copy_(make((272, 400), seed + 10, std=0.05))
        if captured:
            graph.replay()
        else:
            out = work()
        torch.cuda.synchronize()
        with monkeypatch.context() as one_by_one:
            one_by_one.setattr(plan, "call", lambda *a, **k: None)
            want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert _recorded(plan) == (4, 3)

@pytest.mark.parametrize("kind", ["blockwise", "tensorwise", "experts blockwise", "experts rowwise"])
def test_copies_made_inside_a_capture_are_not_kept(dev, kind):
    """The first call of a module that keeps its float8 weight is captured: the copies are the graph's, which has not run yet, and no call outside may read
    them.  Replays see the weight as it is then."""
    from olmo_core_amd.nn import DroplessMoEMLP

    torch.manual_seed(5)
    if kind.startswith("experts"):
        m = DroplessMoEMLP(d_model=256, hidden_size=144, num_experts=3, dtype=BF16, init_device=dev, keep_float8_weights=True, scaling=kind.split()[1])
        sizes = torch.tensor([20, 0, 13], device=dev)
        call, weight = (lambda x: m(x, sizes)), m.w2
    else:
        config = Float8LinearConfig.from_recipe_name(kind)
        config.enable_fsdp_float8_all_gather = True
        m = Float8Linear(256, 64, bias=False, dtype=BF16, device=dev, config=config)
        call, weight = m, m.weight
    x = make((33, 256), 430).to(dev)
    scratch = [torch.full((1 << 20,), 7.0, device=dev) for _ in range(4)]  # (what the graph's memory may hold before its first replay)
    del scratch
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            out = call(x)
        assert m.__dict__.get("_kept") is None and m.__dict__.get("_weight_operands") is None
        eager = call(x).clone()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
        weight.mul_(2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, 2 * eager)
        assert torch.equal(call(x), 2 * eager) and m.weight_operands() is m.weight_operands()
