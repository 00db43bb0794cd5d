"""
Products in bf16 and float16 (``ops.linear``, ``ops.grouped_linear``) against the formulas in 64 bits.

Small integers as inputs: every product and partial sum is a whole number below 2^24, so float32 sums are exact whatever their order and the result is the
exact one rounded once, bit for bit.  Real inputs: a float32 sum of K products is off by at most K 2^-23 times the sum of their magnitudes, the epilogue's
few operations and the exponential by 2^-20 of their largest operand, and the rounding by eps / 2 of the value (:func:`_bound`).
"""

import ctypes
import math

import pytest
import torch

from olmo_core_amd import _C
from olmo_core_amd.ops import linear as L
from olmo_core_amd.ops.linear import grouped_linear, linear

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
VARIANTS = {"256": _C.HALF_256, "128": _C.HALF_128, "64": _C.HALF_64}


def _ints(g, *shape, most=3, dtype=BF16):
    return torch.randint(-most, most + 1, shape, generator=g).to(dtype).cuda()


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _act64(name, z):
    if name == "relu":
        return torch.relu(z)  # (its slope at 0 is 0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    if name == "gelu_tanh":
        # (1 + tanh u) / 2 = 1 / (1 + e^-2u), which keeps its digits where 1 + tanh u has none left in 64 bits
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def _close(got, want, sums, k, what=""):
    """``sums``: the sums of the products' magnitudes (and of what is added to them)."""
    eps = torch.finfo(got.dtype).eps
    bound = eps / 2 * want.abs() * (1 + 1e-3) + (k * 2.0 ** -23 + 2.0 ** -20) * sums + torch.finfo(got.dtype).smallest_normal * eps
    worst = ((got.double() - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, f"{what}: {worst} times the bound"


@pytest.fixture(params=list(VARIANTS))
def variant(request, monkeypatch):
    """The kernel that every product of the test runs on."""
    monkeypatch.setattr(_C, "HALF_ANY", VARIANTS[request.param])
    return request.param


# 1 to more than a tile, odd, of one step of K and of several, none a multiple of a tile
SIZES = [(1, 8, 8), (1, 1, 1), (3, 5, 7), (16, 16, 64), (63, 65, 129), (130, 264, 200), (257, 300, 72), (300, 520, 640), (513, 1031, 331)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_whole_numbers_are_exact(variant, dtype, m, n, k):
    g = _gen(m * n + k)
    x, w, gy = _ints(g, m, k, dtype=dtype), _ints(g, n, k, dtype=dtype), _ints(g, m, n, dtype=dtype)
    x.requires_grad_(True), w.requires_grad_(True)
    y = linear(x, w)
    assert y.shape == (m, n) and y.is_contiguous() and y.dtype == dtype
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    x64, w64, g64 = x.detach().double(), w.detach().double(), gy.double()
    for name, got, want in (("y", y, x64 @ w64.t()), ("gx", gx, g64 @ w64), ("gw", gw, g64.t() @ x64)):
        assert torch.equal(got, want.to(dtype)), name


@pytest.mark.parametrize("m,n,k", [(700, 520, 1100), (300, 2000, 64), (256, 256, 4096)])
def test_several_tiles_a_workgroup(m, n, k, variant, monkeypatch):
    """A grid smaller than the number of tiles: the walk over tiles and what is loaded ahead of it (sizes of a whole chip are in the full shapes)."""
    g = _gen(5)
    many = 9 if variant == "64" else 3
    x, w = _ints(g, m * many, k, most=1), _ints(g, n * many, k, most=1)
    assert torch.equal(linear(x, w), (x.double() @ w.double().t()).to(BF16))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", SIZES + [(192, 256, 128), (193, 257, 64), (777, 520, 1100), (1500, 2000, 264)])
def test_tiles_of_192_rows(monkeypatch, dtype, m, n, k):
    """For products whose A lies by rows: forward with every epilogue, gradient of the input."""
    monkeypatch.setattr(_C, "HALF_ANY", _C.HALF_192)
    g = _gen(m + 3 * n + k)
    x, w, b, r, gy = _ints(g, m, k, dtype=dtype), _ints(g, n, k, dtype=dtype), _ints(g, n, dtype=dtype), _ints(g, m, n, dtype=dtype), _ints(g, m, n, dtype=dtype)
    want = x.double() @ w.double().t()
    assert torch.equal(linear(x, w), want.to(dtype))
    assert torch.equal(linear(x, w, b.float(), activation="relu", residual=r), (torch.relu(want + b.double()) + r.double()).to(dtype))
    x.requires_grad_(True)
    y = linear(x, w, b, activation="relu", residual=r)
    assert torch.equal(y, (torch.relu(want + b.double()) + r.double()).to(dtype))
    (gx,) = torch.autograd.grad(y, x, gy)
    assert torch.equal(gx, ((gy.double() * (want + b.double() > 0)) @ w.double()).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (1, 1, 1), (2, 33, 520), (15, 64, 4096), (16, 16, 72), (16, 100, 1001), (9, 31, 64), (16, 129, 2000), (13, 520, 513), (16, 16, 11008)])
def test_few_rows(monkeypatch, dtype, m, n, k):
    monkeypatch.setattr(_C, "HALF_ANY", _C.HALF_ROWS)
    g = _gen(m + n + k)
    x, w, b, r = _ints(g, m, k, dtype=dtype), _ints(g, n, k, dtype=dtype), _ints(g, n, dtype=dtype), _ints(g, m, n, dtype=dtype)
    want = x.double() @ w.double().t()
    assert torch.equal(linear(x, w), want.to(dtype))
    assert torch.equal(linear(x, w, b, activation="relu", residual=r), (torch.relu(want + b.double()) + r.double()).to(dtype))
    assert torch.equal(linear(x, w, b.float()), (want + b.double()).to(dtype))


@pytest.mark.parametrize("m,n,k,a_by_k,b_by_k", [(48, 4096, 11008, 0, 0), (200, 512, 4096, 0, 1), (100, 131, 3001, 0, 0), (256, 200, 9000, 1, 1), (130, 70, 5000, 1, 1)])
def test_slices_of_k(m, n, k, a_by_k, b_by_k):
    """Few tiles and a long K: cut along K, joined with the epilogue; without a workspace the same product in one piece."""
    slices = ctypes.c_int32()
    assert _C.lib().mi8_gemm_half_variant(m, n, k, a_by_k, b_by_k, slices) in (_C.HALF_64, _C.HALF_128) and slices.value > 1
    g = _gen(k)
    a, b = _ints(g, *((k, m) if a_by_k else (m, k)), most=1), _ints(g, *((k, n) if b_by_k else (n, k)), most=1)
    bias, r = _ints(g, n), _ints(g, m, n)
    ao, bo = L._operand(a), L._operand(b)
    want = (a.double().t() if a_by_k else a.double()) @ (b.double() if b_by_k else b.double().t())
    ep = _C.HalfEpilogue(activation=_C.ACT_RELU, bias=bias.data_ptr(), bias_dtype=_C.MI8_BF16, residual=r.data_ptr(), ld_residual=n)
    assert torch.equal(L._product(ao, bo, m, n, k, a_by_k, b_by_k), want.to(BF16))
    joined = (torch.relu(want + bias.double()) + r.double()).to(BF16)
    assert torch.equal(L._product(ao, bo, m, n, k, a_by_k, b_by_k, ctypes.byref(ep)), joined)
    out = torch.empty(m, n, dtype=BF16, device="cuda")
    _C.check(_C.lib().mi8_gemm_half(_C.MI8_BF16, ao.data_ptr(), L._operand_pitch(ao), a_by_k, bo.data_ptr(), L._operand_pitch(bo), b_by_k, m, n, k, ctypes.byref(ep),
                                    out.data_ptr(), n, _C.HALF_ANY, None, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out, joined)


@pytest.mark.parametrize("m,n,k", [(16384, 1024, 200), (5000, 5000, 320), (200, 33000, 136)])
def test_more_tiles_than_the_chip_holds(m, n, k):
    g = _gen(6)
    x, w = _ints(g, m, k, most=1), _ints(g, n, k, most=1)
    for v in (*VARIANTS.values(), _C.HALF_192):
        out = torch.empty(m, n, dtype=BF16, device="cuda")
        _C.check(_C.lib().mi8_gemm_half(_C.MI8_BF16, x.data_ptr(), k, 0, w.data_ptr(), k, 0, m, n, k, None, out.data_ptr(), n, v, None, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out, (x.double() @ w.double().t()).to(BF16)), v


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k,bias,residual", [(70, 136, 200, True, True), (33, 67, 45, True, True), (260, 264, 128, False, True), (5, 24, 8, True, False)])
def test_epilogue_and_gradients(dtype, activation, m, n, k, bias, residual):
    g = _gen(k)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    x, w = rand(m, k), (rand(n, k).float() * (3 / math.sqrt(k))).to(dtype)
    b = rand(n) if bias else None
    r = rand(m, n) if residual else None
    gy = rand(m, n)
    ins = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    y = linear(x, w, b, activation=activation, residual=r)
    grads = dict(zip([nm for nm, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None], torch.autograd.grad(y, ins, gy)))
    x64, w64, g64 = x.detach().double(), w.detach().double(), gy.double()
    b64 = b.detach().double() if bias else torch.zeros(n, device="cuda").double()
    z = x64 @ w64.t() + b64
    zsum = x64.abs() @ w64.abs().t() + b64.abs()
    want = _act64(activation, z)
    wsum = 1.2 * zsum  # (no activation's slope passes 1.13)
    if residual:
        want, wsum = want + r.detach().double(), wsum + r.detach().double().abs()
        assert torch.equal(grads["r"], gy)
    _close(y.detach(), want, wsum, k, "y")
    # the slope is taken at the rounded argument: it is off by at most its own slope (below 1.2) times the rounding and the sum's error
    zr = z.detach().requires_grad_(True)
    slope = torch.autograd.grad(_act64(activation, zr).sum(), zr)[0]
    eps = torch.finfo(dtype).eps
    dz = g64 * slope
    if activation == "relu":  # (a step at 0: where the argument's sign is in doubt either side is right)
        dz_err = g64.abs() * ((z.abs() <= k * 2.0 ** -22 * zsum).double())
    elif activation is None:
        dz_err = torch.zeros_like(dz)
    else:
        dz_err = g64.abs() * 1.2 * (eps / 2 * z.abs() + k * 2.0 ** -23 * zsum + 2.0 ** -19)
    if activation is not None:
        dz_err = dz_err + eps / 2 * (dz.abs() + dz_err)  # rounded to the operands' type
    for name, got, left, right, length in (("gx", grads["x"], (dz, dz_err), w64, n), ("gw", grads["w"], (dz.t(), dz_err.t()), x64, m)):
        value, err = left
        want = value @ right
        bound = err @ right.abs() + length * 2.0 ** -23 * (value.abs() + err) @ right.abs()
        bound = bound + eps / 2 * (want.abs() + bound) + 1e-7
        worst = ((got.double() - want).abs() / bound).max().item()
        assert worst <= 1, (name, worst)
    if bias:
        err = (g64.abs() * 1.2 * (eps / 2 * z.abs() + k * 2.0 ** -23 * zsum + 2.0 ** -19)).sum(0) if activation not in (None, "relu") else dz_err.sum(0)
        bound = err + (m + 4) * 2.0 ** -23 * (dz.abs().sum(0) + err)
        bound = bound + eps / 2 * (dz.sum(0).abs() + bound) + 1e-7
        assert ((grads["b"].double() - dz.sum(0)).abs() <= bound).all()


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_gradient_agrees_with_differences(activation):
    """The slope of the layer itself, by central differences of its own 64-bit definition around inputs that float16 holds."""
    g = _gen(2)
    x = (torch.randn(40, 32, generator=g)).to(F16).cuda().requires_grad_(True)
    w = (torch.randn(24, 32, generator=g) * 0.3).to(F16).cuda()
    gy = torch.randn(40, 24, generator=g).to(F16).cuda()
    gx = torch.autograd.grad(linear(x, w, activation=activation), x, gy)[0]
    f = lambda v: (_act64(activation, v @ w.double().t()) * gy.double()).sum(1)  # noqa: E731
    x64, h = x.detach().double(), 1e-5
    for c in (0, 7, 31):
        step = torch.zeros_like(x64)
        step[:, c] = h
        slope = (f(x64 + step) - f(x64 - step)) / (2 * h)
        scale = (gy.double().abs() @ w.double().abs())[:, c]
        assert ((gx[:, c].double() - slope).abs() <= 2.0 ** -9 * scale).all()  # (the slope's argument, the slope and the sum: three half steps of 2^-11)


@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu", "gelu_tanh"])
def test_activation_over_its_whole_range(activation):
    """The identity as weight: y is the activation of x itself, within a rounding and 2^-15 of the value (where that is a normal number).

    2^-15: the value is at worst e^a times what is exact to 2^-20, |a| < 100 (e^-100 is below 2^-126), and a is made with at most three roundings of
    2^-24 of itself and the constants' own: a relative error of e^a of 100 * 4 * 2^-24 < 2^-15."""
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(BF16)
    x = x[x.isfinite()]
    x = x[: x.numel() // 64 * 64].view(-1, 64).cuda().requires_grad_(True)
    w = torch.eye(64, dtype=BF16, device="cuda")
    y = linear(x, w, activation=activation)
    x64 = x.detach().double().requires_grad_(True)
    want = _act64(activation, x64)
    slope = torch.autograd.grad(want.sum(), x64)[0].nan_to_num()
    ok = x64.detach().abs() < 1e18
    err = (y.double() - want.detach()).abs()
    assert (err[ok] <= (2.0 ** -8 + 2.0 ** -15) * want.detach().abs()[ok] + 2.0 ** -100).all()
    gx = torch.autograd.grad(y, x, torch.ones_like(y))[0]
    err = (gx.double() - slope).abs()
    assert (err[ok] <= 2.0 ** -7 * slope.abs()[ok] + 2.0 ** -18).all()  # (two roundings: dz, gx)
    assert gx.isfinite().all()


def test_not_finite_values_stay_in_their_row():
    g = _gen(3)
    x, w = _ints(g, 200, 72), _ints(g, 136, 72)
    for bad in (math.nan, math.inf):
        xb = x.clone()
        xb[77, 71] = bad
        w1 = w.clone()
        w1[:, 71] = 1
        y = linear(xb, w1)
        want = (xb.double() @ w1.double().t()).to(BF16)
        rows = torch.arange(200) != 77
        assert torch.equal(y[rows], want[rows])
        assert y[77].isnan().all() if bad != bad else y[77].isinf().all()
    # ... nor does a tensor's neighbourhood reach in: a view of a larger one that is NaN all around
    big = torch.full((300, 200), math.nan, dtype=BF16, device="cuda")
    big[16:216, 8:80] = x
    y = linear(big[16:216, 8:80], w)
    assert torch.equal(y, (x.double() @ w.double().t()).to(BF16))
    big[16:216, 8:77] = x[:, :69]
    big[:, 77:] = math.nan
    assert torch.equal(linear(big[16:216, 8:77], w[:, :69]), (x[:, :69].double() @ w[:, :69].double().t()).to(BF16))


def test_shapes_strides_and_empty():
    g = _gen(4)
    w = _ints(g, 40, 48)
    x = _ints(g, 2, 3, 5, 48)
    want = (x.double() @ w.double().t()).to(BF16)
    assert torch.equal(linear(x, w), want)
    assert torch.equal(linear(x[0, 0, 0], w), want[0, 0, 0])
    assert torch.equal(linear(x.transpose(0, 2), w), want.transpose(0, 2))
    assert torch.equal(linear(x[:, :, ::2], w), want[:, :, ::2])
    assert torch.equal(linear(x.flip(0), w), want.flip(0))
    assert torch.equal(linear(x[:1, :1, :1].expand(4, 2, 3, 48), w), want[:1, :1, :1].expand(4, 2, 3, 40))
    wt = w.t().contiguous()
    assert torch.equal(linear(x, wt.t()), want)
    odd = torch.empty(40 * 48 + 1, dtype=BF16, device="cuda")[1:].view(40, 48).copy_(w)
    assert torch.equal(linear(x, odd), want)
    r = _ints(g, 5, 2, 3, 40)
    assert torch.equal(linear(x, w, residual=r.permute(1, 2, 0, 3)), (want.double() + r.permute(1, 2, 0, 3).double()).to(BF16))
    for shape in ((0, 48), (2, 0, 48)):
        xe = torch.empty(shape, dtype=BF16, device="cuda", requires_grad=True)
        we = w.clone().requires_grad_(True)
        be = torch.zeros(40, device="cuda", requires_grad=True)
        y = linear(xe, we, be, activation="gelu")
        assert y.shape == (*shape[:-1], 40)
        gx, gw, gb = torch.autograd.grad(y, [xe, we, be], torch.empty_like(y))
        assert gx.shape == shape and not gw.any() and not gb.any()
    b = torch.randn(40, generator=g).cuda()
    no_features = linear(torch.empty(7, 0, dtype=BF16, device="cuda"), torch.empty(40, 0, dtype=BF16, device="cuda"), b)
    assert torch.equal(no_features, b.to(BF16).expand(7, 40))
    assert linear(x, w[:0]).shape == (2, 3, 5, 0)


def test_rows_that_lie_over_one_another():
    """Expanded inputs, residuals and gradients (a row's stride of zero), whole chunks or not."""
    g = _gen(21)
    for n, k in ((40, 48), (37, 45)):
        x, w, r, gy = _ints(g, 1, k), _ints(g, n, k), _ints(g, 1, n), _ints(g, 1, n)
        b = _ints(g, n)
        xe, re, ge = x.expand(20, k), r.expand(20, n), gy.expand(20, n)
        want = x.double() @ w.double().t() + b.double()
        assert torch.equal(linear(xe, w, b, residual=re), (want + r.double()).to(BF16).expand(20, n))
        ins = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        for activation, slope in ((None, torch.ones_like(want)), ("relu", (want > 0).double())):
            y = linear(ins[0].expand(20, k), ins[1], ins[2], activation=activation, residual=ins[3].expand(20, n))
            made = torch.autograd.grad(y, ins[1:3], ge)
            dz = gy.double() * slope
            assert torch.equal(made[0], (20 * dz.t() @ x.double()).to(BF16)) and torch.equal(made[1], (20 * dz[0]).to(BF16))
            y = linear(xe.clone().requires_grad_(True), w, b, activation=activation)
            assert torch.equal(torch.autograd.grad(y, y.grad_fn.next_functions[0][0].variable, ge)[0], (dz @ w.double()).to(BF16).expand(20, k))


def test_offsets_past_32_bits():
    """Operands and outputs of more than 2^31 elements: the last rows are what they are alone."""
    rows, k, n = (1 << 19) + 131, 4104, 4120
    w = _ints(_gen(1), n, k, most=1)
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    x[-300:] = _ints(_gen(2), 300, k, most=1)
    y = linear(x, w)
    assert torch.equal(y[-300:], (x[-300:].double() @ w.double().t()).to(BF16)) and not y[:-300].any()
    del y
    sizes = torch.tensor([rows - 200, 200], device="cuda")
    two = torch.cat([torch.zeros_like(w[:64]), w[:64]])
    y = grouped_linear(x, two, sizes)
    assert torch.equal(y[-200:], (x[-200:].double() @ w[:64].double().t()).to(BF16)) and not y[:-200].any()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_tiles_of_all_sizes_give_the_same_bits(dtype):
    """One order of summation, and one rounding whether results pass through LDS or not."""
    g = _gen(31)
    x, w = torch.randn(300, 1000, generator=g).to(dtype).cuda(), torch.randn(520, 1000, generator=g).to(dtype).cuda()
    zero = torch.zeros(520, dtype=dtype, device="cuda")
    outs = []
    for v in (*VARIANTS.values(), _C.HALF_192):
        for ep in (None, _C.HalfEpilogue(bias=zero.data_ptr(), bias_dtype=L._CODE[dtype])):
            out = torch.empty(300, 520, dtype=dtype, device="cuda")
            _C.check(_C.lib().mi8_gemm_half(L._CODE[dtype], x.data_ptr(), 1000, 0, w.data_ptr(), 1000, 0, 300, 520, 1000, ctypes.byref(ep) if ep else None, out.data_ptr(), 520, v,
                                            None, torch.cuda.current_stream().cuda_stream))
            outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_two_threads_on_two_streams():
    import threading

    g = _gen(32)
    ins = [(_ints(g, 200, 264), _ints(g, 136, 264), _ints(g, 136)) for _ in range(2)]
    want = [torch.relu(x.double() @ w.double().t() + b.double()).to(BF16) for x, w, b in ins]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        x, w, b = ins[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y = linear(x, w, b, activation="relu")
                y2 = grouped_linear(x, w, torch.tensor([200], device="cuda"))
            torch.cuda.current_stream().synchronize()
            if not torch.equal(y, want[i]) or not torch.equal(y2, (x.double() @ w.double().t()).to(BF16)):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_gradients_only_of_what_is_asked():
    g = _gen(8)
    x, w, b, r = _ints(g, 9, 16), _ints(g, 24, 16), _ints(g, 24), _ints(g, 9, 24)
    gy = _ints(g, 9, 24)
    for which in range(4):
        ins = [t.clone() for t in (x, w, b, r)]
        ins[which].requires_grad_(True)
        y = linear(ins[0], ins[1], ins[2], residual=ins[3])
        want = (gy.double() @ w.double(), gy.double().t() @ x.double(), gy.double().sum(0), gy.double())[which]
        assert torch.equal(torch.autograd.grad(y, ins[which], gy)[0], want.to(BF16))
    # a gradient that is a view with odd strides, and one value everywhere
    x.requires_grad_(True)
    y = linear(x, w)
    assert torch.equal(torch.autograd.grad(y, x, gy.t().contiguous().t(), retain_graph=True)[0], (gy.double() @ w.double()).to(BF16))
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], w.double().sum(0).to(BF16).expand(9, 16))


# ---- rows sorted by expert -------------------------------------------------------------------------------------

GROUPS = [
    ([5, 0, 17, 1], 30, 72, 40),            # an empty group, one row, rows behind the last group
    ([0, 0, 0], 9, 16, 24),                  # nothing but empty groups
    ([70, 130, 3, 64, 200], 467, 136, 200),  # more than a tile of a group
    ([300, 1, 257], 558, 264, 328),
    ([33, 21, 11], 65, 45, 37),              # nothing a multiple of 8
    ([2] * 70, 140, 24, 16),                 # more groups than lanes
    ([40], 40, 64, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
@pytest.mark.parametrize("sizes,rows,n,k", GROUPS, ids=[str(i) for i in range(len(GROUPS))])
def test_groups(variant, dtype, transposed, sizes, rows, n, k):
    g = _gen(rows + n)
    E = len(sizes)
    x = _ints(g, rows, k, dtype=dtype).requires_grad_(True)
    w = _ints(g, *((E * k, n) if transposed else (E * n, k)), dtype=dtype).requires_grad_(True)
    gy = _ints(g, rows, n, dtype=dtype)
    y = grouped_linear(x, w, torch.tensor(sizes, device="cuda"), transposed=transposed)
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    want_y, want_gx, want_gw = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (y, x, w))
    first = 0
    for e, size in enumerate(sizes):
        here = slice(first, first + size)
        first += size
        we = w.detach().double().chunk(E)[e]
        we = we if transposed else we.t()
        want_y[here] = x.detach().double()[here] @ we
        want_gx[here] = gy.double()[here] @ we.t()
        ge = x.detach().double()[here].t() @ gy.double()[here]
        want_gw.chunk(E)[e].copy_(ge if transposed else ge.t())
    for name, got, want in (("y", y, want_y), ("gx", gx, want_gx), ("gw", gw, want_gw)):
        assert torch.equal(got, want.to(dtype)), name


def test_group_sizes_of_any_kind():
    g = _gen(9)
    x, w = _ints(g, 50, 16), _ints(g, 3 * 8, 16)
    want = grouped_linear(x, w, torch.tensor([10, 15, 25], device="cuda"))
    assert torch.equal(grouped_linear(x, w, torch.tensor([10, 15, 25], device="cuda", dtype=torch.int32)), want)
    assert torch.equal(grouped_linear(x, w, torch.tensor([10, 9, 15, 9, 25], device="cuda")[::2]), want)
    assert torch.equal(grouped_linear(x.view(5, 10, 16), w, torch.tensor([10, 15, 25])), want.view(5, 10, 8))
    # sizes that pass the rows are cut off, negative ones count as none: nothing past the tensors is touched
    got = grouped_linear(x, w, torch.tensor([10, -4, 400], device="cuda"))
    assert torch.equal(got[10:], (x[10:].double() @ w[16:].double().t()).to(BF16)) and torch.equal(got[:10], want[:10])
    empty = grouped_linear(x[:0], w, torch.tensor([0, 0, 0], device="cuda"))
    assert empty.shape == (0, 8)
    we = w.clone().requires_grad_(True)
    assert not torch.autograd.grad(grouped_linear(x[:0], we, torch.tensor([0, 0, 0], device="cuda")).sum(), we)[0].any()


def test_no_rows_at_all():
    w = torch.randn(3 * 16, 24, device="cuda").to(BF16).requires_grad_(True)
    x = torch.empty(0, 24, dtype=BF16, device="cuda", requires_grad=True)
    y = grouped_linear(x, w, torch.zeros(3, dtype=torch.int64, device="cuda"))
    gx, gw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
    assert y.shape == (0, 16) and gx.shape == (0, 24) and gw.shape == w.shape and not gw.any()


def test_rows_behind_the_last_group_do_not_reach_a_gradient():
    g = _gen(10)
    x, w = _ints(g, 50, 16), _ints(g, 2 * 24, 16)
    x[30:] = math.nan
    gy = _ints(g, 50, 24)
    gy[30:] = math.inf
    x.requires_grad_(True), w.requires_grad_(True)
    y = grouped_linear(x, w, torch.tensor([13, 17], device="cuda"))
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    assert not y[30:].any() and not gx[30:].any() and gw.isfinite().all() and gx.isfinite().all()


# ---- streams, graphs, devices' state ------------------------------------------------------------------------------


def test_on_another_stream_and_captured():
    g = _gen(11)
    x, w, b = _ints(g, 130, 72), _ints(g, 264, 72), _ints(g, 264)
    gy = _ints(g, 130, 264)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)

    def step():
        y = linear(x, w, b, activation="relu")
        return (y, *torch.autograd.grad(y, [x, w, b], gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(outs, want):
            assert torch.equal(got, expected)
        eager = step()
        for got, expected in zip(eager, want):
            assert torch.equal(got, expected)
        for t in outs:
            t.detach().zero_()
    # new values in the same places
    with torch.no_grad():
        x.copy_(_ints(g, 130, 72))
    want = [t.clone() for t in step()]
    graph.replay()
    torch.cuda.synchronize()
    for got, expected in zip(outs, want):
        assert torch.equal(got, expected)


def test_weight_modified_between_forward_and_backward_is_noticed():
    x, w = torch.ones(8, 16, dtype=BF16, device="cuda", requires_grad=True), torch.ones(8, 16, dtype=BF16, device="cuda")
    y = linear(x, w)
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_library_refuses_what_its_kernels_cannot_read():
    x = torch.zeros(64, 64, dtype=BF16, device="cuda")
    out = torch.full((64, 64), 3.0, dtype=BF16, device="cuda")

    def call(dtype=_C.MI8_BF16, a=x.data_ptr(), lda=64, a_by_k=0, b=x.data_ptr(), ldb=64, b_by_k=0, m=64, n=64, k=64, ep=None, ldc=64, variant=0):
        return _C.lib().mi8_gemm_half(dtype, a, lda, a_by_k, b, ldb, b_by_k, m, n, k, ep, out.data_ptr(), ldc, variant, None, torch.cuda.current_stream().cuda_stream)

    for bad in (dict(dtype=_C.MI8_F32), dict(a=x.data_ptr() + 2), dict(lda=60), dict(lda=56), dict(ldb=1 << 22), dict(ldc=63), dict(a_by_k=1), dict(m=-1),
                dict(variant=9), dict(variant=_C.HALF_192, a_by_k=1, b_by_k=1), dict(a=None), dict(k=1 << 30), dict(ep=_C.HalfEpilogue(activation=7)), dict(ep=_C.HalfEpilogue(bias=x.data_ptr(), bias_dtype=_C.MI8_F16)),
                dict(ep=_C.HalfEpilogue(residual=x.data_ptr(), ld_residual=63))):
        assert call(**bad) < 0, bad
        assert _C.last_error()
    torch.cuda.synchronize()
    assert (out == 3).all()
    assert call() == 0
    torch.cuda.synchronize()
    assert not out.any()
    assert L._is_operand(x)


# ---- more tiles than workgroups live at once, behind every epilogue -----------------------------------------------------------

# (256 workgroups of the large tiles live on the chip, 512 of the others: 324 tiles of 256 x 256, 414 of 192 x 256, 1225 of 128 x 128, 4761 of 64 x 64)
MANY = (4400, 4360)


@pytest.mark.parametrize("k", [64, 200], ids=["one_step", "steps"])
@pytest.mark.parametrize("n", [MANY[1], MANY[1] - 3], ids=["whole", "odd"])
@pytest.mark.parametrize("name", [*VARIANTS, "192"])
def test_next_tile_behind_every_epilogue(monkeypatch, name, n, k):
    """A workgroup's second tile starts while the first one's results are still being stored: bias, activation, residual and z, alone and together, on
    outputs whose rows are whole chunks and on others.  Sums stay below 2^8, so that bf16 holds them."""
    monkeypatch.setattr(_C, "HALF_ANY", {**VARIANTS, "192": _C.HALF_192}[name])
    m = MANY[0]
    g = _gen(n + k)
    x, w, b, r = _ints(g, m, k, most=1), _ints(g, n, k, most=1), _ints(g, n), _ints(g, m, n)
    xo, wo = L._operand(x), L._operand(w)
    product = x.double() @ w.double().t()
    assert product.abs().max() < 240
    for bias, act, residual, keep in ((True, "relu", True, False), (True, "relu", False, True), (True, "relu", True, True), (True, None, False, False),
                                      (False, None, True, False), (False, None, False, False)):
        z = torch.full((m, L._pad8(n)), math.nan, dtype=BF16, device="cuda") if keep else None
        y = L._forward(xo, wo, n, k, b if bias else None, r if residual else None, L.ACTIVATIONS[act] if act else _C.ACT_NONE, z)
        want = product + b.double() if bias else product
        if keep:
            assert torch.equal(z[:, :n], want.to(BF16)), (bias, act, residual)
        want = torch.relu(want) if act else want
        assert torch.equal(y, (want + r.double() if residual else want).to(BF16)), (bias, act, residual, keep)


@pytest.mark.parametrize("n", [MANY[1], MANY[1] - 3], ids=["whole", "odd"])
@pytest.mark.parametrize("name", [*VARIANTS, "192"])
def test_next_tile_of_gradients(monkeypatch, name, n):
    """The same for operands that lie by K: the gradient of the input, and that of the weight."""
    monkeypatch.setattr(_C, "HALF_ANY", {**VARIANTS, "192": _C.HALF_192}[name])
    m, k = MANY[0], 200
    g = _gen(n)
    a, b = L._operand(_ints(g, m, k, most=1)), L._operand(_ints(g, k, n, most=1))
    assert torch.equal(L._product(a, b, m, n, k, False, True), (a.double() @ b[:, :n].double()).to(BF16))
    if name != "192":
        a = _ints(g, k, m, most=1)
        assert torch.equal(L._product(a, b, m, n, k, True, True), (a.double().t() @ b[:, :n].double()).to(BF16))


@pytest.mark.parametrize("n", [2104, 2101], ids=["whole", "odd"])
def test_next_tile_of_groups(variant, n):
    """Rows in groups: 45 x 9 tiles of 256 x 256 and more of the others."""
    g = _gen(n)
    sizes = [1500, 0, 700, 1, 2500, 64, 900, 2300, 999]
    rows, k = 9000, 136
    x, w = _ints(g, rows, k, most=1), _ints(g, len(sizes) * n, k, most=1)
    y = grouped_linear(x, w, torch.tensor(sizes, device="cuda"))
    parts = [a.double() @ e.double().t() for a, e in zip(x[: sum(sizes)].split(sizes), w.chunk(len(sizes)))]
    assert torch.equal(y[: sum(sizes)], torch.cat(parts).to(BF16)) and not y[sum(sizes):].any()


# ---- balanced groups ------------------------------------------------------------------------------------------------------------

# The weight gradient deals groups to the XCDs by size as long as none has more than a seventh of the rows (and a lane of a wave each): sizes that differ, ties, empty
# groups, a number of groups that is no multiple of eight; the last two stand on either side of a seventh.
BALANCED = {
    "8": [61, 70, 64, 70, 52, 70, 66, 57],
    "9": [40, 41, 42, 43, 44, 45, 46, 47, 48],
    "17": [33, 0, 21, 33, 64, 1, 60, 0, 47, 33, 58, 12, 64, 65, 9, 63, 30],
    "64": [(37 * i) % 83 for i in range(64)],
    "at_a_seventh": [70] * 7,
    "past_a_seventh": [71] + [70] * 6,
}


@pytest.mark.parametrize("transposed", [False, True], ids=["", "transposed"])
@pytest.mark.parametrize("name", list(BALANCED))
@pytest.mark.parametrize("pinned", ["any", *VARIANTS])
def test_balanced_groups(monkeypatch, pinned, name, transposed):
    sizes, n, k = BALANCED[name], 300, 264  # (more than a tile of any size)
    E, rows = len(sizes), sum(sizes)
    assert (max(sizes) * 7 > rows) == (name == "past_a_seventh")
    if pinned != "any":
        monkeypatch.setattr(_C, "HALF_ANY", VARIANTS[pinned])
    g = _gen(E + rows)
    x = _ints(g, rows, k).requires_grad_(True)
    w = _ints(g, *((E * k, n) if transposed else (E * n, k))).requires_grad_(True)
    gy = _ints(g, rows, n)
    y = grouped_linear(x, w, torch.tensor(sizes, device="cuda"), transposed=transposed)
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    x64, g64 = x.detach().double().split(sizes), gy.double().split(sizes)
    w64 = [e if transposed else e.t() for e in w.detach().double().chunk(E)]
    assert torch.equal(y, torch.cat([a @ e for a, e in zip(x64, w64)]).to(BF16))
    assert torch.equal(gx, torch.cat([a @ e.t() for a, e in zip(g64, w64)]).to(BF16))
    assert torch.equal(gw, torch.cat([a.t() @ b if transposed else b.t() @ a for a, b in zip(x64, g64)]).to(BF16))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n", [40, 37])
def test_what_relu_shuts_off_reaches_no_gradient(dtype, n):
    """Where z is not positive the gradient of z is 0 whatever arrives, infinite (a loss scale that was too large) or NaN; elsewhere it is what arrives, also
    where z is NaN."""
    g = _gen(n)
    x, w, b, gy = _ints(g, 21, 24, dtype=dtype), _ints(g, n, 24, dtype=dtype), _ints(g, n, dtype=dtype), _ints(g, 21, n, dtype=dtype)
    z = x.double() @ w.double().t() + b.double()
    off = z <= 0
    assert off.any() and (z == 0).any()
    bad = torch.where(off, torch.where(torch.arange(n, device="cuda") % 2 == 0, math.inf, math.nan).to(dtype), gy)
    ins = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear(*ins, activation="relu")
    want = torch.autograd.grad(y, ins, torch.where(off, 0, gy), retain_graph=True)
    for got, expected in zip(torch.autograd.grad(y, ins, bad), want):
        assert got.isfinite().all() and torch.equal(got, expected)
    with torch.no_grad():
        b[3] = math.nan
    y = linear(*ins, activation="relu")
    assert y[:, 3].isnan().all()
    assert torch.equal(torch.autograd.grad(y, b, gy)[0][3], gy[:, 3].double().sum().to(dtype))


def test_an_operand_is_copied_once():
    """A matrix whose rows are not contiguous is copied; a copy of whole 16-byte chunks is an operand as it is."""
    g = _gen(40)

    def allocations(t):
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        made = L._operand(t)
        return made, torch.cuda.memory_stats()["allocation.all.allocated"] - before

    w = _ints(g, 48, 40)
    made, count = allocations(w.t())
    assert count == 1 and torch.equal(made, w.t()) and L._is_operand(made)
    made, count = allocations(w[:1, :1].expand(24, 32))  # (the gradient of a sum)
    assert count == 1 and (made == w[0, 0]).all()
    made, count = allocations(w)
    assert count == 0 and made is w
    made, count = allocations(w[:, :37])
    assert count == 1 and made.shape == (48, 40) and torch.equal(made[:, :37], w[:, :37]) and not made[:, 37:].any()
    made, count = allocations(w.t()[:, :45])  # (a copy, and one with whole chunks)
    assert count == 2 and made.shape == (40, 48) and torch.equal(made[:, :45], w.t()[:, :45]) and not made[:, 45:].any()


@pytest.mark.parametrize("n", [24, 37])
@pytest.mark.parametrize("activation", ["relu", "gelu"])
def test_gradients_only_of_what_is_asked_behind_an_activation(activation, n):
    """Whichever inputs want a gradient, each gets the bits that it gets together with all others."""
    g = _gen(n)
    t = {"x": _ints(g, 19, 16), "w": _ints(g, n, 16), "b": _ints(g, n), "r": _ints(g, 19, n)}
    gy = torch.randn(n, 19, generator=g).to(BF16).cuda().t()  # (a view with odd strides)

    def grads(wanted):
        ins = {k: v.clone().requires_grad_(k in wanted) for k, v in t.items()}
        y = linear(ins["x"], ins["w"], ins["b"], activation=activation, residual=ins["r"])
        return dict(zip(wanted, torch.autograd.grad(y, [ins[k] for k in wanted], gy)))

    every = grads(list(t))
    for bits in range(1, 15):
        wanted = [k for i, k in enumerate(t) if bits >> i & 1]
        for k, got in grads(wanted).items():
            assert torch.equal(got, every[k]), (k, wanted)


def test_far_apart_rows_and_inference_mode():
    """Rows further apart than the products' 32-bit offsets reach inside a tile, and matrices that are columns of a wider one."""
    g = _gen(50)
    x, w, r = _ints(g, 5, 16), _ints(g, 24, 16), _ints(g, 5, 24)
    want = (torch.relu(x.double() @ w.double().t()) + r.double()).to(BF16)
    far = torch.full((5, 1 << 22), math.nan, dtype=BF16, device="cuda")
    far[:, :16], far[:, 64:88] = x, r
    with torch.inference_mode():
        assert torch.equal(linear(far[:, :16], w, activation="relu", residual=far[:, 64:88]), want)
    wide = torch.full((3 * 24, 40), math.nan, dtype=BF16, device="cuda")
    wide[:, 8:24] = torch.cat([w, 2 * w, 3 * w])
    sizes = torch.tensor([2, 0, 3], device="cuda")
    xg, wg = far[:, :16].detach().requires_grad_(True), wide[:, 8:24].requires_grad_(True)
    y = grouped_linear(xg, wg, sizes)
    exact = torch.cat([x[:2].double() @ w.double().t(), 3 * x[2:].double() @ w.double().t()])
    assert torch.equal(y, exact.to(BF16))
    gx, gw = torch.autograd.grad(y, [xg, wg], r)
    assert torch.equal(gx, torch.cat([r[:2].double() @ w.double(), 3 * r[2:].double() @ w.double()]).to(BF16))
    assert torch.equal(gw, torch.cat([r[:2].double().t() @ x[:2].double(), torch.zeros(24, 16, device="cuda"), r[2:].double().t() @ x[2:].double()]).to(BF16))
