"""
Float8 with block scales in 64 bits: what the casts with one power-of-two scale per 128 elements give, and products of their
values.  Plain torch on the CPU, written from the definition: the scale of a block is the largest power of two (at most 2^120) that
keeps its largest magnitude times the scale within 448, values are rounded to the nearest float8 e4m3 value, ties to even.
"""

from __future__ import annotations

import torch

MAX_SCALE_EXPONENT = 120


def pad128(n: int) -> int:
    return -(-n // 128) * 128


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """float64 values of at most 448 rounded to e4m3 (3 mantissa bits, smallest normal 2^-6)."""
    _, e = torch.frexp(v.abs().clamp(min=2.0 ** -6))
    spacing = torch.ldexp(torch.ones_like(v), e - 4)
    return torch.round(v / spacing) * spacing


def exponent(amax: torch.Tensor) -> torch.Tensor:
    """k of the scale 2^k of blocks with these (finite) largest magnitudes."""
    _, e = torch.frexp(448.0 / amax.double().clamp(min=2.0 ** -140))
    return (e - 1).clamp(max=MAX_SCALE_EXPONENT)


def _blocks(x: torch.Tensor, bm: int, bn: int) -> torch.Tensor:
    """[rows / bm, bm, cols / bn, bn], zero padded."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -cols % bn, 0, -rows % bm))
    return x.view(x.shape[0] // bm, bm, x.shape[1] // bn, bn)


def quantise(x: torch.Tensor, bm: int, bn: int):
    """``(codes, exponents, values)``: float8 values times their scales ``[padded rows, padded cols]`` (as float64), the exponent k of every
    block, and what the codes stand for ``[rows, cols]``.  A block that is not finite is NaN throughout with k = 0."""
    b = _blocks(x, bm, bn)
    amax = b.abs().amax(dim=(1, 3))
    bad = ~torch.isfinite(amax)
    k = torch.where(bad, 0, exponent(torch.where(bad, 1.0, amax)).long())
    scale = torch.ldexp(torch.ones_like(amax), k)[:, None, :, None]
    codes = torch.where(bad[:, None, :, None], float("nan"), round_e4m3(b * scale))
    values = (codes / scale).reshape(b.shape[0] * bm, -1)[: x.shape[0], : x.shape[1]]
    return codes.reshape(b.shape[0] * bm, -1), k, values


def rows_values(x: torch.Tensor) -> torch.Tensor:
    return quantise(x, 1, 128)[2]


def square_values(w: torch.Tensor) -> torch.Tensor:
    return quantise(w, 128, 128)[2]


def scale_bytes(k: torch.Tensor, rows: int) -> torch.Tensor:
    """The exponent bytes of an operand ``[rows, K]`` as they are stored, ``[K / 128, pad128(rows)]`` (rows behind the last: -1), from
    the k of every row and block ``[rows, K / 128]``."""
    blocks = k.shape[1]
    out = torch.full((blocks, pad128(rows)), -1, dtype=torch.int64)
    r = torch.arange(rows)
    out[:, 128 * (r // 128) + 8 * (r % 16) + r % 128 // 16] = (127 - k[:rows]).t()
    return out


def linear(x, w, g=None):
    """``y`` and, with ``g``, ``(y, gx, gw)`` of a linear with block scales, in float64."""
    wv = square_values(w)
    y = rows_values(x) @ wv.t()
    if g is None:
        return y
    return y, rows_values(g) @ wv, rows_values(g.t()) @ rows_values(x.t()).t()


def magnitudes(x, w, g=None):
    """Sums of the magnitudes of the same products: what the errors of their sums are measured against."""
    wv = square_values(w).abs()
    y = rows_values(x).abs() @ wv.t()
    if g is None:
        return y
    return y, rows_values(g).abs() @ wv, rows_values(g.t()).abs() @ rows_values(x.t()).abs().t()
