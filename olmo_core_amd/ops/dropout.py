"""
Dropout whose mask is a function of a seed (``csrc/mi8_dropout.hip``): nothing is stored for the backward pass, which makes the same bits again.

* ``dropout(x, p, seed=, offset=)``  -> ``x`` with each element zero with probability ``p``, the others scaled to keep the mean

The counterpart of the ``nn.Dropout`` modules of the reference's blocks (``src/olmo_core/nn/transformer/block.py``).  Tensors must live on the GPU; there is no CPU
path.
"""

from __future__ import annotations

import operator
from typing import NamedTuple, Optional, Union

import torch

from .. import _C
from ..float8.ops import _on, _require_gpu, _stream, needs_autograd

__all__ = ["dropout"]

_CODE = {torch.bfloat16: _C.MI8_BF16, torch.float16: _C.MI8_F16, torch.float32: _C.MI8_F32}


class _Mask(NamedTuple):
    """Which elements are kept, as the kernels take it."""

    threshold: int
    factor: float
    seed: int
    offset: int


def _word(value, name: str, what: str) -> int:
    """``value``, a whole number of any type (numpy's among them), as one of 64 bits."""
    try:
        number = int(operator.index(value))
    except TypeError:
        number = -1
    if not 0 <= number < 1 << 64:
        raise ValueError(f"{what}: {name} {value} is no 64-bit number")
    return number


def _mask(p: float, seed: Optional[Union[int, torch.Tensor]], offset: int, device: torch.device, what: str):
    """``(_Mask, the seed's tensor or None)``."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: probability {p} is not between 0 and 1")
    offset, place = _word(offset, "offset", what), None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"{what}: a seed on the GPU is one int64 on {device}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")
        place, seed = seed, 0
    else:
        seed = _word(seed, "seed", what)
    threshold = round(65536 * p)
    return _Mask(threshold, 65536 / (65536 - threshold) if threshold < 65536 else 0.0, seed, offset), place


def first_order(backward):
    """For a backward pass of kernels alone, which has no derivative of its own: refuses ``create_graph=True``.  (``once_differentiable`` refuses only where the
    second derivative is taken through the incoming gradient; one through the inputs it would leave out without a word.)"""

    def called(ctx, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError("differentiable once: no backward pass with create_graph=True through this operation")
        return backward(ctx, *grads)

    return called


def _run(x: torch.Tensor, mask: _Mask, place: Optional[torch.Tensor]) -> torch.Tensor:
    x = x.contiguous()
    y = torch.empty_like(x)
    with _on(x.device):
        _C.check(
            _C.lib().mi8_dropout(x.data_ptr(), _CODE[x.dtype], x.numel(), mask.threshold, mask.factor, mask.seed,
                                 place.data_ptr() if place is not None else None, mask.offset, y.data_ptr(), _stream(x)),
            "mi8_dropout",
        )
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, place, mask):
        ctx.mask = mask
        ctx.save_for_backward(place)
        return _run(x, mask, place)

    @staticmethod
    @first_order
    def backward(ctx, gy):
        (place,) = ctx.saved_tensors
        return _run(gy, ctx.mask, place), None, None


def _dropout(x, p, seed, offset):
    _require_gpu(x, "dropout")
    if x.dtype not in _CODE:
        raise TypeError(f"dropout: unsupported type {x.dtype} (bfloat16, float16 or float32)")
    mask, place = _mask(p, seed, offset, x.device, "dropout")
    return _Dropout.apply(x, place, mask) if needs_autograd(x) else _run(x, mask, place)


def dropout(x: torch.Tensor, p: float, *, seed: Union[int, torch.Tensor], offset: int = 0) -> torch.Tensor:
    """
    Zero each element of ``x`` with probability ``p`` (in steps of 2^-16) and divide the others by the probability with which they are kept.
    An element that is not kept is 0 whatever it was, and so is its gradient.

    :param seed: what the mask is made from: the same seed, offset and shape give the same mask.  A tensor (one int64 on ``x``'s device) is read when
        the kernels run, so a captured graph draws another mask whenever the tensor has changed before a replay; the backward
        pass needs it as the forward found it.
    :param offset: tells apart the calls that share a seed (a layer's number, say).
    """
    if torch.compiler.is_compiling():
        return _traced_dropout(x, p, seed, offset)
    return _dropout(x, p, seed, offset)


_traced_dropout = torch.compiler.disable(_dropout)  # (a graph break; asking whether there is a trace costs less than the wrapper does on every call)
