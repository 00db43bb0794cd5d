"""
Norms around a block, fused with what joins them to the residual stream (``csrc/mi8_norm.hip``).

* ``residual_norm(branch, residual, post_weight=, pre_weight=, gate=, ...)``  -> ``(stream, normed)``:

      stream = residual_scale * residual + scale * gate * dropout(norm(branch) * post_weight)
      normed = norm(stream) * pre_weight             norm(a) = a / sqrt(mean(a^2) + eps)

one pass over the data forward and one backward, every part optional: a norm in front of a block (``pre_weight`` alone), behind it (``post_weight`` and the
residual: the reference's reordered norm), on both sides, or only the residual with a gate, a scale or dropout (reference:
``src/olmo_core/nn/transformer/block.py``, ``src/olmo_core/nn/layer_norm.py``).  Tensors must live on the GPU; there is no CPU path.
"""

from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .. import _C
from ..float8.ops import _on, _require_gpu, _stream, needs_autograd
from .dropout import _CODE, _Mask, _mask, first_order

__all__ = ["MOST_FEATURES", "residual_norm"]

MOST_FEATURES = 16384  # a row is held in registers
_NO_MASK = _Mask(0, 1.0, 0, 0)


class _Spec(NamedTuple):
    post_norm: bool
    pre_norm: bool
    scale: float
    residual_scale: float
    eps: float
    mask: _Mask
    has_stream: bool  # the stream is something else than the branch itself


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``[rows, features]`` with contiguous rows, in place where they are."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    rows, features = t.shape
    return t.stride(0) if rows > 1 else features


def _at(t: Optional[torch.Tensor]) -> int:
    return t.data_ptr() if t is not None else 0


def _code(w: Optional[torch.Tensor]) -> int:
    return _CODE[w.dtype] if w is not None else 0


# The library's argument block (``_C.ResidualNorm``) in one piece: field by field it costs more than the launch does on a few rows
_pack = struct.Struct("@19Q6q7iI4f").pack


def _forward(spec: _Spec, branch, residual, post, pre, gate, place, keep: bool):
    """``(stream or None, normed or None, statistics or None)``: one over the root of each row's mean square, of the branch and of the stream, ``[2, rows]``."""
    rows, features = branch.shape
    like = branch if residual is None else residual
    stream = like.new_empty((rows, features)) if spec.has_stream else None
    normed = branch.new_empty((rows, features)) if spec.pre_norm else None
    rstd = branch.new_empty((2, rows), dtype=torch.float32) if keep and (spec.post_norm or spec.pre_norm) else None
    at, mask = _at(rstd), spec.mask
    a = _C.ResidualNorm.from_buffer_copy(_pack(
        branch.data_ptr(), _at(residual), _at(stream), _at(normed), _at(post), _at(pre), _at(gate), at, at + 4 * rows if at else 0, _at(place), 0, 0, 0, 0, 0, 0, 0,
        mask.seed, mask.offset, rows, features, _pitch(branch), _pitch(residual) if residual is not None else 0, 0, 0,
        _CODE[branch.dtype], _CODE[like.dtype], _code(post), _code(pre), _code(gate), spec.post_norm, spec.pre_norm,
        mask.threshold, mask.factor, spec.scale, spec.residual_scale, spec.eps))
    with _on(branch.device):
        _C.check(_C.lib().mi8_residual_norm_forward(a, _stream(branch)), "mi8_residual_norm_forward")
    return stream, normed, rstd


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, branch, residual, post, pre, gate, place, spec):
        stream, normed, rstd = _forward(spec, branch, residual, post, pre, gate, place, True)
        ctx.set_materialize_grads(False)
        # Where the branch is read again, the stream is made again from it and the residual; elsewhere its stored values are taken
        u = branch if spec.post_norm or ctx.needs_input_grad[4] else None
        other = None if not spec.pre_norm else residual if u is not None else stream if spec.has_stream else branch
        ctx.save_for_backward(u, other, post, pre, gate, place, rstd)
        ctx.spec = spec
        ctx.meta = (branch.shape, branch.dtype, branch.dtype if residual is None else residual.dtype)
        return stream, normed

    @staticmethod
    @first_order
    def backward(ctx, gstream, gnormed):
        u, other, post, pre, gate, place, rstd = ctx.saved_tensors
        spec, (shape, dtype, stream_dtype) = ctx.spec, ctx.meta
        need_branch, need_residual, need_post, need_pre, need_gate = ctx.needs_input_grad[:5]
        if gstream is None and gnormed is None:
            return (None,) * 7
        rows, features = shape
        # (kept alive until the launch)
        gstream = _rows(gstream) if gstream is not None else None
        gnormed = _rows(gnormed) if gnormed is not None else None
        like = gnormed if gstream is None else gstream
        need_pre = need_pre and gnormed is not None
        outs = [
            like.new_empty(shape, dtype=dtype) if need_branch else None,
            like.new_empty(shape, dtype=stream_dtype) if need_residual else None,
            torch.empty_like(post) if need_post else None,
            torch.empty_like(pre) if need_pre else None,
            torch.empty_like(gate) if need_gate else None,
        ]
        stored = residual = None  # what the stream is read or made from
        if gnormed is not None:
            if u is None:
                stored = other = other.contiguous()
            else:
                residual = other
        lib = _C.lib()
        ws = like.new_empty(lib.mi8_residual_norm_workspace_words(rows, features), dtype=torch.float32) if need_post or need_pre or need_gate else None
        at, mask = _at(rstd), spec.mask
        a = _C.ResidualNorm.from_buffer_copy(_pack(
            _at(u), _at(residual), _at(stored), 0, _at(post), _at(pre), _at(gate), at, at + 4 * rows if at else 0, _at(place), _at(gstream), _at(gnormed),
            _at(outs[0]), _at(outs[1]), _at(outs[2]), _at(outs[3]), _at(outs[4]),
            mask.seed, mask.offset, rows, features, _pitch(u) if u is not None else 0, _pitch(residual) if residual is not None else 0,
            _pitch(gstream) if gstream is not None else 0, _pitch(gnormed) if gnormed is not None else 0,
            _CODE[dtype], _CODE[stream_dtype], _code(post), _code(pre), _code(gate), spec.post_norm, spec.pre_norm,
            mask.threshold, mask.factor, spec.scale, spec.residual_scale, spec.eps))
        with _on(like.device):
            _C.check(lib.mi8_residual_norm_backward(a, _at(ws), _stream(like)), "mi8_residual_norm_backward")
        return (*outs, None, None)


def _weight(w: torch.Tensor, name: str, branch: torch.Tensor, what: str) -> torch.Tensor:
    if w.shape != branch.shape[-1:] or w.device != branch.device:
        raise ValueError(f"{what}: {name} must be {branch.shape[-1]} numbers on {branch.device}, got {tuple(w.shape)} on {w.device}")
    if w.dtype not in (branch.dtype, torch.float32):
        raise TypeError(f"{what}: {name} is {w.dtype}, the branch {branch.dtype}")
    return w.contiguous()


def _residual_norm(branch, residual, post_norm, post_weight, pre_norm, pre_weight, gate, scale, residual_scale, eps, p, seed, offset):
    what = "residual_norm"
    _require_gpu(branch, what)
    if branch.dtype not in _CODE:
        raise TypeError(f"{what}: unsupported type {branch.dtype} (bfloat16, float16 or float32)")
    if branch.dim() < 1 or not 0 < branch.shape[-1] <= MOST_FEATURES:
        raise ValueError(f"{what}: rows of 1 to {MOST_FEATURES} features, got {tuple(branch.shape)}")
    if residual is not None:
        if residual.shape != branch.shape or residual.device != branch.device:
            raise ValueError(f"{what}: residual {tuple(residual.shape)} on {residual.device} for a branch {tuple(branch.shape)} on {branch.device}")
        if residual.dtype not in (branch.dtype, torch.float32):
            raise TypeError(f"{what}: the residual is {residual.dtype}, the branch {branch.dtype}")
    post = _weight(post_weight, "post_weight", branch, what) if post_weight is not None else None
    pre = _weight(pre_weight, "pre_weight", branch, what) if pre_weight is not None else None
    gate = _weight(gate, "gate", branch, what) if gate is not None else None
    post_norm, pre_norm = bool(post_norm or post is not None), bool(pre_norm or pre is not None)
    mask, place = (_NO_MASK, None) if p == 0 else _mask(p, seed, offset, branch.device, what)
    has_stream = residual is not None or post_norm or gate is not None or mask.threshold > 0 or scale != 1.0
    if not has_stream and not pre_norm:
        return branch, None
    spec = _Spec(post_norm, pre_norm, float(scale), float(residual_scale), float(eps), mask, has_stream)
    b2, r2 = _rows(branch), _rows(residual) if residual is not None else None
    if needs_autograd(*(t for t in (b2, r2, post, pre, gate) if t is not None)):
        stream, normed = _ResidualNorm.apply(b2, r2, post, pre, gate, place, spec)
    else:
        stream, normed = _forward(spec, b2, r2, post, pre, gate, place, False)[:2]
    if branch.dim() != 2:
        stream, normed = (t.reshape(branch.shape) if t is not None else None for t in (stream, normed))
    return stream if has_stream else branch, normed


def residual_norm(
    branch: torch.Tensor, residual: Optional[torch.Tensor] = None, *, post_norm: bool = False, post_weight: Optional[torch.Tensor] = None,
    pre_norm: bool = False, pre_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, scale: float = 1.0,
    residual_scale: float = 1.0, eps: float = 1e-6, p: float = 0.0, seed: Optional[Union[int, torch.Tensor]] = None, offset: int = 0,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """
    Join a block's output with the residual stream and take the norm that the next block starts with, differentiable in all tensors.

    :param branch: ``[*, features]``, what the block computed; bfloat16, float16 or float32, up to 16384 features.
    :param residual: the stream so far, of the branch's shape, and of its type or float32; ``None``: there is none (yet).
    :param post_norm: the branch is normed before it joins the stream; ``post_weight`` ``[features]`` is the norm's weight and implies it.
    :param pre_norm: the norm of the stream is wanted too; ``pre_weight`` ``[features]`` is its weight and implies it.
    :param gate: ``[features]``, multiplies the branch (after its norm and dropout).
    :param scale: factor of the branch, ``residual_scale`` of the residual.
    :param eps: added to both norms' mean squares.
    :param p: dropout of the branch, after its norm, with ``seed`` and ``offset`` as in :func:`~olmo_core_amd.ops.dropout.dropout`, whose mask it is for a
        tensor of this shape.

    Weights and gate are of the branch's type or float32.  Sums, statistics and the stream inside are float32: ``normed`` is that of the unrounded stream,
    and so is its gradient where the branch is normed or gated; elsewhere that is taken at the stored stream.

    :returns: ``(stream, normed)``: the stream, of the residual's type (of the branch's without one; the branch itself where nothing is done to it), and its norm, of
        the branch's type, or ``None``.
    """
    if torch.compiler.is_compiling():
        return _traced_residual_norm(branch, residual, post_norm, post_weight, pre_norm, pre_weight, gate, scale, residual_scale, eps, p, seed, offset)
    return _residual_norm(branch, residual, post_norm, post_weight, pre_norm, pre_weight, gate, scale, residual_scale, eps, p, seed, offset)


# (a graph break under torch.compile; asking whether there is a trace costs less than the wrapper does on every call)
_traced_residual_norm = torch.compiler.disable(_residual_norm)
