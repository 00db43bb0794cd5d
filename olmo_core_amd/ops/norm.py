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
    has_stream: bool  # the stream is something else than the branch itself
    seed: int
    offset: int
    tail: tuple  # the library's argument block from the types on


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``[rows, features]`` with contiguous rows, in place where they are."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


# A call on few rows is bound by what the host does for it: no helper is called for what an expression says, and the library's argument block
# (``_C.ResidualNorm``) is packed in one piece, field by field it costs more than the launch; its tail is made once for forward and backward.  231 x 64 to 1999 x 768
# float32, residual and a norm in front, forward and backward: 66 to 68 us where autograd's thread shares the caller's caches (elementary operations one by one, without
# autograd: 102), 124 where it does not and every line takes twice as long.
_pack = struct.Struct("@19Q6q7iI4f").pack


def _forward(spec: _Spec, branch, residual, post, pre, gate, place, keep: bool):
    """``(stream or None, normed or None, statistics or None)``: one over the root of each row's mean square, of the branch and of the stream, ``[2, rows]``."""
    shape = rows, features = branch.shape
    stream = normed = rstd = None
    at = 0
    if spec.has_stream:
        stream = (branch if residual is None else residual).new_empty(shape)
    if spec.pre_norm:
        normed = branch.new_empty(shape)
    if keep and (spec.post_norm or spec.pre_norm):
        rstd = branch.new_empty((2, rows), dtype=torch.float32)
        at = rstd.data_ptr()
    a = _C.ResidualNorm.from_buffer_copy(_pack(
        branch.data_ptr(), residual.data_ptr() if residual is not None else 0, stream.data_ptr() if stream is not None else 0,
        normed.data_ptr() if normed is not None else 0, post.data_ptr() if post is not None else 0, pre.data_ptr() if pre is not None else 0,
        gate.data_ptr() if gate is not None else 0, at, at + 4 * rows if at else 0, place.data_ptr() if place is not None else 0, 0, 0, 0, 0, 0, 0, 0,
        spec.seed, spec.offset, rows, features, branch.stride(0) if rows > 1 else features,
        0 if residual is None else residual.stride(0) if rows > 1 else features, 0, 0, *spec.tail))
    with _on(branch.device):
        _C.check(_C.lib().mi8_residual_norm_forward(a, _stream(branch)), "mi8_residual_norm_forward")
    return stream, normed, rstd


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, branch, residual, post, pre, gate, place, spec):
        stream, normed, rstd = _forward(spec, branch, residual, post, pre, gate, place, True)
        ctx.set_materialize_grads(False)
        # Where the branch is read again, the stream is made again from it and the residual; elsewhere its stored values are taken, which have to be all of it: a
        # 16-bit stream was rounded when it was stored
        stream_dtype = branch.dtype if residual is None else residual.dtype
        remake = spec.pre_norm and (gate is not None or (spec.has_stream and stream_dtype != torch.float32))
        u = branch if spec.post_norm or remake or ctx.needs_input_grad[4] else None
        other = None if not spec.pre_norm else residual if u is not None else stream if spec.has_stream else branch
        ctx.save_for_backward(u, other, post, pre, gate, place, rstd)
        ctx.meta = (spec, branch.shape, branch.dtype, stream_dtype)
        return stream, normed

    @staticmethod
    @first_order
    def backward(ctx, gstream, gnormed):
        if gstream is None and gnormed is None:
            return (None,) * 7
        u, other, post, pre, gate, place, rstd = ctx.saved_tensors
        spec, shape, dtype, stream_dtype = ctx.meta
        need_branch, need_residual, need_post, need_pre, need_gate = ctx.needs_input_grad[:5]
        rows, features = shape
        several = rows > 1
        like = gnormed if gstream is None else gstream
        at = to_stream = to_normed = pitch_stream = pitch_normed = 0
        if gstream is not None:  # (kept alive until the launch, like all that is made here)
            gstream = _rows(gstream)
            to_stream, pitch_stream = gstream.data_ptr(), gstream.stride(0) if several else features
        if rstd is not None:
            at = rstd.data_ptr()
        residual_at = stored_at = pitch_residual = 0  # what the stream is made or read from
        if gnormed is not None:
            gnormed = _rows(gnormed)
            to_normed, pitch_normed = gnormed.data_ptr(), gnormed.stride(0) if several else features
            if u is None:
                other = other.contiguous()
                stored_at = other.data_ptr()
            elif other is not None:
                residual_at, pitch_residual = other.data_ptr(), other.stride(0) if several else features
        else:
            need_pre = False
        gbranch = like.new_empty(shape, dtype=dtype) if need_branch else None
        gresidual = like.new_empty(shape, dtype=stream_dtype) if need_residual else None
        gpost = torch.empty_like(post) if need_post else None
        gpre = torch.empty_like(pre) if need_pre else None
        ggate = torch.empty_like(gate) if need_gate else None
        lib, ws_at = _C.lib(), 0
        with _on(like.device):
            if need_post or need_pre or need_gate:  # (its size follows from the current device)
                ws = like.new_empty(lib.mi8_residual_norm_workspace_words(rows, features), dtype=torch.float32)
                ws_at = ws.data_ptr()
            a = _C.ResidualNorm.from_buffer_copy(_pack(
                u.data_ptr() if u is not None else 0, residual_at, stored_at, 0, post.data_ptr() if post is not None else 0, pre.data_ptr() if pre is not None else 0,
                gate.data_ptr() if gate is not None else 0, at, at + 4 * rows if at else 0, place.data_ptr() if place is not None else 0, to_stream, to_normed,
                gbranch.data_ptr() if need_branch else 0, gresidual.data_ptr() if need_residual else 0, gpost.data_ptr() if need_post else 0,
                gpre.data_ptr() if need_pre else 0, ggate.data_ptr() if need_gate else 0,
                spec.seed, spec.offset, rows, features, 0 if u is None else u.stride(0) if several else features, pitch_residual, pitch_stream, pitch_normed, *spec.tail))
            _C.check(lib.mi8_residual_norm_backward(a, ws_at, _stream(like)), "mi8_residual_norm_backward")
        return gbranch, gresidual, gpost, gpre, ggate, None, None


def _weight(w: torch.Tensor, name: str, branch: torch.Tensor, features: int, what: str) -> torch.Tensor:
    if w.shape != (features,) or w.device != branch.device:
        raise ValueError(f"{what}: {name} must be {features} numbers on {branch.device}, got {tuple(w.shape)} on {w.device}")
    if w.dtype != branch.dtype and w.dtype != torch.float32:
        raise TypeError(f"{what}: {name} is {w.dtype}, the branch {branch.dtype}")
    return w if w.is_contiguous() else w.contiguous()


def _residual_norm(branch, residual, post_norm, post_weight, pre_norm, pre_weight, gate, scale, residual_scale, eps, p, seed, offset):
    what = "residual_norm"
    _require_gpu(branch, what)
    dtype, shape = branch.dtype, branch.shape
    code = stream_code = _CODE.get(dtype)
    if code is None:
        raise TypeError(f"{what}: unsupported type {dtype} (bfloat16, float16 or float32)")
    features = shape[-1] if shape else 0
    if not 0 < features <= MOST_FEATURES:
        raise ValueError(f"{what}: rows of 1 to {MOST_FEATURES} features, got {tuple(shape)}")
    if residual is not None:
        if residual.shape != shape or residual.device != branch.device:
            raise ValueError(f"{what}: residual {tuple(residual.shape)} on {residual.device} for a branch {tuple(shape)} on {branch.device}")
        if residual.dtype != dtype:
            if residual.dtype != torch.float32:
                raise TypeError(f"{what}: the residual is {residual.dtype}, the branch {dtype}")
            stream_code = _C.MI8_F32
    b2 = _rows(branch)
    tensors, post_code, pre_code, gate_code = [b2], 0, 0, 0
    r2 = None
    if residual is not None:
        r2 = _rows(residual)
        tensors.append(r2)
    if post_weight is not None:
        post_weight = _weight(post_weight, "post_weight", branch, features, what)
        post_norm, post_code = True, _CODE[post_weight.dtype]
        tensors.append(post_weight)
    if pre_weight is not None:
        pre_weight = _weight(pre_weight, "pre_weight", branch, features, what)
        pre_norm, pre_code = True, _CODE[pre_weight.dtype]
        tensors.append(pre_weight)
    if gate is not None:
        gate = _weight(gate, "gate", branch, features, what)
        gate_code = _CODE[gate.dtype]
        tensors.append(gate)
    post_norm, pre_norm = bool(post_norm), bool(pre_norm)
    mask, place = (_NO_MASK, None) if p == 0 else _mask(p, seed, offset, branch.device, what)
    has_stream = residual is not None or post_norm or gate is not None or mask.threshold > 0 or scale != 1.0
    if not has_stream and not pre_norm:
        return branch, None
    spec = _Spec(post_norm, pre_norm, has_stream, mask.seed, mask.offset, (
        code, stream_code, post_code, pre_code, gate_code, post_norm, pre_norm, mask.threshold, mask.factor, float(scale), float(residual_scale), float(eps)))
    if needs_autograd(*tensors):
        stream, normed = _ResidualNorm.apply(b2, r2, post_weight, pre_weight, gate, place, spec)
    else:
        stream, normed = _forward(spec, b2, r2, post_weight, pre_weight, gate, place, False)[:2]
    if branch.dim() != 2:
        stream, normed = (t.reshape(shape) if t is not None else None for t in (stream, normed))
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

    Weights and gate are of the branch's type or float32.  Sums, statistics and the stream inside are float32: ``normed`` is that of the unrounded stream, and
    so is its gradient.  For that the backward pass keeps branch and residual where the stream has 16 bits; a float32 stream is kept itself.

    :returns: ``(stream, normed)``: the stream, of the residual's type (of the branch's without one; the branch itself where nothing is done to it), and its norm, of
        the branch's type, or ``None``.
    """
    if torch.compiler.is_compiling():
        return _traced_residual_norm(branch, residual, post_norm, post_weight, pre_norm, pre_weight, gate, scale, residual_scale, eps, p, seed, offset)
    return _residual_norm(branch, residual, post_norm, post_weight, pre_norm, pre_weight, gate, scale, residual_scale, eps, p, seed, offset)


# (a graph break under torch.compile; asking whether there is a trace costs less than the wrapper does on every call)
_traced_residual_norm = torch.compiler.disable(_residual_norm)
