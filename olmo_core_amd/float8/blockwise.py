"""
Linear layers with block scales: float8 e4m3 operands with one power-of-two scale for each 128 elements of the contracted
axis, 1 x 128 of activations and gradients and 128 x 128 of weights.

    output      y  [M, N] = q(x)   . q(W)^T       blocks along the input features
    grad_input  gx [M, K] = q(g)   . q(W)         blocks along the output features
    grad_weight gW [N, K] = q(g^T) . q(x^T)^T     blocks along the tokens

A block's scale is the largest power of two that keeps its largest magnitude within float8's 448, so an outlier costs the other
values of its 128 their precision, not those of the whole row or tensor.  (No counterpart in the reference.  Powers of two
because gfx950's matrix instructions apply them themselves: the product runs as fast as one without scales.)

:func:`blockwise_linear` is what a :class:`~olmo_core_amd.float8.linear.Float8Linear` of the ``blockwise`` recipe calls,
:func:`blockwise_grouped_linear` what a :class:`~olmo_core_amd.nn.DroplessMoEMLP` with ``scaling="blockwise"`` does for its experts.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import ops

__all__ = ["BlockwiseWeight", "blockwise_weight", "blockwise_linear", "blockwise_grouped_linear"]


class BlockwiseWeight(NamedTuple):
    """Both float8 copies of a weight ``[experts * rows, cols]`` and their scales (:func:`ops.cast_blockwise` with ``square``)."""

    q: torch.Tensor
    scales: torch.Tensor
    q_t: Optional[torch.Tensor]
    scales_t: Optional[torch.Tensor]
    shape: Tuple[int, int]
    experts: int

    @property
    def rows(self) -> int:
        return self.shape[0] // self.experts


def blockwise_weight(weight: torch.Tensor, *, experts: int = 1, transposed: bool = True) -> BlockwiseWeight:
    """Quantise a weight ``[experts * rows, cols]`` once, for calls that pass it as ``kept``: a serving loop, the micro-batches of one
    optimizer step.  ``transposed=False`` leaves out the copy that gradients of the input (and products with the transposed
    weight) read.  The copies are not tied to ``weight``: make them again when it changes."""
    if weight.dim() != 2 or any(d % 16 for d in weight.shape) or weight.shape[0] % experts or (weight.shape[0] // experts) % 16:
        raise ValueError(f"blockwise_weight: {tuple(weight.shape)} is not {experts} matrices whose sizes are multiples of 16")
    with torch.no_grad():
        q, s, q_t, s_t = ops.cast_blockwise(weight.detach(), square=True, matrices=experts, want_transposed=transposed)
    return BlockwiseWeight(q, s, q_t, s_t, tuple(weight.shape), experts)


def _check(x: torch.Tensor, weights, kept, experts: int, features: int, what: str) -> None:
    ops._require_gpu(x, what)
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: unsupported input type {x.dtype} (bfloat16 or float32)")
    for w, k in zip(weights, kept):
        if w.dim() != 2 or w.shape[0] % experts or (w.shape[0] // experts) % 16 or w.shape[1] % 16:
            raise ValueError(f"{what}: weight {tuple(w.shape)} is not {experts} matrices whose sizes are multiples of 16")
        if w.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"{what}: unsupported weight type {w.dtype} (bfloat16 or float32)")
        if w.device != x.device:
            raise ValueError(f"{what}: input on {x.device}, weight on {w.device}")
        if k is not None and (k.shape != tuple(w.shape) or k.experts != experts or k.q.device != x.device):
            raise ValueError(f"{what}: kept copies of {k.experts} matrices {k.shape} for a weight {tuple(w.shape)} of {experts}")
    if x.dim() < 1 or x.shape[-1] != features:
        raise ValueError(f"{what}: input features {x.shape[-1] if x.dim() else 0} do not match {features}")


def _operands(weight, kept, experts: int, rows: bool, transposed: bool):
    """``(q, scales, q_t, scales_t)`` of a weight, ``rows`` / ``transposed``: which of the two copies are needed."""
    if kept is not None:
        if transposed and kept.q_t is None:
            raise ValueError("the kept weight has no transposed copy (blockwise_weight(..., transposed=False))")
        return kept[:4]
    return ops.cast_blockwise(weight, square=True, matrices=experts, want_rowmajor=rows, want_transposed=transposed)


class _Layout:
    """How the products of a call find their rows: one matrix, or groups of rows with matrices of their own."""

    def __init__(self, sizes: Optional[torch.Tensor], experts: int, transposed: bool):
        self.sizes, self.experts, self.transposed = sizes, experts, transposed

    def cast(self, x, rows: bool, columns: bool):
        if self.sizes is None:
            return ops.cast_blockwise(x, want_rowmajor=rows, want_transposed=columns)
        return ops.grouped_cast_blockwise(x, self.sizes, want_rowmajor=rows, want_transposed=columns)

    def product(self, a, sa, w, as_stored: bool, shape, dtype):
        """Rows times the weight's rows (``as_stored``, contracted over its columns) or its columns."""
        rows, cols = shape[0] // self.experts, shape[1]
        n, k = (rows, cols) if as_stored else (cols, rows)
        b, sb = w[:2] if as_stored else w[2:]
        if self.sizes is None:
            return ops.gemm_fp8_blockwise(a, sa, b, sb, k=k, out_dtype=dtype)
        b = b.view(self.experts, n, -1)
        sb = sb.view(self.experts, -1, sb.shape[-1])
        return ops.grouped_gemm_fp8_blockwise(a, sa, b, sb, self.sizes, k=k, out_dtype=dtype)

    def weight_grad(self, g_t, sg, x_t, sx, tokens: int, dtype):
        """``g^T x``, or ``x^T g`` where the weight is used transposed."""
        if self.transposed:
            g_t, sg, x_t, sx = x_t, sx, g_t, sg
        if self.sizes is None:
            return ops.gemm_fp8_blockwise(g_t, sg, x_t, sx, k=tokens, out_dtype=dtype)
        out = ops.grouped_wgrad_fp8_blockwise(g_t, sg, x_t, sx, self.sizes, tokens=tokens, out_dtype=dtype)
        return out.view(-1, out.shape[-1])


class _BlockwiseLinear(torch.autograd.Function):
    """``ys[i] = x @ weights[i]^T`` (or ``x @ weights[i]``), x quantised once; rows in groups or not (``_Layout``)."""

    @staticmethod
    def forward(ctx, x2, layout, n, *rest):
        weights, kept = rest[:n], rest[n:]
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[3:3 + n]
        ctx.set_materialize_grads(False)
        xq, xs, x_t, xs_t = layout.cast(x2, True, any(need_w))
        saved, ys = [], []
        if any(need_w):
            saved += [x_t, xs_t]
        as_stored = not layout.transposed
        for w, k in zip(weights, kept):
            made = _operands(w, k, layout.experts, as_stored or need_x, not as_stored or need_x)
            ys.append(layout.product(xq, xs, made, as_stored, w.shape, x2.dtype))
            if need_x:  # what the gradient of x reads
                saved += made[2:] if as_stored else made[:2]
        ctx.save_for_backward(*saved)
        ctx.layout, ctx.tokens, ctx.x_dtype, ctx.need_w = layout, x2.shape[0], x2.dtype, need_w
        ctx.shapes, ctx.w_dtypes = [tuple(w.shape) for w in weights], [w.dtype for w in weights]
        return tuple(ys)

    @staticmethod
    @once_differentiable
    def backward(ctx, *gos):
        layout, n = ctx.layout, len(ctx.shapes)
        saved = list(ctx.saved_tensors)
        need_x = ctx.needs_input_grad[0]
        x_t, xs_t = (saved.pop(0), saved.pop(0)) if any(ctx.need_w) else (None, None)
        as_stored = not layout.transposed
        gx, gws = None, [None] * n
        for i in reversed(range(n)):  # (the order in which autograd adds the terms of separate calls)
            go = gos[i]
            if go is None or not (need_x or ctx.need_w[i]):
                continue
            if go.dtype != ctx.x_dtype:
                go = go.to(ctx.x_dtype)
            gq, gs, g_t, gs_t = layout.cast(go, need_x, ctx.need_w[i])
            if need_x:
                q, s = saved[2 * i:2 * i + 2]
                w = (None, None, q, s) if as_stored else (q, s, None, None)
                term = layout.product(gq, gs, w, not as_stored, ctx.shapes[i], ctx.x_dtype)
                gx = term if gx is None else gx.add_(term)
            if ctx.need_w[i]:
                gws[i] = layout.weight_grad(g_t, gs_t, x_t, xs_t, ctx.tokens, ctx.w_dtypes[i])
        return (gx, None, None, *gws, *([None] * n))


def _apply(x2, layout: _Layout, weights: Sequence[torch.Tensor], kept) -> Tuple[torch.Tensor, ...]:
    from .linear import needs_autograd

    if needs_autograd(x2, *weights):
        return _BlockwiseLinear.apply(x2, layout, len(weights), *weights, *kept)
    as_stored = not layout.transposed
    xq, xs, _, _ = layout.cast(x2, True, False)
    return tuple(layout.product(xq, xs, _operands(w, k, layout.experts, as_stored, not as_stored), as_stored, w.shape, x2.dtype)
                 for w, k in zip(weights, kept))


@torch.compiler.disable
def _linears(x: torch.Tensor, weights: Sequence[torch.Tensor], kept) -> Tuple[torch.Tensor, ...]:
    """``x @ w.T`` for several weights, x quantised once."""
    _check(x, weights, kept, 1, weights[0].shape[-1], "blockwise_linear")
    for w in weights[1:]:
        if w.shape[-1] != x.shape[-1]:
            raise ValueError(f"blockwise_linear: input features {x.shape[-1]} do not match weight {tuple(w.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    ys = _apply(x2, _Layout(None, 1, False), weights, kept)
    return ys if x.dim() == 2 else tuple(y.reshape(*x.shape[:-1], y.shape[1]) for y in ys)


def blockwise_linear(x: torch.Tensor, weight: torch.Tensor, *, kept: Optional[BlockwiseWeight] = None) -> torch.Tensor:
    """
    ``x [*, K] @ weight[N, K].T`` in float8 with block scales, differentiable in ``x`` and ``weight`` (both bfloat16 or float32; N and
    K multiples of 16).  The output and the gradient of ``x`` have the type of ``x``, the gradient of ``weight`` its own.

    :param kept: copies of ``weight`` made by :func:`blockwise_weight`, which are then used in its place.
    """
    return _linears(x, (weight,), (kept,))[0]


@torch.compiler.disable
def _grouped_linears(x, weights, batch_size_per_expert, kept, transposed: bool) -> Tuple[torch.Tensor, ...]:
    what = "blockwise_grouped_linear"
    sizes = batch_size_per_expert
    if sizes.dim() != 1 or sizes.numel() == 0 or sizes.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: batch_size_per_expert must be a vector of integers, got {sizes.dtype} {tuple(sizes.shape)}")
    experts = sizes.numel()
    w = weights[0]
    _check(x, weights, kept, experts, (w.shape[0] // experts if transposed else w.shape[-1]), what)
    if any(other.shape != w.shape for other in weights):
        raise ValueError(f"{what}: weights of different shapes")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    ys = _apply(x2, _Layout(ops._sizes_i64(sizes, x.device), experts, transposed), weights, kept)
    return ys if x.dim() == 2 else tuple(y.reshape(*x.shape[:-1], y.shape[1]) for y in ys)


def blockwise_grouped_linear(
    x: torch.Tensor, weight: torch.Tensor, batch_size_per_expert: torch.Tensor, *, transposed: bool = False,
    kept: Optional[BlockwiseWeight] = None,
) -> torch.Tensor:
    """
    :func:`blockwise_linear` for rows that are sorted by expert: the first ``batch_size_per_expert[0]`` rows of ``x`` are multiplied with the
    first expert's matrix, the next ones with the second's, and so on (the sizes stay on the GPU).

    :param weight: the experts' matrices one below the other, ``[experts * N, K]``: ``y = x [T, K] @ w[e].T``.
    :param transposed: ``y = x [T, N] @ w[e]`` instead.
    :param kept: copies made by :func:`blockwise_weight` with ``experts=``.

    Rows behind the last group give zeros, and the weight of an expert without rows a gradient of zeros.
    """
    return _grouped_linears(x, (weight,), batch_size_per_expert, (kept,), transposed)[0]
