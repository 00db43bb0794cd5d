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

from . import ops, plan

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
    if experts < 1 or weight.dim() != 2 or any(d % 16 for d in weight.shape) or weight.shape[0] % experts or (weight.shape[0] // experts) % 16:
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


class _Spec(NamedTuple):
    """What the launches of a call follow from, beside the shapes and types of its tensors."""

    experts: int  # 0: one matrix, rows in no groups
    transposed: bool
    shapes: Tuple[Tuple[int, int], ...]  # of the weights
    need_x: bool
    need_w: Tuple[bool, ...]

    @property
    def stored(self) -> bool:
        """The product contracts over the columns of a weight as it is stored."""
        return not self.transposed


def _few_rows(rows: int, experts: int) -> bool:
    """Whether the product quantises its rows itself."""
    return 0 < rows <= (min(512, 8 * experts) if experts else 16) and experts <= 4096


# Bytes read by casts up to which they share a launch: beyond it saves next to nothing, and the copies of all of them would live at once.  us of
# rows and a weight one by one / together: bfloat16 2 MiB 10.0 / 6.1, 9 MiB 11.2 / 7.7, 16 MiB 12.2 / 10.6, 48 MiB 26.1 / 23.2, 64 MiB 31.2 / 31.7,
# 160 MiB 64.7 / 61.6; float32 4 MiB 10.1 / 6.4, 32 MiB 16.3 / 12.4, 96 MiB 35.2 / 36.6, 320 MiB 101.7 / 100.7.
_MOST_TOGETHER = 64 << 20


def _cast_all(casts):
    """The results of :func:`ops.cast_blockwise_batch` of any number of tensors in order: made together where that pays, else each when it is asked for
    (so that no more of them live than are used)."""
    if len(casts) > ops._C.BLOCK_CAST_BATCH or sum(x.numel() * x.dtype.itemsize for x, _ in casts) > _MOST_TOGETHER:
        return (ops.cast_blockwise_batch([c])[0] for c in casts)
    return iter(ops.cast_blockwise_batch(casts) if casts else ())


def _wanted(spec: _Spec, sizes, rows: bool, columns: bool) -> dict:
    """How rows (the input, a gradient) are cast."""
    kw = dict(want_rowmajor=rows, want_transposed=columns)
    return dict(kw, group_sizes=sizes) if spec.experts else kw


def _product(spec: _Spec, a, sa, w, i: int, over_columns: bool, sizes, dtype):
    """Rows of ``a`` times the i-th weight's matrices, contracted over their columns (``w = (q, scales)``) or their rows (of the
    transposed copies)."""
    rows, cols = spec.shapes[i][0] // max(spec.experts, 1), spec.shapes[i][1]
    n, k = (rows, cols) if over_columns else (cols, rows)
    if not spec.experts:
        return ops.gemm_fp8_blockwise(a, sa, *w, k=k, out_dtype=dtype)
    return ops.grouped_gemm_fp8_blockwise(a, sa, *w, sizes, n=n, k=k, out_dtype=dtype)


def _forward(spec: _Spec, x, sizes, weights, kept):
    """``(ys, saved)``: ``saved`` is ``(x_t, its scales)`` and per weight the copy that the gradient of x reads with its scales, ``None`` for what no
    gradient needs.  ``weights[i]`` or ``kept[i] = (q, scales, q_t, scales_t)`` is ``None``."""
    rows = _few_rows(x.shape[0], spec.experts)
    casts = [(x, _wanted(spec, sizes, not rows, any(spec.need_w)))] if not rows or any(spec.need_w) else []
    square = dict(square=True, matrices=max(spec.experts, 1), want_rowmajor=spec.stored or spec.need_x, want_transposed=spec.transposed or spec.need_x)
    casts += [(w, square) for w, k in zip(weights, kept) if k is None]
    done = _cast_all(casts)
    xq, xs, x_t, xs_t = next(done) if not rows or any(spec.need_w) else (None,) * 4
    ys, w_saved = [], []
    for i, made in enumerate(kept):
        if made is None:
            made = next(done)
        here, other = (made[:2], made[2:]) if spec.stored else (made[2:], made[:2])
        if rows:
            n = spec.shapes[i][0] // max(spec.experts, 1) if spec.stored else spec.shapes[i][1]
            ys.append(ops.rows_fp8_blockwise(x, *here, n=n, group_sizes=sizes))
        else:
            ys.append(_product(spec, xq, xs, here, i, spec.stored, sizes, x.dtype))
        w_saved.append(tuple(other) if spec.need_x else None)
    return ys, ((x_t, xs_t) if any(spec.need_w) else None, w_saved)


def _backward(spec: _Spec, saved, sizes, gos, tokens: int, x_dtype, w_dtypes, separate: bool = False):
    """``[gx] + [gw, ...]`` of the gradients that are needed; ``gos[i]`` ``None``: no gradient arrived.  ``separate``: each weight's term of gx by itself, in
    the order in which they are to be added, and the products of all weights at once (what is recorded: the additions are not the library's.  us of forward
    and backward one by one / replayed: 1537 tokens x 2048 to 2048 + 512 + 512 390 / 197, 2 x 32 experts of 1024 x 512 with 4008 rows 225 / 136)."""
    x_op, w_ops = saved
    order = _order(spec, gos)
    cast = _cast_all([(gos[i], _wanted(spec, sizes, spec.need_x, spec.need_w[i])) for i in order])
    terms, gws = [], [None] * len(gos)

    def add(term):
        if separate or not terms:
            terms.append(term)
        else:
            terms[0].add_(term)

    if spec.experts:
        for i in order:
            gq, gs, g_t, gs_t = next(cast)
            if spec.need_x:
                add(_product(spec, gq, gs, w_ops[i], i, spec.transposed, sizes, x_dtype))
            if spec.need_w[i]:
                a, b = ((g_t, gs_t), x_op) if spec.stored else (x_op, (g_t, gs_t))
                gws[i] = ops.grouped_wgrad_fp8_blockwise(*a, *b, sizes, tokens=tokens, out_dtype=w_dtypes[i]).reshape(spec.shapes[i])
    else:
        todo = []  # (weight or None, product)
        for i in order:  # (the products of a linear, or of all of them, in one launch where they are small)
            gq, gs, g_t, gs_t = next(cast)
            if spec.need_x:
                todo.append((None, (gq, gs, *w_ops[i], spec.shapes[i][0], x_dtype)))
            if spec.need_w[i]:
                todo.append((i, (g_t, gs_t, *x_op, tokens, w_dtypes[i])))
            if separate and i != order[-1] and len(todo) + 2 <= ops._C.BLOCK_GEMM_BATCH:
                continue
            for (k, _), made in zip(todo, ops.gemm_fp8_blockwise_batch([t for _, t in todo])):
                if k is None:
                    add(made)
                else:
                    gws[k] = made
            todo = []
    return terms + [g for g in gws if g is not None]


def _order(spec: _Spec, gos) -> list:
    """The weights whose gradients of the output have work to do, in the order in which autograd adds the terms of separate calls."""
    return [i for i in reversed(range(len(gos))) if gos[i] is not None and (spec.need_x or spec.need_w[i])]


def _planned_forward(spec: _Spec, x, sizes, weights, kept):
    """:func:`_forward` from a plan: ``(ys, kept buffer, plan)`` or ``None``."""
    if x.shape[0] == 0 or (spec.need_x and any(k is not None for k in kept)):
        return None  # (a kept weight's copies are saved as they are)
    n = len(weights)
    used = [w if k is None else None for w, k in zip(weights, kept)]
    copies = [t for k in kept for t in (k[:4] if k is not None else (None,) * 4)]

    def recorded(px, psizes, *rest):
        made = [rest[n + 4 * i:n + 4 * i + 4] for i in range(n)]
        return _forward(spec, px, psizes, rest[:n], [m if m[0] is not None else None for m in made])

    return plan.call(recorded, [x, sizes, *used, *copies], ("blockwise", spec), own=4 * n)


class _BlockwiseLinear(torch.autograd.Function):
    """``ys[i] = x @ weights[i]^T`` (or ``x @ weights[i]``), x quantised once; rows in groups or not."""

    @staticmethod
    def forward(ctx, x2, sizes, experts, transposed, n, *rest):
        weights, kept = rest[:n], rest[n:]
        spec = _Spec(experts, transposed, tuple(tuple(w.shape) for w in weights), ctx.needs_input_grad[0], tuple(ctx.needs_input_grad[5:5 + n]))
        ctx.set_materialize_grads(False)
        ctx.spec, ctx.tokens, ctx.x_dtype, ctx.w_dtypes = spec, x2.shape[0], x2.dtype, [w.dtype for w in weights]
        done = _planned_forward(spec, x2, sizes, weights, kept)
        ctx.plan = None
        if done is not None:
            ys, buffer, ctx.plan = done
            ctx.save_for_backward(buffer, sizes)
            return tuple(ys)
        ys, (x_op, w_ops) = _forward(spec, x2, sizes, weights, [k[:4] if k is not None else None for k in kept])
        ctx.has_x = x_op is not None
        flat = list(x_op or ())
        for w in w_ops:
            flat += w or ()
        ctx.save_for_backward(sizes, *flat)
        return tuple(ys)

    @staticmethod
    @once_differentiable
    def backward(ctx, *gos):
        spec, n = ctx.spec, len(ctx.spec.shapes)
        gos = [None if g is None else g if g.dtype == ctx.x_dtype else g.to(ctx.x_dtype) for g in gos]
        done = None
        if ctx.plan is not None:
            buffer, sizes = ctx.saved_tensors

            def recorded(slab, psizes, *places):
                return _backward(spec, ctx.plan.saved_places(slab), psizes, places, ctx.tokens, ctx.x_dtype, ctx.w_dtypes, separate=True), None

            if any(g is not None for g in gos):
                done = plan.call(recorded, [buffer, sizes, *gos], ("blockwise backward", tuple(ctx.w_dtypes)), within=ctx.plan)
            saved = ctx.plan.saved_tensors(buffer) if done is None else None
        else:
            sizes, *flat = ctx.saved_tensors
            x_op = (flat.pop(0), flat.pop(0)) if ctx.has_x else None
            saved = x_op, [(flat[2 * i], flat[2 * i + 1]) if spec.need_x else None for i in range(n)]
        outs = list(done[0] if done is not None else _backward(spec, saved, sizes, gos, ctx.tokens, ctx.x_dtype, ctx.w_dtypes))
        gx = outs.pop(0) if spec.need_x and any(g is not None for g in gos) else None
        if spec.need_x and done is not None:
            for _ in _order(spec, gos)[1:]:
                gx = gx.add_(outs.pop(0))
        gws = [outs.pop(0) if need and g is not None else None for need, g in zip(spec.need_w, gos)]
        return (gx, None, None, None, None, *gws, *([None] * n))


def _apply(x2, sizes, experts: int, transposed: bool, weights: Sequence[torch.Tensor], kept) -> Tuple[torch.Tensor, ...]:
    differentiate = ops.needs_autograd(x2, *weights)
    if (transposed or (differentiate and x2.requires_grad)) and any(k is not None and k.q_t is None for k in kept):
        raise ValueError("the kept weight has no transposed copy (blockwise_weight(..., transposed=False))")
    if differentiate:
        return _BlockwiseLinear.apply(x2, sizes, experts, transposed, len(weights), *weights, *kept)
    spec = _Spec(experts, transposed, tuple(tuple(w.shape) for w in weights), False, (False,) * len(weights))
    if all(k is not None for k in kept) and _few_rows(x2.shape[0], experts):  # (one launch a product: nothing to record)
        return tuple(_forward(spec, x2, sizes, weights, [k[:4] for k in kept])[0])
    done = _planned_forward(spec, x2, sizes, weights, kept)
    if done is not None:
        return tuple(done[0])
    return tuple(_forward(spec, x2, sizes, weights, [k[:4] if k is not None else None for k in kept])[0])


def _linears(x: torch.Tensor, weights: Sequence[torch.Tensor], kept) -> Tuple[torch.Tensor, ...]:
    """``x @ w.T`` for several weights, x quantised once."""
    if torch.compiler.is_compiling():
        return _traced_linears(x, weights, kept)
    _check(x, weights, kept, 1, weights[0].shape[-1], "blockwise_linear")
    for w in weights[1:]:
        if w.shape[-1] != x.shape[-1]:
            raise ValueError(f"blockwise_linear: input features {x.shape[-1]} do not match weight {tuple(w.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    with ops._on(x.device):
        ys = _apply(x2, None, 0, False, weights, kept)
    return ys if x.dim() == 2 else tuple(y.reshape(*x.shape[:-1], y.shape[1]) for y in ys)


def blockwise_linear(x: torch.Tensor, weight: torch.Tensor, *, kept: Optional[BlockwiseWeight] = None) -> torch.Tensor:
    """
    ``x [*, K] @ weight[N, K].T`` in float8 with block scales, differentiable in ``x`` and ``weight`` (both bfloat16 or float32; N and
    K multiples of 16).  The output and the gradient of ``x`` have the type of ``x``, the gradient of ``weight`` its own.

    :param kept: copies of ``weight`` made by :func:`blockwise_weight`, which are then used in its place.
    """
    return _linears(x, (weight,), (kept,))[0]


def _grouped_linears(x, weights, batch_size_per_expert, kept, transposed: bool) -> Tuple[torch.Tensor, ...]:
    if torch.compiler.is_compiling():
        return _traced_grouped_linears(x, weights, batch_size_per_expert, kept, transposed)
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
    with ops._on(x.device):
        ys = _apply(x2, ops._sizes_i64(sizes, x.device), experts, transposed, weights, kept)
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


# (a graph break under torch.compile; asking whether there is a trace costs less than the wrapper does on every call)
_traced_linears = torch.compiler.disable(_linears)
_traced_grouped_linears = torch.compiler.disable(_grouped_linears)
