"""
MoE token-permutation ops: the interface of ``olmo_core.ops.moe`` (reference ``src/olmo_core/ops/moe.py:26-205``,
``:289-304``) on the HIP kernels of ``csrc/mi8_permute.hip`` (which replace the Triton kernels of
``src/olmo_core/kernels/moe.py``).

Same functions, argument order and gradients as the reference:

* ``gather(x, indices, bin_ids, bins, top_k)``            -> ``[tokens * top_k, hidden]`` rows sorted by expert
* ``scatter(x, indices, bin_ids, weights, bins, top_k)``  -> ``[tokens, hidden]`` weighted sum over a token's slots
* ``binned_gather(x, indices, bins, bin_size, top_k)``    -> ``[experts, bin_size, hidden]``
* ``binned_scatter(x, indices, weights, bins, top_k)``    -> ``[tokens, hidden]``
* ``batched_histc(x, num_classes)``, ``histc(x, num_classes)``

and what makes their expert ids, weights and batch sizes (``csrc/mi8_route.hip``):

* ``route(logits, top_k, ...)``  -> expert weights, expert indices, token slots per expert

``bin_ids`` is accepted for signature compatibility; the dropless kernels do not need it (row ``i`` of the sorted
side is row ``i`` of ``indices``).  Tensors must live on the GPU; there is no CPU path.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _C
from ..float8.ops import _empty, _on, _stream, needs_autograd

_DT = {torch.bfloat16: _C.MI8_BF16, torch.float32: _C.MI8_F32, torch.float16: _C.MI8_F16}
_RAW = (torch.float8_e4m3fn, torch.float8_e5m2, torch.uint8, torch.int8)


def _dt(x: torch.Tensor, what: str, allow_raw: bool = False) -> int:
    if not x.is_cuda:
        raise RuntimeError(f"{what}: tensors must live on the GPU (the permutation ops have no CPU implementation)")
    if x.dtype in _DT:
        return _DT[x.dtype]
    if allow_raw and x.dtype in _RAW:
        return _C.MI8_RAW8
    raise TypeError(f"{what}: unsupported element type {x.dtype}")


def _i32(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dim() != 1:
        raise ValueError(f"{what}: expected a vector, got {t.dim()} dimensions")
    return t if (t.dtype == torch.int32 and t.is_contiguous()) else t.to(torch.int32).contiguous()


def _weights(w: Optional[torch.Tensor], n: int, what: str):
    if w is None:
        return None, None, 0
    if w.dim() != 1 or w.shape[0] != n:
        raise ValueError(f"{what}: expected {n} weights, got {tuple(w.shape)}")
    w = w.contiguous()
    return w, w.data_ptr(), _dt(w, what)


# ---- kernels (no autograd) -----------------------------------------------------------------------------------


def _sort_slots(ids: torch.Tensor, sizes: torch.Tensor):
    """``(indices, bin_ids, bins)``: the slots stably sorted by expert id, their ids, the inclusive prefix sums of
    ``sizes`` (all int32).  One launch up to ``mi8_moe_sort_slots_max()`` slots, two beyond; torch's sort for other types, for
    more slots or experts than ``mi8_moe_sort_workspace_words`` takes, and wherever something other than plain GPU tensors is at work (tracing, vmap, subclasses)."""
    n = ids.numel()
    if (type(ids) is torch.Tensor and type(sizes) is torch.Tensor and not torch.compiler.is_compiling() and ids.is_cuda
            and sizes.device == ids.device and ids.dim() == sizes.dim() == 1 and ids.dtype in (torch.int32, torch.int64)
            and sizes.dtype == torch.int64 and ids.is_contiguous() and sizes.is_contiguous() and sizes.numel()
            and torch._C._len_torch_dispatch_stack() == 0 and torch._C._functorch.peek_interpreter_stack() is None
            and 0 < n and (n <= _C.lib().mi8_moe_sort_slots_max() or _C.lib().mi8_moe_sort_workspace_words(n, sizes.shape[0]))):
        indices, bin_ids = (torch.empty(n, dtype=torch.int32, device=ids.device) for _ in range(2))
        bins = torch.empty(sizes.shape[0], dtype=torch.int32, device=ids.device)
        if n > _C.lib().mi8_moe_sort_slots_max():
            counts = torch.empty(_C.lib().mi8_moe_sort_workspace_words(n, sizes.shape[0]), dtype=torch.int32, device=ids.device)
            _C.check(
                _C.lib().mi8_moe_sort_many_slots(ids.data_ptr(), int(ids.dtype == torch.int64), n, sizes.data_ptr(), sizes.shape[0],
                                                 counts.data_ptr(), indices.data_ptr(), bin_ids.data_ptr(), bins.data_ptr(),
                                                 _stream(ids)),
                "mi8_moe_sort_many_slots",
            )
            return indices, bin_ids, bins
        _C.check(
            _C.lib().mi8_moe_sort_slots(ids.data_ptr(), int(ids.dtype == torch.int64), n, sizes.data_ptr(), sizes.shape[0],
                                        indices.data_ptr(), bin_ids.data_ptr(), bins.data_ptr(), _stream(ids)),
            "mi8_moe_sort_slots",
        )
        return indices, bin_ids, bins
    bin_ids, indices = torch.sort(ids.int())
    return indices.int(), bin_ids, torch.cumsum(sizes, 0).to(torch.int32)


def _gather(x, indices, weights, top_k: int) -> torch.Tensor:
    if x.dim() != 2:
        raise ValueError(f"gather: expected a matrix, got {x.dim()} dimensions")
    x = x.contiguous()
    tokens, hidden = x.shape
    indices = _i32(indices, "gather")
    if indices.shape[0] != tokens * top_k:
        raise ValueError(f"gather: expected {tokens * top_k} indices, got {indices.shape[0]}")
    w, wp, wd = _weights(weights, tokens * top_k, "gather")
    out = torch.empty((tokens * top_k, hidden), dtype=x.dtype, device=x.device)
    if out.numel():
        _C.check(
            _C.lib().mi8_moe_gather(x.data_ptr(), _dt(x, "gather", allow_raw=w is None), tokens, hidden,
                                    indices.data_ptr(), wp, wd, top_k, out.data_ptr(), _stream(x)),
            "mi8_moe_gather",
        )
    return out


def _scatter(x, indices, weights, top_k: int) -> torch.Tensor:
    if x.dim() != 2:
        raise ValueError(f"scatter: expected a matrix, got {x.dim()} dimensions")
    x = x.contiguous()
    n, hidden = x.shape
    indices = _i32(indices, "scatter")
    if indices.shape[0] != n or n % top_k:
        raise ValueError(f"scatter: {n} rows, {indices.shape[0]} indices, top_k {top_k} do not fit together")
    tokens = n // top_k
    w, wp, wd = _weights(weights, n, "scatter")
    out = _empty((tokens, hidden), dtype=x.dtype, device=x.device)
    if out.numel():
        inverse = _empty(n, dtype=torch.int32, device=x.device)
        _C.check(
            _C.lib().mi8_moe_scatter(x.data_ptr(), _dt(x, "scatter"), tokens, hidden, indices.data_ptr(), wp, wd, top_k,
                                     inverse.data_ptr(), out.data_ptr(), _stream(x)),
            "mi8_moe_scatter",
        )
    return out


def _scatter_wgrad(x, grad, indices, top_k: int) -> torch.Tensor:
    x, grad = x.contiguous(), grad.contiguous()
    n, hidden = x.shape
    indices = _i32(indices, "scatter_wgrad")
    tokens = n // top_k
    if grad.shape != (tokens, hidden) or grad.dtype != x.dtype:
        raise ValueError(f"scatter_wgrad: grad {tuple(grad.shape)} {grad.dtype} does not match x {tuple(x.shape)} {x.dtype}")
    out = torch.empty(n, dtype=x.dtype, device=x.device)
    if n and hidden:
        _C.check(
            _C.lib().mi8_moe_scatter_wgrad(x.data_ptr(), grad.data_ptr(), _dt(x, "scatter_wgrad"), tokens, hidden,
                                           indices.data_ptr(), top_k, out.data_ptr(), _stream(x)),
            "mi8_moe_scatter_wgrad",
        )
    return out


def _binned_gather(x, indices, weights, bins, bin_size: int, top_k: int) -> torch.Tensor:
    if x.dim() != 2:
        raise ValueError(f"binned_gather: expected a matrix, got {x.dim()} dimensions")
    x = x.contiguous()
    tokens, hidden = x.shape
    indices, bins = _i32(indices, "binned_gather"), _i32(bins, "binned_gather")
    if indices.shape[0] != tokens * top_k:
        raise ValueError(f"binned_gather: expected {tokens * top_k} indices, got {indices.shape[0]}")
    w, wp, wd = _weights(weights, tokens * top_k, "binned_gather")
    experts = bins.shape[0]
    out = torch.empty((experts, bin_size, hidden), dtype=x.dtype, device=x.device)
    if out.numel():
        _C.check(
            _C.lib().mi8_moe_binned_gather(x.data_ptr(), _dt(x, "binned_gather", allow_raw=w is None), tokens, hidden,
                                           indices.data_ptr(), wp, wd, bins.data_ptr(), experts, bin_size, top_k,
                                           out.data_ptr(), _stream(x)),
            "mi8_moe_binned_gather",
        )
    return out


def _binned_scatter(x, indices, weights, bins, top_k: int) -> torch.Tensor:
    if x.dim() != 3:
        raise ValueError(f"binned_scatter: expected a 3-tensor, got {x.dim()} dimensions")
    x = x.contiguous()
    experts, bin_size, hidden = x.shape
    indices, bins = _i32(indices, "binned_scatter"), _i32(bins, "binned_scatter")
    if bins.shape[0] != experts or indices.shape[0] % top_k:
        raise ValueError("binned_scatter: bins / indices do not match x and top_k")
    n = indices.shape[0]
    tokens = n // top_k
    w, wp, wd = _weights(weights, n, "binned_scatter")
    out = torch.empty((tokens, hidden), dtype=x.dtype, device=x.device)
    if out.numel():
        inverse = torch.empty(n, dtype=torch.int32, device=x.device)
        _C.check(
            _C.lib().mi8_moe_binned_scatter(x.data_ptr(), _dt(x, "binned_scatter"), tokens, hidden, indices.data_ptr(),
                                            wp, wd, bins.data_ptr(), experts, bin_size, top_k, inverse.data_ptr(),
                                            out.data_ptr(), _stream(x)),
            "mi8_moe_binned_scatter",
        )
    return out


def _binned_scatter_wgrad(x, grad, indices, bins, top_k: int) -> torch.Tensor:
    x, grad = x.contiguous(), grad.contiguous()
    experts, bin_size, hidden = x.shape
    indices, bins = _i32(indices, "binned_scatter_wgrad"), _i32(bins, "binned_scatter_wgrad")
    n = indices.shape[0]
    tokens = n // top_k
    if grad.shape != (tokens, hidden) or grad.dtype != x.dtype:
        raise ValueError("binned_scatter_wgrad: grad does not match x")
    out = torch.empty(n, dtype=x.dtype, device=x.device)
    if n:
        _C.check(
            _C.lib().mi8_moe_binned_scatter_wgrad(x.data_ptr(), grad.data_ptr(), _dt(x, "binned_scatter_wgrad"), tokens,
                                                  hidden, indices.data_ptr(), bins.data_ptr(), experts, bin_size, top_k,
                                                  out.data_ptr(), _stream(x)),
            "mi8_moe_binned_scatter_wgrad",
        )
    return out


# ---- autograd functions (reference: src/olmo_core/ops/moe.py:26-205) -------------------------------------------


class GatherOp(torch.autograd.Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    def forward(ctx: Any, x, indices, bin_ids, bins, top_k: int):
        ctx.save_for_backward(indices)
        ctx.top_k = top_k
        return _gather(x, indices, None, top_k)

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    def backward(ctx: Any, grad):
        (indices,) = ctx.saved_tensors
        return _scatter(grad.contiguous(), indices, None, ctx.top_k), None, None, None, None


@torch.compiler.disable
def gather(x, indices, bin_ids, bins, top_k: int) -> torch.Tensor:
    return GatherOp.apply(x, indices, bin_ids, bins, top_k)


class ScatterOp(torch.autograd.Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    def forward(ctx: Any, x, indices, bin_ids, weights, bins, top_k: int):
        maybe_x = [x] if ctx.needs_input_grad[3] else []
        ctx.save_for_backward(indices, weights, *maybe_x)
        ctx.top_k = top_k
        return _scatter(x, indices, weights, top_k)

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    def backward(ctx: Any, grad):
        grad = grad.contiguous()
        indices, weights = ctx.saved_tensors[:2]
        dgrad = _gather(grad, indices, weights, ctx.top_k) if ctx.needs_input_grad[0] else None
        wgrad = None
        if ctx.needs_input_grad[3]:
            wgrad = _scatter_wgrad(ctx.saved_tensors[-1], grad, indices, ctx.top_k)
        return dgrad, None, None, wgrad, None, None


@torch.compiler.disable
def scatter(x, indices, bin_ids, weights, bins, top_k: int) -> torch.Tensor:
    return ScatterOp.apply(x, indices, bin_ids, weights, bins, top_k)


class BinnedGatherOp(torch.autograd.Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    def forward(ctx: Any, x, indices, bins, bin_size: int, top_k: int):
        ctx.save_for_backward(indices, bins)
        ctx.top_k = top_k
        return _binned_gather(x, indices, None, bins, bin_size, top_k)

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    def backward(ctx: Any, grad):
        indices, bins = ctx.saved_tensors
        return _binned_scatter(grad.contiguous(), indices, None, bins, ctx.top_k), None, None, None, None


@torch.compiler.disable
def binned_gather(x, indices, bins, bin_size: int, top_k: int) -> torch.Tensor:
    return BinnedGatherOp.apply(x, indices, bins, bin_size, top_k)


class BinnedScatterOp(torch.autograd.Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    def forward(ctx: Any, x, indices, weights, bins, top_k: int):
        if x.dim() != 3:
            raise ValueError("binned_scatter: expected a 3-tensor")
        ctx.bin_size = x.size(1)
        ctx.top_k = top_k
        ctx.save_for_backward(x, indices, weights, bins)
        return _binned_scatter(x, indices, weights, bins, top_k)

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    def backward(ctx: Any, grad):
        grad = grad.contiguous()
        x, indices, weights, bins = ctx.saved_tensors
        out = _binned_gather(grad, indices, weights, bins, ctx.bin_size, ctx.top_k)
        wgrad = _binned_scatter_wgrad(x, grad, indices, bins, ctx.top_k) if ctx.needs_input_grad[2] else None
        return out, None, wgrad, None, None


@torch.compiler.disable
def binned_scatter(x, indices, weights, bins, top_k: int) -> torch.Tensor:
    return BinnedScatterOp.apply(x, indices, weights, bins, top_k)


def batched_histc(x: torch.Tensor, num_classes: int) -> torch.Tensor:
    """A batched ``torch.histc`` over the last axis (integer class ids in ``[0, num_classes)``)."""
    hist = torch.zeros((*x.shape[:-1], num_classes), dtype=x.dtype, device=x.device)
    hist.scatter_add_(-1, x, torch.ones_like(x))
    return hist


def histc(x: torch.Tensor, num_classes: int) -> torch.Tensor:
    return batched_histc(x.reshape(1, -1), num_classes).reshape(num_classes)


# ---- routing ---------------------------------------------------------------------------------------------------

MOST_EXPERTS, MOST_TOP_K, MOST_GROUPS = 512, 64, 32


def _route(logits, bias, top_k: int, softmax: bool, groups: int, kept: int, normalize: bool, scale: float):
    n, experts = logits.shape
    dev = logits.device
    weights = torch.empty((n, top_k), dtype=torch.float32, device=dev)
    indices = torch.empty((n, top_k), dtype=torch.int64, device=dev)
    if n == 0:
        return weights, indices, torch.zeros(experts, dtype=torch.int64, device=dev)
    counts = torch.empty(experts, dtype=torch.int64, device=dev)
    words = _C.lib().mi8_moe_route_workspace_words(n, experts)
    ws = torch.empty(words, dtype=torch.int32, device=dev) if words else None
    with _on(dev):
        _C.check(
            _C.lib().mi8_moe_route(logits.data_ptr(), _dt(logits, "route"), n, experts, top_k, int(softmax),
                                   bias.data_ptr() if bias is not None else None, groups, kept, int(normalize), scale,
                                   ws.data_ptr() if ws is not None else None, weights.data_ptr(), indices.data_ptr(), counts.data_ptr(),
                                   _stream(logits)),
            "mi8_moe_route",
        )
    return weights, indices, counts


class RouteOp(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, logits, bias, top_k, softmax, groups, kept, normalize, scale):
        weights, indices, counts = _route(logits, bias, top_k, softmax, groups, kept, normalize, scale)
        ctx.mark_non_differentiable(indices, counts)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, weights, indices)
        ctx.options = (softmax, normalize, scale)
        return weights, indices, counts

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad, _indices, _counts):
        if grad is None:
            return (None,) * 8
        logits, weights, indices = ctx.saved_tensors
        softmax, normalize, scale = ctx.options
        n, experts = logits.shape
        out = torch.empty_like(logits)
        if n:
            grad = grad.to(torch.float32).contiguous()
            with _on(logits.device):
                _C.check(
                    _C.lib().mi8_moe_route_grad(logits.data_ptr(), _dt(logits, "route"), n, experts, weights.shape[1], int(softmax), int(normalize),
                                                scale, weights.data_ptr(), indices.data_ptr(), grad.data_ptr(), out.data_ptr(),
                                                _stream(logits)),
                    "mi8_moe_route_grad",
                )
        return (out,) + (None,) * 7


def route(
    logits: torch.Tensor, top_k: int, *, gating: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
    groups_kept: int = 1, normalize: bool = False, scale: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    Choose ``top_k`` experts for every token from router logits ``[*, experts]`` (bfloat16, float16 or float32).

    :param gating: the scores are the ``"softmax"`` or the ``"sigmoid"`` of the logits.
    :param bias: ``[experts]``, added to the scores for the choice alone (it balances the load and gets no gradient).
    :param groups: the experts are this many groups of equal size; only the ``groups_kept`` groups with the largest sum of their two
        largest (biased) scores are chosen from.  With as many kept as there are, groups change nothing.
    :param normalize: divide the weights of a token by their sum.
    :param scale: factor of the weights.

    :returns: ``(expert_weights float32 [*, top_k], expert_indices int64 [*, top_k], batch_size_per_expert int64 [experts])``, what
        :class:`~olmo_core_amd.nn.ParallelDroplessMLP` takes.  The expert with the largest score comes first, the lowest index of equal ones.
        The weights are differentiable in the logits.  The choice is that of 64-bit scores (without a bias or groups that of the logits
        themselves); a NaN comes last.  A token whose chosen scores are all below 2^-1024 (every logit minus infinity, say) has normalised
        weights of zero.
    """
    if torch.compiler.is_compiling():
        return _traced_route(logits, top_k, gating=gating, bias=bias, groups=groups, groups_kept=groups_kept, normalize=normalize, scale=scale)
    if logits.dim() < 1:
        raise ValueError("route: logits need a dimension of experts")
    _dt(logits, "route")
    experts = logits.shape[-1]
    if gating not in ("softmax", "sigmoid"):
        raise ValueError(f"route: unknown gating '{gating}' (softmax or sigmoid)")
    if not 0 < experts <= MOST_EXPERTS or not 0 < groups <= MOST_GROUPS or experts % groups or not 0 < groups_kept <= groups:
        raise ValueError(f"route: {experts} experts in {groups} groups of which {groups_kept} are kept (at most {MOST_EXPERTS} experts in at most "
                         f"{MOST_GROUPS} groups of equal size)")
    if not 0 < top_k <= min(MOST_TOP_K, experts // groups * groups_kept):
        raise ValueError(f"route: cannot choose {top_k} of {experts // groups * groups_kept} experts (at most {MOST_TOP_K})")
    if bias is not None:
        if bias.shape != (experts,) or bias.device != logits.device or not torch.is_floating_point(bias):
            raise ValueError(f"route: bias must be {experts} floating point numbers on {logits.device}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
        bias = bias.detach().to(torch.float32).contiguous()
    flat = (logits if logits.dim() == 2 else logits.reshape(-1, experts)).contiguous()  # (a reshape is a node of the graph also where it changes nothing)
    args = (bias, top_k, gating == "softmax", groups, groups_kept, normalize, float(scale))
    if needs_autograd(flat):
        weights, indices, counts = RouteOp.apply(flat, *args)
    else:
        weights, indices, counts = _route(flat, *args)
    if logits.dim() != 2:
        weights, indices = (t.reshape(*logits.shape[:-1], top_k) for t in (weights, indices))
    return weights, indices, counts


_traced_route = torch.compiler.disable(route)  # (a graph break; asking whether there is a trace costs less than the wrapper does on every call)
