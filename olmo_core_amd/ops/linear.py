"""
Linear layers in the model's own type (bfloat16 or float16): what a model keeps beside its float8 layers, on the matrix kernels of
``csrc/mi8_half_gemm.hip``.

* ``linear(x, weight, bias, activation=, residual=)``      -> ``residual + act(x @ weight.T + bias)``
* ``grouped_linear(x, weight, batch_size_per_expert)``     -> the product for rows sorted by expert, each group with a matrix of its own

Both are differentiable in every floating point argument.  Sums are float32 and rounded to the type once, after bias, activation and
residual.  Two more roundings are in a training step behind an activation, because the matrix units take 16-bit operands: of the activation's argument,
which is stored for the backward pass, and of its gradient in front of both products (in float16 the gradients' error is 3.0e-4 where that of the outputs'
rounding alone is 2.1e-4).  The counterparts of the float8 layers :func:`olmo_core_amd.float8.blockwise_linear` and
:func:`olmo_core_amd.float8.blockwise_grouped_linear` (reference: ``nn.Linear`` in ``src/olmo_core/nn/feed_forward.py:114-171`` and ``grouped_gemm.ops.gmm`` in
``src/olmo_core/nn/moe/mlp.py:177-292``).  Tensors must live on the GPU; there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from .. import _C
from ..float8.ops import _on, _require_gpu, _sizes_i64, _stream, needs_autograd
from .dropout import first_order

__all__ = ["ACTIVATIONS", "linear", "grouped_linear"]

#: what ``linear`` takes as ``activation`` beside ``None``
ACTIVATIONS = {"relu": _C.ACT_RELU, "silu": _C.ACT_SILU, "gelu": _C.ACT_GELU, "gelu_tanh": _C.ACT_GELU_TANH}

_CODE = {torch.bfloat16: _C.MI8_BF16, torch.float16: _C.MI8_F16, torch.float32: _C.MI8_F32}
_MOST_PITCH = 1 << 22
_MOST_SIZE = 1 << 30


def _pad8(n: int) -> int:
    return (n + 7) // 8 * 8


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` (2-D) with its rows contiguous, in place where they are."""
    return t if t.stride(1) == 1 or t.shape[1] <= 1 or t.numel() == 0 else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    """Elements from a row of ``t`` to the next (a single row has none: its own length)."""
    rows, cols = t.shape
    return t.stride(0) if rows > 1 and cols else cols


def _is_operand(t: torch.Tensor) -> bool:
    """Whether the products read ``t`` where it is: whole 16-byte chunks."""
    (rows, cols), (pitch, step) = t.shape, t.stride()
    if rows <= 1 or not cols:
        pitch = cols
    return cols % 8 == 0 and pitch % 8 == 0 and cols <= pitch < _MOST_PITCH and t.data_ptr() % 16 == 0 and (step == 1 or cols == 0)


def _operand(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy of it whose rows are whole 16-byte chunks (zeros behind the last column)."""
    if _is_operand(t):
        return t
    if t.stride(1) != 1:
        t = _rows(t)
        if _is_operand(t):  # (that copy has whole chunks already)
            return t
    rows, cols = t.shape
    padded = _pad8(cols)
    copy = t.new_empty((rows, padded))
    _C.check(_C.lib().mi8_half_pad(t.data_ptr(), _pitch(t), rows, cols, copy.data_ptr(), padded, _stream(t)), "mi8_half_pad")
    return copy


def _product(a, b, m: int, n: int, k: int, a_by_k: bool, b_by_k: bool, epilogue=None) -> torch.Tensor:
    out, lib = a.new_empty((m, n)), _C.lib()
    words = lib.mi8_gemm_half_workspace_bytes(m, n, k, a_by_k, b_by_k)
    ws = a.new_empty(words, dtype=torch.uint8) if words else None
    _C.check(
        lib.mi8_gemm_half(_CODE[a.dtype], a.data_ptr(), _operand_pitch(a), a_by_k, b.data_ptr(), _operand_pitch(b), b_by_k, m, n, k,
                               epilogue, out.data_ptr(), n, _C.HALF_ANY, ws.data_ptr() if words else None, _stream(a)),
        "mi8_gemm_half",
    )
    return out


def _operand_pitch(t: torch.Tensor) -> int:
    rows, cols = t.shape
    return t.stride(0) if rows > 1 and cols else _pad8(cols)


def _forward(x, weight, n: int, k: int, bias, residual, act: int, z):
    """``x``, ``weight``: operands; ``z``: ``None``, or the buffer that takes what the activation is applied to."""
    if bias is None and residual is None and z is None and act == _C.ACT_NONE:
        return _product(x, weight, x.shape[0], n, k, False, False)
    ep = _C.HalfEpilogue(activation=act)
    if bias is not None:
        ep.bias, ep.bias_dtype = bias.data_ptr(), _CODE[bias.dtype]
    if residual is not None:
        ep.residual, ep.ld_residual = residual.data_ptr(), _pitch(residual)
    if z is not None:
        ep.z, ep.ld_z = z.data_ptr(), z.shape[1]
    return _product(x, weight, x.shape[0], n, k, False, False, ctypes.byref(ep))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        n, k = weight.shape
        m = x.shape[0]
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        with _on(x.device):
            xo, wo = _operand(x), _operand(weight)
            # (the value the activation is applied to, rounded, is what its slope is taken at)
            z = x.new_empty((m, _pad8(n))) if act != _C.ACT_NONE and (need_x or need_w or need_b) else None
            y = _forward(xo, wo, n, k, bias, residual, act, z)
        ctx.save_for_backward(xo if need_w else None, wo if need_x else None, z)
        ctx.meta = (m, n, k, act, bias.dtype if bias is not None else None)
        return y

    @staticmethod
    @first_order
    def backward(ctx, gy):
        x, weight, z = ctx.saved_tensors
        m, n, k, act, bias_dtype = ctx.meta
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        gx = gw = gb = None
        gr = gy if need_r else None
        with _on(gy.device):
            gy = _rows(gy)
            products = need_x or need_w
            dz = gy
            if z is not None or need_b:
                write = products and (z is not None or not _is_operand(gy))
                if write:
                    dz = gy.new_empty((m, _pad8(n)))
                ws = None
                if need_b:
                    gb = gy.new_empty(n, dtype=bias_dtype)
                    ws = gy.new_empty(_C.lib().mi8_half_epilogue_grad_workspace_words(m, n), dtype=torch.float32)
                _C.check(
                    _C.lib().mi8_half_epilogue_grad(
                        _CODE[gy.dtype], gy.data_ptr(), _pitch(gy), z.data_ptr() if z is not None else None, _pad8(n), act, m, n,
                        dz.data_ptr() if write else None, _pad8(n), gb.data_ptr() if need_b else None, _CODE[bias_dtype] if need_b else 0,
                        ws.data_ptr() if need_b else None, _stream(gy)),
                    "mi8_half_epilogue_grad",
                )
            elif products:
                dz = _operand(gy)
            if need_x:
                gx = _product(dz, weight, m, k, n, False, True)
            if need_w:
                gw = _product(dz, x, n, k, m, True, True)
        return gx, gw, gb, gr, None


def _check_tensor(t: torch.Tensor, x: torch.Tensor, name: str, what: str, also=()) -> None:
    if t.dtype != x.dtype and t.dtype not in also:
        raise TypeError(f"{what}: {name} is {t.dtype}, the input {x.dtype}")
    if t.device != x.device:
        raise ValueError(f"{what}: input on {x.device}, {name} on {t.device}")


def _check_input(x: torch.Tensor, weight: torch.Tensor, what: str) -> None:
    _require_gpu(x, what)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{what}: unsupported input type {x.dtype} (bfloat16 or float16)")
    _check_tensor(weight, x, "weight", what)
    if weight.dim() != 2:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} is not a matrix")
    if x.dim() < 1:
        raise ValueError(f"{what}: the input needs a dimension of features")


def _flat(x: torch.Tensor) -> torch.Tensor:
    return x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def _linear(x, weight, bias, activation, residual):
    what = "linear"
    _check_input(x, weight, what)
    n, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"{what}: input features {x.shape[-1]} do not match weight {tuple(weight.shape)}")
    if activation is not None and activation not in ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation '{activation}' ({', '.join(ACTIVATIONS)} or None)")
    if bias is not None:
        _check_tensor(bias, x, "bias", what, (torch.float32,))
        if bias.shape != (n,):
            raise ValueError(f"{what}: bias {tuple(bias.shape)} for {n} output features")
        bias = bias.contiguous()
    shape = (*x.shape[:-1], n)
    if residual is not None:
        _check_tensor(residual, x, "residual", what)
        if residual.shape != shape:
            raise ValueError(f"{what}: residual {tuple(residual.shape)} for an output {shape}")
    x2 = _flat(x)
    if max(x2.shape[0], n, k) >= _MOST_SIZE or max(_pad8(n), _pad8(k)) >= _MOST_PITCH:
        raise ValueError(f"{what}: {tuple(x2.shape)} by {tuple(weight.shape)} is more than the kernels address ({_MOST_SIZE} rows, {_MOST_PITCH} features)")
    act = ACTIVATIONS[activation] if activation is not None else _C.ACT_NONE
    r2 = _rows(_flat(residual)) if residual is not None else None
    if r2 is not None and _pitch(r2) < n:  # (rows that lie over one another)
        r2 = r2.contiguous()
    if needs_autograd(*(t for t in (x, weight, bias, residual) if t is not None)):
        y = _Linear.apply(x2, weight, bias, r2, act)
    else:
        with _on(x.device):
            y = _forward(_operand(x2), _operand(weight), n, k, bias, r2, act, None)
    return y if x.dim() == 2 else y.reshape(shape)


def linear(
    x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """
    ``residual + act(x [*, K] @ weight[N, K].T + bias)`` in bfloat16 or float16, differentiable in all four tensors.  One launch; two where few tiles and a long K
    have it cut along K, and one more for each operand that is copied.

    :param bias: ``[N]``, of the input's type or float32.
    :param activation: ``"relu"``, ``"silu"``, ``"gelu"`` (the exact one), ``"gelu_tanh"`` or ``None``.
    :param residual: a tensor of the output's shape and type.

    Sizes, strides and alignment may be anything; operands whose rows are not whole 16-byte chunks are copied first.
    The activation's slope is taken at its argument rounded to the type, and the argument's gradient is rounded to it.  What ReLU shuts off has no gradient,
    whatever arrives.
    """
    if torch.compiler.is_compiling():
        return _traced_linear(x, weight, bias, activation, residual)
    return _linear(x, weight, bias, activation, residual)


# ---- rows sorted by expert -------------------------------------------------------------------------------------


def _grouped_product(x, w, sizes, n: int, k: int, w_by_k: bool) -> torch.Tensor:
    """Rows of ``x`` (an operand) in groups, times the group's matrix: ``w`` operand of ``experts`` matrices one below the other, ``[n, k]`` each or,
    ``w_by_k``, ``[k, n]``."""
    out = x.new_empty((x.shape[0], n))
    pitch = _operand_pitch(w)
    _C.check(
        _C.lib().mi8_grouped_gemm_half(_CODE[x.dtype], x.data_ptr(), _operand_pitch(x), w.data_ptr(), pitch, w_by_k, (k if w_by_k else n) * pitch,
                                       sizes.data_ptr(), sizes.numel(), x.shape[0], n, k, out.data_ptr(), n, _C.HALF_ANY, _stream(x)),
        "mi8_grouped_gemm_half",
    )
    return out


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, sizes, transposed):
        n, k = _features(weight, sizes.numel(), transposed)
        with _on(x.device):
            xo, wo = _operand(x), _operand(weight)
            y = _grouped_product(xo, wo, sizes, n, k, transposed)
        ctx.save_for_backward(xo if ctx.needs_input_grad[1] else None, wo if ctx.needs_input_grad[0] else None, sizes)
        ctx.meta = (tuple(weight.shape), transposed)
        return y

    @staticmethod
    @first_order
    def backward(ctx, gy):
        x, weight, sizes = ctx.saved_tensors
        shape, transposed = ctx.meta
        experts = sizes.numel()
        rows = shape[0] // experts
        n, k = (shape[1], rows) if transposed else (rows, shape[1])
        gx = gw = None
        with _on(gy.device):
            g = _operand(gy)
            if ctx.needs_input_grad[0]:
                gx = _grouped_product(g, weight, sizes, k, n, not transposed)
            if ctx.needs_input_grad[1]:
                a, b = (x, g) if transposed else (g, x)
                gw = gy.new_empty(shape)
                _C.check(
                    _C.lib().mi8_grouped_wgrad_half(_CODE[gy.dtype], a.data_ptr(), _operand_pitch(a), b.data_ptr(), _operand_pitch(b), sizes.data_ptr(),
                                                    experts, gy.shape[0], rows, shape[1], gw.data_ptr(), _C.HALF_ANY, _stream(gy)),
                    "mi8_grouped_wgrad_half",
                )
        return gx, gw, None, None


def _features(weight: torch.Tensor, experts: int, transposed: bool):
    """Output and input features of one expert."""
    rows, cols = weight.shape[0] // experts, weight.shape[1]
    return (cols, rows) if transposed else (rows, cols)


def _grouped_linear(x, weight, batch_size_per_expert, transposed):
    what = "grouped_linear"
    sizes = batch_size_per_expert
    if sizes.dim() != 1 or sizes.numel() == 0 or sizes.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: batch_size_per_expert must be a vector of integers, got {sizes.dtype} {tuple(sizes.shape)}")
    _check_input(x, weight, what)
    experts = sizes.numel()
    if weight.shape[0] % experts:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} is not {experts} matrices of equal size")
    n, k = _features(weight, experts, transposed)
    if x.shape[-1] != k:
        raise ValueError(f"{what}: input features {x.shape[-1]} do not match {k}")
    x2 = _flat(x)
    if max(x2.shape[0], n, k) >= _MOST_SIZE or max(_pad8(n), _pad8(k), _pad8(weight.shape[1])) >= _MOST_PITCH:
        raise ValueError(f"{what}: {tuple(x2.shape)} by {tuple(weight.shape)} is more than the kernels address ({_MOST_SIZE} rows, {_MOST_PITCH} features)")
    sizes = _sizes_i64(sizes, x.device)
    if needs_autograd(x, weight):
        y = _GroupedLinear.apply(x2, weight, sizes, transposed)
    else:
        with _on(x.device):
            y = _grouped_product(_operand(x2), _operand(weight), sizes, n, k, transposed)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], n)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, batch_size_per_expert: torch.Tensor, *, transposed: bool = False) -> torch.Tensor:
    """
    :func:`linear` without bias for rows that are sorted by expert: the first ``batch_size_per_expert[0]`` rows of ``x`` are multiplied with the
    first expert's matrix, the next ones with the second's, and so on (the sizes stay on the GPU).

    :param weight: the experts' matrices one below the other, ``[experts * N, K]``: ``y = x [T, K] @ w[e].T``.
    :param transposed: ``y = x [T, N] @ w[e]`` instead.

    Sizes count up to the number of rows in all.  Rows behind the last group give zeros, also as the gradient of ``x``, and the
    weight of an expert without rows a gradient of zeros.
    """
    if torch.compiler.is_compiling():
        return _traced_grouped_linear(x, weight, batch_size_per_expert, transposed)
    return _grouped_linear(x, weight, batch_size_per_expert, transposed)


# (a graph break under torch.compile; asking whether there is a trace costs less than the wrapper does on every call)
_traced_linear = torch.compiler.disable(_linear)
_traced_grouped_linear = torch.compiler.disable(_grouped_linear)
