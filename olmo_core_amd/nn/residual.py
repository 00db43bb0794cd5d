"""
Blocks on a residual stream, with the norms and the dropout between them in one pass (:func:`olmo_core_amd.ops.norm.residual_norm`).

The reference writes a block as ``h = x + dropout(block(norm(x)))``, or ``h = x + dropout(norm(block(x)))`` with the norm reordered
(``src/olmo_core/nn/transformer/block.py``).  Read along the stream, what stands between two blocks is always the same: the last block's output,
normed or not, dropped, joins the stream, and the next block wants the stream's norm.  :class:`ResidualNorm` is that place with its parameters,
:class:`ResidualBlocks` a chain of blocks joined by them.
"""

from __future__ import annotations

from typing import Iterable, Optional, Tuple, Union

import torch
import torch.nn as nn

from ..ops.norm import MOST_FEATURES, residual_norm

__all__ = ["ResidualNorm", "ResidualBlocks"]


def _seed(p: float, seed: Optional[Union[int, torch.Tensor]], device: torch.device) -> Optional[Union[int, torch.Tensor]]:
    """``seed``, or one drawn from the generator of the CPU (:func:`torch.manual_seed`) where dropout needs one."""
    if p == 0.0 or seed is not None:
        return seed
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("dropout inside a captured graph needs a seed on the GPU: one drawn here would be the same in every replay")
    return int(torch.randint(0, 2**63 - 1, (), device="cpu"))


class ResidualNorm(nn.Module):
    """
    Where a block's output joins the residual stream: ``forward(branch, residual) -> (stream, normed)``, see
    :func:`~olmo_core_amd.ops.norm.residual_norm`.

    :param post_norm, pre_norm: a norm of the branch, of the stream, each with a weight (``post_weight``, ``pre_weight``).
    :param gate: a learnt factor for each feature of the branch, this much at first (``None``: no gate).
    :param dropout: of the branch, in training.
    """

    def __init__(
        self, *, d_model: int, post_norm: bool = False, pre_norm: bool = False, gate: Optional[float] = None, dropout: float = 0.0, eps: float = 1e-6,
        dtype: torch.dtype = torch.float32, init_device: str = "cpu",
    ):
        super().__init__()
        if not 0 < d_model <= MOST_FEATURES:
            raise ValueError(f"d_model {d_model} is not between 1 and {MOST_FEATURES}")
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout {dropout} is not between 0 and 1")
        self.d_model, self.dropout, self.eps, self.first_gate = d_model, dropout, eps, gate

        def weight(wanted: bool):
            return nn.Parameter(torch.empty(d_model, device=init_device, dtype=dtype)) if wanted else None

        self.post_weight, self.pre_weight, self.gate = weight(post_norm), weight(pre_norm), weight(gate is not None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        for w, value in ((self.post_weight, 1.0), (self.pre_weight, 1.0), (self.gate, self.first_gate)):
            if w is not None and not w.is_meta:
                nn.init.constant_(w, value)

    def forward(
        self, branch: torch.Tensor, residual: Optional[torch.Tensor] = None, *, seed: Optional[Union[int, torch.Tensor]] = None, offset: int = 0,
    ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """
        :param branch, residual: ``[*, d_model]``.
        :param seed, offset: what the dropout's mask is made from, see :func:`~olmo_core_amd.ops.dropout.dropout`; ``None``: a seed is drawn.
        """
        p = self.dropout if self.training else 0.0
        # (a weight is of the branch's type or float32)
        post, pre, gate = (w if w is None or w.dtype in (torch.float32, branch.dtype) else w.to(torch.float32)
                           for w in (self.post_weight, self.pre_weight, self.gate))
        return residual_norm(branch, residual, post_weight=post, pre_weight=pre, gate=gate, eps=self.eps, p=p, seed=_seed(p, seed, branch.device), offset=offset)

    def extra_repr(self) -> str:
        return f"d_model={self.d_model}, dropout={self.dropout}, eps={self.eps}"


class ResidualBlocks(nn.Module):
    """
    A chain of blocks (:class:`FeedForward`, :class:`DroplessMoE`, anything that maps ``[*, d_model]`` to itself) on a residual stream:
    ``forward(x)`` is the stream behind the last block, or its norm.

    :param norm: ``"before"``: each block sees the stream's norm; ``"after"``: it sees the stream, and its output is normed (the reference's
        reordered norm); ``"both"``.
    :param final_norm: the result is the norm of the stream behind the last block.
    :param gate, dropout, eps: see :class:`ResidualNorm`.
    :param block_dtype: the type that the blocks work in (``None``: the stream's).  A float32 stream around bfloat16 blocks keeps what they add.
    """

    def __init__(
        self, blocks: Iterable[nn.Module], *, d_model: int, norm: str = "before", final_norm: bool = True, gate: Optional[float] = None, dropout: float = 0.0,
        eps: float = 1e-6, block_dtype: Optional[torch.dtype] = None, dtype: torch.dtype = torch.float32, init_device: str = "cpu",
    ):
        super().__init__()
        if norm not in ("before", "after", "both"):
            raise ValueError(f"unknown norm '{norm}' (before, after or both)")
        self.blocks = nn.ModuleList(blocks)
        self.norm, self.block_dtype = norm, block_dtype
        n = len(self.blocks)
        before, after = norm != "after", norm != "before"
        shared = {"d_model": d_model, "eps": eps, "dtype": dtype, "init_device": init_device}
        # joins[i] stands in front of block i, the last one behind them all
        self.joins = nn.ModuleList(
            ResidualNorm(post_norm=after and i > 0, pre_norm=before if i < n else final_norm, gate=gate if i > 0 else None,
                         dropout=dropout if i > 0 else 0.0, **shared)
            for i in range(n + 1)
        )

    def reset_parameters(self) -> None:
        for join in self.joins:
            join.reset_parameters()

    def forward(self, x: torch.Tensor, *, seed: Optional[Union[int, torch.Tensor]] = None, offset: int = 0) -> torch.Tensor:
        """
        :param x: ``[*, d_model]``, the stream in front of the first block.
        :param seed: of the dropout of all blocks, which take different masks of it; ``None``: one is drawn.
        :param offset: of the first block's mask, one more for each further block.  What else takes masks from the same seed (another chain in the same
            captured graph, say) needs offsets apart from these ``len(blocks)``, or its masks are the same.
        """
        seed = _seed(max(join.dropout for join in self.joins) if self.training else 0.0, seed, x.device)
        stream, normed = self.joins[0](x)
        for i, block in enumerate(self.blocks):
            into = normed if normed is not None else stream
            branch = block(into if self.block_dtype is None else into.to(self.block_dtype))
            stream, normed = self.joins[i + 1](branch, stream, seed=seed, offset=offset + i)
        return normed if normed is not None else stream
