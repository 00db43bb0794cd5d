from .feed_forward import FeedForward, swiglu
from .moe import DroplessMoE, DroplessMoEMLP, MoERouter, ParallelDroplessMLP, float8_dropless_mlp

__all__ = ["FeedForward", "swiglu", "DroplessMoE", "DroplessMoEMLP", "MoERouter", "ParallelDroplessMLP", "float8_dropless_mlp"]
