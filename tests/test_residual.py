"""``nn.ResidualNorm``, ``nn.ResidualBlocks`` and the unquantised experts: parameters and refusals (no GPU)."""

import pytest
import torch

from olmo_core_amd.nn import DroplessMoEMLP, FeedForward, ParallelDroplessMLP, ResidualBlocks, ResidualNorm


@pytest.mark.parametrize("norm,names", [
    ("before", ["joins.0.pre_weight", "joins.1.pre_weight", "joins.2.pre_weight"]),
    ("after", ["joins.1.post_weight", "joins.2.post_weight", "joins.2.pre_weight"]),
    ("both", ["joins.0.pre_weight", "joins.1.post_weight", "joins.1.pre_weight", "joins.2.post_weight", "joins.2.pre_weight"]),
])
def test_parameters(norm, names):
    blocks = ResidualBlocks([torch.nn.Identity(), torch.nn.Identity()], d_model=24, norm=norm)
    assert [n for n, _ in blocks.named_parameters()] == names
    assert all(torch.equal(p, torch.ones(24)) for p in blocks.parameters())
    without = ResidualBlocks([torch.nn.Identity(), torch.nn.Identity()], d_model=24, norm=norm, final_norm=False)
    assert [n for n, _ in without.named_parameters()] == [n for n in names if n != "joins.2.pre_weight"]


def test_gate_and_meta():
    join = ResidualNorm(d_model=8, pre_norm=True, gate=0.25, init_device="meta")
    assert join.pre_weight.is_meta and join.post_weight is None
    join.to_empty(device="cpu").reset_parameters()
    assert torch.equal(join.gate, torch.full((8,), 0.25)) and torch.equal(join.pre_weight, torch.ones(8))
    blocks = ResidualBlocks([FeedForward(d_model=8, hidden_size=16)], d_model=8, gate=0.5, dtype=torch.bfloat16)
    assert [j.gate is not None for j in blocks.joins] == [False, True]
    assert all(p.dtype == torch.bfloat16 for p in blocks.joins.parameters())


@pytest.mark.parametrize("make,match", [
    (lambda: ResidualNorm(d_model=0), "d_model"),
    (lambda: ResidualNorm(d_model=16385), "d_model"),
    (lambda: ResidualNorm(d_model=8, dropout=1.5), "dropout"),
    (lambda: ResidualBlocks([], d_model=8, norm="first"), "unknown norm"),
    (lambda: DroplessMoEMLP(d_model=32, hidden_size=32, num_experts=2, scaling="tensorwise"), "unknown scaling"),
    (lambda: DroplessMoEMLP(d_model=32, hidden_size=32, num_experts=2, scaling="none", keep_float8_weights=True), "no float8 weights"),
    (lambda: DroplessMoEMLP(d_model=33, hidden_size=32, num_experts=2), "multiples of 16"),
])
def test_refusals(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        ResidualNorm(d_model=8, pre_norm=True)(torch.zeros(4, 8))
    mlp = DroplessMoEMLP(d_model=9, hidden_size=5, num_experts=2, scaling="none")
    with pytest.raises(RuntimeError, match="no CPU path"):
        mlp(torch.zeros(4, 9), torch.tensor([3, 1]))
    with pytest.raises(NotImplementedError, match="scales per row"):
        mlp.forward_gathered(torch.zeros(4, 9), torch.arange(4), 1, torch.tensor([3, 1]))
    assert ParallelDroplessMLP(mlp=mlp, top_k=1).d_model == 9
