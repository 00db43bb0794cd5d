"""Routing without a GPU: refusals, the C ABI's checks of arguments, the layers' configuration."""

import pytest
import torch

from olmo_core_amd import _C
from olmo_core_amd.nn import DroplessMoE, DroplessMoEMLP, MoERouter, ParallelDroplessMLP
from olmo_core_amd.ops.moe import route
from oracle import route_oracle as R


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="GPU"):
        route(torch.randn(4, 8), 2)


def test_entry_points_check_their_arguments():
    L = _C.lib()
    p = 1 << 20  # (never read: every call is refused on the host)
    call = lambda l=p, dt=0, n=200, e=64, k=8, groups=1, kept=1, ws=p, w=p: L.mi8_moe_route(  # noqa: E731
        l, dt, n, e, k, 1, None, groups, kept, 0, 1.0, ws, w, p, p, None)
    assert call(l=None) == call(w=None) == call(dt=3) == call(n=0) == call(k=0) == call(e=0) == call(ws=None) == -1
    assert call(e=513) == call(k=65) == call(k=9, e=8) == call(groups=7) == call(groups=64) == call(groups=8, kept=9) == call(groups=8, kept=0) == -2
    assert call(groups=16, kept=1) == -2  # 4 experts to choose 8 from
    assert L.mi8_moe_route_grad(p, 0, 4, 64, 8, 1, 0, 1.0, p, p, None, p, None) == -1
    assert L.mi8_moe_route_workspace_words(128, 64) == 0 and L.mi8_moe_route_workspace_words(129, 64) == 9 * 64
    assert L.mi8_moe_route_workspace_words(0, 64) == 0


def test_layers_fit_together():
    mlp = DroplessMoEMLP(d_model=64, hidden_size=32, num_experts=4, scaling="blockwise")
    with pytest.raises(ValueError, match="scaling"):
        DroplessMoEMLP(d_model=64, hidden_size=32, num_experts=4, scaling="tensorwise")
    experts = ParallelDroplessMLP(mlp=mlp, top_k=2)
    DroplessMoE(router=MoERouter(d_model=64, num_experts=4, top_k=2), experts=experts)
    for kw in (dict(d_model=64, num_experts=4, top_k=1), dict(d_model=64, num_experts=8, top_k=2), dict(d_model=32, num_experts=4, top_k=2)):
        with pytest.raises(ValueError, match="fit"):
            DroplessMoE(router=MoERouter(**kw), experts=experts)
    router = MoERouter(d_model=64, num_experts=4, top_k=2, bias_gamma=0.1)
    assert set(router.state_dict()) == {"weight", "score_bias"}


def test_oracle_agrees_with_topk():
    g = torch.Generator().manual_seed(0)
    l = torch.randn(50, 16, generator=g)
    w, i, n = R.route(l, 4)
    want = torch.softmax(l.double(), -1).topk(4)
    assert torch.equal(i, want.indices) and torch.allclose(w, want.values) and int(n.sum()) == 200


@pytest.mark.parametrize("to", [torch.bfloat16, torch.float16, torch.float64])
def test_bias_stays_float32(to):
    """A bias of half and more, in steps that bfloat16 would round away."""
    router = MoERouter(d_model=64, num_experts=4, top_k=2, gating="sigmoid", bias_gamma=1e-3)
    start = torch.tensor([0.6, 0.7, -0.3, 0.0123])
    router.score_bias.copy_(start)
    router = router.to(to)
    assert router.weight.dtype == to and router.score_bias.dtype == torch.float32 and torch.equal(router.score_bias, start)
    router.slots_since.copy_(torch.tensor([9, 1, 1, 1]))
    router.post_batch()
    assert torch.equal(router.score_bias, start + 1e-3 * torch.tensor([-1.0, 1.0, 1.0, 1.0]))
    assert set(router.state_dict()) == {"weight", "score_bias"}
    meta = MoERouter(d_model=64, num_experts=4, top_k=2, bias_gamma=1e-3, init_device="meta").to(to).to_empty(device="cpu")
    meta.reset_parameters()
    assert meta.score_bias.dtype == torch.float32 and not meta.score_bias.any()
    other = MoERouter(d_model=64, num_experts=4, top_k=2, bias_gamma=1e-3)
    other.load_state_dict({k: v.to(torch.bfloat16) for k, v in router.state_dict().items()}, assign=True)
    other.slots_since.copy_(torch.tensor([9, 1, 1, 1]))
    other.post_batch()
    assert other.score_bias.dtype == torch.float32
    holder = torch.nn.ModuleList([router]).to("meta")
    assert holder[0].score_bias.is_meta and holder[0].score_bias.dtype == torch.float32
