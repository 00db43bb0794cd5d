"""Block scales without a GPU: configuration, refusals, the C ABI's checks of arguments, the oracle itself."""

import pytest
import torch

from olmo_core_amd import _C
from olmo_core_amd.float8 import AOFloat8LinearRecipe, Float8Config, blockwise_grouped_linear, blockwise_linear, blockwise_weight, ops
from olmo_core_amd.float8.ao import AOCastConfig, AOFloat8LinearConfig, AOScalingGranularity
from olmo_core_amd.float8.native_config import CastConfig, Float8LinearConfig, ScalingGranularity, ScalingType
from oracle import block_oracle as B


def test_recipe():
    c = Float8LinearConfig.from_recipe_name(AOFloat8LinearRecipe.blockwise.to_ao_type())
    assert c.any_blockwise and not c.any_axiswise
    assert all(k.scaling_granularity is ScalingGranularity.BLOCKWISE and k.target_dtype == torch.float8_e4m3fn for k in c._casts)
    assert c.cast_config_input.short_str() == "dyn_blk_e4m3"
    again = Float8Config.from_dict(Float8Config(ao_recipe=AOFloat8LinearRecipe.blockwise).as_config_dict())
    assert again.ao_recipe == AOFloat8LinearRecipe.blockwise


def test_all_casts_or_none():
    block = AOCastConfig(scaling_granularity=AOScalingGranularity.blockwise)
    with pytest.raises(ValueError, match="all casts"):
        AOFloat8LinearConfig(cast_config_input=block).to_ao_type()
    c = AOFloat8LinearConfig(cast_config_input=block, cast_config_weight=block, cast_config_grad_output=block).to_ao_type()
    assert c.cast_config_grad_output_for_grad_weight.target_dtype == torch.float8_e4m3fn
    with pytest.raises(ValueError, match="e4m3"):
        CastConfig(scaling_granularity=ScalingGranularity.BLOCKWISE, target_dtype=torch.float8_e5m2)
    with pytest.raises(ValueError, match="dynamic"):
        CastConfig(scaling_granularity=ScalingGranularity.BLOCKWISE, scaling_type=ScalingType.DISABLED)


def test_no_cpu_path():
    x, w = torch.randn(4, 32).bfloat16(), torch.randn(16, 32).bfloat16()
    with pytest.raises(RuntimeError, match="GPU"):
        blockwise_linear(x, w)
    with pytest.raises(RuntimeError, match="GPU"):
        blockwise_grouped_linear(x, w, torch.tensor([4]))
    with pytest.raises(RuntimeError, match="GPU"):
        blockwise_weight(w)
    with pytest.raises(ValueError, match="multiples of 16"):
        blockwise_weight(torch.randn(20, 32))


def test_entry_points_check_their_arguments():
    L = _C.lib()
    assert L.mi8_block_scale_bytes(1, 1) == 128 and L.mi8_block_scale_bytes(129, 257) == 256 * 3 and L.mi8_block_scale_bytes(0, 4) == 0
    p = 1 << 20  # (never read: every call is refused on the host)
    cast = lambda x=p, dt=0, rows=4, cols=32, n=1, out=p, ld=128, s=p, out_t=p, ld_t=128, s_t=p: L.mi8_cast_block(  # noqa: E731
        x, dt, rows, cols, n, 0, out, ld, s, out_t, ld_t, s_t, None)
    assert cast(x=None) == cast(out=None, out_t=None) == cast(dt=2) == cast(rows=0) == cast(n=0) == -1
    for bad in (dict(cols=24), dict(x=p + 8), dict(ld=112), dict(ld=136), dict(s=None), dict(ld_t=112), dict(s_t=None), dict(out=p + 8), dict(rows=1 << 31)):
        assert cast(**bad) == -2, bad
    gemm = lambda a=p, lda=128, b=p, M=4, N=16, K=100, out=p, dt=0, ldc=16, v=-1: L.mi8_gemm_fp8_block(  # noqa: E731
        a, lda, p, b, 128, p, M, N, K, out, dt, ldc, v, None)
    assert gemm(a=None) == gemm(out=None) == gemm(dt=4) == gemm(M=0) == gemm(K=0) == -1
    for bad in (dict(N=12), dict(ldc=8), dict(ldc=20), dict(K=129), dict(lda=136), dict(a=p + 4), dict(out=p + 8), dict(M=1 << 30), dict(lda=1 << 24), dict(v=4), dict(v=-2), dict(v=3, dt=1)):
        assert gemm(**bad) == -2, bad
    assert L.mi8_grouped_gemm_fp8_block(p, 128, p, p, 128, 2048, p, None, 4, 10, 16, 100, p, 0, 16, None) == -1
    assert L.mi8_grouped_gemm_fp8_block(p, 128, p, p, 128, 2050, p, p, 4, 10, 16, 100, p, 0, 16, None) == -2
    assert L.mi8_grouped_wgrad_fp8_block(p, p, p, p, 128, p, 2, 200, 16, 16, p, 0, None) == -2


def test_batches_check_their_arguments():
    L = _C.lib()
    p = 1 << 20  # (never read: every call is refused on the host)

    def cast(n=2, count=None, **kw):
        items = (_C.BlockCastItem * n)(*[_C.BlockCastItem(x=p, rows=4, cols=32, out=p, ld_out=128, scales=p, out_t=p, ld_t=128, scales_t=p, matrices=1)
                                         for _ in range(n)])
        for name, v in kw.items():
            setattr(items[n - 1], name, v)
        return L.mi8_cast_block_batch(items, n if count is None else count, None)

    assert cast(count=0) == cast(n=9) == cast(count=-1) == L.mi8_cast_block_batch(None, 1, None) == -1
    groups = dict(group_sizes=p, num_groups=2, ld_t=384)
    for bad in (dict(x=None), dict(rows=0), dict(matrices=0), dict(out=None, out_t=None), dict(group_sizes=p), dict(num_groups=2), dict(num_groups=-1),
                dict(groups, square=1), dict(groups, matrices=2)):
        assert cast(**bad) == -1, bad
    for bad in (dict(hp_dtype=1), dict(cols=24), dict(x=p + 8), dict(ld_out=112), dict(ld_t=112), dict(scales=None), dict(groups, ld_t=112),
                dict(rows=1 << 31), dict(rows=(1 << 31) - 256, cols=(1 << 31) - 256, ld_out=1 << 31, ld_t=1 << 31, matrices=(1 << 31) - 1)):
        assert cast(**bad) == -2, bad

    def gemm(n=2, count=None, **kw):
        items = (_C.BlockProduct * n)(*[_C.BlockProduct(a=p, lda=128, a_scales=p, b=p, ldb=128, b_scales=p, M=4, N=16, K=100, out=p, ldc=16) for _ in range(n)])
        for name, v in kw.items():
            setattr(items[n - 1], name, v)
        return L.mi8_gemm_fp8_block_batch(items, n if count is None else count, None)

    assert gemm(count=0) == gemm(n=9) == L.mi8_gemm_fp8_block_batch(None, 1, None) == -1
    for bad in (dict(a=None), dict(b_scales=None), dict(out=None), dict(out_dtype=4), dict(M=0), dict(K=0)):
        assert gemm(**bad) == -1, bad
    for bad in (dict(N=12), dict(ldc=8), dict(K=129), dict(lda=136), dict(a=p + 4), dict(out=p + 8), dict(M=1 << 30), dict(ldb=1 << 24)):
        assert gemm(**bad) == -2, bad
    for items in ([], [None] * 9):
        with pytest.raises(ValueError):
            ops.cast_blockwise_batch(items)
        with pytest.raises(ValueError):
            ops.gemm_fp8_blockwise_batch(items)
    with pytest.raises(RuntimeError):
        ops.cast_blockwise_batch([(torch.zeros(16, 16), {})])


def test_batch_of_casts_refuses_options_that_do_not_fit():
    x, sizes = torch.zeros(32, 16), torch.tensor([16, 16])
    for kw in (dict(group_sizes=sizes, square=True), dict(group_sizes=sizes, matrices=2)):
        with pytest.raises(ValueError):
            ops.cast_blockwise_batch([(x, kw)])
    for kw in (dict(sqare=True), dict(sizes=sizes)):
        with pytest.raises(TypeError):
            ops.cast_blockwise_batch([(x, kw)])


def test_oracle_rounds_as_torch_does():
    v = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.05, 0.05, 5001)]).double()
    assert torch.equal(B.round_e4m3(v.float().double()), v.float().to(torch.float8_e4m3fn).double())


def test_oracle_scales():
    amax = torch.tensor([448.0, 448.5, 1.75, 1.76, 1.0, 3e38, 2.0 ** -112, 0.0])
    k = B.exponent(amax)
    assert k.tolist() == [0, -1, 8, 7, 8, -120, 120, 120]
    assert bool((torch.ldexp(amax.double(), k) <= 448).all())


def test_which_recipe_is_asked_of_one_cast(monkeypatch):
    """Every call of every float8 linear asks: blockwise is for all casts or for none."""
    configs = [(Float8LinearConfig.from_recipe_name(name), name == "blockwise") for name in ("tensorwise", "rowwise", "rowwise_with_gw_hp", "blockwise")]
    monkeypatch.setattr(Float8LinearConfig, "_casts", property(lambda self: pytest.fail("all six casts are looked at")))
    assert all(c.any_blockwise is want for c, want in configs)


def test_an_expert_layer_of_before_is_rowwise():
    """A module that was pickled whole before there was a choice has no such attribute of its own."""
    from olmo_core_amd.nn import DroplessMoEMLP

    mlp = DroplessMoEMLP(d_model=64, hidden_size=32, num_experts=4)
    del mlp.__dict__["scaling"]
    assert mlp.scaling == "rowwise"
    mlp._only_rowwise("forward_gathered")


def test_kernels_of_grouped_products():
    """Large groups take the 256 x 256 tiles, small problems and float32 outputs the ring tiles; an empty problem none."""
    L = _C.lib()
    assert L.mi8_grouped_gemm_fp8_block_variant(131072, 1024, 2048, 128, 0) == L.mi8_grouped_wgrad_fp8_block_variant(131072, 1024, 2048, 128, 0) == 3
    f32 = ops._HP_CODE[torch.float32]
    for f in (L.mi8_grouped_gemm_fp8_block_variant, L.mi8_grouped_wgrad_fp8_block_variant):
        assert 0 <= f(200, 128, 256, 4, 0) < 3 and 0 <= f(131072, 1024, 2048, 128, f32) < 3
        assert f(0, 1024, 2048, 64, 0) == f(200, 0, 2048, 64, 0) == f(200, 1024, 0, 64, 0) == f(200, 1024, 2048, 0, 0) == -1
