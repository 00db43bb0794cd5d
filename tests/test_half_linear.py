"""What ``ops.linear`` and ``ops.grouped_linear`` refuse before anything runs, and what the library says of sizes (no GPU)."""

import pytest
import torch

from olmo_core_amd import _C
from olmo_core_amd.ops import linear as linear_module
from olmo_core_amd.ops.linear import grouped_linear, linear


def test_no_cpu_path():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        grouped_linear(x, w, torch.tensor([2, 2]))


@pytest.fixture
def on_gpu(monkeypatch):
    """The checks behind the one for the device."""
    import olmo_core_amd.ops.linear as module

    monkeypatch.setattr(module, "_require_gpu", lambda t, what: None)


@pytest.mark.parametrize("call,error,match", [
    (lambda x, w: linear(x.float(), w.float()), TypeError, "unsupported input type"),
    (lambda x, w: linear(x, w.half()), TypeError, "weight is torch.float16"),
    (lambda x, w: linear(x, w[0]), ValueError, "not a matrix"),
    (lambda x, w: linear(x[0, 0], w), ValueError, "needs a dimension"),
    (lambda x, w: linear(x[:, :7], w), ValueError, "do not match"),
    (lambda x, w: linear(x, w, activation="tanh"), ValueError, "unknown activation"),
    (lambda x, w: linear(x, w, torch.zeros(6)[:5]), ValueError, "bias"),
    (lambda x, w: linear(x, w, torch.zeros(6, dtype=torch.float64)), TypeError, "bias"),
    (lambda x, w: linear(x, w, residual=torch.zeros(6, dtype=torch.bfloat16)), ValueError, "residual"),
    (lambda x, w: linear(x, w, residual=torch.zeros(4, 6)), TypeError, "residual"),
    (lambda x, w: linear(x, w.to("meta")), ValueError, "weight on meta"),
    (lambda x, w: linear(x[:, :1].expand(4, 1 << 22), w[:, :1].expand(6, 1 << 22)), ValueError, "more than the kernels address"),
    (lambda x, w: grouped_linear(x, w, torch.zeros(0, dtype=torch.int64)), ValueError, "vector of integers"),
    (lambda x, w: grouped_linear(x, w, torch.zeros(2)), ValueError, "vector of integers"),
    (lambda x, w: grouped_linear(x, w, torch.zeros(2, 1, dtype=torch.int64)), ValueError, "vector of integers"),
    (lambda x, w: grouped_linear(x, w, torch.zeros(4, dtype=torch.int64)), ValueError, "4 matrices"),
    (lambda x, w: grouped_linear(x[:, :7], w, torch.zeros(2, dtype=torch.int64)), ValueError, "do not match"),
    (lambda x, w: grouped_linear(x, w, torch.zeros(2, dtype=torch.int64), transposed=True), ValueError, "do not match 3"),
])
def test_refusals(on_gpu, call, error, match):
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(error, match=match):
        call(x, w)


def test_column_sums_have_room():
    words = _C.lib().mi8_half_epilogue_grad_workspace_words
    assert words(0, 8) == words(8, 0) == 0
    assert words(1, 1) == 1 and words(33, 5) % 5 == 0 and words(33, 5) > 0
    assert words(16384, 4096) % 4096 == 0


def test_which_tiles_groups_take():
    """What the library says it chooses, at sizes whose launches were recorded."""
    lib = _C.lib()
    assert lib.mi8_grouped_gemm_half_variant(131072, 1024, 2048, 64) == lib.mi8_grouped_gemm_half_variant(131072, 2048, 1024, 64) == _C.HALF_256
    assert lib.mi8_grouped_wgrad_half_variant(131072, 1024, 2048, 64) == _C.HALF_256
    assert lib.mi8_grouped_gemm_half_variant(4008, 1024, 512, 32) == lib.mi8_grouped_gemm_half_variant(4008, 512, 1024, 32) == _C.HALF_128
    assert lib.mi8_grouped_wgrad_half_variant(4008, 512, 1024, 32) == _C.HALF_128
    assert lib.mi8_grouped_gemm_half_variant(384, 1024, 2048, 64) == _C.HALF_64
    for call in (lib.mi8_grouped_gemm_half_variant, lib.mi8_grouped_wgrad_half_variant):
        assert call(0, 8, 0, 1) == call(8, 8, 8, 0) == -1
        assert all(call(t, n, k, e) in (_C.HALF_256, _C.HALF_128, _C.HALF_64) for t in (1, 999, 1 << 29) for n in (1, 1 << 20) for k in (1, 5000) for e in (1, 7, 1000))


def test_a_contiguous_copy_of_whole_chunks_is_an_operand(monkeypatch):
    """Of a transposed or expanded matrix: the library is not asked for another copy."""
    monkeypatch.setattr(_C, "lib", lambda: pytest.fail("copied twice"))
    w = torch.arange(48 * 40).view(48, 40).to(torch.bfloat16)
    for t in (w.t(), w[:1, :1].expand(24, 32), w[::2, ::5]):
        made = linear_module._operand(t)
        assert torch.equal(made, t) and linear_module._is_operand(made)
