"""What ``ops.norm`` and ``ops.dropout`` refuse before anything runs, and what the library says of sizes (no GPU)."""

import pytest
import torch

from olmo_core_amd import _C
from olmo_core_amd.ops import dropout as dropout_module
from olmo_core_amd.ops import norm as norm_module
from olmo_core_amd.ops.dropout import dropout
from olmo_core_amd.ops.norm import MOST_FEATURES, residual_norm


def test_no_cpu_path():
    x = torch.zeros(4, 8)
    for call in (lambda: dropout(x, 0.1, seed=1), lambda: residual_norm(x, pre_norm=True)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.fixture
def on_gpu(monkeypatch):
    """The checks behind the one for the device."""
    for module in (dropout_module, norm_module):
        monkeypatch.setattr(module, "_require_gpu", lambda t, what: None)


@pytest.mark.parametrize("call,error,match", [
    (lambda x: dropout(x.double(), 0.1, seed=1), TypeError, "unsupported type"),
    (lambda x: dropout(x, 1.5, seed=1), ValueError, "between 0 and 1"),
    (lambda x: dropout(x, float("nan"), seed=1), ValueError, "between 0 and 1"),
    (lambda x: dropout(x, 0.1, seed=-1), ValueError, "64-bit"),
    (lambda x: dropout(x, 0.1, seed=1, offset=1 << 64), ValueError, "64-bit"),
    (lambda x: dropout(x, 0.1, seed=torch.zeros(1)), ValueError, "one int64"),
    (lambda x: dropout(x, 0.1, seed=torch.zeros(2, dtype=torch.int64)), ValueError, "one int64"),
    (lambda x: residual_norm(x.double()), TypeError, "unsupported type"),
    (lambda x: residual_norm(x[0, 0]), ValueError, "features"),
    (lambda x: residual_norm(x[:, :0]), ValueError, "features"),
    (lambda x: residual_norm(x[:, :1].expand(4, MOST_FEATURES + 1)), ValueError, "features"),
    (lambda x: residual_norm(x, x[:1]), ValueError, "residual"),
    (lambda x: residual_norm(x, x.half()), TypeError, "residual"),
    (lambda x: residual_norm(x, post_weight=x[0, :7]), ValueError, "post_weight"),
    (lambda x: residual_norm(x, pre_weight=x[0].half()), TypeError, "pre_weight"),
    (lambda x: residual_norm(x, gate=x), ValueError, "gate"),
    (lambda x: residual_norm(x, p=0.1), ValueError, "seed"),
    (lambda x: residual_norm(x, p=2.0, seed=1), ValueError, "between 0 and 1"),
])
def test_refusals(on_gpu, call, error, match):
    with pytest.raises(error, match=match):
        call(torch.zeros(4, 8))


def test_workspace():
    words = _C.lib().mi8_residual_norm_workspace_words
    assert words(0, 8) == words(8, 0) == 0
    assert words(1, 4096) == 3 * 4096
    assert words(1 << 20, 64) == words(1 << 22, 64)


def test_argument_block():
    """The block that calls are packed into is the structure, field by field."""
    import ctypes
    import struct

    fields = _C.ResidualNorm._fields_
    codes = {ctypes.c_void_p: "Q", ctypes.c_uint64: "Q", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_uint32: "I", ctypes.c_float: "f"}
    assert struct.calcsize("@19Q6q7iI4f") == ctypes.sizeof(_C.ResidualNorm)
    assert "".join(codes[t] for _, t in fields) == "Q" * 19 + "q" * 6 + "i" * 7 + "I" + "f" * 4
    values = [i + 1 for i in range(len(fields))]
    a = _C.ResidualNorm.from_buffer_copy(norm_module._pack(*values))
    assert [getattr(a, name) for name, _ in fields] == values


@pytest.mark.parametrize("number", [5, (1 << 64) - 1])
def test_seeds_and_offsets_of_any_whole_number_type(number):
    import numpy as np

    want = dropout_module._mask(0.1, number, number, torch.device("cpu"), "call")
    made = dropout_module._mask(0.1, np.uint64(number), np.uint64(number), torch.device("cpu"), "call")
    assert made == want and type(made[0].seed) is int and type(made[0].offset) is int


@pytest.mark.parametrize("call", [lambda x, **kw: dropout(x, 0.1, **kw), lambda x, **kw: residual_norm(x, p=0.1, **kw)], ids=["dropout", "residual_norm"])
@pytest.mark.parametrize("kw,name", [({"seed": 1.5}, "seed"), ({"seed": "7"}, "seed"), ({"seed": 1, "offset": 2.0}, "offset"), ({"seed": 1, "offset": None}, "offset")])
def test_seeds_and_offsets_that_are_no_whole_numbers(on_gpu, call, kw, name):
    with pytest.raises(ValueError, match=f"{name} .* no 64-bit number"):
        call(torch.zeros(4, 8), **kw)


@pytest.mark.parametrize("residual,gate", [(False, False), (True, False), (True, True)])
def test_few_python_calls(on_gpu, monkeypatch, residual, gate):
    """Small calls are bound by the host: what a step with gradients calls of this package's functions, the library's own left out (they do nothing here)."""
    import contextlib
    import sys

    class Nothing:
        mi8_residual_norm_forward = mi8_residual_norm_backward = staticmethod(lambda *args: 0)
        mi8_residual_norm_workspace_words = staticmethod(lambda rows, features: 3 * features)

    monkeypatch.setattr(norm_module, "_on", lambda device, here=contextlib.nullcontext(): here)
    monkeypatch.setattr(norm_module, "_stream", lambda t: 0)
    monkeypatch.setattr(norm_module._C, "lib", lambda: Nothing)
    x, r = torch.zeros(5, 8, requires_grad=True), torch.zeros(5, 8, requires_grad=True) if residual else None
    w, s = torch.zeros(8, requires_grad=True), torch.zeros(8, requires_grad=True) if gate else None
    names = []

    def note(frame, event, arg):
        if event == "call" and "olmo_core_amd" in frame.f_code.co_filename:
            names.append(frame.f_code.co_name)

    ins = [t for t in (x, r, w, s) if t is not None]
    sys.setprofile(note)
    try:
        outs = residual_norm(x, r, post_weight=w, pre_norm=True, gate=s)
        made = torch.autograd.grad(outs, ins, [torch.zeros(5, 8), torch.zeros(5, 8)])
    finally:
        sys.setprofile(None)
    assert [t.shape for t in made] == [t.shape for t in ins]
    # the call and what is behind it, its checks, two passes of the autograd function, a launch and its status in each
    assert len(names) <= 24, names


def test_the_workspace_is_that_of_the_tensors_device(on_gpu, monkeypatch):
    """Its size follows from the device that is current when the library is asked, which has to be the tensors' own."""
    import contextlib

    current = []

    @contextlib.contextmanager
    def on(device):
        current.append(device)
        yield
        current.pop()

    class Asked:
        @staticmethod
        def mi8_residual_norm_forward(*args):
            return 0 if current else 1

        mi8_residual_norm_backward = mi8_residual_norm_forward

        @staticmethod
        def mi8_residual_norm_workspace_words(rows, features):
            assert current
            return 3 * features

    monkeypatch.setattr(norm_module, "_on", on)
    monkeypatch.setattr(norm_module, "_stream", lambda t: 0)
    monkeypatch.setattr(norm_module._C, "lib", lambda: Asked)
    x, w = torch.zeros(5, 8, requires_grad=True), torch.zeros(8, requires_grad=True)
    out = residual_norm(x, post_weight=w)[0]
    assert [t.shape for t in torch.autograd.grad(out, [x, w], torch.zeros(5, 8))] == [(5, 8), (8,)]
