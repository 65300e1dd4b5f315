"""Refusals and host-side checks of gated_linear and lora_linear that need no GPU."""
import ctypes
import os

import pytest
import torch

from opengda_b200.ops.ffn import gated_linear, gated_linear_backward, gated_linear_forward
from opengda_b200.ops.lora import lora_linear

BF = torch.bfloat16


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 16, dtype=BF), torch.zeros(8, 16, dtype=BF)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear(x, w, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear_forward(x, w, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear_backward(torch.zeros(4, 8, dtype=BF), x, w, w, torch.zeros(0))
    with pytest.raises(RuntimeError, match="CUDA"):
        lora_linear(x, w, torch.zeros(1, 8, 16, dtype=BF), torch.zeros(1, 8, 8, dtype=BF), torch.zeros(4, dtype=torch.int32))


def test_types_and_activation_are_refused():
    x, w = torch.zeros(4, 16), torch.zeros(8, 16)
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        gated_linear(x, w, w)
    with pytest.raises(ValueError, match="act"):
        gated_linear(x.to(BF), w.to(BF), w.to(BF), act="tanh")


def test_lora_refuses_gradients():
    x, w = torch.zeros(4, 16, dtype=BF), torch.zeros(8, 16, dtype=BF)
    a, b, i = torch.zeros(1, 8, 16, dtype=BF, requires_grad=True), torch.zeros(1, 8, 8, dtype=BF), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no backward"):
        lora_linear(x, w, a, b, i)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        lora_linear(x, w, a, b, i)


def test_out_that_requires_a_gradient_is_refused():
    x, w = torch.zeros(4, 16, dtype=BF), torch.zeros(8, 16, dtype=BF)
    out = torch.zeros(4, 8, dtype=BF, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        gated_linear(x, w, w, out=out)


def test_c_entry_points_report_and_do_not_throw():
    """The C entries return -1 on misuse (checked before anything touches a GPU)."""
    lib = ctypes.CDLL(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "opengda_b200", "lib",
                                   "libgicc.so"))
    p, ll, i = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int
    f = lib.gicc_gated_linear
    f.argtypes = [p, p, p, p, i, i, i, ll, ll, ll, ll, i, i, p, p]
    assert f(None, None, None, None, 4, 16, 8, 16, 16, 16, 8, 0, 1, None, None) == -1   # no pointers
    assert f(16, 16, 16, 16, 4, 12, 8, 16, 16, 16, 8, 0, 1, None, None) == -1           # H % 8
    assert f(16, 16, 16, 16, 4, 16, 8, 16, 16, 16, 8, 7, 1, None, None) == -1           # unknown activation
    assert f(16, 24, 16, 16, 4, 16, 8, 16, 16, 16, 8, 0, 1, None, None) == -1           # unaligned w_gate
    assert f(16, 16, 16, 16, 4, 16, 8, 16, 16, 16, 7, 0, 1, None, None) == -1           # ldh < I
    b = lib.gicc_gated_linear_backward
    b.argtypes = [p] * 9 + [i] * 3 + [ll] * 6 + [i, i, p]
    assert b(16, 16, 16, 16, None, 16, 16, None, None, 4, 16, 8, 8, 16, 16, 16, 16, 16, 0, 1, None) == -1  # no saved
    assert b(16, 16, 16, 16, 16, 16, None, 16, None, 4, 16, 8, 8, 16, 16, 16, 16, 16, 0, 1, None) == -1    # one gradient
    g = lib.gicc_lora_linear
    g.argtypes = [p] * 8 + [i] * 5 + [ll] * 3 + [i, p]
    assert g(16, 16, 16, 16, 16, None, 16, 16, 4, 16, 8, 1, 12, 16, 16, 8, 1, None) == -1      # r % 8
    assert g(16, 16, 16, 16, 16, None, 16, 16, 4, 16, 8, 1, 136, 16, 16, 8, 1, None) == -1     # r > 128
    assert g(16, 16, 16, 16, 16, None, 16, 16, 4, 16, 8, 8193, 8, 16, 16, 8, 1, None) == -1    # too many adapters
    assert g(16, 16, 16, 16, None, None, 16, 16, 4, 16, 8, 1, 8, 16, 16, 8, 1, None) == -1     # no indexes
    assert g(16, 16, 16, 16, 16, None, 16, 16, 2 ** 30, 16, 8, 1, 8, 16, 16, 8, 1, None) == -1  # too many rows
