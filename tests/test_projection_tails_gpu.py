"""The activations of gated_linear far from zero, element by element and relative to their value."""
import math

import pytest
import torch

from projection_ref import act_ref, half_step

pytestmark = pytest.mark.gpu

# Gates whose activation is computed: gelu's to the last normal bf16 number (1.2e-38); the logistic
# function is 0 where its argument is below -87.3 (there |silu| < 1.1e-36).
RANGE = {"silu": 87.0, "gelu": 12.5, "gelu_tanh": 9.9}


def _run(gates, act, dt, tile):
    """act(g) and act'(g) as the operator computes them: with x = (1, 1, 0 ..), w_gate = (g, 0 ..) and
    w_up = (0, 1, 0 ..) every g is exact and u = 1, so h = act(g); with dh = 1 the rows of dw_up are
    du = act(g) and those of dw_gate are dg = act'(g)."""
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    from opengda_b200.ops.gemm import check_errors
    n = gates.numel()
    x = torch.zeros(1, 16, device="cuda", dtype=dt)
    x[0, :2] = 1.0
    wg, wu = torch.zeros(n, 16, device="cuda", dtype=dt), torch.zeros(n, 16, device="cuda", dtype=dt)
    wg[:, 0], wu[:, 1] = gates, 1.0
    h, saved = gated_linear_forward(x, wg, wu, act, tile=tile)
    _, dwg, dwu = gated_linear_backward(torch.ones_like(h), x, wg, wu, saved, act, need_dx=False, tile=tile)
    torch.cuda.synchronize()
    check_errors()
    return h[0].double(), dwu[:, 0].double(), dwg[:, 0].double()


def _slack(g, act):
    """The f32 evaluation's error relative to the value, in units of 2^-23.

    silu, gelu_tanh: the exponential of t, with t off by at most 4 roundings and __expf by 2 + 1.173 |t|
    ulp, then a sum, a division (2 ulp) and two products.  gelu: the exponential of t = g^2 / 2 (one
    rounding of g^2) and a polynomial in a quotient (2 ulp), 2^-21 together with its fit; three products."""
    if act == "gelu":
        t = g * g / 2
        return t / 2 + 2 + 1.173 * t + 2 + 4 + 3
    t = g.abs() if act == "silu" else 2 * math.sqrt(2 / math.pi) * g.abs() * (1 + 0.044715 * g * g)
    return 2 * t + 2 + 1.173 * t + 1 + 2 + 2


def _check_tails(dt, act, tile):
    gates = torch.cat([-torch.linspace(0.25, RANGE[act], 120), torch.linspace(0.0, RANGE[act], 40)]).to(dt).cuda()
    g = gates.double()
    a, da = act_ref(g, act)
    if act == "gelu_tanh":  # 1 + tanh cancels in 64 bits too: logistic(2 z) is the same value
        z2 = 2 * math.sqrt(2 / math.pi) * g * (1 + 0.044715 * g * g)
        s = torch.sigmoid(z2)
        a, da = g * s, s + g * 2 * s * torch.sigmoid(-z2) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    e, unit = half_step(dt), _slack(g, act) * 2.0 ** -23
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0  # half of f16's smallest subnormal; bf16's range is f32's
    h, du, dg = _run(gates, act, dt, tile)
    bound = (e + 2 * unit) * a.abs() + sub
    assert bool(((h - a).abs() <= bound).all()), (h, a)
    assert bool(((du - a).abs() <= bound).all())
    # act' is a sum of two terms of either sign, each off by its units: below 2 g^2 of the larger together
    terms = da.abs() + 2 * a.abs() * (1 + g.abs()) / g.abs().clamp_min(0.25)
    assert bool(((dg - da).abs() <= e * da.abs() + 4 * unit * terms + sub).all()), (dg, da)


@pytest.mark.parametrize("tile", [1, 2, 3])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gelu_tail(dt, tile):
    _check_tails(dt, "gelu", tile)


@pytest.mark.parametrize("tile", [1, 2, 3])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_logistic_tails(dt, act, tile):
    _check_tails(dt, act, tile)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_huge_gates(act):
    """Beyond the square root of f32's largest value: the gate itself or 0, slopes 1 or 0, no NaN."""
    gates = torch.tensor([2e19, -2e19, 1e30, -1e30, 3e38, -3e38], device="cuda").to(torch.bfloat16)
    for tile in (1, 2, 3):
        h, du, dg = _run(gates, act, torch.bfloat16, tile)
        g = gates.double()
        assert torch.equal(h, g.clamp_min(0)) and torch.equal(du, g.clamp_min(0)), (h, du)
        assert torch.equal(dg, (g > 0).double()), dg
