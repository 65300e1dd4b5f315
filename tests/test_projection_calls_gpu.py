"""Calls of the projection operators around a training step: captures, gradients' storage, size limits."""
import pytest
import torch

from projection_ref import check, gated_ref

pytestmark = pytest.mark.gpu


def _make(T, H, I, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).to(dt)  # noqa: E731
    return r(T, H), r(I, H, std=H ** -0.5), r(I, H, std=H ** -0.5), r(T, I, std=0.1)


def _sync():
    from opengda_b200.ops.gemm import check_errors
    torch.cuda.synchronize()
    check_errors()


def test_capture_beside_a_live_graph_of_the_weights_source():
    """The weights are 16-bit copies of 32-bit parameters, and an eager graph of the parameters is
    alive: the captured backward pass would reach their accumulation on the other stream."""
    from opengda_b200.ops.ffn import gated_linear
    x, w, _, dh = _make(8, 64, 64, torch.bfloat16, seed=1)
    master = w.float().requires_grad_(True)
    live = master * 2.0
    torch.cuda.synchronize()
    refused = False
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        low = master.to(torch.bfloat16)
        try:
            gated_linear(x, low, low)
        except RuntimeError as e:
            refused = "still alive" in str(e)
    assert refused
    del live, low
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        low = master.to(torch.bfloat16)
        grad, = torch.autograd.grad(gated_linear(x, low, low), (master,), dh)
    g.replay()
    _sync()
    r = gated_ref(x, w, w, "silu", dh)
    check(grad, (r[2][0] + r[3][0], 1.01 * (r[2][1] + r[3][1]) + 2.0 ** -8 * (r[2][0] + r[3][0]).abs()))
