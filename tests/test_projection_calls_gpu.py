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


def test_weight_gradients_do_not_share_memory():
    """A user may free or overwrite one weight's gradient without the other's."""
    from opengda_b200.ops.ffn import gated_linear, gated_linear_backward, gated_linear_forward
    for T in (0, 3, 300):
        x, wg, wu, dh = _make(T, 64, 40, torch.bfloat16)
        _, saved = gated_linear_forward(x, wg, wu)
        _, a, b = gated_linear_backward(dh, x, wg, wu, saved)
        assert a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr()
        assert a.untyped_storage().nbytes() == b.untyped_storage().nbytes() == 40 * 64 * 2
        version = b._version
        a.mul_(2)
        assert b._version == version
        ws = [w.clone().requires_grad_(True) for w in (wg, wu)]
        gated_linear(x, *ws).backward(dh)
        _sync()
        assert ws[0].grad.untyped_storage().data_ptr() != ws[1].grad.untyped_storage().data_ptr()
        if T:
            ref = gated_ref(x, wg, wu, "silu", dh)
            check(ws[0].grad, ref[2])
            check(ws[1].grad, ref[3])


def test_a_refused_size_leaves_no_error_behind():
    """More row blocks than a grid of the split clusters takes: refused, and the next call works."""
    from opengda_b200.ops.ffn import gated_linear
    x = torch.zeros(65536 * 128 + 1, 8, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(1, 8, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="rows"):
        gated_linear(x, w, w, tile=1)
    assert not gated_linear(x, w, w).any()
    _sync()


def test_more_rows_than_the_split_clusters_take():
    """By shape such a call runs on the pairs; the backward products too, where a weight has that many rows."""
    from opengda_b200.ops.ffn import gated_linear, gated_linear_backward, gated_linear_forward
    x = torch.zeros(65536 * 128 + 1, 8, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(1, 8, device="cuda", dtype=torch.bfloat16)
    x[-1, :2] = 1.0
    h = gated_linear(x, w, w)
    _sync()
    check(h[-1:], gated_ref(x[-1:], w, w, "silu")[0])
    assert not h[:-1].any()
    del h
    rows, H = 32768 * 128 + 1, 8
    x, wg, wu, dh = _make(2, H, rows, torch.bfloat16, seed=2)
    h, saved = gated_linear_forward(x, wg, wu)
    with pytest.raises(RuntimeError, match="rows"):
        gated_linear_backward(dh, x, wg, wu, saved, tile=1)
    got = (h, *gated_linear_backward(dh, x, wg, wu, saved))
    _sync()
    for t, r in zip(got, gated_ref(x, wg, wu, "silu", dh)):
        check(t, r)


def test_capture_beside_a_live_graph_of_another_side_stream():
    """A warm-up on a stream of its own whose result is still held: the engine joins that stream."""
    from opengda_b200.ops.ffn import gated_linear
    x, wg, wu, dh = _make(130, 72, 96, torch.bfloat16, seed=3)
    wg.requires_grad_(True)
    wu.requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        live = gated_linear(x, wg, wu)
        torch.autograd.grad(live, (wg, wu), dh, retain_graph=True)
    torch.cuda.synchronize()
    g, acc = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grads = torch.autograd.grad(gated_linear(x, wg, wu), (wg, wu), dh)
    wg.grad, wu.grad = torch.zeros_like(wg), torch.zeros_like(wu)
    with torch.cuda.graph(acc):
        wg.grad.zero_()
        wu.grad.zero_()
        gated_linear(x, wg, wu).backward(dh)
    x.copy_(_make(130, 72, 96, torch.bfloat16, seed=4)[0])
    g.replay()
    acc.replay()
    _sync()
    ref = gated_ref(x, wg.detach(), wu.detach(), "silu", dh)
    for got in (grads, (wg.grad, wu.grad)):
        check(got[0], ref[2])
        check(got[1], ref[3])
    assert live.requires_grad


def test_make_graphed_callables():
    """torch's own way to capture a module's forward and backward pass."""
    from opengda_b200.ops.ffn import gated_linear

    class Block(torch.nn.Module):
        def __init__(self, wg, wu):
            super().__init__()
            self.wg, self.wu = torch.nn.Parameter(wg), torch.nn.Parameter(wu)

        def forward(self, x):
            return gated_linear(x, self.wg, self.wu, act="gelu")

    x, wg, wu, dh = _make(70, 264, 130, torch.bfloat16, seed=5)
    block = Block(wg, wu)
    graphed = torch.cuda.make_graphed_callables(block, (x.clone().requires_grad_(True),))
    for seed in (6, 7):
        x, _, _, dh = _make(70, 264, 130, torch.bfloat16, seed=seed)
        x.requires_grad_(True)
        h = graphed(x)
        got = (h.detach().clone(), *(t.clone() for t in torch.autograd.grad(h, (x, block.wg, block.wu), dh)))
        _sync()
        for t, r in zip(got, gated_ref(x.detach(), wg, wu, "gelu", dh)):
            check(t, r)
