"""gated_linear on the GPU against its definition in 64 bits."""
import pytest
import torch

from projection_ref import check, gated_ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _make(T, H, I, dt, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + T * 31 + H * 7 + I)
    x = (torch.randn(T, H, device="cuda", generator=g) * scale).to(dt)
    wg = (torch.randn(I, H, device="cuda", generator=g) * H ** -0.5).to(dt)
    wu = (torch.randn(I, H, device="cuda", generator=g) * H ** -0.5).to(dt)
    dh = (torch.randn(T, I, device="cuda", generator=g) * 0.1).to(dt)
    return x, wg, wu, dh


def _sync():
    from opengda_b200.ops.gemm import check_errors
    torch.cuda.synchronize()
    check_errors()


@pytest.mark.parametrize("tile", [1, 2, 3])
@pytest.mark.parametrize("dt,act", [("bf16", "silu"), ("fp16", "gelu"), ("bf16", "gelu_tanh")])
@pytest.mark.parametrize("T,H,I", [(1, 8, 1), (1, 512, 256), (5, 72, 33), (127, 136, 129), (128, 64, 128), (129, 264, 300),
                                   (257, 520, 513), (700, 128, 1000)])
def test_forward(T, H, I, dt, act, tile):
    from opengda_b200.ops.ffn import gated_linear
    x, wg, wu, _ = _make(T, H, I, DT[dt])
    h = gated_linear(x, wg, wu, act=act, tile=tile)
    _sync()
    check(h, gated_ref(x, wg, wu, act)[0], "h")


@pytest.mark.parametrize("tile", [1, 2, 3])
@pytest.mark.parametrize("dt,act", [("bf16", "silu"), ("fp16", "gelu_tanh"), ("fp16", "silu"), ("bf16", "gelu")])
@pytest.mark.parametrize("T,H,I", [(1, 8, 1), (3, 520, 17), (64, 64, 64), (65, 72, 130), (300, 264, 513), (1030, 136, 200),
                                   (40, 72, 1100), (2100, 72, 40)])
def test_backward(T, H, I, dt, act, tile):
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    x, wg, wu, dh = _make(T, H, I, DT[dt], seed=1)
    h, saved = gated_linear_forward(x, wg, wu, act, tile=tile)
    got = (h, *gated_linear_backward(dh, x, wg, wu, saved, act, tile=tile))
    _sync()
    for g, r, name in zip(got, gated_ref(x, wg, wu, act, dh), ("h", "dx", "dw_gate", "dw_up")):
        check(g, r, name)


def test_chosen_tile_matches_over_shapes():
    """The launches picked by shape, at sizes on both sides of every choice."""
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    for T, H, I in ((2, 1024, 512), (160, 512, 2048), (900, 256, 1030), (2600, 128, 260), (33, 2048, 96)):
        x, wg, wu, dh = _make(T, H, I, torch.bfloat16, seed=2)
        h, saved = gated_linear_forward(x, wg, wu)
        got = (h, *gated_linear_backward(dh, x, wg, wu, saved))
        _sync()
        for g, r, name in zip(got, gated_ref(x, wg, wu, "silu", dh), ("h", "dx", "dw_gate", "dw_up")):
            check(g, r, (T, H, I, name))


@pytest.mark.parametrize("tile", [1, 2, 3])
def test_strided_inputs_and_out(tile):
    """Row pitches beyond the row, single-row views, an unaligned out; rows around out untouched."""
    from opengda_b200.ops.ffn import gated_linear
    T, H, I = 70, 136, 75
    big = _make(T + 3, H + 24, I + 9, torch.bfloat16, seed=3)
    x, wg, wu = big[0][2:T + 2, 8:H + 8], big[1][:I, 16:H + 16], big[2][5:I + 5, :H]
    out = torch.full((T + 2, I + 11), 7.0, device="cuda", dtype=torch.bfloat16)
    got = gated_linear(x, wg, wu, out=out[1:T + 1, 3:I + 3], tile=tile)
    _sync()
    assert got.data_ptr() == out[1:, 3:].data_ptr()
    check(got, gated_ref(x, wg, wu, "silu")[0])
    out[1:T + 1, 3:I + 3] = 7.0
    assert bool((out == 7.0).all())
    one = gated_linear(x[3:4], wg, wu, tile=tile)
    _sync()
    check(one, gated_ref(x[3:4], wg, wu, "silu")[0])


@pytest.mark.parametrize("tile", [1, 2, 3])
def test_backward_of_strided_gradient_and_guards(tile):
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    T, H, I = 61, 72, 37
    x, wg, wu, dh = _make(T, H, I, torch.float16, seed=4)
    wide = torch.zeros(T, I + 6, device="cuda", dtype=torch.float16)
    wide[:, 3:I + 3] = dh
    _, saved = gated_linear_forward(x, wg, wu, tile=tile)
    ref = gated_ref(x, wg, wu, "silu", dh)
    got = gated_linear_backward(wide[:, 3:I + 3], x, wg, wu, saved, tile=tile)
    _sync()
    for g, r in zip(got, ref[1:]):
        check(g, r)
    dx, a, b = gated_linear_backward(dh, x, wg, wu, saved, need_dw=False, tile=tile)
    assert a is None and b is None
    check(dx, ref[1])
    none, a, b = gated_linear_backward(dh, x, wg, wu, saved, need_dx=False, tile=tile)
    assert none is None
    _sync()
    check(a, ref[2])
    check(b, ref[3])


def test_rows_and_columns_stay_apart():
    """Infinities and NaN in one row of x, one row of a weight, reach that row and column alone."""
    from opengda_b200.ops.ffn import gated_linear
    for T, H, I in ((40, 264, 130), (300, 264, 300)):
        for tile in (1, 2, 3):
            x, wg, wu, _ = _make(T, H, I, torch.bfloat16, seed=5)
            want = gated_linear(x, wg, wu, tile=tile)
            x2, wg2 = x.clone(), wg.clone()
            x2[17, 5] = float("nan")
            x2[18, 6] = float("inf")
            wg2[9, 3] = float("nan")
            got = gated_linear(x2, wg2, wu, tile=tile)
            _sync()
            rows = [r for r in range(T) if r not in (17, 18)]
            cols = [c for c in range(I) if c != 9]
            assert torch.equal(got[rows][:, cols], want[rows][:, cols])
            assert bool(got[17].isnan().all()) and bool(got[rows][:, 9].isnan().all())


def test_extreme_gates():
    """Gates far from zero: the activations go to 0 or the gate itself, without NaN."""
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    for act in ("silu", "gelu", "gelu_tanh"):
        x = torch.zeros(4, 16, device="cuda", dtype=torch.bfloat16)
        x[:, 0] = torch.tensor([3e4, -3e4, 200.0, -200.0], device="cuda")
        wg = torch.zeros(8, 16, device="cuda", dtype=torch.bfloat16)
        wg[:, 0] = 1.0
        wu = torch.zeros_like(wg)
        wu[:, 0] = 2.0 ** -6
        h, saved = gated_linear_forward(x, wg, wu, act)
        dh = torch.ones_like(h)
        dx, dwg, dwu = gated_linear_backward(dh, x, wg, wu, saved, act)
        _sync()
        g, u = x[:, :1].double(), x[:, :1].double() * 2.0 ** -6
        want = torch.where(g > 0, g * u, torch.zeros_like(g)).expand(4, 8)
        assert torch.allclose(h.double(), want, rtol=2.0 ** -8, atol=0)
        assert not dx.isnan().any() and not dwg.isnan().any() and not dwu.isnan().any()
        # dx: (u + g/64) summed over the 8 columns where the gate is open, 0 where it is shut;
        # its first column only
        open_ = torch.where(g > 0, 8 * (u + g * 2.0 ** -6), torch.zeros_like(g))[:, 0]
        assert torch.allclose(dx[:, 0].double(), open_, rtol=2.0 ** -6, atol=0)


def test_empty_batch():
    from opengda_b200.ops.ffn import gated_linear
    x = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(40, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
    h = gated_linear(x, w, w)
    assert h.shape == (0, 40)
    dx, dw = torch.autograd.grad(h, (x, w), torch.zeros_like(h))
    _sync()
    assert dx.shape == (0, 64) and dw.shape == (40, 64) and not dw.any()


def test_autograd():
    from opengda_b200.ops.ffn import gated_linear
    T, H, I = 50, 128, 90
    x, wg, wu, dh = _make(T, H, I, torch.bfloat16, seed=6)
    ref = gated_ref(x, wg, wu, "gelu", dh)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    h = gated_linear(*leaves, act="gelu")
    h.backward(dh)
    _sync()
    for t, r in zip((h, *(t.grad for t in leaves)), ref):
        check(t.detach(), r)
    # a subset of the inputs; a broadcast gradient
    leaves = [x.clone(), wg.clone().requires_grad_(True), wu.clone()]
    g, = torch.autograd.grad(gated_linear(*leaves, act="gelu").sum(), (leaves[1],))
    _sync()
    check(g, gated_ref(x, wg, wu, "gelu", torch.ones_like(dh))[2])
    # the same tensor for both weights: its gradient is the sum of both
    w = wg.clone().requires_grad_(True)
    both = torch.autograd.grad(gated_linear(x, w, w), (w,), dh)[0]
    r = gated_ref(x, wg, wg, "silu", dh)
    half = 2.0 ** -8
    check(both, (r[2][0] + r[3][0], r[2][1] + r[3][1] + half * (r[2][0].abs() + r[3][0].abs() + r[2][1] + r[3][1])))
    # changed after the forward pass: refused by its version
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    h = gated_linear(*leaves)
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.backward(dh)
    # no second derivative
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    g, = torch.autograd.grad(gated_linear(*leaves), (leaves[0],), dh, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        g.float().sum().backward()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradient_against_differences(act):
    """d(sum h * dh) along a direction in x and the weights, by the operator's own forward pass.

    The step e moves every g and u by about e; the difference quotient of the 64-bit definition is
    off by O(e^2).  The 16-bit gradients are off by the bounds of gated_ref, summed along the
    direction."""
    T, H, I = 24, 64, 40
    x, wg, wu, dh = _make(T, H, I, torch.float16, seed=7)
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    _, saved = gated_linear_forward(x, wg, wu, act)
    grads = gated_linear_backward(dh, x, wg, wu, saved, act)
    _sync()
    g = torch.Generator(device="cuda").manual_seed(8)
    dirs = [torch.randn(t.shape, device="cuda", generator=g).double() * t.abs().double().mean() for t in (x, wg, wu)]

    def value(s):
        from projection_ref import act_ref
        X, G, U = (t.double() + s * d for t, d in zip((x, wg, wu), dirs))
        return (act_ref(X @ G.t(), act)[0] * (X @ U.t()) * dh.double()).sum().item()

    e = 1e-4
    quotient = (value(e) - value(-e)) / (2 * e)
    third = abs((value(2 * e) - 2 * value(e) + 2 * value(-e) - value(-2 * e)) / (2 * e ** 3)) * e * e / 6
    along = sum((a.double() * d).sum().item() for a, d in zip(grads, dirs))
    slack = sum((r[1] * d.abs()).sum().item() for r, d in zip(gated_ref(x, wg, wu, act, dh)[1:], dirs))
    assert abs(along - quotient) <= slack + 2 * third + 1e-9 * abs(quotient)


def test_graph_capture_and_replay():
    """Forward and backward captured together, replayed with new contents; two graphs at once."""
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    shapes = ((5, 264, 130), (700, 264, 300))
    made = []
    for T, H, I in shapes:
        x, wg, wu, dh = _make(T, H, I, torch.bfloat16, seed=9)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            gated_linear_forward(x, wg, wu)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h, saved = gated_linear_forward(x, wg, wu)
            out = (h, *gated_linear_backward(dh, x, wg, wu, saved))
        made.append((g, (x, wg, wu, dh), out))
    for rep in range(3):
        for g, ins, _ in made:
            for t, n in zip(ins, _make(ins[0].shape[0], ins[0].shape[1], ins[1].shape[0], torch.bfloat16, seed=10 + rep)):
                t.copy_(n)
            g.replay()
        _sync()
        for _, ins, out in made:
            for t, r in zip(out, gated_ref(ins[0], ins[1], ins[2], "silu", ins[3])):
                check(t, r)


def test_autograd_step_captured():
    """A whole step (forward and autograd) captured in a graph, as a training loop does it."""
    from opengda_b200.ops.ffn import gated_linear
    T, H, I = 130, 72, 96
    x, wg, wu, dh = _make(T, H, I, torch.bfloat16, seed=13)
    wg.requires_grad_(True)
    wu.requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(gated_linear(x, wg, wu), (wg, wu), dh)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grads = torch.autograd.grad(gated_linear(x, wg, wu), (wg, wu), dh)
    x.copy_(_make(T, H, I, torch.bfloat16, seed=14)[0])
    g.replay()
    _sync()
    ref = gated_ref(x, wg.detach(), wu.detach(), "silu", dh)
    check(grads[0], ref[2])
    check(grads[1], ref[3])


def test_capture_beside_a_live_graph_is_refused():
    """An autograd graph of the same parameter that is alive outside the capture: refused with a
    reason, and everything works again once it is gone."""
    from opengda_b200.ops.ffn import gated_linear
    x, w, _, dh = _make(8, 64, 64, torch.bfloat16, seed=15)
    w.requires_grad_(True)
    live = gated_linear(x, w, w)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gated_linear(x, w, w)
    live.backward(dh)
    _sync()
    r = gated_ref(x, w.detach(), w.detach(), "silu", dh)
    check(w.grad, (r[2][0] + r[3][0], 1.01 * (r[2][1] + r[3][1]) + 2.0 ** -8 * (r[2][0] + r[3][0]).abs()))
    del live
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grad, = torch.autograd.grad(gated_linear(x, w, w), (w,), dh)
    g.replay()
    _sync()
    assert torch.equal(grad, w.grad)


def test_side_streams_at_once():
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    jobs = []
    for k, (T, H, I) in enumerate(((3, 512, 260), (400, 264, 500), (90, 1024, 70), (1500, 136, 64))):
        jobs.append((torch.cuda.Stream(), _make(T, H, I, torch.bfloat16, seed=20 + k)))
    torch.cuda.synchronize()
    got = []
    for s, (x, wg, wu, dh) in jobs:
        with torch.cuda.stream(s):
            h, saved = gated_linear_forward(x, wg, wu)
            got.append((h, *gated_linear_backward(dh, x, wg, wu, saved)))
    _sync()
    for out, (_, (x, wg, wu, dh)) in zip(got, jobs):
        for t, r in zip(out, gated_ref(x, wg, wu, "silu", dh)):
            check(t, r)


def test_results_repeat():
    """Every sum has a fixed order: the same inputs give the same bits."""
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    for T, H, I in ((7, 2048, 300), (300, 264, 513), (2100, 72, 40)):
        x, wg, wu, dh = _make(T, H, I, torch.bfloat16, seed=30)
        runs = []
        for _ in range(3):
            h, saved = gated_linear_forward(x, wg, wu)
            runs.append((h, *gated_linear_backward(dh, x, wg, wu, saved)))
        _sync()
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_long_rows():
    """Offsets beyond 2^31 elements in h, the saved planes and dg."""
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    T, H, I = 65600, 8, 32800  # 2.15e9 elements
    x, wg, wu, _ = _make(T, H, I, torch.bfloat16, seed=31)
    h, saved = gated_linear_forward(x, wg, wu)
    rows = torch.tensor([0, 31, 32767, 65500, T - 1], device="cuda")
    dh = torch.zeros_like(h)
    dh[rows] = 0.125
    dx, dwg, dwu = gated_linear_backward(dh, x, wg, wu, saved)
    _sync()
    check(h[rows], gated_ref(x[rows], wg, wu, "silu")[0])
    ref = gated_ref(x[rows], wg, wu, "silu", dh[rows])
    check(dx[rows], ref[1])
    check(dwg, ref[2])
    check(dwu, ref[3])
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert not dx[rest].any()


def test_refusals():
    from opengda_b200.ops.ffn import gated_linear, gated_linear_backward, gated_linear_forward
    x, wg, wu, dh = _make(16, 64, 24, torch.bfloat16)
    bad = [
        ((x.float(), wg.float(), wu.float()), "bfloat16 or float16"),
        ((x, wg.half(), wu), "dtype"),
        ((x, wg.cpu(), wu), "CUDA"),
        ((x, wg, wu[:20]), "share"),
        ((x[:, :56], wg, wu), "share"),
        ((x[:, :60].contiguous(), wg[:, :60].contiguous(), wu[:, :60].contiguous()), "multiple of 8|16-byte"),
        ((x.t().contiguous().t(), wg, wu), "row-major"),
        ((x[:1].expand(16, 64), wg, wu), "overlap"),
        ((x.flatten(), wg, wu), "2-D"),
        ((torch.empty(16 * 64 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(16, 64), wg, wu), "16-byte"),
    ]
    for args, what in bad:
        with pytest.raises(RuntimeError, match=what):
            gated_linear(*args)
    for out in (torch.empty(16, 25, device="cuda", dtype=torch.bfloat16), torch.empty(16, 24, device="cuda"),
                torch.empty(24, 16, device="cuda", dtype=torch.bfloat16).t()):
        with pytest.raises(RuntimeError):
            gated_linear(x, wg, wu, out=out)
    with pytest.raises(RuntimeError, match="tile"):
        gated_linear(x, wg, wu, tile=4)
    with pytest.raises(RuntimeError, match="overlap"):
        gated_linear(x, wg, wu, out=x[:, :24])
    side = torch.empty(16, 88, device="cuda", dtype=torch.bfloat16)  # x and out side by side in one buffer
    side[:, :64] = x
    check(gated_linear(side[:, :64], wg, wu, out=side[:, 64:]), gated_ref(x, wg, wu, "silu")[0])
    with pytest.raises(RuntimeError, match="overlap"):
        gated_linear(side[:, :64], wg, wu, out=side[:, 56:80])
    _, saved = gated_linear_forward(x, wg, wu)
    with pytest.raises(RuntimeError, match="saved"):
        gated_linear_backward(dh, x, wg, wu, saved[:-1])
    with pytest.raises(RuntimeError, match="share"):
        gated_linear_backward(dh[:8], x, wg, wu, saved)
    with pytest.raises(ValueError, match="without gradients"):
        gated_linear(x.clone().requires_grad_(True), wg, wu, tile=1)
    _sync()
