"""lora_linear on the GPU against its definition in 64 bits."""
import pytest
import torch

from projection_ref import check, lora_ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _make(T, K, N, L, r, dt, idx="random", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + T * 31 + K * 7 + N + L * 13 + r)
    rnd = lambda *s, std: (torch.randn(*s, device="cuda", generator=g) * std).to(dt)  # noqa: E731
    x, w = rnd(T, K, std=1.0), rnd(N, K, std=K ** -0.5)
    a, b = rnd(L, r, K, std=K ** -0.5), rnd(L, N, r, std=r ** -0.5)
    if idx == "random":
        ids = torch.randint(-1, L, (T,), device="cuda", generator=g)
    elif idx == "none":
        ids = torch.full((T,), -1, device="cuda")
    elif idx == "distinct":
        ids = torch.arange(T, device="cuda") % L
    else:  # runs
        ids = (torch.arange(T, device="cuda") * 7 // max(T, 1)) % (L + 1) - 1
    scale = torch.rand(L, device="cuda", generator=g) * 2 - 0.5
    return x, w, a, b, ids.to(torch.int32), scale


def _sync():
    from opengda_b200.ops.gemm import check_errors
    torch.cuda.synchronize()
    check_errors()


@pytest.mark.parametrize("tile", [1, 2, 3])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N,L,r,idx", [
    (1, 8, 1, 1, 8, "distinct"), (1, 520, 256, 3, 16, "distinct"), (7, 136, 33, 4, 24, "random"),
    (64, 256, 512, 64, 16, "distinct"), (128, 72, 130, 200, 8, "distinct"), (130, 264, 300, 5, 64, "random"),
    (200, 512, 257, 2, 128, "runs"), (300, 128, 1024, 300, 16, "distinct"), (1000, 264, 515, 9, 72, "runs"),
    (600, 64, 64, 1, 32, "none"), (513, 136, 260, 40, 16, "random")])
def test_lora(T, K, N, L, r, idx, dt, tile):
    from opengda_b200.ops.lora import lora_linear
    x, w, a, b, ids, scale = _make(T, K, N, L, r, DT[dt], idx)
    y = lora_linear(x, w, a, b, ids, scale, tile=tile)
    _sync()
    check(y, lora_ref(x, w, a, b, ids, scale), "y")


@pytest.mark.parametrize("tile", [1, 2, 3])
def test_rows_apart(tile):
    """A row without an adapter, or of another one, sees nothing of an adapter's NaN or infinity;
    the same row alone gives the same bits."""
    from opengda_b200.ops.lora import lora_linear
    for T in (60, 300):
        x, w, a, b, ids, scale = _make(T, 264, 130, 6, 24, torch.bfloat16, seed=3)
        want = lora_linear(x, w, a, b, ids, scale, tile=tile)
        a2, b2 = a.clone(), b.clone()
        a2[2, 3, 5] = float("nan")
        b2[4] = float("inf")
        x2 = x.clone()
        x2[11] = float("nan")
        got = lora_linear(x2, w, a2, b2, ids, scale, tile=tile)
        _sync()
        keep = (ids != 2) & (ids != 4)
        keep[11] = False
        assert torch.equal(got[keep], want[keep])
        assert bool(got[ids == 2].isnan().all())


@pytest.mark.parametrize("tile", [1, 2, 3])
def test_no_adapter_is_the_plain_projection(tile):
    from opengda_b200.ops.lora import lora_linear
    x, w, a, b, ids, scale = _make(140, 512, 260, 3, 16, torch.bfloat16, idx="none", seed=4)
    a.fill_(float("nan"))
    got = lora_linear(x, w, a, b, ids, scale, tile=tile)
    none = lora_linear(x, w, a[:1].zero_().contiguous(), b[:1].zero_().contiguous(), torch.zeros_like(ids), tile=tile)
    _sync()
    assert torch.equal(got, none)


@pytest.mark.parametrize("tile", [1, 2, 3])
def test_strides_and_out(tile):
    from opengda_b200.ops.lora import lora_linear
    T, K, N = 90, 136, 75
    x, w, a, b, ids, scale = _make(T + 3, K + 24, N + 9, 4, 16, torch.float16, seed=5)
    x, w = x[1:T + 1, 8:K + 8], w[2:N + 2, 16:K + 16]
    a, b, ids = a[:, :, :K].contiguous(), b[:, :N].contiguous(), ids[:T].contiguous()
    out = torch.full((T + 2, N + 11), 7.0, device="cuda", dtype=torch.float16)
    got = lora_linear(x, w, a, b, ids, scale, out=out[1:T + 1, 3:N + 3], tile=tile)
    _sync()
    check(got, lora_ref(x, w, a, b, ids, scale))
    out[1:T + 1, 3:N + 3] = 7.0
    assert bool((out == 7.0).all())
    one = lora_linear(x[4:5], w, a, b, ids[4:5].contiguous(), tile=tile)
    _sync()
    check(one, lora_ref(x[4:5], w, a, b, ids[4:5]))


def test_chosen_tile_over_shapes():
    from opengda_b200.ops.lora import lora_linear
    for T, K, N, L, r, idx in ((1, 2048, 512, 2000, 16, "distinct"), (3, 64, 4096, 8192, 8, "random"), (180, 512, 700, 7, 32, "runs"),
                               (1100, 256, 640, 30, 48, "random"), (5000, 72, 300, 3, 64, "runs"), (256, 136, 260, 256, 128, "distinct")):
        x, w, a, b, ids, scale = _make(T, K, N, L, r, torch.bfloat16, idx, seed=6)
        y = lora_linear(x, w, a, b, ids, scale)
        _sync()
        check(y, lora_ref(x, w, a, b, ids, scale), (T, K, N, L, r, idx))


def test_empty_batch():
    from opengda_b200.ops.lora import lora_linear
    x, w, a, b, ids, scale = _make(8, 64, 40, 2, 8, torch.bfloat16)
    assert lora_linear(x[:0], w, a, b, ids[:0], scale).shape == (0, 40)


@pytest.mark.parametrize("tile", [1, 2, 3])
def test_indexes_out_of_range_are_reported(tile):
    from opengda_b200.ops.gemm import check_errors
    from opengda_b200.ops.lora import lora_linear
    x, w, a, b, ids, scale = _make(300, 136, 70, 5, 16, torch.bfloat16, idx="runs", seed=7)
    good = ids.clone()
    ids[10], ids[200], good[10], good[200] = 5, -2, -1, -1
    y = lora_linear(x, w, a, b, ids, scale, tile=tile)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="ERANGE"):
        check_errors()
    check_errors()
    check(y, lora_ref(x, w, a, b, good, scale))


def test_graph_capture_and_replay():
    from opengda_b200.ops.lora import lora_linear
    made = []
    for T in (9, 400):
        ins = _make(T, 264, 300, 6, 16, torch.bfloat16, seed=8)
        lora_linear(*ins)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = lora_linear(*ins)
        made.append((g, ins, y))
    for rep in range(3):
        for g, ins, _ in made:
            for t, n in zip(ins, _make(ins[0].shape[0], 264, 300, 6, 16, torch.bfloat16, seed=9 + rep)):
                t.copy_(n)
            g.replay()
        _sync()
        for _, ins, y in made:
            check(y, lora_ref(*ins))


def test_first_call_inside_a_capture():
    """A process whose first call of the library is captured."""
    import os
    import subprocess
    import sys
    code = """
import sys; sys.path[:0] = [%r, %r]
import torch
from test_lora_gpu import _make, _sync
from projection_ref import check, lora_ref
from opengda_b200.ops.lora import lora_linear
for T in (9, 400):
    ins = _make(T, 264, 300, 6, 16, torch.bfloat16, seed=8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lora_linear(*ins)
    g.replay()
    _sync()
    check(y, lora_ref(*ins))
print("captured")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", code % (os.path.dirname(here), here)], capture_output=True, text=True, timeout=180)
    assert "captured" in r.stdout, r.stdout + r.stderr


def test_side_streams_at_once():
    from opengda_b200.ops.lora import lora_linear
    jobs = [(torch.cuda.Stream(), _make(T, 512, 520, 8, 16, torch.bfloat16, seed=40 + T)) for T in (1, 64, 300, 2000)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, ins in jobs:
            with torch.cuda.stream(s):
                got.append((lora_linear(*ins), ins))
    _sync()
    for y, ins in got:
        check(y, lora_ref(*ins))


def test_results_repeat():
    from opengda_b200.ops.lora import lora_linear
    for T in (40, 700):
        ins = _make(T, 1032, 300, 12, 32, torch.bfloat16, seed=50)
        runs = [lora_linear(*ins) for _ in range(3)]
        _sync()
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_block_of_both_operators():
    """A feed-forward block as a server runs it: gated_linear, then the down projection with each
    request's adapter, in one captured graph; against the two definitions in sequence."""
    from opengda_b200.ops.ffn import gated_linear
    from opengda_b200.ops.lora import lora_linear
    from projection_ref import gated_ref
    for T in (1, 33, 600):
        H, I = 264, 392
        x, wd, a, b, ids, scale = _make(T, H, I, 5, 16, torch.bfloat16, seed=60)
        wg, wu = wd, wd.flip(0).contiguous()
        down = _make(T, I, H, 5, 16, torch.bfloat16, seed=61)
        lora_linear(gated_linear(x, wg, wu), *down[1:])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h = gated_linear(x, wg, wu)
            y = lora_linear(h, *down[1:])
        g.replay()
        _sync()
        check(h, gated_ref(x, wg, wu, "silu")[0])
        check(y, lora_ref(h, *down[1:]))


def test_long_outputs():
    """Offsets beyond 2^31 elements in y."""
    from opengda_b200.ops.lora import lora_linear
    T, K, N = 65600, 8, 32800
    x, w, a, b, ids, scale = _make(T, K, N, 3, 8, torch.bfloat16, idx="runs", seed=70)
    y = lora_linear(x, w, a, b, ids, scale)
    rows = torch.tensor([0, 255, 32767, 65500, T - 1], device="cuda")
    _sync()
    check(y[rows], lora_ref(x[rows], w, a, b, ids[rows], scale))


def test_refusals():
    from opengda_b200.ops.lora import lora_linear
    x, w, a, b, ids, scale = _make(16, 64, 24, 3, 16, torch.bfloat16)
    bad = [
        ((x.float(), w, a, b, ids), "bfloat16 or float16"),
        ((x, w.half(), a, b, ids), "dtype"),
        ((x, w, a[:, :, :56], b, ids), "contiguous|share"),
        ((x, w, a, b[:, :20].contiguous(), ids), "share"),
        ((x, w, a, b, ids.long()), "int32"),
        ((x, w, a, b, ids[:8]), "adapter"),
        ((x, w, a, b, torch.stack([ids, ids], 1)[:, 0]), "contiguous"),
        ((x, w, a, b, ids.cpu()), "adapter"),
        ((x, w, a, b, ids, scale.double()), "scale"),
        ((x, w, a, b, ids, scale[:2]), "scale"),
        ((x, w, a[:, :12].contiguous(), b[:, :, :12].contiguous(), ids), "multiples of 8"),
        ((x, w, a.repeat(1, 9, 1), b.repeat(1, 1, 9), ids), "128"),
        ((x.t().contiguous().t(), w, a, b, ids), "row-major"),
        ((x[:, :60].contiguous(), w[:, :60].contiguous(), a[:, :, :60].contiguous(), b, ids), "multiples of 8|16-byte"),
    ]
    for args, what in bad:
        with pytest.raises(RuntimeError, match=what):
            lora_linear(*args)
    with pytest.raises(RuntimeError, match="overlap"):
        lora_linear(x, w, a, b, ids, out=x[:, :24])
    with pytest.raises(RuntimeError, match="tile"):
        lora_linear(x, w, a, b, ids, tile=4)
    _sync()
