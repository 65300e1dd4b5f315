"""Every kernel path of the projections in the ways that a program runs it: several tiles and ring turns per
CTA, captured and replayed, several streams at once, repeated bits; and that each is picked by shape."""
import pytest
import torch

from projection_ref import check, gated_ref, lora_ref

pytestmark = pytest.mark.gpu
TILES = [1, 2, 3]


def _gated(T, H, I, dt=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).to(dt)  # noqa: E731
    return r(T, H), r(I, H, std=H ** -0.5), r(I, H, std=H ** -0.5), r(T, I, std=0.1)


def _lora(T, K, N, L, r, dt=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std).to(dt)  # noqa: E731
    ids = torch.randint(-1, L, (T,), device="cuda", generator=g).to(torch.int32)
    return (m(T, K), m(N, K, std=K ** -0.5), m(L, r, K, std=K ** -0.5), m(L, N, r, std=r ** -0.5), ids,
            torch.rand(L, device="cuda", generator=g) + 0.5)


def _step(ins, act, tile):
    from opengda_b200.ops.ffn import gated_linear_backward, gated_linear_forward
    x, wg, wu, dh = ins
    h, saved = gated_linear_forward(x, wg, wu, act, tile=tile)
    return (h, *gated_linear_backward(dh, x, wg, wu, saved, act, tile=tile))


def _check_step(out, ins, act, what=""):
    for t, r, name in zip(out, gated_ref(*ins[:3], act, ins[3]), ("h", "dx", "dw_gate", "dw_up")):
        check(t, r, (what, name))


def _sync():
    from opengda_b200.ops.gemm import check_errors
    torch.cuda.synchronize()
    check_errors()


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("act,dt", [("silu", torch.bfloat16), ("gelu", torch.float16)])
@pytest.mark.parametrize("T,H,I", [(2600, 520, 2100), (2600, 1104, 2100), (1000, 2056, 5000)])
def test_gated_with_several_tiles_per_pair(T, H, I, act, dt, tile):
    """More tiles than CTA pairs and more k-blocks than ring stages, in the forward and the three products."""
    from opengda_b200.ops.ffn import gated_linear
    ins = _gated(T, H, I, dt)
    out = _step(ins, act, tile)
    plain = gated_linear(*ins[:3], act=act, tile=tile)
    _sync()
    _check_step(out, ins, act, (T, H, I))
    assert torch.equal(plain, out[0])


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("T,K,N,L,r,dt", [(2600, 520, 4200, 9, 24, torch.bfloat16), (2600, 520, 4200, 300, 64, torch.float16),
                                          (1500, 1032, 8200, 40, 16, torch.bfloat16), (5000, 264, 1029, 70, 128, torch.bfloat16)])
def test_lora_with_several_tiles_per_pair(T, K, N, L, r, dt, tile):
    from opengda_b200.ops.lora import lora_linear
    ins = _lora(T, K, N, L, r, dt)
    y = lora_linear(*ins, tile=tile)
    _sync()
    check(y, lora_ref(*ins))


@pytest.mark.parametrize("tile", TILES)
def test_captured_and_replayed(tile):
    """Two graphs of each operator, replayed in turn with new contents."""
    from opengda_b200.ops.lora import lora_linear
    gated_sizes, lora_sizes = ((300, 264, 300), (2600, 136, 2100)), ((300, 264, 300, 6, 16), (2600, 136, 4200, 9, 24))
    made = []
    for k, (gs, ls) in enumerate(zip(gated_sizes, lora_sizes)):
        gi, li = _gated(*gs), _lora(*ls)
        _step(gi, "silu", tile)
        lora_linear(*li, tile=tile)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, y = _step(gi, "silu", tile), lora_linear(*li, tile=tile)
        made.append((graph, gs, ls, gi, li, out, y))
    for rep in range(3):
        for graph, gs, ls, gi, li, _, _ in made:
            for t, n in zip((*gi, *li), (*_gated(*gs, seed=1 + rep), *_lora(*ls, seed=1 + rep))):
                t.copy_(n)
            graph.replay()
        _sync()
        for _, _, _, gi, li, out, y in made:
            _check_step(out, gi, "silu", rep)
            check(y, lora_ref(*li))


@pytest.mark.parametrize("tile", TILES)
def test_several_streams_at_once(tile):
    from opengda_b200.ops.lora import lora_linear
    jobs = [(torch.cuda.Stream(), _gated(T, H, I, seed=T), _lora(T, H, I, 7, 16, seed=T))
            for T, H, I in ((5, 1032, 300), (300, 520, 1030), (1300, 264, 2100), (2600, 136, 520))]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, gi, li in jobs:
            with torch.cuda.stream(s):
                got.append((_step(gi, "silu", tile), gi, lora_linear(*li, tile=tile), li))
    _sync()
    for out, gi, y, li in got:
        _check_step(out, gi, "silu")
        check(y, lora_ref(*li))


@pytest.mark.parametrize("tile", TILES)
def test_same_bits_again(tile):
    from opengda_b200.ops.lora import lora_linear
    gi, li = _gated(2600, 520, 2100), _lora(2600, 520, 4200, 9, 24)
    runs = [(*_step(gi, "silu", tile), lora_linear(*li, tile=tile)) for _ in range(4)]
    _sync()
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_each_path_is_picked_by_shape():
    """Sizes for which the choice by shape takes each of the three launches, and their results."""
    from opengda_b200 import native
    from opengda_b200.ops.lora import lora_linear
    hit = set()
    for T, H, I in ((1, 1024, 512), (700, 1024, 2048), (1500, 512, 1030), (2048, 1024, 2048), (4096, 512, 2048)):
        tile = native().gated_linear_tile(T, H, I)
        hit.add(("gated", tile))
        ins = _gated(T, H, I)
        auto, forced = _step(ins, "silu", 0), _step(ins, "silu", tile)
        _sync()
        assert torch.equal(auto[0], forced[0])
        _check_step(auto, ins, "silu", (T, H, I))
    for T, K, N, L, r in ((1, 1024, 512, 3, 16), (1000, 1024, 2048, 5, 16), (2600, 520, 2100, 9, 24), (2048, 1024, 4096, 9, 24),
                          (4096, 1024, 4096, 40, 16)):
        tile = native().lora_linear_tile(T, K, N, r)
        hit.add(("lora", tile))
        ins = _lora(T, K, N, L, r)
        y, forced = lora_linear(*ins), lora_linear(*ins, tile=tile)
        _sync()
        assert torch.equal(y, forced)
        check(y, lora_ref(*ins))
    assert hit == {(op, t) for op in ("gated", "lora") for t in TILES}, hit
