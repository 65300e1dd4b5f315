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
