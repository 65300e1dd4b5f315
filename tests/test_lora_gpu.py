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
