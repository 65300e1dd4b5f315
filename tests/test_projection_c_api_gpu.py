"""The C entry points of the projections (gicc/projections.h), called with the buffers that they ask for."""
import ctypes
import os

import pytest
import torch

from projection_ref import check, gated_ref, lora_ref

pytestmark = pytest.mark.gpu
P, LL, I = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int
GUARD = 4096  # bytes behind a buffer that have to stay as they are


@pytest.fixture(scope="module")
def lib():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = ctypes.CDLL(os.path.join(root, "opengda_b200", "lib", "libgicc.so"))
    for f, n in (("gicc_gated_saved_floats", 2), ("gicc_gated_grad_bytes", 2), ("gicc_lora_work_bytes", 3)):
        getattr(lib, f).argtypes, getattr(lib, f).restype = [I] * n, ctypes.c_size_t
    lib.gicc_gated_linear.argtypes = [P, P, P, P, I, I, I, LL, LL, LL, LL, I, I, P, P]
    lib.gicc_gated_linear_backward.argtypes = [P] * 9 + [I] * 3 + [LL] * 6 + [I, I, P]
    lib.gicc_lora_linear.argtypes = [P] * 8 + [I] * 5 + [LL] * 3 + [I, P]
    return lib


def _buffer(nbytes):
    return torch.full((nbytes + GUARD,), 0x5A, dtype=torch.uint8, device="cuda")


def _sync():
    from opengda_b200.ops.gemm import check_errors
    torch.cuda.synchronize()
    check_errors()


@pytest.mark.parametrize("T,H,n", [(1, 8, 1), (5, 72, 33), (61, 72, 37), (300, 264, 513), (1030, 136, 200)])
def test_gated(lib, T, H, n):
    g = torch.Generator(device="cuda").manual_seed(T + H + n)
    x, wg, wu, dh = ((torch.randn(*s, device="cuda", generator=g) * k).to(torch.float16)
                     for s, k in (((T, H), 1.0), ((n, H), H ** -0.5), ((n, H), H ** -0.5), ((T, n), 0.1)))
    nsaved, nwork = 4 * lib.gicc_gated_saved_floats(T, n), lib.gicc_gated_grad_bytes(T, n)
    saved, work = _buffer(nsaved), _buffer(nwork)
    h, dx, dwg, dwu = (torch.empty_like(t) for t in (dh, x, wg, wu))
    s = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    assert lib.gicc_gated_linear(p(x), p(wg), p(wu), p(h), T, H, n, H, H, H, n, 1, 0, p(saved), s) == 0
    assert lib.gicc_gated_linear_backward(p(dh), p(x), p(wg), p(wu), p(saved), p(work), p(dx), p(dwg), p(dwu), T, H, n, n, H, H,
                                          H, H, H, 1, 0, s) == 0
    _sync()
    for t, r in zip((h, dx, dwg, dwu), gated_ref(x, wg, wu, "gelu", dh)):
        check(t, r)
    assert bool((saved[nsaved:] == 0x5A).all()) and bool((work[nwork:] == 0x5A).all())


@pytest.mark.parametrize("T,K,n,L,r", [(1, 8, 1, 1, 8), (33, 136, 75, 4, 24), (300, 264, 515, 9, 72), (5000, 72, 300, 40, 16)])
def test_lora(lib, T, K, n, L, r):
    g = torch.Generator(device="cuda").manual_seed(T + K + n)
    x, w, a, b = ((torch.randn(*s, device="cuda", generator=g) * k).to(torch.bfloat16)
                  for s, k in (((T, K), 1.0), ((n, K), K ** -0.5), ((L, r, K), K ** -0.5), ((L, n, r), r ** -0.5)))
    ids = torch.randint(-1, L, (T,), device="cuda", generator=g).to(torch.int32)
    scale = torch.rand(L, device="cuda", generator=g) + 0.5
    nwork = lib.gicc_lora_work_bytes(T, L, r)
    work, y = _buffer(nwork), torch.empty(T, n, dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    assert lib.gicc_lora_linear(p(x), p(w), p(a), p(b), p(ids), p(scale), p(y), p(work), T, K, n, L, r, K, K, n, 1, s) == 0
    _sync()
    check(y, lora_ref(x, w, a, b, ids, scale))
    assert bool((work[nwork:] == 0x5A).all())


def test_first_calls_from_several_threads():
    """A process whose first calls come from several host threads at once, each on a stream of its own
    (ctypes leaves the interpreter's lock)."""
    import subprocess
    import sys
    code = """
import sys; sys.path[:0] = [%r, %r]
import threading
import torch
from projection_ref import check, gated_ref
from opengda_b200 import native
native()
import ctypes, os
P, LL, I = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int
lib = ctypes.CDLL(os.path.join(%r, "opengda_b200", "lib", "libgicc.so"))
for f in ("gicc_gated_saved_floats", "gicc_gated_grad_bytes"):
    getattr(lib, f).argtypes, getattr(lib, f).restype = [I] * 2, ctypes.c_size_t
lib.gicc_gated_linear.argtypes = [P, P, P, P, I, I, I, LL, LL, LL, LL, I, I, P, P]
lib.gicc_gated_linear_backward.argtypes = [P] * 9 + [I] * 3 + [LL] * 6 + [I, I, P]
jobs = []
for k, (T, H, n) in enumerate([(5, 264, 130), (700, 264, 300), (33, 512, 96), (1500, 136, 64)] * 2):
    g = torch.Generator(device="cuda").manual_seed(k)
    x, wg, wu, dh = ((torch.randn(*s, device="cuda", generator=g) * c).to(torch.bfloat16)
                     for s, c in (((T, H), 1.0), ((n, H), H ** -0.5), ((n, H), H ** -0.5), ((T, n), 0.1)))
    saved = torch.empty(lib.gicc_gated_saved_floats(T, n), device="cuda")
    work = torch.empty(lib.gicc_gated_grad_bytes(T, n), dtype=torch.uint8, device="cuda")
    jobs.append((torch.cuda.Stream(), T, H, n, x, wg, wu, dh, saved, work, [torch.empty_like(t) for t in (dh, x, wg, wu)]))
torch.cuda.synchronize()
start, rcs = threading.Barrier(len(jobs)), []
def run(job):
    s, T, H, n, x, wg, wu, dh, saved, work, out = job
    p = [t.data_ptr() for t in (x, wg, wu, dh, saved, work, *out)]
    torch.cuda.set_device(0)
    start.wait()
    for _ in range(3):
        rcs.append(lib.gicc_gated_linear(p[0], p[1], p[2], p[6], T, H, n, H, H, H, n, 0, 1, p[4], s.cuda_stream))
        rcs.append(lib.gicc_gated_linear_backward(p[3], p[0], p[1], p[2], p[4], p[5], p[7], p[8], p[9], T, H, n, n, H, H, H, H,
                                                  H, 0, 1, s.cuda_stream))
threads = [threading.Thread(target=run, args=(j,)) for j in jobs]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
from opengda_b200.ops.gemm import check_errors
check_errors()
assert len(rcs) == 6 * len(jobs) and not any(rcs), rcs
for _, _, _, _, x, wg, wu, dh, _, _, out in jobs:
    for t, r in zip(out, gated_ref(x, wg, wu, "silu", dh)):
        check(t, r)
print("done")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    root = os.path.dirname(here)
    r = subprocess.run([sys.executable, "-c", code % (root, here, root)], capture_output=True, text=True, timeout=180)
    assert "done" in r.stdout, r.stdout + r.stderr
