"""Calls of gated_linear and lora_linear that are refused on the host, before anything touches a GPU."""
import ctypes
import os

import pytest
import torch

P, LL, I = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int


@pytest.fixture(scope="module")
def lib():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = ctypes.CDLL(os.path.join(root, "opengda_b200", "lib", "libgicc.so"))
    lib.gicc_gated_linear.argtypes = [P, P, P, P, I, I, I, LL, LL, LL, LL, I, I, P, P]
    lib.gicc_gated_linear_backward.argtypes = [P] * 9 + [I] * 3 + [LL] * 6 + [I, I, P]
    lib.gicc_lora_linear.argtypes = [P] * 8 + [I] * 5 + [LL] * 3 + [I, P]
    return lib


def _refused(rc, capfd, what):
    assert rc == -1
    err = capfd.readouterr().err
    assert what in err, err


def test_unaligned_saved(lib, capfd):
    """The kernels write and read saved in 16-byte pieces."""
    for off in (4, 8, 24):
        what = "saved must be 16-byte aligned"
        _refused(lib.gicc_gated_linear(16, 16, 16, 16, 4, 16, 8, 16, 16, 16, 8, 0, 1, off, None), capfd, what)
        _refused(lib.gicc_gated_linear_backward(16, 16, 16, 16, off, 16, 16, 16, 16, 4, 16, 8, 8, 16, 16, 16, 16, 16, 0, 1,
                                                None), capfd, what)


def _args():
    """Valid but for the device: reaches the check of the device where nothing before it refuses."""
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    gated = {"x": z(4, 16), "w_gate": z(8, 16), "w_up": z(8, 16)}
    lora = {"x": z(4, 16), "w": z(8, 16), "lora_a": z(1, 8, 16), "lora_b": z(1, 8, 8), "adapter": torch.zeros(4, dtype=torch.int32),
            "scale": torch.ones(1)}
    return gated, lora


def test_forward_mode_tangents():
    """A dual tensor does not require a gradient: without a check its tangent is dropped."""
    import torch.autograd.forward_ad as fwd
    from opengda_b200.ops.ffn import gated_linear, gated_linear_backward, gated_linear_forward
    from opengda_b200.ops.lora import lora_linear
    gated, lora = _args()
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for name in gated:
            for grads in (False, True):
                args = {k: t.clone().requires_grad_(grads and k != name) for k, t in gated.items()}
                args[name] = dual(args[name])
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    gated_linear(**args)
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                gated_linear_forward(**dict(gated, **{name: dual(gated[name])}))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            gated_linear(**gated, out=dual(torch.zeros(4, 8, dtype=torch.bfloat16)))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            gated_linear_backward(dual(torch.zeros(4, 8, dtype=torch.bfloat16)), **gated, saved=torch.zeros(1024))
        for name in ("x", "w", "lora_a", "lora_b", "scale"):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                lora_linear(**dict(lora, **{name: dual(lora[name])}))
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):  # a dual level alone refuses nothing
            gated_linear(**gated)
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            lora_linear(**lora)


@pytest.mark.filterwarnings("ignore")
def test_tracing():
    """A trace holds the output's allocation and not the launch: what it returns would be whatever the
    memory held."""
    from opengda_b200.ops.ffn import gated_linear, gated_linear_backward, gated_linear_forward
    from opengda_b200.ops.lora import lora_linear
    gated, lora = _args()
    dh, saved = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(1024)
    for f in (lambda x: gated_linear(**dict(gated, x=x)), lambda x: gated_linear_forward(**dict(gated, x=x))[0],
              lambda x: gated_linear(x, gated["w_gate"].requires_grad_(True), gated["w_up"]),
              lambda x: gated_linear_backward(dh, **dict(gated, x=x), saved=saved)[0], lambda x: lora_linear(**dict(lora, x=x))):
        gated["w_gate"].requires_grad_(False)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (gated["x"],))


def test_sizes_next_to_the_integers_end(lib, capfd):
    """Rounded up to a tile such a size would overflow into a negative grid."""
    big, what = 2 ** 31 - 8, "sizes from 1 to"
    for T, H, n in ((big, 16, 8), (4, big, 8), (4, 16, big)):
        _refused(lib.gicc_gated_linear(16, 16, 16, 16, T, H, n, H, H, H, n, 0, 1, None, None), capfd, what)
        _refused(lib.gicc_gated_linear_backward(16, 16, 16, 16, 16, 16, 16, 16, 16, T, H, n, n, H, H, H, H, H, 0, 1, None), capfd,
                 what)
    for T, K, n in ((big, 16, 8), (4, big, 8), (4, 16, big)):
        _refused(lib.gicc_lora_linear(16, 16, 16, 16, 16, None, 16, 16, T, K, n, 1, 8, K, K, n, 1, None), capfd, what)


def test_work_sizes_of_the_c_interface(lib):
    """What a C caller has to allocate: at least the plain arrays, padded; 0 for sizes that are refused."""
    for f, n in (("gicc_gated_saved_floats", 2), ("gicc_gated_grad_bytes", 2), ("gicc_lora_work_bytes", 3)):
        getattr(lib, f).argtypes, getattr(lib, f).restype = [I] * n, ctypes.c_size_t
    for T, n in ((1, 1), (5, 33), (32, 16), (61, 37), (8192, 8192), (65600, 32800)):
        saved = lib.gicc_gated_saved_floats(T, n)
        assert saved == 2 * ((T + 31) // 32 * 32) * ((n + 15) // 16 * 16) >= 2 * T * n
        assert lib.gicc_gated_grad_bytes(T, n) >= 2 * T * n * 2 + 4
        assert lib.gicc_lora_work_bytes(T, 3, 24) >= T * 24 * 2
    for a, b in ((0, 4), (4, 0), (-1, 4), (2 ** 31 - 1, 4), (4, 2 ** 31 - 1)):
        assert lib.gicc_gated_saved_floats(a, b) == lib.gicc_gated_grad_bytes(a, b) == 0
    for a, b, c in ((0, 4, 8), (4, 0, 8), (4, 8193, 8), (4, 4, 136), (2 ** 31 - 1, 4, 8)):
        assert lib.gicc_lora_work_bytes(a, b, c) == 0


def test_c_header_is_c(tmp_path):
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "p.c"
    src.write_text("#include <gicc/projections.h>\n"
                   "int main(void) { return gicc_gated_saved_floats(4, GICC_ACT_GELU) == 0; }\n")
    p = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I" + os.path.join(root, "csrc", "include"), "-I/usr/local/cuda/include",
                        "-fsyntax-only", str(src)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stderr


def test_sizes_asked_for_their_tile():
    from opengda_b200 import native
    for sizes in ((0, 64, 8), (4, 0, 8), (4, 64, 0), (2 ** 31 - 8, 64, 8)):
        with pytest.raises(RuntimeError, match="sizes from 1 to"):
            native().gated_linear_tile(*sizes)
        with pytest.raises(RuntimeError, match="sizes from 1 to"):
            native().lora_linear_tile(*sizes, 8)
