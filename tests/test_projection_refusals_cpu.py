"""Calls of gated_linear and lora_linear that are refused on the host, before anything touches a GPU."""
import ctypes
import os

import pytest

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
