"""C entries of the 8-bit-activation experts: pointers that the kernels' wide pieces do not fit are
refused before a launch, on the CPU."""

import ctypes
import os

import pytest


@pytest.fixture(scope="module")
def lib():
    from torchtitan_amd import _lib

    if not os.path.exists(_lib.library_path()):
        from torchtitan_amd import build

        build.build()
    return _lib.lib()


def test_gate_up_keep8_alignment(lib):
    """g and u are written in 8-byte pieces, their scales byte by byte."""
    buf = ctypes.create_string_buffer(80)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    run = lambda *kept, rows=4: lib.moe_grouped_gemm_gate_up_keep8(at, at, at, at, rows, 2, 64, 64, *kept, at, None)  # noqa: E731
    for off in (1, 2, 4):
        assert run(at + off, at, at, at) == -1 and run(at, at, at + off, at) == -1
    assert run(at + 8, at + 1, at + 8, at + 3, rows=0) == 0  # nothing to write
