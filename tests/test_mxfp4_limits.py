"""Sizes that a launch of the MXFP4 products cannot hold are refused before any work, on the CPU."""
from __future__ import annotations

import ctypes

import pytest

P = ctypes.c_void_p
A = 1 << 20  # an aligned address that is never read


@pytest.mark.parametrize("rows,n,m", [(16 * 65535, 40960, 16), (16 * 65535, 32768, 1024), (300000, 1 << 17, 512)])
def test_quantized_inputs_of_2_to_the_32_lanes(rows, n, m):
    """The rows' launch takes 8 values a lane, of rows padded to whole 512 inputs, and the weight's
    scales four bytes a lane."""
    from rwkv7mi import _lib

    lib = _lib.load()
    assert 64 * rows * -(-n // 512) + 4 * m * -(-n // 512) > 2 ** 32 - 1024
    for dt in (_lib.F16, _lib.BF16):
        # (as any call that is refused, it asks for no workspace)
        assert lib.rwkv7mi_mxfp4_linear_workspace_bytes(1, rows, m, n, dt, 1) == 0
        assert lib.rwkv7mi_mxfp4_linear1(A, A, A, None, None, A, 0, rows, m, n, dt, 1, None, 0, None) == -1
        assert b"too large" in lib.rwkv7mi_last_error()
    # a fraction of the rows is no such call: it only lacks its workspace
    need = lib.rwkv7mi_mxfp4_linear_workspace_bytes(1, rows // 8, m, n, _lib.F16, 1)
    assert need > 0
    assert lib.rwkv7mi_mxfp4_linear1(A, A, A, None, None, A, 0, rows // 8, m, n, _lib.F16, 1, None, 0, None) == -3


@pytest.mark.parametrize("rows,n,m", [(262144, 1 << 21, 256), (65536, 4096, 4096), (4001, 96, 16325)])
def test_long_batches_ask_for_the_weight_in_16_bits_alone(rows, n, m):
    """Also for inputs so wide that a chunk of rows below 2 GiB is a single tile."""
    from rwkv7mi import _lib

    records, factors = 2 * -(-m // 32) * -(-n // 64) * 2048, -(-4 * m // 256) * 256
    assert _lib.load().rwkv7mi_mxfp4_linear_workspace_bytes(1, rows, m, n, _lib.BF16, 0) == records + factors
