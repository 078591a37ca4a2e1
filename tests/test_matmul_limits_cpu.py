"""Matmuls of few rows whose launch would hold 2^32 threads or more (2^27 columns) are
refused (such a grid wraps without an error); on the host, nothing is launched."""

import ctypes

import pytest

from mlx_batch_invariant_amd import _lib

P = ctypes.c_void_p(256)                                 # never dereferenced
BIG = 1 << 62


@pytest.mark.parametrize("M", [1, 16, 24])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_columns_of_the_row_kernels(M, dtype):
    lib = _lib.load()
    rc = lib.bi_matmul(P, 32, P, 32, P, M, 1 << 27, 32, dtype, P, BIG, None)
    assert rc == -2 and "grid too large" in lib.bi_last_error().decode()
    # ... and the next call is not blamed for it
    assert lib.bi_matmul(P, 32, P, 32, P, 0, 64, 32, dtype, P, BIG, None) == 0
