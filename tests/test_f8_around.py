"""Which outputs of the 8-bit products go around the caches (host arithmetic, no GPU):
those that the last cache could not keep for their reader, in whole lines."""
import pytest

import q4mi

A = 1 << 20


@pytest.mark.parametrize("yt,size", [(0, 4), (1, 2), (30, 2)])
def test_by_output_size(yt, size):
    M = q4mi.meas()
    for n, rows in ((640, 1024), (129, 16384), (2048, 8192), ((128 << 20) // 8192 // size, 8192)):
        assert not M.q4mi_f8_around(A, yt, rows, n, rows), (n, rows)
    n = (128 << 20) // 8192 // size + 1
    assert M.q4mi_f8_around(A, yt, 8192, n, 8192)
    assert M.q4mi_f8_around(A + 64, yt, 8192 + 64 // size, n, 8192)
    assert not M.q4mi_f8_around(A + 32, yt, 8192, n, 8192)
    assert not M.q4mi_f8_around(A, yt, 8193, n, 8192)
