"""Which row of the weights' scales a wave of the 8-bit tiles reads (host
arithmetic, no GPU).  Weights have [ceil(rows / 128)] of them: a wave whose weight
rows all lie past the last reads none beyond.  What it computes from them is not
stored, so no output shows where it read."""
import pytest

import q4mi


@pytest.mark.parametrize("bn,waves", [(32, 2), (64, 2), (128, 2), (256, 4), (256, 2)])
def test_scale_rows_exist(bn, waves):
    M = q4mi.meas()
    sizes = list(range(1, 4 * 256 + 2)) + [6500, 54613, 151936, 15232, (1 << 30) - 1, 1 << 30]
    for rows in sizes:
        have, tiles = -(-rows // 128), -(-rows // bn)
        for tile in {0, max(tiles - 2, 0), tiles - 1}:
            for wave in range(waves):
                first = wave * (bn // waves)
                row = M.q4mi_f8_tile_scale_row(rows, tile * bn, first)
                assert row < have, (rows, tile, wave)
                if tile * bn + first < rows:
                    assert row == (tile * bn + first) // 128, (rows, tile, wave)
