"""Overlaps of the two gradients that the 8-bit backward refuses at its C entry, before any device is touched."""
import pytest

from kernel_pocs_b200 import _lib


@pytest.mark.parametrize("distance,pitch,rows,es", [
    (0, 40, 4, 4), (39, 40, 4, 4), (-39, 40, 4, 4),        # contiguous rows, shifted by less than all of them
    (40, 40, 4, 4), (-80, 40, 4, 2),                       # by whole rows
    (20, 80, 4, 2), (-39, 100, 4, 2), (39, 100, 4, 4),     # interleaved rows that reach into one another
    (70, 100, 4, 2),                                       # into the next row
    (1, 40, 1, 4), (-39, 1000, 1, 2),                      # one row, whatever its pitch
])
def test_gradients_whose_rows_overlap_are_refused(distance, pitch, rows, es):
    p = 0x1000000
    cols, dgate, kept = 40, p + 0x100000, p + 0x400000
    dtype = _lib.F32 if es == 4 else _lib.BF16
    for h in (None, p + 0x800000):
        assert _lib.lib.swiglu_b200_ckpt8_bwd(h, dgate, dgate + distance * es, p, kept, kept + 0x1000, kept + 0x2000,
                                              kept + 0x3000, rows, cols, pitch, cols, cols, dtype, 0, 1.0, 1.0, -1, None) == 5
