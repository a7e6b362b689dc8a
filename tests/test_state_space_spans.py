"""Which memory the state-space entry points and the 4-bit product take for overlapping: refusals
of outputs that share bytes with inputs, counted by rows of a common stride, on the CPU."""
import ctypes
import random

import pytest
import torch

from cpp1_b200 import _lib

BUF = ctypes.create_string_buffer(1 << 18)
P0 = (ctypes.addressof(BUF) + 255) // 256 * 256
FAR = P0 + (1 << 17)


def touches(ax, rows_a, wa, la, bx, rows_b, wb, lb):
    a = {ax + i * la + j for i in range(rows_a) for j in range(wa)}
    return any(bx + i * lb + j in a for i in range(rows_b) for j in range(wb))


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused would be launched on host memory")
def test_random_columns_of_one_matrix():
    """A convolution's x and y as columns (in floats) of one matrix: refused if and only if they share one."""
    L = _lib.load()
    rng = random.Random(3)
    seen = set()
    for _ in range(4000):
        c, rows = rng.randint(1, 6), rng.randint(1, 5)
        ld = rng.randint(c, 14)
        ldy = ld if rng.random() < 0.8 or rows > 1 else rng.randint(c, 14)
        ox, oy = rng.randint(0, 70), rng.randint(0, 70)
        rc = L.smm_causal_conv(P0 + 4 * ox, FAR, None, None, None, None, None, P0 + 4 * oy, rows, c, 2, 1, 0, ld, ldy,
                               0, 0, None)
        hit = touches(ox, rows, c, ld, oy, rows, c, ldy)
        seen.add(hit)
        assert (rc == _lib.SMM_ERR_INVALID) == hit, (c, rows, ld, ox, oy)
    assert seen == {True, False}


@pytest.mark.parametrize("oy,ldx,ldy", [(0, 64, 64), (64 + 31, 64, 64), (65 - 32, 64, 64), (32, 64, 72), (64 * 3, 64, 64),
                                        (-31, 64, 64)])
def test_scan_columns_that_share_elements(oy, ldx, ldy):
    """y against x (four rows of 32 floats): the same columns, columns shifted by less than a row's
    width, other strides."""
    L = _lib.load()
    x = P0 + 4096
    rc = L.smm_selective_scan(x, FAR, FAR + 4096, FAR + 8192, FAR + 16384, None, None, None, None, None, None, None,
                              x + 4 * oy, 4, 1, 0, 2, 16, 1, 8, ldx, 2, 8, 8, 0, ldy, 0, 0, 0, None, 0, None)
    assert rc == _lib.SMM_ERR_INVALID and "overlaps" in _lib.last_error()
