"""What the state-space entry points and the 4-bit product refuse of the memory they are given, on the
CPU: outputs that share bytes with inputs, counted by rows of a common stride, pointers that
are not aligned to their elements, dimensions that do not fit the entries' integers."""
import ctypes
import random

import pytest
import torch

from cpp1_b200 import _lib, ops

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


Q = [P0 + 4096 * i for i in range(16)]  # places 4 KB apart


@pytest.mark.parametrize("which", range(8))
@pytest.mark.parametrize("dtype,shift", [(0, 2), (0, 1), (1, 1)])
def test_conv_pointers_off_their_elements(which, dtype, shift):
    ptrs = Q[:8]  # x, w, bias, offsets, state_in, state_out, slots, y
    ptrs[which] += shift
    rc = _lib.load().smm_causal_conv(*ptrs, 4, 8, 4, 1, 2, 8, 8, dtype, 0, None)
    assert rc == _lib.SMM_ERR_INVALID and "not aligned" in _lib.last_error()


@pytest.mark.parametrize("which", range(13))
@pytest.mark.parametrize("dtype,shift", [(0, 2), (0, 1), (1, 1)])
def test_scan_pointers_off_their_elements(which, dtype, shift):
    # x, dt, A, B, C, D, z, dt_bias, offsets, state_in, state_out, slots, y
    ptrs = Q[:13]
    ptrs[which] += shift
    rc = _lib.load().smm_selective_scan(*ptrs, 4, 1, 2, 2, 16, 1, 8, 32, 2, 8, 8, 32, 32, dtype, dtype, 0, None, 0, None)
    assert rc == _lib.SMM_ERR_INVALID and "not aligned" in _lib.last_error()
    if which == 8:
        return
    step = ptrs[:8] + ptrs[9:]
    rc = _lib.load().smm_selective_step(*step, 2, 2, 2, 16, 1, 8, 32, 2, 8, 8, 32, 32, dtype, dtype, 0, None)
    assert rc == _lib.SMM_ERR_INVALID and "not aligned" in _lib.last_error()


@pytest.mark.parametrize("which,dtype,sd,shift", [(1, 0, 0, 2), (1, 0, 1, 1), (4, 0, 0, 2), (4, 1, 0, 1), (1, 1, 0, 2)])
def test_q4_pointers_off_their_elements(which, dtype, sd, shift):
    ptrs = Q[:5]  # q, scales, zeros, x, y
    ptrs[which] += shift
    rc = _lib.load().smm_q4_matvec(*ptrs, 2, 8, 64, 64, 64, 8, dtype, sd, None)
    assert rc == _lib.SMM_ERR_INVALID and "not aligned" in _lib.last_error()


def huge(*shape, dtype=torch.float32):
    """A tensor of one element seen as many."""
    return torch.zeros((), dtype=dtype).expand(shape)


MANY = (1 << 32) + 8  # would count as 8 in 32 bits


@pytest.mark.parametrize("call", [
    lambda: ops.q4_matvec(huge(MANY, 16, dtype=torch.uint8), huge(MANY, 1), torch.zeros(1, 32)),
    lambda: ops.q4_matvec(huge(4, 16, dtype=torch.uint8), huge(4, 1), huge(MANY, 32)),
    lambda: ops.causal_conv(huge(MANY, 4), torch.zeros(4, 4)),
    lambda: ops.causal_conv(torch.zeros(4, 4), torch.zeros(4, 4), state=huge(MANY, 4, 3)),
    lambda: ops.causal_conv(torch.zeros(4, 4), torch.zeros(4, 4), offsets=huge(MANY, dtype=torch.int32)),
    lambda: ops.causal_conv_step(huge(MANY, 4), torch.zeros(4, 4), state=huge(MANY, 4, 3)),
    lambda: ops.causal_conv_step(huge(1, MANY), huge(MANY, 4), state=huge(1, MANY, 3)),
    lambda: ops.selective_scan(huge(MANY, 2, 16), huge(MANY, 2), torch.zeros(2), huge(MANY, 1, 8), huge(MANY, 1, 8)),
    lambda: ops.selective_step(torch.zeros(3, 2, 16), torch.zeros(3, 2), torch.zeros(2), torch.zeros(3, 1, 8),
                               torch.zeros(3, 1, 8), state=huge(MANY, 2, 16, 8)),
])
def test_dimensions_beyond_31_bits(call):
    with pytest.raises(ValueError, match="31 bits"):
        call()
