"""Refusals of the state-space and 4-bit entry points, on the CPU: bad calls are
rejected before any device work, by the Python functions and by the C entries."""
import ctypes

import pytest
import torch

from cpp1_b200 import _lib, ops

bf = torch.bfloat16


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def conv_args(**kw):
    a = dict(x=z(6, 8), weight=z(8, 4), bias=z(8))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,err", [
    (dict(x=z(6, 8, 1)), ValueError),
    (dict(x=z(6, 8, dtype=torch.float16)), TypeError),
    (dict(x=[1.0]), TypeError),
    (dict(weight=z(7, 4)), ValueError),
    (dict(weight=z(8, 1)), ValueError),
    (dict(weight=z(8, 9)), ValueError),
    (dict(weight=z(8, 4, dtype=bf)), TypeError),
    (dict(bias=z(9)), ValueError),
    (dict(bias=z(8, dtype=bf)), TypeError),
    (dict(activation="relu"), ValueError),
    (dict(activation=["silu"]), ValueError),
    (dict(state=z(1, 8, 4)), ValueError),
    (dict(state=z(1, 8, 3, dtype=bf)), TypeError),
    (dict(state=z(1, 3, 8).transpose(1, 2)), ValueError),
    (dict(state=z(1, 8, 3), state_out=z(2, 8, 3)), ValueError),
    (dict(offsets=torch.tensor([0, 6])), TypeError),
    (dict(offsets=i32(0, 6)[:0]), ValueError),
    (dict(offsets=i32(0, 6), slots=i32(0, 1)), ValueError),
    (dict(), ValueError),  # a CPU tensor, last of all
])
def test_conv_refusals(kw, err):
    with pytest.raises(err):
        ops.causal_conv(**conv_args(**kw))


@pytest.mark.parametrize("kw,err", [
    (dict(state=None), TypeError),
    (dict(state=z(6, 8, 2)), ValueError),
    (dict(slots=i32(0, 1)), ValueError),
    (dict(slots=torch.zeros(6)), TypeError),
    (dict(weight=z(8, 9)), ValueError),
    (dict(bias=z(8, 1)), ValueError),
    (dict(), ValueError),
])
def test_conv_step_refusals(kw, err):
    a = dict(state=z(6, 8, 3))
    a.update(kw)
    with pytest.raises(err):
        ops.causal_conv_step(**conv_args(**a))


def scan_args(**kw):
    a = dict(x=z(6, 4, 16), dt=z(6, 4), A=z(4), B=z(6, 2, 8), C=z(6, 2, 8))
    a.update(kw)
    return a


SCAN_BAD = [
    (dict(x=z(6, 64)), ValueError),
    (dict(x=z(6, 4, 16, dtype=torch.float64)), TypeError),
    (dict(dt=z(6, 3)), ValueError),
    (dict(dt=z(6, 4, dtype=bf)), TypeError),
    (dict(dt=None), TypeError),
    (dict(A=z(4, 1)), ValueError),
    (dict(A=z(4, dtype=bf)), TypeError),
    (dict(B=z(5, 2, 8)), ValueError),
    (dict(B=z(6, 3, 8), C=z(6, 3, 8)), ValueError),
    (dict(C=z(6, 2, 9)), ValueError),
    (dict(C=z(6, 2, 8, dtype=bf)), TypeError),
    (dict(B=z(6, 2, 257), C=z(6, 2, 257)), ValueError),
    (dict(B=z(6, 2, 0), C=z(6, 2, 0)), ValueError),
    (dict(x=z(6, 4, 257)), ValueError),
    (dict(D=z(5)), ValueError),
    (dict(dt_bias=z(4, dtype=bf)), TypeError),
    (dict(z=z(6, 4, 15)), ValueError),
    (dict(state=z(1, 4, 16, 9)), ValueError),
    (dict(state=z(1, 4, 16, 8, dtype=bf)), TypeError),
    (dict(), ValueError),
]


@pytest.mark.parametrize("kw,err", SCAN_BAD)
def test_scan_refusals(kw, err):
    with pytest.raises(err):
        ops.selective_scan(**scan_args(**kw))


@pytest.mark.parametrize("kw,err", SCAN_BAD + [(dict(state=None), TypeError)])
def test_step_refusals(kw, err):
    a = dict(state=z(6, 4, 16, 8))
    a.update(kw)
    with pytest.raises(err):
        ops.selective_step(**scan_args(**a))


@pytest.mark.parametrize("kw,err", [
    (dict(x=z(2, 64, 1)), ValueError),
    (dict(q=z(8, 32)), TypeError),
    (dict(q=z(8, 31, dtype=torch.uint8)), ValueError),
    (dict(x=z(2, 63)), ValueError),
    (dict(scales=z(8, 3)), ValueError),
    (dict(scales=z(8, 4)), ValueError),       # groups of 16
    (dict(scales=z(8, 0)), ValueError),
    (dict(scales=z(7, 1)), ValueError),
    (dict(scales=z(8, 1, dtype=torch.float16)), TypeError),
    (dict(scales=None), TypeError),
    (dict(zeros=z(8, 1)), TypeError),
    (dict(zeros=z(8, 2, dtype=torch.uint8)), ValueError),
    (dict(), ValueError),
])
def test_q4_refusals(kw, err):
    a = dict(q=z(8, 32, dtype=torch.uint8), scales=z(8, 1), x=z(2, 64))
    a.update(kw)
    with pytest.raises(err):
        ops.q4_matvec(**a)


# ---------------------------------------------------------------- C entries
BUF = ctypes.create_string_buffer(1 << 16)
P0 = (ctypes.addressof(BUF) + 255) // 256 * 256


def at(off):
    return P0 + off


def conv(x=at(0), w=at(4096), bias=None, offsets=None, si=None, so=None, slots=None, y=at(8192), tokens=4, channels=8,
         width=4, nseq=1, nslots=0, ldx=8, ldy=8, dtype=0, act=0):
    return _lib.load().smm_causal_conv(x, w, bias, offsets, si, so, slots, y, tokens, channels, width, nseq, nslots,
                                       ldx, ldy, dtype, act, None)


@pytest.mark.parametrize("kw", [
    dict(tokens=-1), dict(channels=-8), dict(nseq=-1), dict(nslots=-1), dict(width=1), dict(width=9), dict(dtype=2),
    dict(act=2), dict(ldx=7), dict(ldy=7), dict(x=None), dict(w=None), dict(y=None), dict(nseq=2), dict(so=at(16384)),
    dict(y=at(0)), dict(y=at(64)), dict(y=at(4096)), dict(tokens=1 << 31),
    dict(si=at(16384), so=at(16384 + 32), nslots=1), dict(so=at(0), nslots=1), dict(y=at(16384), so=at(16384), nslots=1),
])
def test_conv_entry_rejects(kw):
    assert conv(**kw) == _lib.SMM_ERR_INVALID
    assert _lib.last_error()


def test_empty_calls_do_nothing():
    L = _lib.load()
    assert conv(channels=0, x=None, y=None, w=None) == _lib.SMM_OK
    assert conv(tokens=0, nseq=0, x=None, y=None) == _lib.SMM_OK
    assert L.smm_causal_conv_step(None, at(0), None, None, None, None, None, 0, 8, 4, 0, 8, 8, 0, 0, None) == _lib.SMM_OK
    assert scan(tokens=0, nseq=0) == _lib.SMM_OK
    assert scan(heads=0, ldx=0, ldy=0, lddt=0) == _lib.SMM_OK
    assert q4(batch=0) == _lib.SMM_OK
    assert q4(rows=0, ldy=0) == _lib.SMM_OK


def scan(x=at(0), dt=at(8192), A=at(12288), B=at(16384), C=at(20480), D=None, zz=None, db=None, offsets=None, si=None,
         so=None, slots=None, y=at(4096), tokens=4, nseq=1, nslots=0, heads=2, dim=16, groups=1, n=8, ldx=32, lddt=2,
         ldb=8, ldc=8, ldz=0, ldy=32, dtype=0, dtd=0, ws=None, wsb=0):
    return _lib.load().smm_selective_scan(x, dt, A, B, C, D, zz, db, offsets, si, so, slots, y, tokens, nseq, nslots,
                                          heads, dim, groups, n, ldx, lddt, ldb, ldc, ldz, ldy, dtype, dtd, 0, ws, wsb,
                                          None)


@pytest.mark.parametrize("kw", [
    dict(tokens=-1), dict(nseq=-1), dict(heads=-2), dict(nslots=-1), dict(dim=0), dict(dim=257), dict(n=0),
    dict(n=257, ldb=257, ldc=257), dict(groups=0), dict(groups=3), dict(dtype=7), dict(dtd=-1), dict(ldx=31),
    dict(ldy=31), dict(ldb=7), dict(ldc=7), dict(lddt=1), dict(zz=at(24576), ldz=31), dict(x=None), dict(dt=None),
    dict(A=None), dict(B=None), dict(C=None), dict(y=None), dict(nseq=2), dict(si=at(32768)), dict(y=at(0)),
    dict(y=at(16384)), dict(y=at(8192)), dict(so=at(20480), nslots=1), dict(si=at(32768), so=at(32768 + 64), nslots=1),
    dict(tokens=1 << 31),
])
def test_scan_entry_rejects(kw):
    assert scan(**kw) == _lib.SMM_ERR_INVALID
    assert _lib.last_error()


def q4(q=at(0), scales=at(4096), zeros=None, x=at(8192), y=at(16384), batch=2, rows=8, cols=64, group=64, ldx=64, ldy=8,
       dtype=0, sd=0):
    return _lib.load().smm_q4_matvec(q, scales, zeros, x, y, batch, rows, cols, group, ldx, ldy, dtype, sd, None)


@pytest.mark.parametrize("kw", [
    dict(batch=-1), dict(rows=-1), dict(cols=-64), dict(group=16), dict(group=0), dict(group=48), dict(group=128),
    dict(dtype=3), dict(sd=3), dict(ldx=63), dict(ldy=7), dict(q=None), dict(scales=None), dict(x=None), dict(y=None),
    dict(q=at(8)), dict(x=at(8192 + 4)), dict(ldx=65), dict(y=at(8192 + 256)), dict(y=at(0)), dict(y=at(4096)),
    dict(batch=65536, y=at(1 << 26)),
])
def test_q4_entry_rejects(kw):
    assert q4(**kw) == _lib.SMM_ERR_INVALID
    assert _lib.last_error()


def test_scan_workspace_query():
    L = _lib.load()
    size = L.smm_selective_scan_workspace_size
    assert size(0, 1, 4, 64, 1, 128, 0) == 0
    assert size(100, 0, 4, 64, 1, 128, 0) == 0
    # few heads and one long prompt: split, with room for the segments' states
    assert size(65536, 1, 4, 64, 1, 128, 0) >= 2 * 4 * 64 * 128 * 4
    # enough heads: not split in fp32
    assert size(65536, 1, 128, 64, 1, 128, 0) == 0


def test_scan_reports_a_small_workspace():
    need = _lib.load().smm_selective_scan_workspace_size(65536, 1, 1, 16, 1, 8, 0)
    assert need > 0
    big = ctypes.create_string_buffer(65536 * (16 * 4 * 2 + 8 * 4 * 2 + 8) + 4096)
    p = (ctypes.addressof(big) + 255) // 256 * 256
    xs, bs = 65536 * 64, 65536 * 32
    rc = scan(x=p, y=p + xs, B=p + 2 * xs, C=p + 2 * xs + bs, dt=p + 2 * xs + 2 * bs, A=p + 2 * xs + 2 * bs + 65536 * 4,
              tokens=65536, heads=1, dim=16, n=8, ldx=16, ldy=16, lddt=1, ws=P0, wsb=need - 1)
    assert rc == _lib.SMM_ERR_WORKSPACE
    assert "required" in _lib.last_error()
