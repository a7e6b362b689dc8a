"""State-space operators and the 4-bit product where they can go wrong: busy memory,
accuracy, decays, non-finite values, calls from several threads and streams, limits."""
import threading

import pytest
import torch

from cpp1_b200 import _lib, ops
from test_gpu_state_space import SCAN_CASES, TYPES, U, conv_ref, conv_tol, gen, half_step, i32, make_scan, offs, q4_ref, rnd, scan_ref, scan_tol, state_tol, within

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("lens,h,n", [([128] * 24, 64, 128), ([256] * 9, 40, 128), ([300, 90, 513], 148, 64)])
def test_scan_beside_busy_memory(cuda, lens, h, n):
    """The tensor-core scan's loads arrive in any order when other streams keep the memory
    busy: chunks whose C lands long after B and x give the same bits as on a quiet GPU."""
    b = offs(lens)
    a = make_scan(h, b[-1], h, 64, 1, n, "bf16")
    st = rnd(gen(h), len(lens), h, 64, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    o = i32(b)
    y = ops.selective_scan(**a, offsets=o, state=st, state_out=so)
    within(y, ref, scan_tol(ref, mag, n, max(lens), BF, True), "y")
    within(so, fin, state_tol(fin, fmag, max(lens), True), "state")
    big = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    other = torch.empty_like(big)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(15):
        for s in side:
            with torch.cuda.stream(s):
                other.copy_(big)
        so2 = torch.empty_like(st)
        y2 = ops.selective_scan(**a, offsets=o, state=st, state_out=so2)
        torch.cuda.synchronize()
        assert torch.equal(y2, y) and torch.equal(so2, so)


# ---------------------------------------------------------------- accuracy
def on_tensor_cores(a, lens):
    """The rule by which bf16 prompts take the tensor cores (aligned pieces, one tile of state)."""
    t, _, p = a["x"].shape
    n = a["B"].shape[2]
    return (a["x"].dtype is BF and p % 8 == 0 and n % 8 == 0 and n <= 128
            and t * (n + 15) * p >= 3500 * len(lens) * 64 * ((p + 63) // 64))


def once_rounded_tol(ref, mag, n, longest, dtype):
    """One rounding to the output's type, and behind it what 32-bit sums leave: the recurrence's
    roundings as in scan_tol; on the tensor cores two terms of 2^-17 each for the scores and the state,
    and 40 additions truncated to 2^-23 of the sum, 2^-17.7."""
    return scan_tol(ref, mag, n, longest, dtype, False) + (2.0 ** -16 + 2.0 ** -17.7) * mag


@pytest.mark.parametrize("lens,h,p,g_,n", [
    ([128], 4, 64, 1, 128), ([127, 129, 1, 0, 256], 4, 64, 2, 128), ([300, 100], 8, 64, 8, 64), ([513], 2, 128, 1, 128),
    ([200, 131], 3, 96, 1, 96), ([260], 5, 40, 1, 24), ([1000], 2, 64, 1, 128), ([64] * 9, 2, 32, 1, 16),
    ([600, 1400], 1, 64, 1, 8), ([700, 37, 260], 160, 64, 8, 128), ([130, 900, 1, 0, 128], 200, 64, 1, 64)])
@pytest.mark.parametrize("with_state", [False, True])
def test_bf16_scan_rounds_its_outputs_alone(cuda, lens, h, p, g_, n, with_state):
    """Scores, decays and states are not cut to the inputs' 8 bits on their way: where the terms
    of an output cancel, its error stays that of its own rounding."""
    b = offs(lens)
    a = make_scan(h + n, b[-1], h, p, g_, n, "bf16", z=h % 2 == 0)
    st = rnd(gen(n), len(lens), h, p, n) if with_state else None
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty(len(lens), h, p, n, device="cuda")
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    within(y, ref, once_rounded_tol(ref, mag, n, max(lens), BF), "y")
    # a rounding of the exact result, and 2^-16 of the terms beside it
    best = float((ref.to(BF).double() - ref).norm())
    assert float((y.double() - ref).norm()) <= best + 2.0 ** -16 * float(mag.norm())


@pytest.mark.parametrize("lens,h,p,n", [([2048], 16, 64, 128), ([700, 37, 260], 40, 64, 64), ([4097], 2, 64, 128),
                                        ([300] * 6, 8, 128, 16)])
def test_tensor_core_states_keep_32_bits(cuda, lens, h, p, n):
    """Over all elements a final state is within 2^-20: three terms of the weighted x leave 2^-24, 24
    truncated additions of random signs 5 x 2^-24, two exponentials 2^-22 each.  Two terms would leave 2^-18.7."""
    b = offs(lens)
    a = make_scan(n, b[-1], h, p, 1, n, "bf16")
    assert on_tensor_cores(a, lens)
    st = rnd(gen(h), len(lens), h, p, n)
    _, _, (fin, _) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    assert float((so.double() - fin).norm()) <= 2.0 ** -20 * float(fin.norm())


@pytest.mark.parametrize("lens,h,p,g_,n", SCAN_CASES)
def test_bf16_recurrence_sums_in_32_bits(cuda, lens, h, p, g_, n):
    """bf16 prompts that are too short or too odd for the tensor cores: the fp32 recurrence's tolerance."""
    b = offs(lens)
    a = make_scan(h + p + n, b[-1], h, p, g_, n, "bf16", strided=p % 32 != 0)
    if on_tensor_cores(a, lens):
        a = {k: v[..., 1:] if k in ("B", "C") else v for k, v in a.items()}  # an odd state size goes there too
        n -= 1
    st = rnd(gen(n), len(lens), h, p, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    longest = max(max(lens), 1)
    within(y, ref, scan_tol(ref, mag, n, longest, BF, False), "y")
    within(so, fin, state_tol(fin, fmag, longest, False), "state")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,h,p,n", [([40, 7, 65], 64, 64, 256), ([40, 7, 65], 16, 64, 256), ([30] * 9, 72, 20, 136),
                                        ([200], 64, 64, 200), ([50, 90], 96, 64, 16), ([50, 90], 9, 64, 12)])
def test_recurrence_variants(cuda, dtype, lens, h, p, n):
    """Both sides of the recurrence's choices: one or two dims a lane, one or two CTAs on an SM."""
    b = offs(lens)
    a = make_scan(h + n, b[-1], h, p, 1, n, dtype)
    st = rnd(gen(n), len(lens), h, p, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    tensor = on_tensor_cores(a, lens)
    within(y, ref, (once_rounded_tol if tensor else lambda *v: scan_tol(*v, False))(ref, mag, n, max(lens), TYPES[dtype]), "y")
    within(so, fin, state_tol(fin, fmag, max(lens), tensor), "state")


# ---------------------------------------------------------------- giving up
@pytest.mark.parametrize("lens,h,n", [([700, 37, 260], 160, 128), ([100] * 40, 24, 64), ([6000], 2, 128), ([5000, 90], 3, 64)])
def test_scan_that_gives_up_leaves_cleanly(cuda, lens, h, n):
    """With a wait limit of a microsecond some wait of the tensor-core scan runs out: the
    expiry is reported once, whatever was under way has landed, and the next call is right."""
    L = _lib.load()
    b = offs(lens)
    a = make_scan(h, b[-1], h, 64, 1, n, "bf16")
    assert on_tensor_cores(a, lens)
    o = i32(b)
    so = torch.empty(len(lens), h, 64, n, device="cuda")
    y = ops.selective_scan(**a, offsets=o, state_out=so)
    ops.device_status()
    for _ in range(3):
        so2 = torch.empty_like(so)
        assert L.smm_debug_wait_limit_next(1000) == _lib.SMM_OK
        ops.selective_scan(**a, offsets=o, state_out=so2)
        with pytest.raises(_lib.SmmError) as e:
            ops.device_status()
        assert e.value.status == _lib.SMM_ERR_DEVICE_TIMEOUT
        ops.device_status()  # consumed
        y2 = ops.selective_scan(**a, offsets=o, state_out=so2)
        ops.device_status()  # and the limit was for one call
        assert torch.equal(y2, y) and torch.equal(so2, so)


# ---------------------------------------------------------------- strong resets
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("strength", [1e3, 1e4, 1e5, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("empty", [False, True])
def test_tokens_behind_a_reset(cuda, dtype, strength, empty):
    """A token whose d A is large and negative forgets the state; what it adds itself (nothing, if
    its x is zero) and the tokens behind it decay as they would without it."""
    lens, h, n = [300, 140], 4, 128
    b = offs(lens)
    a = make_scan(3, b[-1], h, 64, 1, n, dtype, strided=False, dt_f32=True)
    a["dt"] = 0.01 + 0.1 * torch.rand(b[-1], h, generator=gen(5), device="cuda")
    a["dt_bias"], a["dt_softplus"] = None, False
    a["A"] = torch.tensor([-1.0, -0.01, -8.0, -0.5], device="cuda")
    resets = [0, 5, 37, 38, 64, 200, 255, 300 + 1, 300 + 70, 300 + 99]
    for r in resets:
        a["dt"][r] = strength
        if empty:
            a["x"][r] = 0
    st = rnd(gen(4), 2, h, 64, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    # Exponents within 32 tokens are differences of two sums of five additions each.  Two
    # resets in a row count as 130 binary orders each at most, what is below is zero.
    sums = 10 * U * 0.7 * (2 * 130 + 32 * 0.11 * 8 * 1.45)
    tol = once_rounded_tol(ref, mag, n, 300, TYPES[dtype]) + (sums * mag if dtype == "bf16" else 0)
    within(y, ref, tol, "y")
    within(so, fin, state_tol(fin, fmag, 300, False) + sums * fmag, "state")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("every", [2, 5])
def test_resets_all_over(cuda, dtype, every):
    """Every second (fifth) token forgets."""
    t, h, n = 260, 4, 64
    a = make_scan(4, t, h, 64, 1, n, dtype, strided=False, dt_f32=True)
    a["dt"] = 0.01 + 0.1 * torch.rand(t, h, generator=gen(5), device="cuda")
    a["dt"][1::every] = 2e4
    a["x"][1::every] = 0
    a["dt_bias"], a["dt_softplus"] = None, False
    a["A"] = torch.tensor([-1.0, -0.01, -8.0, -0.5], device="cuda")
    ref, mag, (fin, fmag) = scan_ref(a, [0, t], None)
    so = torch.empty(1, h, 64, n, device="cuda")
    y = ops.selective_scan(**a, state_out=so)
    sums = 10 * U * 0.7 * (32 / every * 130 + 32 * 0.11 * 8 * 1.45)  # as in test_tokens_behind_a_reset
    tol = once_rounded_tol(ref, mag, n, t, TYPES[dtype]) + (sums * mag if dtype == "bf16" else 0)
    within(y, ref, tol, "y")
    within(so, fin, state_tol(fin, fmag, t, False) + sums * fmag, "state")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,h", [([300, 17], 4), ([3000], 4)])
def test_states_that_grow(cuda, dtype, lens, h):
    """Steps of both signs and rates of both signs: states grow and shrink."""
    b = offs(lens)
    n = 128
    a = make_scan(5, b[-1], h, 64, 1, n, dtype, strided=False, dt_f32=True)
    a["dt"] = 0.6 * torch.rand(b[-1], h, generator=gen(7), device="cuda") - 0.3
    a["dt_bias"], a["dt_softplus"] = None, False
    a["A"] = torch.tensor([0.3, -0.3, 0.05, 0.0], device="cuda")
    st = rnd(gen(8), len(lens), h, 64, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    within(y, ref, once_rounded_tol(ref, mag, n, max(lens), TYPES[dtype]), "y")
    within(so, fin, state_tol(fin, fmag, max(lens), dtype == "bf16"), "state")


# ---------------------------------------------------------------- non-finite inputs
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,h,p,n", [([140, 70, 300], 2, 64, 128), ([128, 128], 3, 128, 64), ([5, 9, 16], 4, 64, 16), ([6000], 2, 64, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_values_reach_no_token_before_them(cuda, dtype, lens, h, p, n, value):
    """What does not depend on a non-finite element keeps its bits, what does is not finite."""
    b = offs(lens)
    t = b[-1]
    dt = TYPES[dtype]
    clean = make_scan(6, t, h, p, 1, n, dtype, strided=False, dt_f32=True)
    st = rnd(gen(4), len(lens), h, p, n)

    def call(a):
        so = torch.empty_like(st)
        return ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so), so

    good, gst = call(clean)
    seq = len(lens) - 1
    toks = sorted({b[seq], b[seq] + 3, b[seq + 1] - 1, b[seq] + lens[seq] // 2})
    for what in ("x", "B", "C", "dt", "z"):
        a = dict(clean)
        a[what] = clean[what].clone()
        hit = torch.zeros(t, h, p, dtype=torch.bool, device="cuda")  # outputs that depend on it
        hst = torch.zeros(h, p, n, dtype=torch.bool, device="cuda")
        for i, k in enumerate(toks[1:3] if what in ("B", "dt") else toks):
            head, dim = i % h, (7 * i + 3) % p
            if what == "x":
                a["x"][k, head, dim] = value
                hit[k:, head, dim] = True
                hst[head, dim] = True
            elif what == "z":
                a["z"][k, head, dim] = value
                hit[k, head, dim] = True
            elif what == "dt":
                a["dt"][k, head] = float("nan")
                hit[k:, head] = True
                hst[head] = True
            elif what == "B":
                a["B"][k, 0, i] = value
                hit[k:] = True
                hst[:, :, i] = True
            else:
                a["C"][k, 0, i] = value
                hit[k] = True
        y, so = call(a)
        if what == "z" and value == float("-inf"):
            hit &= ~y.isfinite()  # a gate of minus infinity is zero at its limit, or no number
        assert torch.equal(y[~hit], good[~hit]), what
        assert not y[hit].isfinite().any(), what
        assert torch.equal(so[:seq], gst[:seq])
        assert torch.equal(so[seq][~hst], gst[seq][~hst]), what
        assert not so[seq][hst].isfinite().any(), what
    assert y.dtype == dt


# ---------------------------------------------------------------- several callers
def test_q4_from_several_threads(cuda):
    """Calls of one kernel with different amounts of shared memory, each thread on its own stream."""
    L = _lib.load()
    g = gen(2)
    failed = []
    start = threading.Barrier(6)

    def work(args, stream):
        torch.cuda.set_device(0)
        start.wait()
        bad = sum(L.smm_q4_matvec(*args, stream.cuda_stream) != _lib.SMM_OK for _ in range(20000))
        if bad:
            failed.append((bad, _lib.last_error()))

    jobs = []
    for i in range(6):
        cols = (8192, 4096)[i % 2]  # 128 and 64 KB for x: both above the 48 that need no leave
        q = torch.randint(0, 256, (16, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
        s = torch.rand(16, cols // 128, generator=g, device="cuda")
        x = rnd(g, 8, cols, dtype=BF)
        y = torch.empty(8, 16, device="cuda", dtype=BF)
        ref = ops.q4_matvec(q, s, x)
        args = (q.data_ptr(), s.data_ptr(), None, x.data_ptr(), y.data_ptr(), 8, 16, cols, 128, cols, 16,
                _lib.DTYPE_BF16, _lib.DTYPE_F32)
        jobs.append((args, torch.cuda.Stream(), y, ref, (q, s, x)))
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=j[:2]) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for _, _, y, ref, _ in jobs:
        assert torch.equal(y, ref)


# ---------------------------------------------------------------- padded batches
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,channels", [([0] * 70, 24), ([0] * 300 + [9, 0, 70] + [0] * 500, 40), ([3] + [0] * 90, 4352),
                                           ([64, 64, 0, 0, 64] + [0] * 33, 130), ([1, 0] * 120, 33)])
def test_many_empty_sequences(cuda, dtype, lens, channels):
    """Empty sequences in front, between and behind: their states pass through the convolution and the
    scan (zero where there is none), in place too, padded ones without a slot leave nothing."""
    dt = TYPES[dtype]
    b = offs(lens)
    k = len(lens)
    slots = torch.randperm(k, generator=torch.Generator().manual_seed(k)).tolist()
    for i in range(0, k, 3):
        slots[i] = -1
    x, w = rnd(gen(1), b[-1], channels, dtype=dt), rnd(gen(2), channels, 4, dtype=dt)
    st = rnd(gen(3), k, channels, 3, dtype=dt)
    start = torch.stack([st[s] if s >= 0 else torch.zeros_like(st[0]) for s in slots])
    ref, mag, final = conv_ref(x, w, None, b, start, True)
    live = [i for i in range(k) if slots[i] >= 0]
    rest = sorted(set(range(k)) - {slots[i] for i in live})
    where = [slots[i] for i in live]
    out = torch.full_like(st, 5.0)
    y = ops.causal_conv(x, w, offsets=i32(b), state=st, state_out=out, slots=i32(slots))
    within(y, ref, conv_tol(ref, mag, 4, dt), "y")
    assert torch.equal(out[where].double(), final[live]) and (out[rest] == 5).all()
    again = st.clone()
    assert torch.equal(ops.causal_conv(x, w, offsets=i32(b), state=again, slots=i32(slots)), y)
    assert torch.equal(again[where], out[where]) and torch.equal(again[rest], st[rest])
    out.fill_(5.0)
    ops.causal_conv(x, w, offsets=i32(b), state_out=out, slots=i32(slots))
    for i in live:
        if lens[i] == 0:
            assert (out[slots[i]] == 0).all()
    assert (out[rest] == 5).all()
    h, p, n = 2, 16, 8
    a = make_scan(4, b[-1], h, p, 1, n, dtype)
    ss = rnd(gen(5), k, h, p, n)
    start = torch.stack([ss[s] if s >= 0 else torch.zeros_like(ss[0]) for s in slots])
    ref, mag, (fin, fmag) = scan_ref(a, b, start)
    out = torch.full_like(ss, 5.0)
    y = ops.selective_scan(**a, offsets=i32(b), state=ss, state_out=out, slots=i32(slots))
    within(y, ref, scan_tol(ref, mag, n, max(lens), dt, dtype == "bf16"), "y")
    within(out[where], fin[live], state_tol(fin[live], fmag[live], max(lens), False), "state")
    assert (out[rest] == 5).all()
    ops.device_status()


# ---------------------------------------------------------------- 4-bit product: ranges
def q4_tol(ref, mag, cols, group, dtype):
    """As in test_q4_matches_definition."""
    steps = 2 * 24 + 2 * cols // min(group, 128) / 8 + 16
    return half_step(dtype) * ref.abs() * 1.01 + 2 * steps * U * mag + 1e-30


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("batch,group", [(1, 128), (8, 32), (12, 64)])
def test_q4_zero_points_up_to_127(cuda, dtype, batch, group):
    g = gen(group)
    x = rnd(g, batch, 512, dtype=TYPES[dtype])
    q = torch.randint(0, 256, (70, 256), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.rand(70, 512 // group, generator=g, device="cuda") * 0.02
    z = torch.randint(0, 128, s.shape, generator=g, device="cuda", dtype=torch.uint8)
    z[0], z[1], z[2], z[3] = 16, 127, 0, 15
    ref, mag = q4_ref(q, s, z, x)
    within(ops.q4_matvec(q, s, x, z), ref, q4_tol(ref, mag, 512, group, TYPES[dtype]))


def test_q4_keeps_every_nan(cuda):
    """Not-a-numbers whose payload lies in their low bits alone, beside an infinity."""
    g = gen(6)
    q = torch.randint(0, 256, (40, 64), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.rand(40, 1, generator=g, device="cuda") + 0.01
    x = rnd(g, 5, 128)
    clean = ops.q4_matvec(q, s, x)
    bits = x.view(torch.int32)
    for row, v in ((0, 0x7F800001), (1, -0x007FFFFF), (2, 0x7FC00000), (3, 0x7F800000)):
        bits[row, 9 * row + 4] = v
    y = ops.q4_matvec(q, s, x)
    assert y[:3].isnan().all()
    assert not y[3].isfinite().any() and torch.equal(y[4], clean[4])


# ---------------------------------------------------------------- C entries
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [128, 20, 7])
def test_step_entries_without_states(cuda, dtype, n):
    """No states at all (null pointers, no entries): every row starts from zero, and nothing is reported."""
    L = _lib.load()
    batch, h, p = 5, 3, 40
    ty = _lib.DTYPE_F32 if dtype == "fp32" else _lib.DTYPE_BF16
    a = make_scan(n, batch, h, p, 1, n, dtype, z=False, d=False, strided=False)
    pool = rnd(gen(1), batch, h, p, n)
    none = i32([-1] * batch)
    ref = ops.selective_step(**a, state=pool, slots=none)
    y = torch.full_like(ref, float("nan"))
    ops.device_status()
    rc = L.smm_selective_step(a["x"].data_ptr(), a["dt"].data_ptr(), a["A"].data_ptr(), a["B"].data_ptr(),
                              a["C"].data_ptr(), None, None, a["dt_bias"].data_ptr(), None, None, None, y.data_ptr(),
                              batch, 0, h, p, 1, n, h * p, h, n, n, 0, h * p, ty, ty, 1, None)
    assert rc == _lib.SMM_OK
    ops.device_status()
    assert torch.equal(y, ref)
    x, w = rnd(gen(2), batch, n, dtype=TYPES[dtype]), rnd(gen(3), n, 4, dtype=TYPES[dtype])
    cs = rnd(gen(4), batch, n, 3, dtype=TYPES[dtype])
    ref = ops.causal_conv_step(x, w, state=cs, slots=none)
    y = torch.full_like(ref, float("nan"))
    rc = L.smm_causal_conv_step(x.data_ptr(), w.data_ptr(), None, None, None, None, y.data_ptr(), batch, n, 4, 0, n, n,
                                ty, 1, None)
    assert rc == _lib.SMM_OK
    ops.device_status()
    assert torch.equal(y, ref)


# ---------------------------------------------------------------- streams
def test_strided_offsets_and_slots_on_another_stream(cuda):
    """Arguments that have to be copied are copied on the stream that the call runs on,
    however busy the current one is."""
    h, p, n = 2, 64, 128
    lens = [100, 30, 70]
    b = offs(lens)
    a = make_scan(1, b[-1], h, p, 1, n, "bf16")
    x = rnd(gen(2), b[-1], 64)
    w = rnd(gen(3), 64, 4)
    st, cs = rnd(gen(4), 4, h, p, n), rnd(gen(5), 4, 64, 3)
    one = {k: v[:3] if isinstance(v, torch.Tensor) and v.dim() > 1 else v for k, v in a.items()}
    off, sl = i32(b), i32([3, 0, 2])
    off2, sl2 = torch.stack([off, off * 0 + 7], 1)[:, 0], torch.stack([sl, sl * 0 + 1], 1)[:, 0]
    assert not off2.is_contiguous() and not sl2.is_contiguous()

    def calls(o, s, stream):
        kw = dict(stream=stream)
        so, co = torch.zeros_like(st), torch.zeros_like(cs)
        s1, c1 = st.clone(), cs.clone()
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
            torch.cuda._sleep(400_000_000)  # the current stream is busy from here on
        res = [ops.selective_scan(**a, offsets=o, state=st, state_out=so, slots=s, **kw), so,
               ops.causal_conv(x, w, offsets=o, state=cs, state_out=co, slots=s, **kw), co,
               ops.selective_step(**one, state=s1, slots=s, **kw), s1,
               ops.causal_conv_step(x[:3], w, state=c1, slots=s, **kw), c1]
        if stream is not None:
            stream.synchronize()
            res = [r.cpu() for r in res]
        return res

    ref = [r.cpu() for r in calls(off, sl, None)]
    got = calls(off2, sl2, torch.cuda.Stream())
    for r, v in zip(ref, got):
        assert torch.equal(r, v)


# ---------------------------------------------------------------- one matrix for all
@pytest.mark.parametrize("dtype,lens,h,n", [("bf16", [300, 41], 4, 64), ("bf16", [5, 2], 4, 64), ("fp32", [70, 30], 4, 20),
                                            ("bf16", [4200], 1, 128), ("fp32", [3000], 1, 32)])
def test_outputs_beside_inputs_in_one_matrix(cuda, dtype, lens, h, n):
    """out= as columns of the rows that hold the inputs: the result, and no other column changed."""
    dt, p = TYPES[dtype], 64
    b = offs(lens)
    t, hp = b[-1], h * p
    a = make_scan(9, t, h, p, 1, n, dtype, strided=False)
    ref = ops.selective_scan(**a, offsets=i32(b))
    widths = dict(x=hp, y=hp, B=n, C=n, z=hp, dt=8)
    m = rnd(gen(1), t, sum(widths.values()) + 8, dtype=dt)
    col, at = {}, 0
    for k, v in widths.items():
        col[k], at = m[:, at:at + v], at + v
    for k in ("x", "B", "C", "z"):
        col[k].copy_(a[k].reshape(t, -1))
    col["dt"][:, :h].copy_(a["dt"])
    keep = m.clone()
    args = dict(a, x=col["x"].unflatten(1, (h, p)), B=col["B"].unflatten(1, (1, n)), C=col["C"].unflatten(1, (1, n)),
                z=col["z"].unflatten(1, (h, p)), dt=col["dt"][:, :h])
    out = col["y"].unflatten(1, (h, p))
    ops.selective_scan(**args, offsets=i32(b), out=out)
    assert torch.equal(out, ref)
    keep[:, hp:2 * hp] = ref.view(t, hp)
    assert torch.equal(m, keep)
    st = rnd(gen(2), t, h, p, n)
    ops.selective_step(**args, state=st.clone(), out=out)
    keep[:, hp:2 * hp] = ops.selective_step(**a, state=st.clone()).view(t, hp)
    assert torch.equal(m, keep)
    w, cs = rnd(gen(3), hp, 4, dtype=dt), rnd(gen(4), t, hp, 3, dtype=dt)
    x = a["x"].reshape(t, hp)
    ops.causal_conv(col["x"], w, offsets=i32(b), out=col["y"])
    keep[:, hp:2 * hp] = ops.causal_conv(x, w, offsets=i32(b))
    assert torch.equal(m, keep)
    ops.causal_conv_step(col["x"], w, state=cs.clone(), out=col["y"])
    keep[:, hp:2 * hp] = ops.causal_conv_step(x, w, state=cs.clone())
    assert torch.equal(m, keep)
    q = torch.randint(0, 256, (hp, hp // 2), generator=gen(5), device="cuda", dtype=torch.uint8)
    s = torch.rand(hp, hp // 32, generator=gen(6), device="cuda")
    ops.q4_matvec(q, s, col["x"], out=col["y"])
    keep[:, hp:2 * hp] = ops.q4_matvec(q, s, x)
    assert torch.equal(m, keep)
    with pytest.raises(_lib.SmmError) as e:
        ops.causal_conv(col["x"], w, offsets=i32(b), out=m[:, hp - 1:2 * hp - 1])
    assert e.value.status == _lib.SMM_ERR_INVALID


# ---------------------------------------------------------------- long rows
@pytest.mark.parametrize("dtype,cols", [("fp32", 32768), ("bf16", 98304)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("batch,zeros", [(2, True), (11, False)])
def test_q4_rows_beyond_shared_memory(cuda, dtype, cols, group, batch, zeros):
    """Rows of x of which one fills the shared memory's share, and longer ones that are read beside the products."""
    for c in (cols, cols + group):
        g = gen(c)
        x = rnd(g, batch, c, dtype=TYPES[dtype])
        q = torch.randint(0, 256, (33, c // 2), generator=g, device="cuda", dtype=torch.uint8)
        s = torch.rand(33, c // group, generator=g, device="cuda") * 0.02
        z = torch.randint(0, 16, s.shape, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
        ref, mag = q4_ref(q, s, z, x)
        within(ops.q4_matvec(q, s, x, z), ref, q4_tol(ref, mag, c, group, TYPES[dtype]))


def test_q4_most_rows(cuda):
    """Nearly 2^31 rows of 32 columns: 34 GB of codes."""
    rows = (1 << 31) - 3
    q = torch.zeros(rows, 16, device="cuda", dtype=torch.uint8)
    s = torch.ones(rows, 1, device="cuda", dtype=BF)
    g = gen(8)
    some = (0, rows // 2, rows - 40)
    for r in some:
        q[r:r + 40] = torch.randint(0, 256, (40, 16), generator=g, device="cuda", dtype=torch.uint8)
        s[r:r + 40] = torch.rand(40, 1, generator=g, device="cuda").to(BF)
    x = rnd(g, 1, 32, dtype=BF)
    y = ops.q4_matvec(q, s, x)
    for r in some:
        ref, mag = q4_ref(q[r:r + 40], s[r:r + 40], None, x)
        within(y[:, r:r + 40], ref, q4_tol(ref, mag, 32, 32, BF))
    ref, mag = q4_ref(q[100:101], s[100:101], None, x)
    assert (y[:, 100:rows // 2] == y[:, 100:101]).all()
    within(y[:, 100:101], ref, q4_tol(ref, mag, 32, 32, BF))
