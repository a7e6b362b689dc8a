"""The state-space operators against their definitions in 64 bits.

Tolerances are derived from the roundings.  With u = 2^-24 and M the sum of the
magnitudes of an output's terms (computed beside it in 64 bits):
  - an fp32 chain of k operations on the terms is within k u M;
  - exp, log1p and the quotient of silu are within a few u relative, and an
    exponent's own error reaches the result as at most 0.37 times it (x exp(-x));
  - a product on the tensor cores whose operand was rounded to bf16 adds 2^-8 M,
    one whose operand is the sum of three bf16 terms 2^-27 M, and its 24 products of
    16 terms with truncated additions less than 2^-16 M;
  - the result's rounding is half a step of its type, eps/2.
"""
import pytest
import torch

from cpp1_b200 import _lib, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def offs(lens, start=0):
    o = [start]
    for n in lens:
        o.append(o[-1] + n)
    return o


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def within(got, ref, tol, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance, worst {float((err / tol).nan_to_num(1e9).max()):.3g} x"


# ---------------------------------------------------------------- convolution
def conv_ref(x, w, b, bounds, state, act):
    """(y, tolerance's magnitude, final states) in float64."""
    x, w = x.double(), w.double()
    c, width = w.shape
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    final = []
    for i, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
        head = state[i].double().t() if state is not None else x.new_zeros(width - 1, c)
        s = torch.cat([head, x[lo:hi]])
        for j in range(width):
            y[lo:hi] += s[j:j + hi - lo] * w[:, j]
            mag[lo:hi] += (s[j:j + hi - lo] * w[:, j]).abs()
        final.append(s[hi - lo:].t())
    if b is not None:
        y += b.double()
        mag += b.double().abs()
    return (y * torch.sigmoid(y) if act else y), mag, torch.stack(final) if final else None


def conv_tol(ref, mag, width, dtype):
    # 2 width operations per term; silu's slope is at most 1.1 and its own error 16 u relative
    return half_step(dtype) * ref.abs() * 1.01 + (1.1 * (2 * width + 2)) * U * mag + 16 * U * ref.abs() + 1e-30


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,channels,width", [
    ([1], 8, 4), ([0], 64, 4), ([0, 1, 2, 3, 0, 4, 5, 0], 96, 4), ([16, 15, 17, 1, 33], 1001, 3), ([200], 257, 2),
    ([5, 64, 3], 130, 8), ([31, 2], 48, 5), ([1, 7, 100], 520, 6), ([6, 7, 8], 16, 7), ([1500, 0, 700], 4352, 4),
])
@pytest.mark.parametrize("with_state", [False, True])
def test_conv_matches_definition(cuda, dtype, lens, channels, width, with_state):
    dt = TYPES[dtype]
    g = gen(channels * 10 + width)
    b = offs(lens)
    x, w = rnd(g, b[-1], channels, dtype=dt), rnd(g, channels, width, dtype=dt, scale=0.5)
    bias = rnd(g, channels, dtype=dt) if width % 2 == 0 else None
    st = rnd(g, len(lens), channels, width - 1, dtype=dt) if with_state else None
    act = "silu" if width != 3 else None
    ref, mag, final = conv_ref(x, w, bias, b, st, act)
    out_st = torch.full((len(lens), channels, width - 1), float("nan"), device="cuda", dtype=dt)
    y = ops.causal_conv(x, w, bias, offsets=i32(b), state=st, state_out=out_st, activation=act)
    within(y, ref, conv_tol(ref, mag, width, dt), "y")
    assert torch.equal(out_st.double(), final)
    if with_state:  # in place
        y2 = ops.causal_conv(x, w, bias, offsets=i32(b), state=st, activation=act)
        assert torch.equal(y2, y) and torch.equal(st, out_st)
    ops.device_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_conv_strides_slots_and_rows_outside(cuda, dtype):
    dt = TYPES[dtype]
    g = gen(7)
    lens, c, w = [9, 0, 40, 3], 24, 4
    b = offs(lens, start=5)
    base = torch.full((b[-1] + 11, 80), float("nan"), device="cuda", dtype=dt)
    base[5:b[-1], 8:8 + c] = rnd(g, b[-1] - 5, c, dtype=dt)
    x = base[:, 8:8 + c]
    wt = rnd(g, c, w, dtype=dt)
    pool = rnd(g, 6, c, w - 1, dtype=dt)
    slots = [4, 2, -1, 0]
    st = torch.stack([pool[s] if s >= 0 else torch.zeros_like(pool[0]) for s in slots])
    ref, mag, final = conv_ref(x.nan_to_num(0), wt, None, b, st, True)
    keep = pool.clone()
    out = torch.full((x.shape[0], 40), 3.0, device="cuda", dtype=dt)[:, :c]
    y = ops.causal_conv(x, wt, offsets=i32(b), state=pool, slots=i32(slots), out=out)
    assert y is out
    within(y[5:b[-1]], ref[5:b[-1]], conv_tol(ref, mag, w, dt)[5:b[-1]])
    assert (y[:5] == 3).all() and (y[b[-1]:] == 3).all()
    for i, s in enumerate(slots):
        if s >= 0:
            assert torch.equal(pool[s].double(), final[i])
            keep[s] = pool[s]
    assert torch.equal(keep, pool)
    # the same through a column layout that has to be copied, and unaligned rows
    xt = x[5:b[-1]].t().contiguous().t()
    y2 = ops.causal_conv(xt, wt, offsets=i32([v - 5 for v in b]), state=st.clone())
    assert torch.equal(y2, y[5:b[-1]])
    odd = torch.empty(b[-1] - 5, 2 * c + 1, device="cuda", dtype=dt)[:, 1:1 + c]
    odd.copy_(x[5:b[-1]])
    y3 = ops.causal_conv(odd, wt, offsets=i32([v - 5 for v in b]), state=st.clone())
    assert torch.equal(y3, y2)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("channels,width,batch", [(8, 4, 1), (4352, 4, 3), (33, 2, 5), (40, 8, 2), (1000, 3, 65)])
def test_conv_steps_continue_a_prompt(cuda, dtype, channels, width, batch):
    dt = TYPES[dtype]
    g = gen(channels)
    n = 7
    x, w = rnd(g, batch, n + 3, channels, dtype=dt), rnd(g, channels, width, dtype=dt)
    bias = rnd(g, channels, dtype=dt)
    st = torch.empty(batch, channels, width - 1, device="cuda", dtype=dt)
    b = i32([i * n for i in range(batch + 1)])
    ops.causal_conv(x[:, :n].reshape(-1, channels), w, bias, offsets=b, state_out=st)
    whole = ops.causal_conv(x.reshape(-1, channels), w, bias, offsets=i32([i * (n + 3) for i in range(batch + 1)]))
    whole = whole.view(batch, n + 3, channels)
    for j in range(3):
        nxt = torch.empty_like(st)
        y = ops.causal_conv_step(x[:, n + j], w, bias, state=st, state_out=nxt)
        assert torch.equal(y, whole[:, n + j])
        y2 = ops.causal_conv_step(x[:, n + j], w, bias, state=st)
        assert torch.equal(y2, y) and torch.equal(st, nxt)
    # a padded row takes no state and leaves none
    slots = i32([-1] * batch)
    keep = st.clone()
    y = ops.causal_conv_step(x[:, 0], w, bias, state=st, slots=slots)
    one = ops.causal_conv(x[:, 0].contiguous(), w, bias, offsets=i32(list(range(batch + 1))))
    assert torch.equal(y, one) and torch.equal(st, keep)


def test_conv_bad_slot_is_reported(cuda):
    x, w, st = torch.ones(2, 8, device="cuda"), torch.ones(8, 4, device="cuda"), torch.ones(2, 8, 3, device="cuda")
    ops.causal_conv_step(x, w, state=st, slots=i32([0, 2]))
    with pytest.raises(_lib.SmmError) as e:
        ops.device_status()
    assert e.value.status == _lib.SMM_ERR_BOUNDS
    ops.device_status()
    assert (st[1] == 1).all()


# ---------------------------------------------------------------- scan
def make_scan(seed, t, h, p, g_, n, dtype, z=True, d=True, dt_f32=False, strided=True):
    g = gen(seed)
    dt = TYPES[dtype]
    if strided:
        m = rnd(g, t, h * p + 2 * g_ * n, dtype=dt)
        x = m[:, :h * p].view(t, h, p)
        B = m[:, h * p:h * p + g_ * n].view(t, g_, n)
        C = m[:, h * p + g_ * n:].view(t, g_, n)
    else:
        x, B, C = rnd(g, t, h, p, dtype=dt), rnd(g, t, g_, n, dtype=dt), rnd(g, t, g_, n, dtype=dt)
    a = dict(x=x, dt=rnd(g, t, h, dtype=torch.float32 if dt_f32 else dt),
             A=-(0.5 + 15 * torch.rand(h, generator=g, device="cuda")), B=B, C=C,
             D=rnd(g, h) if d else None, z=rnd(g, t, h, p, dtype=dt) if z else None,
             dt_bias=rnd(g, h, scale=0.5) - 3.0, dt_softplus=True)
    return a


def scan_ref(a, bounds, state):
    """The recurrence in float64: y, magnitude of its terms, final states and theirs."""
    f = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    x = f["x"]
    t, h, p = x.shape
    per = h // f["B"].shape[1]
    d = f["dt"] + (f["dt_bias"] if f["dt_bias"] is not None else 0)
    if f["dt_softplus"]:
        d = torch.logaddexp(d, torch.zeros_like(d))
    dec = torch.exp(d * f["A"])
    B, C = f["B"].repeat_interleave(per, 1), f["C"].repeat_interleave(per, 1)
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    fin, fmag = [], []
    for i, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
        s = state[i].double().clone() if state is not None else x.new_zeros(h, p, B.shape[2])
        m = s.abs()
        for j in range(lo, hi):
            add = (d[j][:, None] * x[j])[:, :, None] * B[j][:, None, :]
            s = s * dec[j][:, None, None] + add
            m = m * dec[j][:, None, None] + add.abs()
            y[j] = torch.einsum("hpn,hn->hp", s, C[j])
            mag[j] = torch.einsum("hpn,hn->hp", m, C[j].abs())
        fin.append(s)
        fmag.append(m)
    if f["D"] is not None:
        y += f["D"][:, None] * x
        mag += (f["D"][:, None] * x).abs()
    if f["z"] is not None:
        gate = f["z"] * torch.sigmoid(f["z"])
        y, mag = y * gate, mag * gate.abs()
    return y, mag, (torch.stack(fin), torch.stack(fmag)) if fin else None


def scan_tol(ref, mag, n, longest, dtype, tensor):
    """fp32 recurrence: 3 roundings a token and an exp of 3 u, n + 2 additions, exponents
    and softplus 2^-19; on the tensor cores two operands rounded to bf16."""
    fp = (6 * longest + 2 * n + 8) * U + 2.0 ** -19
    return half_step(dtype) * ref.abs() * 1.01 + (fp + (2.0 ** -8 * 1.01 if tensor else 0)) * mag + 1e-30


def state_tol(ref, mag, longest, tensor):
    return ((6 * longest + 8) * U + 2.0 ** -19 + (2.0 ** -16 if tensor else 0)) * mag + 1e-30


SCAN_CASES = [
    # lens, heads, dim, groups, state_dim
    ([1], 1, 1, 1, 1), ([3], 2, 64, 1, 128), ([0], 2, 16, 1, 8), ([0, 5, 0, 1, 17], 4, 48, 2, 16),
    ([16, 15, 33], 3, 33, 1, 20), ([70, 2], 6, 64, 3, 64), ([40], 2, 128, 1, 32), ([21, 19], 2, 256, 2, 256),
    ([128], 4, 64, 1, 128), ([127, 129, 1, 0, 256], 4, 64, 2, 128), ([300, 100], 8, 64, 8, 64),
    ([513], 2, 128, 1, 128), ([200, 131], 3, 96, 1, 96), ([260], 5, 40, 1, 24), ([129], 2, 64, 1, 256),
    ([1000], 2, 64, 1, 128), ([64] * 9, 2, 32, 1, 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,h,p,g_,n", SCAN_CASES)
@pytest.mark.parametrize("with_state", [False, True])
def test_scan_matches_definition(cuda, dtype, lens, h, p, g_, n, with_state):
    b = offs(lens)
    seed = h * 1000 + p + n
    a = make_scan(seed, b[-1], h, p, g_, n, dtype, z=h % 2 == 0, d=h != 3, dt_f32=p == 48, strided=p % 32 != 0)
    st = rnd(gen(seed + 1), len(lens), h, p, n) if with_state else None
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.full((len(lens), h, p, n), float("nan"), device="cuda")
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    tensor = dtype == "bf16"
    longest = max(max(lens), 1)
    within(y, ref, scan_tol(ref, mag, n, longest, TYPES[dtype], tensor), "y")
    within(so, fin, state_tol(fin, fmag, longest, tensor), "state")
    y2 = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=st)
    assert torch.equal(y2, y)
    if with_state:
        assert torch.equal(st, so)
    ops.device_status()


@pytest.mark.parametrize("dtype,h,p,n,t", [("fp32", 1, 64, 128, 3000), ("fp32", 2, 16, 16, 5001), ("bf16", 1, 64, 128, 6000),
                                           ("bf16", 3, 64, 64, 4097), ("bf16", 1, 8, 8, 4000)])
def test_long_sequences_are_split(cuda, dtype, h, p, n, t):
    """Few heads and many tokens: segments, with states passed between them; in place too."""
    lens = [t, 0, t // 3]
    b = offs(lens)
    assert _lib.load().smm_selective_scan_workspace_size(b[-1], 3, h, p, 1, n, 0 if dtype == "fp32" else 1) > 0
    a = make_scan(t, b[-1], h, p, 1, n, dtype)
    st = rnd(gen(1), 4, h, p, n)
    slots = [3, 0, 2]
    ref, mag, (fin, fmag) = scan_ref(a, b, st[slots])
    keep = st.clone()
    so = torch.zeros_like(st)
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so, slots=i32(slots))
    assert torch.equal(st, keep)
    within(y, ref, scan_tol(ref, mag, n, t, TYPES[dtype], dtype == "bf16"), "y")
    within(so[slots], fin, state_tol(fin, fmag, t, dtype == "bf16"), "state")
    y2 = ops.selective_scan(**a, offsets=i32(b), state=st, slots=i32(slots))
    assert torch.equal(y2, y) and torch.equal(st[slots], so[slots]) and torch.equal(st[1], keep[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_scan_rows_outside_and_slots(cuda, dtype):
    """NaN and infinities around the sequences, sequences without a state, rows left alone."""
    lens, h, p, g_, n = [150, 0, 20, 129], 2, 64, 1, 128
    b = offs(lens, start=3)
    t = b[-1] + 140
    a = make_scan(5, t, h, p, g_, n, dtype, strided=False)
    clean = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    for k, bad in (("x", float("nan")), ("B", float("inf")), ("C", float("-inf")), ("dt", float("nan")),
                   ("z", float("nan"))):
        a[k][:3] = bad
        a[k][b[-1]:] = bad
    pool = rnd(gen(9), 5, h, p, n)
    slots = [4, 1, -1, 0]
    st = torch.stack([pool[s] if s >= 0 else torch.zeros_like(pool[0]) for s in slots])
    ref, mag, (fin, fmag) = scan_ref(clean, b, st)
    out = torch.full((t, h, p), 3.0, device="cuda", dtype=TYPES[dtype])
    keep = pool.clone()
    ops.selective_scan(**a, offsets=i32(b), state=pool, slots=i32(slots), out=out)
    tensor = dtype == "bf16"
    tol = scan_tol(ref, mag, n, 150, TYPES[dtype], tensor)
    within(out[3:b[-1]], ref[3:b[-1]], tol[3:b[-1]], "y")
    assert (out[:3] == 3).all() and (out[b[-1]:] == 3).all()
    for i, s in enumerate(slots):
        if s >= 0:
            within(pool[s], fin[i], state_tol(fin[i], fmag[i], 150, tensor), f"state {s}")
            keep[s] = pool[s]
    assert torch.equal(keep, pool)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_nan_stays_in_its_sequence(cuda, dtype):
    """One sequence's NaN reaches neither its neighbours nor its own tokens a tile before."""
    lens, h, p, n = [140, 70, 300], 2, 64, 128
    b = offs(lens)
    a = make_scan(6, b[-1], h, p, 1, n, dtype, strided=False)
    good = ops.selective_scan(**a, offsets=i32(b))
    a["x"][b[1] + 10] = float("nan")
    a["B"][b[2] + 290, 0, 3] = float("inf")
    so = torch.empty(3, h, p, n, device="cuda")
    y = ops.selective_scan(**a, offsets=i32(b), state_out=so)
    assert torch.equal(y[:b[1]], good[:b[1]])
    assert y[b[1] + 10:b[2]].isnan().all() and so[1].isnan().all()
    assert torch.equal(y[b[2]:b[2] + 290 - 127], good[b[2]:b[2] + 290 - 127])
    assert so[0].isfinite().all() and not so[2][:, :, 3].isfinite().any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_extreme_decays(cuda, dtype):
    """d of zero (a token that does nothing), of 20 and more (softplus' linear part) and of
    e^-30; A of zero (no decay) and of -1000 (nothing is kept)."""
    t, h, p, n = 300, 4, 64, 128
    a = make_scan(8, t, h, p, 1, n, dtype, strided=False)
    a["A"] = torch.tensor([0.0, -1000.0, -1e-6, -3.0], device="cuda")
    a["dt"][::7] = -30.0
    a["dt"][3::50] = 25.0
    b = [0, t]
    ref, mag, (fin, fmag) = scan_ref(a, b, None)
    so = torch.empty(1, h, p, n, device="cuda")
    y = ops.selective_scan(**a, state_out=so)
    tensor = dtype == "bf16"
    within(y, ref, scan_tol(ref, mag, n, t, TYPES[dtype], tensor), "y")
    within(so, fin, state_tol(fin, fmag, t, tensor), "state")
    a["dt_softplus"], a["dt_bias"] = False, None
    a["dt"].zero_()
    a["dt"][100] = 0.5
    st = rnd(gen(3), 1, h, p, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    y = ops.selective_scan(**a, state=st, state_out=so)
    within(y, ref, scan_tol(ref, mag, n, t, TYPES[dtype], tensor), "y")
    within(so, fin, state_tol(fin, fmag, t, tensor), "state")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("batch,h,p,g_,n", [(1, 64, 64, 1, 128), (5, 6, 48, 2, 16), (3, 2, 33, 1, 20), (2, 2, 256, 1, 256),
                                            (7, 1, 1, 1, 1), (2, 4, 64, 4, 200), (3, 2, 30, 1, 33), (33, 8, 64, 8, 64)])
def test_step_matches_definition(cuda, dtype, batch, h, p, g_, n):
    a = make_scan(batch + n, batch, h, p, g_, n, dtype, z=h != 6, d=h != 8, dt_f32=h == 2)
    st = rnd(gen(n), batch, h, p, n)
    ref, mag, (fin, fmag) = scan_ref(a, list(range(batch + 1)), st)
    so = torch.empty_like(st)
    y = ops.selective_step(**a, state=st, state_out=so)
    within(y, ref, scan_tol(ref, mag, n, 1, TYPES[dtype], False), "y")
    within(so, fin, state_tol(fin, fmag, 1, False), "state")
    pool = rnd(gen(2), batch + 2, h, p, n)
    perm = torch.randperm(batch + 2, generator=torch.Generator().manual_seed(0))[:batch].tolist()
    pool[perm] = st
    keep = pool.clone()
    y2 = ops.selective_step(**a, state=pool, slots=i32(perm))
    assert torch.equal(y2, y) and torch.equal(pool[perm], so)
    keep[perm] = so
    assert torch.equal(keep, pool)
    # a padded row: from zero, leaving nothing
    y3 = ops.selective_step(**a, state=pool, slots=i32([-1] * batch))
    ref, mag, _ = scan_ref(a, list(range(batch + 1)), None)
    within(y3, ref, scan_tol(ref, mag, n, 1, TYPES[dtype], False), "y")
    assert torch.equal(keep, pool)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("batch,h,p,g_,n", [(60, 64, 64, 8, 128), (70, 48, 50, 2, 100), (40, 64, 40, 1, 200), (150, 40, 64, 1, 16),
                                            (50, 64, 72, 4, 36), (3, 300, 64, 1, 64), (90, 64, 33, 1, 45)])
def test_step_over_many_tiles(cuda, dtype, batch, h, p, g_, n):
    """States that every warp walks several tiles of, some without a slot."""
    a = make_scan(batch + n, batch, h, p, g_, n, dtype)
    pool = rnd(gen(n), batch, h, p, n)
    keep = pool.clone()
    slots = torch.randperm(batch, generator=torch.Generator().manual_seed(1))
    slots[batch // 2] = -1
    st = pool[slots]
    st[batch // 2] = 0
    ref, mag, (fin, fmag) = scan_ref(a, list(range(batch + 1)), st)
    y = ops.selective_step(**a, state=pool, slots=i32(slots.tolist()))
    within(y, ref, scan_tol(ref, mag, n, 1, TYPES[dtype], False), "y")
    live = slots >= 0
    within(pool[slots[live]], fin[live], state_tol(fin[live], fmag[live], 1, False), "state")
    keep[slots[live]] = pool[slots[live]]
    assert torch.equal(keep, pool)


@pytest.mark.parametrize("dtype,lens,h,g_,n,gate", [
    ("bf16", [700, 37, 260], 160, 8, 128, True), ("bf16", [130, 900, 1, 0, 128], 200, 1, 64, False),
    ("bf16", [60] * 40, 24, 3, 128, True), ("bf16", [9] * 30, 64, 1, 16, True), ("bf16", [300] * 6, 64, 1, 16, True),
    ("fp32", [500, 37, 130], 160, 8, 128, True), ("fp32", [200] * 5, 64, 2, 64, False), ("fp32", [400], 16, 1, 128, True)])
def test_scan_on_every_sm_repeats_itself(cuda, dtype, lens, h, g_, n, gate):
    """All SMs at work, several items to each: right, and the same bits every time."""
    b = offs(lens)
    a = make_scan(h + n, b[-1], h, 64, g_, n, dtype, z=gate)
    st = rnd(gen(h), len(lens), h, 64, n)
    ref, mag, (fin, fmag) = scan_ref(a, b, st)
    so = torch.empty_like(st)
    y = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so)
    tensor = dtype == "bf16"
    within(y, ref, scan_tol(ref, mag, n, max(lens), TYPES[dtype], tensor), "y")
    within(so, fin, state_tol(fin, fmag, max(lens), tensor), "state")
    for _ in range(20):
        so2 = torch.empty_like(st)
        y2 = ops.selective_scan(**a, offsets=i32(b), state=st, state_out=so2)
        assert torch.equal(y2, y) and torch.equal(so2, so)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,channels,width", [([3, 130, 64, 1, 0, 65, 7000], 4352, 4), ([4000, 63, 65, 2500, 500], 4400, 8),
                                                 ([7129], 4354, 2)])
def test_conv_long_runs(cuda, dtype, lens, channels, width):
    dt = TYPES[dtype]
    g = gen(channels)
    b = offs(lens)
    x, w, bias = rnd(g, b[-1], channels, dtype=dt), rnd(g, channels, width, dtype=dt), rnd(g, channels, dtype=dt)
    st = rnd(g, len(lens), channels, width - 1, dtype=dt)
    ref, mag, final = conv_ref(x, w, bias, b, st, True)
    y = ops.causal_conv(x, w, bias, offsets=i32(b), state=st)
    within(y, ref, conv_tol(ref, mag, width, dt), "y")
    assert torch.equal(st.double(), final)


def test_step_bad_slot_is_reported(cuda):
    a = make_scan(1, 3, 2, 16, 1, 8, "fp32")
    st = rnd(gen(1), 3, 2, 16, 8)
    keep = st.clone()
    y = ops.selective_step(**a, state=st, slots=i32([3, 1, 1 << 30]))
    assert y.isfinite().all()
    with pytest.raises(_lib.SmmError) as e:
        ops.device_status()
    assert e.value.status == _lib.SMM_ERR_BOUNDS
    assert torch.equal(st[0], keep[0]) and torch.equal(st[2], keep[2])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_bad_offsets_stay_in_bounds(cuda, dtype):
    """Offsets that decrease or leave the rows: some result, no access outside."""
    a = make_scan(1, 300, 2, 64, 1, 128, dtype)
    for o in ([0, 400, 500], [-7, 100, 50], [290, 10, 1 << 30], [0, 0, 0]):
        out = torch.zeros(300, 2, 64, device="cuda", dtype=TYPES[dtype])
        so = torch.zeros(2, 2, 64, 128, device="cuda")
        ops.selective_scan(**a, offsets=i32(o), state_out=so, out=out)
        x = a["x"].reshape(300, 128)
        ops.causal_conv(x, torch.ones(128, 4, device="cuda", dtype=x.dtype), offsets=i32(o))
    ops.device_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_overlapping_sequences_of_a_split_scan_stay_in_bounds(cuda, dtype):
    """Offsets that decrease can count more segments than the workspace holds."""
    t, h, n = 6000, 1, 128
    a = make_scan(2, t, h, 64, 1, n, dtype)
    for o in ([0, t, 10, t], [0, t, 0, t, 0, t], [t, 0, t, 0]):
        nseq = len(o) - 1
        assert _lib.load().smm_selective_scan_workspace_size(t, nseq, h, 64, 1, n, 0 if dtype == "fp32" else 1) > 0
        so = torch.zeros(nseq, h, 64, n, device="cuda")
        ops.selective_scan(**a, offsets=i32(o), state=rnd(gen(1), nseq, h, 64, n), state_out=so)
    ops.device_status()
    ref = ops.selective_scan(**a)
    assert ref.isfinite().all()


def test_no_sequences_and_no_tokens(cuda):
    a = make_scan(1, 0, 2, 64, 1, 128, "bf16")
    st = rnd(gen(1), 1, 2, 64, 128)
    so = torch.zeros_like(st)
    assert ops.selective_scan(**a, state=st, state_out=so).shape == (0, 2, 64)
    assert torch.equal(so, st)
    w = torch.ones(128, 4, device="cuda", dtype=torch.bfloat16)
    cs = rnd(gen(1), 1, 128, 3, dtype=torch.bfloat16)
    co = torch.zeros_like(cs)
    assert ops.causal_conv(a["x"].reshape(0, 128), w, state=cs, state_out=co).shape == (0, 128)
    assert torch.equal(co, cs)
    a = make_scan(1, 5, 2, 64, 1, 128, "bf16")
    out = torch.full((5, 2, 64), 2.0, device="cuda", dtype=torch.bfloat16)
    ops.selective_scan(**a, offsets=i32([0]), out=out)
    assert (out == 2).all()


# ---------------------------------------------------------------- 4-bit
def q4_ref(q, s, z, x):
    codes = torch.stack([q & 15, q >> 4], 2).reshape(q.shape[0], -1).double()
    grp = codes.shape[1] // s.shape[1]
    zero = z.double().repeat_interleave(grp, 1) if z is not None else 8.0
    w = (codes - zero) * s.double().repeat_interleave(grp, 1)
    return x.double() @ w.t(), x.double().abs() @ w.abs().t()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("batch,rows,cols,group,zeros,sf32", [
    (1, 1, 32, 32, False, False), (1, 16, 128, 128, True, True), (2, 17, 64, 64, True, False), (8, 250, 1024, 32, False, True),
    (9, 33, 4096, 256, True, False), (1, 1000, 8192, 128, False, False), (16, 64, 640, 64, True, True), (3, 100, 96, 96, True, False),
    (33, 40, 384, 128, False, False), (70, 129, 1280, 64, True, False), (5, 48, 12288, 4096, False, True),
])
def test_q4_matches_definition(cuda, dtype, batch, rows, cols, group, zeros, sf32):
    dt = TYPES[dtype]
    g = gen(rows + cols)
    x = rnd(g, batch, cols, dtype=dt)
    q = torch.randint(0, 256, (rows, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand(rows, cols // group, generator=g, device="cuda") * 0.02 - 0.005).to(torch.float32 if sf32 else dt)
    z = torch.randint(0, 16, s.shape, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    ref, mag = q4_ref(q, s, z, x)
    y = ops.q4_matvec(q, s, x, z)
    # exact products; a tensor-core sum truncates to 2^-23 of its largest term at each of up to
    # 2 (bf16) or 6 (fp32) additions per 32 columns of a 128-column run, then fp32 additions over the runs
    steps = 2 * 24 + 2 * cols // min(group, 128) / 8 + 16
    within(y, ref, half_step(dt) * ref.abs() * 1.01 + 2 * steps * U * mag + 1e-30)
    assert torch.equal(ops.q4_matvec(q, s, x, z), y)


def test_q4_strides_and_range(cuda):
    g = gen(4)
    q = torch.randint(0, 256, (40, 64), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.rand(40, 1, generator=g, device="cuda")
    base = rnd(g, 6, 200)
    for x in (base[:, 8:136], base[:, 3:131], base[:5, 4:132:1], base[:, :128].t().contiguous().t()):
        y = ops.q4_matvec(q, s, x)
        assert torch.equal(y, ops.q4_matvec(q, s, x.clone(memory_format=torch.contiguous_format)))
    out = torch.full((6, 50), 7.0, device="cuda")
    ops.q4_matvec(q, s, base[:, :128], out=out[:, :40])
    assert torch.equal(out[:, :40], ops.q4_matvec(q, s, base[:, :128])) and (out[:, 40:] == 7).all()
    # fp32's whole range: the three terms are exact, and infinities stay infinities
    x = torch.zeros(3, 128, device="cuda")
    x[0, 5], x[1, 7], x[2, 9] = 3.3e38, float("inf"), 1.1754944e-38
    w = (torch.stack([q & 15, q >> 4], 2).reshape(40, 128).double() - 8) * s.double()
    y = ops.q4_matvec(q, s, x * torch.tensor([[0.01], [1.0], [1.0]], device="cuda"))
    ref = (x[0, 5] * 0.01).double() * w[:, 5]
    within(y[0], ref, 16 * U * ref.abs())
    pos = w[:, 7] != 0
    assert (y[1][pos] == torch.sign(w[pos, 7]) * float("inf")).all() and y[1][~pos].isnan().all()
    ref = x[2, 9].double() * w[:, 9]
    within(y[2], ref, 16 * U * ref.abs() + 2.0 ** -149)


# ---------------------------------------------------------------- together
def block(m, x, conv_state, ssm_state, step, offsets=None):
    """One state-space block: projections in 4 bits, convolution, scan, gate."""
    h, p, g_, n = m["shape"]
    hp, gn = h * p, g_ * n
    row = ops.q4_matvec(m["qin"], m["sin"], x)
    z, xbc, dt = row[:, :hp], row[:, hp:2 * hp + 2 * gn], row[:, 2 * hp + 2 * gn:]
    if step:
        u = ops.causal_conv_step(xbc, m["cw"], m["cb"], state=conv_state)
    else:
        u = ops.causal_conv(xbc, m["cw"], m["cb"], offsets=offsets, state=conv_state)
    t = x.shape[0]
    kw = dict(D=m["D"], z=z.unflatten(1, (h, p)), dt_bias=m["db"], dt_softplus=True, state=ssm_state)
    args = (u[:, :hp].unflatten(1, (h, p)), dt, m["A"], u[:, hp:hp + gn].unflatten(1, (g_, n)),
            u[:, hp + gn:].unflatten(1, (g_, n)))
    y = ops.selective_step(*args, **kw) if step else ops.selective_scan(*args, offsets=offsets, **kw)
    return ops.q4_matvec(m["qout"], m["sout"], y.view(t, hp))


def make_block(dtype, h=4, p=64, g_=1, n=64, width=256):
    g = gen(11)
    hp, gn = h * p, g_ * n
    rows = 2 * hp + 2 * gn + h
    dt = TYPES[dtype]
    return dict(shape=(h, p, g_, n),
                qin=torch.randint(0, 256, (rows, width // 2), generator=g, device="cuda", dtype=torch.uint8),
                sin=(torch.rand(rows, width // 64, generator=g, device="cuda") * 0.02).to(dt),
                qout=torch.randint(0, 256, (width, hp // 2), generator=g, device="cuda", dtype=torch.uint8),
                sout=(torch.rand(width, hp // 64, generator=g, device="cuda") * 0.02).to(dt),
                cw=rnd(g, hp + 2 * gn, 4, dtype=dt, scale=0.5), cb=rnd(g, hp + 2 * gn, dtype=dt, scale=0.1),
                A=-(1 + 4 * torch.rand(h, generator=g, device="cuda")), D=rnd(g, h), db=rnd(g, h) - 2)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_block_prompt_then_tokens(cuda, dtype):
    """A prompt and then single tokens, through captured graphs as a server replays them,
    give what the whole text gives as one prompt."""
    m = make_block(dtype)
    h, p, g_, n = m["shape"]
    c = h * p + 2 * g_ * n
    lens, extra = [37, 130, 1], 5
    g = gen(12)
    texts = [rnd(g, k + extra, 256, dtype=TYPES[dtype]) for k in lens]
    conv, ssm = torch.zeros(3, c, 3, device="cuda", dtype=TYPES[dtype]), torch.zeros(3, h, p, n, device="cuda")
    whole = block(m, torch.cat(texts), conv.clone(), ssm.clone(), False, i32(offs([k + extra for k in lens])))
    whole = torch.split(whole, [k + extra for k in lens])
    first = torch.split(block(m, torch.cat([t[:k] for t, k in zip(texts, lens)]), conv, ssm, False, i32(offs(lens))), lens)
    # relative to the outputs' size: the roundings to the type at each of the four steps, twice
    eps = 16 * half_step(TYPES[dtype]) if dtype == "bf16" else 1e-4

    def close(a, b):
        assert float((a.double() - b.double()).norm()) <= eps * float(b.double().norm())

    for a, b, k in zip(first, whole, lens):
        close(a, b[:k])
    tok = torch.stack([t[k] for t, k in zip(texts, lens)])
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        block(m, tok, conv.clone(), ssm.clone(), True)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(m, tok, conv, ssm, True)
    for j in range(extra):
        tok.copy_(torch.stack([t[k + j] for t, k in zip(texts, lens)]))
        graph.replay()
        close(y, torch.stack([b[k + j] for b, k in zip(whole, lens)]))
    ops.device_status()


def test_two_captured_scans_and_a_side_stream(cuda):
    """Graphs of split scans share no workspace: replayed on two streams at once
    they give what each gives alone; so does an explicit stream argument."""
    calls = []
    for seed in (1, 2):
        a = make_scan(seed, 5000, 2, 64, 1, 128, "bf16")
        calls.append((a, ops.selective_scan(**a)))
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for a, _ in calls:
        gph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gph):
            outs.append(ops.selective_scan(**a))
        graphs.append(gph)
    torch.cuda.synchronize()
    for _ in range(3):
        for gph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gph.replay()
    torch.cuda.synchronize()
    for (_, ref), o in zip(calls, outs):
        assert torch.equal(ref, o)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y = ops.selective_scan(**calls[0][0], stream=s)
    s.synchronize()
    assert torch.equal(y, calls[0][1])


def test_offsets_beyond_32_bits(cuda):
    """Slots, rows and columns whose element offsets pass 2^32."""
    h, p, n = 8, 64, 128
    entries = (1 << 32) // (h * p * n) + 3
    pool = torch.empty(entries, h, p, n, device="cuda")
    pool[-1].normal_()
    st = pool[-1].clone()
    a = make_scan(3, 1, h, p, 1, n, "bf16")
    so = torch.empty(1, h, p, n, device="cuda")
    ref = ops.selective_step(**a, state=st[None], state_out=so)
    y = ops.selective_step(**a, state=pool, slots=i32([entries - 1]))
    assert torch.equal(y, ref) and torch.equal(pool[-1], so[0])
    pool[-1] = st
    ref = ops.selective_scan(**a, state=st[None], state_out=so)
    y = ops.selective_scan(**a, state=pool, slots=i32([entries - 1]))
    assert torch.equal(y, ref) and torch.equal(pool[-1], so[0])
    del pool
    wide = torch.empty(3, (1 << 31) + 64, device="cuda", dtype=torch.bfloat16)
    x = wide[:, -512:].view(3, 8, 64)
    small = rnd(gen(1), 3, 8, 64, dtype=torch.bfloat16)
    x.copy_(small)
    a = make_scan(4, 3, 8, 64, 1, 128, "bf16")
    a["x"] = small
    ref = ops.selective_scan(**a)
    a["x"] = x
    assert torch.equal(ops.selective_scan(**a), ref)
    w = rnd(gen(2), 512, 4, dtype=torch.bfloat16)
    assert torch.equal(ops.causal_conv(wide[:, -512:], w), ops.causal_conv(small.view(3, 512), w))
