"""The operators of a state-space block, as they are measured.

Three operators in five calls, on the shapes a served language model meets:

  conv       short causal convolution of packed prompts (a banded
             lower-triangular Toeplitz matrix per channel)
  conv_step  the same for one new token of each sequence
  scan       selective state space scan of packed prompts (a lower-triangular
             semiseparable matrix per head)
  step       the same for one new token of each sequence
  q4         a few activations times a matrix held in 4 bits with group scales

``run`` computes them either in plain torch operations (32 bits throughout,
rounded once at the end) or, with ``own`` set, through cpp1_b200.ops.
``exact`` computes them from their definitions in 64 bits.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one long prompt, the convolved channels of 64 heads of 64 and one group of 128
        {"name": "conv_prompt", "kind": "conv", "dtype": "bf16", "tokens": 8192, "seqs": 1, "cut": 0,
         "channels": 4352, "width": 4, "bias": True, "state": True},
        # a batch of short ragged prompts in fp32, odd channel count
        {"name": "conv_ragged", "kind": "conv", "dtype": "fp32", "tokens": 3001, "seqs": 17, "cut": 1,
         "channels": 1001, "width": 3, "bias": False, "state": True},
        # one token of one sequence: latency
        {"name": "conv_step_one", "kind": "conv_step", "dtype": "bf16", "batch": 1, "channels": 4352, "width": 4,
         "bias": True},
        # one token of each sequence of a full batch
        {"name": "conv_step_batch", "kind": "conv_step", "dtype": "bf16", "batch": 192, "channels": 8448, "width": 4,
         "bias": True},
        # one prompt of ordinary length
        {"name": "scan_prompt", "kind": "scan", "dtype": "bf16", "tokens": 4096, "seqs": 1, "cut": 0, "heads": 64,
         "dim": 64, "groups": 1, "state_dim": 128, "gate": True, "state": False},
        # a batch of ragged prompts that continue from kept states
        {"name": "scan_ragged", "kind": "scan", "dtype": "bf16", "tokens": 8190, "seqs": 24, "cut": 2, "heads": 32,
         "dim": 64, "groups": 4, "state_dim": 64, "gate": False, "state": True},
        # the longest prompt, wide heads' groups
        {"name": "scan_long", "kind": "scan", "dtype": "bf16", "tokens": 32768, "seqs": 1, "cut": 0, "heads": 80,
         "dim": 64, "groups": 8, "state_dim": 128, "gate": True, "state": True},
        # full precision, odd sizes
        {"name": "scan_fp32", "kind": "scan", "dtype": "fp32", "tokens": 1023, "seqs": 5, "cut": 3, "heads": 13,
         "dim": 48, "groups": 1, "state_dim": 16, "gate": True, "state": True},
        # one token of one sequence: latency
        {"name": "step_one", "kind": "step", "dtype": "bf16", "batch": 1, "heads": 64, "dim": 64, "groups": 1,
         "state_dim": 128, "gate": True},
        # one token of each sequence of a full batch: the states' traffic
        {"name": "step_batch", "kind": "step", "dtype": "bf16", "batch": 160, "heads": 64, "dim": 64, "groups": 8,
         "state_dim": 128, "gate": True},
        # one token through a projection
        {"name": "q4_one", "kind": "q4", "dtype": "bf16", "batch": 1, "rows": 8192, "cols": 4096, "group": 128,
         "zeros": False},
        # a small batch through a larger projection with zero points and finer groups
        {"name": "q4_batch", "kind": "q4", "dtype": "bf16", "batch": 8, "rows": 8200, "cols": 8192, "group": 64,
         "zeros": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    groups = rng.choice([1, 1, 2, 4, 8])
    return groups * rng.randint(1, 80 // groups), groups


def draw(rng):
    kind = rng.choice(["conv", "conv_step", "scan", "scan", "step", "q4", "q4"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "conv":
        t = _log(rng, 1, 8192)
        return {"kind": kind, "dtype": dtype, "tokens": t, "seqs": _log(rng, 1, min(64, t)),
                "cut": rng.randrange(1 << 20), "channels": _log(rng, 64, 4352 if dtype == "bf16" else 2176),
                "width": rng.choice([2, 3, 4, 4]), "bias": rng.random() < 0.5, "state": rng.random() < 0.5}
    if kind == "conv_step":
        return {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, 256), "channels": _log(rng, 64, 8448),
                "width": rng.choice([2, 3, 4, 4]), "bias": rng.random() < 0.5}
    if kind == "scan":
        heads, groups = _heads(rng)
        t = _log(rng, 1, 16384 if dtype == "bf16" else 4096)
        return {"kind": kind, "dtype": dtype, "tokens": t, "seqs": _log(rng, 1, min(48, t)),
                "cut": rng.randrange(1 << 20), "heads": heads, "dim": rng.choice([32, 48, 64, 64, 64, 128]),
                "groups": groups, "state_dim": rng.choice([16, 32, 64, 128, 128]), "gate": rng.random() < 0.5,
                "state": rng.random() < 0.5}
    if kind == "step":
        heads, groups = _heads(rng)
        return {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, 128), "heads": heads,
                "dim": rng.choice([32, 48, 64, 64, 64]), "groups": groups,
                "state_dim": rng.choice([16, 32, 64, 128, 128]), "gate": rng.random() < 0.5}
    group = rng.choice([32, 64, 128, 128])
    return {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, 16), "rows": _log(rng, 256, 16384),
            "cols": group * _log(rng, 1024 // group, 8192 // group), "group": group, "zeros": rng.random() < 0.5}


def _offsets(case):
    """Sequence boundaries: `seqs` random cuts of `tokens` (ragged, some may be empty)."""
    t, s = case["tokens"], case["seqs"]
    g = torch.Generator().manual_seed(case["cut"])
    cuts = torch.randint(0, t + 1, (s - 1,), generator=g).sort().values.tolist()
    return [0] + cuts + [t]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    dt = _DT[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    kind = case["kind"]
    s = {"kind": kind, "case": case}
    if kind in ("conv", "conv_step"):
        c, w = case["channels"], case["width"]
        n = case["tokens"] if kind == "conv" else case["batch"]
        s["x"] = randn(n, c)
        s["weight"] = randn(c, w, scale=w ** -0.5)
        s["bias"] = randn(c, scale=0.1) if case["bias"] else None
        seqs = case["seqs"] if kind == "conv" else n
        keep = kind == "conv_step" or case["state"]
        s["state"] = randn(seqs, c, w - 1) if keep else None
        s["state_out"] = torch.empty(seqs, c, w - 1, device=dev, dtype=dt)
        if kind == "conv":
            s["offsets"] = torch.tensor(_offsets(case), dtype=torch.int32, device=dev)
    elif kind in ("scan", "step"):
        h, p, gr, n = case["heads"], case["dim"], case["groups"], case["state_dim"]
        t = case["tokens"] if kind == "scan" else case["batch"]
        # x, B and C as they come out of the convolution: columns of one row
        act = torch.randn(t, h * p + 2 * gr * n, generator=g, device=dev)
        act = (act / (1 + torch.exp(-act))).to(dt)
        s["x"] = act[:, :h * p].view(t, h, p)
        s["B"] = act[:, h * p:h * p + gr * n].view(t, gr, n)
        s["C"] = act[:, h * p + gr * n:].view(t, gr, n)
        s["dt"] = randn(t, h)
        s["A"] = -(1 + 15 * rand(h))
        s["D"] = 1 + 0.1 * randn(h, dtype=torch.float32)
        # softplus(dt_bias) is log-uniform in [0.001, 0.1]
        d0 = torch.exp(rand(h) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["dt_bias"] = d0 + torch.log(-torch.expm1(-d0))
        s["z"] = randn(t, h, p) if case["gate"] else None
        seqs = case["seqs"] if kind == "scan" else t
        keep = kind == "step" or case["state"]
        s["state"] = randn(seqs, h, p, n, dtype=torch.float32, scale=0.5) if keep else None
        s["state_out"] = torch.empty(seqs, h, p, n, device=dev)
        if kind == "scan":
            s["bounds"] = _offsets(case)
            s["offsets"] = torch.tensor(s["bounds"], dtype=torch.int32, device=dev)
    else:
        r, k, gs = case["rows"], case["cols"], case["group"]
        s["x"] = randn(case["batch"], k)
        s["q"] = torch.randint(0, 256, (r, k // 2), generator=g, device=dev, dtype=torch.uint8)
        s["scales"] = (rand(r, k // gs) * 0.02 + 0.002).to(dt)
        s["zeros"] = (torch.randint(0, 16, (r, k // gs), generator=g, device=dev, dtype=torch.uint8)
                      if case["zeros"] else None)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    kind = s["kind"]
    if own:
        from cpp1_b200 import ops
        if kind == "conv":
            y = ops.causal_conv(s["x"], s["weight"], s["bias"], offsets=s["offsets"], state=s["state"],
                                state_out=s["state_out"], activation="silu")
            return y, s["state_out"]
        if kind == "conv_step":
            y = ops.causal_conv_step(s["x"], s["weight"], s["bias"], state=s["state"], state_out=s["state_out"],
                                     activation="silu")
            return y, s["state_out"]
        if kind == "scan":
            y = ops.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                   dt_bias=s["dt_bias"], dt_softplus=True, offsets=s["offsets"], state=s["state"],
                                   state_out=s["state_out"])
            return y, s["state_out"]
        if kind == "step":
            y = ops.selective_step(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                   dt_bias=s["dt_bias"], dt_softplus=True, state=s["state"],
                                   state_out=s["state_out"])
            return y, s["state_out"]
        return ops.q4_matvec(s["q"], s["scales"], s["x"], zeros=s["zeros"])
    if kind == "conv":
        return _conv_plain(s)
    if kind == "conv_step":
        return _conv_step_plain(s)
    if kind == "scan":
        return _scan_plain(s)
    if kind == "step":
        return _step_plain(s)
    return _q4_plain(s)


# ------------------------------------------------------------------ plain forms
def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(torch.clamp(v, max=20))))


def _conv_plain(s):
    x, off = s["x"].float(), s["offsets"].long()
    w = s["weight"].float()
    width = w.shape[1]
    t = x.shape[0]
    rows = torch.arange(t, device=x.device)
    seq = (rows[:, None] >= off[None, 1:]).sum(1)
    begin = off[seq]
    old = s["state"].float() if s["state"] is not None else None
    acc = torch.zeros_like(x) if s["bias"] is None else s["bias"].float().expand_as(x).clone()
    for j in range(width):
        src = rows - (width - 1) + j
        inside = (src >= begin)[:, None]
        v = x[src.clamp(min=0)]
        if old is None:
            v = torch.where(inside, v, torch.zeros((), device=x.device))
        else:
            v = torch.where(inside, v, old[seq, :, (src - begin + width - 1).clamp(0, width - 2)])
        acc += v * w[:, j]
    y = _silu(acc).to(s["x"].dtype)
    new = s["state_out"]
    for j in range(width - 1):
        src = off[1:] - (width - 1) + j
        inside = (src >= off[:-1])[:, None]
        kept = (torch.zeros(len(src), x.shape[1], device=x.device) if old is None
                else old[torch.arange(len(src), device=x.device), :, (src - off[:-1] + width - 1).clamp(0, width - 2)])
        new[:, :, j] = torch.where(inside, x[src.clamp(min=0)], kept).to(new.dtype)
    return y, new


def _conv_step_plain(s):
    x, w = s["x"].float(), s["weight"].float()
    win = torch.cat([s["state"].float(), x[:, :, None]], dim=2)
    acc = (win * w).sum(2)
    if s["bias"] is not None:
        acc = acc + s["bias"].float()
    s["state_out"].copy_(win[:, :, 1:])
    return _silu(acc).to(s["x"].dtype), s["state_out"]


_CHUNK = 64


def _scan_plain(s):
    """Chunks of 64 tokens: products within a chunk, a loop over the chunks' states."""
    x, bm, cm = s["x"].float(), s["B"].float(), s["C"].float()
    dev = x.device
    t, h, p = x.shape
    g, n = bm.shape[1], bm.shape[2]
    q = _CHUNK
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    # every chunk's rows; rows behind a sequence's end point at an extra row of zeros
    bounds = s["bounds"]
    first, last, count = [], [], []
    for b, e in zip(bounds[:-1], bounds[1:]):
        starts = list(range(b, e, q))
        first += starts
        last += [min(c + q, e) for c in starts]
        count.append(len(starts))
    nc = len(first)
    rows = torch.tensor(first, device=dev)[:, None] + torch.arange(q, device=dev)
    rows = torch.where(rows < torch.tensor(last, device=dev)[:, None], rows, t)

    def chunks(v):
        return torch.cat([v, torch.zeros_like(v[:1])])[rows]

    xc, bc, cc, dc = chunks(x), chunks(bm), chunks(cm), chunks(dt)
    cum = torch.cumsum(dc * s["A"], dim=1).transpose(1, 2)                      # nc, h, q
    xc = (xc * dc[..., None]).transpose(1, 2)                                   # nc, h, q, p
    bc, cc = bc.transpose(1, 2), cc.transpose(1, 2)                             # nc, g, q, n
    low = torch.ones(q, q, dtype=torch.bool, device=dev).tril()
    m = torch.exp(torch.where(low, cum[..., :, None] - cum[..., None, :], -math.inf))
    m = (m.view(nc, g, h // g, q, q) * (cc @ bc.transpose(2, 3))[:, :, None]).view(nc, h, q, q)
    y = m @ xc                                                                  # nc, h, q, p
    del m
    tail = torch.exp(cum[..., -1:] - cum)
    add = ((xc * tail[..., None]).transpose(2, 3).reshape(nc, g, h // g * p, q) @ bc).view(nc, h, p, n)
    decay = torch.exp(cum[..., -1])
    # the states before each chunk
    hs = (s["state"].clone() if s["state"] is not None else torch.zeros(len(count), h, p, n, device=dev))
    begin = [sum(count[:i]) for i in range(len(count))]
    before = torch.empty(nc, h, p, n, device=dev)
    for j in range(max(count)):
        live = [i for i in range(len(count)) if count[i] > j]
        if len(live) == len(count) == 1:
            before[j] = hs[0]
            hs = hs * decay[j, :, None, None] + add[j]
            continue
        li = torch.tensor(live, device=dev)
        ci = torch.tensor([begin[i] + j for i in live], device=dev)
        cur = hs[li]
        before[ci] = cur
        hs[li] = cur * decay[ci][..., None, None] + add[ci]
    off = (before.view(nc, g, h // g * p, n) @ cc.transpose(2, 3)).view(nc, h, p, q).transpose(2, 3)
    y = y + off * torch.exp(cum)[..., None]
    out = torch.empty(t + 1, h, p, device=dev)
    out[rows] = y.transpose(1, 2)
    out = out[:t] + x * s["D"][:, None]
    if s["z"] is not None:
        out = out * _silu(s["z"].float())
    s["state_out"].copy_(hs)
    return out.to(s["x"].dtype), s["state_out"]


def _step_plain(s):
    x, bm, cm = s["x"].float(), s["B"].float(), s["C"].float()
    b, h, p = x.shape
    per = h // bm.shape[1]
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    bh, ch = bm.repeat_interleave(per, 1), cm.repeat_interleave(per, 1)
    new = (s["state"] * torch.exp(dt * s["A"])[..., None, None]
           + (x * dt[..., None])[..., None] * bh[:, :, None, :])
    y = (new * ch[:, :, None, :]).sum(3) + x * s["D"][:, None]
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    s["state_out"].copy_(new)
    return y.to(s["x"].dtype), s["state_out"]


def _q4_plain(s):
    q = s["q"]
    r, half = q.shape
    codes = torch.stack([q & 15, q >> 4], dim=2).view(r, 2 * half).float()
    groups = s["scales"].shape[1]
    zero = s["zeros"].float()[:, :, None] if s["zeros"] is not None else 8.0
    w = ((codes.view(r, groups, -1) - zero) * s["scales"].float()[:, :, None]).view(r, 2 * half)
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


# ------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = {k: (v.double() if isinstance(v, torch.Tensor) and v.dtype.is_floating_point else v) for k, v in s.items()}
    kind = case["kind"]
    if kind == "conv":
        ys, sts = [], []
        off = _offsets(case)
        w = f["weight"]
        width = w.shape[1]
        for i, (b, e) in enumerate(zip(off[:-1], off[1:])):
            head = f["state"][i].t() if f["state"] is not None else torch.zeros_like(w[:, 1:]).t()
            seq = torch.cat([head, f["x"][b:e]])
            u = sum(seq[j:j + e - b] * w[:, j] for j in range(width))
            if f["bias"] is not None:
                u = u + f["bias"]
            ys.append(u * torch.sigmoid(u))
            sts.append(seq[e - b:].t())
        return torch.cat(ys), torch.stack(sts)
    if kind == "conv_step":
        u = torch.einsum("bcw,cw->bc", f["state"], f["weight"][:, :-1]) + f["x"] * f["weight"][:, -1]
        if f["bias"] is not None:
            u = u + f["bias"]
        return u * torch.sigmoid(u), torch.cat([f["state"][:, :, 1:], f["x"][:, :, None]], dim=2)
    if kind in ("scan", "step"):
        h, p, n = case["heads"], case["dim"], case["state_dim"]
        per = h // case["groups"]
        dt = torch.nn.functional.softplus(f["dt"] + f["dt_bias"], threshold=700)
        a = torch.exp(dt * f["A"])
        off = _offsets(case) if kind == "scan" else list(range(case["batch"] + 1))
        lens = [e - b for b, e in zip(off[:-1], off[1:])]
        order = sorted(range(len(lens)), key=lambda i: -lens[i])
        hs = torch.zeros(len(lens), h, p, n, dtype=torch.float64, device="cuda")
        if f["state"] is not None:
            hs += f["state"][order]
        starts = torch.tensor([off[i] for i in order], device="cuda")
        y = torch.empty(f["x"].shape, dtype=torch.float64, device="cuda")
        live = len(lens)
        for j in range(max(lens)):
            while lens[order[live - 1]] <= j:
                live -= 1
            r = starts[:live] + j
            b = f["B"][r].repeat_interleave(per, 1)
            c = f["C"][r].repeat_interleave(per, 1)
            cur = hs[:live]
            cur *= a[r][:, :, None, None]
            cur += (f["x"][r] * dt[r][:, :, None])[..., None] * b[:, :, None, :]
            y[r] = torch.einsum("bhpn,bhn->bhp", cur, c)
        y += f["x"] * f["D"][:, None]
        if f["z"] is not None:
            y *= f["z"] * torch.sigmoid(f["z"])
        out = torch.empty_like(hs)
        out[torch.tensor(order, device="cuda")] = hs
        return y, out
    lo, hi = (f["q"] % 16).double(), torch.div(f["q"], 16, rounding_mode="floor").double()
    w = torch.empty(lo.shape[0], 2 * lo.shape[1], dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = lo, hi
    gs = case["group"]
    w -= f["zeros"].double().repeat_interleave(gs, 1) if f["zeros"] is not None else 8
    w *= f["scales"].repeat_interleave(gs, 1)
    return f["x"] @ w.t()


# ------------------------------------------------------------------ work of one pass
def work(case):
    e = _SIZE[case["dtype"]]
    kind = case["kind"]
    if kind in ("conv", "conv_step"):
        c, w = case["channels"], case["width"]
        rows = case["tokens"] if kind == "conv" else case["batch"]
        seqs = case["seqs"] if kind == "conv" else rows
        reads = 2 if kind == "conv_step" or case["state"] else 1
        nbytes = 2 * rows * c * e + c * w * e + (c * e if case["bias"] else 0) + reads * seqs * c * (w - 1) * e
        return {"bytes": nbytes, "flops": rows * c * (2 * w + 4)}
    if kind in ("scan", "step"):
        h, p, g, n = case["heads"], case["dim"], case["groups"], case["state_dim"]
        rows = case["tokens"] if kind == "scan" else case["batch"]
        seqs = case["seqs"] if kind == "scan" else rows
        reads = 2 if kind == "step" or case["state"] else 1
        nbytes = (rows * (h * p * (3 if case["gate"] else 2) + 2 * g * n + h) * e + 12 * h
                  + reads * seqs * h * p * n * 4)
        # the recurrence: decay, add and read each element of the state
        return {"bytes": nbytes, "flops": rows * h * (5 * p * n + 4 * p)}
    r, k, gs, b = case["rows"], case["cols"], case["group"], case["batch"]
    nbytes = r * k // 2 + r * (k // gs) * (e + (1 if case["zeros"] else 0)) + b * (r + k) * e
    return {"bytes": nbytes, "flops": 2 * b * r * k}
