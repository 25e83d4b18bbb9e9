"""Cases of the event-history operators, for measuring them: the short causal convolution and the selective state space
scan over packed histories (forward, and as a training step), both for single events against per-node state tables, and
dropout in front of a residual sum.

`run` computes a case in plain elementary torch operations (fp32 whatever the inputs' type, rounded once at the end),
or, with `own` set, through fast_b200.ops, as a user calls it.  `exact` restates the definitions in fp64.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # -- short causal convolution over packed histories ------------------------------------------------------
        # the histories of a 600-edge batch's roots (about 20 events each, some nodes without any) at width 200, fp32
        dict(name="conv roots fp32", op="conv", train=True, dtype="fp32", rows=12000, seqs=600, d=200, k=4, pad=0,
             carry=False, tail=0),
        # 64 long histories at a wide inner width, read from one half of a projection's output rows
        dict(name="conv wide bf16", op="conv", train=True, dtype="bf16", rows=32768, seqs=64, d=2048, k=4, pad=2048,
             carry=False, tail=0),
        # -- selective scan over packed histories ----------------------------------------------------------------
        # the same 600-edge batch: short ragged histories, fp32
        dict(name="scan roots fp32", op="scan", train=True, dtype="fp32", rows=12000, seqs=600, d=200, n=16, g=1, pad=0,
             carry=False, tail=0, gate=True),
        # one long history encoded before its events are followed one by one: states in and out, forward only
        dict(name="scan one history", op="scan", train=False, dtype="bf16", rows=2048, seqs=1, d=2048, n=16, g=1, pad=0,
             carry=True, tail=0, gate=True),
        # odd widths in wider buffers, an odd number of states, and rows behind the last history
        dict(name="scan odd widths", op="scan", train=True, dtype="bf16", rows=5003, seqs=7, d=413, n=13, g=1, pad=3,
             carry=True, tail=19, gate=False),
        # the largest training batch: 64 ragged histories
        dict(name="scan packed bf16", op="scan", train=True, dtype="bf16", rows=16384, seqs=64, d=1024, n=16, g=1,
             pad=0, carry=False, tail=0, gate=True),
        # -- single events against state tables ------------------------------------------------------------------
        # one event of one node while a query is answered: launch latency alone
        dict(name="conv event", op="conv_step", dtype="bf16", rows=1, nodes=2000, d=2048, k=4, pad=0, repeat=1),
        # a large batch of events in chronological order, busy nodes several times in it
        dict(name="conv events", op="conv_step", dtype="fp32", rows=4000, nodes=16700, d=200, k=4, pad=0, repeat=4),
        dict(name="scan event", op="scan_step", dtype="bf16", rows=1, nodes=1000, d=2048, n=16, g=1, pad=0, repeat=1,
             gate=True),
        dict(name="scan events", op="scan_step", dtype="fp32", rows=4000, nodes=16700, d=200, n=16, g=1, pad=0,
             repeat=4, gate=True),
        # -- dropout in front of a residual sum ------------------------------------------------------------------
        # the 12,000 roots of a training batch at hidden width 100, fp32
        dict(name="dropout roots fp32", op="dropout", train=True, dtype="fp32", rows=12000, d=100, pad=0, res=True,
             p=0.1),
        # a wide block over a long batch: bound by memory, or by the generator
        dict(name="dropout wide bf16", op="dropout", train=True, dtype="bf16", rows=16384, d=4096, pad=0, res=True,
             p=0.2),
    ]


def draw(rng):
    def span(lo, hi):
        """Log-uniform whole number; an eighth of them rounded to a multiple of 64."""
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return min(hi, max(lo, n // 64 * 64)) if rng.random() < 0.125 and n >= 64 else n

    while True:
        op = rng.choice(["conv", "conv", "scan", "scan", "scan", "conv_step", "scan_step", "dropout"])
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp32"]), pad=rng.choice([0, 0, 0, 3, 4, 8]))
        if op in ("conv", "scan"):
            c.update(train=rng.random() < 0.7, rows=span(1, 32768), d=span(8, 4096), carry=rng.random() < 0.4,
                     tail=rng.choice([0, 0, 0, 1, 37]))
            c["seqs"] = span(1, max(1, min(2000, c["rows"])))
            if op == "conv":
                c["k"] = rng.choice([2, 3, 4, 4, 4, 5, 8])
                cost, top = c["rows"] * c["d"], 32768 * 2048
            else:
                c.update(n=rng.choice([1, 4, 8, 13, 16, 16, 16, 32, 64]), gate=rng.random() < 0.7)
                c["g"] = rng.choice([q for q in (1, 1, 1, 2, 4) if c["d"] % q == 0])
                cost, top = c["rows"] * c["d"] * c["n"], 16384 * 1024 * 16
        elif op in ("conv_step", "scan_step"):
            c.update(rows=span(1, 4000), d=span(8, 4096), repeat=rng.choice([1, 1, 2, 5]))
            c["nodes"] = c["rows"] + span(1, 4000)
            if op == "conv_step":
                c["k"] = rng.choice([2, 3, 4, 4, 4, 5, 8])
                cost, top = c["nodes"] * c["d"] * (c["k"] - 1), 16700 * 200 * 16
            else:
                c.update(n=rng.choice([1, 4, 8, 13, 16, 16, 16, 32, 64]), gate=rng.random() < 0.7)
                c["g"] = rng.choice([q for q in (1, 1, 1, 2, 4) if c["d"] % q == 0])
                cost, top = c["nodes"] * c["d"] * c["n"], 16700 * 200 * 16
        else:
            c.update(train=rng.random() < 0.7, rows=span(1, 16384), d=span(8, 4096), res=rng.random() < 0.6,
                     p=rng.choice([0.0, 0.1, 0.2, 0.5]))
            cost, top = c["rows"] * c["d"], 16384 * 4096
        if cost <= top:
            return c


def work(case):
    op, n, d, e = case["op"], case["rows"], case["d"], TYPES[case["dtype"]].itemsize
    if op == "conv":
        k, state = case["k"], case["seqs"] * (case["k"] - 1) * d * e if case["carry"] else 0
        planes = 4 if case["train"] else 2                       # x in, y out; dy in, dx out
        return {"bytes": planes * n * d * e + 2 * state + (k + 1) * d * 4,
                "flops": ((6 * k + 16) if case["train"] else (2 * k + 5)) * n * d}
    if op == "scan":
        s, g = case["n"], case["g"]
        planes = (3 + case["gate"]) + ((3 + case["gate"]) if case["train"] else 0)   # u, delta, z in, y out; dy in, du, ddelta, dz out
        small = (4 if case["train"] else 2) * n * g * s * e + (2 if case["train"] else 1) * d * (s + 2) * 4
        state = case["seqs"] * d * s * 4 * (3 if case["train"] else 2) if case["carry"] else 0
        return {"bytes": planes * n * d * e + small + state, "flops": (28 if case["train"] else 7) * n * d * s}
    if op == "conv_step":
        return {"bytes": n * d * e * (2 + 2 * (case["k"] - 1)) + (case["k"] + 1) * d * 4, "flops": (2 * case["k"] + 5) * n * d}
    if op == "scan_step":
        s = case["n"]
        return {"bytes": n * d * (8 * s + e * (3 + case["gate"])) + d * (s + 2) * 4 + 2 * n * case["g"] * s * e,
                "flops": 7 * n * d * s}
    planes = (3 if case["res"] else 2) + (2 if case["train"] else 0)
    return {"bytes": planes * n * d * e, "flops": (32 if case["train"] else 16) * n * d}


# ----------------------------------------------------------------------------------------------------------------------
def _normal(g, rows, cols, dtype, scale=1.0, pad=0):
    """N(0, scale^2) rows in a buffer `pad` elements wider than they are."""
    t = torch.empty(rows, cols + pad, device="cuda", dtype=torch.float32).normal_(generator=g).mul_(scale).to(dtype)
    return t[:, :cols]


def _starts(case, seed):
    """Ragged histories of rows - tail rows in all: the cuts are drawn with repetition, so some histories are empty."""
    rng, rows = random.Random(seed), case["rows"] - min(case["tail"], case["rows"] - 1)
    return [0] + sorted(rng.randint(0, rows) for _ in range(case["seqs"] - 1)) + [rows]


def _scan_weights(g, d, n):
    """Decays -1 .. -n of each channel, a little apart; a bias that puts softplus between 0.001 and 0.1."""
    A = -(torch.arange(1, n + 1, device="cuda", dtype=torch.float32).expand(d, n) * (0.8 + 0.4 * torch.rand(d, n, device="cuda", generator=g)))
    dt = torch.exp(torch.rand(d, device="cuda", generator=g) * math.log(100.0) + math.log(1e-3))
    return dict(A=A.contiguous(), D=torch.ones(d, device="cuda") + 0.1 * torch.randn(d, device="cuda", generator=g),
                delta_bias=torch.log(torch.expm1(dt)))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows, d, pad, op = TYPES[case["dtype"]], case["rows"], case["d"], case["pad"], case["op"]
    s = {"op": op, "train": case.get("train", False)}
    if op == "conv_step" or op == "scan_step":
        # events in chronological order; a few busy nodes come `repeat` times
        rng = random.Random(seed)
        index = rng.sample(range(case["nodes"]), rows)
        if case["repeat"] > 1 and rows > case["repeat"]:
            for _ in range(max(1, rows // 50)):
                at = rng.sample(range(rows), case["repeat"])
                for i in at[1:]:
                    index[i] = index[at[0]]
        count = {}
        for i in index:
            count[i] = count.get(i, 0) + 1
        s["most"] = max(count.values())
        s["index"] = torch.tensor(index, device="cuda")
    if op == "conv" or op == "conv_step":
        k = case["k"]
        s["x"] = _normal(g, rows, d, dt, 1.0, pad)
        s["w"] = _normal(g, d, k, torch.float32, k ** -0.5)
        s["bias"] = _normal(g, 1, d, torch.float32, 0.1)[0]
        if op == "conv_step":
            s["table"] = _normal(g, case["nodes"] + 1, (k - 1) * d, dt).view(-1, k - 1, d)    # a spare row: see _put
            s["state"] = s["table"][:-1]
            return s
        starts = _starts(case, seed)
        s["starts"] = torch.tensor(starts, device="cuda")
        s["init"] = _normal(g, case["seqs"] * (k - 1), d, dt).view(-1, k - 1, d) if case["carry"] else None
        if s["train"]:
            s["dy"] = _normal(g, rows, d, dt, 1e-3)
    elif op == "scan" or op == "scan_step":
        n, groups = case["n"], case["g"]
        s["u"] = _normal(g, rows, d, dt, 1.0, pad)
        s["delta"] = _normal(g, rows, d, dt, 0.7, pad)
        s["B"] = _normal(g, rows, groups * n, dt, 1.0, pad).unflatten(1, (groups, n))
        s["C"] = _normal(g, rows, groups * n, dt, 1.0, pad).unflatten(1, (groups, n))
        s["z"] = _normal(g, rows, d, dt, 1.0, pad) if case["gate"] else None
        s.update(_scan_weights(g, d, n))
        if op == "scan_step":
            s["table"] = _normal(g, (case["nodes"] + 1) * d, n, torch.float32, 0.3).view(-1, d, n)
            s["state"] = s["table"][:-1]
            return s
        starts = _starts(case, seed)
        s["starts"] = torch.tensor(starts, device="cuda")
        s["longest"] = max(b - a for a, b in zip(starts, starts[1:]))
        s["init"] = _normal(g, case["seqs"] * d, n, torch.float32, 0.3).view(-1, d, n) if case["carry"] else None
        if s["train"]:
            s["dy"] = _normal(g, rows, d, dt, 1e-3)
    else:
        s["x"] = _normal(g, rows, d, dt, 1.0, pad)
        s["res"] = _normal(g, rows, d, dt, 1.0, pad) if case["res"] else None
        s["p"], s["seed"], s["offset"] = case["p"], seed * 7919 + 12345678901, 3 + (seed << 20)
        if s["train"]:
            s["dy"] = _normal(g, rows, d, dt, 1e-3)
    return s


# ----------------------------------------------------------------------------------------------------------------------
def _silu(x):
    """silu(x) and its derivative."""
    sg = 1 / (1 + torch.exp(-x))
    return x * sg, sg * (1 + x * (1 - sg))


def _softplus(x):
    """log(1 + e^x) and its derivative."""
    e = torch.exp(-x.abs())
    return x.clamp(min=0) + torch.log1p(e), torch.where(x >= 0, 1 / (1 + e), e / (1 + e))


def _owner(starts, rows):
    """Sequence of each row (-1 behind the last one), and the row's place in it."""
    t = torch.arange(rows, device=starts.device)
    seq = torch.searchsorted(starts, t, right=True) - 1
    inside = t < starts[-1]
    seq = torch.where(inside, seq, -1)
    pos = torch.where(inside, t - starts[seq.clamp(min=0)], 0)
    return seq, pos


def _taps(x, init, seq, pos, k):
    """The k inputs of each row, oldest first, and which of them lie in the row's own sequence."""
    rows = x.shape[0]
    t = torch.arange(rows, device=x.device)
    for j in range(k - 1, -1, -1):                              # j rows back
        here = (pos >= j) & (seq >= 0)
        v = x[(t - j).clamp(min=0)] * here.unsqueeze(1)
        if init is not None and j:
            at = (k - 1 + pos - j).clamp(max=k - 2)
            v = v + init[seq.clamp(min=0), at] * ((pos < j) & (seq >= 0)).unsqueeze(1)
        yield j, v, here


def _plain_conv(s):
    dt, x, w, bias = s["x"].dtype, s["x"].float(), s["w"].float(), s["bias"].float()
    init = None if s["init"] is None else s["init"].float()
    k, rows = w.shape[1], x.shape[0]
    seq, pos = _owner(s["starts"], rows)
    inside = (seq >= 0).unsqueeze(1)
    p = bias.expand(rows, -1).clone()
    for j, v, _ in _taps(x, init, seq, pos, k):
        p = p + w[:, k - 1 - j] * v
    y, dact = _silu(p)
    out = {"y": (y * inside).to(dt)}
    if init is not None:
        # the k - 1 newest inputs of each history, older ones shifted up where it is shorter
        start, end = s["starts"][:-1], s["starts"][1:]
        slots = []
        for i in range(k - 1):
            back = k - 1 - i                                     # inputs back from the end
            have = end - start >= back
            new = x[(end - back).clamp(min=0)] * have.unsqueeze(1)
            at = (i + (end - start)).clamp(max=k - 2)
            old = init[torch.arange(len(start), device=x.device), at] * (~have).unsqueeze(1)
            slots.append(new + old)
        out["final"] = torch.stack(slots, 1).to(dt)
    if s["train"]:
        dp = s["dy"].float() * dact * inside
        dx, dw = torch.zeros_like(x), torch.empty_like(w)
        dinit = None if init is None else torch.zeros_like(init)
        for j, v, here in _taps(x, init, seq, pos, k):
            wj = w[:, k - 1 - j]
            dw[:, k - 1 - j] = (dp * v).sum(0)
            dx[:rows - j] += ((dp * here.unsqueeze(1)) * wj)[j:]
            if dinit is not None and j:
                back = (pos < j) & (seq >= 0)
                at = (k - 1 + pos - j).clamp(max=k - 2)
                dinit.index_put_((seq.clamp(min=0), at), (dp * wj) * back.unsqueeze(1), accumulate=True)
        out.update(dx=dx.to(dt), dw=dw, dbias=dp.sum(0))
        if dinit is not None:
            out["dinit"] = dinit.to(dt)
    return out


def _doubling(a, b, longest):
    """h[t] = a[t] h[t-1] + b[t] down the rows, in log2(longest) rounds; a is 0 where a sequence begins."""
    a, b, k = a.clone(), b.clone(), 1
    while k < longest:
        b[k:] = b[k:] + a[k:] * b[:-k]
        a[k:] = a[k:] * a[:-k]
        k *= 2
    return b


def _plain_scan(s):
    dtype, u, dy = s["u"].dtype, s["u"].float(), None
    x = s["delta"].float() + s["delta_bias"]
    dt, ddt_dx = _softplus(x)
    rows, d = u.shape
    groups, n = s["B"].shape[1:]
    A, D = s["A"], s["D"]
    seq, pos = _owner(s["starts"], rows)
    inside, first = (seq >= 0).view(-1, 1, 1), ((pos == 0) & (seq >= 0)).view(-1, 1, 1)

    def wide(t):
        """[rows, groups, n] to each channel's [rows, d, n]."""
        return t.float().unsqueeze(2).expand(rows, groups, d // groups, n).reshape(rows, d, n)

    def narrow(t):
        return t.view(rows, groups, d // groups, n).sum(2)

    a = torch.exp(dt.unsqueeze(2) * A)
    b = (dt * u).unsqueeze(2) * wide(s["B"]) * inside
    init = s["init"]
    if init is not None:
        b = b + first * a * init[seq.clamp(min=0)]
    a0 = a * (inside & ~first)
    h = _doubling(a0, b, s["longest"])
    del b
    v = (h * wide(s["C"])).sum(2) + D * u
    zs, dzs = _silu(s["z"].float()) if s["z"] is not None else (torch.ones_like(v), None)
    keep = inside.squeeze(2)
    out = {"y": (v * zs * keep).to(dtype)}
    if init is not None:
        end, some = s["starts"][1:], (s["starts"][1:] > s["starts"][:-1]).view(-1, 1, 1)
        out["final"] = torch.where(some, h[(end - 1).clamp(min=0)], init)
    if s["train"]:
        dy = s["dy"].float() * keep
        gv = dy * zs
        b = gv.unsqueeze(2) * wide(s["C"])
        shifted = torch.cat([a0[1:], torch.zeros_like(a0[:1])])
        g = _doubling(shifted.flip(0), b.flip(0), s["longest"]).flip(0)
        del b, shifted
        prev = torch.cat([torch.zeros_like(h[:1]), h[:-1]]) * (~first)
        if init is not None:
            prev = prev + first * init[seq.clamp(min=0)]
        gB = (g * wide(s["B"])).sum(2)
        q = g * a * prev
        ddelta = ((q * A).sum(2) + u * gB) * ddt_dx
        out.update(du=(dt * gB + D * gv).to(dtype), ddelta=ddelta.to(dtype), dA=(q * dt.unsqueeze(2)).sum(0),
                   dB=narrow(g * (dt * u).unsqueeze(2)).to(dtype), dC=narrow(gv.unsqueeze(2) * h).to(dtype),
                   dD=(gv * u).sum(0), ddelta_bias=ddelta.sum(0))
        if dzs is not None:
            out["dz"] = (dy * v * dzs).to(dtype)
        if init is not None:
            begin = s["starts"][:-1].clamp(max=rows - 1)
            out["dinit"] = torch.where(some, a[begin] * g[begin], torch.zeros_like(init))
    return out


def _turns(s):
    """Which occurrence of its node each row is: events of one node take their turns in the rows' order."""
    i = s["index"]
    before = torch.ones(len(i), len(i), device=i.device, dtype=torch.bool).tril(-1)
    return ((i.unsqueeze(1) == i.unsqueeze(0)) & before).sum(1)


def _put(s, now, rows):
    """Writes the rows whose turn it is to their nodes, the others to the spare row behind the table."""
    s["table"][torch.where(now.squeeze(1), s["index"], len(s["state"]))] = rows


def _plain_conv_step(s):
    dt, x, w, state, index = s["x"].dtype, s["x"].float(), s["w"].float(), s["state"], s["index"]
    turn, y = _turns(s), torch.zeros_like(x)
    for i in range(s["most"]):
        now = (turn == i).unsqueeze(1)
        window = torch.cat([state[index].float(), x.unsqueeze(1)], 1)          # [rows, k, d]
        y = torch.where(now, _silu((window * w.t()).sum(1) + s["bias"])[0], y)
        _put(s, now, window[:, 1:].to(dt))
    return {"y": y.to(dt), "state": state}


def _plain_scan_step(s):
    dtype, u, state, index = s["u"].dtype, s["u"].float(), s["state"], s["index"]
    dt = _softplus(s["delta"].float() + s["delta_bias"])[0]
    rows, d = u.shape
    groups, n = s["B"].shape[1:]

    def wide(t):
        return t.float().unsqueeze(2).expand(rows, groups, d // groups, n).reshape(rows, d, n)

    a, b, c = torch.exp(dt.unsqueeze(2) * s["A"]), (dt * u).unsqueeze(2) * wide(s["B"]), wide(s["C"])
    turn, v = _turns(s), torch.zeros_like(u)
    for i in range(s["most"]):
        now = (turn == i).unsqueeze(1)
        h = a * state[index] + b
        v = torch.where(now, (h * c).sum(2), v)
        _put(s, now, h)
    v = v + s["D"] * u
    if s["z"] is not None:
        v = v * _silu(s["z"].float())[0]
    return {"y": v.to(dtype), "state": state}


def _mulhilo(m, c):
    """High and low words of the 64-bit product of two 32-bit words held as int64."""
    low, high = (c & 0xFFFF) * m, (c >> 16) * m                # below 2^48 each
    t = low + ((high & 0xFFFF) << 16)                          # below 2^49
    return (high >> 16) + (t >> 32), t & 0xFFFFFFFF


def _plain_dropout(s):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011): counter (column / 4, row, offset), key seed; a column keeps
    its value where the top 24 bits of its word, as a fraction, are not below p."""
    dt, x = s["x"].dtype, s["x"].float()
    rows, d = x.shape
    dev, quads = x.device, -(-d // 4)
    c = [torch.arange(quads, device=dev).expand(rows, quads), torch.arange(rows, device=dev).unsqueeze(1).expand(rows, quads),
         torch.full((rows, quads), s["offset"] & 0xFFFFFFFF, device=dev), torch.full((rows, quads), s["offset"] >> 32, device=dev)]
    k0, k1 = s["seed"] & 0xFFFFFFFF, s["seed"] >> 32
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, c[0])
        h1, l1 = _mulhilo(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    word = torch.stack(c, 2).view(rows, quads * 4)[:, :d]
    p = torch.tensor(s["p"], dtype=torch.float32, device=dev)
    scale = ((word >> 8).float() * 2.0 ** -24 >= p) * (1 / (1 - p))
    y = x * scale
    if s["res"] is not None:
        y = y + s["res"].float()
    out = {"y": y.to(dt)}
    if s["train"]:
        out["dx"] = (s["dy"].float() * scale).to(dt)
    return out


def _own(s):
    from fast_b200 import ops
    if s["op"] == "conv":
        kw = dict(bias=s["bias"], starts=s["starts"], init=s["init"])
        if s["init"] is None:
            out = {"y": ops.short_conv_fwd(s["x"], s["w"], **kw)}
        else:
            y, final = ops.short_conv_fwd(s["x"], s["w"], final=True, **kw)
            out = {"y": y, "final": final}
        if s["train"]:
            out["dx"], out["dw"], out["dbias"], dinit = ops.short_conv_bwd(s["dy"], s["x"], s["w"], **kw)
            if dinit is not None:
                out["dinit"] = dinit
        return out
    if s["op"] == "scan":
        kw = dict(D=s["D"], z=s["z"], delta_bias=s["delta_bias"], starts=s["starts"], init=s["init"])
        args = s["u"], s["delta"], s["A"], s["B"], s["C"]
        y, carry, final = ops.selective_scan_fwd(*args, final=s["init"] is not None, keep=s["train"], **kw)
        out = {"y": y}
        if final is not None:
            out["final"] = final
        if s["train"]:
            grads = ops.selective_scan_bwd(s["dy"], *args, carry, **kw)
            names = "du", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dinit"
            out.update((k, v) for k, v in zip(names, grads) if v is not None)
        return out
    if s["op"] == "conv_step":
        return {"y": ops.short_conv_step(s["x"], s["state"], s["w"], bias=s["bias"], index=s["index"]), "state": s["state"]}
    if s["op"] == "scan_step":
        y = ops.selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                    delta_bias=s["delta_bias"], index=s["index"])
        return {"y": y, "state": s["state"]}
    out = {"y": ops.dropout_fwd(s["x"], s["p"], s["seed"], s["offset"], res=s["res"])}
    if s["train"]:
        out["dx"] = ops.dropout_bwd(s["dy"], s["p"], s["seed"], s["offset"])
    return out


def run(state):
    if own:
        return _own(state)
    return {"conv": _plain_conv, "scan": _plain_scan, "conv_step": _plain_conv_step, "scan_step": _plain_scan_step,
            "dropout": _plain_dropout}[state["op"]](state)


# ----------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """The definitions in fp64: histories one by one or position by position."""
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "conv_step": _exact_conv_step, "scan_step": _exact_scan_step,
            "dropout": _exact_dropout}[case["op"]](s)


def _exact_conv(s):
    F = torch.nn.functional
    x, w, bias = (s[k].double().requires_grad_(s["train"]) for k in ("x", "w", "bias"))
    d, k = w.shape
    starts = s["starts"].tolist()
    init = None if s["init"] is None else s["init"].double().requires_grad_(s["train"])
    before = torch.zeros(len(starts) - 1, k - 1, d, device=x.device, dtype=x.dtype) if init is None else init
    ys, finals = [], []
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        xe = torch.cat([before[i], x[a:b]])
        finals.append(xe[len(xe) - (k - 1):])
        if b > a:
            ys.append(F.silu(F.conv1d(xe.t().unsqueeze(0), w.unsqueeze(1), bias, groups=d))[0].t())
    ys.append(x.new_zeros(len(x) - starts[-1], d))
    y = torch.cat(ys)
    out = {"y": y}
    if init is not None:
        out["final"] = torch.stack(finals)
    if s["train"]:
        want = [x, w, bias] + ([] if init is None else [init])
        grads = torch.autograd.grad(y, want, s["dy"].double())
        out.update(zip(("dx", "dw", "dbias", "dinit"), grads))
    return {k: v.detach() for k, v in out.items()}


def _exact_scan(s):
    F = torch.nn.functional
    u, B, C, A, D = (s[k].double() for k in ("u", "B", "C", "A", "D"))
    x = s["delta"].double() + s["delta_bias"].double()
    dt = F.softplus(x, threshold=1000)
    rows, d = u.shape
    per = d // B.shape[1]
    n = A.shape[1]
    starts = s["starts"]
    lens = (starts[1:] - starts[:-1]).tolist()
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    order_dev = torch.tensor(order, device=u.device)
    first = starts[:-1][order_dev]
    init = torch.zeros(len(lens), d, n, device=u.device, dtype=u.dtype) if s["init"] is None else s["init"].double()
    longest = lens[order[0]]
    active = [sum(1 for i in order if lens[i] > j) for j in range(longest)] if longest < 4096 or len(lens) < 300 else None
    if active is None:
        return None
    before = torch.zeros(rows, d, n, device=u.device, dtype=u.dtype)            # the state each row finds
    h, final, v = init[order_dev].clone(), init.clone(), torch.zeros_like(u)
    for j, m in enumerate(active):
        r = first[:m] + j
        before[r] = h[:m]
        a = torch.exp(dt[r].unsqueeze(2) * A)
        Bj, Cj = B[r].repeat_interleave(per, 1), C[r].repeat_interleave(per, 1)
        h[:m] = a * h[:m] + (dt[r] * u[r]).unsqueeze(2) * Bj
        v[r] = (Cj * h[:m]).sum(2) + D * u[r]
    final[order_dev] = h
    zs = F.silu(s["z"].double()) if s["z"] is not None else 1.0
    out = {"y": v * zs}
    if s["init"] is not None:
        out["final"] = final
    if not s["train"]:
        return out
    dy = s["dy"].double()
    dy[int(starts[-1]):] = 0
    gv = dy * zs
    du, ddt, dA = D * gv, torch.zeros_like(u), torch.zeros_like(A)
    dB, dC = torch.zeros_like(B), torch.zeros_like(C)
    g = torch.zeros_like(h)
    for j in range(longest - 1, -1, -1):
        m = active[j]
        r = first[:m] + j
        a = torch.exp(dt[r].unsqueeze(2) * A)
        Bj, Cj = B[r].repeat_interleave(per, 1), C[r].repeat_interleave(per, 1)
        hj = a * before[r] + (dt[r] * u[r]).unsqueeze(2) * Bj
        gj = g[:m] + Cj * gv[r].unsqueeze(2)
        dC[r] = (gv[r].unsqueeze(2) * hj).unflatten(1, (-1, per)).sum(2)
        dB[r] = (gj * (dt[r] * u[r]).unsqueeze(2)).unflatten(1, (-1, per)).sum(2)
        gB = (gj * Bj).sum(2)
        q = gj * a * before[r]
        du[r] += dt[r] * gB
        ddt[r] = (q * A).sum(2) + u[r] * gB
        dA += (q * dt[r].unsqueeze(2)).sum(0)
        g[:m] = a * gj
    ddelta = ddt * torch.sigmoid(x)
    out.update(du=du, ddelta=ddelta, dA=dA, dB=dB, dC=dC, dD=(gv * u).sum(0), ddelta_bias=ddelta.sum(0))
    if s["z"] is not None:
        z = s["z"].double()
        sg = torch.sigmoid(z)
        out["dz"] = dy * v * (sg + z * sg * (1 - sg))
    if s["init"] is not None:
        dinit = torch.zeros_like(init)
        dinit[order_dev] = g
        out["dinit"] = dinit
    return out


def _exact_conv_step(s):
    x, w, bias, state = (s[k].double() for k in ("x", "w", "bias", "state"))
    y = torch.zeros_like(x)
    for rows in _by_turn(s["index"].tolist(), x.device):
        at = s["index"][rows]
        window = torch.cat([state[at], x[rows].unsqueeze(1)], 1)
        y[rows] = torch.nn.functional.silu(torch.einsum("rkd,dk->rd", window, w) + bias)
        state[at] = window[:, 1:]
    return {"y": y, "state": state}


def _exact_scan_step(s):
    u, B, C, A, D, state = (s[k].double() for k in ("u", "B", "C", "A", "D", "state"))
    dt = torch.nn.functional.softplus(s["delta"].double() + s["delta_bias"].double(), threshold=1000)
    per, y = u.shape[1] // B.shape[1], torch.zeros_like(u)
    for rows in _by_turn(s["index"].tolist(), u.device):
        at = s["index"][rows]
        h = torch.exp(dt[rows].unsqueeze(2) * A) * state[at] + (dt[rows] * u[rows]).unsqueeze(2) * B[rows].repeat_interleave(per, 1)
        state[at] = h
        y[rows] = (C[rows].repeat_interleave(per, 1) * h).sum(2) + D * u[rows]
    if s["z"] is not None:
        y = y * torch.nn.functional.silu(s["z"].double())
    return {"y": y, "state": state}


def _by_turn(index, device):
    """The rows of every node's first event, of every second event, ..."""
    seen, turns = {}, []
    for r, i in enumerate(index):
        t = seen.get(i, 0)
        seen[i] = t + 1
        if t == len(turns):
            turns.append([])
        turns[t].append(r)
    return [torch.tensor(t, device=device) for t in turns]


def _exact_dropout(s):
    rows, d = s["x"].shape
    quads, word = -(-d // 4), np.uint64(0xFFFFFFFF)
    c0 = np.broadcast_to(np.arange(quads, dtype=np.uint64), (rows, quads))
    c1 = np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], (rows, quads))
    c2, c3 = np.full((rows, quads), s["offset"] & 0xFFFFFFFF, np.uint64), np.full((rows, quads), s["offset"] >> 32, np.uint64)
    k0, k1 = s["seed"] & 0xFFFFFFFF, s["seed"] >> 32
    for _ in range(10):
        p0, p1 = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = (p1 >> np.uint64(32)) ^ c1 ^ np.uint64(k0), p1 & word, (p0 >> np.uint64(32)) ^ c3 ^ np.uint64(k1), p0 & word
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack([c0, c1, c2, c3], 2).reshape(rows, quads * 4)[:, :d]
    keep = (words >> np.uint64(8)).astype(np.float64) * 2.0 ** -24 >= float(np.float32(s["p"]))
    scale = torch.from_numpy(keep).to(s["x"].device).double() / (1 - s["p"])
    y = s["x"].double() * scale
    if s["res"] is not None:
        y = y + s["res"].double()
    out = {"y": y}
    if s["train"]:
        out["dx"] = s["dy"].double() * scale
    return out
