"""Cases of the node-ranking head's operators, for measuring them: layer norm, the gated feed-forward block and the
softmax cross entropy over every candidate node, each forward and as a training step.

`run` computes a case in plain elementary torch operations (fp32 whatever the inputs' type, rounded once at the end),
or, with `own` set, through fast_b200.ops, as a user calls it.  `exact` restates the definitions in fp64.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # -- layer norm ------------------------------------------------------------------------------------------
        # one root embedding normalised while answering a single ranking query: launch latency alone
        dict(name="norm one row", op="norm", train=False, dtype="bf16", rows=1, d=1024, pad=0, res=False),
        # the 12,000 roots (4,000 edges, their ends and negatives) of a training batch at hidden width 100, fp32 mode
        dict(name="norm roots fp32", op="norm", train=True, dtype="fp32", rows=12000, d=100, pad=0, res=False),
        # an odd width in a wider buffer: rows that no vector load lines up with
        dict(name="norm odd rows", op="norm", train=True, dtype="bf16", rows=20011, d=413, pad=6, res=False),
        # a wide head over a long batch, the residual sum included: bound by memory
        dict(name="norm wide residual", op="norm", train=True, dtype="bf16", rows=16384, d=4096, pad=0, res=True),
        # -- gated feed-forward block ----------------------------------------------------------------------------
        # a single ranking query through a wide head: every weight is read for one row
        dict(name="ffn one row", op="ffn", train=False, dtype="bf16", rows=1, d=2048, f=8192, pad=0, act="silu"),
        # a 600-edge batch's 1,800 roots at hidden width 100 in the fp32 mode
        dict(name="ffn roots fp32", op="ffn", train=True, dtype="fp32", rows=1800, d=100, f=400, pad=0, act="silu"),
        # the 12,000 roots of the large batch in the bf16 mode, rows padded to 16 bytes as the mode's layouts are
        dict(name="ffn roots bf16", op="ffn", train=True, dtype="bf16", rows=12000, d=172, f=688, pad=4, act="gelu"),
        # a large head: bound by the tensor cores
        dict(name="ffn large", op="ffn", train=True, dtype="bf16", rows=8192, d=2048, f=8192, pad=0, act="silu"),
        # -- softmax cross entropy over all nodes ----------------------------------------------------------------
        # the answer to one query scored against 50,000 nodes: the node table is read once
        dict(name="xent one row", op="xent", train=False, dtype="bf16", rows=1, d=1024, v=50000, pad=0, ignore=0.0),
        # 600 edges ranked against 10,000 nodes in the fp32 mode
        dict(name="xent nodes fp32", op="xent", train=True, dtype="fp32", rows=600, d=100, v=10000, pad=0, ignore=0.0),
        # 4,000 edges ranked against 16,700 nodes in the bf16 mode, some edges held out of the loss
        dict(name="xent nodes bf16", op="xent", train=True, dtype="bf16", rows=4000, d=100, v=16700, pad=4,
             ignore=0.05),
        # a wide head over a long batch: bound by the tensor cores
        dict(name="xent large", op="xent", train=True, dtype="bf16", rows=8192, d=1024, v=50000, pad=0, ignore=0.02),
    ]


def draw(rng):
    def span(lo, hi):
        """Log-uniform whole number; an eighth of them rounded to a multiple of 64."""
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return min(hi, max(lo, n // 64 * 64)) if rng.random() < 0.125 and n >= 64 else n

    while True:
        op = rng.choice(["norm", "ffn", "xent"])
        c = dict(op=op, train=rng.random() < 0.7, dtype=rng.choice(["bf16", "bf16", "fp32"]), rows=span(1, 16384),
                 d=span(16, 4096), pad=rng.choice([0, 0, 0, 4, 8, 12]))
        if op == "norm":
            c["res"] = rng.random() < 0.4
            top = 16384 * 4096
            cost = c["rows"] * c["d"]
        elif op == "ffn":
            c["f"] = min(16384, max(16, int(c["d"] * rng.uniform(1.5, 4.5))))
            c["act"] = rng.choice(["silu", "gelu", "relu"])
            top = 8192 * 2048 * 8192 // (4 if c["dtype"] == "fp32" else 1)
            cost = c["rows"] * c["d"] * c["f"]
        else:
            c["v"] = span(500, 60000)
            c["ignore"] = rng.choice([0.0, 0.05, 0.3])
            top = 8192 * 1024 * 50000 // (4 if c["dtype"] == "fp32" else 1)
            cost = c["rows"] * c["d"] * c["v"]
        if cost <= top:
            return c


def work(case):
    n, d, e = case["rows"], case["d"], TYPES[case["dtype"]].itemsize
    train = case["train"]
    if case["op"] == "norm":
        # x (and the residual) in, y (and the sum) out; backward: dy (and the sum's gradient) in, dx out
        planes = (4 if case["res"] else 2) + ((3 if case["res"] else 2) if train else 0)
        return {"bytes": planes * n * d * e + (4 if train else 2) * d * e, "flops": (18 if train else 8) * n * d}
    if case["op"] == "ffn":
        f = case["f"]
        weights = 3 * d * f * e
        return {"bytes": (2 * n * d * e + weights) * (2 if train else 1), "flops": (18 if train else 6) * n * d * f}
    v = case["v"]
    operands = (n + v) * d * e
    return {"bytes": operands * (2 if train else 1) + n * (20 if train else 12), "flops": (6 if train else 2) * n * d * v}


# ----------------------------------------------------------------------------------------------------------------------
def _normal(g, rows, cols, dtype, scale=1.0, pad=0):
    """N(0, scale^2) rows in a buffer `pad` elements wider than they are."""
    t = torch.empty(rows, cols + pad, device="cuda", dtype=torch.float32).normal_(generator=g).mul_(scale).to(dtype)
    return t[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, n, d, pad = TYPES[case["dtype"]], case["rows"], case["d"], case["pad"]
    s = {"op": case["op"], "train": case["train"]}
    if case["op"] == "norm":
        # embeddings away from mean 0 and scale 1, a weight near 1
        s["x"] = _normal(g, n, d, dt, 1.7, pad).add_(0.4)
        s["res"] = _normal(g, n, d, dt, 0.8, pad) if case["res"] else None
        s["gamma"] = _normal(g, 1, d, dt, 0.2)[0].add_(1)
        s["beta"] = _normal(g, 1, d, dt, 0.2)[0]
        if case["train"]:
            s["dy"] = _normal(g, n, d, dt, 1e-3, pad)
            s["ds"] = _normal(g, n, d, dt, 1e-3, pad) if case["res"] else None
    elif case["op"] == "ffn":
        f = case["f"]
        s["act"] = case["act"]
        s["x"] = _normal(g, n, d, dt, 1.0, pad)
        s["w_gate"] = _normal(g, f, d, dt, d ** -0.5, pad)
        s["w_up"] = _normal(g, f, d, dt, d ** -0.5, pad)
        s["w_down"] = _normal(g, d, f, dt, f ** -0.5, pad)
        if case["train"]:
            s["dy"] = _normal(g, n, d, dt, 1e-3, pad)
    else:
        v = case["v"]
        s["h"] = _normal(g, n, d, dt, 1.0, pad)
        s["w"] = _normal(g, v, d, dt, 2 * d ** -0.5, pad)
        # popular nodes are met more often; held-out edges carry -1
        t = (torch.rand(n, device="cuda", generator=g).pow(3) * v).long().clamp_(max=v - 1)
        held = torch.rand(n, device="cuda", generator=g) < case["ignore"]
        s["target"] = t.masked_fill_(held, -1)
        if case["train"]:
            s["dloss"] = torch.rand(n, device="cuda", generator=g).add_(0.5).div_(n)
    return s


# ----------------------------------------------------------------------------------------------------------------------
def _act(name, g):
    """act(g) and act'(g)."""
    if name == "silu":
        sg = 1 / (1 + torch.exp(-g))
        return g * sg, sg * (1 + g * (1 - sg))
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(g * 2 ** -0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    pos = (g > 0).float()
    return g * pos, pos


def _plain_norm(s):
    dt = s["x"].dtype
    x, gamma, beta = s["x"].float(), s["gamma"].float(), s["beta"].float()
    if s["res"] is not None:
        x = (x + s["res"].float()).to(dt).float()   # the sum is a result of its own: what is normalised is what is kept
    c = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
    xhat = c * rstd
    out = {"y": (xhat * gamma + beta).to(dt)}
    if s["res"] is not None:
        out["sum"] = x.to(dt)
    if s["train"]:
        dy = s["dy"].float()
        a = dy * gamma
        dx = rstd * (a - a.mean(1, keepdim=True) - xhat * (a * xhat).mean(1, keepdim=True))
        if s["res"] is not None:
            dx = dx + s["ds"].float()
        out.update(dx=dx.to(dt), dgamma=(dy * xhat).sum(0).to(dt), dbeta=dy.sum(0).to(dt))
    return out


def _plain_ffn(s):
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(s["act"], g)
    h = a * u
    out = {"y": (h @ wd.t()).to(dt)}
    if s["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * da, dh * a
        out.update(dx=(dg @ wg + du @ wu).to(dt), dw_gate=(dg.t() @ x).to(dt), dw_up=(du.t() @ x).to(dt),
                   dw_down=(dy.t() @ h).to(dt))
    return out


def _plain_xent(s):
    dt = s["h"].dtype
    h, w, t = s["h"].float(), s["w"].float(), s["target"]
    keep = t >= 0
    at = t.clamp(min=0).unsqueeze(1)
    logits = h @ w.t()
    m = logits.max(1, keepdim=True).values
    e = torch.exp(logits - m)
    z = e.sum(1, keepdim=True)
    loss = (m + torch.log(z) - logits.gather(1, at)).squeeze(1) * keep
    out = {"loss": loss}
    if s["train"]:
        p = e / z
        p.scatter_add_(1, at, torch.full_like(at, -1, dtype=p.dtype))
        p = p * (s["dloss"] * keep).unsqueeze(1)
        out.update(dh=(p @ w).to(dt), dw=(p.t() @ h).to(dt))
    return out


def _own(s):
    from fast_b200 import ops
    if s["op"] == "norm":
        if s["res"] is None:
            y, mean, rstd = ops.layer_norm_fwd(s["x"], s["gamma"], s["beta"])
            out, x = {"y": y}, s["x"]
        else:
            y, x, mean, rstd = ops.layer_norm_fwd(s["x"], s["gamma"], s["beta"], res=s["res"])
            out = {"y": y, "sum": x}
        if s["train"]:
            out["dx"], out["dgamma"], out["dbeta"] = ops.layer_norm_bwd(s["dy"], x, s["gamma"], mean, rstd, ds=s["ds"])
    elif s["op"] == "ffn":
        w = s["w_gate"], s["w_up"], s["w_down"]
        out = {"y": ops.gated_ffn_fwd(s["x"], *w, act=s["act"])}
        if s["train"]:
            out["dx"], out["dw_gate"], out["dw_up"], out["dw_down"] = ops.gated_ffn_bwd(s["dy"], s["x"], *w,
                                                                                         act=s["act"])
    else:
        loss, lse = ops.softmax_xent_fwd(s["h"], s["w"], s["target"])
        out = {"loss": loss}
        if s["train"]:
            out["dh"], out["dw"] = ops.softmax_xent_bwd(s["h"], s["w"], s["target"], lse, s["dloss"])
    return out


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "ffn": _plain_ffn, "xent": _plain_xent}[state["op"]](state)


# ----------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """The definitions in fp64; the gradients are autograd's."""
    s = prepare(case, seed)
    F = torch.nn.functional
    need = case["train"]

    def wide(name):
        return s[name].double().requires_grad_(need)

    if case["op"] == "norm":
        x, gamma, beta = wide("x"), wide("gamma"), wide("beta")
        if case["res"]:
            # by definition the sum is kept in the rows' type, and the kept sum is normalised; d(sum)/dx = 1
            x = (s["x"].double() + s["res"].double()).to(s["x"].dtype).double().requires_grad_(need)
        y = F.layer_norm(x, (case["d"],), gamma, beta, 1e-5)
        out = {"y": y}
        if case["res"]:
            out["sum"] = x
        if need:
            out["dx"], out["dgamma"], out["dbeta"] = torch.autograd.grad(y, [x, gamma, beta], s["dy"].double())
            if case["res"]:
                out["dx"] = out["dx"] + s["ds"].double()
    elif case["op"] == "ffn":
        x, wg, wu, wd = wide("x"), wide("w_gate"), wide("w_up"), wide("w_down")
        act = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}[case["act"]]
        y = F.linear(act(F.linear(x, wg)) * F.linear(x, wu), wd)
        out = {"y": y}
        if need:
            grads = torch.autograd.grad(y, [x, wg, wu, wd], s["dy"].double())
            out["dx"], out["dw_gate"], out["dw_up"], out["dw_down"] = grads
    else:
        h, w = wide("h"), wide("w")
        loss = F.cross_entropy(F.linear(h, w), s["target"], ignore_index=-1, reduction="none")
        out = {"loss": loss}
        if need:
            out["dh"], out["dw"] = torch.autograd.grad(loss, [h, w], s["dloss"].double())
    return {k: v.detach() for k, v in out.items()}
