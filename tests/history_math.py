"""Event histories in plain torch: the short causal convolution, the selective
state space scan and dropout's draws, written from their definitions, row by row,
differentiable, in whatever precision the inputs have."""
import torch


def spans(starts, rows):
    """(begin, end) of every sequence; starts None: one sequence."""
    s = [0, rows] if starts is None else [int(v) for v in starts]
    return list(zip(s, s[1:]))


def short_conv(x, w, bias, starts, init, act):
    """(y, final) of fast_b200.ops.short_conv_fwd."""
    k, y, final = w.shape[1], [None] * x.shape[0], []
    for i, (b, e) in enumerate(spans(starts, x.shape[0])):
        past = x.new_zeros(k - 1, x.shape[1]) if init is None else init[i]
        xe = torch.cat([past, x[b:e]])
        for t in range(e - b):
            p = (xe[t:t + k] * w.t()).sum(0) + (0 if bias is None else bias)
            y[b + t] = p * torch.sigmoid(p) if act == "silu" else p
        final.append(xe[e - b:])
    zero = torch.zeros_like(x[0]) if len(x) else None
    y = torch.stack([zero if v is None else v for v in y]) if y else torch.zeros_like(x)
    return y, torch.stack(final) if final else x.new_zeros(0, k - 1, x.shape[1])


def selective_scan(u, delta, A, B, C, D, z, delta_bias, starts, init, softplus):
    """(y, final) of fast_b200.ops.selective_scan_fwd; B, C [rows, groups, N]."""
    rows, d = u.shape
    per = d // B.shape[1]
    x = delta if delta_bias is None else delta + delta_bias
    dt = torch.logaddexp(x, torch.zeros_like(x)) if softplus else x
    y, final = [None] * rows, []
    for i, (b, e) in enumerate(spans(starts, rows)):
        h = torch.zeros_like(A) if init is None else init[i]
        for t in range(b, e):
            h = torch.exp(dt[t].unsqueeze(1) * A) * h + (dt[t] * u[t]).unsqueeze(1) * B[t].repeat_interleave(per, 0)
            v = (C[t].repeat_interleave(per, 0) * h).sum(1)
            if D is not None:
                v = v + D * u[t]
            y[t] = v if z is None else v * z[t] * torch.sigmoid(z[t])
        final.append(h)
    zero = torch.zeros_like(u[0]) if rows else None
    y = torch.stack([zero if v is None else v for v in y]) if rows else torch.zeros_like(u)
    return y, torch.stack(final) if final else A.new_zeros(0, *A.shape)


def philox(rows, cols, seed, offset):
    """Words [rows, cols] of Philox4x32-10: word c % 4 at counter (c / 4, row, offset), key seed."""
    out, mask = [], 0xFFFFFFFF
    for r in range(rows):
        line = []
        for q in range((cols + 3) // 4):
            c, k = [q, r, offset & mask, offset >> 32 & mask], [seed & mask, seed >> 32]
            for _ in range(10):
                p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
                c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & mask, (p0 >> 32) ^ c[3] ^ k[1], p0 & mask]
                k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
            line += c
        out.append(line[:cols])
    return torch.tensor(out, dtype=torch.int64).view(rows, cols)


def keep_scale(rows, cols, p, seed, offset):
    """0 or 1 / (1 - p) for every element, fp64."""
    f = (philox(rows, cols, seed, offset) >> 8).double() * 2.0 ** -24
    p32 = float(torch.tensor(p, dtype=torch.float32))
    return (f >= p32).double() / (1 - p)
