"""Windowed / cached attention in 64 bits, with elementwise bounds on what the bf16 kernels may be off by.

Roundings the kernels make (each at most half a step, h = finfo(bf16).eps / 2 = 2**-8, relative to the value): the outputs and
gradients, once, when written; P before P.V and before dV's product; dS before dQ's and dK's products; and o before
delta = do.o.  Everything else is fp32, bounded by ``F32`` relative to the sums of absolute values: products accumulate over at most a few
hundred terms (2**-24 each), the exponent's argument carries 2**-24 of its own size (below 2**6 here) and ex2.approx 2**-22.
"""
import torch

H = torch.finfo(torch.bfloat16).eps / 2
F32 = 2.0 ** -14


def visible(s, t, window, ns, lengths=None, device=None):
    p = torch.arange(t - s, t, device=device)[:, None]
    j = torch.arange(t, device=device)[None]
    w = t + s + 1 if window is None else window
    m = ((j <= p) & ((p - j < w) | (j < ns)))[None]
    return m if lengths is None else m & (j[None] < lengths.view(-1, 1, 1))


def attention64(q, k, v, seen, sinks=None, scale=None, do=None):
    """q [B,S,H,D], k/v [B,T,Hk,D], seen [B|1,S,T].  Returns {name: (value, bound)} for o and, with ``do``, dq, dk, dv, ds."""
    b, s, h, d = q.shape
    t, hk = k.shape[1], k.shape[2]
    g = h // hk
    scale = d ** -0.5 if scale is None else scale
    seen = seen.expand(b, s, t)
    clean = lambda x: torch.where(seen.any(1)[:, :, None, None], x, torch.zeros_like(x)).double()  # noqa: E731
    q, k, v = q.double(), clean(k), clean(v)
    kk, vv = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    sc = torch.einsum("bshd,bthd->bhst", q, kk) * scale
    sc = sc.masked_fill(~seen[:, None], float("-inf"))
    full = sc if sinks is None else torch.cat([sc, sinks.double().view(1, h, 1, 1).expand(b, h, s, 1)], -1)
    w = torch.nan_to_num(torch.softmax(full, -1))
    p, ps = w[..., :t], w[..., t:]
    o = torch.einsum("bhst,bthd->bshd", p, vv)
    oa = torch.einsum("bhst,bthd->bshd", p, vv.abs())
    eo = (H + F32) * oa + H * o.abs() * (1 + H) + 1e-30
    res = {"o": (o, eo)}
    if do is None:
        return res
    do = do.double()
    dp = torch.einsum("bshd,bthd->bhst", do, vv)
    delta = (do * o).sum(-1).transpose(1, 2)[..., None]                       # [B,H,S,1]
    edelta = (do.abs() * eo).sum(-1).transpose(1, 2)[..., None]
    ds = p * (dp - delta)
    # error of dS itself: its rounding, delta's, and fp32 in p and dp
    dpa = torch.einsum("bshd,bthd->bhst", do.abs(), vv.abs())
    eds = H * ds.abs() + p * (edelta + F32 * (dpa + delta.abs())) * (1 + H)
    group = lambda x: x.view(b, t, hk, g, -1).sum(3)  # noqa: E731

    def out(value, bound):
        return value, (bound + H * (value.abs() + bound)) * 1.01 + 1e-30
    res["dq"] = out(scale * torch.einsum("bhst,bthd->bshd", ds, kk),
                    scale * torch.einsum("bhst,bthd->bshd", eds + F32 * ds.abs(), kk.abs()))
    res["dk"] = out(scale * group(torch.einsum("bhst,bshd->bthd", ds, q)),
                    scale * group(torch.einsum("bhst,bshd->bthd", eds + F32 * ds.abs(), q.abs())))
    res["dv"] = out(group(torch.einsum("bhst,bshd->bthd", p, do)), (H + F32) * group(torch.einsum("bhst,bshd->bthd", p, do.abs())))
    if sinks is not None:
        res["ds"] = out(-(ps * delta).sum((0, 2, 3)), F32 * (ps * dpa.mul(p).sum(-1, keepdim=True)).sum((0, 2, 3)))
    return res


def check(got, want, name):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    over = (got.double() - value).abs() - bound
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    worst = int(over.argmax())
    assert float(over.max()) <= 0, (f"{name}: off by {float((got.double() - value).abs().flatten()[worst]):.3g} where "
                                    f"{float(bound.flatten()[worst]):.3g} is allowed, at {worst}")


def cached_visible(prefix, n, t, bits, window, ns, device=None):
    """[B, N, T] by the definition, token by token (bits: [B][N][N] lists of truth values)."""
    b = len(prefix)
    seen = torch.zeros(b, n, t, dtype=torch.bool)
    for i in range(b):
        depth = [sum(row) - 1 for row in bits[i]]
        for x in range(n):
            if depth[x] < 0:
                continue
            pos = prefix[i] + depth[x]
            for j in range(prefix[i]):
                seen[i, x, j] = window is None or pos - j < window or j < ns
            for m in range(n):
                if bits[i][x][m]:
                    pm = prefix[i] + depth[m]
                    seen[i, x, prefix[i] + m] = window is None or pos - pm < window or pm < ns
    return seen.to(device)
