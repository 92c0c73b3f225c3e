"""Attention over a sliding window with visible first tokens, attention of drafted tokens over a paged cache, and the
movements of that cache's pages: the workloads they are measured on, in their plain forms and through the framework.

A case is a dict of plain values; ``kind`` names the operator:

* ``window``: ``ops.window_attention`` on queries, keys and values that are slices of one packed projection, with its
  gradients where ``grad`` is set (a training step of a sliding-window layer) or without (a prompt over a filled cache);
* ``cached``: ``ops.cached_attention`` — the tokens drafted for each sequence (a tree of them, or a chain) or its single
  next token, over pages or over a contiguous cache;
* ``copy``: ``ops.copy_pages`` — pages duplicated when sequences fork;
* ``compact``: ``ops.compact_rows`` — the accepted path of a drafted tree moved to the end of each sequence's cache.
"""
import math

import torch
import torch.nn.functional as F

own = False

UNLIMITED = 1 << 30


# ------------------------------------------------------------------------------------------------------------- cases
def _window(name=None, *, B, S, T, H, Hk, D, W, ns, logits, ragged, grad):
    c = dict(kind="window", B=B, S=S, T=T, H=H, Hk=Hk, D=D, W=W, ns=ns, logits=logits, ragged=ragged, grad=grad)
    return c if name is None else {"name": name, **c}


def _cached(name=None, *, B, N, H, Hk, D, prefix, page, tree, W, ns, logits):
    c = dict(kind="cached", B=B, N=N, H=H, Hk=Hk, D=D, prefix=prefix, page=page, tree=tree, W=W, ns=ns, logits=logits)
    return c if name is None else {"name": name, **c}


def _copy(name=None, *, blocks, layers, page, Hk, D, pairs):
    c = dict(kind="copy", blocks=blocks, layers=layers, page=page, Hk=Hk, D=D, pairs=pairs)
    return c if name is None else {"name": name, **c}


def _compact(name=None, *, B, prefix, layers, page, Hk, D, N, path):
    c = dict(kind="compact", B=B, prefix=prefix, layers=layers, page=page, Hk=Hk, D=D, N=N, path=path)
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # a training step of one sliding-window layer with grouped heads: two sequences of 4096
        _window("window_step", B=2, S=4096, T=4096, H=16, Hk=4, D=128, W=1024, ns=4, logits=False, ragged=False, grad=True),
        # the same layer on one long document
        _window("window_long", B=1, S=16384, T=16384, H=16, Hk=4, D=128, W=2048, ns=16, logits=False, ragged=False, grad=True),
        # a padded batch of short, odd-sized sequences; three query heads to a key head, learned sink logits
        _window("window_padded", B=3, S=1333, T=1333, H=6, Hk=2, D=64, W=200, ns=3, logits=True, ragged=True, grad=True),
        # the last 77 tokens of a prompt over a cache that holds the others
        _window("window_prompt", B=1, S=77, T=650, H=8, Hk=8, D=96, W=256, ns=1, logits=False, ragged=False, grad=False),
        # one request's next token: latency alone
        _cached("decode_one", B=1, N=1, H=16, Hk=4, D=128, prefix=900, page=16, tree="chain", W=512, ns=4, logits=False),
        # a batch of single next tokens over a contiguous cache, a window of each
        _cached("decode_window", B=128, N=1, H=16, Hk=4, D=64, prefix=8000, page=0, tree="chain", W=1024, ns=4, logits=True),
        # a serving batch that verifies a small drafted tree for every request
        _cached("tree_batch", B=64, N=12, H=32, Hk=8, D=128, prefix=8192, page=64, tree="own", W=0, ns=0, logits=False),
        # one long conversation that verifies a large drafted tree
        _cached("tree_long", B=1, N=61, H=16, Hk=2, D=128, prefix=131000, page=64, tree="shared", W=0, ns=0, logits=False),
        # one request forks: its last, partly filled page is duplicated
        _copy("fork_one", blocks=64, layers=4, page=16, Hk=4, D=128, pairs=1),
        # a batch of forks, or a pool that is put in order
        _copy("fork_batch", blocks=1024, layers=16, page=16, Hk=8, D=128, pairs=500),
        # one request accepts a path of its drafted tree
        _compact("accept_one", B=1, prefix=700, layers=4, page=16, Hk=4, D=128, N=16, path=3),
        # every request of a batch does
        _compact("accept_batch", B=64, prefix=500, layers=8, page=64, Hk=8, D=128, N=60, path=7),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["window", "window", "cached", "cached", "cached", "copy", "compact"])
    if kind == "window":
        Hk, g = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 5, 8])
        while Hk * g > 16:
            Hk, g = max(1, Hk // 2), max(1, g - 1)
        grad = rng.random() < 0.7
        S = _spread(rng, 2 if grad else 1, 8192)
        B = max(1, min(rng.choice([1, 2, 3, 5]), 12000 // S))
        T = S if grad and rng.random() < 0.8 else S + _spread(rng, 1, 2000)
        # where every query sees a single key the scores' gradients are zero: a window of two keys is the least to train with
        W = rng.choice([0, _spread(rng, 2 if grad else 1, 2048), _spread(rng, 32, 2048)]) if S <= 2048 else _spread(rng, 16, 2048)
        return _window(B=B, S=S, T=T, H=Hk * g, Hk=Hk, D=rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128]), W=W,
                       ns=rng.choice([0, 1, 4, 4, 17, 130]), logits=rng.random() < 0.3, ragged=rng.random() < 0.4, grad=grad)
    if kind == "cached":
        Hk, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        tree = rng.choice(["chain", "own", "own", "shared"])
        N = rng.choice([1, _spread(rng, 1, 400)]) if tree == "chain" else _spread(rng, 1, 64)
        B = _spread(rng, 1, 64)
        prefix = _spread(rng, 1, max(2, min(100000, 2_000_000 // (B * Hk), 100_000_000 // (B * Hk * g * N))))
        return _cached(B=B, N=N, H=Hk * g, Hk=Hk, D=rng.choice([32, 64, 64, 96, 128, 128]), prefix=prefix,
                       page=rng.choice([0, 8, 16, 16, 24, 32, 48, 64, 128, 256]), tree=tree,
                       W=rng.choice([0, 0, _spread(rng, 1, 4096)]), ns=rng.choice([0, 1, 4, 20, 150]), logits=rng.random() < 0.3)
    if kind == "copy":
        blocks = _spread(rng, 4, 1024)
        return _copy(blocks=blocks, layers=_spread(rng, 1, 16), page=rng.choice([1, 8, 15, 16, 16]), Hk=rng.choice([1, 2, 3, 4, 8]),
                     D=rng.choice([24, 64, 80, 128]), pairs=_spread(rng, 1, blocks // 2))
    path = _spread(rng, 1, 16)
    return _compact(B=_spread(rng, 1, 64), prefix=_spread(rng, 1, 1500), layers=_spread(rng, 1, 16), page=rng.choice([1, 7, 16, 16, 64]),
                    Hk=rng.choice([1, 2, 3, 4, 8]), D=rng.choice([24, 64, 80, 128]), N=rng.randint(2 * path, 64), path=path)


# ------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _lengths(B, most, seed):
    """B lengths from about half of ``most`` up to it, in an order that goes by the seed; their sum is the case's."""
    n = torch.tensor([most - (b * (most // 2)) // max(1, B - 1) if B > 1 else most for b in range(B)], dtype=torch.int32)
    return n[torch.randperm(B, generator=torch.Generator().manual_seed(int(seed)))]


def _trees(count, N, seed):
    """``count`` random trees of drafted tokens in the order in which they were drafted: bit m of word n is set where node n
    is node m or descends from it. All but the first have a few places at the end that hold no node (words of 0)."""
    r = torch.Generator().manual_seed(int(seed) + 101)
    words = []
    for t in range(count):
        n_nodes = N if t == 0 else max(1, N - int(torch.randint(0, max(1, N // 4), (1,), generator=r)))
        row = []
        for n in range(n_nodes):
            parent = int(torch.randint(-1, n, (1,), generator=r)) if n else -1
            row.append((row[parent] if parent >= 0 else 0) | (1 << n))
        row += [0] * (N - n_nodes)
        words.append([w - (1 << 64) if w >= 1 << 63 else w for w in row])
    return torch.tensor(words, dtype=torch.int64)


def prepare(case, seed):
    g, c = _gen(seed), case
    bf = torch.bfloat16
    rand = lambda *s: torch.randn(*s, device="cuda", dtype=bf, generator=g)  # noqa: E731
    if c["kind"] == "window":
        B, S, T, H, Hk, D = (c[n] for n in ("B", "S", "T", "H", "Hk", "D"))
        packed = rand(B, T, (H + 2 * Hk) * D)          # one projection; the queries are its last S rows
        part = lambda a, n: packed[..., a * D:(a + n) * D].view(B, T, n, D)  # noqa: E731
        q, k, v = part(0, H)[:, T - S:], part(H, Hk), part(H + Hk, Hk)
        sinks = rand(H) if c["logits"] else None
        state = {"case": c, "lengths": _lengths(B, T, seed).cuda() if c["ragged"] else None}
        if c["grad"]:
            q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
            sinks = sinks.requires_grad_() if sinks is not None else None
            state["do"] = rand(B, S, H, D)
        return {**state, "q": q, "k": k, "v": v, "sinks": sinks}
    if c["kind"] == "cached":
        B, N, H, Hk, D, page = (c[n] for n in ("B", "N", "H", "Hk", "D", "page"))
        prefix = _lengths(B, c["prefix"], seed).cuda()
        rows = c["prefix"] + N + 5
        if page:
            width = -(-rows // page)
            k, v = rand(B * width + 3, page, Hk, D), rand(B * width + 3, page, Hk, D)
            table = torch.randperm(B * width + 3, device="cuda", generator=g)[:B * width].view(B, width).int()
        else:
            k, v, table = rand(B, rows, Hk, D), rand(B, rows, Hk, D), None
        tree = None if c["tree"] == "chain" else _trees(1, N, seed)[0] if c["tree"] == "shared" else _trees(B, N, seed)
        return {"case": c, "q": rand(B, N, H, D), "k": k, "v": v, "table": table, "prefix": prefix,
                "tree": None if tree is None else tree.cuda(), "sinks": rand(H) if c["logits"] else None}
    layers, page, Hk, D = (c[n] for n in ("layers", "page", "Hk", "D"))
    if c["kind"] == "copy":
        k, v = rand(c["blocks"], layers, page, Hk, D), rand(c["blocks"], layers, page, Hk, D)
        ids = torch.randperm(c["blocks"], generator=torch.Generator().manual_seed(int(seed)))[:2 * c["pairs"]]
        return {"case": c, "k": k, "v": v, "src": ids[:c["pairs"]].int().cuda(), "dst": ids[c["pairs"]:].int().cuda()}
    B, N, path = c["B"], c["N"], c["path"]
    width = -(-(c["prefix"] + N) // page)
    k, v = rand(B * width, layers, page, Hk, D), rand(B * width, layers, page, Hk, D)
    table = torch.randperm(B * width, device="cuda", generator=g).view(B, width).int()
    r = torch.Generator().manual_seed(int(seed))
    # the tree's first level is wider than any path is long, so a path begins behind the places that it moves to
    picks = torch.stack([torch.randperm(N - path, generator=r)[:path].sort().values + path for _ in range(B)])
    counts = torch.randint(0, path + 1, (B,), generator=r)
    counts[0] = path
    return {"case": c, "k": k, "v": v, "table": table, "start": _lengths(B, c["prefix"], seed).cuda(), "path": picks.int().cuda(),
            "counts": counts.int().cuda()}


# ------------------------------------------------------------------------------------------------------------- plain forms
def _plain_weights(scores, seen, sinks):
    """Softmax over the last axis where ``seen``, in 32 bits; ``sinks`` (broadcast to the rows) is the logit of one more key
    whose value is 0. A row that sees nothing has no weights at all."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top)).detach()
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _plain_window(q, k, v, sinks, lengths, W, ns):
    """Blocks of C queries against the C + W − 1 keys that their windows cover and against the first ``ns`` keys."""
    B, S, H, D = q.shape
    T, Hk = k.shape[1], k.shape[2]
    off, g = T - S, H // k.shape[2]
    W = min(W or T, T)
    C = min(S, 512)
    nb = -(-S // C)
    dev = q.device
    qb = F.pad(q, (0, 0, 0, 0, 0, nb * C - S)).view(B, nb, C, Hk, g, D)
    back = nb * C - S
    first = min(ns, T)

    def blocks(x):          # [B, nb, C + W - 1, Hk, D], and the first rows behind them
        wide = F.pad(x, (0, 0, 0, 0, W - 1, back))[:, off:].unfold(1, C + W - 1, C).permute(0, 1, 4, 2, 3)
        return torch.cat([wide, x[:, None, :first].expand(B, nb, first, Hk, D)], 2)

    kb, vb = blocks(k), blocks(v)
    row = torch.arange(nb, device=dev)[:, None] * C
    qp = off + row + torch.arange(C, device=dev)                                     # [nb, C] positions
    kp = off + row + torch.arange(C + W - 1, device=dev) - (W - 1)                   # [nb, C + W - 1]
    near = (kp[:, None] <= qp[:, :, None]) & (qp[:, :, None] - kp[:, None] < W) & (kp[:, None] >= 0)
    sp = torch.arange(first, device=dev)
    far = (qp[:, :, None] - sp >= W) & (sp <= qp[:, :, None])
    seen = torch.cat([near, far], -1)[None]                                          # [1, nb, C, K]
    at = torch.cat([kp, sp.expand(nb, first)], 1)
    if lengths is not None:
        seen = seen & (at[None, :, None] < lengths.view(B, 1, 1, 1))
    vb = torch.where(seen.any(2)[..., None, None], vb, torch.zeros_like(vb))
    s = torch.einsum("bnchgd,bnkhd->bnhgck", qb, kb) * D ** -0.5
    p = _plain_weights(s, seen[:, :, None, None], None if sinks is None else sinks.view(1, 1, Hk, g, 1, 1))
    o = torch.einsum("bnhgck,bnkhd->bnchgd", p, vb)
    return o.reshape(B, nb * C, H, D)[:, :S]


def _plain_cached(q, k, v, table, prefix, tree, sinks, W, ns):
    B, N, H, D = q.shape
    Hk = k.shape[2]
    if table is not None:
        k, v = (x[table.long()].flatten(1, 2) for x in (k, v))
    T, dev = k.shape[1], q.device
    W = W or UNLIMITED
    if tree is None:
        bits = torch.ones(N, N, dtype=torch.bool, device=dev).tril()[None].expand(B, N, N)
    else:
        bits = ((tree.view(-1, N, 1) >> torch.arange(N, device=dev)) & 1).bool().expand(B, N, N)
    depth = bits.sum(-1) - 1                                                         # [B, N]
    pos = prefix[:, None] + depth
    kp = torch.arange(T, device=dev)
    old = (kp < prefix[:, None])[:, None] & ((pos[..., None] - kp < W) | (kp < ns)) & (depth >= 0)[..., None]
    node = (kp - prefix[:, None]).clamp(0, N - 1)                                    # [B, T]
    is_node = (kp >= prefix[:, None]) & (kp < prefix[:, None] + N)
    kdepth = depth.gather(1, node)
    new = bits.gather(2, node[:, None].expand(B, N, T)) & is_node[:, None]
    new = new & ((depth[..., None] - kdepth[:, None] < W) | (prefix[:, None] + kdepth < ns)[:, None])
    seen = old | new                                                                 # [B, N, T]
    v = torch.where(seen.any(1)[..., None, None], v, torch.zeros_like(v)).float()
    s = torch.einsum("bnhgd,bkhd->bhgnk", q.float().view(B, N, Hk, H // Hk, D), k.float()) * D ** -0.5
    p = _plain_weights(s, seen[:, None, None], None if sinks is None else sinks.float().view(1, Hk, H // Hk, 1, 1))
    return torch.einsum("bhgnk,bkhd->bnhgd", p, v).reshape(B, N, H, D).to(q.dtype)


def _plain_compact(pool, table, start, path, counts):
    page = pool.shape[2]
    at = torch.arange(path.shape[1], device=path.device)
    to = (start[:, None] + at).long()
    fro = torch.where(at < counts[:, None], start[:, None] + path, to).long()         # the others stay where they are
    rows = pool[table.gather(1, fro // page).long(), :, fro % page]
    pool[table.gather(1, to // page).long(), :, to % page] = rows


def run(state):
    c = state["case"]
    if c["kind"] == "window":
        q, k, v, sinks = (state[n] for n in ("q", "k", "v", "sinks"))
        leaves = [t for t in (q, k, v, sinks) if t is not None]
        if own:
            from cppmega_mlx_b200 import ops
            o = ops.window_attention(q, k, v, window=c["W"] or None, sink_tokens=c["ns"], sinks=sinks, key_lengths=state["lengths"])
        else:
            wide = [None if t is None else t.float() for t in (q, k, v, sinks)]
            o = _plain_window(*wide, state["lengths"], c["W"], c["ns"]).to(q.dtype)
        out = {"o": o.detach()}
        if c["grad"]:
            out["grads"] = list(torch.autograd.grad(o, leaves, state["do"]))
        return out
    if c["kind"] == "cached":
        args = [state[n] for n in ("q", "k", "v", "table", "prefix")]
        if own:
            from cppmega_mlx_b200 import ops
            return ops.cached_attention(*args, tree=state["tree"], window=c["W"] or None, sink_tokens=c["ns"], sinks=state["sinks"])
        return _plain_cached(*args, state["tree"], state["sinks"], c["W"], c["ns"])
    k, v = state["k"], state["v"]
    if c["kind"] == "copy":
        src, dst = state["src"], state["dst"]
        if own:
            from cppmega_mlx_b200 import ops
            ops.copy_pages((k, v), src, dst)
        else:
            k[dst.long()] = k[src.long()]
            v[dst.long()] = v[src.long()]
        return k, v
    args = [state[n] for n in ("table", "start", "path", "counts")]
    if own:
        from cppmega_mlx_b200 import ops
        ops.compact_rows((k, v), *args)
    else:
        _plain_compact(k, *args)
        _plain_compact(v, *args)
    return k, v


# ------------------------------------------------------------------------------------------------------------- sizes
def work(case):
    c = case
    if c["kind"] == "window":
        B, S, T, H, Hk, D = (c[n] for n in ("B", "S", "T", "H", "Hk", "D"))
        W = c["W"] or T
        lens = _lengths(B, T, 0).tolist() if c["ragged"] else [T] * B
        pairs = sum(max(0, min(p + 1, n) - max(0, p - W + 1)) + min(c["ns"], n, max(0, p - W + 1)) for n in lens for p in range(T - S, T))
        fwd = 4.0 * D * H * pairs
        moved = 2.0 * D * B * (2 * S * H + 2 * T * Hk)
        return {"flops": fwd * 3.5, "bytes": moved * 2 + 2.0 * D * B * S * H} if c["grad"] else {"flops": fwd, "bytes": moved}
    if c["kind"] == "cached":
        B, N, H, Hk, D = (c[n] for n in ("B", "N", "H", "Hk", "D"))
        W = c["W"] or UNLIMITED
        keys = sum(min(n, W) + min(c["ns"], max(0, n - W)) + N for n in _lengths(B, c["prefix"], 0).tolist())
        return {"flops": 4.0 * D * H * N * keys, "bytes": 4.0 * D * Hk * keys + 4.0 * B * N * H * D}
    row = 2.0 * 2.0 * c["layers"] * c["Hk"] * c["D"]           # one token's keys and values, all layers
    if c["kind"] == "copy":
        return {"bytes": 2.0 * row * c["page"] * c["pairs"], "flops": 0}
    return {"bytes": 2.0 * row * (c["path"] + (c["B"] - 1) * c["path"] / 2), "flops": 0}


# ------------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_window(st, c):
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    B, S, H, D = q.shape
    T, Hk = k.shape[1], k.shape[2]
    g, off, W, ns = H // Hk, T - S, c["W"] or T, c["ns"]
    do = st["do"].double() if c["grad"] else None
    out = torch.zeros_like(q)
    dq, dk, dv, ds = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), q.new_zeros(H)
    scale = 1.0 / math.sqrt(D)
    step = 256
    for b in range(B):
        n_keys = T if st["lengths"] is None else int(st["lengths"][b])
        for i0 in range(0, S, step):
            i1 = min(S, i0 + step)
            p = torch.arange(off + i0, off + i1, device=q.device)
            lo = max(0, off + i0 - W + 1)
            j = torch.arange(n_keys, device=q.device)
            j = j[(j < ns) | ((j >= lo) & (j < off + i1))]
            allowed = (j[None] <= p[:, None]) & ((j[None] > p[:, None] - W) | (j[None] < ns))
            for h in range(H):
                hk = h // g
                qi, kj, vj = q[b, i0:i1, h], k[b, j, hk], v[b, j, hk]
                e = torch.where(allowed, (qi @ kj.T) * scale, q.new_tensor(-math.inf))
                if st["sinks"] is not None:
                    e = torch.cat([e, st["sinks"].detach().double()[h].expand(i1 - i0, 1)], 1)
                w = torch.nan_to_num(torch.softmax(e, 1)) if e.shape[1] else e
                a, rest = w[:, :j.numel()], w[:, j.numel():]
                oi = a @ vj
                out[b, i0:i1, h] = oi
                if do is None:
                    continue
                gi = do[b, i0:i1, h]
                along = (gi * oi).sum(1, keepdim=True)
                dv[b].index_put_((j, torch.full_like(j, hk)), a.T @ gi, accumulate=True)
                da = a * (gi @ vj.T - along) * scale
                dq[b, i0:i1, h] = da @ kj
                dk[b].index_put_((j, torch.full_like(j, hk)), da.T @ qi, accumulate=True)
                ds[h] -= (rest * along).sum()
    res = {"o": out}
    if do is not None:
        res["grads"] = [dq, dk, dv] + ([ds] if st["sinks"] is not None else [])
    return res


def _exact_cached(st, c):
    q = st["q"].double()
    B, N, H, D = q.shape
    Hk = st["k"].shape[2]
    g, W, ns = H // Hk, c["W"] or UNLIMITED, c["ns"]
    out = torch.zeros_like(q)
    for b in range(B):
        n_old = int(st["prefix"][b])
        at = torch.arange(n_old + N, device=q.device)
        if st["table"] is None:
            k, v = st["k"][b, :n_old + N].double(), st["v"][b, :n_old + N].double()
        else:
            ps = st["k"].shape[1]
            pages = st["table"][b].long()[at // ps]
            k, v = st["k"][pages, at % ps].double(), st["v"][pages, at % ps].double()
        if st["tree"] is None:
            words = [(1 << (n + 1)) - 1 for n in range(N)]
        else:
            words = [w % (1 << 64) for w in (st["tree"] if st["tree"].dim() == 1 else st["tree"][b]).tolist()]
        deep = [bin(w).count("1") - 1 for w in words]
        allowed = torch.zeros(N, n_old + N, dtype=torch.bool)
        far = torch.arange(n_old)
        for n, w in enumerate(words):
            if not w:
                continue
            allowed[n, :n_old] = (n_old + deep[n] - far < W) | (far < ns)
            allowed[n, n_old:] = torch.tensor([bool(w >> m & 1) and (deep[n] - deep[m] < W or n_old + deep[m] < ns) for m in range(N)])
        allowed = allowed.to(q.device)
        for h in range(H):
            e = torch.where(allowed, q[b, :, h] @ k[:, h // g].T / math.sqrt(D), q.new_tensor(-math.inf))
            if st["sinks"] is not None:
                e = torch.cat([e, st["sinks"].double()[h].expand(N, 1)], 1)
            w = torch.nan_to_num(torch.softmax(e, 1))[:, :n_old + N]
            out[b, :, h] = w @ v[:, h // g]
    return out


def exact(case, seed):
    if case["kind"] in ("copy", "compact"):
        return None                                    # rows are moved, nothing is computed
    st = prepare(case, seed)
    return (_exact_window if case["kind"] == "window" else _exact_cached)(st, case)
