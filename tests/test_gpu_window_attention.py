"""The kernels of windowed attention, cached attention and page movements against 64-bit oracles with derived bounds."""
import pytest
import torch

from tests import _window_oracle as W

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _done():
    from cppmega_mlx_b200.ops import _backend as B
    torch.cuda.synchronize()
    B.check_status()


def _rand(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale).to(BF)


WINDOW = [
    # B, S, T, H, Hk, Dq, Dv, window, ns, logits, lengths
    (1, 1, 1, 1, 1, 8, 8, None, 0, False, None),
    (1, 1, 700, 4, 2, 64, 64, 100, 3, True, None),              # a single next token
    (2, 33, 33, 4, 1, 64, 64, 5, 2, False, None),
    (2, 129, 129, 3, 3, 128, 128, None, 0, False, None),        # one row past a tile
    (1, 128, 300, 8, 2, 128, 128, 40, 17, True, [131]),         # lengths end inside the cache
    (2, 200, 200, 6, 2, 96, 40, 64, 130, False, [200, 77]),     # three heads to a group, more first tokens than a tile, ragged
    (1, 515, 515, 7, 1, 80, 128, 129, 1, True, None),
    (1, 700, 700, 4, 4, 64, 64, 1, 0, True, None),              # a window of the token itself
    (2, 384, 384, 2, 1, 128, 64, 128, 0, False, [0, 384]),      # a sequence without any key
    (1, 260, 391, 64, 1, 32, 32, 50, 4, False, None),           # 64 heads to a group
    (1, 2100, 2100, 2, 2, 64, 64, 33, 20, True, [2050]),        # many rows behind the first tokens: split over thread blocks
    (1, 90, 90, 5, 5, 16, 24, 300, 300, False, None),           # window and first tokens past the sequence
]


def _window_inputs(case, seed=0):
    b, s, t, h, hk, dq, dv, window, ns, logits, lengths = case
    q, k, v, do = _rand(b, s, h, dq, seed=seed), _rand(b, t, hk, dq, seed=seed + 1), _rand(b, t, hk, dv, seed=seed + 2), _rand(b, s, h, dv, seed=seed + 3)
    sinks = _rand(h, seed=seed + 4) if logits else None
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return q, k, v, do, sinks, n, dict(window=window, sink_tokens=ns, key_lengths=n)


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_window_forward_and_backward(case):
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    b, s, t, window, ns = case[0], case[1], case[2], case[7], case[8]
    q, k, v, do, sinks, n, kw = _window_inputs(case)
    leaves = [x.requires_grad_() for x in (q, k, v, sinks) if x is not None]
    before = B.launch_count("window_fwd"), B.launch_count("window_bwd")
    o = ops.window_attention(q, k, v, sinks=sinks, **kw)
    grads = torch.autograd.grad(o, leaves, do)
    assert (B.launch_count("window_fwd"), B.launch_count("window_bwd")) == (before[0] + 1, before[1] + 1)
    _done()
    with torch.no_grad():
        alone = ops.window_attention(q, k, v, sinks=sinks, **kw)
    assert torch.equal(alone, o)
    ref = W.attention64(*(x.detach() for x in (q, k, v)), W.visible(s, t, window, ns, n, "cuda"), None if sinks is None else sinks.detach(), do=do)
    for got, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv", "ds")):
        W.check(got, ref[name], name)


@pytest.mark.parametrize("scale,mag", [(1.0, 1.0), (0.01, 1.0), (None, 6.0)])
def test_window_scales_and_sharp_rows(scale, mag):
    from cppmega_mlx_b200 import ops
    q, k, v, do = (_rand(1, 300, 2, 64, seed=i, scale=mag if i < 2 else 1.0) for i in range(4))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = ops.window_attention(q, k, v, window=90, sink_tokens=5, scale=scale)
    grads = torch.autograd.grad(o, leaves, do)
    _done()
    ref = W.attention64(*(x.detach() for x in leaves), W.visible(300, 300, 90, 5, device="cuda"), scale=scale, do=do)
    # scores reach mag^2 * 64^0.5 * 4 (or * 8 with scale 1): their fp32 error, 2^-24 of the sum of 64 products, grows with them
    grow = 1 + 8 * mag * mag * (8 if scale == 1.0 else 1) * 2.0 ** -17 / W.H
    for got, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv")):
        W.check(got, (ref[name][0], ref[name][1] * grow), name)


def test_window_layouts_and_partial_gradients():
    """Slices of a packed projection, an expanded output gradient, a broadcast key head, a transposed layout; only some gradients."""
    from cppmega_mlx_b200 import ops
    x = _rand(2, 150, (4 + 2 + 2) * 64)
    q, k, v = x[..., :256].view(2, 150, 4, 64), x[..., 256:384].view(2, 150, 2, 64), x[..., 384:].view(2, 150, 2, 64)
    seen = W.visible(150, 150, 40, 2, device="cuda")

    def run(q, k, v, do, which):
        leaves = [(t.detach().requires_grad_() if n in which else t.detach()) for n, t in zip("qkv", (q, k, v))]
        o = ops.window_attention(*leaves, window=40, sink_tokens=2)
        g = torch.autograd.grad(o, [t for t in leaves if t.requires_grad], do)
        _done()
        ref = W.attention64(q, k, v, seen, do=do)
        W.check(o.detach(), ref["o"], "o")
        for got, n in zip(g, which):
            W.check(got, ref["d" + n], "d" + n)
    do = _rand(2, 150, 4, 64, seed=9)
    run(q, k, v, do, "qkv")
    run(q, k, v, do[:, :1].expand(2, 150, 4, 64), "q")
    run(q, k[:, :, :1].expand(2, 150, 2, 64), v, do, "kv")
    run(q.transpose(1, 2).contiguous().transpose(1, 2), k, v[..., torch.arange(63, -1, -1, device="cuda")], do.transpose(1, 3).contiguous().transpose(1, 3), "v")
    whole = x.detach().clone().requires_grad_()       # through the views, as a layer does
    qq, kk, vv = whole[..., :256].view(2, 150, 4, 64), whole[..., 256:384].view(2, 150, 2, 64), whole[..., 384:].view(2, 150, 2, 64)
    ops.window_attention(qq, kk, vv, window=40, sink_tokens=2).backward(do)
    ref = W.attention64(q, k, v, seen, do=do)
    W.check(whole.grad[..., 256:384].reshape(2, 150, 2, 64), ref["dk"], "dk")


def test_window_unseen_values_and_repeatability():
    """What lies behind the lengths may be NaN; the same call gives the same bits."""
    from cppmega_mlx_b200 import ops
    case = (2, 500, 500, 4, 2, 128, 128, 70, 150, True, [500, 301])
    outs = []
    for poison in (False, True, True):
        q, k, v, do, sinks, n, kw = _window_inputs(case)
        if poison:
            k[1, 301:], v[1, 301:] = float("nan"), float("inf")
        leaves = [x.requires_grad_() for x in (q, k, v, sinks)]
        o = ops.window_attention(q, k, v, sinks=sinks, **kw)
        outs.append([o.detach(), *torch.autograd.grad(o, leaves, do)])
        _done()
    for a, b, c in zip(*outs):
        assert torch.equal(a, b) and torch.equal(b, c) and bool(torch.isfinite(b).all())
    assert float(outs[1][2][1, 301:].abs().max()) == 0 and float(outs[1][3][1, 301:].abs().max()) == 0


def test_window_sinks_far_from_the_scores():
    from cppmega_mlx_b200 import ops
    q, k, v = (_rand(1, 140, 4, 64, seed=i) for i in range(3))
    sinks = torch.tensor([-300.0, 300.0, 0.0, float("-inf")], device="cuda")
    o = ops.window_attention(q, k, v, window=30, sinks=sinks)
    _done()
    W.check(o, W.attention64(q, k, v, W.visible(140, 140, 30, 0, device="cuda"), sinks)["o"], "o")
    assert float(o[:, :, 1].abs().max()) == 0


CACHED = [
    # B, N, H, Hk, D, Dv, prefixes, page, tree, window, ns, logits
    (1, 1, 4, 2, 64, 64, [0], 16, None, None, 0, False),
    (3, 1, 16, 4, 128, 128, [900, 1, 130], 16, None, 100, 4, True),
    (2, 5, 8, 1, 128, 128, [300, 64], 8, "own", None, 0, False),
    (2, 20, 8, 2, 64, 64, [500, 3], 48, "own", 7, 2, False),           # the window ends inside the tree
    (1, 61, 16, 2, 128, 128, [1500], 64, "shared", None, 0, False),     # four row tiles, split over the keys
    (2, 64, 6, 2, 96, 32, [77, 200], 24, "own", 60, 40, True),          # 64 nodes, three heads to a group, pages inside tiles
    (2, 150, 4, 2, 64, 64, [333, 0], 32, None, 90, 5, False),           # a chunk of a prompt
    (3, 7, 40, 1, 128, 128, [50, 2000, 700], 256, "own", 512, 0, True),
    (2, 9, 8, 8, 64, 128, [400, 127], 0, "own", 33, 1, False),          # contiguous
    (130, 1, 8, 2, 64, 64, None, 0, None, 64, 4, False),
    (2, 3, 4, 2, 64, 64, [40, 9], 7, "own", None, 0, False),            # a page size the kernel does not take: the plain form
]


def _cached_inputs(case, poison=True):
    b, n, h, hk, d, dv, prefix, page, tree, window, ns, logits = case
    from cppmega_mlx_b200 import ops
    r = torch.Generator().manual_seed(b * 100 + n)
    prefix = [int(x) for x in torch.randint(0, 300, (b,), generator=r)] if prefix is None else prefix
    t = max(prefix) + n + 3
    k, v, q = _rand(b, t, hk, d, seed=1), _rand(b, t, hk, dv, seed=2), _rand(b, n, h, d, seed=3)
    words = None
    if tree is not None:
        par = [[int(torch.randint(-1, m, (1,), generator=r)) if m else -1 for m in range(n)] for _ in range(b if tree == "own" else 1)]
        if tree == "own" and n > 4:
            par[-1][n - 2:] = [-2, -2]                       # two places that hold no node
        words = ops.tree_words(par if tree == "own" else par[0])
    rows = [[(1 << (i + 1)) - 1 for i in range(n)]] * b if words is None else (words.tolist() if words.dim() == 2 else [words.tolist()] * b)
    bits = [[[bool(w >> m & 1) for m in range(n)] for w in row] for row in rows]
    seen = W.cached_visible(prefix, n, t, bits, window, ns, "cuda")
    bad = float("nan") if poison else 0.0
    unseen = ~seen.any(1)
    k[unseen], v[unseen] = bad, bad
    kr, vr, table = k, v, None
    if page:
        width = -(-t // page) + 1
        kr, vr = (torch.full((b * width + 2, 3, page, hk, x), bad, device="cuda", dtype=BF) for x in (d, dv))
        table = torch.randperm(b * width + 2, generator=r)[:b * width].view(b, width)
        for i in range(b):
            at = torch.arange(prefix[i] + n)
            kr[table[i, at // page].cuda(), 1, (at % page).cuda()] = k[i, :prefix[i] + n]
            vr[table[i, at // page].cuda(), 1, (at % page).cuda()] = v[i, :prefix[i] + n]
            table[i, -(-(prefix[i] + n) // page):] = -1
        kr, vr, table = kr[:, 1], vr[:, 1], table.int().cuda()
    sinks = _rand(h, seed=5) if logits else None
    args = (q, kr, vr, table, torch.tensor(prefix, dtype=torch.int32, device="cuda"))
    kw = dict(tree=None if words is None else words.cuda(), window=window, sink_tokens=ns, sinks=sinks)
    return args, kw, (k, v, seen)


@pytest.mark.parametrize("case", CACHED, ids=str)
def test_cached_attention(case):
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    args, kw, (k, v, seen) = _cached_inputs(case)
    before = B.launch_count("window_fwd")
    o = ops.cached_attention(*args, **kw)
    _done()
    assert B.launch_count("window_fwd") == before + (0 if case[7] == 7 else 1)
    W.check(o, W.attention64(args[0], k, v, seen, kw["sinks"])["o"], "o")
    again = ops.cached_attention(*args, **kw, max_keys=64)          # another split of the work
    _done()
    W.check(again, W.attention64(args[0], k, v, seen, kw["sinks"])["o"], "o")


def test_cached_reports_what_the_pool_cannot_hold():
    """A page id outside the pool and a length outside the table are reported; the kernel reads inside the pool all the same."""
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    args, kw, _ = _cached_inputs((2, 3, 4, 2, 64, 64, [40, 9], 8, "own", None, 0, False), poison=False)
    good = ops.cached_attention(*args, **kw)
    _done()
    q, k, v, table, prefix = args
    for tbl, n in ((torch.where(table == table[0, 1], table.new_tensor(10 ** 6), table), prefix),
                   (torch.where(table == table[0, 1], table.new_tensor(-5), table), prefix), (table, prefix + 100000), (table, prefix - 100)):
        out = ops.cached_attention(q, k, v, tbl, n, **kw)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="status"):
            B.check_status()
        if n is prefix:
            assert torch.equal(out[1], good[1])          # the other sequence is as it was
    assert torch.equal(ops.cached_attention(*args, **kw), good)
    _done()


def test_graph_replay_and_streams():
    """Captured calls follow their inputs; a call on a side stream equals one on the default stream; two graphs do not share scratch."""
    from cppmega_mlx_b200 import ops
    args, kw, _ = _cached_inputs((1, 7, 16, 2, 128, 128, [1700], 16, "own", None, 0, True), poison=False)
    wq, wk, wv = (_rand(1, 300, n, 64, seed=n) for n in (4, 2, 2))
    calls = [lambda: ops.cached_attention(*args, **kw), lambda: ops.window_attention(wq, wk, wv, window=50, sink_tokens=4)]
    want = [f() for f in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [f() for f in calls]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for f in [calls[0], calls[0], calls[1]]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out, f))
    args[0].mul_(-0.5), wq.mul_(2.0)
    want = [f() for _, _, f in graphs]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    a.wait_stream(torch.cuda.current_stream()), b.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(a):
            graphs[0][0].replay()
        with torch.cuda.stream(b):
            graphs[1][0].replay()
            graphs[2][0].replay()
    _done()
    assert all(torch.equal(w, o) for w, (_, o, _) in zip(want, graphs))


def test_training_step_in_a_graph():
    from cppmega_mlx_b200 import ops
    q, k, v = (_rand(1, 200, n, 64, seed=n).requires_grad_() for n in (4, 2, 2))
    do = _rand(1, 200, 4, 64, seed=8)

    def step():
        o = ops.window_attention(q, k, v, window=60, sink_tokens=4)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    with torch.no_grad():
        q.mul_(0.5), do.mul_(-2)
    g.replay()
    _done()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("dtype,shape", [(BF, (40, 3, 16, 2, 64)), (torch.float32, (9, 5, 3)), (torch.uint8, (17, 1, 7, 3)), (torch.int64, (6, 1)),
                                         (BF, (33, 5, 11, 9, 125))])
def test_copy_pages(dtype, shape):
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    a = torch.randint(0, 200, shape, device="cuda").to(dtype)
    b = torch.randint(0, 200, (shape[0], 2, shape[-1]), device="cuda").to(torch.float32)[:, 1:]      # pages of a larger tensor
    n = shape[0]
    perm = torch.randperm(n)
    src, dst = perm[:n // 2], perm[n // 2:2 * (n // 2)]
    want = [x.clone() for x in (a, b)]
    for w in want:
        w[dst.cuda()] = w[src.cuda()]
    before = B.launch_count("copy_pages")
    ops.copy_pages((a, b), src.tolist(), dst.tolist())
    _done()
    assert B.launch_count("copy_pages") == before + 1 and torch.equal(a, want[0]) and torch.equal(b, want[1])
    pad = torch.tensor([-1], dtype=torch.int32)
    ops.copy_pages([a] * 1, torch.cat([dst.int(), pad]).cuda(), torch.cat([src.int(), pad]).cuda())      # device lists, an unused place
    _done()
    assert torch.equal(a, want[0])
    for s, d in (([0], [n]), ([-7], [0]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        ops.copy_pages(a, torch.tensor(s, device="cuda"), torch.tensor(d, device="cuda"))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="status"):
            B.check_status()


@pytest.mark.parametrize("dtype,layers,page,row", [(BF, 3, 16, (2, 64)), (BF, 2, 7, (1, 9)), (torch.uint8, 1, 8, (33,)), (torch.float32, 4, 64, (8, 128))])
def test_compact_rows(dtype, layers, page, row):
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    from cppmega_mlx_b200.ops.pages import compact_rows_reference
    r = torch.Generator().manual_seed(page)
    bsz, most = 5, 64
    width = -(-200 // page)
    pools = [torch.randint(0, 200, (bsz * width, layers, page, *row), device="cuda").to(dtype) for _ in range(2)]
    table = torch.randperm(bsz * width, generator=r).view(bsz, width).int().cuda()
    start = torch.tensor([0, 5, 130, 17, 64], dtype=torch.int32, device="cuda")
    path = torch.stack([torch.randperm(70, generator=r)[:most].sort().values for _ in range(bsz)])
    path[4] = torch.randperm(most, generator=r)                        # any order, sources written by others
    path[3, 1] = path[3, 0]                                            # the same row twice
    counts = torch.tensor([64, 1, 40, 30, 64], dtype=torch.int32, device="cuda")
    path = path.int().cuda()
    want = [p.clone() for p in pools]
    compact_rows_reference(want, table, start, path, counts)
    before = B.launch_count("compact_rows")
    ops.compact_rows(pools, table, start, path, counts)
    _done()
    assert B.launch_count("compact_rows") == before + 1 and all(torch.equal(a, b) for a, b in zip(pools, want))
    keep = [p.clone() for p in pools]
    for st, pa, co, tb in ((start + 10 ** 6, path, counts, table), (start, path - 99, counts, table), (start, path, counts + 1, table),
                           (start, path, counts - 9, table), (start, path, counts, table + 10 ** 6)):
        ops.compact_rows(pools, tb, st, pa, co)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="status"):
            B.check_status()
        for p, k in zip(pools, keep):
            p.copy_(k)


def test_serving_run_verify_accept_fork_decode():
    """Prompt, drafted tree, acceptance, a fork, next tokens on both, through the block manager and the kernels."""
    from cppmega_mlx_b200 import inference as I
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    torch.manual_seed(0)
    m = I.PagedKVBlockManager(num_blocks=64, num_layers=2, block_size=16, kv_heads=2, head_dim=64, device="cuda")
    m.k_pool.fill_(float("nan")), m.v_pool.fill_(float("nan"))
    rows = {1: _rand(2, 100, 2, 64, seed=1), 2: _rand(2, 41, 2, 64, seed=2)}
    par = [-1, -1, 0, 1, 3, 3, 5]
    path = {1: [1, 3, 5, 6], 2: [0, 2]}
    nodes = {s: _rand(2, 7, 2, 64, seed=10 + s) for s in (1, 2)}
    for s in (1, 2):
        m.allocate(s, 0)
        for layer in range(2):
            m.append(s, layer, *rows[s], advance=layer == 1)
        for layer in range(2):
            m.append(s, layer, *nodes[s], advance=False)
    q, qn = _rand(2, 7, 8, 64, seed=3), _rand(3, 8, 64, seed=4)
    table, lens = I.build_paged_block_table(m, [1, 2])
    tree = ops.tree_words(par).cuda()
    names = ("window_fwd", "compact_rows", "copy_pages")
    before = [B.launch_count(n) for n in names]
    out = I.paged_tree_attention(q, m, 1, table, lens, tree, window=60, sink_tokens=4)
    m.accept(path)
    m.fork(2, 3)
    nxt = _rand(3, 2, 1, 2, 64, seed=5)
    for i, s in enumerate((1, 2, 3)):
        for layer in range(2):
            m.append(s, layer, *nxt[i], advance=layer == 1)
    table, lens = I.build_paged_block_table(m, [1, 2, 3])
    last = I.paged_decode_attention(qn, m, 1, table, lens, window=60, sink_tokens=4)
    _done()
    assert [B.launch_count(n) - x for n, x in zip(names, before)] == [2, 1, 1]
    for i, s in enumerate((1, 2, 3)):
        o = 2 if s == 3 else s
        k, v = (torch.cat([rows[o][x], nodes[o][x][path[o]], nxt[i, x]])[None] for x in range(2))
        n_q = len(path[o]) if s < 3 else 0
        qs = torch.cat([q[o - 1, path[o]][:n_q], qn[i:i + 1]])[None]
        want = W.attention64(qs, k, v, W.visible(len(path[o]) + 1, k.shape[1], 60, 4, device="cuda")[:, len(path[o]) - n_q:])["o"]
        got = torch.cat([out[o - 1, path[o]][:n_q], last[i:i + 1]])[None]
        W.check(got, want, f"sequence {s}")


def test_module_routes_windows_to_the_kernels():
    from cppmega_mlx_b200 import inference as I
    from cppmega_mlx_b200.nn.attention import AttentionConfig, CausalSelfAttention
    from cppmega_mlx_b200.ops import _backend as B
    from tests.test_gpu_blocks import _compare
    torch.manual_seed(0)
    cfg = AttentionConfig(256, 4, num_kv_heads=2, mode="gqa", sliding_window=50, sink_tokens=3)
    m = CausalSelfAttention(cfg).cuda()
    _compare(m, torch.randn(2, 200, 256, device="cuda"), lambda mod, x: mod(x), expect=("window_fwd", "window_bwd"))
    m = m.eval()
    x, sinks = _rand(2, 90, 256, seed=3), _rand(4, seed=4)
    with torch.no_grad():
        full = m(x, sinks=sinks)
        caches = [I.StaticDecodeCache(1, 2, 96, "cuda"), I.PagedDecodeCache(1, 2, num_pages=12, page_size=16, max_pages_per_seq=6, device="cuda")]
        caches[1].set_pages(0, [3, 5, 7, 9, 11, 1]), caches[1].set_pages(1, [0, 2, 4, 6, 8, 10])
        for cache in caches:
            before = B.launch_count("window_fwd")
            y = []
            for i in range(90):
                y.append(m(x[:, i:i + 1], kv_cache=cache, sinks=sinks))
                cache.advance()
            assert B.launch_count("window_fwd") == before + 90
            y = torch.cat(y, 1).float()
            # two bf16 projections of 256 terms apart: a few half steps of the largest value
            assert float((y - full.float()).abs().max()) <= 8 * W.H * float(full.float().abs().max())
    _done()
