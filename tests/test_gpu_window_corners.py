"""Windowed and cached attention and page movements at the corners of their contracts: layouts and values of the sink logits, rows and
nodes that see nothing, words with stray bits, indexes that do not fit, autograd's rarer modes."""
import pytest
import torch

from tests import _window_oracle as W

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _rand(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale).to(BF)


def _done():
    from cppmega_mlx_b200.ops import _backend as B
    torch.cuda.synchronize()
    B.check_status()


def _reported():
    from cppmega_mlx_b200.ops import _backend as B
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status"):
        B.check_status()


def _sinks(layout, dtype, h, seed=4):
    if layout == "expanded":
        return _rand(1, seed=seed).to(dtype).expand(h)
    x = _rand(2 * h, 3, seed=seed).to(dtype)
    return {"dense": x[:h, 0].contiguous(), "strided": x[::2, 1], "column": x[:h, 2]}[layout]


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("layout", ["dense", "strided", "column", "expanded"])
def test_sinks_of_any_layout_and_type(layout, dtype):
    from cppmega_mlx_b200 import ops
    q, k, v, do = _rand(2, 90, 8, 64, seed=1), _rand(2, 90, 2, 64, seed=2), _rand(2, 90, 2, 64, seed=3), _rand(2, 90, 8, 64, seed=5)
    sinks = _sinks(layout, dtype, 8).detach()
    leaves = [x.requires_grad_() for x in (q, k, v, sinks)]
    o = ops.window_attention(q, k, v, window=30, sink_tokens=2, sinks=sinks)
    grads = torch.autograd.grad(o, leaves, do)
    _done()
    ref = W.attention64(*(x.detach() for x in leaves[:3]), W.visible(90, 90, 30, 2, device="cuda"), sinks.detach(), do=do)
    for got, name in zip((o.detach(), *grads[:3]), ("o", "dq", "dk", "dv")):
        W.check(got, ref[name], name)
    value, bound = ref["ds"]
    W.check(grads[3], (value, bound + torch.finfo(dtype).eps / 2 * value.abs()), "ds")         # written in the logits' type
    with torch.no_grad():
        n = torch.tensor([85, 3], dtype=torch.int32, device="cuda")
        c = ops.cached_attention(q[:, :5], k, v, None, n, sinks=sinks)
    _done()
    bits = [[[m <= i for m in range(5)] for i in range(5)]] * 2
    W.check(c, W.attention64(q[:, :5].detach(), k.detach(), v.detach(), W.cached_visible([85, 3], 5, 90, bits, None, 0, "cuda"), sinks.detach())["o"], "cached")


@pytest.mark.parametrize("s,t", [(1, 60), (1, 1500), (1, 5000), (12, 700), (100, 100), (100, 4000)])     # whole, joined in a cluster, by a second kernel
def test_rows_without_a_key_whose_sink_is_off(s, t):
    """A logit of -inf is no key at all: a row that sees nothing yields zeros and adds nothing to any gradient."""
    from cppmega_mlx_b200 import ops
    q, k, v, do = _rand(2, s, 4, 64, seed=1), _rand(2, t, 2, 64, seed=2), _rand(2, t, 2, 64, seed=3), _rand(2, s, 4, 64, seed=4)
    sinks = torch.tensor([float("-inf"), 0.5, float("-inf"), -2.0], device="cuda")
    n = torch.tensor([0, t], dtype=torch.int32, device="cuda")
    seen = W.visible(s, t, None, 0, n, "cuda")
    with torch.no_grad():
        alone = ops.window_attention(q, k, v, sinks=sinks, key_lengths=n)
    leaves = [x.requires_grad_() for x in (q, k, v, sinks)]
    o = ops.window_attention(q, k, v, sinks=sinks, key_lengths=n)
    grads = torch.autograd.grad(o, leaves, do)
    _done()
    assert torch.equal(o, alone) and float(o[0].detach().abs().max()) == 0
    ref = W.attention64(*(x.detach() for x in leaves[:3]), seen, sinks.detach(), do=do)
    for got, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv", "ds")):
        W.check(got, ref[name], name)
    assert float(grads[3][0]) == 0 and float(grads[3][2]) == 0


@pytest.mark.parametrize("prefix", [20, 900, 6000])
@pytest.mark.parametrize("h", [2, 8, 40])
def test_padding_nodes_whose_sink_is_off(prefix, h):
    from cppmega_mlx_b200 import ops
    par = [-1, 0, 0, -2, -2]
    tree = ops.tree_words(par).cuda()
    q, k, v = _rand(1, 5, h, 64, seed=1), _rand(1, prefix + 5, 2, 64, seed=2), _rand(1, prefix + 5, 2, 64, seed=3)
    sinks = torch.zeros(h, device="cuda")
    sinks[::2] = float("-inf")
    o = ops.cached_attention(q, k, v, None, torch.tensor([prefix], device="cuda"), tree=tree, sinks=sinks)
    _done()
    bits = [[[bool(w >> m & 1) for m in range(5)] for w in tree.tolist()]]
    W.check(o, W.attention64(q, k, v, W.cached_visible([prefix], 5, prefix + 5, bits, None, 0, "cuda"), sinks)["o"], "o")
    assert float(o[:, 3:].abs().max()) == 0


@pytest.mark.parametrize("batch,prefix", [(2, 20), (2, 700), (2, 6000), (160, 300)])      # one tile, split and joined both ways, whole
@pytest.mark.parametrize("n,h", [(6, 4), (12, 8), (30, 8), (60, 16)])                     # up to 32 rows, up to 64, more, many
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_padding_nodes_with_anything_in_their_queries(batch, prefix, n, h, bad):
    """Unused places of a captured step: zeros come out, and the others' results are what they are without them."""
    from cppmega_mlx_b200 import ops
    hk = 2
    par = [(i - 1) // 2 for i in range(n)]
    hole = [n - 1, n - 2, n // 2 + 1]                      # (leaves: a parent is no padding)
    for i in hole:
        par[i] = -2
    tree = ops.tree_words(par).cuda()
    q, k, v = _rand(batch, n, h, 64, seed=1), _rand(batch, prefix + n, hk, 64, seed=2), _rand(batch, prefix + n, hk, 64, seed=3)
    sinks = _rand(h, seed=4)
    lens = torch.full((batch,), prefix, dtype=torch.int32, device="cuda")
    for sk in (None, sinks):
        q[:, hole] = 0
        want = ops.cached_attention(q, k, v, None, lens, tree=tree, sinks=sk)
        q[:, hole] = bad
        got = ops.cached_attention(q, k, v, None, lens, tree=tree, sinks=sk)
        _done()
        assert torch.equal(got, want) and float(got[:, hole].abs().max()) == 0


def test_plain_forms_on_the_gpu_report_what_the_pool_cannot_hold():
    """Pages that are not dense, page sizes that the kernels do not take and kernels turned off: the same contract, no failed assertion."""
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    pool = torch.arange(96., device="cuda").view(6, 4, 4)
    t = lambda *x: torch.tensor(x, device="cuda")  # noqa: E731
    for thin in (pool[:, :, ::2], pool):
        keep = pool.clone()
        with B.use_kernels(thin is not pool):
            before = B.launch_count("copy_pages")
            ops.copy_pages(thin, t(1, 9, -3, -1), t(3, 0, 0, -1))
            assert B.launch_count("copy_pages") == before
        _reported()
        assert torch.equal(thin[3], thin[1]) and torch.equal(thin[0], (keep[:, :, ::2] if thin is not pool else keep)[0])
    pool = torch.randn(5, 2, 4, 3, 2, device="cuda")
    keep, table = pool.clone(), t([4, 0], [2, 1])
    for thin in (pool[..., :1], pool):
        with B.use_kernels(thin is not pool):
            for start, tbl in ((t(9, 0), table), (t(4, 0), t([4, 7], [2, 1])), (t(4, 0), t([4, -2], [2, 1]))):
                ops.compact_rows(thin.transpose(-1, -2), tbl, start, t([1], [0]), t(1, 0))
                _reported()
                assert torch.equal(pool, keep)
    q, k = _rand(2, 2, 2, 8), _rand(6, 7, 1, 8)
    table, n = t([0, 1, 2], [3, 4, 5]), t(9, 3)
    want = ops.cached_attention(q, k, k, table, n)
    _done()
    for tbl, lens in ((t([0, 6, 2], [3, 4, 5]), n), (t([-4, 1, 2], [3, 4, 5]), n), (table, t(10 ** 6, 3)), (table, t(-2, 3))):
        got = ops.cached_attention(q, k, k, tbl, lens)
        _reported()
        assert torch.equal(got[1], want[1])


def test_host_indexes_are_the_caller_s_again_when_the_call_returns():
    """Pinned lists that are overwritten behind queued work: the pages copied are those that were checked.  A graph, which would read the
    lists again at every replay, takes none from the host."""
    from cppmega_mlx_b200 import ops
    n = 50000                                          # long enough for a copy that the device makes when it comes to it
    pool = torch.arange(8 * n, device="cuda").view(2 * n, 4).clone()
    want = pool.clone()
    want[n:] = want[:n]
    src, dst = torch.arange(n, dtype=torch.int32).pin_memory(), torch.arange(n, 2 * n, dtype=torch.int32).pin_memory()
    other = src.flip(0)
    ops.copy_pages(pool, [0], [0])                     # (the library is loaded)
    _done()
    torch.cuda._sleep(1_000_000_000)                   # half a second: the call returns long before
    ops.copy_pages(pool, src, dst)
    src.copy_(other)
    _done()
    assert torch.equal(pool, want)
    a, b = torch.tensor([2], device="cuda"), torch.tensor([9], device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_pages(pool, a, b)
        for x, y in (([3], [4]), (torch.tensor([3]), torch.tensor([4])), (src[:1], src[1:2])):
            with pytest.raises(RuntimeError, match="capture"):
                ops.copy_pages(pool, x, y)
    a.fill_(5)
    g.replay()
    _done()
    want[9] = want[5]
    assert torch.equal(pool, want)


@pytest.mark.parametrize("far", [2 ** 32 + 3, -2 ** 32 + 3, 2 ** 31 + 1, 2 ** 40])
def test_indexes_past_32_bits_are_reported(far):
    """64-bit indexes are not cut to a page, a length or a row that happens to exist."""
    from cppmega_mlx_b200 import ops
    pool = torch.randn(8, 2, 8, 1, 8, device="cuda").to(BF)
    keep = pool.clone()
    t = lambda *x: torch.tensor(x, device="cuda")  # noqa: E731
    for src, dst in ((t(far), t(1)), (t(1), t(far))):
        ops.copy_pages(pool, src, dst)
        _reported()
        assert torch.equal(pool, keep)
    table = t([0, 1, 2, 3])
    bad = table.clone()
    bad[0, 0] = far
    for args in ((bad, t(1), t([2]), t(1)), (table, t(far), t([2]), t(1)), (table, t(1), t([far]), t(1)), (table, t(1), t([2]), t(far))):
        ops.compact_rows(pool, *args)
        _reported()
        pool.copy_(keep)
    q = _rand(1, 1, 2, 8)
    for tbl, n in ((bad, t(5)), (table, t(far))):
        ops.cached_attention(q, pool[:, 0], pool[:, 1], tbl, n)
        _reported()
    k = _rand(1, 20, 2, 8)
    ops.window_attention(q, k, k, key_lengths=t(far))
    _reported()
    ops.copy_pages(pool, t(-1, 3), t(-1, 5))                 # an unused place stays one
    _done()
    assert torch.equal(pool[5], keep[3])


@pytest.mark.parametrize("d,logits", [(64, False), (64, True), (32, True), (128, False)])
def test_backwards_side_by_side(d, logits):
    """A block that waits for the key gradients' blocks holds no tensor memory that one of them, or of another stream's, may still need."""
    from cppmega_mlx_b200 import ops
    sides, work = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(3):
        s = 1200 + 333 * i
        leaves = [_rand(1, s, n, d, seed=10 * i + j).requires_grad_() for j, n in enumerate((8, 4, 4))]
        if logits:
            leaves.append(_rand(8, seed=10 * i + 5).requires_grad_())
        do = _rand(1, s, 8, d, seed=10 * i + 4)
        o = ops.window_attention(*leaves[:3], window=300, sink_tokens=4, sinks=leaves[3] if logits else None)
        work.append((o, leaves, do, torch.autograd.grad(o, leaves, do, retain_graph=True)))
    _done()
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        got = []
        for side, (o, leaves, do, _) in zip(sides, work):
            with torch.cuda.stream(side):
                got.append([x.clone() for x in torch.autograd.grad(o, leaves, do, retain_graph=True)])
        for side in sides:
            side.synchronize()
        assert all(torch.equal(a, b) for g, (_, _, _, want) in zip(got, work) for a, b in zip(g, want))
    _done()


def test_layer_takes_sinks_of_any_shape_and_type():
    from cppmega_mlx_b200.nn.attention import AttentionConfig, CausalSelfAttention
    from cppmega_mlx_b200.ops import _backend as B
    torch.manual_seed(0)
    m = CausalSelfAttention(AttentionConfig(128, 4, num_kv_heads=2, mode="gqa")).cuda().to(BF).eval()
    x, sinks = _rand(2, 70, 128, seed=1), torch.tensor([1, -2, 0, 3], device="cuda")
    with torch.no_grad():
        want = m(x, sinks=sinks.float())
        before = B.launch_count("window_fwd")
        for other in (sinks, sinks.view(1, 4, 1, 1), sinks.to(BF).view(2, 2)):
            assert torch.equal(m(x, sinks=other), want)
        assert B.launch_count("window_fwd") == before + 3
    leaf = sinks.float().view(1, 4, 1, 1).requires_grad_()
    m(x, sinks=leaf).float().square().sum().backward()
    assert leaf.grad.shape == leaf.shape and float(leaf.grad.abs().min()) > 0
    _done()


def test_forward_mode_derivatives():
    """Tangents pass through the plain form, with or without gradients wanted beside them; a cache has none and says so."""
    from torch.autograd import forward_ad as F

    from cppmega_mlx_b200 import ops
    q, k, v, dk = _rand(1, 20, 4, 64, seed=1), _rand(1, 20, 2, 64, seed=2), _rand(1, 20, 2, 64, seed=3), _rand(1, 20, 2, 64, seed=4)
    f = lambda x: ops.window_attention_reference(q, x, v, window=7, sink_tokens=1)  # noqa: E731
    want = torch.func.jvp(f, (k,), (dk,))[1]
    assert float(want.abs().max()) > 0.01
    for grad in (False, True):
        with F.dual_level():
            o = ops.window_attention(q.detach().requires_grad_(grad), F.make_dual(k, dk), v, window=7, sink_tokens=1)
            assert torch.equal(F.unpack_dual(o).tangent.detach(), want)
            with torch.no_grad(), pytest.raises(ValueError, match="no gradient"):
                ops.cached_attention(q, F.make_dual(k, dk), v, None, torch.zeros(1, dtype=torch.int32, device="cuda"))
            with pytest.raises(ValueError, match="gradient"):
                ops.copy_pages(F.make_dual(k[0], dk[0]), [0], [1])
    _done()


@pytest.mark.parametrize("n", [1, 5, 31, 63])
@pytest.mark.parametrize("window", [None, 2])
def test_bits_past_the_last_token_say_nothing(n, window):
    from cppmega_mlx_b200 import ops
    par = [(i - 1) // 2 for i in range(n)]
    par[-1] = -2 if n > 1 else -1
    tree = ops.tree_words(par).cuda()
    q, k, v = _rand(2, n, 4, 64, seed=1), _rand(2, 200, 2, 64, seed=2), _rand(2, 200, 2, 64, seed=3)
    lens = torch.tensor([100, 0], dtype=torch.int32, device="cuda")
    want = ops.cached_attention(q, k, v, None, lens, tree=tree, window=window)
    stray = tree | (-1 << n)                                     # every bit from n on
    got = ops.cached_attention(q, k, v, None, lens, tree=stray, window=window)
    _done()
    assert torch.equal(got, want)
    plain = ops.cached_attention_reference(q, k, v, None, lens, tree=stray, window=window)
    assert torch.equal(plain, ops.cached_attention_reference(q, k, v, None, lens, tree=tree, window=window))


def test_trees_of_any_layout_run_the_kernel():
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    tree = ops.tree_words([[-1, 0, 0, 2, 2], [-1, -1, 1, 1, 0]]).cuda()
    q, k, v = _rand(2, 5, 4, 64, seed=1), _rand(2, 200, 2, 64, seed=2), _rand(2, 200, 2, 64, seed=3)
    lens = torch.tensor([100, 9], dtype=torch.int32, device="cuda")
    wide = torch.zeros(2, 9, dtype=torch.int64, device="cuda")
    wide[:, 2:7] = tree
    for same, other in ((tree, wide[:, 2:7]), (tree, tree.t().contiguous().t()), (tree[:1].repeat(2, 1), tree[:1].expand(2, 5)), (tree[1], wide[1, 2:7])):
        want = ops.cached_attention(q, k, v, None, lens, tree=same)
        before = B.launch_count("window_fwd")
        assert torch.equal(ops.cached_attention(q, k, v, None, lens, tree=other), want)
        assert B.launch_count("window_fwd") == before + 1
    _done()


def test_second_derivatives():
    """A layer's sink logits had them before there was a kernel: they come from the plain form, the first ones that carry a graph too."""
    from cppmega_mlx_b200 import ops
    leaves = [_rand(1, 20, n, 64, seed=n).requires_grad_() for n in (4, 2)] + [_rand(1, 20, 2, 64, seed=9).requires_grad_(), _rand(4, seed=7).requires_grad_()]
    do, dd = _rand(1, 20, 4, 64, seed=8).requires_grad_(), _rand(1, 20, 2, 64, seed=6)
    res = []
    for f in (ops.window_attention, ops.window_attention_reference):
        o = f(*leaves[:3], window=7, sink_tokens=1, sinks=leaves[3])
        first = torch.autograd.grad(o, leaves, do, create_graph=True)
        res.append([*first, *torch.autograd.grad((first[1] * dd).float().sum() + first[3].float().sum(), [*leaves, do])])
    _done()
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(*res))
    x = leaves[1]                                                 # one tensor as keys and as values: each use counts once
    got, want = (torch.autograd.grad(f(leaves[0], x, x, window=7), x, do.detach(), create_graph=True)[0] for f in (ops.window_attention, ops.window_attention_reference))
    assert torch.equal(got, want)


def test_layers_whose_groups_the_backward_does_not_take_train_as_before(monkeypatch):
    """Groups of more than 64 heads: the library's attention under a window, not the fp32 form of every pair."""
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.nn import attention as A
    torch.manual_seed(0)
    m = A.CausalSelfAttention(A.AttentionConfig(65 * 16, 65, num_kv_heads=1, mode="gqa", sliding_window=20)).cuda().to(BF)
    x = _rand(1, 50, 65 * 16, seed=1)
    asked = []
    real = ops.window_attention
    monkeypatch.setattr(ops, "window_attention", lambda *a, **kw: asked.append(1) or real(*a, **kw))
    m(x).float().sum().backward()
    assert not asked and all(p.grad is not None for p in m.parameters())
    with torch.no_grad():
        m(x)
    assert len(asked) == 1
    _done()


def test_more_heads_than_a_grid_has_rows():
    from cppmega_mlx_b200 import ops
    h, g = 2 * 33000, 2
    leaves = [_rand(1, 2, n, 8, seed=1 + i).requires_grad_() for i, n in enumerate((h, h // g, h // g))]
    do = _rand(1, 2, h, 8, seed=5)
    o = ops.window_attention(*leaves, window=2)
    grads = torch.autograd.grad(o, leaves, do)
    _done()
    ref = W.attention64(*(x.detach() for x in leaves), W.visible(2, 2, 2, 0, device="cuda"), do=do)
    for got, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv")):
        W.check(got, ref[name], name)


@pytest.mark.parametrize("s,t,g,d,window,ns,lengths", [(16, 16, 2, 64, None, 0, None), (40, 300, 3, 128, 9, 3, None), (70, 70, 1, 40, 12, 4, None),
                                                       (33, 700, 4, 96, 13, 0, None), (20, 200, 2, 64, None, 0, [11, 16])])
def test_rows_that_see_nine_to_sixteen_keys(s, t, g, d, window, ns, lengths):
    """As for a handful of keys: delta comes from p and dP there, three and four rounds of four keys."""
    from cppmega_mlx_b200 import ops
    b = 2
    q, k, v, do = _rand(b, s, 2 * g, d, seed=1), _rand(b, t, 2, d, seed=2), _rand(b, t, 2, d, seed=3), _rand(b, s, 2 * g, d, seed=4)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(ops.window_attention(q, k, v, window=window, sink_tokens=ns, key_lengths=n), leaves, do)
    _done()
    q, k, v, do = (x.detach().double() for x in (q, k, v, do))
    seen = W.visible(s, t, window, ns, n, "cuda").expand(b, s, t)
    most = seen.sum(-1).max()
    assert 9 <= int(most) <= 16
    kk, vv = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    p = torch.softmax((torch.einsum("bshd,bthd->bhst", q, kk) * d ** -0.5).masked_fill(~seen[:, None], float("-inf")), -1)
    dp, dpa = torch.einsum("bshd,bthd->bhst", do, vv), torch.einsum("bshd,bthd->bhst", do.abs(), vv.abs())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    # dS's rounding and fp32 in p, dP and delta
    eds = (W.H + W.F32) * ds.abs() + 2 * W.F32 * p * (dpa + (p * dpa).sum(-1, keepdim=True))
    for got, a, name in ((dq, kk, "dq"), (dk, q, "dk")):
        eq = "bhst,bthd->bshd" if name == "dq" else "bhst,bshd->bthd"
        value, bound = d ** -0.5 * torch.einsum(eq, ds, a), d ** -0.5 * torch.einsum(eq, eds, a.abs())
        if name == "dk":
            value, bound = (x.view(b, t, 2, g, d).sum(3) for x in (value, bound))
        W.check(got, (value, (bound + W.H * (value.abs() + bound)) * 1.01 + 1e-30), name)
