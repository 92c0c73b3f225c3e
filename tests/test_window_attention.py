"""Windowed attention, attention of drafted tokens over a cache, and page movements: plain forms, refusals, the block manager."""
import pytest
import torch

from cppmega_mlx_b200 import inference as I
from cppmega_mlx_b200 import ops
from cppmega_mlx_b200.inference.serving import OutOfBlocks
from tests import _window_oracle as W

# the plain forms compute in fp32: products of up to a few hundred terms, 2**-24 each
TOL = dict(rtol=2e-5, atol=2e-6)


@pytest.mark.parametrize("s,t,h,hk,window,ns", [(1, 1, 2, 1, None, 0), (9, 9, 4, 2, 3, 1), (7, 20, 3, 3, 5, 2), (5, 5, 2, 2, 100, 0),
                                                (12, 12, 2, 1, 1, 0), (6, 9, 4, 1, 2, 30)])
@pytest.mark.parametrize("logits", [False, True])
def test_window_reference_and_gradients(s, t, h, hk, window, ns, logits):
    torch.manual_seed(s * 31 + t)
    q, k, v = torch.randn(2, s, h, 8), torch.randn(2, t, hk, 8), torch.randn(2, t, hk, 12)
    sinks = torch.randn(h).requires_grad_() if logits else None
    lengths = torch.tensor([t, max(0, t - 4)], dtype=torch.int32)
    leaves = [x.requires_grad_() for x in (q, k, v)] + ([sinks] if logits else [])
    do = torch.randn(2, s, h, 12)
    o = ops.window_attention(q, k, v, window=window, sink_tokens=ns, sinks=sinks, key_lengths=lengths)
    grads = torch.autograd.grad(o, leaves, do)
    ref = W.attention64(*(x.detach() for x in (q, k, v)), W.visible(s, t, window, ns, lengths), None if sinks is None else sinks.detach(), do=do)
    for got, name in zip((o, *grads), ("o", "dq", "dk", "dv", "ds")):
        torch.testing.assert_close(got.detach().double(), ref[name][0], **TOL)


def test_window_gradient_against_differences():
    torch.manual_seed(0)
    args = [torch.randn(*n, dtype=torch.float64) for n in ((1, 4, 2, 4), (1, 6, 1, 4), (1, 6, 1, 4), (2,))]
    seen = W.visible(4, 6, 3, 1)
    do = torch.randn(1, 4, 2, 4, dtype=torch.float64)
    ref = W.attention64(*args[:3], seen, args[3], do=do)
    value = lambda a: float((W.attention64(*a[:3], seen, a[3])["o"][0] * do).sum())  # noqa: E731
    for i, name in enumerate(("dq", "dk", "dv", "ds")):
        for at in range(0, args[i].numel(), 3):
            d = torch.zeros(args[i].numel(), dtype=torch.float64)
            d[at] = 1e-6
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + d.view_as(args[i]), args[i] - d.view_as(args[i])
            slope = (value(up) - value(down)) / 2e-6     # central: off by 1e-12 f''' plus 1e-16 / 1e-6
            assert abs(slope - float(ref[name][0].flatten()[at])) < 1e-7


def test_rows_without_a_key_and_unseen_nan():
    q, k, v = torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8)
    lengths = torch.tensor([0])
    assert float(ops.window_attention(q, k, v, key_lengths=lengths).abs().max()) == 0
    want = ops.window_attention(q, k, v, window=2, key_lengths=torch.tensor([3]))
    k[:, 3], v[:, 3] = float("nan"), float("inf")
    k.requires_grad_(), v.requires_grad_()
    got = ops.window_attention(q, k, v, window=2, key_lengths=torch.tensor([3]))
    assert torch.equal(got, want)
    assert ops.window_attention(q[:, :0], k, v).shape == (1, 0, 2, 8)


@pytest.mark.parametrize("change,match", [
    (dict(window=0), "window must be positive"), (dict(sink_tokens=-1), "sink_tokens"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(sinks=torch.zeros(3)), "sinks must be"), (dict(key_lengths=torch.zeros(2)), "key_lengths"),
    (dict(k=torch.zeros(1, 5, 2, 8)), "at least as many keys"), (dict(k=torch.zeros(1, 6, 2, 4)), "head size"),
    (dict(v=torch.zeros(1, 7, 2, 8)), "differ in more"), (dict(q=torch.zeros(1, 6, 3, 8)), "not a multiple"),
    (dict(q=torch.zeros(1, 6, 4, 8, dtype=torch.bfloat16)), "one floating type"), (dict(q=torch.zeros(2, 6, 4, 8)), "batches")])
def test_window_refusals(change, match):
    a = dict(q=torch.zeros(1, 6, 4, 8), k=torch.zeros(1, 6, 2, 8), v=torch.zeros(1, 6, 2, 8))
    if "k" in change and change["k"].shape[1] == 5:
        a["v"] = torch.zeros(1, 5, 2, 8)
    a.update(change)
    with pytest.raises(ValueError, match=match):
        ops.window_attention(a.pop("q"), a.pop("k"), a.pop("v"), **a)


def _bits(words, n):
    return [[[bool(w >> m & 1) for m in range(n)] for w in row] for row in words]


def test_tree_words():
    w = ops.tree_words([-1, 0, 0, 1, -1, -2])
    assert w.tolist() == [1, 0b11, 0b101, 0b1011, 0b10000, 0]
    assert ops.tree_words([[-1] * 64, list(range(-1, 63))])[1, 63].item() == -1          # a chain of 64 sees all of itself
    for bad in ([0], [-1, 2, -1], [-3], [-2, 0], [[-1] * 65]):
        with pytest.raises(ValueError):
            ops.tree_words(bad)


@pytest.mark.parametrize("window,ns", [(None, 0), (4, 1), (2, 0), (1, 3)])
@pytest.mark.parametrize("paged", [True, False])
def test_cached_reference(window, ns, paged):
    torch.manual_seed(1)
    n, prefix = 6, [9, 0, 4]
    tree = ops.tree_words([[-1, 0, 0, 1, 3, -1], [-1, -1, 1, 2, -2, -2], [-1, 0, 1, 2, 3, 4]])
    t = 16
    k, v = torch.randn(3, t, 2, 8), torch.randn(3, t, 2, 8)
    q, sinks = torch.randn(3, n, 4, 8), torch.randn(4)
    for tr in (tree, tree[0], None):
        bits = _bits([[(1 << (i + 1)) - 1 for i in range(n)]] * 3 if tr is None else (tr.tolist() if tr.dim() == 2 else [tr.tolist()] * 3), n)
        ref = W.attention64(q, k, v, W.cached_visible(prefix, n, t, bits, window, ns), sinks)["o"][0]
        kr, vr, table = k, v, None
        if paged:
            perm = torch.randperm(12)
            table = perm.view(3, 4).int()
            kr, vr = torch.full((12, 4, 2, 8), float("nan")), torch.full((12, 4, 2, 8), float("nan"))
            for b in range(3):
                for i in range(prefix[b] + n):
                    kr[table[b, i // 4], i % 4], vr[table[b, i // 4], i % 4] = k[b, i], v[b, i]
            table[1, 2:] = -1                                        # nothing of sequence 1 lies there
        got = ops.cached_attention(q, kr, vr, table, torch.tensor(prefix), tree=tr, window=window, sink_tokens=ns, sinks=sinks)
        torch.testing.assert_close(got.double(), ref, **TOL)


def test_cached_refusals():
    q, k = torch.zeros(2, 3, 4, 8), torch.zeros(2, 9, 2, 8)
    n = torch.zeros(2, dtype=torch.int32)
    ok = lambda **kw: ops.cached_attention(q, kw.pop("k", k), k, kw.pop("table", None), kw.pop("n", n), **kw)  # noqa: E731
    ok()
    for kw, match in ((dict(n=torch.zeros(3, dtype=torch.int32)), "prefix_lengths"), (dict(table=torch.zeros(1, 4, dtype=torch.int32)), "table"),
                      (dict(tree=torch.zeros(2, dtype=torch.int64)), "tree must"), (dict(tree=torch.zeros(3, dtype=torch.int32)), "tree must"),
                      (dict(window=-1), "window"), (dict(k=k.clone().requires_grad_()), "no gradient"), (dict(n=n.float()), "prefix_lengths")):
        with pytest.raises(ValueError, match=match):
            ok(**kw)
    with pytest.raises(ValueError, match="at most 64"):
        ops.cached_attention(torch.zeros(1, 65, 1, 8), torch.zeros(1, 99, 1, 8), torch.zeros(1, 99, 1, 8), None,
                             torch.zeros(1, dtype=torch.int32), tree=torch.zeros(65, dtype=torch.int64))
    with pytest.raises(ValueError, match="contiguous cache"):
        ops.cached_attention(q, k[:1], k[:1], None, n)


def test_copy_pages_and_refusals():
    a, b = torch.randn(6, 3, 2), torch.arange(12).view(6, 2)
    a0, b0 = a.clone(), b.clone()
    ops.copy_pages((a, b), [0, -1, 3], [5, -1, 1])
    for x, x0 in ((a, a0), (b, b0)):
        assert torch.equal(x[5], x0[0]) and torch.equal(x[1], x0[3]) and torch.equal(x[[0, 2, 3, 4]], x0[[0, 2, 3, 4]])
    ops.copy_pages(a, [], [])
    ops.copy_pages(a, torch.tensor([2]), torch.tensor([2]))
    for src, dst in (([6], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1, 2])):
        with pytest.raises(ValueError):
            ops.copy_pages((a, b), src, dst)
    with pytest.raises(ValueError, match="pools"):
        ops.copy_pages((a, b[:5]), [0], [1])
    with pytest.raises(ValueError, match="gradient"):
        ops.copy_pages(a.clone().requires_grad_(), [0], [1])


def test_compact_rows_and_refusals():
    pool = torch.randn(5, 2, 4, 3)
    table = torch.tensor([[4, 0], [2, 1]])
    want = pool.clone()
    rows = lambda p, b, i: p[table[b, i // 4], :, i % 4]  # noqa: E731
    for b, start, path in ((0, 2, [1, 2, 5]), (1, 0, [3])):
        for i, x in enumerate(path):
            want[table[b, (start + i) // 4], :, (start + i) % 4] = rows(pool, b, start + x)
    ops.compact_rows(pool, table, torch.tensor([2, 0]), torch.tensor([[1, 2, 5], [3, 99, -9]]), torch.tensor([3, 1]))
    assert torch.equal(pool, want)
    for start, path, counts, tbl in (([2, 0], [[6], [0]], [1, 0], table), ([0, 0], [[-1], [0]], [1, 0], table), ([0, 0], [[0], [0]], [2, 0], table),
                                     ([-1, 0], [[0], [0]], [1, 0], table), ([4, 0], [[1], [0]], [1, 0], torch.tensor([[4, 7], [2, 1]]))):
        with pytest.raises(ValueError):
            ops.compact_rows(pool, tbl, torch.tensor(start), torch.tensor(path), torch.tensor(counts))
    with pytest.raises(ValueError, match="at most"):
        ops.compact_rows(pool, table, torch.tensor([0, 0]), torch.zeros(2, 2049, dtype=torch.int64), torch.tensor([0, 0]))


def _manager(**kw):
    return I.PagedKVBlockManager(**{**dict(num_blocks=12, num_layers=2, block_size=4, kv_heads=1, head_dim=8, dtype=torch.float32), **kw})


def _fill(m, sid, n, advance=True):
    ks = [torch.randn(n, 1, 8) for _ in range(2)]
    for layer in range(2):
        m.append(sid, layer, ks[layer], -ks[layer], advance=advance and layer == 1)
    return ks


def test_fork_copies_when_written():
    m = _manager()
    m.allocate(1, 0)
    a = _fill(m, 1, 6)
    m.fork(1, 2)
    assert m.tables[1] == m.tables[2] and m.num_free_blocks == 10
    b1, b2 = _fill(m, 1, 3), _fill(m, 2, 1)
    assert m.tables[1][0] == m.tables[2][0] and m.tables[1][1] != m.tables[2][1]
    for layer in range(2):
        assert torch.equal(m.gather(1, layer)[0], torch.cat([a[layer], b1[layer]]))
        assert torch.equal(m.gather(2, layer)[1], -torch.cat([a[layer], b2[layer]]))
    m.free(1)
    assert torch.equal(m.gather(2, 0)[0], torch.cat([a[0], b2[0]]))
    m.free(2)
    assert m.num_free_blocks == 12 and not any(m._refs)
    with pytest.raises(KeyError):
        m.fork(1, 5)
    m.allocate(3, 4 * 11)
    _fill(m, 3, 43)
    m.fork(3, 4)
    m.allocate(5, 4)
    with pytest.raises(OutOfBlocks):
        _fill(m, 4, 1)
    assert m.tables[3] == m.tables[4]


def test_accept_truncate_release_compact():
    m = _manager(num_blocks=24)
    m.allocate(1, 0), m.allocate(2, 0)
    a1, a2 = _fill(m, 1, 6), _fill(m, 2, 3)
    m.fork(1, 3)
    d1, d2, d3 = (_fill(m, s, 9, advance=False) for s in (1, 2, 3))
    m.accept({1: [0, 2, 7], 2: [0, 1], 3: []})
    assert m.lengths == {1: 9, 2: 5, 3: 6} and [len(m.tables[s]) for s in (1, 2, 3)] == [3, 2, 2]
    for layer in range(2):
        assert torch.equal(m.gather(1, layer)[0], torch.cat([a1[layer], d1[layer][[0, 2, 7]]]))
        assert torch.equal(m.gather(2, layer)[1], -torch.cat([a2[layer], d2[layer][:2]]))
        assert torch.equal(m.gather(3, layer)[0], a1[layer])
    for bad in ([2, 1], [0, 0], [-1], [400]):
        with pytest.raises(ValueError):
            m.accept({1: bad})
    before = {s: [m.gather(s, layer) for layer in range(2)] for s in (1, 2, 3)}
    m.allocate(9, 20)
    m.truncate(1, 7)
    m.free(2)
    moved = m.compact()
    used = {b for t in m.tables.values() for b in t}
    assert moved and used == set(range(len(used))) and m.num_free_blocks == 24 - len(used)
    for s, n in ((1, 7), (3, 6)):
        for layer in range(2):
            got = m.gather(s, layer)
            assert all(torch.equal(x, y[:n]) for x, y in zip(got, before[s][layer]))
    with pytest.raises(ValueError):
        m.truncate(1, 8)
    # a window of 5 over 23 tokens, 2 of them visible for good: blocks 1..3 of 6 are behind it
    m.allocate(5, 0)
    _fill(m, 5, 23)
    free = m.num_free_blocks
    assert m.release_window(5, 5, 2) == 3 and m.num_free_blocks == free + 3 and m.release_window(5, 5, 2) == 0
    assert [b < 0 for b in m.tables[5]] == [False, True, True, True, False, False]
    with pytest.raises(ValueError, match="released"):
        m.gather(5, 0)
    with pytest.raises(ValueError, match="released"):
        m.make_writable(5, 5, 6)
    m.fork(5, 6)
    m.free(5), m.free(6)
    assert m.num_free_blocks == free + 6


def test_greedy_tree_accept():
    par, tok = [-1, -1, 1, 1, 3], [5, 6, 7, 8, 9]
    assert I.greedy_tree_accept(par, tok, [6, 0, 8, 0, 9, 4]) == ([1, 3, 4], 4)
    assert I.greedy_tree_accept(par, tok, [1, 0, 0, 0, 0, 0]) == ([], 1)
    with pytest.raises(ValueError):
        I.greedy_tree_accept(par, tok, [1])


@pytest.mark.parametrize("window,ns", [(None, 0), (6, 2)])
def test_verify_accept_decode_equals_a_plain_chain(window, ns):
    """Prompt, drafted tree, acceptance, next token, through the manager: equal to attention over the accepted tokens alone."""
    torch.manual_seed(3)
    m = _manager(kv_heads=2, num_layers=1, num_blocks=20)
    m.allocate(1, 0), m.allocate(2, 0)
    rows = {}
    for sid, n in ((1, 7), (2, 10)):
        rows[sid] = torch.randn(2, n, 2, 8)
        m.append(sid, 0, *rows[sid])
    par = [-1, -1, 0, 1, 3, 3]
    nodes = {sid: torch.randn(2, 6, 2, 8) for sid in (1, 2)}
    for sid in (1, 2):
        m.append(sid, 0, *nodes[sid], advance=False)
    q = torch.randn(2, 6, 4, 8)
    table, lens = I.build_paged_block_table(m, [1, 2])
    out = I.paged_tree_attention(q, m, 0, table, lens, ops.tree_words(par), window=window, sink_tokens=ns)
    path = {1: [1, 3, 5], 2: [0, 2]}
    m.accept(path)
    nxt = torch.randn(2, 1, 2, 2, 8)
    qn = torch.randn(2, 4, 8)
    for i, sid in enumerate((1, 2)):
        m.append(sid, 0, nxt[i, :, 0], nxt[i, :, 1])
    table, lens = I.build_paged_block_table(m, [1, 2])
    last = I.paged_decode_attention(qn, m, 0, table, lens, window=window, sink_tokens=ns)
    for i, sid in enumerate((1, 2)):
        k, v = (torch.cat([rows[sid][x], nodes[sid][x][path[sid]], nxt[i, :, x]])[None] for x in range(2))
        qs = torch.cat([q[i, path[sid]], qn[i:i + 1]])[None]
        want = W.attention64(qs, k, v, W.visible(qs.shape[1], k.shape[1], window, ns))["o"][0][0]
        torch.testing.assert_close(torch.cat([out[i, path[sid]], last[i:i + 1]]).double(), want, **TOL)


def test_module_window_with_first_tokens():
    """The layer's mask route on the CPU: training, prompt over a cache, static one-token steps agree."""
    from cppmega_mlx_b200.nn.attention import AttentionConfig, CausalSelfAttention, causal_sdpa_mask
    with pytest.raises(ValueError):
        AttentionConfig(32, 4, mode="full", sink_tokens=1)
    with pytest.raises(ValueError):
        AttentionConfig(32, 4, mode="full", sliding_window=4, sink_tokens=-1)
    assert torch.equal(causal_sdpa_mask(9, sliding_window=3, sink_tokens=2), W.visible(9, 9, 3, 2)[0])
    torch.manual_seed(0)
    m = CausalSelfAttention(AttentionConfig(32, 4, num_kv_heads=2, mode="gqa", sliding_window=5, sink_tokens=2)).eval()
    x = torch.randn(2, 12, 32)
    sinks = torch.randn(4)
    with torch.no_grad():
        for sk in (None, sinks):
            full = m(x, sinks=sk)
            cache = I.StaticDecodeCache(1, 2, 16, "cpu")
            for i in range(12):
                y = m(x[:, i:i + 1], kv_cache=cache, sinks=sk)
                cache.advance()
                torch.testing.assert_close(y[:, 0], full[:, i], rtol=1e-4, atol=1e-5)
