"""Windowed and cached attention where the kernels take their rarer ways: a row's reference that has to rise, sequences far shorter than
the splits were made for, rows that see a handful of keys, groups larger than the backward takes, calls from several threads."""
import threading

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


def _levels(kind, t):
    """k's first column; whole numbers up to 80, so that bf16 holds them."""
    j = torch.arange(t)
    if kind == "step":
        return torch.where(j < t // 2, -80, 80)
    if kind == "ramp":
        return (160 * j // max(t - 1, 1)) - 80
    if kind == "fall":
        return 80 - (160 * j // max(t - 1, 1))
    if kind == "spike":
        return torch.where(j == (2 * t) // 3, 80, -80)
    return torch.randint(-80, 81, (t,), generator=torch.Generator().manual_seed(t))


# Scores are 16 * level / 8: exact in fp32 up to the multiplication with log2(e) / 8, whose arguments stay below 2.9 * 80 < 2^8.  One
# rounding there and one in the reference or the log-sum-exp (and one more in its conversion) are 2^-16 each, times ln 2: below the 2^-14
# that the bounds allow for fp32 everywhere.  A tile that rises by 15 levels lifts its sums by 2^43.
KINDS = ["step", "ramp", "fall", "spike", "random"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s,h,hk,window,ns", [(300, 4, 2, None, 0), (200, 2, 2, 90, 5), (450, 3, 1, 128, 64)])
def test_scores_far_apart_in_training(kind, s, h, hk, window, ns):
    from cppmega_mlx_b200 import ops
    q = torch.zeros(1, s, h, 64, device="cuda", dtype=BF)
    q[..., 0] = 16.0
    q[:, 1::2, :, 0] = -16.0                       # every other row meets the levels upside down
    k = _rand(1, s, hk, 64, seed=1)
    k[..., 0] = _levels(kind, s).to("cuda", BF)[None, :, None]
    v, do = _rand(1, s, hk, 64, seed=2), _rand(1, s, h, 64, seed=3)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = ops.window_attention(q, k, v, window=window, sink_tokens=ns)
    grads = torch.autograd.grad(o, leaves, do)
    _done()
    ref = W.attention64(*(x.detach() for x in leaves), W.visible(s, s, window, ns, device="cuda"), do=do)
    for got, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv")):
        W.check(got, ref[name], name)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,h,hk,t", [(1, 4, 1, 700), (1, 4, 1, 5000), (10, 4, 1, 1500), (25, 4, 1, 1500), (70, 8, 2, 900), (5, 128, 1, 400)])
def test_scores_far_apart_in_a_cache(kind, n, h, hk, t):
    from cppmega_mlx_b200 import ops
    q = torch.zeros(2, n, h, 64, device="cuda", dtype=BF)
    q[..., 0] = 16.0
    q[:, :, 1::2, 0] = -16.0
    k, v = _rand(2, t, hk, 64, seed=1), _rand(2, t, hk, 64, seed=2)
    k[..., 0] = _levels(kind, t).to("cuda", BF)[None, :, None]
    prefix = torch.tensor([t - n, (t - n) // 2], dtype=torch.int32, device="cuda")
    o = ops.cached_attention(q, k, v, None, prefix)
    _done()
    bits = [[[m <= i for m in range(n)] for i in range(n)]] * 2
    W.check(o, W.attention64(q, k, v, W.cached_visible(prefix.tolist(), n, t, bits, None, 0, "cuda"))["o"], "o")


@pytest.mark.parametrize("n,h", [(1, 4), (10, 4), (30, 4), (40, 8)])
@pytest.mark.parametrize("capacity", [300, 1900, 2400, 20000])
def test_sequences_far_shorter_than_the_cache(n, h, capacity):
    """The work is split for the cache's capacity; most splits of a short sequence then hold nothing."""
    from cppmega_mlx_b200 import ops
    prefix = torch.tensor([0, 3, 130], dtype=torch.int32, device="cuda")
    q, k, v = _rand(3, n, h, 64, seed=1), _rand(3, capacity, 1, 64, seed=2), _rand(3, capacity, 1, 64, seed=3)
    sinks = _rand(h, seed=4)
    bits = [[[m <= i for m in range(n)] for i in range(n)]] * 3
    t = 130 + n
    seen = W.cached_visible(prefix.tolist(), n, t, bits, 60, 2, "cuda")
    for i in range(3):
        k[i, int(prefix[i]) + n:], v[i, int(prefix[i]) + n:] = float("nan"), float("nan")
    for window, ns, vis in ((60, 2, seen), (None, 0, W.cached_visible(prefix.tolist(), n, t, bits, None, 0, "cuda"))):
        o = ops.cached_attention(q, k, v, None, prefix, window=window, sink_tokens=ns, sinks=sinks)
        _done()
        W.check(o, W.attention64(q, k[:, :t], v[:, :t], vis, sinks)["o"], "o")


@pytest.mark.parametrize("s,g,d,window,ns", [(1, 1, 64, None, 0), (2, 4, 128, None, 0), (5, 3, 40, None, 0), (8, 1, 128, None, 0), (90, 2, 64, 3, 4), (70, 64, 64, 1, 0)])
def test_rows_that_see_a_handful_of_keys(s, g, d, window, ns):
    """delta = sum p dP in fp32 there: no rounding of o enters dq.  A row that sees one key has a gradient of zero."""
    from cppmega_mlx_b200 import ops
    q, k, v, do = _rand(2, s, 2 * g, d, seed=1), _rand(2, s, 2, d, seed=2), _rand(2, s, 2, d, seed=3), _rand(2, s, 2 * g, d, seed=4)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(ops.window_attention(q, k, v, window=window, sink_tokens=ns), leaves, do)
    _done()
    q, k, v, do = (x.detach().double() for x in (q, k, v, do))
    seen = W.visible(s, s, window, ns, device="cuda")[0]
    kk, vv = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    p = torch.softmax((torch.einsum("bshd,bthd->bhst", q, kk) * d ** -0.5).masked_fill(~seen, float("-inf")), -1)
    dp, dpa = torch.einsum("bshd,bthd->bhst", do, vv), torch.einsum("bshd,bthd->bhst", do.abs(), vv.abs())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    # dS's rounding and fp32 in p, dP and delta; every row here sees at most eight keys
    assert int(seen.sum(-1).max()) <= 8
    eds = (W.H + W.F32) * ds.abs() + 2 * W.F32 * p * (dpa + (p * dpa).sum(-1, keepdim=True))
    for got, a, name in ((dq, kk, "dq"), (dk, q, "dk")):
        eq = "bhst,bthd->bshd" if name == "dq" else "bhst,bshd->bthd"
        value, bound = d ** -0.5 * torch.einsum(eq, ds, a), d ** -0.5 * torch.einsum(eq, eds, a.abs())
        if name == "dk":
            value, bound = (x.view(2, s, 2, g, d).sum(3) for x in (value, bound))
        W.check(got, (value, (bound + W.H * (value.abs() + bound)) * 1.01 + 1e-30), name)
    if window == 1:
        assert float(dq.abs().max()) <= 2.0 ** -10


@pytest.mark.parametrize("h", [65, 100, 128])
def test_groups_that_the_backward_leaves_to_the_plain_form(h):
    from cppmega_mlx_b200 import ops
    from cppmega_mlx_b200.ops import _backend as B
    q, k, v, do = _rand(1, 40, h, 32, seed=1), _rand(1, 40, 1, 32, seed=2), _rand(1, 40, 1, 32, seed=3), _rand(1, 40, h, 32, seed=4)
    ref = W.attention64(q, k, v, W.visible(40, 40, 9, 1, device="cuda"), do=do)
    before = B.launch_count("window_fwd"), B.launch_count("window_bwd")
    with torch.no_grad():
        W.check(ops.window_attention(q, k, v, window=9, sink_tokens=1), ref["o"], "o")
    assert B.launch_count("window_fwd") == before[0] + 1
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = ops.window_attention(q, k, v, window=9, sink_tokens=1)
    grads = torch.autograd.grad(o, leaves, do)
    _done()
    assert B.launch_count("window_bwd") == before[1]
    for got, name in zip((o.detach(), *grads), ("o", "dq", "dk", "dv")):
        W.check(got, ref[name], name)


def test_threads_with_streams_of_their_own():
    from cppmega_mlx_b200 import ops
    work = []
    for i in range(4):
        q, k, v = _rand(1, 150 + 40 * i, 4, 64, seed=i), _rand(1, 150 + 40 * i, 2, 64, seed=10 + i), _rand(1, 150 + 40 * i, 2, 64, seed=20 + i)
        c = _rand(2, 1 + 9 * i, 4, 64, seed=30 + i), _rand(2, 900, 2, 64, seed=40 + i), _rand(2, 900, 2, 64, seed=50 + i)
        n = torch.tensor([800, 17 * i], dtype=torch.int32, device="cuda")
        work.append((q, k, v, c, n))

    def run(item):
        q, k, v, c, n = item
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o = ops.window_attention(*leaves, window=70, sink_tokens=3)
        return [o.detach(), *torch.autograd.grad(o, leaves, q), ops.cached_attention(*c, None, n, window=500, sink_tokens=1)]
    want = [run(w) for w in work]
    _done()
    got, errors = [None] * 4, []

    def body(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[i] = run(work[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=body, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    _done()
    assert not errors and all(torch.equal(a, b) for x, y in zip(want, got) for a, b in zip(x, y))


def test_backward_beside_other_work_on_the_stream():
    """The gradients of keys and of queries run side by side; what follows on the stream finds both complete."""
    from cppmega_mlx_b200 import ops
    q, k, v = (_rand(1, 3000, n, 128, seed=n).requires_grad_() for n in (8, 2, 2))
    do = _rand(1, 3000, 8, 128, seed=9)
    o = ops.window_attention(q, k, v, window=700, sink_tokens=8)
    want = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    _done()
    for _ in range(20):
        sums = [x.float().sum() for x in torch.autograd.grad(o, (q, k, v), do, retain_graph=True)]
        for s, w in zip(sums, want):
            assert torch.equal(s, w.float().sum())
    _done()


def test_captured_backwards_with_joined_keys_side_by_side():
    """Two captured training steps whose first tokens' keys are split and joined and whose sinks are trained, replayed on two streams."""
    from cppmega_mlx_b200 import ops

    def make(seed, s):
        leaves = [_rand(1, s, n, 64, seed=seed + n).requires_grad_() for n in (4, 2, 1)]
        leaves[2] = _rand(1, s, 2, 64, seed=seed + 9).requires_grad_()
        leaves.append(_rand(4, seed=seed + 5).requires_grad_())
        do = _rand(1, s, 4, 64, seed=seed + 6)

        def step():
            o = ops.window_attention(*leaves[:3], window=60, sink_tokens=6, sinks=leaves[3])
            return [o.detach(), *torch.autograd.grad(o, leaves, do)]
        return leaves, step
    sides, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for side, (seed, s) in zip(sides, ((0, 2100), (50, 1500))):
        leaves, step = make(seed, s)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        with torch.no_grad():
            leaves[0].mul_(-0.5)
        graphs.append((g, out, step))
    want = [step() for _, _, step in graphs]
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for side, (g, _, _) in zip(sides, graphs):
            with torch.cuda.stream(side):
                g.replay()
    _done()
    for w, (_, out, _) in zip(want, graphs):
        assert all(torch.equal(a, b) for a, b in zip(w, out))
