"""Windowed and cached attention, page movements and the block manager at the corners of their contracts, on the CPU."""
import pytest
import torch

from cppmega_mlx_b200 import inference as I
from cppmega_mlx_b200 import ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("layout", ["dense", "strided", "expanded"])
def test_packed_type_of_the_sinks_is_that_of_what_the_kernel_reads(dtype, layout):
    import importlib
    wa = importlib.import_module("cppmega_mlx_b200.ops.window_attention")
    sinks = {"dense": torch.randn(4), "strided": torch.randn(8)[::2], "expanded": torch.randn(1).expand(4)}[layout].to(dtype)
    if layout == "strided":
        sinks = torch.randn(8).to(dtype)[::2]
    if layout == "expanded":
        sinks = torch.randn(1).to(dtype).expand(4)
    q, k = torch.zeros(1, 3, 4, 8, dtype=torch.bfloat16), torch.zeros(1, 5, 2, 8, dtype=torch.bfloat16)
    plan = wa.plan_forward(q, k, k, t=5, lengths=None, cached=False, tree=None, table=None, page=0, window=None, sink_tokens=0, sinks=sinks, scale=1.0)
    read = wa.converted(plan, None, None, sinks)[2]
    assert read.is_contiguous() and read.dtype == (torch.bfloat16 if wa._CALL.unpack(plan.call)[16] else torch.float32)
    assert torch.equal(read.double(), sinks.to(read.dtype).double())


def _released(n=32, window=8, sink=0, bs=4):
    m = I.PagedKVBlockManager(num_blocks=24, num_layers=1, block_size=bs, kv_heads=1, head_dim=8, dtype=torch.float32)
    m.allocate(1, 0)
    m.append(1, 0, torch.randn(n, 1, 8), torch.randn(n, 1, 8))
    m.release_window(1, window, sink)
    return m


def test_truncate_keeps_what_the_released_window_needs():
    for keep in (20, 28, 30):                       # the next token at 20 sees 13 .. 20; at 30 it sees 23 .. 30; block 5 holds 20 .. 23
        m = _released()
        table, free = list(m.tables[1]), m.num_free_blocks
        with pytest.raises(ValueError, match="released"):
            m.truncate(1, keep)
        assert m.tables[1] == table and m.lengths[1] == 32 and m.num_free_blocks == free
    m = _released()
    m.truncate(1, 31)                               # sees 24 .. 31
    assert m.lengths[1] == 31 and len(m.tables[1]) == 8
    m.append(1, 0, torch.ones(2, 1, 8), torch.ones(2, 1, 8))
    m = _released()
    m.truncate(1, 0)                                # nothing is left to see
    assert m.tables[1] == [] and m.num_free_blocks == 24
    m.append(1, 0, torch.ones(9, 1, 8), torch.ones(9, 1, 8))
    m.truncate(1, 5)
    m = _released(window=1)
    with pytest.raises(ValueError, match="released"):
        m.truncate(1, 30)                           # the next token would be written into a block that is gone
    m.truncate(1, 28)                               # … into a new one
    m.append(1, 0, torch.ones(1, 1, 8), torch.ones(1, 1, 8))
    m = _released(sink=6)
    with pytest.raises(ValueError, match="released"):
        m.truncate(1, 11)
    m.fork(1, 2)                                    # a fork has seen the same release
    with pytest.raises(ValueError, match="released"):
        m.truncate(2, 20)
    m.truncate(2, 31)
    m.free(1), m.free(2)
    assert m.num_free_blocks == 24
    m = _released(window=20)                        # a later, narrower release asks for less
    m.release_window(1, 4)
    m.truncate(1, 31)
    with pytest.raises(ValueError, match="released"):
        m.truncate(1, 30)


def test_plain_page_copies_skip_what_the_pool_does_not_hold():
    """The plain forms serve CUDA tensors too (pages that are not dense, kernels turned off): there an index outside is skipped and
    reported as the kernels do, and never reaches an indexing operation, which would end the process's context."""
    from cppmega_mlx_b200.ops.pages import compact_rows_reference, copy_pages_reference
    pool = torch.arange(24.).view(6, 4)
    want = pool.clone()
    want[3] = want[1]
    t = torch.tensor
    assert bool(copy_pages_reference((pool,), t([1, 9, -3, 2, -1]), t([3, 0, 0, 6, 2])))
    assert torch.equal(pool, want)
    assert not bool(copy_pages_reference((pool,), t([0, -1]), t([5, -1]))) and torch.equal(pool[5], want[0])
    assert bool(copy_pages_reference((pool,), t([0, 1]), t([2, 2]))) and bool(copy_pages_reference((pool,), t([0, 1]), t([1, 2])))
    assert not bool(copy_pages_reference((pool,), t([4]), t([4])))
    pool = torch.randn(5, 2, 4, 3)
    table = t([[4, 0], [2, 1]])
    keep = pool.clone()
    for start, path, counts, tbl in (([9, 0], [[1], [0]], [1, 0], table), ([0, 0], [[-1], [0]], [1, 0], table), ([0, 0], [[0], [0]], [2, 0], table),
                                     ([-3, 0], [[2], [0]], [1, 0], table), ([4, 0], [[1], [0]], [1, 0], t([[4, 7], [2, 1]])),
                                     ([4, 0], [[1], [0]], [1, 0], t([[4, -2], [2, 1]])), ([0, 0], [[0], [0]], [-1, 0], table)):
        assert bool(compact_rows_reference((pool,), tbl, t(start), t(path), t(counts)))
        assert torch.equal(pool, keep)
    assert not bool(compact_rows_reference((pool,), table, t([2, 0]), t([[1, 2, 5], [3, 99, -9]]), t([3, 1])))
    want = keep.clone()             # positions 3, 4 and 7 of the first sequence close up behind its second, 3 of the other moves to its start
    want[4, :, 2], want[4, :, 3], want[0, :, 0], want[2, :, 0] = keep[4, :, 3], keep[0, :, 0], keep[0, :, 3], keep[2, :, 3]
    assert torch.equal(pool, want)


def test_plain_cached_attention_stays_inside_the_pool():
    """On the CPU an entry that is read, or a length, that the pool or the table cannot hold is refused; what nobody reads may be anything."""
    q, k = torch.randn(2, 2, 2, 8), torch.randn(6, 4, 1, 8)
    table, n = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32), torch.tensor([9, 3])
    want = ops.cached_attention(q, k, k, table, n)
    hole = table.clone()
    hole[1, 2] = 10 ** 6                                        # behind the sequence's end
    assert torch.equal(ops.cached_attention(q, k, k, hole, n), want)
    narrow = ops.cached_attention(q, k, k, table, n, window=3)
    hole[0, :1] = -1                                            # behind the window: the first token at 9 sees 7, 8, 9
    assert torch.equal(ops.cached_attention(q, k, k, hole, n, window=3), narrow)
    for bad in (-1, 6, 2 ** 40):
        tbl = table.long()
        tbl[0, 1] = bad
        with pytest.raises(ValueError, match="page"):
            ops.cached_attention(q, k, k, tbl, n)
    for lens in ([-1, 3], [11, 3], [9, 2 ** 40]):
        with pytest.raises(ValueError, match="prefix"):
            ops.cached_attention(q, k, k, table, torch.tensor(lens))
    with pytest.raises(ValueError, match="page"):
        ops.cached_attention(q, k[:0], k[:0], table, n)


@pytest.mark.parametrize("shape", [(4,), (1, 4, 1, 1), (4, 1), (2, 2)])
def test_layer_takes_sinks_of_any_shape(shape):
    from cppmega_mlx_b200.nn.attention import AttentionConfig, CausalSelfAttention, flat_sinks
    torch.manual_seed(0)
    m = CausalSelfAttention(AttentionConfig(32, 4, num_kv_heads=2, mode="gqa", sliding_window=5)).eval()
    x, sinks = torch.randn(2, 9, 32), torch.randn(4)
    with torch.no_grad():
        want = m(x, sinks=sinks)
        assert torch.equal(m(x, sinks=sinks.view(shape)), want)
        cache = I.StaticDecodeCache(1, 2, 16, "cpu")
        for i in range(9):
            y = m(x[:, i:i + 1], kv_cache=cache, sinks=sinks.view(shape))
            cache.advance()
            torch.testing.assert_close(y[:, 0], want[:, i], rtol=1e-4, atol=1e-5)
    assert flat_sinks(None) is None and flat_sinks(torch.ones(2, 2, dtype=torch.int64)).dtype == torch.float32


def test_greedy_tree_accept_among_equal_siblings():
    """Two drafts of one token: the path goes on where it is longest."""
    par, tok = [-1, -1, 1, 0, 2], [5, 5, 7, 8, 9]
    assert I.greedy_tree_accept(par, tok, [5, 7, 7, 9, 0, 4]) == ([1, 2, 4], 4)
    assert I.greedy_tree_accept(par, tok, [5, 8, 8, 9, 1, 4]) == ([0, 3], 1)
    assert I.greedy_tree_accept([-1, -1], [5, 5], [5, 6, 6]) == ([0], 6)            # the first of equally long ones
    assert I.greedy_tree_accept([-1, -2, 0], [5, 5, 6], [5, 6, 0, 3]) == ([0, 2], 3)
    assert I.greedy_tree_accept([], [], [8]) == ([], 8)


@pytest.mark.parametrize("change,match", [(dict(window=torch.tensor(3)), "window"), (dict(window=2.5), "window"), (dict(sink_tokens=1.5), "sink_tokens"),
                                          (dict(sink_tokens=torch.tensor(1)), "sink_tokens"), (dict(scale=torch.tensor(0.5)), "scale")])
def test_options_are_plain_numbers(change, match):
    """Prepared calls are found by their options' values: a tensor, which is found by its identity and may change, is refused."""
    q = torch.randn(1, 6, 2, 8)
    with pytest.raises(ValueError, match=match):
        ops.window_attention(q, q, q, **{"window": 3, **change})
    with pytest.raises(ValueError, match=match):
        ops.cached_attention(q, q, q, None, torch.zeros(1, dtype=torch.int32), **{"window": 3, **change})


def test_numpy_numbers_are_numbers():
    import numpy as np
    q = torch.randn(1, 6, 2, 8)
    assert torch.equal(ops.window_attention(q, q, q, window=np.int64(3), sink_tokens=np.int32(1), scale=np.float32(0.5)),
                       ops.window_attention(q, q, q, window=3, sink_tokens=1, scale=0.5))


def test_sequences_that_move_nothing_may_stand_anywhere():
    pool = torch.randn(5, 2, 4, 3)
    keep, t = pool.clone(), torch.tensor
    ops.compact_rows(pool, t([[-1, 99], [2, 1]]), t([-1, 0]), t([[7], [0]]), t([0, 1]))
    ops.compact_rows(pool, t([[-1, 99], [2, 1]]), t([400, 0]), t([[7], [0]]), t([0, 1]))
    assert torch.equal(pool, keep)
    for start in (-1, 400):
        with pytest.raises(ValueError):
            ops.compact_rows(pool, t([[4, 0], [2, 1]]), t([start, 0]), t([[7], [0]]), t([1, 1]))


def test_positions_past_32_bits_are_refused():
    """int32 starts and paths whose sum does not fit: not wrapped to a position in front of the table."""
    pool = torch.randn(5, 2, 4, 3)
    keep = pool.clone()
    t = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="outside"):
        ops.compact_rows(pool, t([4, 0]), t(5), t([2 ** 31 - 3]), t(1))
    assert torch.equal(pool, keep)
