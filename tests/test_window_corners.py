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
