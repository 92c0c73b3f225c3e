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
