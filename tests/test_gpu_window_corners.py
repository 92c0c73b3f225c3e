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
