"""Causal attention over a sliding window, with a few first tokens that stay visible to every query.

``window_attention(q, k, v)`` takes ``q`` [B, S, H, Dq], ``k`` [B, T, Hk, Dq] and ``v`` [B, T, Hk, Dv] with ``T >= S``: the queries are
the last S positions of the T that the keys hold (``T == S`` in training; a prompt over a filled cache has more keys).  The query
at position P sees key j when

* ``j <= P``, and ``j < key_lengths[b]`` where lengths are given (padding at the end of a row of the batch), and
* ``P - j < window`` (the window counts the query's own position) or ``j < sink_tokens``.

``sinks`` [H] adds, per head, one key of that logit whose value is 0 (learned sink logits).  Softmax statistics are fp32; a query
that sees no key yields zeros.  Gradients flow to q, k, v and ``sinks``; a grouped key head's gradient is the sum over its heads.
A key that no query sees may hold anything (NaN included) and gets zero gradients.

CUDA bf16 tensors whose head sizes are multiples of 8 up to 128 run ``csrc/window_attn.cu`` and ``csrc/window_attn_bwd.cu``
(tcgen05; work and memory proportional to the visible pairs, no S x T tensor, no atomics: results do not depend on the order
in which thread blocks run).  Everything else uses ``window_attention_reference``, which is also the test oracle.  The module
form is ``nn.attention.CausalSelfAttention`` (``sliding_window``, ``sink_tokens``); single tokens and drafted tokens over a cache:
``ops.cached_attention``.  Window semantics: ``cppmega_mlx/nn/attention.py:214-248``.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import _backend as B

NO_WINDOW = 1 << 30
NUM_SMS = 148
MAX_HEAD_DIM = 128
MAX_GROUP = 128
MAX_GROUP_GRAD = 64        # the backward's sub-tiles hold 64 rows


def _check(q, k, v, window, sink_tokens, sinks, scale, what: str) -> float:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{what}: q, k and v have 4 dimensions, got {q.dim()}, {k.dim()}, {v.dim()}")
    if not (q.dtype == k.dtype == v.dtype) or not q.is_floating_point():
        raise ValueError(f"{what}: q, k and v have one floating type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if not (q.device == k.device == v.device):
        raise ValueError(f"{what}: q, k and v are on one device")
    if k.shape[:3] != v.shape[:3]:
        raise ValueError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ in more than the head size")
    if q.shape[3] != k.shape[3]:
        raise ValueError(f"{what}: head size of q ({q.shape[3]}) and k ({k.shape[3]}) differ")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"{what}: {q.shape[2]} query heads are not a multiple of {k.shape[2]} key heads")
    if q.shape[3] == 0 or v.shape[3] == 0:
        raise ValueError(f"{what}: head sizes must be positive")
    if window is not None and window < 1:
        raise ValueError(f"{what}: window must be positive, got {window}")
    if sink_tokens < 0:
        raise ValueError(f"{what}: sink_tokens must not be negative, got {sink_tokens}")
    if sinks is not None and (sinks.shape != (q.shape[2],) or sinks.device != q.device or not sinks.is_floating_point()):
        raise ValueError(f"{what}: sinks must be {q.shape[2]} logits on {q.device}, got {tuple(sinks.shape)} on {sinks.device}")
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be positive and finite, got {scale}")
    return scale


def _check_lengths(n, batch: int, device, what: str) -> None:
    if n.shape != (batch,) or n.dtype not in (torch.int32, torch.int64) or n.device != device:
        raise ValueError(f"{what} must be {batch} int32 / int64 values on {device}, got {tuple(n.shape)} {n.dtype} on {n.device}")


def masked_softmax_attention(q, k, v, seen, sinks, scale):
    """The plain form: ``seen`` [B | 1, S, T] (True = visible); fp32 throughout, rounded once; zeros where a row sees nothing."""
    b, s, h, d = q.shape
    hk = k.shape[2]
    sc = torch.einsum("bsgrd,btgd->bgrst", q.float().reshape(b, s, hk, h // hk, d), k.float()) * scale
    sc = sc.masked_fill(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True) if sc.shape[-1] else sc.new_full((*sc.shape[:-1], 1), float("-inf"))
    sk = None if sinks is None else sinks.float().view(1, hk, h // hk, 1, 1)
    if sk is not None:
        top = torch.maximum(top, sk)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top).detach()
    e = torch.exp(sc - top)
    total = e.sum(-1, keepdim=True)
    if sk is not None:
        total = total + torch.exp(sk - top)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    vf = torch.where(seen.any(1)[:, :, None, None], v.float(), v.new_zeros(()).float())   # what nobody sees may hold anything
    return torch.einsum("bgrst,btgd->bsgrd", p, vf).reshape(b, s, h, v.shape[3]).to(q.dtype)


def window_mask(s: int, t: int, window: int | None, sink_tokens: int, key_lengths=None, device=None) -> torch.Tensor:
    """[B | 1, S, T] visibility of ``window_attention``."""
    p = torch.arange(t - s, t, device=device)[:, None]
    j = torch.arange(t, device=device)[None]
    seen = j <= p
    if window is not None:
        seen = seen & ((p - j < window) | (j < sink_tokens))
    seen = seen[None]
    return seen if key_lengths is None else seen & (j[None] < key_lengths.view(-1, 1, 1))


def window_attention_reference(q, k, v, *, window: int | None = None, sink_tokens: int = 0, sinks=None, key_lengths=None,
                               scale: float | None = None):
    scale = _check(q, k, v, window, sink_tokens, sinks, scale, "window_attention")
    return masked_softmax_attention(q, k, v, window_mask(q.shape[1], k.shape[1], window, sink_tokens, key_lengths, q.device), sinks, scale)


# ------------------------------------------------------------------------------------------------------------ kernel path
@contextlib.contextmanager
def on_device(device: torch.device):
    """Kernels run on the current device's current stream: make it the tensors' device for the call."""
    if device.index == torch.cuda.current_device():
        yield
    else:
        with torch.cuda.device(device):
            yield


def usable(t: torch.Tensor) -> bool:
    """A layout that the kernels read in place: unit inner stride, other strides (of dimensions longer than 1) positive
    multiples of 8 elements, 16-byte aligned."""
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1])))


def strides3(t: torch.Tensor) -> tuple[int, int, int]:
    """Element strides of the first three dimensions; 0 where a dimension has one entry (its stride says nothing)."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3]))


def kernel_covers(q, k, v) -> bool:
    """Types, head sizes and devices of the kernels (layouts apart)."""
    dq, dv = q.shape[3], v.shape[3]
    return (B.on_gpu(q, k, v) and q.dtype == k.dtype == v.dtype == torch.bfloat16 and dq % 8 == 0 and dv % 8 == 0
            and dq <= MAX_HEAD_DIM and dv <= MAX_HEAD_DIM and q.shape[2] // k.shape[2] <= MAX_GROUP and k.shape[2] <= 65535)


def choose_splits(ctas: int, tiles: int) -> int:
    """How many ways to split the key axis of ``ctas`` thread blocks whose rows see about ``tiles`` 128-key tiles: enough blocks for
    every SM, two tiles (one per stream of the kernel) or more to a block."""
    return max(1, min(NUM_SMS // max(1, ctas), (tiles + 1) // 2, 64))


def row_blocks(s: int, g: int) -> int:
    """Thread blocks per (sequence, key head): up to 128 rows in one, else two row tiles of 128 // g queries each."""
    return 1 if s * g <= 128 else -(-s // (2 * (128 // g)))


def sink_split(s: int, t: int, window: int, sink_tokens: int, g: int) -> tuple[int, int]:
    """(key tiles of the first tokens, thread blocks that share the rows of each) for the backward: every row sees the first
    tokens' keys, where another key tile is seen by about ``window + 128`` positions."""
    if window >= t or sink_tokens == 0:
        return 0, 1
    tiles = -(-min(sink_tokens, t) // 128)
    return tiles, max(1, min(64, -(-s // (window + 128))))


def launch_forward(q, k, v, *, t: int, lengths, cached: bool, tree, table, page: int, window, sink_tokens, sinks, scale, want_lse: bool,
                   max_keys: int | None = None):
    """``cmb_window_fwd`` on checked arguments in usable layouts; (o, lse or None)."""
    lib = B.load_library()
    b, s, h, dq = q.shape
    hk, dv = v.shape[2], v.shape[3]
    dev = q.device
    w = NO_WINDOW if window is None else min(int(window), NO_WINDOW)
    g = h // hk
    blocks = row_blocks(s, g)
    span = s if tree is not None or blocks == 1 else 2 * (128 // g)
    reach = min(t if max_keys is None else min(t, max_keys), w + span)
    splits = choose_splits(b * hk * blocks, -(-reach // 128) + -(-min(sink_tokens, t) // 128))
    if b * splits > 65535:
        splits = 1
    one_tile = s * g <= 128                                # the kernel's form for few rows: 128 keys a tile, else 64
    box_k = 32 if one_tile else 64
    if table is not None:
        box_k = min(128 if one_tile else 64, page & -page)
    out = torch.empty(b, s, h, dv, dtype=torch.bfloat16, device=dev)
    lse = torch.empty(b, h, s, dtype=torch.float32, device=dev) if want_lse else None
    ws = torch.empty(b * s * h * splits * (dv + 2), dtype=torch.float32, device=dev) if splits > 1 else None
    ml = None if ws is None else ws[b * s * h * splits * dv:]
    ip = (ctypes.c_int * 16)(b, s, t, h, hk, dq, dv, w, min(sink_tokens, NO_WINDOW), int(cached),
                             s if tree is not None and tree.dim() == 2 else 0, 0 if table is None else table.shape[1], page,
                             k.shape[0] if table is not None else 0, box_k, splits)
    lp = (ctypes.c_longlong * 12)(*strides3(q), *strides3(k), *strides3(v), *strides3(out))
    B.check(lib.cmb_window_fwd(B.ptr(q), B.ptr(k), B.ptr(v), B.ptr(lengths), B.ptr(tree), B.ptr(table), B.ptr(sinks), B.ptr(out),
                               B.ptr(lse), B.ptr(ws), B.ptr(ml), ip, lp, ctypes.c_float(scale), B.ptr(B.status_buffer(dev)),
                               B.stream_ptr()), "window_fwd")
    return out, lse


class _WindowAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sinks, key_lengths, window, sink_tokens, scale):
        with on_device(q.device):
            sk = None if sinks is None else sinks.float().contiguous()
            out, lse = launch_forward(q, k, v, t=k.shape[1], lengths=key_lengths, cached=False, tree=None, table=None, page=0,
                                      window=window, sink_tokens=sink_tokens, sinks=sk, scale=scale, want_lse=True)
        ctx.save_for_backward(q, k, v, sinks, key_lengths, out, lse)
        ctx.args = (window, sink_tokens, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, sinks, lengths, out, lse = ctx.saved_tensors
        window, sink_tokens, scale = ctx.args
        need_q, need_k, need_v, need_s = ctx.needs_input_grad[:4]
        b, s, h, dq_ = q.shape
        t, hk, dv_ = v.shape[1:]
        do = do if usable(do) else do.contiguous()
        lib = B.load_library()
        with on_device(q.device):
            f32 = lambda *n: torch.empty(*n, dtype=torch.float32, device=q.device)  # noqa: E731
            sk = None if sinks is None else sinks.float().contiguous()
            sink_part = f32(h, b * -(-s // min(s, 128 // (h // hk)))) if sinks is not None and need_s else None
            dq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if need_q or need_s else None
            dk, dv = ((torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (k, v)) if need_k or need_v else (None, None))
            w = NO_WINDOW if window is None else min(int(window), NO_WINDOW)
            tiles, splits = sink_split(s, t, w, sink_tokens, h // hk)
            part = f32(b * hk * tiles * splits * 128 * (dq_ + dv_)) if splits > 1 and dk is not None else None
            ip = (ctypes.c_int * 11)(b, s, t, h, hk, dq_, dv_, w, min(sink_tokens, NO_WINDOW), tiles, splits if part is not None else 1)
            lp = (ctypes.c_longlong * 24)(*(st for x in (q, k, v, out, do, dq, dk, dv) for st in ((0, 0, 0) if x is None else strides3(x))))
            stats = f32(2 * b * s * h)
            B.check(lib.cmb_window_bwd(B.ptr(q), B.ptr(k), B.ptr(v), B.ptr(out), B.ptr(do), B.ptr(lengths), B.ptr(sk), B.ptr(lse),
                                       B.ptr(dq), B.ptr(dk), B.ptr(dv), B.ptr(stats), B.ptr(sink_part), B.ptr(part), ip, lp,
                                       ctypes.c_float(scale), B.ptr(B.status_buffer(q.device)), B.stream_ptr()), "window_bwd")
            ds = None if sink_part is None else sink_part.sum(1).to(sinks.dtype)
        return dq if need_q else None, dk if need_k else None, dv if need_v else None, ds, None, None, None, None


def window_attention(q, k, v, *, window: int | None = None, sink_tokens: int = 0, sinks: torch.Tensor | None = None,
                     key_lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """See the module docstring; returns [B, S, H, Dv] in ``q.dtype``."""
    scale = _check(q, k, v, window, sink_tokens, sinks, scale, "window_attention")
    if q.shape[0] != k.shape[0]:
        raise ValueError(f"window_attention: batches of q ({q.shape[0]}) and k ({k.shape[0]}) differ")
    if k.shape[1] < q.shape[1]:
        raise ValueError(f"window_attention: {q.shape[1]} queries are the last positions of at least as many keys, got {k.shape[1]}")
    if key_lengths is not None:
        _check_lengths(key_lengths, q.shape[0], q.device, "window_attention: key_lengths")
    if not kernel_covers(q, k, v) or k.shape[1] > NO_WINDOW // 2 or q.shape[0] > 65535:
        return window_attention_reference(q, k, v, window=window, sink_tokens=sink_tokens, sinks=sinks, key_lengths=key_lengths, scale=scale)
    if q.shape[0] == 0 or q.shape[1] == 0:
        return q.new_zeros(*q.shape[:3], v.shape[3])
    q, k, v = (x if usable(x) else x.contiguous() for x in (q, k, v))
    lengths = None if key_lengths is None else key_lengths.to(torch.int32).contiguous()
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, sinks)):
        if q.shape[2] // k.shape[2] > MAX_GROUP_GRAD:
            return window_attention_reference(q, k, v, window=window, sink_tokens=sink_tokens, sinks=sinks, key_lengths=key_lengths,
                                              scale=scale)
        return _WindowAttentionFn.apply(q, k, v, sinks, lengths, window, int(sink_tokens), scale)
    with on_device(q.device):
        sk = None if sinks is None else sinks.float().contiguous()
        return launch_forward(q, k, v, t=k.shape[1], lengths=lengths, cached=False, tree=None, table=None, page=0, window=window,
                              sink_tokens=int(sink_tokens), sinks=sk, scale=scale, want_lse=False)[0]
