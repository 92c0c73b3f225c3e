"""Causal attention over a sliding window, with a few first tokens that stay visible to every query.

``window_attention(q, k, v)`` takes ``q`` [B, S, H, Dq], ``k`` [B, T, Hk, Dq] and ``v`` [B, T, Hk, Dv] with ``T >= S``: the queries are
the last S positions of the T that the keys hold (``T == S`` in training; a prompt over a filled cache has more keys).  The query
at position P sees key j when

* ``j <= P``, and ``j < key_lengths[b]`` where lengths are given (padding at the end of a row of the batch; lengths outside 0 .. T
  count as the nearest inside, and the kernel reports them through ``ops.check_status``), and
* ``P - j < window`` (the window counts the query's own position) or ``j < sink_tokens``.

``sinks`` [H] adds, per head, one key of that logit whose value is 0 (learned sink logits).  Softmax statistics are fp32; a query
that sees no key yields zeros.  Gradients flow to q, k, v and ``sinks``; a grouped key head's gradient is the sum over its heads.
A key that no query sees may hold anything (NaN included) and gets zero gradients.

CUDA bf16 tensors whose head sizes are multiples of 8 up to 128 run ``csrc/window_attn.cu`` and ``csrc/window_attn_bwd.cu``
(tcgen05; work and memory proportional to the visible pairs, no S x T tensor, no atomics: results do not depend on the order
in which thread blocks run).  Everything else, forward-mode derivatives and gradients with ``create_graph`` among it, uses
``window_attention_reference``, which is also the test oracle.  The module
form is ``nn.attention.CausalSelfAttention`` (``sliding_window``, ``sink_tokens``); single tokens and drafted tokens over a cache:
``ops.cached_attention``.  Window semantics: ``cppmega_mlx/nn/attention.py:214-248``.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import numbers
import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _backend as B

NO_WINDOW = 1 << 30
NUM_SMS = 148
JOIN_ROWS = 64         # as the kernel has it
JOIN_TILES = 32        # 4 tiles for each of 8 blocks take as long as a second kernel that joins more of them (8 heads over 2048 keys: 9.4, 10.4 us)
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
    # plain numbers only: prepared calls are found by their options' values, and a tensor's may change
    if window is not None and (not isinstance(window, numbers.Integral) or window < 1):
        raise ValueError(f"{what}: window must be positive and whole, got {window}")
    if not isinstance(sink_tokens, numbers.Integral) or sink_tokens < 0:
        raise ValueError(f"{what}: sink_tokens must be whole and not negative, got {sink_tokens}")
    if sinks is not None and (sinks.shape != (q.shape[2],) or sinks.device != q.device or not sinks.is_floating_point()):
        raise ValueError(f"{what}: sinks must be {q.shape[2]} logits on {q.device}, got {tuple(sinks.shape)} on {sinks.device}")
    scale = q.shape[3] ** -0.5 if scale is None else scale
    if not (isinstance(scale, numbers.Real) and scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be a positive and finite number, got {scale}")
    return float(scale)


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
def _other_device(device: torch.device):
    with torch.cuda.device(device):
        yield


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """Kernels run on the current device's current stream: make it the tensors' device for the call."""
    return _HERE if device.index == torch.cuda.current_device() else _other_device(device)


def usable(t: torch.Tensor) -> bool:
    """A layout that the kernels read in place (its address apart, which must be a multiple of 16 bytes): unit inner stride, other
    strides (of dimensions longer than 1) positive multiples of 8 elements."""
    return t.stride(-1) == 1 and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def in_place(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a dense copy of it where the kernels cannot read it as it lies."""
    if usable(t):
        return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
    return t.contiguous()


def strides3(t: torch.Tensor) -> tuple[int, int, int]:
    """Element strides of the first three dimensions; 0 where a dimension has one entry (its stride says nothing)."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3]))


def kernel_covers(q, k, v, sinks=None) -> bool:
    """Types, head sizes, groups and devices of the kernels (layouts apart), with the backward where gradients are wanted."""
    return B.on_gpu(q, k, v) and _sizes_covered(q, k, v) and (_heads_covered_grad(q, k) or not _wants_grad(q, k, v, sinks))


def _heads_covered_grad(q, k) -> bool:
    return q.shape[2] // k.shape[2] <= MAX_GROUP_GRAD and q.shape[2] <= 65535


def _wants_grad(q, k, v, sinks) -> bool:
    return torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (sinks is not None and sinks.requires_grad))


def _sizes_covered(q, k, v) -> bool:
    dq, dv = q.shape[3], v.shape[3]
    return (q.is_cuda and q.dtype == k.dtype == v.dtype == torch.bfloat16 and dq % 8 == 0 and dv % 8 == 0 and dq <= MAX_HEAD_DIM
            and dv <= MAX_HEAD_DIM and q.shape[2] // k.shape[2] <= MAX_GROUP and k.shape[2] <= 65535 and q.shape[0] <= 65535)


def choose_splits(ctas: int, tiles: int, rows: int) -> int:
    """How many ways to split the key axis of ``ctas`` thread blocks whose rows see about ``tiles`` 64-key tiles: enough blocks for
    every SM, which holds two, and a tile or more to a block.  Up to 8 of up to 64 ``rows`` are joined within the kernel, so few tiles
    get no more there."""
    return max(1, min(2 * NUM_SMS // max(1, ctas), tiles, 8 if rows <= JOIN_ROWS and tiles <= JOIN_TILES else 64))


def row_blocks(s: int, g: int) -> int:
    """Thread blocks per (sequence, key head): 128 // g queries each."""
    return -(-s // (128 // g))


def sink_split(s: int, t: int, window: int, sink_tokens: int, g: int) -> tuple[int, int]:
    """(key tiles of the first tokens, thread blocks that share the rows of each) for the backward: every row sees the first
    tokens' keys, where another key tile is seen by about ``window + 128`` positions."""
    if window >= t or sink_tokens == 0:
        return 0, 1
    tiles = -(-min(sink_tokens, t) // 128)
    return tiles, max(1, min(64, -(-s // (window + 128))))


def meta(t):
    """What a call's preparation depends on of a tensor: nothing of its address or contents."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def has_tangent(*tensors) -> bool:
    """Whether forward-mode differentiation runs through any of them: the kernels would lose the tangent without a word."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class Plans:
    """Prepared calls by their tensors' layouts and their options (checks done, arguments packed); forgotten when there are many."""

    def __init__(self, most: int = 1024):
        self.most, self.plans = most, {}

    def get(self, key, make, *args):
        plan = self.plans.get(key)
        if plan is None:
            plan = make(*args)
            if len(self.plans) >= self.most:
                self.plans.clear()
            self.plans[key] = plan
        return plan


_CALL, _AT = struct.Struct("18i12qd"), struct.Struct("12Q")               # cmb_window_call, cmb_window_ptrs
_BWD_CALL, _BWD_AT = struct.Struct("12i24qd"), struct.Struct("16Q")       # cmb_window_bwd_call, cmb_window_bwd_ptrs
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_entries: dict[str, object] = {}


def entry(name: str, *argtypes):
    fn = _entries.get(name)
    if fn is None:
        fn = getattr(B.load_library(), name)
        fn.argtypes, fn.restype = argtypes, ctypes.c_int
        _entries[name] = fn
    return fn


def addr(t) -> int:
    return 0 if t is None else t.data_ptr()


class ForwardPlan(NamedTuple):
    covered: bool              # by the kernel, as far as types and sizes go
    ready: bool                # the layouts are read in place
    scale: float
    call: bytes = b""
    out_shape: tuple = ()
    rows: int = 0              # B S H
    ws: int = 0                # floats of scratch; the (max, sum) pairs begin at ws_ml
    ws_ml: int = 0
    convert: tuple = (False, False, False)    # lengths, table, sinks need another type or layout
    window: int = 0
    sink_tokens: int = 0
    bwd: dict | None = None


def plan_forward(q, k, v, *, t: int, lengths, cached: bool, tree, table, page: int, window, sink_tokens, sinks, scale,
                 max_keys: int | None = None) -> ForwardPlan:
    """Arguments of ``cmb_window_fwd`` for checked tensors in usable layouts."""
    b, s, h, dq = q.shape
    hk, dv = v.shape[2], v.shape[3]
    w = NO_WINDOW if window is None else min(int(window), NO_WINDOW)
    g = h // hk
    blocks = row_blocks(s, g)
    span = s if tree is not None or blocks == 1 else 128 // g
    reach = min(t if max_keys is None else min(t, max_keys), w + span)
    splits = choose_splits(b * hk * blocks, -(-reach // 64) + -(-min(sink_tokens, t) // 64), s * g)
    if b * splits > 65535:
        splits = 1
    box_k = 64 if table is None else min(64, page & -page)     # key rows of one copy; a tile is 64 keys
    out_shape = (b, s, h, dv)
    o = tuple(x if n > 1 else 0 for n, x in zip(out_shape, (s * h * dv, h * dv, dv)))
    sinks_bf16 = sinks is not None and sinks.dtype == torch.bfloat16
    rows = b * s * h
    call = _CALL.pack(b, s, t, h, hk, dq, dv, w, min(int(sink_tokens), NO_WINDOW), int(cached),
                      s if tree is not None and tree.dim() == 2 else 0, 0 if table is None else table.shape[1], page,
                      k.shape[0] if table is not None else 0, box_k, splits, int(sinks_bf16), 0, *strides3(q), *strides3(k), *strides3(v),
                      *o, scale)
    plain = lambda x: x is not None and (x.dtype != torch.int32 or not x.is_contiguous())  # noqa: E731
    return ForwardPlan(True, True, scale, call, out_shape, rows, rows * splits * (dv + 2) if splits > 8 or (splits > 1 and s * g > JOIN_ROWS) else 0, rows * splits * dv,
                       (plain(lengths), plain(table), sinks is not None and (sinks.dtype not in (torch.bfloat16, torch.float32)
                                                                            or not sinks.is_contiguous())), w, int(sink_tokens), {})


def launch_forward(plan: ForwardPlan, q, k, v, lengths, tree, table, sinks, want_lse: bool):
    """(o, lse or None) of a plan whose tensors are converted; the current device is theirs."""
    dev = q.device
    out = q.new_empty(plan.out_shape)
    b, s, h, _ = plan.out_shape
    lse = q.new_empty((b, h, s), dtype=torch.float32) if want_lse else None
    ws = q.new_empty(plan.ws, dtype=torch.float32) if plan.ws else None
    w0 = addr(ws)
    at = _AT.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), addr(lengths), addr(tree), addr(table), addr(sinks), out.data_ptr(), addr(lse),
                  w0, w0 + 4 * plan.ws_ml if w0 else 0, B.status_buffer(dev).data_ptr())
    B.check(entry("cmb_window_fwd", ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p)(plan.call, at, _raw_stream(dev.index)), "window_fwd")
    return out, lse


_INT32 = torch.iinfo(torch.int32)


def int32(x: torch.Tensor) -> torch.Tensor:
    """Indexes as the kernels read them: dense int32.  What does not fit becomes the nearest value that does, which no pool, table or cache
    holds either: it is reported, and never cut to an index that happens to exist."""
    return (x if x.dtype == torch.int32 else x.clamp(_INT32.min, _INT32.max).to(torch.int32)).contiguous()


def converted(plan: ForwardPlan, lengths, table, sinks):
    a, b, c = plan.convert
    return (int32(lengths) if a else lengths, int32(table) if b else table,
            (sinks if sinks.dtype == torch.bfloat16 else sinks.float()).contiguous() if c else sinks)     # bf16 stays: the call says so


def _plan_backward(q, k, v, do, sinks, plan: ForwardPlan, need_q: bool, need_kv: bool, need_s: bool):
    b, s, h, dq = q.shape
    t, hk, dv = v.shape[1:]
    g = h // hk
    tiles, splits = sink_split(s, t, plan.window, plan.sink_tokens, g)
    if not need_kv:
        splits = 1
    dense = lambda x: tuple(st if n > 1 else 0 for n, st in zip(x.shape, (x.shape[1] * x.shape[2] * x.shape[3], x.shape[2] * x.shape[3], x.shape[3])))  # noqa: E731
    o = tuple(st if n > 1 else 0 for n, st in zip(plan.out_shape, (s * h * dv, h * dv, dv)))
    call = _BWD_CALL.pack(b, s, t, h, hk, dq, dv, plan.window, min(plan.sink_tokens, NO_WINDOW), tiles, splits,
                          int(sinks is not None and sinks.dtype == torch.bfloat16), *strides3(q), *strides3(k), *strides3(v), *o, *strides3(do),
                          *dense(q), *dense(k), *dense(v), plan.scale)
    n_stats = 2 * plan.rows
    n_sink = h * b * -(-s // min(s, 128 // g)) if need_s else 0
    n_part = b * hk * tiles * splits * 128 * (dq + dv) if splits > 1 else 0
    return call, n_stats, n_sink, n_part


class _WindowAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sinks, lengths, plan):
        out, lse = launch_forward(plan, q, k, v, lengths, None, None, sinks, True)
        ctx.save_for_backward(q, k, v, sinks, lengths, out, lse)
        ctx.plan = plan
        return out

    @staticmethod
    def backward(ctx, do):
        q, k, v, sinks, lengths, out, lse = ctx.saved_tensors
        plan = ctx.plan
        need_q, need_k, need_v, need_s = ctx.needs_input_grad[:4]
        if torch.is_grad_enabled():        # gradients that are differentiated again (create_graph): the plain form's
            need = (need_q, need_k, need_v, need_s)
            # (each input as a tensor of its own: one that is used twice gets each use's part)
            own = [None if t is None else t.view_as(t) for t in (q, k, v, sinks)]
            o = window_attention_reference(*own[:3], window=plan.window, sink_tokens=plan.sink_tokens, sinks=own[3], key_lengths=lengths, scale=plan.scale)
            grads = iter(torch.autograd.grad(o, [t for t, n in zip(own, need) if n], do, create_graph=True))
            return *(next(grads) if n else None for n in need), None, None
        need_kv = need_k or need_v
        do = in_place(do)
        dev = q.device
        key = (do.stride(), need_q, need_kv, need_s)
        prepared = plan.bwd.get(key)
        if prepared is None:
            prepared = plan.bwd[key] = _plan_backward(q, k, v, do, sinks, plan, need_q, need_kv, need_s)
        call, n_stats, n_sink, n_part = prepared
        with on_device(dev):
            dq = q.new_empty(q.shape) if need_q or need_s else None
            dk = k.new_empty(k.shape) if need_kv else None
            dv = v.new_empty(v.shape) if need_kv else None
            ds = sinks.new_empty(sinks.shape) if need_s else None
            n_stats_up = -(-n_stats // 4) * 4                # every part of the scratch begins on 16 bytes
            ws = q.new_empty(n_stats_up + n_part + n_sink, dtype=torch.float32)
            w0 = ws.data_ptr()
            at = _BWD_AT.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), do.data_ptr(), addr(lengths), addr(sinks), lse.data_ptr(),
                              addr(dq), addr(dk), addr(dv), addr(ds), w0, w0 + 4 * (n_stats_up + n_part) if n_sink else 0,
                              w0 + 4 * n_stats_up if n_part else 0, B.status_buffer(dev).data_ptr())
            B.check(entry("cmb_window_bwd", ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p)(call, at, _raw_stream(dev.index)), "window_bwd")
        return dq if need_q else None, dk if need_k else None, dv if need_v else None, ds, None, None


_plans = Plans()


def _plan(q, k, v, window, sink_tokens, sinks, key_lengths, scale) -> ForwardPlan:
    scale = _check(q, k, v, window, sink_tokens, sinks, scale, "window_attention")
    if q.shape[0] != k.shape[0]:
        raise ValueError(f"window_attention: batches of q ({q.shape[0]}) and k ({k.shape[0]}) differ")
    if k.shape[1] < q.shape[1]:
        raise ValueError(f"window_attention: {q.shape[1]} queries are the last positions of at least as many keys, got {k.shape[1]}")
    if key_lengths is not None:
        _check_lengths(key_lengths, q.shape[0], q.device, "window_attention: key_lengths")
    if not _sizes_covered(q, k, v) or k.shape[1] > NO_WINDOW // 2 or q.shape[0] == 0 or q.shape[1] == 0:
        return ForwardPlan(False, False, scale)
    if not (usable(q) and usable(k) and usable(v)):
        return ForwardPlan(True, False, scale)
    return plan_forward(q, k, v, t=k.shape[1], lengths=key_lengths, cached=False, tree=None, table=None, page=0, window=window,
                        sink_tokens=sink_tokens, sinks=sinks, scale=scale)


def window_attention(q, k, v, *, window: int | None = None, sink_tokens: int = 0, sinks: torch.Tensor | None = None,
                     key_lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """See the module docstring; returns [B, S, H, Dv] in ``q.dtype``."""
    plan = _plans.get((meta(q), meta(k), meta(v), meta(sinks), meta(key_lengths), window, sink_tokens, scale),
                      _plan, q, k, v, window, sink_tokens, sinks, key_lengths, scale)
    grad = _wants_grad(q, k, v, sinks)
    if not plan.covered or not B.kernels_enabled() or (grad and not _heads_covered_grad(q, k)) or has_tangent(q, k, v, sinks):
        return window_attention_reference(q, k, v, window=window, sink_tokens=sink_tokens, sinks=sinks, key_lengths=key_lengths, scale=scale)
    if not plan.ready or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        return window_attention(in_place(q), in_place(k), in_place(v), window=window, sink_tokens=sink_tokens, sinks=sinks,
                                key_lengths=key_lengths, scale=scale)
    with on_device(q.device):
        lengths, _, sk = converted(plan, key_lengths, None, sinks)
        if grad:
            return _WindowAttentionFn.apply(q, k, v, sk, lengths, plan)
        return launch_forward(plan, q, k, v, lengths, None, None, sk, False)[0]
