"""Attention of the newest tokens of every sequence over its cache: a tree of drafted tokens, a chain of them (a chunk of a prompt),
or a single next token; with an optional sliding window and first tokens that stay visible.

``q`` [B, N, H, Dq] are N new tokens per sequence whose keys and values have been written to the cache already, at positions
``prefix_lengths[b] .. prefix_lengths[b] + N - 1``.  The cache is read in place:

* paged: ``k_rows`` / ``v_rows`` are views ``[num_pages, page_size, kv_heads, D]`` of one layer of a block pool and ``table`` [B, W]
  int32 maps a sequence's logical pages to pool pages;
* contiguous: ``table is None`` and the views are ``[B, T, kv_heads, D]``.

``tree`` [N] (one for the batch) or [B, N] int64, N <= 64: bit m of word n is set where token n sees token m — itself and its
ancestors (``tree_words``); bits from N on say nothing.  Token n then stands at position ``prefix + (bits of word n) - 1``, a token whose word is 0 is padding
and yields zeros.  ``tree is None``: a chain, token n sees all tokens up to itself (any N).  Every token sees the sequence's
prefix.  ``window`` and ``sink_tokens`` restrict both by position: a key at position j is seen from position P when ``P - j < window``
or ``j < sink_tokens``.  ``sinks`` [H]: one more key per head with that logit and value 0.

What no token sees — rows past a sequence's end, table entries past them, pages behind the window — may hold anything.  A table
entry or a length that the pool or the table cannot hold is reported by ``ops.check_status`` (nothing is read outside the pool); with
CPU tensors it is a ``ValueError``.

CUDA bf16 tensors run ``csrc/window_attn.cu`` (tcgen05, split over the keys when there are few rows).  CPU tensors, other types, heads that
are not a multiple of 8 or larger than 128, page sizes that are not a multiple of 8, and cache rows whose address or strides are not
multiples of 16 bytes use ``cached_attention_reference``, the test oracle, which gathers every sequence's whole capacity in fp32.  No gradients,
neither mode: inputs that require one are refused.  The reference verifies drafts as a plain chain (``cppmega_mlx/inference/speculative_decode.py:92``) and never attends
over its pages (``cppmega_mlx/inference/serving.py:522``).
"""
from __future__ import annotations

import torch

from . import _backend as B
from .window_attention import (NO_WINDOW, ForwardPlan, Plans, _check, _check_lengths, _sizes_covered, _wants_grad, converted,
                               has_tangent, in_place, launch_forward, masked_softmax_attention, meta, on_device, plan_forward, usable)

MAX_TREE = 64


def tree_words(parents) -> torch.Tensor:
    """[N] or [B, N] parents (the index of each drafted token's parent among the drafted tokens; -1: it follows the prefix; -2:
    padding) in an order where a parent stands before its children → int64 words for ``cached_attention(tree=...)``, on the CPU."""
    par = torch.as_tensor(parents, dtype=torch.int64).cpu()
    if par.dim() not in (1, 2) or par.shape[-1] > MAX_TREE:
        raise ValueError(f"tree_words: parents must be [N] or [B, N] with N <= {MAX_TREE}, got {tuple(par.shape)}")
    rows = []
    for row in par.reshape(-1, par.shape[-1]).tolist():
        words: list[int] = []
        for n, m in enumerate(row):
            if m >= n or m < -2 or (m >= 0 and words[m] == 0):
                raise ValueError(f"tree_words: token {n} has parent {m}: parents stand before their children and are no padding")
            words.append(0 if m == -2 else (words[m] if m >= 0 else 0) | (1 << n))
        rows.append([w - (1 << 64) if w >> 63 else w for w in words])
    return torch.tensor(rows, dtype=torch.int64).reshape(par.shape)


def _checked(q, k_rows, v_rows, table, prefix_lengths, tree, window, sink_tokens, sinks, scale):
    scale = _check(q, k_rows, v_rows, window, sink_tokens, sinks, scale, "cached_attention")
    b, n = q.shape[:2]
    _check_lengths(prefix_lengths, b, q.device, "cached_attention: prefix_lengths")
    if table is not None:
        if table.dim() != 2 or table.shape[0] != b or table.dtype not in (torch.int32, torch.int64) or table.device != q.device:
            raise ValueError(f"cached_attention: table must be [{b}, pages] int32 / int64 on {q.device}, got {tuple(table.shape)} "
                             f"{table.dtype} on {table.device}")
    elif k_rows.shape[0] != b:
        raise ValueError(f"cached_attention: a contiguous cache has {b} rows, got {k_rows.shape[0]}")
    if tree is not None:
        if tree.shape not in ((n,), (b, n)) or tree.dtype != torch.int64 or tree.device != q.device:
            raise ValueError(f"cached_attention: tree must be int64 words [{n}] or [{b}, {n}] on {q.device}, got {tuple(tree.shape)} "
                             f"{tree.dtype} on {tree.device}")
        if n > MAX_TREE:
            raise ValueError(f"cached_attention: a tree has at most {MAX_TREE} tokens, got {n}")
    return scale


def _no_gradient(q, k_rows, v_rows, sinks) -> None:
    if _wants_grad(q, k_rows, v_rows, sinks) or has_tangent(q, k_rows, v_rows, sinks):
        raise ValueError("cached_attention has no gradient: call it under torch.no_grad(), or use window_attention")


def _refuse(bad: torch.Tensor, what: str) -> None:
    """As the kernel does: reported by ``ops.check_status``; on the CPU, where reading ``bad`` costs nothing, raised."""
    if bad.device.type != "cpu":
        B.report(bad)
    elif bool(bad):
        raise ValueError(f"cached_attention: {what}")


def cached_attention_reference(q, k_rows, v_rows, table, prefix_lengths, *, tree=None, window: int | None = None, sink_tokens: int = 0,
                               sinks=None, scale: float | None = None):
    scale = _checked(q, k_rows, v_rows, table, prefix_lengths, tree, window, sink_tokens, sinks, scale)
    _no_gradient(q, k_rows, v_rows, sinks)
    b, n = q.shape[:2]
    dev = q.device
    page = k_rows.shape[1]
    t = page * (1 if table is None else table.shape[1])
    asked = prefix_lengths.long()
    prefix = asked.clamp(0, max(0, t - n))
    _refuse((prefix != asked).any() if t >= n else torch.ones((), dtype=torch.bool, device=dev), f"prefix_lengths and {n} tokens do not fit into {t} rows")
    idx = torch.arange(n, device=dev)
    bits = (idx[None] <= idx[:, None])[None] if tree is None else ((tree.reshape(-1, n, 1) >> idx) & 1).bool()
    bits = bits.expand(b, n, n)
    depth = bits.sum(-1) - 1
    pos = (prefix[:, None] + depth)[..., None]                            # [B, N, 1]
    j = torch.arange(t, device=dev)[None, None]
    w = NO_WINDOW if window is None else window
    old = (j < prefix[:, None, None]) & ((pos - j < w) | (j < sink_tokens)) & (depth >= 0)[..., None]
    m = (j[:, 0] - prefix[:, None]).clamp(0, max(n - 1, 0))               # [B, T]: which drafted token a row holds
    held = (j >= prefix[:, None, None]) & (j < prefix[:, None, None] + n)
    mpos = (prefix[:, None] + depth.gather(1, m))[:, None]                # [B, 1, T]
    new = bits.gather(2, m[:, None].expand(b, n, t)) & held & ((pos - mpos < w) | (mpos < sink_tokens))
    k, v = k_rows, v_rows
    if table is not None:       # entries that no token reads may be anything
        pages = table.long()
        inside = (pages >= 0) & (pages < k_rows.shape[0])
        _refuse(((old | new).any(1).view(b, table.shape[1], page).any(-1) & ~inside).any(), f"table names a page outside the pool of {k_rows.shape[0]}")
        pages = torch.where(inside, pages, torch.zeros_like(pages))
        k, v = (x[pages].flatten(1, 2) if x.shape[0] else x.new_zeros(b, t, *x.shape[2:]) for x in (k_rows, v_rows))
    return masked_softmax_attention(q, k, v, old | new, sinks, scale)


_plans = Plans()


def _plan(q, k_rows, v_rows, table, prefix_lengths, tree, window, sink_tokens, sinks, scale, max_keys) -> ForwardPlan:
    scale = _checked(q, k_rows, v_rows, table, prefix_lengths, tree, window, sink_tokens, sinks, scale)
    rows = k_rows.shape[1]
    t = rows * (1 if table is None else table.shape[1])
    if (not _sizes_covered(q, k_rows, v_rows) or not (usable(k_rows) and usable(v_rows)) or 0 in q.shape[:2] or not q.shape[1] <= t <= NO_WINDOW // 2
            or (table is not None and (rows % 8 or not k_rows.shape[0]))):
        return ForwardPlan(False, False, scale)
    if not usable(q):
        return ForwardPlan(True, False, scale)
    return plan_forward(q, k_rows, v_rows, t=t, lengths=prefix_lengths, cached=True, tree=tree, table=table, page=rows if table is not None else 0,
                        window=window, sink_tokens=sink_tokens, sinks=sinks, scale=scale, max_keys=max_keys)


def cached_attention(q, k_rows, v_rows, table, prefix_lengths, *, tree: torch.Tensor | None = None, window: int | None = None,
                     sink_tokens: int = 0, sinks: torch.Tensor | None = None, scale: float | None = None,
                     max_keys: int | None = None) -> torch.Tensor:
    """See the module docstring; returns [B, N, H, Dv] in ``q.dtype``.  ``max_keys`` (a bound on ``prefix_lengths + N``) only tunes how
    the work is split and never costs correctness."""
    if tree is not None:
        tree = tree.contiguous()
    plan = _plans.get((meta(q), meta(k_rows), meta(v_rows), meta(table), meta(prefix_lengths), meta(tree), meta(sinks), window, sink_tokens, scale,
                       max_keys), _plan, q, k_rows, v_rows, table, prefix_lengths, tree, window, sink_tokens, sinks, scale, max_keys)
    _no_gradient(q, k_rows, v_rows, sinks)
    if q.shape[0] == 0 or q.shape[1] == 0:
        return q.new_zeros(*q.shape[:3], v_rows.shape[3])
    if not plan.covered or not B.kernels_enabled() or (k_rows.data_ptr() | v_rows.data_ptr()) % 16:
        return cached_attention_reference(q, k_rows, v_rows, table, prefix_lengths, tree=tree,
                                          window=window, sink_tokens=sink_tokens, sinks=sinks, scale=scale)
    if not plan.ready or q.data_ptr() % 16:
        return cached_attention(in_place(q), k_rows, v_rows, table, prefix_lengths, tree=tree, window=window, sink_tokens=sink_tokens,
                                sinks=sinks, scale=scale, max_keys=max_keys)
    with on_device(q.device):
        lengths, tbl, sk = converted(plan, prefix_lengths, table, sinks)
        return launch_forward(plan, q, k_rows, v_rows, lengths, tree, tbl, sk, False)[0]
