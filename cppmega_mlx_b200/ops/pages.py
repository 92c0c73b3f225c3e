"""Movements of a paged cache: pages duplicated, rows closed up within sequences.

``copy_pages(pools, src, dst)`` copies page ``src[i]`` of every pool to page ``dst[i]`` (a sequence forks, a page that others share is
about to be written, the pool is put in order).  A pool is ``[num_pages, ...]`` with dense pages.  A page is written at most once in a
call and not read in the same call; a pair (-1, -1) is an unused place of the list.

``compact_rows(pools, table, start, path, counts)`` moves, in every sequence b, the cached rows of tokens ``start[b] + path[b, i]`` to
``start[b] + i`` for ``i < counts[b]``, as if all were read before any is written: the accepted path of a drafted tree closes up
behind the prefix.  Pools are ``[num_pages, layers, page_size, ...]`` with dense rows.  The pages that a sequence's rows move to are its own:
no other sequence of the call reads or writes them.

Both work in place on CPU and CUDA tensors of any type, one launch for all pools of a cache (``csrc/pages.cu``; pages or rows that are
not dense take the plain forms).  Indexes given as Python lists or CPU tensors are checked before anything moves, and cannot be captured
into a graph with CUDA pools; in CUDA tensors, which the kernels never read back, what lies outside the pool or the table is skipped and
reported by ``ops.check_status``.  ``inference.PagedKVBlockManager`` builds fork, copy on write,
acceptance and compaction of the pool on them.  The reference's manager only hands blocks out and takes them back
(``cppmega_mlx/inference/serving.py:47-215``).
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _backend as B
from .window_attention import Plans, _raw_stream, entry, has_tangent, int32, meta, on_device

MAX_POOLS = 32          # of one launch
MAX_PAIRS = 65535
MAX_MOVES = 2048        # rows of one sequence in one call


_POOL = struct.Struct("Q4q")                     # cmb_page_pool
_plans = Plans()


def _pools(pools) -> tuple[torch.Tensor, ...]:
    return (pools,) if isinstance(pools, torch.Tensor) else tuple(pools)


def _check_pools(pools, rank: int, what: str) -> None:
    if not pools:
        raise ValueError(f"{what}: no pools")
    for p in pools:
        if p.dim() < rank or p.shape[0] != pools[0].shape[0] or p.device != pools[0].device:
            raise ValueError(f"{what}: pools have at least {rank} dimensions, one number of pages and one device")


def _check_grad(pools, what: str) -> None:
    if (torch.is_grad_enabled() and any(p.requires_grad for p in pools)) or has_tangent(*pools):
        raise ValueError(f"{what}: pools are written in place and cannot require a gradient")


def _dense(t: torch.Tensor, first: int) -> bool:
    """Whether the dimensions from ``first`` on are one dense piece of memory."""
    want = 1
    for n, s in zip(reversed(t.shape[first:]), reversed(t.stride()[first:])):
        if n != 1 and s != want:
            return False
        want *= n
    return True


def _indexes(x, what: str) -> torch.Tensor:
    t = x if isinstance(x, torch.Tensor) else torch.as_tensor(list(x), dtype=torch.int64)
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what} must be int32 / int64, got {t.dtype}")
    return t


def _plan_copy(pools, src, dst):
    """(whether the kernel serves the call, (page stride, bytes of a page) of every pool that has any)."""
    _check_pools(pools, 2, "copy_pages")
    if src.dim() != 1 or src.shape != dst.shape or src.device != dst.device:
        raise ValueError(f"copy_pages: src and dst are one list each, got {tuple(src.shape)} and {tuple(dst.shape)}")
    dev = pools[0].device
    if src.device.type != "cpu" and src.device != dev:
        raise ValueError(f"copy_pages: indexes on {src.device}, pools on {dev}")
    covered = dev.type == "cuda" and all(_dense(p, 1) for p in pools) and src.shape[0] <= MAX_PAIRS
    return covered, tuple((p.stride(0) * p.element_size(), 0, 0, (p.numel() // p.shape[0]) * p.element_size()) if p.numel() else None for p in pools)


def copy_pages_reference(pools, src, dst) -> torch.Tensor:
    """The plain form.  Pairs that the pool does not hold are left out; returns whether there were any (or pages written twice, or read and
    written)."""
    n = pools[0].shape[0]
    inside = (src >= 0) & (src < n) & (dst >= 0) & (dst < n)
    bad = (~inside & ((src != -1) | (dst != -1))).any()
    s, d = src[inside], dst[inside]
    for p in pools:
        p[d] = p[s]
    by_target = d.sort().values
    return bad | (by_target[1:] == by_target[:-1]).any() | torch.isin(s[s != d], d).any()


def copy_pages(pools, src, dst) -> None:
    """See the module docstring."""
    pools = _pools(pools)
    src, dst = _indexes(src, "copy_pages: src"), _indexes(dst, "copy_pages: dst")
    covered, shapes = _plans.get((*map(meta, pools), meta(src), meta(dst)), _plan_copy, pools, src, dst)
    _check_grad(pools, "copy_pages")
    dev, n = pools[0].device, pools[0].shape[0]
    if src.device.type == "cpu":
        used = [(s, d) for s, d in zip(src.tolist(), dst.tolist()) if (s, d) != (-1, -1)]
        for s, d in used:
            if not (0 <= s < n and 0 <= d < n):
                raise ValueError(f"copy_pages: page {s} to page {d} of {n}")
        to = [d for _, d in used]
        if len(set(to)) != len(to) or set(to) & {s for s, d in used if s != d}:
            raise ValueError("copy_pages: a page is written twice, or read and written")
        if not used:
            return
        # the lists that were checked, in memory of their own that is not pinned: it has been read when the upload's call returns, and
        # what the caller writes into its own then (pinned memory is read when the device comes to it) changes nothing
        src, dst = torch.tensor([[s for s, _ in used], to], dtype=torch.int32).to(dev, non_blocking=True)
    if src.shape[0] == 0 or n == 0:
        return
    if not covered or not B.kernels_enabled():
        bad = copy_pages_reference(pools, src.to(dev, torch.int64), dst.to(dev, torch.int64))
        if dev.type == "cuda":
            B.report(bad)
        return
    with on_device(dev):
        src, dst = int32(src), int32(dst)
        packed = [_POOL.pack(p.data_ptr(), *x) for p, x in zip(pools, shapes) if x is not None]
        fn = entry("cmb_copy_pages", ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p,
                   ctypes.c_void_p)
        for at in range(0, len(packed), MAX_POOLS):
            part = packed[at:at + MAX_POOLS]
            B.check(fn(b"".join(part), len(part), src.data_ptr(), dst.data_ptr(), src.shape[0], n, B.status_buffer(dev).data_ptr(),
                       _raw_stream(dev.index)), "copy_pages")


def compact_rows_reference(pools, table, start, path, counts) -> torch.Tensor:
    """The plain form.  Rows outside the table or the pool are left out; returns whether there were any (or counts outside the path)."""
    n, page, width, most = pools[0].shape[0], pools[0].shape[2], table.shape[1], path.shape[1]
    i = torch.arange(most, device=path.device)
    rows = counts.clamp(0, most)
    use = (i < rows[:, None]) & (path != i)
    bad = (rows != counts).any()
    if width == 0:
        return bad | use.any()
    to = start.long()[:, None] + i
    fro = start.long()[:, None] + path

    def pool_page(pos):        # and whether the table and the pool hold the position
        ids = table.long().gather(1, (pos // page).clamp(0, width - 1))
        return ids, (pos >= 0) & (pos < width * page) & (ids >= 0) & (ids < n)
    (to_page, to_held), (fro_page, fro_held) = pool_page(to), pool_page(fro)
    held = use & to_held & fro_held & (path >= 0)
    for p in pools:
        p[to_page[held], :, (to % page)[held]] = p[fro_page[held], :, (fro % page)[held]]
    return bad | (use & ~held).any()


def _plan_compact(pools, table, start, path, counts):
    """(whether the kernel serves the call, (strides, bytes of a row) of every pool, the entry's sizes)."""
    _check_pools(pools, 4, "compact_rows")
    dev = pools[0].device
    if any(p.shape[:3] != pools[0].shape[:3] for p in pools):
        raise ValueError("compact_rows: pools differ in pages, layers or page size")
    b = table.shape[0]
    if table.dim() != 2 or path.dim() != 2 or path.shape[0] != b or start.shape != (b,) or counts.shape != (b,):
        raise ValueError(f"compact_rows: table {tuple(table.shape)}, start {tuple(start.shape)}, path {tuple(path.shape)} and counts "
                         f"{tuple(counts.shape)} do not fit")
    if any(x.device != dev for x in (table, start, path, counts)):
        raise ValueError(f"compact_rows: indexes and pools are on one device ({dev})")
    if path.shape[1] > MAX_MOVES:
        raise ValueError(f"compact_rows: at most {MAX_MOVES} rows of a sequence, got {path.shape[1]}")
    n, layers, page = pools[0].shape[:3]
    covered = (dev.type == "cuda" and all(_dense(p, 3) for p in pools) and b <= 65535 and min(len(pools), MAX_POOLS) * layers <= 65535
               and table.shape[1] > 0)
    size = [p.element_size() for p in pools]
    shapes = tuple((p.stride(0) * e, p.stride(1) * e, p.stride(2) * e, p.numel() // max(1, n * layers * page) * e) for p, e in zip(pools, size))
    return covered, shapes, struct.pack("6i", b, table.shape[1], path.shape[1], page, n, layers)


def compact_rows(pools, table, start, path, counts) -> None:
    """See the module docstring.  table [B, W], start [B], path [B, P], counts [B], int32 / int64 on the pools' device."""
    pools = _pools(pools)
    table, start, path, counts = (_indexes(table, "compact_rows: table"), _indexes(start, "compact_rows: start"),
                                  _indexes(path, "compact_rows: path"), _indexes(counts, "compact_rows: counts"))
    covered, shapes, ip = _plans.get((*map(meta, pools), meta(table), meta(start), meta(path), meta(counts)), _plan_compact, pools, table, start,
                                     path, counts)
    _check_grad(pools, "compact_rows")
    dev = pools[0].device
    if path.shape[0] == 0 or path.shape[1] == 0 or any(p.numel() == 0 for p in pools):
        return
    n, page = pools[0].shape[0], pools[0].shape[2]
    if dev.type == "cpu":
        i = torch.arange(path.shape[1])
        use = i < counts[:, None]
        moves = use.any(1)                  # (a sequence that moves nothing may stand anywhere)
        far = torch.where(use, torch.maximum(path.long(), i), -1).amax(1) + start.long()
        if bool((counts < 0).any()) or bool((counts > path.shape[1]).any()) or bool((path[use] < 0).any()) or \
                bool((moves & ((start < 0) | (far >= table.shape[1] * page))).any()):
            raise ValueError("compact_rows: a row outside the table")
        need = torch.arange(table.shape[1]) * page <= far[:, None]
        need &= (torch.arange(table.shape[1]) + 1) * page > start[:, None]
        need &= moves[:, None]
        if bool(((table < 0) | (table >= n))[need].any()):
            raise ValueError(f"compact_rows: a page outside the pool of {n}")
    if not covered or not B.kernels_enabled():
        bad = compact_rows_reference(pools, table, start, path, counts)
        if dev.type == "cuda":
            B.report(bad)
        return
    with on_device(dev):
        table, start, path, counts = int32(table), int32(start), int32(path), int32(counts)
        packed = [_POOL.pack(p.data_ptr(), *x) for p, x in zip(pools, shapes)]
        fn = entry("cmb_compact_rows", ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                   ctypes.c_char_p, ctypes.c_void_p, ctypes.c_void_p)
        for at in range(0, len(packed), MAX_POOLS):
            part = packed[at:at + MAX_POOLS]
            B.check(fn(b"".join(part), len(part), table.data_ptr(), start.data_ptr(), path.data_ptr(), counts.data_ptr(), ip,
                       B.status_buffer(dev).data_ptr(), _raw_stream(dev.index)), "compact_rows")
