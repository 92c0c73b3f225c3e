"""Serving: paged KV block manager, continuous-batching scheduler, and paged decode attention.

``PagedKVBlockManager`` owns fixed-size blocks in two pools ``[num_blocks, layers, block_size, kv_heads, head_dim]``, hands them
out from a LIFO free list and keeps one block table per sequence.  ``ContinuousBatchScheduler`` admits waiting requests by
priority then arrival, groups by adapter key, and preempts the lowest-priority running request when blocks run out.  The
reference stops there (``cppmega_mlx/inference/serving.py:47-215`` manager, ``:265-489`` scheduler, ``:379`` adapter grouping,
``:472`` preemption, ``:492`` block table; ``:522`` raises because paged attention is not wired into the model).  Here
``paged_decode_attention`` / ``paged_tree_attention`` / ``paged_latent_decode_attention`` read keys straight through the block table,
so a decode step never materialises a contiguous copy of a sequence's cache.

Blocks are shared: ``fork`` gives a new sequence its parent's blocks, and a block is copied when a sequence is about to write into one
that others hold (``ops.copy_pages``, every layer's keys and values in one launch).  Drafted tokens are appended without advancing, verified
by ``paged_tree_attention``, and ``accept`` keeps one path of them (``ops.compact_rows``); ``release_window`` gives back what a sliding window
has passed, ``truncate`` what lies behind a length, and ``compact`` moves the blocks in use to the front of the pools.
"""
from __future__ import annotations

import heapq
import itertools
from dataclasses import dataclass, field

import torch

from ..ops.cached_attention import cached_attention
from ..ops.decode_attention import decode_attention
from ..ops.pages import MAX_MOVES, compact_rows, copy_pages


class OutOfBlocks(RuntimeError):
    pass


class PagedKVBlockManager:
    def __init__(self, *, num_blocks: int, num_layers: int, block_size: int, kv_heads: int, head_dim: int, v_head_dim: int | None = None,
                 dtype=torch.bfloat16, device=None):
        for n, v in (("num_blocks", num_blocks), ("num_layers", num_layers), ("block_size", block_size), ("kv_heads", kv_heads),
                     ("head_dim", head_dim)):
            if v <= 0:
                raise ValueError(f"{n} must be positive")
        self.num_blocks, self.num_layers, self.block_size = num_blocks, num_layers, block_size
        self.k_pool = torch.zeros(num_blocks, num_layers, block_size, kv_heads, head_dim, dtype=dtype, device=device)
        self.v_pool = torch.zeros(num_blocks, num_layers, block_size, kv_heads, v_head_dim or head_dim, dtype=dtype, device=device)
        self._free = list(range(num_blocks - 1, -1, -1))      # LIFO: pop() hands out block 0 first, freed blocks are reused first
        self._refs = [0] * num_blocks                          # sequences that hold each block
        self.tables: dict[int, list[int]] = {}                 # -1: a block that a window has passed (release_window)
        self.lengths: dict[int, int] = {}
        self._released: dict[int, tuple[int, int]] = {}        # (window, sink_tokens) of a sequence's latest release_window

    # -- accounting ------------------------------------------------------------------------------
    @property
    def num_free_blocks(self) -> int:
        return len(self._free)

    def blocks_needed(self, num_tokens: int) -> int:
        return -(-num_tokens // self.block_size)

    def can_allocate(self, num_tokens: int) -> bool:
        return self.blocks_needed(num_tokens) <= len(self._free)

    def allocate(self, seq_id: int, num_tokens: int) -> list[int]:
        if seq_id in self.tables:
            raise ValueError(f"sequence {seq_id} already has blocks")
        need = self.blocks_needed(num_tokens)
        if need > len(self._free):
            raise OutOfBlocks(f"need {need} blocks, {len(self._free)} free")
        self.tables[seq_id] = [self._take() for _ in range(need)]
        self.lengths[seq_id] = 0
        return self.tables[seq_id]

    def ensure_capacity(self, seq_id: int, total_tokens: int) -> None:
        tbl = self.tables[seq_id]
        need = self.blocks_needed(total_tokens) - len(tbl)
        if need > len(self._free):
            raise OutOfBlocks(f"need {need} more blocks, {len(self._free)} free")
        tbl.extend(self._take() for _ in range(max(0, need)))

    def free(self, seq_id: int) -> None:
        for b in reversed(self.tables.pop(seq_id)):
            self._drop(b)
        self.lengths.pop(seq_id, None)
        self._released.pop(seq_id, None)

    def _take(self) -> int:
        b = self._free.pop()
        self._refs[b] = 1
        return b

    def _drop(self, block: int) -> None:
        if block < 0:
            return
        self._refs[block] -= 1
        if self._refs[block] == 0:
            self._free.append(block)

    def fork(self, seq_id: int, new_id: int) -> list[int]:
        """``new_id`` continues from where ``seq_id`` is, on the same blocks (copied only when either writes into one)."""
        if new_id in self.tables:
            raise ValueError(f"sequence {new_id} already has blocks")
        self.tables[new_id] = list(self.tables[seq_id][:self.blocks_needed(self.lengths[seq_id])])
        self.lengths[new_id] = self.lengths[seq_id]
        if seq_id in self._released:
            self._released[new_id] = self._released[seq_id]
        for b in self.tables[new_id]:
            if b >= 0:
                self._refs[b] += 1
        return self.tables[new_id]

    def make_writable(self, seq_id: int, start: int, end: int) -> None:
        """Positions ``start .. end - 1`` of a sequence are about to be written: blocks that others hold too are copied first."""
        tbl = self.tables[seq_id]
        if not 0 <= start <= end <= len(tbl) * self.block_size:
            raise ValueError(f"positions {start} to {end} of a sequence with {len(tbl)} blocks of {self.block_size}")
        if start == end:
            return
        at = [i for i in range(start // self.block_size, (end - 1) // self.block_size + 1)]
        if any(tbl[i] < 0 for i in at):
            raise ValueError(f"sequence {seq_id}: positions {start} to {end} lie in blocks that its window has released")
        at = [i for i in at if self._refs[tbl[i]] > 1]
        if len(at) > len(self._free):
            raise OutOfBlocks(f"need {len(at)} blocks to copy, {len(self._free)} free")
        if at:
            src = [tbl[i] for i in at]
            for i in at:
                self._drop(tbl[i])
                tbl[i] = self._take()
            copy_pages((self.k_pool, self.v_pool), src, [tbl[i] for i in at])

    def truncate(self, seq_id: int, num_tokens: int) -> None:
        """Forget what a sequence holds behind its first ``num_tokens`` tokens; whole blocks behind them are freed.  Refused where the next
        token would see, or be written into, a block that ``release_window`` has given back."""
        if not 0 <= num_tokens <= self.lengths[seq_id]:
            raise ValueError(f"sequence {seq_id} has {self.lengths[seq_id]} tokens, cannot keep {num_tokens}")
        tbl = self.tables[seq_id]
        keep = self.blocks_needed(num_tokens)
        if num_tokens and seq_id in self._released:
            window, sink_tokens = self._released[seq_id]
            near = range(max(0, num_tokens - window + 1) // self.block_size, keep)
            if any(tbl[i] < 0 for i in (*range(min(keep, self.blocks_needed(sink_tokens))), *near)):
                raise ValueError(f"sequence {seq_id}: the window of {window} before token {num_tokens} lies in blocks that were released")
        for b in reversed(tbl[keep:]):
            self._drop(b)
        del tbl[keep:]
        self.lengths[seq_id] = num_tokens
        if not num_tokens:
            self._released.pop(seq_id, None)

    def release_window(self, seq_id: int, window: int, sink_tokens: int = 0) -> int:
        """Free the blocks that no later token sees under a sliding window with visible first tokens; how many."""
        if window < 1 or sink_tokens < 0:
            raise ValueError("window must be positive and sink_tokens non-negative")
        tbl, bs, n = self.tables[seq_id], self.block_size, 0
        first = self.lengths[seq_id] - window + 1               # the next token stands at position lengths[seq_id]
        for i in range(self.blocks_needed(sink_tokens), min(len(tbl), max(0, first) // bs)):
            if tbl[i] >= 0:
                self._drop(tbl[i])
                tbl[i] = -1
                n += 1
        self._released[seq_id] = (window, sink_tokens)
        return n

    def accept(self, paths: dict[int, list[int]]) -> None:
        """Drafted tokens were appended without advancing, token n of a sequence at position ``lengths + n``.  ``paths[seq]`` are the
        accepted ones, root first: they become the sequence's next tokens, the others are dropped.  One launch for all sequences."""
        for sid, path in paths.items():
            if list(path) != sorted(set(path)) or (path and (path[0] < 0 or path[-1] >= self._room(sid))):
                raise ValueError(f"sequence {sid}: path {path} must ascend within the {self._room(sid)} appended places")
            if len(path) > MAX_MOVES:
                raise ValueError(f"sequence {sid}: a path has at most {MAX_MOVES} tokens")
        moved = {sid: p for sid, p in paths.items() if list(p) != list(range(len(p)))}
        for sid, path in moved.items():
            self.make_writable(sid, self.lengths[sid], self.lengths[sid] + len(path))
        if moved:
            dev, most = self.k_pool.device, max(len(p) for p in moved.values())
            width = max(len(self.tables[s]) for s in moved)
            rows = [(self.tables[s] + [-1] * (width - len(self.tables[s])), [self.lengths[s]], list(p) + [0] * (most - len(p)), [len(p)])
                    for s, p in moved.items()]
            packed = torch.tensor([t + n + p + c for t, n, p, c in rows], dtype=torch.int32).to(dev)
            compact_rows((self.k_pool, self.v_pool), packed[:, :width], packed[:, width], packed[:, width + 1:width + 1 + most],
                         packed[:, -1])
        for sid, path in paths.items():
            self.lengths[sid] += len(path)
            tbl, keep = self.tables[sid], self.blocks_needed(self.lengths[sid])
            for b in reversed(tbl[keep:]):
                self._drop(b)
            del tbl[keep:]

    def _room(self, seq_id: int) -> int:
        return len(self.tables[seq_id]) * self.block_size - self.lengths[seq_id]

    def compact(self) -> dict[int, int]:
        """Move the blocks in use to the front of the pools; {old: new} of those that moved.  Block tables handed out before are stale."""
        used = [b for b, n in enumerate(self._refs) if n]
        holes = [b for b in range(len(used)) if not self._refs[b]]
        moved = dict(zip([b for b in used if b >= len(used)], holes))
        if moved:
            copy_pages((self.k_pool, self.v_pool), list(moved), list(moved.values()))
            for old, new in moved.items():
                self._refs[new], self._refs[old] = self._refs[old], 0
            for tbl in self.tables.values():
                tbl[:] = [moved.get(b, b) for b in tbl]
        self._free = list(range(self.num_blocks - 1, len(used) - 1, -1))
        return moved

    # -- data ------------------------------------------------------------------------------------
    def append(self, seq_id: int, layer: int, k: torch.Tensor, v: torch.Tensor, *, advance: bool = True) -> None:
        """k,v [S, kv_heads, dim] for one sequence; written at its current length (advance on the last layer only; drafted tokens
        never advance: ``accept`` does)."""
        pos = self.lengths[seq_id]
        s = k.shape[0]
        self.ensure_capacity(seq_id, pos + s)
        self.make_writable(seq_id, pos, pos + s)
        tbl = torch.tensor(self.tables[seq_id], device=k.device)
        p = pos + torch.arange(s, device=k.device)
        blk, off = tbl[p // self.block_size], p % self.block_size
        self.k_pool[blk, layer, off] = k.to(self.k_pool.dtype)
        self.v_pool[blk, layer, off] = v.to(self.v_pool.dtype)
        if advance:
            self.lengths[seq_id] = pos + s

    def gather(self, seq_id: int, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Contiguous [L, kv_heads, dim] copy of one sequence's cache (tests / fallbacks)."""
        n = self.lengths[seq_id]
        if any(b < 0 for b in self.tables[seq_id]):
            raise ValueError(f"sequence {seq_id} has released blocks")
        tbl = torch.tensor(self.tables[seq_id], device=self.k_pool.device)
        p = torch.arange(n, device=self.k_pool.device)
        blk, off = tbl[p // self.block_size], p % self.block_size
        return self.k_pool[blk, layer, off], self.v_pool[blk, layer, off]


def build_paged_block_table(manager: PagedKVBlockManager, seq_ids, *, pad: int = -1) -> tuple[torch.Tensor, torch.Tensor]:
    """([B, max_blocks] int32 table padded with ``pad``, [B] int32 lengths) for a batch of sequences."""
    rows = [manager.tables[s] for s in seq_ids]
    width = max((len(r) for r in rows), default=0)
    dev = manager.k_pool.device
    table = torch.full((len(rows), max(width, 1)), pad, dtype=torch.int32, device=dev)
    for i, r in enumerate(rows):
        if r:
            table[i, :len(r)] = torch.tensor(r, dtype=torch.int32, device=dev)
    lengths = torch.tensor([manager.lengths[s] for s in seq_ids], dtype=torch.int32, device=dev)
    return table, lengths


def paged_decode_attention(q: torch.Tensor, manager: PagedKVBlockManager, layer: int, block_table: torch.Tensor,
                           lengths: torch.Tensor, *, scale: float | None = None, window: int | None = None, sink_tokens: int = 0,
                           sinks: torch.Tensor | None = None) -> torch.Tensor:
    """One new query per sequence. q [B,H,D] → [B,H,Dv]; keys/values are read through ``block_table`` (GQA by head groups), ``lengths``
    count the query's own key.  CUDA tensors run the split-KV tcgen05 decode kernel (``ops/decode_attention.py``); nothing is gathered into
    a contiguous copy.  ``window`` / ``sink_tokens`` / ``sinks``: as in ``ops.cached_attention``, which then serves the step."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if window is not None or sinks is not None:
        return cached_attention(q[:, None], manager.k_pool[:, layer], manager.v_pool[:, layer], block_table, lengths - 1, window=window,
                                sink_tokens=sink_tokens, sinks=sinks, scale=scale)[:, 0]
    return decode_attention(q, manager.k_pool[:, layer], manager.v_pool[:, layer], block_table, lengths, scale=scale)


def paged_tree_attention(q: torch.Tensor, manager: PagedKVBlockManager, layer: int, block_table: torch.Tensor, lengths: torch.Tensor,
                         tree: torch.Tensor | None = None, *, scale: float | None = None, window: int | None = None, sink_tokens: int = 0,
                         sinks: torch.Tensor | None = None) -> torch.Tensor:
    """N drafted tokens per sequence, q [B,N,H,D] → [B,N,H,Dv].  Their keys and values have been appended without advancing, so they
    stand behind ``lengths`` (the manager's, without them); ``tree``: ``ops.tree_words`` of their parents, None for a chain."""
    return cached_attention(q, manager.k_pool[:, layer], manager.v_pool[:, layer], block_table, lengths, tree=tree, window=window,
                            sink_tokens=sink_tokens, sinks=sinks, scale=scale)


def paged_latent_decode_attention(q_lat: torch.Tensor, manager: PagedKVBlockManager, layer: int, block_table, lengths, *,
                                  d_v: int, scale: float, topk_idx: torch.Tensor | None = None) -> torch.Tensor:
    """MLA decode in latent form: q_lat [B,H,576]; pool rows hold the 576-wide latent in ``k_pool`` (kv_heads = 1); the value is
    the first ``d_v`` columns. ``topk_idx`` [B,K] (−1 padded) restricts attention to the indexer's selection."""
    return decode_attention(q_lat, manager.k_pool[:, layer], None, block_table, lengths, scale=scale, topk=topk_idx, d_v=d_v)


# ----------------------------------------------------------------------------------------------- scheduler
@dataclass
class Request:
    request_id: int
    prompt_len: int
    max_new_tokens: int
    priority: int = 0                 # larger runs first
    adapter_key: str | None = None
    arrival: int = 0
    generated: int = 0
    preemptions: int = 0

    @property
    def total_tokens(self) -> int:
        return self.prompt_len + self.generated

    @property
    def finished(self) -> bool:
        return self.generated >= self.max_new_tokens


@dataclass
class ScheduleStep:
    prefill: list[int] = field(default_factory=list)      # request ids admitted this step (need a prefill)
    decode: list[int] = field(default_factory=list)       # request ids decoding one token this step
    preempted: list[int] = field(default_factory=list)
    adapter_key: str | None = None


class ContinuousBatchScheduler:
    """Token-level continuous batching over a ``PagedKVBlockManager``."""

    def __init__(self, manager: PagedKVBlockManager, *, max_batch_size: int, policy: str = "priority"):
        if policy not in ("priority", "fifo"):
            raise ValueError("policy must be 'priority' or 'fifo'")
        if max_batch_size <= 0:
            raise ValueError("max_batch_size must be positive")
        self.manager, self.max_batch_size, self.policy = manager, max_batch_size, policy
        self._waiting: list[tuple] = []
        self._tick = itertools.count()
        self.requests: dict[int, Request] = {}
        self.running: list[int] = []
        self.finished: list[int] = []

    def _key(self, r: Request):
        return ((-r.priority) if self.policy == "priority" else 0, r.arrival, r.request_id)

    def add_request(self, request_id: int, prompt_len: int, max_new_tokens: int, *, priority: int = 0, adapter_key: str | None = None) -> Request:
        if request_id in self.requests:
            raise ValueError(f"duplicate request id {request_id}")
        if prompt_len <= 0 or max_new_tokens <= 0:
            raise ValueError("prompt_len and max_new_tokens must be positive")
        if self.manager.blocks_needed(prompt_len + max_new_tokens) > self.manager.num_blocks:
            raise ValueError("request can never fit in the block pool")
        r = Request(request_id, prompt_len, max_new_tokens, priority, adapter_key, next(self._tick))
        self.requests[request_id] = r
        heapq.heappush(self._waiting, (self._key(r), request_id))
        return r

    @property
    def num_waiting(self) -> int:
        return len(self._waiting)

    def _preempt_one(self, protect: set[int]) -> int | None:
        cands = [self.requests[i] for i in self.running if i not in protect]
        if not cands:
            return None
        victim = max(cands, key=lambda r: (-r.priority if self.policy == "priority" else 0, r.arrival))  # lowest priority, newest
        self.running.remove(victim.request_id)
        self.manager.free(victim.request_id)
        victim.preemptions += 1
        victim.prompt_len, victim.max_new_tokens = victim.total_tokens, victim.max_new_tokens - victim.generated   # recompute on resume
        victim.generated = 0
        heapq.heappush(self._waiting, (self._key(victim), victim.request_id))
        return victim.request_id

    def schedule(self) -> ScheduleStep:
        step = ScheduleStep()
        # the batch serves one adapter at a time: the running set's key, else the best waiting request's
        key = self.requests[self.running[0]].adapter_key if self.running else (
            self.requests[self._waiting[0][1]].adapter_key if self._waiting else None)
        step.adapter_key = key
        # 1. make room for every running request's next token
        for rid in list(self.running):
            if rid not in self.running:
                continue
            r = self.requests[rid]
            while True:
                try:
                    self.manager.ensure_capacity(rid, r.total_tokens + 1)
                    break
                except OutOfBlocks:
                    v = self._preempt_one(protect={rid})
                    if v is None:
                        raise
                    step.preempted.append(v)
        step.decode = list(self.running)
        # 2. admit waiting requests of the same adapter while slots and blocks last
        skipped = []
        while self._waiting and len(self.running) < self.max_batch_size:
            k, rid = heapq.heappop(self._waiting)
            r = self.requests[rid]
            if r.adapter_key != key or rid in step.preempted:
                skipped.append((k, rid))
                continue
            if not self.manager.can_allocate(r.prompt_len + 1):
                skipped.append((k, rid))
                break
            self.manager.allocate(rid, r.prompt_len + 1)
            self.running.append(rid)
            step.prefill.append(rid)
        for item in skipped:
            heapq.heappush(self._waiting, item)
        return step

    def complete_step(self, step: ScheduleStep, *, finished_ids=()) -> None:
        """Account one generated token for every request that ran; retire finished ones."""
        done = set(finished_ids)
        for rid in step.prefill + step.decode:
            if rid not in self.running:
                continue
            r = self.requests[rid]
            r.generated += 1
            if r.finished or rid in done:
                self.running.remove(rid)
                self.manager.free(rid)
                self.finished.append(rid)

    def idle(self) -> bool:
        return not self.running and not self._waiting
