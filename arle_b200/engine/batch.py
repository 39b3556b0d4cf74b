"""One step's batch as the kernels see it.

A step is a list of entries ``(request, its next tokens, wanted places)``.  The
entries are laid end to end into T token rows; a decoded token is simply an entry
with one token.  All integer tables of the step are packed into ONE pinned host
array and copied to the device in one transfer, the way cklxx/arle uploads
positions / indptr / page indices per step (crates/cuda-kernels/src/tilelang.rs:424-612,
:703-818), but without separate code paths for decode, prefill and mixed batches.
With the cache manager's ``device_tables`` only tokens, slots, lengths and newly given pages
are copied, and a kernel (``ops.step_tables``) makes the tables from them.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch


@dataclass
class StepEntry:
    request: object                 # request id (any hashable)
    tokens: Sequence[int]           # its next tokens, in order
    want: Sequence[int] = ()        # indices into ``tokens`` whose logits are wanted


class Workspace:
    """Named scratch buffers that live across steps.  ``get`` returns a view of the
    wanted shape on a buffer that only ever grows, so steady-state steps allocate
    nothing."""

    def __init__(self, device):
        self.device = torch.device(device)
        self._bufs: Dict[Tuple[str, torch.dtype], torch.Tensor] = {}
        self._views: Dict[Tuple[str, torch.dtype], Tuple[Tuple[int, ...], torch.Tensor]] = {}     # the shape asked for last, and its view
        self._cuts: Dict[Tuple[str, torch.dtype], Dict[Tuple[int, int], torch.Tensor]] = {}                # columns of those views
        self.frozen = False
        self.generation = 0            # counts (re)allocations: addresses handed out earlier may be stale after one

    def get(self, name: str, shape: Tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
        key = (name, dtype)
        last = self._views.get(key)
        if last is not None and last[0] == shape:
            return last[1]
        n = 1
        for s in shape:
            n *= int(s)
        buf = self._bufs.get(key)
        if buf is None or buf.numel() < n:
            if self.frozen:
                raise RuntimeError(f"workspace buffer '{name}' would have to grow inside a captured graph")
            last = buf = None                       # or they would keep the smaller one
            buf = self._grown(torch.empty, key, n)
        view = buf[:n].view(shape)
        self._views[key] = (tuple(shape), view)
        self._cuts.pop(key, None)
        return view

    def get_zeroed(self, name: str, shape: Tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
        """Like ``get``, but the buffer is zero when it is first handed out (and after it
        had to grow).  For flags and counters that kernels leave at zero."""
        key = (name, dtype)
        last = self._views.get(key)
        if last is not None and last[0] == shape:
            return last[1]
        n = 1
        for s in shape:
            n *= int(s)
        buf = self._bufs.get(key)
        if buf is None or buf.numel() < n:
            if self.frozen:
                raise RuntimeError(f"workspace buffer '{name}' would have to grow inside a captured graph")
            last = buf = None                       # or they would keep the smaller one
            buf = self._grown(torch.zeros, key, n)
        view = buf[:n].view(shape)
        self._views[key] = (tuple(shape), view)
        self._cuts.pop(key, None)
        return view

    def _grown(self, make, key, n: int) -> torch.Tensor:
        """A larger buffer in the place of the one there was, which goes first: the device never has to hold both."""
        for kept in (self._bufs, self._views, self._cuts):
            kept.pop(key, None)
        self.generation += 1
        buf = self._bufs[key] = make(max(n, 1), dtype=key[1], device=self.device)
        return buf

    def cut(self, name: str, view: torch.Tensor, first: int, last: int) -> torch.Tensor:
        """``view[:, first: last]`` of a view that ``get`` handed out under this name.  Kept as long as the view is: making one costs the host as
        much as a launch."""
        key = (name, view.dtype)
        last_view = self._views.get(key)
        if last_view is None or last_view[1] is not view:
            return view[:, first: last]
        cuts = self._cuts.setdefault(key, {})
        piece = cuts.get((first, last))
        if piece is None:
            piece = cuts[(first, last)] = view[:, first: last]
        return piece

    def nbytes(self) -> int:
        return sum(b.numel() * b.element_size() for b in self._bufs.values())


@dataclass
class GroupTables:
    block_table: torch.Tensor       # int32 [R, width]
    slot_mapping: torch.Tensor      # int32 [T]


class TablesStatus:
    """What ``ops.step_tables`` says of a step (a word for each cache group), on its way to the host.  ``check()`` waits for the words alone, which are
    copied in front of the step's layers, and raises if a group's tables were not in order: that step ran as an empty one, its logits mean nothing.  The pinned
    words and the event are its context's, which reads them before it hands them to the next step."""

    def __init__(self, host: torch.Tensor, copied):
        self._host, self._copied, self._codes = host, copied, None

    def check(self) -> None:
        if self._codes is None:
            if self._copied is not None:
                self._copied.synchronize()
            self._codes = self._host.tolist()
        for gi, code in enumerate(self._codes):
            if code != 0:
                raise RuntimeError(f"the device's tables of cache group {gi} were not in order (status {code}, see ops.step_tables): the step ran without tokens and "
                                   "its results are invalid")


class StepContext:
    """Device-side description of one step, handed to every part.

    token_ids, positions, row_of_token, slot_of_token: int32 [T] (a negative token id
    stands for the token its request sampled last, kept on the device in ``last_token``).
    q_indptr: int32 [R+1] (row r owns token rows q_indptr[r] .. q_indptr[r+1]-1).
    kv_lens: int32 [R], tokens the request holds after this step.  state_slots: int32 [R].
    want_rows, want_slots: int32 [W] (token row and request slot of each wanted place).
    Host-side copies of what launch shapes depend on: q_lens, kv_lens_host,
    max_q_len, max_kv_len, decode_only."""

    def __init__(self, cache_manager, ws: Workspace):
        self.cache = cache_manager
        self.ws = ws
        self.device = ws.device
        self.num_tokens = 0
        self.num_rows = 0
        self.num_wanted = 0
        self.requests: List[object] = []
        self.q_lens: List[int] = []
        self.kv_lens_host: List[int] = []
        self.max_q_len = 0
        self.max_kv_len = 0
        self.decode_only = False
        self.num_single = 0
        self.table_width = 0
        self.token_ids = self.positions = self.row_of_token = None
        self.q_indptr = self.kv_lens = self.state_slots = self.want_rows = None
        self.slot_of_token = self.want_slots = None
        self.last_token: Optional[torch.Tensor] = None       # int32 [slots]: each request's last sampled token
        self.h2d_bytes = 0
        self.groups: List[GroupTables] = []
        self.memo: dict = {}                                 # what parts derive from a step once for all layers (cleared per step)
        self._pinned: Optional[torch.Tensor] = None
        self._dev: Optional[torch.Tensor] = None
        self._made: Optional[torch.Tensor] = None            # tables made on the device
        self.tables_status: Optional[TablesStatus] = None    # of this step, if they were
        self._status_host: Optional[torch.Tensor] = None     # pinned
        self._copied = torch.cuda.Event() if self.device.type == "cuda" else None

    # ------------------------------------------------------------------ build
    def build(self, entries: Sequence[StepEntry], starts: Sequence[int], table_width: Optional[int] = None) -> "StepContext":
        """``starts[i]`` is the number of tokens request i held before this step; the
        cache manager has already made room for the new ones.  ``table_width`` fixes
        the width of every block table (a captured graph needs the same layout at
        every replay); by default each is as wide as the longest request needs."""
        cm = self.cache
        self.memo.clear()
        R = len(entries)
        q_lens = [len(e.tokens) for e in entries]
        T = sum(q_lens)
        W = sum(len(e.want) for e in entries)
        self.num_tokens, self.num_rows, self.num_wanted = T, R, W
        self.requests = [e.request for e in entries]
        self.q_lens = q_lens
        self.kv_lens_host = [s + n for s, n in zip(starts, q_lens)]
        self.max_q_len = max(q_lens)
        self.max_kv_len = max(self.kv_lens_host)
        self.decode_only = self.max_q_len == 1
        self.num_single = sum(1 for n in q_lens if n == 1)
        n_groups = len(cm.groups)
        widths = []
        for gi, g in enumerate(cm.groups):
            need = max(1, max(-(-kv // g.page_size) for kv in self.kv_lens_host))
            if table_width is not None and need > table_width:
                raise ValueError(f"a request needs {need} pages, the fixed table width is {table_width}")
            widths.append(table_width if table_width is not None else need)
        self.table_width = max(widths) if widths else 0
        if cm.device_tables and n_groups:
            if self.tables_status is not None:
                self.tables_status.check()      # of the step before this one
            return self._build_on_device(entries, starts, widths)
        # layout of the packed int32 array
        sizes = [T, T, T, R + 1, R, R, max(W, 1), T, max(W, 1)]
        for gi in range(n_groups):
            sizes += [R * widths[gi], T]
        offs = np.concatenate([[0], np.cumsum([(s + 3) // 4 * 4 for s in sizes])])
        total = int(offs[-1])
        host = self._host_buffer(total)
        h = host.numpy()
        tok = h[offs[0]:offs[0] + T]
        pos = h[offs[1]:offs[1] + T]
        row = h[offs[2]:offs[2] + T]
        qi = h[offs[3]:offs[3] + R + 1]
        kvl = h[offs[4]:offs[4] + R]
        sts = h[offs[5]:offs[5] + R]
        want = h[offs[6]:offs[6] + W]
        slot_tok = h[offs[7]:offs[7] + T]
        want_slot = h[offs[8]:offs[8] + W]
        slots = np.fromiter((cm.slot(e.request) for e in entries), dtype=np.int64, count=R)
        starts_np = np.asarray(starts, dtype=np.int64)
        sts[:] = slots
        if self.max_q_len == 1 and W == R and all(tuple(e.want) == (0,) for e in entries):
            # every entry is one decoded token whose logits are wanted: no loops over requests
            tok[:] = [e.tokens[0] for e in entries]
            pos[:] = starts_np
            row[:] = np.arange(R)
            qi[:] = np.arange(R + 1)
            kvl[:] = starts_np + 1
            want[:] = np.arange(R)
            slot_tok[:] = slots
            want_slot[:] = slots
            for gi, g in enumerate(cm.groups):
                bt = h[offs[9 + 2 * gi]:offs[9 + 2 * gi] + R * widths[gi]].reshape(R, widths[gi])
                bt[:] = g.table[slots, :widths[gi]]
                pages = g.table[slots, starts_np // g.page_size].astype(np.int64)
                if (pages < 0).any():
                    raise RuntimeError(f"a token of this step has no page in cache group {gi}")
                h[offs[10 + 2 * gi]:offs[10 + 2 * gi] + T] = pages * g.page_size + starts_np % g.page_size
        else:
            at = 0
            wi = 0
            qi[0] = 0
            for r, (e, st, n) in enumerate(zip(entries, starts, q_lens)):
                tok[at:at + n] = np.asarray(e.tokens, dtype=np.int32)
                pos[at:at + n] = np.arange(st, st + n, dtype=np.int32)
                row[at:at + n] = r
                slot_tok[at:at + n] = slots[r]
                for w in e.want:
                    if not 0 <= w < n:
                        raise ValueError(f"request {e.request!r}: wanted place {w} is not among its {n} tokens")
                    want[wi] = at + w
                    want_slot[wi] = slots[r]
                    wi += 1
                at += n
                qi[r + 1] = at
                kvl[r] = st + n
            for gi in range(n_groups):
                bt = h[offs[9 + 2 * gi]:offs[9 + 2 * gi] + R * widths[gi]].reshape(R, widths[gi])
                bt[:] = cm.block_rows(gi, self.requests, widths[gi])
                sm = h[offs[10 + 2 * gi]:offs[10 + 2 * gi] + T]
                at = 0
                for e, st, n in zip(entries, starts, q_lens):
                    sm[at:at + n] = cm.slot_mapping(gi, e.request, st, n)
                    at += n
        dev = self._device_buffer(total)
        dev[:total].copy_(host[:total], non_blocking=True)
        if self._copied is not None:
            self._copied.record()
        self.h2d_bytes = total * 4
        d = dev
        self.token_ids = d[offs[0]:offs[0] + T]
        self.positions = d[offs[1]:offs[1] + T]
        self.row_of_token = d[offs[2]:offs[2] + T]
        self.q_indptr = d[offs[3]:offs[3] + R + 1]
        self.kv_lens = d[offs[4]:offs[4] + R]
        self.state_slots = d[offs[5]:offs[5] + R]
        self.want_rows = d[offs[6]:offs[6] + W]
        self.slot_of_token = d[offs[7]:offs[7] + T]
        self.want_slots = d[offs[8]:offs[8] + W]
        self.groups = []
        for gi in range(n_groups):
            bt = d[offs[9 + 2 * gi]:offs[9 + 2 * gi] + R * widths[gi]].view(R, widths[gi])
            sm = d[offs[10 + 2 * gi]:offs[10 + 2 * gi] + T]
            self.groups.append(GroupTables(bt, sm))
        return self

    def _build_on_device(self, entries, starts, widths) -> "StepContext":
        from .. import ops

        cm, T, R, W = self.cache, self.num_tokens, self.num_rows, self.num_wanted
        starts_np, lens = np.asarray(starts, dtype=np.int64), np.asarray(self.q_lens, dtype=np.int64)
        slots = np.fromiter((cm.slot(e.request) for e in entries), dtype=np.int64, count=R)
        # room for the pages that a step of these lengths may gain: what follows lies where it lay in a step of the same shape
        room = [int((-(-lens // g.page_size) + 1).sum()) for g in cm.groups]
        sizes = [T, max(W, 1), max(W, 1), R, R, R] + room
        offs = np.concatenate([[0], np.cumsum([(s + 3) // 4 * 4 for s in sizes])])
        host = self._host_buffer(int(offs[-1]))
        h = host.numpy()
        h[offs[0]:offs[0] + T] = np.concatenate([np.asarray(e.tokens, dtype=np.int32) for e in entries])
        firsts = np.cumsum(lens) - lens
        for e, n in zip(entries, self.q_lens):
            for w in e.want:
                if not 0 <= w < n:
                    raise ValueError(f"request {e.request!r}: wanted place {w} is not among its {n} tokens")
        counts = [len(e.want) for e in entries]
        if W:
            h[offs[1]:offs[1] + W] = np.repeat(firsts, counts) + np.concatenate([np.asarray(e.want, dtype=np.int64) for e in entries if len(e.want)])
            h[offs[2]:offs[2] + W] = np.repeat(slots, counts)
        h[offs[3]:offs[3] + R] = slots
        h[offs[4]:offs[4] + R] = starts_np
        h[offs[5]:offs[5] + R] = lens
        gained, listed = [], []
        for gi, g in enumerate(cm.groups):
            ps = g.page_size
            held, pages = -(-starts_np // ps), -(-(starts_np + lens) // ps)
            # room that was made without a step: the kernel reads the device's table up to the tokens in front of this one
            for r in np.nonzero(g.num_listed[slots] < held)[0]:
                first, late = int(g.num_listed[slots[r]]), g.table[slots[r], :held[r]]
                g.device_table[int(slots[r]), first:int(held[r])].copy_(torch.from_numpy(late[first:].copy()))
            listed.append(pages)
            more = np.nonzero(pages > held)[0]
            new = np.concatenate([g.table[slots[r], held[r]:pages[r]] for r in more]) if more.size else np.zeros(0, dtype=np.int32)
            if (new < 0).any():
                raise RuntimeError(f"a token of this step has no page in cache group {gi}")
            h[offs[6 + gi]:offs[6 + gi] + new.size] = new
            gained.append(int(new.size))
        last = len(cm.groups) - 1
        total = int(offs[6 + last]) + gained[last]
        dev = self._device_buffer(int(offs[-1]))
        dev[:total].copy_(host[:total], non_blocking=True)
        self.h2d_bytes = total * 4
        cut = lambda k, n: dev[offs[k]:offs[k] + n]      # noqa: E731
        self.token_ids, self.want_rows, self.want_slots, self.state_slots = cut(0, T), cut(1, W), cut(2, W), cut(3, R)
        made = [T, T, T, R + 1, R, len(cm.groups)] + [x for w in widths for x in (R * w, T)]
        at = np.concatenate([[0], np.cumsum([(s + 3) // 4 * 4 for s in made])])
        if self._made is None or self._made.numel() < at[-1]:
            self._made = torch.zeros(max(int(at[-1]), 4096), dtype=torch.int32, device=self.device)
        piece = lambda k: self._made[at[k]:at[k] + made[k]]      # noqa: E731
        self.positions, self.row_of_token, self.slot_of_token, self.q_indptr, self.kv_lens = (piece(k) for k in range(5))
        self.groups, status = [], piece(5)
        if self._status_host is None:
            self._status_host = torch.empty(len(cm.groups), dtype=torch.int32, pin_memory=self._copied is not None)
        try:
            for gi, g in enumerate(cm.groups):
                bt, sm = piece(6 + 2 * gi).view(R, widths[gi]), piece(7 + 2 * gi)
                ops.step_tables(self.state_slots, cut(4, R), cut(5, R), cut(6 + gi, gained[gi]), g.device_table, g.pool.num_pages, g.page_size, self.q_indptr, self.kv_lens,
                                self.positions, self.row_of_token, self.slot_of_token, sm, bt, status[gi: gi + 1])
                g.num_listed[slots] = listed[gi]
                self.groups.append(GroupTables(bt, sm))
            self._status_host.copy_(status, non_blocking=True)
        finally:
            if self._copied is not None:
                self._copied.record()           # one event for the copy to the device and the one from it
        self.tables_status = TablesStatus(self._status_host, self._copied)
        return self

    def _host_buffer(self, n: int) -> torch.Tensor:
        if self._copied is not None:
            self._copied.synchronize()      # the last step's copy has read the pinned array
        if self._pinned is None or self._pinned.numel() < n:
            cap = max(n, 4096)
            self._pinned = torch.empty(cap, dtype=torch.int32, pin_memory=self.device.type == "cuda")
        return self._pinned

    def _device_buffer(self, n: int) -> torch.Tensor:
        if self._dev is None or self._dev.numel() < n:
            self._dev = torch.empty(max(n, 4096), dtype=torch.int32, device=self.device)
        return self._dev

    # ------------------------------------------------------------------ views
    def cache_view(self, cache_layer: int, writable: bool = True):
        gi = self.cache.group_of_layer(cache_layer)
        t = self.groups[gi]
        return self.cache.layer_view(cache_layer, t.block_table, t.slot_mapping, writable)

    def state_view(self, state_index: int) -> torch.Tensor:
        return self.cache.states[state_index]
