"""The cache on the GPU: page tensors, block tables and state arrays, driven by `CacheBooks`.

Layout of a group's pages, per cache of the group: keys [num_pages, n_kv_heads, page_tokens,
k_dim] and values [num_pages, n_kv_heads, page_tokens, v_dim] in the compute type (the two widths
may differ, and a spec with v_dim 0 keeps the key tensor alone), so one (page, kv head) slab of
page_tokens * width elements is contiguous.  (The reference keeps a fixed region
per slot, [layer][kv head][position][head_dim]: src/cuda/engine.zig:234,393-401.)  The block
table of a group is int32 [max_requests, max_pages_per_request] on the device, a copy of the
host books' table; rows that changed are uploaded before a step runs.  A mixer with state of
fixed size gets an array [max_requests, *shape], zeroed when a request takes its slot.

A forked request shares the pages of the one that it was forked from and has a copy of its states; where one of them is about to
write a shared page, its rows are copied first (`sync_tables`).  All arrays of a group, and all states, are copied by one launch
each, and so are the rows of an accepted path moved (`keep`).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import numpy as np
import torch

from ..csrc import ops
from ..parts.base import KVCacheSpec, Precision, StateSpec
from .pages import CacheBooks


@dataclass
class LayerCache:
    """What one schedule entry's mixer is handed."""
    kind: str                                  # "pages" or "state"
    k_pages: Optional[torch.Tensor] = None
    v_pages: Optional[torch.Tensor] = None
    block_table: Optional[torch.Tensor] = None
    page_tokens: int = 0
    window: Optional[int] = None
    state: Optional[torch.Tensor] = None
    group: int = -1


class PagedCache:
    def __init__(self, cache_specs: Sequence[object], precision: Precision, page_tokens: int, num_pages: int,
                 max_requests: int, max_context: int):
        """`cache_specs`: per schedule entry, the list of specs of the caches its block keeps (a bare spec counts
        as a list of one; None or an empty list: the entry keeps none).  `layers[i]` is the list of `LayerCache`
        that entry's block is handed, in the order of its specs."""
        self.precision = precision
        self.page_tokens = page_tokens
        self.num_pages = num_pages
        entries: List[List[object]] = []
        for spec in cache_specs:
            if spec is None:
                entries.append([])
            elif isinstance(spec, (list, tuple)):
                entries.append([s for s in spec if s is not None])
            else:
                entries.append([spec])
        keys: List[tuple] = []
        for specs in entries:
            for spec in specs:
                if isinstance(spec, KVCacheSpec):
                    key = (spec.n_kv_heads, spec.k_dim, spec.v_dim, spec.window)
                    if key not in keys:
                        keys.append(key)
                elif not isinstance(spec, StateSpec):
                    raise TypeError(f"a cache spec of type {type(spec).__name__}; KVCacheSpec, StateSpec or None are known")
        self.books = CacheBooks([k[3] for k in keys], page_tokens, num_pages, max_requests, max_context)
        dev = precision.device
        self.tables = [torch.full((max_requests, self.books.max_pages_per_request), -1, dtype=torch.int32, device=dev)
                       for _ in keys]
        self.uploaded_bytes = 0
        self.layers: List[List[LayerCache]] = []
        self._states: List[torch.Tensor] = []
        for specs in entries:
            caches: List[LayerCache] = []
            for spec in specs:
                if isinstance(spec, KVCacheSpec):
                    gi = keys.index((spec.n_kv_heads, spec.k_dim, spec.v_dim, spec.window))
                    # zeros, not empty: a page that was never written must not hold NaN patterns
                    k = torch.zeros((num_pages, spec.n_kv_heads, page_tokens, spec.k_dim), dtype=precision.compute, device=dev)
                    v = None
                    if spec.v_dim > 0:
                        v = torch.zeros((num_pages, spec.n_kv_heads, page_tokens, spec.v_dim), dtype=precision.compute, device=dev)
                    caches.append(LayerCache("pages", k, v, self.tables[gi], page_tokens, spec.window, None, gi))
                else:
                    st = torch.zeros((max_requests, *spec.shape), dtype=spec.dtype, device=dev)
                    self._states.append(st)
                    caches.append(LayerCache("state", state=st))
            self.layers.append(caches)
        # what the kernels that copy blocks and move rows read, one record an array (see csrc/ops.py)
        self._page_tables: List[torch.Tensor] = []
        self._row_tables: List[torch.Tensor] = []
        self._page_arrays: List[List[torch.Tensor]] = [[] for _ in keys]
        for caches in self.layers:
            for lc in caches:
                if lc.kind == "pages":
                    self._page_arrays[lc.group] += [t for t in (lc.k_pages, lc.v_pages) if t is not None]
        for gi, arrays in enumerate(self._page_arrays):
            row = [t.shape[3] * t.element_size() for t in arrays]
            self._page_tables.append(torch.tensor([[t.data_ptr(), num_pages, t.shape[1], page_tokens * r, r] for t, r in zip(arrays, row)],
                                                  dtype=torch.int64, device=dev))
            self._row_tables.append(torch.tensor([[t.data_ptr(), t.shape[1], r, self.tables[gi].data_ptr()] for t, r in zip(arrays, row)],
                                                 dtype=torch.int64, device=dev))
        sizes = [st[0].numel() * st.element_size() for st in self._states]
        self._state_bytes = max(sizes, default=0)
        self._state_table = None
        if self._states and torch.device(dev).type == "cuda":
            self._state_table = torch.tensor([[st.data_ptr(), b] for st, b in zip(self._states, sizes)], dtype=torch.int64, device=dev)
            self._slot_table = torch.tensor([[st.data_ptr(), max_requests, 1, b, b] for st, b in zip(self._states, sizes)], dtype=torch.int64,
                                            device=dev)

    def has_state(self) -> bool:
        """Whether any mixer keeps a state of fixed size (which running a row twice would advance twice)."""
        return bool(self._states)

    # -- requests ----------------------------------------------------------------------------
    def open(self) -> int:
        slot = self.books.open()
        if self._state_table is not None:       # one launch for all states: of two, each a launch of its own, 7 us less on the host
            ops.zero_slot(self._state_table, slot, self._state_bytes)
        else:
            for st in self._states:
                st[slot].zero_()
        return slot

    def close(self, slot: int) -> None:
        self.books.close(slot)

    def fork(self, slots: Sequence[int]) -> List[int]:
        """A new slot for each of `slots`, with its tokens: pages shared, states copied."""
        new = []
        try:
            for s in slots:
                new.append(self.books.fork(int(s)))
        except Exception:
            for s in new:
                self.books.close(s)
            raise
        if self._states and new:
            if self._state_table is not None:
                moves = torch.tensor([[int(a), b, 1] for a, b in zip(slots, new)], dtype=torch.int32, device=self._slot_table.device)
                ops.copy_blocks(self._slot_table, moves, self._state_bytes)
            else:
                for st in self._states:
                    for a, b in zip(slots, new):
                        st[b].copy_(st[int(a)])
        return new

    def keep(self, paths: Sequence[tuple]) -> None:
        """Moves the accepted rows of drafted trees up in every cache of the model.  `paths`: (slot, the cache's row where the tree
        begins, the accepted rows of the tree in ascending order); the books' lengths stay the caller's business."""
        width = max((len(kept) for _, _, kept in paths), default=0)
        if not any(list(kept) != list(range(len(kept))) for _, _, kept in paths):
            return                              # every row is where it has to be
        rec = np.full((len(paths), 2 + width), -1, dtype=np.int32)
        for i, (slot, first, kept) in enumerate(paths):
            rec[i, :2] = slot, first
            rec[i, 2:2 + len(kept)] = kept
        dev = torch.from_numpy(rec).to(self.precision.device)
        self.uploaded_bytes += rec.nbytes
        for table, arrays, bt in zip(self._row_tables, self._page_arrays, self.tables):
            if arrays:
                ops.compact_rows(table, dev, bt.shape[0], bt.shape[1], self.page_tokens, max(t.shape[1] for t in arrays),
                                 max(t.shape[3] * t.element_size() for t in arrays), self.num_pages)

    def _copy_pages(self) -> None:
        """Makes the copies that the books owe.  One that reads or writes a page which an earlier one of them writes, or writes one which an
        earlier one reads, waits for a launch of its own."""
        owed = self.books.take_copies()
        for gi, arrays in enumerate(self._page_arrays):
            batch, busy_to, busy_from = [], set(), set()

            def launch():
                if not batch:
                    return
                if arrays[0].is_cuda:
                    moves = torch.tensor(batch, dtype=torch.int32, device=arrays[0].device)
                    ops.copy_blocks(self._page_tables[gi], moves, max(t[0].numel() * t.element_size() for t in arrays))
                else:
                    for a, b, rows in batch:
                        for t in arrays:
                            t[b, :, :rows].copy_(t[a, :, :rows])
                self.uploaded_bytes += 12 * len(batch)
                batch.clear(), busy_to.clear(), busy_from.clear()

            for a, b, rows in owed[owed[:, 0] == gi, 1:].tolist():
                if a in busy_to or b in busy_to or b in busy_from:
                    launch()
                batch.append((a, b, rows))
                busy_to.add(b), busy_from.add(a)
            launch()

    def sync_tables(self) -> None:
        """Makes the copies that the books owe and uploads the block-table rows that changed since the last call.  The copies read
        pageable host memory, so they are complete (staged) when the call returns and the
        books may change again at once."""
        if self.books.owes_copies():         # (8 us a step otherwise, for nothing in all steps without forks)
            self._copy_pages()
        if not self.books.dirty:
            return
        if len(self.books.dirty) > 4:            # many rows (a batch of beams): one upload, not one a row
            rows = sorted(self.books.dirty)
            for g, dev_table in zip(self.books.groups, self.tables):
                at = torch.tensor(rows, dtype=torch.int64, device=dev_table.device)
                dev_table.index_copy_(0, at, torch.from_numpy(g.table[rows]).to(dev_table.device))
                self.uploaded_bytes += (g.table.shape[1] * 4 + 8) * len(rows)
            self.books.dirty.clear()
            return
        for slot in sorted(self.books.dirty):
            for g, dev_table in zip(self.books.groups, self.tables):
                dev_table[slot].copy_(torch.from_numpy(g.table[slot].copy()))
                self.uploaded_bytes += g.table.shape[1] * 4
        self.books.dirty.clear()

    def bytes(self) -> int:
        n = 0
        for caches in self.layers:
            for lc in caches:
                for t in (lc.k_pages, lc.v_pages, lc.state):
                    if t is not None:
                        n += t.numel() * t.element_size()
        return n
