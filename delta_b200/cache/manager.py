"""The cache manager: pages of keys and values with a block table per request,
in groups, and slots of fixed-size state per request.

Reference counterparts: ``KVCache`` (one buffer [pages, 2, 16, heads, head_dim] per
layer, DELTA/Engine/DELTA/model.py:99-127), ``PageManager`` and
``Request.plan/initialize_pages`` (scheduler.py:8-40, 60-74), the slot block table
(backend.py:1835-1848) and the slot-indexed arrays ``cachelens`` and the selected
pages (backend.py:263, page_selector_v2.py:62-63).

What differs, on purpose:
  * Layers are sorted into groups by what they keep per token (the layout of a
    page, which the mixer declares, and the window or chunk).  A group has a pool and block tables of its own; all layers
    of a group share a request's page ids.  A group with a window or chunk gives pages back
    as soon as the window or chunk has passed them; the others when the request ends.
  * A request holds ceil(len / page_size) pages: no empty page in advance
    (the reference allocates one whenever the length reaches a page's end,
    scheduler.py:60-66).
  * Growing a request is all or nothing over the groups; ``OutOfPages`` leaves
    everything as it was, and the scheduler decides what happens then.
  * A request can be forked: the new ones hold the same whole pages (a page counts its holders) and a copy of
    the last one as far as it is filled, so nothing that is shared is ever written again.  The reference gives every
    request pages of its own and computes a prompt once for every sample of it.
  * What a page holds is the mixer's business: the manager allocates
    [layers of the group][page][*layout] from the layout the mixer declares.  The
    attention part keeps [K|V][kv head][offset][head_dim], so that the keys of one
    (page, head) are one contiguous tile.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..kernels import ops
from ..parts.base import PAGE, CacheSpec, StateSpec
from .page_pool import OutOfPages, PagePool


@dataclass
class LayerCacheView:
    """What a mixer gets for one run: its layer's pages and the block table of its group
    for the rows of this step."""
    pages: torch.Tensor         # [num_pages, *page layout]: the pages of this layer
    block_table: torch.Tensor   # [rows, max_pages] int32 (device), -1 where no page is held
    page_size: int
    writes: bool
    window: Optional[int]
    group: str
    state: Optional[dict] = None    # per-run state tensors of a mixer that declares some beside its pages


class CacheGroup:
    def __init__(self, name: str, spec: CacheSpec, cache_ids: List[int], num_pages: int, page_size: int,
                 max_slots: int, max_pages_per_request: int, dtype, device, shuffle_seed=None, page_runs=True):
        self.name, self.spec, self.cache_ids = name, spec, list(cache_ids)
        self.page_size = page_size
        self.pool = PagePool(num_pages, shuffle_seed, run_pages=max(1, spec.run_tokens // page_size) if page_runs else 1)
        self.index_of = {cid: i for i, cid in enumerate(self.cache_ids)}
        # one page more than the pool hands out: the spare page that the padding slot points at
        self.pages = torch.zeros((len(self.cache_ids), num_pages + 1, *spec.page_shape(page_size)), dtype=dtype, device=device)
        self.spare_page = num_pages
        # host block tables; -1 = no page.  first_page[slot]: pages below it were given back.
        # Row max_slots is the padding slot: one logical page, the spare one, for ever.
        self.table = np.full((max_slots + 1, max_pages_per_request), -1, dtype=np.int32)
        self.first_page = np.zeros(max_slots + 1, dtype=np.int64)
        self.num_logical = np.zeros(max_slots + 1, dtype=np.int64)  # logical pages ever reached
        self.table[max_slots, 0] = self.spare_page
        self.num_logical[max_slots] = 1

    def pages_needed(self, slot: int, new_len: int) -> int:
        want = (new_len + self.page_size - 1) // self.page_size
        return max(0, want - int(self.num_logical[slot]))

    def held(self, slot: int) -> List[int]:
        row = self.table[slot, int(self.first_page[slot]):int(self.num_logical[slot])]
        return [int(p) for p in row if p >= 0]


class CacheManager:
    """Owns every cache group and every state slot.  ``device`` may be "cpu" for tests of
    the bookkeeping; kernels only ever see CUDA tensors.

    Beside the ``max_slots`` slots that requests get there is one padding slot
    (``padding_slot``), which no request ever holds: it has a row in every block table
    with one page, a spare page outside the pool, and a row in every state.  A decode step
    captured for a rounded-up batch size points its spare rows at it (position 0), so that
    they read and write nothing that belongs to a request."""

    def __init__(self, cache_specs: Dict[int, CacheSpec], state_specs: Dict[str, StateSpec], *, max_slots: int,
                 max_seq_len: int, page_size: int, num_pages, dtype=torch.bfloat16, device="cuda", shuffle_seed=None,
                 page_runs: bool = True, states_follow_tokens: bool = True):
        """``states_follow_tokens``: a request's states belong to the tokens it holds now, so it can be forked at its present
        length only.  False: they are made anew in every step, and a fork at a shorter length starts with fresh ones."""
        self.max_slots, self.max_seq_len, self.page_size = int(max_slots), int(max_seq_len), int(page_size)
        self.max_pages_per_request = (self.max_seq_len + page_size - 1) // page_size
        self.device = device
        by_spec: Dict[CacheSpec, List[int]] = {}
        for cid, spec in sorted(cache_specs.items()):
            by_spec.setdefault(spec, []).append(cid)
        self.groups: Dict[str, CacheGroup] = {}
        self.group_of_cache: Dict[int, CacheGroup] = {}
        for spec, cids in by_spec.items():
            name = spec.describe()
            n = num_pages[name] if isinstance(num_pages, dict) else int(num_pages)
            g = CacheGroup(name, spec, cids, n, page_size, self.max_slots, self.max_pages_per_request, dtype, device, shuffle_seed,
                           page_runs)
            self.groups[name] = g
            for cid in cids:
                self.group_of_cache[cid] = g
        self.state_specs = dict(state_specs)
        self.states: Dict[str, torch.Tensor] = {
            k: torch.full((self.max_slots + 1, *s.shape), s.fill, dtype=s.dtype, device=device) for k, s in state_specs.items()}
        self.padding_slot = self.max_slots
        self.seq_len = np.zeros(self.max_slots, dtype=np.int64)
        self._free_slots = list(range(self.max_slots - 1, -1, -1))
        self._live = [False] * self.max_slots
        self.states_follow_tokens = bool(states_follow_tokens)
        self._shared: Dict[tuple, list] = {}      # (group, slots) -> what ``shared_prefixes`` found, until a holder comes or goes

    # ---- slots -------------------------------------------------------------
    @property
    def free_slots(self) -> int:
        return len(self._free_slots)

    def acquire_slot(self) -> int:
        """A free request slot with empty block tables and its state reset."""
        slot = self._take_slot()
        for k, s in self.state_specs.items():
            self.states[k][slot] = s.fill
        return slot

    def _take_slot(self) -> int:
        """A free slot with empty block tables; its state is what the last request left."""
        if not self._free_slots:
            raise RuntimeError("no free request slot")
        slot = self._free_slots.pop()
        self._shared.clear()
        self._live[slot] = True
        self.seq_len[slot] = 0
        for g in self.groups.values():
            g.table[slot].fill(-1)
            g.first_page[slot] = 0
            g.num_logical[slot] = 0
        return slot

    def release_slot(self, slot: int) -> None:
        """Gives back every page the request holds, and the slot."""
        if not self._live[slot]:
            raise ValueError(f"slot {slot} is released twice (or was never acquired)")
        self._shared.clear()
        for g in self.groups.values():
            g.pool.free(g.held(slot))
            g.table[slot].fill(-1)
            g.first_page[slot] = 0
            g.num_logical[slot] = 0
        self.seq_len[slot] = 0
        self._live[slot] = False
        self._free_slots.append(slot)

    def is_live(self, slot: int) -> bool:
        return self._live[slot]

    # ---- pages ---------------------------------------------------------------
    def pages_needed(self, slot: int, new_len: int) -> Dict[str, int]:
        return {n: g.pages_needed(slot, new_len) for n, g in self.groups.items()}

    def can_grow(self, slot: int, new_len: int, reserve: Optional[Dict[str, int]] = None) -> bool:
        """True when every group can give the pages that ``new_len`` tokens need, on top of
        ``reserve`` pages per group that are already spoken for in this step."""
        if new_len > self.max_seq_len:
            return False
        for n, g in self.groups.items():
            if g.pages_needed(slot, new_len) + (reserve or {}).get(n, 0) > g.pool.free_pages:
                return False
        return True

    def grow(self, slot: int, new_len: int) -> None:
        """Makes room for the request to hold ``new_len`` tokens.  All groups or none."""
        if not self._live[slot]:
            raise ValueError(f"slot {slot} is not live")
        if new_len > self.max_seq_len:
            raise OutOfPages(f"a request of {new_len} tokens is above the limit of {self.max_seq_len}")
        need = self.pages_needed(slot, new_len)
        for n, g in self.groups.items():
            if need[n] > g.pool.free_pages:
                raise OutOfPages(f"out of cache pages in group {n}: {need[n]} needed, {g.pool.free_pages} free")
        for n, g in self.groups.items():
            if need[n]:
                a = int(g.num_logical[slot])
                last = int(g.table[slot, a - 1]) if a > 0 else -1
                pages = g.pool.alloc(need[n], after=last if last >= 0 else None)
                g.table[slot, a:a + need[n]] = pages
                g.num_logical[slot] = a + need[n]

    def advance(self, slot: int, new_len: int) -> None:
        """Records that the request now holds ``new_len`` tokens, and gives back the pages
        that every later query's window or chunk has passed."""
        self.seq_len[slot] = new_len
        for g in self.groups.values():
            if not g.spec.reach:
                continue
            first_needed = g.spec.first_needed(new_len) // g.page_size
            a = int(g.first_page[slot])
            if first_needed > a:
                row = g.table[slot, a:first_needed]
                g.pool.free([int(p) for p in row if p >= 0])
                g.table[slot, a:first_needed] = -1
                g.first_page[slot] = first_needed

    # ---- requests that share their beginning -----------------------------------
    def can_fork(self, slot: int, length: int) -> bool:
        """Whether the request still holds what a fork at its first ``length`` tokens needs."""
        if not self._live[slot] or not 0 < length <= int(self.seq_len[slot]):
            return False
        if self.states and self.states_follow_tokens and length != int(self.seq_len[slot]):
            return False
        return all(not g.spec.reach or g.spec.first_needed(length) // g.page_size >= int(g.first_page[slot]) for g in self.groups.values())

    def fork(self, slot: int, length: Optional[int] = None, count: int = 1) -> List[int]:
        """``count`` new requests that hold the first ``length`` tokens of a live one (all of them when None), as slots: the whole pages
        are shared, the tokens of the last page and the states are copied, one launch for each (states that are made anew are filled).  The copies are enqueued on the
        current stream.  All or nothing: ``OutOfPages`` and a lack of slots leave everything as it was."""
        length = int(self.seq_len[slot]) if length is None else int(length)
        if not self.can_fork(slot, length):
            raise ValueError(f"slot {slot} cannot be forked at {length} tokens: it holds {int(self.seq_len[slot]) if self._live[slot] else 0}, and what a window "
                             "or a state has passed is gone")
        if count > self.free_slots:
            raise RuntimeError("no free request slot")
        whole, rest = divmod(length, self.page_size)
        for n, g in self.groups.items():
            if rest and count > g.pool.free_pages:
                raise OutOfPages(f"out of cache pages in group {n}: {count} needed for the forks' last pages, {g.pool.free_pages} free")
        present = length == int(self.seq_len[slot])
        new = [self._take_slot() for _ in range(count)]
        for g in self.groups.values():
            first = max(int(g.first_page[slot]), g.spec.first_needed(length) // g.page_size if g.spec.reach else 0)
            shared = g.table[slot, first:whole].tolist() if whole > first else []
            copies = []
            for s in new:
                g.table[s, first:whole] = shared
                g.first_page[s], g.num_logical[s] = first, whole + (1 if rest else 0)
                g.pool.share(shared)
                if rest:
                    page = g.pool.alloc(1, after=shared[-1] if shared else None)[0]
                    g.table[s, whole] = page
                    copies.append(page)
            if copies:
                self._copy_pages(g, [int(g.table[slot, whole])] * count, copies, [rest] * count)
        if self.states and present:
            self._copy_slots([slot] * count, new)
        elif self.states and new:
            at = torch.tensor(new, device=self.device)
            for k, s in self.state_specs.items():
                self.states[k].index_fill_(0, at, s.fill)
        for s in new:
            self.seq_len[s] = length
        return new

    def shared_prefixes(self, group: str, slots: Sequence[int]) -> List[Tuple[List[int], int]]:
        """[(places in ``slots``, pages)]: which of these requests hold the same first pages of a group, two or more to each entry.  Where
        some of them share more than all of them do, the way to divide them that saves the most reading is taken."""
        key = (group, tuple(slots))
        found = self._shared.get(key)
        if found is None:
            g = self.groups[group]
            table = g.table[list(slots)]
            n = g.num_logical[list(slots)]

            def divide(rows: np.ndarray, known: int):       # rows that agree on the first ``known`` pages -> (pages saved, entries)
                most = int(n[rows].min())
                same = (table[rows, known:most] == table[rows[0], known:most]).all(axis=0)
                k = known + (int(same.argmin()) if not same.all() else most - known)
                best = ((len(rows) - 1) * k, [(rows.tolist(), k)] if k else [])
                longer = rows[n[rows] > k]
                parts = [divide(longer[table[longer, k] == p], k + 1) for p in np.unique(table[longer, k]) if (table[longer, k] == p).sum() > 1 and p >= 0] if len(longer) > 1 else []
                apart = (sum(x for x, _ in parts), [e for _, es in parts for e in es])
                return apart if apart[0] > best[0] else best

            rows = np.array([i for i in range(len(slots)) if table[i, 0] >= 0 and g.pool.holders(int(table[i, 0])) > 1], dtype=np.int64)
            found = []
            for p in np.unique(table[rows, 0]) if len(rows) else []:
                mine = rows[table[rows, 0] == p]
                if len(mine) > 1:
                    found += divide(mine, 1)[1]
            if len(self._shared) >= 256:
                self._shared.clear()
            self._shared[key] = found
        return found

    def compact(self) -> Dict[str, int]:
        """Moves pages, in place, so that a request's pages follow one another in aligned runs again (see ``PagePool``), where serving has
        scattered them; requests that lie in runs stay where they are.  Tables, shared pages and free pages are booked anew; the copies are
        enqueued on the current stream, one launch for each group.  Returns how many pages moved, by group."""
        self._shared.clear()
        return {name: self._compact_group(g) for name, g in self.groups.items()}

    def _compact_group(self, g: CacheGroup) -> int:
        R, total = g.pool.run_pages, g.pool.num_pages
        if R == 1:
            return 0
        slots = [s for s in range(self.max_slots) if self._live[s]]
        held = {s: g.held(s) for s in slots}

        def broken(pages):      # steps from page to page that neither stay in a run nor begin the next one
            return sum(1 for a, b in zip(pages, pages[1:]) if b != a + 1 and not (a % R == R - 1 and b % R == 0))
        fixed = {p for s in slots if not broken(held[s]) for p in held[s]}
        movable, seen = [], set(fixed)
        for s in sorted(slots, key=lambda s: -len(held[s])):      # shared pages go with the longest request that holds them
            mine = [p for p in held[s] if p not in seen]
            seen.update(mine)
            if mine:
                movable.append(mine)
        runs = [r for r in range(total // R) if not any(q in fixed for q in range(r * R, r * R + R))]
        if sum(-(-len(m) // R) for m in movable) <= len(runs):
            places, at = [], 0
            for m in movable:
                places += [runs[at + i // R] * R + i % R for i in range(len(m))]
                at += -(-len(m) // R)
        else:
            places = [q for q in range(total) if q not in fixed]
        moved = {p: q for p, q in zip((p for m in movable for p in m), places) if p != q}
        if not moved:
            return 0
        g.pool.relocate(moved)          # (refuses, before anything is copied, what would overwrite a page that is held but stands in no table)
        self._copy_pages(g, list(moved), list(moved.values()), None)
        new_id = np.arange(total + 1, dtype=np.int32)
        new_id[list(moved)] = list(moved.values())
        for s in slots:
            row = g.table[s]
            row[row >= 0] = new_id[row[row >= 0]]
        return len(moved)

    def _copy_pages(self, g: CacheGroup, src, dst, tokens) -> None:
        axis = g.spec.layout.index(PAGE)
        if g.pages.is_cuda:
            ops.copy_pages(g.pages, src, dst, tokens=tokens, token_axis=axis)
        elif tokens is None:                    # the bookkeeping's tests
            g.pages[:, dst] = g.pages[:, src]
        else:
            for a, b, n in zip(src, dst, tokens):
                g.pages[:, b].narrow(axis + 1, 0, n).copy_(g.pages[:, a].narrow(axis + 1, 0, n))

    def _copy_slots(self, src, dst) -> None:
        if next(iter(self.states.values())).is_cuda:
            ops.copy_slots(self.states, src, dst)
        else:
            for s in self.states.values():
                s[dst] = s[src]

    # ---- views for a step ------------------------------------------------------
    def layer_pages(self, cache_id: int) -> torch.Tensor:
        g = self.group_of_cache[cache_id]
        return g.pages[g.index_of[cache_id]]

    def check(self) -> None:
        """Bookkeeping invariants: every held page belongs to live requests, as many as it has holders."""
        for g in self.groups.values():
            g.pool.check()
            seen: Dict[int, int] = {}
            for slot in range(self.max_slots):
                pages = g.held(slot)
                if pages and not self._live[slot]:
                    raise AssertionError(f"slot {slot} is free but holds pages in group {g.name}")
                if len(set(pages)) != len(pages):
                    raise AssertionError(f"slot {slot} holds a page of group {g.name} twice")
                for p in pages:
                    seen[p] = seen.get(p, 0) + 1
            for p, n in seen.items():
                if n != g.pool.holders(p):
                    raise AssertionError(f"page {p} of group {g.name} is held twice" if n > g.pool.holders(p) else f"page {p} of group {g.name} has lost a holder")
            if len(seen) != g.pool.held_pages:
                raise AssertionError(f"group {g.name}: {g.pool.held_pages} pages are out, requests hold {len(seen)}")

    def pages_in_use(self) -> Dict[str, int]:
        return {n: g.pool.held_pages for n, g in self.groups.items()}
