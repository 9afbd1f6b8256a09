"""The cache manager: pages of keys and values, block tables, and state slots.

Storage
-------
Every schedule entry that owns a cache says, as a `KVSpec`, what it stores per
position: a list of rows `(heads, width)` (an attention mixer's keys and values are two
equal rows; a latent cache is one), a window, and how many positions share a stored row.
Entries whose specs are equal form a *group*; a group has its own pool of pages and, per
request, its own block table. One tensor per group holds its pages: page `p` of entry
`e` is `tensor[e, p]`, laid out row after row, each row `[heads, page_size, width]`; a
group of equal rows is shaped `[entries, pages, rows, heads, page_size, width]` (keys at
index 0 and values at index 1 of the rows' axis for attention), any other
`[entries, pages, elements per page]`. A request's logical page `i` holds stored rows
`i * page_size` to `(i + 1) * page_size - 1` and maps to the same physical page number
in every entry of the group. Groups may differ in how many pages a request needs of
them (`KVSpec.stride`), so every count below is per group.

A group with a window gives a page back as soon as every position in it is behind
the window of all tokens still to come; its block-table entry becomes -1. So does a group
whose queries read only their own run of positions (`KVSpec.chunk`), once the latest
position has left a page's run behind. Pages that hold
one of the first `keep_first` positions of such a group are kept until the request ends. All pages
return when the request ends. Freed pages are handed out again, last freed first.

A request may be *forked* (`CacheManager.fork`): the new one holds the first positions of the old
one. Whole pages of these are then in both requests' block tables (the pool counts the references, a page
is free again once the last is given back; nobody writes to a page that is in two tables, since
positions only grow), the rows in the page that they end in are copied to a page of its own, and so is
per-request state. Which requests share what (`SharedRun`) is kept with them, so that a step of
single tokens can read shared positions once for all of them. `CacheManager.resize` gives the pools another
number of pages while requests live: what is held moves to the front of the new ones.

Beside the pages there are *state slots*: a request holds one slot number for its
whole life, and every entry that declares a `StateSpec` has a tensor
`[slots + 1, *shape]` indexed by it (an entry that declares several by name has one
each, and so has a block that declares state of its own); the last row is a scratch slot that belongs to no
request (the padding rows of a captured step point at it). A slot is set to the mixer's
initial state when a request's first step runs. Muse-Glimmer declares no state; the
slots exist so a mixer with state of its own needs no change here.

The reference keeps one growing buffer per request and layer instead
(src/mlx_omnia/engine/core/cache/kv.py:18-128) and says which rows a window makes
unreadable through `Rows.keep` (src/mlx_omnia/engine/core/cache/layout.py:14-24);
paging, groups and slots are this engine's own design.

All bookkeeping is host-side Python and runs without a GPU (`device="meta"` or
`allocate=False` skips the tensors).
"""

from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

from mlx_omnia_b200.parts.base import KVSpec
from mlx_omnia_b200.parts.model import CacheNeed


class CacheError(RuntimeError):
    """Misuse of the cache manager: a page freed twice, an unknown request, ..."""


class PagePool:
    """Page numbers 0..count-1, each held so many times; a stack of free ones (last freed, first reused)."""

    def __init__(self, count: int) -> None:
        self.count = count
        self._free = list(range(count - 1, -1, -1))
        self._held = [0] * count

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self) -> int:
        if not self._free:
            raise CacheError("no free page")
        page = self._free.pop()
        self._held[page] = 1
        return page

    def share(self, page: int) -> None:
        """Hold a page once more; it is free after as many `give`s."""
        if not 0 <= page < self.count or not self._held[page]:
            raise CacheError(f"page {page} is not held and cannot be shared")
        self._held[page] += 1

    def give(self, page: int) -> None:
        if not 0 <= page < self.count:
            raise CacheError(f"page {page} is not in a pool of {self.count}")
        if not self._held[page]:
            raise CacheError(f"page {page} is freed twice")
        self._held[page] -= 1
        if not self._held[page]:
            self._free.append(page)

    def held(self) -> list[int]:
        return [p for p, h in enumerate(self._held) if h]

    def references(self, page: int) -> int:
        return self._held[page]

    def resized(self, count: int) -> "tuple[PagePool, dict[int, int]]":
        """A pool of `count` pages that holds what this one does, from page 0 on, and where each held page went."""
        to = {page: i for i, page in enumerate(self.held())}
        if len(to) > count:
            raise CacheError(f"{len(to)} pages are held, which a pool of {count} does not take")
        pool = PagePool(count)
        for page in to:
            pool._held[pool.take()] = self._held[page]
        return pool, to


@dataclass
class Group:
    spec: KVSpec
    entries: list[int]  # schedule entries stored in this group, in tensor order
    pool: PagePool
    pages: torch.Tensor | None  # [entries, pages, rows, heads, page_size, width] or [entries, pages, elements]


@dataclass(eq=False, frozen=True)
class SharedRun:
    """The first `positions` positions that forks of one request hold alike; requests of one run carry the same object."""

    positions: int


@dataclass
class RequestCache:
    """What one live request holds."""

    request_id: str
    tokens: int = 0  # positions written so far
    tables: list[list[int]] = field(default_factory=list)  # per group: physical page per logical page (-1 freed)
    slot: int = -1
    fresh: bool = True  # no step has run for it yet
    # int32 copies of `tables` (capacity grown by doubling; entries beyond len(tables[g]) are -1),
    # so that a step lays its block tables out with array copies instead of Python loops
    arrays: list[np.ndarray] = field(default_factory=list)
    runs: list[SharedRun] = field(default_factory=list)  # what it shares with others, shortest first

    def table_array(self, group: int) -> np.ndarray:
        return self.arrays[group][: len(self.tables[group])]


class CacheManager:
    def __init__(self, needs: list[CacheNeed], *, page_size: int, pages_per_group: int | dict[KVSpec, int],
                 max_requests: int, dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cpu",
                 allocate: bool = True, model_state: "dict | None" = None) -> None:
        if page_size < 1:
            raise ValueError("page_size must be at least 1")
        self.page_size = page_size
        self.needs = needs
        self.groups: list[Group] = []
        self.group_of_entry: dict[int, tuple[int, int]] = {}  # entry -> (group, index in group)
        by_spec: dict[KVSpec, int] = {}
        for entry, need in enumerate(needs):
            if need.kv is None:
                continue
            g = by_spec.get(need.kv)
            if g is None:
                g = by_spec[need.kv] = len(self.groups)
                count = pages_per_group[need.kv] if isinstance(pages_per_group, dict) else pages_per_group
                self.groups.append(Group(need.kv, [], PagePool(count), None))
            self.group_of_entry[entry] = (g, len(self.groups[g].entries))
            self.groups[g].entries.append(entry)
        for entry, need in enumerate(needs):
            if need.reads is not None:
                if need.reads not in self.group_of_entry:
                    raise ValueError(f"schedule entry {entry} reads entry {need.reads}, which keeps no pages")
                self.group_of_entry[entry] = self.group_of_entry[need.reads]
        if allocate:
            for group in self.groups:
                s = group.spec
                shape = (len(s.rows), *s.rows[0][:1], page_size, s.rows[0][1]) if s.uniform else \
                    (s.elements_per_position * page_size,)
                group.pages = torch.zeros(len(group.entries), group.pool.count, *shape, dtype=dtype, device=device)
        self.slots = PagePool(max_requests)
        self.scratch_slot = max_requests  # the state row that padding rows of a captured step point at
        self.state: dict[int, torch.Tensor | dict[str, torch.Tensor]] = {}  # a mixer's: one tensor, or by name
        self.block_state: dict[int, dict[str, torch.Tensor]] = {}  # a block's own, by name
        self.initial_state: dict[int, torch.Tensor] = {}  # entries whose state does not start as zeros

        def slots_of(spec):
            return torch.zeros(max_requests + 1, *spec.shape, dtype=spec.dtype, device=device)

        for entry, need in enumerate(needs):
            if not allocate:
                continue
            if isinstance(need.state, dict):
                self.state[entry] = {name: slots_of(spec) for name, spec in need.state.items()}
            elif need.state is not None:
                self.state[entry] = slots_of(need.state)
                if need.initial_state is not None:
                    start = need.initial_state.to(need.state.dtype).to(device)  # whatever can be written to a slot
                    self.initial_state[entry] = start.expand(1, *need.state.shape)[0].contiguous()
            if getattr(need, "block_state", None):
                self.block_state[entry] = {name: slots_of(spec) for name, spec in need.block_state.items()}
        self.has_state = bool(model_state) or any(need.state is not None or getattr(need, "block_state", None) for need in needs)
        # State that belongs to the model and to no schedule entry (an embedding that looks at the token before).
        self.model_state: dict[str, torch.Tensor] = \
            {name: slots_of(spec) for name, spec in (model_state or {}).items()} if allocate else {}
        self.requests: dict[str, RequestCache] = {}

    def state_tensors(self) -> list[tuple[torch.Tensor, torch.Tensor | None]]:
        """Every tensor indexed by state slots, with what a slot starts as (None: zeros)."""
        held: list[tuple[torch.Tensor, torch.Tensor | None]] = [(t, None) for t in self.model_state.values()]
        for entry in sorted(set(self.state) | set(self.block_state)):
            own = self.state.get(entry)
            if isinstance(own, dict):
                held += [(t, None) for t in own.values()]
            elif own is not None:
                held.append((own, self.initial_state.get(entry)))
            held += [(t, None) for t in self.block_state.get(entry, {}).values()]
        return held

    def reset_slots(self, slots: list[int]) -> None:
        """Set the state of `slots` (of requests about to run their first step) to its start:
        the mixer's `initial_state()` where it gave one, zeros everywhere else."""
        if not slots or not (self.state or self.block_state or self.model_state):
            return
        held = self.state_tensors()
        if held and held[0][0].is_cuda:
            from mlx_omnia_b200.kernels import ops

            ops.fill_slots(held, slots)
            return
        index = torch.as_tensor(slots)
        for tensor, initial in held:
            if initial is None:
                tensor.index_fill_(0, index, 0)
            else:
                tensor[index] = initial

    # -- sizes -----------------------------------------------------------------------
    @staticmethod
    def bytes_per_token(needs: list[CacheNeed], element_size: int) -> int:
        """Cache bytes one position costs over all entries that own pages (what a pool is
        sized by when the caller names no size)."""
        return sum(-(-need.kv.elements_per_position // need.kv.stride) * element_size
                   for need in needs if need.kv is not None)

    def bytes_per_page(self, group: int, element_size: int) -> int:
        g = self.groups[group]
        return len(g.entries) * g.spec.elements_per_position * self.page_size * element_size

    def pages_for(self, group: int, tokens: int) -> int:
        """Pages of `group` that a request of `tokens` positions occupies (none given back)."""
        return -(-self.groups[group].spec.stored(tokens) // self.page_size)

    def pages_needed(self, request: RequestCache, new_tokens: int) -> list[int]:
        """Pages each group must take for `request` to grow by `new_tokens`."""
        return [self.pages_for(g, request.tokens + new_tokens) - self.pages_for(g, request.tokens)
                for g in range(len(self.groups))]

    def capacity_tokens(self) -> int:
        """The longest request the pools can hold (the tightest group decides)."""
        return min((g.pool.count * self.page_size * g.spec.stride for g in self.groups), default=1 << 30)

    def can_grow(self, request: RequestCache, new_tokens: int, reserve: list[int] | None = None) -> bool:
        need = self.pages_needed(request, new_tokens)
        return all(n <= g.pool.free - (reserve[i] if reserve else 0)
                   for i, (n, g) in enumerate(zip(need, self.groups)))

    # -- life of a request -------------------------------------------------------------
    def open(self, request_id: str) -> RequestCache:
        if request_id in self.requests:
            raise CacheError(f"request {request_id!r} is already open")
        if self.slots.free == 0:
            raise CacheError("no free request slot")
        request = RequestCache(request_id, tables=[[] for _ in self.groups], slot=self.slots.take(),
                               arrays=[np.full(16, -1, dtype=np.int32) for _ in self.groups])
        self.requests[request_id] = request
        return request

    def grow(self, request: RequestCache, new_tokens: int) -> None:
        """Take the pages for the next `new_tokens` positions in every group, or none
        at all (CacheError) when some group has too few free pages."""
        if new_tokens < 0:
            raise ValueError("new_tokens must not be negative")
        need = self.pages_needed(request, new_tokens)
        for n, group in zip(need, self.groups):
            if n > group.pool.free:
                raise CacheError(f"group {group.spec} needs {n} pages, {group.pool.free} free")
        for g, (n, group, table) in enumerate(zip(need, self.groups, request.tables)):
            if len(table) + n > len(request.arrays[g]):
                grown = np.full(max(2 * len(request.arrays[g]), len(table) + n), -1, dtype=np.int32)
                grown[: len(table)] = request.arrays[g][: len(table)]
                request.arrays[g] = grown
            for _ in range(n):
                request.arrays[g][len(table)] = page = group.pool.take()
                table.append(page)
        request.tokens += new_tokens

    # -- forks -------------------------------------------------------------------------
    def fork_pages(self, positions: int) -> list[int]:
        """Pages each group takes for a fork at `positions`: the one that these end in, where they do not fill it."""
        return [int(g.spec.stored(positions) > self._whole_pages(i, positions) * self.page_size) for i, g in enumerate(self.groups)]

    def _whole_pages(self, group: int, positions: int) -> int:
        """Pages of `group` that `positions` positions fill: no later position is written to them."""
        return positions // self.groups[group].spec.stride // self.page_size

    def why_not_fork(self, request: RequestCache, positions: int) -> str | None:
        """Why `request` cannot be forked at `positions` (None: it can; pages and slots may still be short)."""
        if not 1 <= positions <= request.tokens:
            return f"a fork takes between 1 and the {request.tokens} positions that request {request.request_id!r} holds, not {positions}"
        # (The page that they end in is the fork's to write on, so its first rows have to be there. None is given back while it can be written to.)
        if any(n and table[self._whole_pages(g, positions)] < 0
               for g, (n, table) in enumerate(zip(self.fork_pages(positions), request.tables))):
            return f"the page that position {positions - 1} of request {request.request_id!r} lies in was given back"
        if request.tokens == positions:
            return None
        if self.has_state:
            return f"the state of request {request.request_id!r} is that of {request.tokens} positions, not of {positions}"
        for g, (group, table) in enumerate(zip(self.groups, request.tables)):
            spec = group.spec
            if positions % spec.stride:
                return f"a stored row of {spec.stride} positions has gone on past position {positions}"
            dead = max(spec.dead_below(positions), 0) // spec.stride // self.page_size if spec.forgets else 0
            kept = -(-spec.stored(spec.keep_first) // self.page_size) if spec.keep_first else 0
            if any(page < 0 and (i < kept or i >= dead) for i, page in enumerate(table[: self.pages_for(g, positions)])):
                return f"positions that a request of {positions} reads were given back"
        return None

    def fork(self, request: RequestCache, request_id: str, positions: int | None = None) -> RequestCache:
        """Open `request_id` with the first `positions` positions of `request` (None: all of them) as its own. Whole pages are
        shared, the rest and the state are copied (on the current stream). Nothing is taken when it cannot be done (CacheError), or when a
        copy fails."""
        positions = request.tokens if positions is None else positions
        why = self.why_not_fork(request, positions)
        if why is not None:
            raise CacheError(why)
        need = self.fork_pages(positions)
        for n, group in zip(need, self.groups):
            if n > group.pool.free:
                raise CacheError(f"group {group.spec} needs {n} pages, {group.pool.free} free")
        new = self.open(request_id)
        try:
            self._take_over(request, new, positions, need)
        except BaseException:
            self.close(request_id)  # what it had taken by then
            raise
        run = next((r for r in request.runs if r.positions == positions), None)
        if run is None:
            run = SharedRun(positions)
            request.runs = sorted([*request.runs, run], key=lambda r: r.positions)
        new.runs = [r for r in request.runs if r.positions <= positions]
        return new

    def _take_over(self, request: RequestCache, new: RequestCache, positions: int, need: list[int]) -> None:
        """Pages, rows and state of a fork. (Its table names a page as soon as it is held, so that closing it gives all of them back.)"""
        new.tokens, new.fresh = positions, request.fresh
        for g, (n, group, table) in enumerate(zip(need, self.groups, request.tables)):
            whole, mine = self._whole_pages(g, positions), new.tables[g]
            for page in table[:whole]:
                if page >= 0:
                    group.pool.share(page)
                mine.append(page)
            if n:
                mine.append(group.pool.take())
                if group.pages is not None:
                    self._copy_rows(group, table[whole], mine[-1], group.spec.stored(positions) - whole * self.page_size)
            if len(mine) > len(new.arrays[g]):
                new.arrays[g] = np.full(2 * len(mine), -1, dtype=np.int32)
            new.arrays[g][: len(mine)] = mine
        tensors = [t for t, _ in self.state_tensors()]
        if tensors and tensors[0].is_cuda:
            from mlx_omnia_b200.kernels import ops

            ops.copy_slots(tensors, [(request.slot, new.slot)])
        else:
            for tensor in tensors:
                tensor[new.slot] = tensor[request.slot]

    def _copy_rows(self, group: Group, page: int, to: int, rows: int) -> None:
        if group.pages.is_cuda:
            from mlx_omnia_b200.kernels import ops

            ops.copy_pages(group.pages, group.spec.rows, self.page_size, [(page, to, rows)])
            return
        flat, at = group.pages.flatten(2), 0
        for heads, width in group.spec.rows:
            size = heads * self.page_size * width
            block = flat[:, :, at: at + size].unflatten(2, (heads, self.page_size, width))
            block[:, to, :, :rows] = block[:, page, :, :rows]
            at += size

    def resize(self, pages_per_group: "int | dict[KVSpec, int]") -> None:
        """Give every group's pool another number of pages, more or fewer, while requests live: what is held moves to the front of a
        new tensor (old and new ones of all groups exist side by side meanwhile). CacheError where a pool would not take what it holds;
        then, and where an allocation or a copy fails, nothing has changed. No step may be in flight, and
        steps captured on the old tensors are dead afterwards (`StepRunner.forget_graphs`)."""
        counts = [pages_per_group[g.spec] if isinstance(pages_per_group, dict) else pages_per_group for g in self.groups]
        if any(count < 1 for count in counts):
            raise ValueError("a pool has at least one page")
        pools = [group.pool.resized(count) for group, count in zip(self.groups, counts)]
        # Every group's new tensor is made and filled ahead of the first change: an allocation that fails leaves all as it was.
        tensors: list[torch.Tensor | None] = []
        for group, (pool, to) in zip(self.groups, pools):
            old, new = group.pages, None
            if old is not None:
                new = torch.zeros(old.shape[0], pool.count, *old.shape[2:], dtype=old.dtype, device=old.device)
                if old.is_cuda:
                    from mlx_omnia_b200.kernels import ops

                    ops.copy_pages(old, group.spec.rows, self.page_size, [(a, b, self.page_size) for a, b in to.items()], to=new)
                elif to:
                    new[:, list(to.values())] = old[:, list(to)]
            tensors.append(new)
        for g, (group, (pool, to), new) in enumerate(zip(self.groups, pools, tensors)):
            group.pool, group.pages = pool, new
            for request in self.requests.values():
                table = [to.get(page, -1) for page in request.tables[g]]
                request.tables[g], request.arrays[g][: len(table)] = table, table

    def slot_of(self, request: RequestCache, group: int, position: int) -> int:
        row = position // self.groups[group].spec.stride
        page = request.tables[group][row // self.page_size]
        if page < 0:
            raise CacheError(f"position {position} of {request.request_id!r} lies in a page already given back")
        return page * self.page_size + row % self.page_size

    def release_behind_window(self, request: RequestCache) -> int:
        """Give back pages of groups with a window or runs that no later token can read. With
        `tokens` positions written, the next query sits at position >= tokens and sees
        keys >= tokens - window + 1, and none before the start of its own run. Returns how many
        pages were freed."""
        freed = 0
        for g, (group, table) in enumerate(zip(self.groups, request.tables)):
            if not group.spec.forgets:
                continue
            dead_below = group.spec.dead_below(request.tokens)  # positions < this are never read again
            dead_rows = max(dead_below, 0) // group.spec.stride  # stored rows wholly below it
            # Pages that hold any of the first `keep_first` positions stay for the request's whole life.
            kept = -(-group.spec.stored(group.spec.keep_first) // self.page_size) if group.spec.keep_first else 0
            for index in range(min(len(table), dead_rows // self.page_size) - 1, kept - 1, -1):
                if table[index] < 0:
                    break  # everything below was given back earlier
                group.pool.give(table[index])
                table[index] = request.arrays[g][index] = -1
                freed += 1
        return freed

    def close(self, request_id: str) -> None:
        """The request ended: everything it holds is given back."""
        request = self.requests.pop(request_id, None)
        if request is None:
            raise CacheError(f"request {request_id!r} is not open")
        for group, table in zip(self.groups, request.tables):
            for page in table:
                if page >= 0:
                    group.pool.give(page)
            table.clear()
        self.slots.give(request.slot)
        request.slot = -1

    # -- views for a step --------------------------------------------------------------
    def entry_pages(self, entry: int) -> torch.Tensor:
        g, index = self.group_of_entry[entry]
        return self.groups[g].pages[index]

    def check(self) -> None:
        """Every page is either free or in as many tables as it is held times, at one place in all of them, and forks apart no
        request writes to it (used by tests)."""
        for g, group in enumerate(self.groups):
            seen: dict[int, list[tuple[int, str]]] = {}
            for request in self.requests.values():
                for place, page in enumerate(request.tables[g]):
                    if page < 0:
                        continue
                    holders = seen.setdefault(page, [])
                    shared = max((r.positions for r in request.runs), default=0)
                    if holders and (holders[0][0] != place or holders[-1][1] == request.request_id or
                                    place >= self._whole_pages(g, shared)):
                        raise CacheError(f"page {page} of group {g} is held by {holders[-1][1]!r} and {request.request_id!r}")
                    holders.append((place, request.request_id))
            for page, holders in seen.items():
                if group.pool.references(page) != len(holders):
                    raise CacheError(f"page {page} of group {g} is held {group.pool.references(page)} times, by {len(holders)} tables")
            if sorted(seen) != group.pool.held():
                raise CacheError(f"group {g}: pages in tables {sorted(seen)} differ from pages taken {group.pool.held()}")
            if len(seen) + group.pool.free != group.pool.count:
                raise CacheError(f"group {g}: a page was lost")
