"""The cache manager: keys and values in fixed-size pages with a block table for each request,
one pool per group of layers with the same needs, and slots for per-request state of fixed size.

The reference keeps one contiguous, grown-by-copy buffer per layer (main + tail of up to 63 rows,
src/model.br:1670-1695) for its single sequence, truncates by setting a length (:2313-2314) and
treats windows as masks over the full cache (README.md:237). Pages, block tables, groups and
slots are this engine's own design in the role of src/kvplane.br; what carries over is that a
cache is only ever read up to the request's length, so freed pages need no clearing.

Everything here is host-side bookkeeping and runs without a GPU; `storage.CacheStorage` owns the
device tensors that the page and slot numbers index.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Callable, Dict, List, Optional, Sequence, Tuple, Union


@dataclass(frozen=True)
class PagedKVSpec:
    """What a mixer that caches keys and values needs: `window` 0 keeps every key, n > 0 only the
    last n positions (the query's own included). `v_head_dim` 0: values have the keys' head size.
    `chunk` n > 0: a query sees only the keys of its own run of n positions counted from 0, so the
    pages before the run of the next position are never read again. `values_in_keys`: a key row's first
    `v_head_dim` values are also its value (attention over one cached latent per token), so the layer
    keeps one tensor and its values are a view into it."""
    n_kv_heads: int
    head_dim: int
    window: int = 0
    v_head_dim: int = 0
    chunk: int = 0
    values_in_keys: bool = False

    def first_needed(self, next_pos: int) -> int:
        """The first key that the query at `next_pos`, or any later one, can still see."""
        lo = 0
        if self.window > 0:
            lo = max(lo, next_pos - self.window + 1)
        if self.chunk > 0:
            lo = max(lo, next_pos - next_pos % self.chunk)
        return lo

    @property
    def value_dim(self) -> int:
        return self.v_head_dim if self.v_head_dim > 0 else self.head_dim


@dataclass(frozen=True)
class StateSpec:
    """Per-request state of fixed size (a recurrent state, a running sum): one tensor of `shape`
    per request and cache layer, zero when the request is admitted."""
    shape: Tuple[int, ...]
    dtype: str = "float32"


CacheSpec = Union[PagedKVSpec, StateSpec, None]


class CacheError(RuntimeError):
    """A misuse of the manager (unknown request, double free, ...): a bug of the caller."""


class PagePool:
    """Free pages of one group, handed out last-freed-first so that small pools reuse pages at once."""

    def __init__(self, num_pages: int):
        if num_pages <= 0:
            raise ValueError(f"a page pool needs at least one page, got {num_pages}")
        self.num_pages = num_pages
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._owner: List[Optional[object]] = [None] * num_pages
        self._others: Dict[int, List[object]] = {}     # page -> its further owners (requests that were forked share pages)
        self.high_water = 0
        self.freed_log: Optional[List[int]] = None     # when a list: every page given back is noted here (debugging)

    @property
    def num_free(self) -> int:
        return len(self._free)

    def take(self, owner) -> int:
        if not self._free:
            raise CacheError("page pool is empty (reserve() must check before taking)")
        p = self._free.pop()
        if self._owner[p] is not None:
            raise CacheError(f"page {p} was on the free list while owned by {self._owner[p]!r}")
        self._owner[p] = owner
        self.high_water = max(self.high_water, self.num_pages - len(self._free))
        return p

    def give_back(self, page: int, owner) -> None:
        if not 0 <= page < self.num_pages:
            raise CacheError(f"page {page} is outside the pool")
        if self._owner[page] is None:
            raise CacheError(f"page {page} freed twice")
        others = self._others.get(page)
        if others and (self._owner[page] == owner or owner in others):
            if self._owner[page] == owner:             # the page stays with the others
                self._owner[page] = others.pop(0)
            else:
                others.remove(owner)
            if not others:
                del self._others[page]
            return
        if self._owner[page] != owner:
            raise CacheError(f"page {page} is owned by {self._owner[page]!r}, not by {owner!r}")
        self._owner[page] = None
        self._free.append(page)
        if self.freed_log is not None:
            self.freed_log.append(page)

    def owner_of(self, page: int):
        return self._owner[page]

    def share(self, page: int, owner) -> None:
        """One more owner of a page that is held."""
        if self._owner[page] is None:
            raise CacheError(f"page {page} is free and cannot be shared")
        if owner in self.owners_of(page):
            raise CacheError(f"page {page} is held by {owner!r} already")
        self._others.setdefault(page, []).append(owner)

    def is_shared(self, page: int) -> bool:
        return page in self._others

    def owners_of(self, page: int) -> List[object]:
        return ([] if self._owner[page] is None else [self._owner[page]]) + self._others.get(page, [])


@dataclass
class PagedGroup:
    spec: PagedKVSpec
    cache_layers: List[int]          # cache ids that share this group's block tables
    pool: PagePool


@dataclass
class StateGroup:
    spec: StateSpec
    cache_layers: List[int]


@dataclass
class RequestCache:
    """What one live request holds: a slot, its length, and one block table per paged group.
    A table entry of -1 is a page that a window has passed and that was given back."""
    request_id: object
    slot: int
    num_tokens: int = 0
    tables: List[List[int]] = field(default_factory=list)
    uid: int = 0          # unlike request_id never used twice by one manager
    version: int = 0      # counts the changes of `tables`: (uid, version) names one state of the block tables
    forked: bool = False  # this request may share pages with others: the one that it writes next has to be looked at


class CacheManager:
    def __init__(self, specs: Sequence[CacheSpec], page_size: int, capacity_tokens: int,
                 max_requests: int, on_slot_assigned: Optional[Callable[[int], None]] = None):
        """`specs[c]` is what cache layer `c` needs (None: nothing). Layers with equal needs form
        a group; every paged group gets a pool of ceil(capacity_tokens / page_size) pages."""
        if page_size <= 0 or capacity_tokens <= 0 or max_requests <= 0:
            raise ValueError("page_size, capacity_tokens and max_requests must be positive")
        self.page_size = page_size
        self.capacity_tokens = capacity_tokens
        self.max_requests = max_requests
        self.num_pages = -(-capacity_tokens // page_size)
        self.paged_groups: List[PagedGroup] = []
        self.state_groups: List[StateGroup] = []
        # cache layer -> ("paged" | "state", group index, index inside the group)
        self.layer_location: Dict[int, Tuple[str, int, int]] = {}
        for c, spec in enumerate(specs):
            if spec is None:
                continue
            if isinstance(spec, PagedKVSpec):
                if spec.window < 0 or spec.chunk < 0:
                    raise ValueError(f"cache layer {c}: window and chunk must not be negative")
                for gi, g in enumerate(self.paged_groups):
                    if g.spec == spec:
                        break
                else:
                    gi = len(self.paged_groups)
                    self.paged_groups.append(PagedGroup(spec, [], PagePool(self.num_pages)))
                g = self.paged_groups[gi]
                self.layer_location[c] = ("paged", gi, len(g.cache_layers))
                g.cache_layers.append(c)
            elif isinstance(spec, StateSpec):
                for gi, sg in enumerate(self.state_groups):
                    if sg.spec == spec:
                        break
                else:
                    gi = len(self.state_groups)
                    self.state_groups.append(StateGroup(spec, []))
                sg = self.state_groups[gi]
                self.layer_location[c] = ("state", gi, len(sg.cache_layers))
                sg.cache_layers.append(c)
            else:
                raise TypeError(f"cache layer {c}: unknown cache spec {spec!r}")
        self._free_slots: List[int] = list(range(max_requests - 1, -1, -1))
        self._requests: Dict[object, RequestCache] = {}
        self._on_slot_assigned = on_slot_assigned
        self._next_uid = 0
        # per paged group: (page, its copy) pairs that have to be copied before the next step writes (`take_copies`)
        self._copies: List[List[Tuple[int, int]]] = [[] for _ in self.paged_groups]

    # ---- requests -------------------------------------------------------------------------
    def has_free_slot(self) -> bool:
        return bool(self._free_slots)

    def add_request(self, request_id) -> RequestCache:
        if request_id in self._requests:
            raise CacheError(f"request {request_id!r} is already live")
        if not self._free_slots:
            raise CacheError("no free request slot (check has_free_slot() before admitting)")
        slot = self._free_slots.pop()
        rc = RequestCache(request_id, slot, 0, [[] for _ in self.paged_groups], self._next_uid)
        self._next_uid += 1
        self._requests[request_id] = rc
        if self._on_slot_assigned is not None:
            self._on_slot_assigned(slot)       # the storage zeroes the slot's state
        return rc

    def get(self, request_id) -> RequestCache:
        try:
            return self._requests[request_id]
        except KeyError:
            raise CacheError(f"request {request_id!r} is not live") from None

    def find(self, request_id) -> Optional[RequestCache]:
        """The live request's record, or None."""
        return self._requests.get(request_id)

    def __contains__(self, request_id) -> bool:
        return request_id in self._requests

    def live_requests(self):
        return list(self._requests)

    # ---- pages ----------------------------------------------------------------------------
    def _pages_needed(self, rc: RequestCache, n_new: int) -> List[int]:
        total = -(-(rc.num_tokens + n_new) // self.page_size)
        return [max(0, total - len(t)) + (1 if rc.forked and self._writes_shared(rc, g, t) else 0) for g, t in zip(self.paged_groups, rc.tables)]

    def _writes_shared(self, rc: RequestCache, group: PagedGroup, table: List[int]) -> bool:
        """Whether the page that the request's next token goes to is one that other requests hold, too."""
        at = rc.num_tokens // self.page_size
        return rc.num_tokens % self.page_size != 0 and at < len(table) and table[at] >= 0 and group.pool.is_shared(table[at])

    def pages_needed(self, request_id, n_new: int) -> List[int]:
        """Pages that `n_new` more tokens take from each group's pool (the copy of a shared page among them)."""
        return self._pages_needed(self.get(request_id), n_new)

    def pages_needed_together(self, wants: Sequence[Tuple[object, int]]) -> List[int]:
        """Pages that a step takes from each group's pool: (request, new tokens) pairs, reserved one behind the other. Of a shared page's
        owners the last one writes in place if all of them write."""
        need = [0] * len(self.paged_groups)
        writers: Dict[Tuple[int, int], int] = {}              # (group, shared page) -> requests that are about to write to it
        for request_id, n_new in wants:
            rc = self.get(request_id)
            for gi, (n, group, table) in enumerate(zip(self._pages_needed(rc, n_new), self.paged_groups, rc.tables)):
                need[gi] += n
                if rc.forked and self._writes_shared(rc, group, table):
                    at = gi, table[rc.num_tokens // self.page_size]
                    writers[at] = writers.get(at, 0) + 1
        for (gi, page), n in writers.items():
            if n == len(self.paged_groups[gi].pool.owners_of(page)):
                need[gi] -= 1
        return need

    def can_reserve(self, request_id, n_new: int) -> bool:
        rc = self.get(request_id)
        need = self._pages_needed(rc, n_new)
        return all(n <= g.pool.num_free for n, g in zip(need, self.paged_groups))

    def pages_short(self, request_id, n_new: int) -> int:
        """How many pages the fullest group lacks for `n_new` more tokens (0: it fits)."""
        rc = self.get(request_id)
        need = self._pages_needed(rc, n_new)
        return max([0] + [n - g.pool.num_free for n, g in zip(need, self.paged_groups)])

    def reserve(self, request_id, n_new: int) -> bool:
        """Gives the request pages for `n_new` more tokens in every group, or none at all."""
        if n_new <= 0:
            raise CacheError("reserve() needs a positive number of tokens")
        rc = self.get(request_id)
        need = self._pages_needed(rc, n_new)
        if any(n > g.pool.num_free for n, g in zip(need, self.paged_groups)):
            return False
        for gi, (n, g, table) in enumerate(zip(need, self.paged_groups, rc.tables)):
            if n and rc.forked and self._writes_shared(rc, g, table):
                # the next token goes to a page that others read: this request goes on in a copy of its own
                at, page = rc.num_tokens // self.page_size, g.pool.take(request_id)
                self._copies[gi].append((table[at], page))
                g.pool.give_back(table[at], request_id)
                table[at] = page
                rc.version += 1
                n -= 1
            for _ in range(n):
                table.append(g.pool.take(request_id))
            if n:
                rc.version += 1
        return True

    def fork(self, request_id, new_id, n_keep: Optional[int] = None) -> RequestCache:
        """A new request that holds the first `n_keep` tokens (default: all) of a live one: it shares their pages, and whoever
        writes to a shared page first goes on in a copy (`reserve`; the storage copies what `take_copies` returns before the
        next step). Costs no pages now. The caller copies the state slot, if there are state groups (then `n_keep` must be all). Not
        possible once a window has given pages back that the shorter prefix needs."""
        rc = self.get(request_id)
        n_keep = rc.num_tokens if n_keep is None else n_keep
        if not 0 <= n_keep <= rc.num_tokens:
            raise CacheError(f"fork: {n_keep} tokens outside 0..{rc.num_tokens}")
        if self.state_groups and n_keep != rc.num_tokens:
            raise CacheError("fork: state of fixed size holds all of a request's tokens, not a prefix")
        keep_pages = -(-n_keep // self.page_size)
        for g, table in zip(self.paged_groups, rc.tables):
            first = max(0, g.spec.first_needed(n_keep)) // self.page_size
            if any(p < 0 for p in table[first:keep_pages]):
                raise CacheError("fork: a window has already given pages of the kept prefix back")
        new = self.add_request(new_id)
        new.num_tokens = n_keep
        for g, table, into in zip(self.paged_groups, rc.tables, new.tables):
            for p in table[:keep_pages]:
                if p >= 0:
                    g.pool.share(p, new_id)
                into.append(p)
        rc.forked = new.forked = True
        new.version += 1
        return new

    def take_copies(self) -> List[List[Tuple[int, int]]]:
        """Per paged group the (page, copy) pairs that have come up since the last call, each copy once."""
        out, self._copies = self._copies, [[] for _ in self.paged_groups]
        return out

    @property
    def has_copies(self) -> bool:
        return any(self._copies)

    def commit(self, request_id, n_new: int) -> None:
        """The step has written `n_new` tokens. Pages that every later query's window has passed
        go back to their pool: a query at position p sees keys j with j + window > p
        (src/math.br:327-328), so page i is dead once (i + 1) * page_size <= p - window + 1."""
        rc = self.get(request_id)
        rc.num_tokens += n_new
        for table in rc.tables:
            if rc.num_tokens > len(table) * self.page_size:
                raise CacheError(f"request {request_id!r}: committed past its reserved pages")
        for g, table in zip(self.paged_groups, rc.tables):
            if g.spec.window <= 0 and g.spec.chunk <= 0:
                continue
            first_needed = g.spec.first_needed(rc.num_tokens) if g.spec.chunk > 0 else rc.num_tokens - g.spec.window + 1
            dead = min(len(table), max(0, first_needed) // self.page_size)
            for i in range(dead):
                if table[i] >= 0:
                    g.pool.give_back(table[i], request_id)
                    table[i] = -1
                    rc.version += 1

    def truncate(self, request_id, n_keep: int) -> None:
        """Keeps the first `n_keep` tokens (the reference truncates by setting a length,
        src/model.br:2313-2314). Not possible once a window has given pages of that prefix back."""
        rc = self.get(request_id)
        if not 0 <= n_keep <= rc.num_tokens:
            raise CacheError(f"truncate({n_keep}) outside 0..{rc.num_tokens}")
        keep_pages = -(-n_keep // self.page_size)
        for g, table in zip(self.paged_groups, rc.tables):
            if (g.spec.window > 0 or g.spec.chunk > 0) and n_keep < rc.num_tokens:
                first_needed = (g.spec.first_needed(n_keep) if g.spec.chunk > 0 else max(0, n_keep - g.spec.window + 1)) // self.page_size
                if any(p < 0 for p in table[first_needed:keep_pages]):
                    raise CacheError("truncate: a window has already given pages of the kept prefix back")
            while len(table) > keep_pages:
                p = table.pop()
                rc.version += 1
                if p >= 0:
                    g.pool.give_back(p, request_id)
        rc.num_tokens = n_keep

    def release_ahead(self, request_id) -> None:
        """Gives back the pages that were reserved for tokens which have not come: what lies behind the last token's page."""
        self.truncate(request_id, self.get(request_id).num_tokens)

    def free(self, request_id) -> None:
        """The request ends (or is preempted): every page and its slot go back."""
        rc = self.get(request_id)
        for g, table in zip(self.paged_groups, rc.tables):
            for p in reversed(table):
                if p >= 0:
                    g.pool.give_back(p, request_id)
            table.clear()
        del self._requests[request_id]
        self._free_slots.append(rc.slot)

    # ---- figures and checks ---------------------------------------------------------------
    def free_pages(self) -> List[int]:
        return [g.pool.num_free for g in self.paged_groups]

    def stats(self) -> dict:
        return {
            "pages_total": self.num_pages,
            "pages_in_use": [self.num_pages - g.pool.num_free for g in self.paged_groups],
            "pages_high_water": [g.pool.high_water for g in self.paged_groups],
            "live_requests": len(self._requests),
        }

    def check(self) -> None:
        """No page lost, held twice or both free and held; slots likewise. Raises CacheError."""
        for gi, g in enumerate(self.paged_groups):
            held: Dict[int, List[object]] = {}
            for rid, rc in self._requests.items():
                for p in rc.tables[gi]:
                    if p < 0:
                        continue
                    owners = g.pool.owners_of(p)
                    if rid not in owners:
                        raise CacheError(f"group {gi}: page {p} in {rid!r}'s table but owned by {owners!r}")
                    if rid in held.setdefault(p, []) or len(held[p]) == len(owners):
                        raise CacheError(f"group {gi}: page {p} held by {held[p]!r} and {rid!r}")
                    held[p].append(rid)
            for p, rids in held.items():
                if len(rids) != len(g.pool.owners_of(p)):
                    raise CacheError(f"group {gi}: page {p} owned by {g.pool.owners_of(p)!r}, in the tables of {rids!r}")
            free = list(g.pool._free)
            if len(set(free)) != len(free):
                raise CacheError(f"group {gi}: a page is on the free list twice")
            if set(free) & set(held):
                raise CacheError(f"group {gi}: pages both free and held: {sorted(set(free) & set(held))}")
            if len(free) + len(held) != g.pool.num_pages:
                raise CacheError(f"group {gi}: {g.pool.num_pages - len(free) - len(held)} pages lost")
        slots = [rc.slot for rc in self._requests.values()]
        if len(set(slots)) != len(slots) or set(slots) & set(self._free_slots):
            raise CacheError("a request slot is held twice or both free and held")
        if len(slots) + len(self._free_slots) != self.max_requests:
            raise CacheError("a request slot is lost")
