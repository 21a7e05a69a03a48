"""Cache manager: pages of keys and values for groups of layers, and slots of per-request state.

Layers whose caches have the same needs (kv heads, head size, all keys or a window of W keys)
form a group.  A group has its own pool of pages and, for every request, its own block table;
one page id is valid in every layer of its group.  Pages go back to the pool when a request
ends, when it is preempted, and, in a window group, as soon as the window has passed them.
Beside the pages every request holds one slot of fixed-size state for mixers that ask for it.

lucciola has one group (every layer keeps all keys), takes pages when a request crosses a page
boundary or for a whole portion of a prompt at once (src/scheduler.cc:55-58, 89-97) and gives
them back when the request ends or is preempted (src/scheduler.cc:20-40); the same rules hold
here for each group.  Everything in this file is host bookkeeping; device memory is in
device_cache.py.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Optional, Hashable, Sequence

from ..parts.base import KVPages, StateSlot
from .page_pool import PagePool, PagePoolError

NO_PAGE = -1


@dataclass(frozen=True)
class CacheGroup:
    num_kv_heads: int
    head_dim: int
    window: int                      # 0: all keys
    cache_ids: tuple                 # the model's caches that live in this group: cache ids, or (cache id, place) for a
                                     # member of a cache id that asked for a tuple
    shared: bool = False             # one vector a token is key and value at once
    v_head_dim: int = 0              # size of a value head when it differs from the keys' (0: the same)
    every: int = 1                   # P > 1: the group holds one entry for every P tokens of a sequence (n // P for n tokens)


def flat_requests(requests: Sequence[KVPages | StateSlot | None | tuple]) -> list[tuple[object, object]]:
    """Every single thing the model's caches hold: (key, request), the key being the cache id, or (cache id, place)
    for the members of a cache id that asks for a tuple."""
    out = []
    for cid, r in enumerate(requests):
        if isinstance(r, tuple):
            out += [((cid, j), one) for j, one in enumerate(r)]
        else:
            out.append((cid, r))
    return out


def plan_groups(requests: Sequence[KVPages | StateSlot | None | tuple]) -> tuple[list[CacheGroup], list]:
    """Group the model's paged caches by their needs.  Returns the groups and the keys (see flat_requests) that hold state."""
    by_key: dict[tuple, list] = {}
    state_ids: list = []
    for key, r in flat_requests(requests):
        if isinstance(r, KVPages):
            by_key.setdefault((r.num_kv_heads, r.head_dim, r.window, r.shared, r.v_head_dim if r.v_head_dim != r.head_dim else 0,
                               max(1, r.every)), []).append(key)
        elif isinstance(r, StateSlot):
            state_ids.append(key)
    groups = [CacheGroup(k[0], k[1], k[2], tuple(v), k[3], k[4], k[5]) for k, v in by_key.items()]
    return groups, state_ids


@dataclass
class _RequestCache:
    slot: int
    tables: list[list[int]]          # per group: page of each logical page index, NO_PAGE once released
    length: int = 0                  # tokens whose keys are (or are about to be) in the cache
    version: int = 0                 # new, manager-wide unique number whenever a table changes (lets callers cache a converted copy)
    cuts: set[int] = field(default_factory=set)      # numbers of first pages that it has, or had, in common with others


@dataclass(eq=False)
class _Alike:
    """Requests of a step (by their places in it) that have their first pages in common, and the groups chosen among them."""
    members: list[int]
    spared: int                      # pages that need not be read again
    groups: list[tuple[list[int], int]]              # members and pages
    rest: list[int]                  # members of no group


# Keys that attention reads at a time (ops.attention_shared): a group with fewer in common reads nothing less.
_BLOCK_KEYS = 64


class CacheManager:
    def __init__(self, groups: Sequence[CacheGroup], page_size: int, num_pages: int | Sequence[int], num_slots: int):
        self.groups = list(groups)
        self.page_size = page_size
        counts = [num_pages] * len(self.groups) if isinstance(num_pages, int) else list(num_pages)
        self.pools = [PagePool(n) for n in counts]
        self.num_slots = num_slots
        self._free_slots = list(range(num_slots - 1, -1, -1))
        self._requests: dict[Hashable, _RequestCache] = {}
        self._versions = 0
        self._shares = 0                 # changes whenever a request takes over pages, or one that has some in common with others ends
        self._groups_of: tuple = (None, None, None)          # requests, self._shares and the answer of the last prefix_groups

    # ---- requests ------------------------------------------------------
    def has_request(self, rid: Hashable) -> bool:
        return rid in self._requests

    def can_admit(self) -> bool:
        return bool(self._free_slots)

    def admit(self, rid: Hashable) -> int:
        """Give a new request its state slot and empty block tables."""
        if rid in self._requests:
            raise PagePoolError(f"request {rid!r} is already admitted")
        if not self._free_slots:
            raise PagePoolError("no free state slot")
        slot = self._free_slots.pop()
        self._versions += 1
        self._requests[rid] = _RequestCache(slot, [[] for _ in self.groups], version=self._versions)
        return slot

    def release(self, rid: Hashable) -> None:
        """Give back everything a request holds (it ended or is preempted)."""
        rc = self._requests.pop(rid)
        self._shares += bool(rc.cuts)
        for g, table in enumerate(rc.tables):
            for p in table:
                if p != NO_PAGE:
                    self.pools[g].free(p)
        self._free_slots.append(rc.slot)

    # ---- requests that begin alike ------------------------------------------
    def can_share(self) -> bool:
        """Whether requests may hold pages in common: every group keeps one entry for every token to the end, and nothing else is kept."""
        return bool(self.groups) and all(g.window <= 0 and g.every <= 1 for g in self.groups)

    def share_prefix(self, rid: Hashable, donor: Hashable, pages: int) -> None:
        """The first `pages` pages of `donor`, which hold computed tokens, become the first of `rid`, which has been admitted and
        has none yet: its length is that many pages then."""
        if not self.can_share():
            raise PagePoolError("requests of these cache groups cannot hold pages in common")
        rc, dc = self._requests[rid], self._requests[donor]
        if rc.length or any(rc.tables) or rid == donor:
            raise PagePoolError(f"request {rid!r} cannot take over pages: it has some")
        if not 0 < pages <= dc.length // self.page_size:
            raise PagePoolError(f"{pages} pages of request {donor!r}, which has filled {dc.length // self.page_size}")
        for g, table in enumerate(dc.tables):
            for p in table[:pages]:
                self.pools[g].share(p)
            rc.tables[g].extend(table[:pages])
        # Whoever has these pages has them as its first: a page has the same place in all tables.
        last = dc.tables[0][pages - 1]
        for other in self._requests.values():
            if len(other.tables[0]) >= pages and other.tables[0][pages - 1] == last:
                other.cuts.add(pages)
        rc.cuts |= {c for c in dc.cuts if c < pages}
        self._shares += 1
        rc.length = pages * self.page_size
        self._versions += 1
        rc.version = self._versions

    def prefix_groups(self, rids: Sequence[Hashable]) -> Optional[tuple[list[int], list[int]]]:
        """Which of these requests begin with the same pages: for each the place in the list of the request whose pages stand for
        its group's (-1: no group), and for that one how many tokens the group has in common (0 for the others).  Where requests share a
        short beginning and some of them a long one, there are as many groups as spare most keys.  None when there is no group."""
        rids = tuple(rids)
        if self._groups_of[:2] != (rids, self._shares):
            self._groups_of = rids, self._shares, self._find_groups(rids)
        found = self._groups_of[2]
        return None if found is None else (list(found[0]), list(found[1]))

    def _find_groups(self, rids: Sequence[Hashable]) -> Optional[tuple[list[int], list[int]]]:
        # Requests with the same page in front of a cut have all pages up to there in common.  Two sets of such requests are one inside the
        # other, or have nobody in common: a tree, in which a deeper set has more pages.
        sets: dict[tuple[int, int], list[int]] = {}
        for i, rid in enumerate(rids):
            rc = self._requests.get(rid)
            if rc is not None and rc.cuts:
                rc.cuts = {c for c in rc.cuts if self.pools[0].holders(rc.tables[0][c - 1]) > 1}
                for c in rc.cuts:
                    sets.setdefault((c, rc.tables[0][c - 1]), []).append(i)
        innermost: dict[int, _Alike] = {}                     # of each member the last set that went by
        for (pages, _), members in sorted(sets.items(), key=lambda kv: -kv[0][0]):
            if len(members) > 1:
                below = {id(innermost[i]): innermost[i] for i in members if i in innermost}
                node = self._alike(pages, members, [i for i in members if i not in innermost], list(below.values()))
                innermost.update(dict.fromkeys(members, node))
        groups = [g for node in {id(n): n for n in innermost.values()}.values() for g in node.groups]
        if not groups:
            return None
        prefix_of, prefix_lens = [-1] * len(rids), [0] * len(rids)
        for members, pages in groups:
            leader = min(members)
            prefix_lens[leader] = pages * self.page_size
            for i in members:
                prefix_of[i] = leader
        return prefix_of, prefix_lens

    def _alike(self, pages: int, members: list[int], direct: list[int], below: list["_Alike"]) -> "_Alike":
        """The best of three for a set of requests: the groups of the sets in it alone; all in one group; a group of those whom these
        leave over (and of sets whose members gain more that way), if they have a block of the kernels' in common."""
        groups = [g for n in below for g in n.groups]
        best = _Alike(members, sum(n.spared for n in below), groups, direct + [i for n in below for i in n.rest])
        whole = (len(members) - 1) * pages
        if whole > best.spared:
            best = _Alike(members, whole, [(members, pages)], [])
        kept = [n for n in below if n.spared + len(n.rest) * pages >= len(n.members) * pages]
        rest = direct + [i for n in below for i in (n.rest if n in kept else n.members)]
        spared = sum(n.spared for n in kept) + (len(rest) - 1) * pages
        if kept and len(rest) > 1 and pages * self.page_size >= _BLOCK_KEYS and spared > best.spared:
            best = _Alike(members, spared, [g for n in kept for g in n.groups] + [(rest, pages)], [])
        return best

    # ---- pages ---------------------------------------------------------
    def _first_needed_page(self, g: int, start: int) -> int:
        """Index of the first page a query at position `start` can still see in group g."""
        w = self.groups[g].window
        return max(0, start - w + 1) // self.page_size if w > 0 else 0

    def pages_for(self, g: int, length: int) -> int:
        """Pages of group g that back a sequence of `length` tokens: one entry a token, or one for every whole block of
        `every` tokens."""
        every = self.groups[g].every
        entries = length // every if every > 1 else length
        return -(-entries // self.page_size)

    def pages_needed(self, rid: Hashable, new_length: int) -> list[int]:
        """Pages each group has to take so that positions below new_length are backed."""
        rc = self._requests[rid]
        return [max(0, self.pages_for(g, new_length) - len(t)) for g, t in enumerate(rc.tables)]

    def can_extend(self, rid: Hashable, new_length: int) -> bool:
        return all(self.pools[g].can_allocate(n) for g, n in enumerate(self.pages_needed(rid, new_length)))

    def extend(self, rid: Hashable, new_length: int) -> bool:
        """Take the pages for positions [length, new_length) in every group, all or nothing."""
        rc = self._requests[rid]
        if new_length < rc.length:
            raise PagePoolError(f"request {rid!r} cannot shrink from {rc.length} to {new_length}")
        need = self.pages_needed(rid, new_length)
        if not all(self.pools[g].can_allocate(n) for g, n in enumerate(need)):
            return False
        for g, n in enumerate(need):
            for _ in range(n):
                rc.tables[g].append(self.pools[g].allocate())
        if any(need):
            self._versions += 1
            rc.version = self._versions
        rc.length = new_length
        return True

    def extend_by_one(self, rids: Sequence[Hashable]) -> Optional[list[int]]:
        """One more position for each of these admitted requests, all or nothing: the step of a decoding batch.
        Returns the positions the new tokens take (the lengths before), or None when a group lacks the pages."""
        ps = self.page_size
        reqs = [self._requests[rid] for rid in rids]
        need = [0] * len(self.groups)
        for rc in reqs:
            for g, t in enumerate(rc.tables):
                want = self.pages_for(g, rc.length + 1)      # pages that back positions 0 .. length
                if want > len(t):
                    need[g] += want - len(t)
        if any(need) and not all(self.pools[g].can_allocate(n) for g, n in enumerate(need)):
            return None
        starts = []
        for rc in reqs:
            grew = False
            for g, t in enumerate(rc.tables):
                want = self.pages_for(g, rc.length + 1)
                while len(t) < want:
                    t.append(self.pools[g].allocate())
                    grew = True
            if grew:
                self._versions += 1
                rc.version = self._versions
            starts.append(rc.length)
            rc.length += 1
        return starts

    def retract_by_one(self, rids: Sequence[Hashable]) -> None:
        """Undo extend_by_one for a step that was prepared and will not run.  A page that was taken for the position
        stays in the request's table (the position's next step finds it there; a request that ends gives it back)."""
        for rid in rids:
            rc = self._requests.get(rid)
            if rc is not None and rc.length > 0:
                rc.length -= 1

    def max_extension(self, rid: Hashable, upto: int) -> int:
        """The largest length <= upto that the free pages allow for this request."""
        rc = self._requests[rid]
        best = upto
        for g, t in enumerate(rc.tables):
            every = self.groups[g].every
            best = min(best, (len(t) + self.pools[g].num_free) * self.page_size * every + (every - 1))
        return max(min(best, upto), rc.length)

    def release_behind_window(self, rid: Hashable) -> int:
        """After a step: free the pages that no later query of this request can see.  Returns how many."""
        rc = self._requests[rid]
        freed = 0
        for g, table in enumerate(rc.tables):
            if self.groups[g].window <= 0:
                continue
            first = min(self._first_needed_page(g, rc.length), len(table))
            for i in range(first):
                if table[i] != NO_PAGE:
                    self.pools[g].free(table[i])
                    table[i] = NO_PAGE
                    freed += 1
        if freed:
            self._versions += 1
            rc.version = self._versions
        return freed

    # ---- views ---------------------------------------------------------
    def length(self, rid: Hashable) -> int:
        return self._requests[rid].length

    def slot(self, rid: Hashable) -> int:
        return self._requests[rid].slot

    def block_table(self, rid: Hashable, group: int) -> list[int]:
        return self._requests[rid].tables[group]

    def version(self, rid: Hashable) -> int:
        return self._requests[rid].version

    def num_requests(self) -> int:
        return len(self._requests)

    def check_invariants(self) -> None:
        """No page lost, none held twice: every page is free or in as many tables as it has holders, at the same place in all of them."""
        for g, pool in enumerate(self.pools):
            places: dict[int, list[int]] = {}
            for rid, rc in self._requests.items():
                for i, p in enumerate(rc.tables[g]):
                    if p != NO_PAGE:
                        places.setdefault(p, []).append(i)
            for p, at in places.items():
                if len(at) != pool.holders(p) or len(set(at)) > 1:
                    raise PagePoolError(f"page {p} of group {g} is held twice ({len(at)} tables, {pool.holders(p)} holders)")
            seen = set(places)
            free = set(pool._free)
            if len(free) != len(pool._free):
                raise PagePoolError(f"group {g}: a page is twice in the free list")
            if seen & free:
                raise PagePoolError(f"group {g}: pages {sorted(seen & free)} are both held and free")
            if len(seen) + len(free) != pool.num_pages:
                raise PagePoolError(f"group {g}: {pool.num_pages - len(seen) - len(free)} page(s) lost")
        slots = [rc.slot for rc in self._requests.values()]
        if len(set(slots)) != len(slots) or set(slots) & set(self._free_slots):
            raise PagePoolError("a state slot is held twice")
        if len(slots) + len(self._free_slots) != self.num_slots:
            raise PagePoolError("a state slot is lost")
