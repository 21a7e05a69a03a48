"""Which running requests begin with which tokens: a tree of runs of whole pages, so that a request that is to be admitted is compared
once along the tree and not with every running request."""
from __future__ import annotations

from typing import Hashable, Optional, Sequence

from .request import Request


class _Run:
    """Pages start .. end - 1 of its holders' tokens, which are the same ones for all of them, as is what stands in front."""
    __slots__ = ("tokens", "start", "end", "above", "below", "holders")

    def __init__(self, tokens: Sequence[int], start: int, end: int, above: Optional["_Run"]):
        self.tokens, self.start, self.end, self.above = tokens, start, end, above      # tokens: all of some holder's, now or once
        self.below: dict[tuple, _Run] = {}               # by their first page
        self.holders: dict[Hashable, Request] = {}       # in the order in which they came


class PrefixTree:
    def __init__(self, page_size: int):
        self.page_size = page_size
        self._root = _Run((), 0, 0, None)
        self._last: dict[Hashable, _Run] = {}            # of each request the run in which its whole pages end

    def _page(self, tokens: Sequence[int], i: int) -> tuple:
        return tuple(tokens[i * self.page_size:(i + 1) * self.page_size])

    def _alike(self, run: _Run, tokens: Sequence[int], pages: int) -> int:
        """Up to which page the run's tokens are these, of which there are `pages` pages; the run's first page is known to be."""
        ps = self.page_size
        lo, hi = run.start + 1, min(run.end, pages)
        if run.tokens[lo * ps:hi * ps] == tokens[lo * ps:hi * ps]:
            return hi
        while hi - lo > 1:                               # the same up to lo, not up to hi
            mid = (lo + hi) // 2
            if run.tokens[lo * ps:mid * ps] == tokens[lo * ps:mid * ps]:
                lo = mid
            else:
                hi = mid
        return lo

    def walk(self, tokens: Sequence[int], pages: int) -> list[tuple[_Run, int]]:
        """The runs along the first `pages` pages of these tokens, each with the number of pages up to which it goes along."""
        path, at, run = [], 0, self._root
        while at < pages and at == run.end:
            run = run.below.get(self._page(tokens, at))
            if run is None:
                break
            at = self._alike(run, tokens, pages)
            path.append((run, at))
        return path

    def add(self, r: Request) -> None:
        """A request, or one that is there and has more tokens now."""
        pages, run = r.length // self.page_size, self._last.get(r.rid, self._root)
        while run.end < pages:
            if len(run.holders) == 1 and not run.below:  # its own last run (the root has no holders)
                run.tokens, run.end = r.tokens, pages
                break
            page = self._page(r.tokens, run.end)
            below = run.below.get(page)
            if below is None:
                below = run.below[page] = _Run(r.tokens, run.end, pages, run)
            else:
                at = self._alike(below, r.tokens, pages)
                if at < below.end:
                    below = self._split(below, at)
            below.holders[r.rid] = r
            self._join(run)
            run = below
        self._last[r.rid] = run

    def _split(self, run: _Run, at: int) -> _Run:
        """The part of a run in front of page `at` as a run of its own; the run itself is what is behind (requests end there)."""
        upper = _Run(run.tokens, run.start, at, run.above)
        upper.holders = dict(run.holders)
        upper.below[self._page(run.tokens, at)] = run
        run.above.below[self._page(run.tokens, run.start)] = upper
        run.start, run.above = at, upper
        return upper

    def remove(self, rid: Hashable) -> None:
        run = self._last.pop(rid, self._root)
        while run is not self._root:
            del run.holders[rid]
            above, page = run.above, self._page(run.tokens, run.start)
            if not run.holders:
                del above.below[page]
            else:
                self._join(run)
            run = above

    def _join(self, run: _Run) -> None:
        """A run behind which only one lies, with the same holders, becomes a part of that one."""
        if run is not self._root and len(run.below) == 1:
            (only,) = run.below.values()
            if len(only.holders) == len(run.holders):
                only.start, only.above = run.start, run.above
                run.above.below[self._page(run.tokens, run.start)] = only

    def __len__(self) -> int:
        """Requests that are in the tree."""
        return len(self._last)

    def num_runs(self) -> int:
        n, runs = 0, list(self._root.below.values())
        while runs:
            n += 1
            runs.extend(runs.pop().below.values())
        return n
