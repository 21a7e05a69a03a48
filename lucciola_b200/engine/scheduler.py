"""The scheduler: admits requests, cuts prompts into portions under a token budget, decodes,
finishes and frees.  Host code only; it sees the cache through the CacheManager.

What it keeps of lucciola's scheduler (src/scheduler.cc:42-139): requests that decode go first and
are not limited by the token budget; what is left of the budget goes to prompts, first come first
served, in portions of any size; a page is taken when a request crosses a page boundary; a
finished request gives its pages back at once.

What it decides differently:
  * Several prompts may have portions in one step.  A request is admitted when the pages for its
    whole prompt are free; later portions of a running prompt shrink to the pages that are free
    (lucciola schedules one portion of one prompt, all or nothing, src/scheduler.cc:89-97, and a
    prompt that does not fit blocks the queue for ever).
  * When pages run out, the request admitted last is preempted: its pages go back, it returns to
    the FRONT of the waiting queue and is later recomputed from its prompt plus what it has
    generated, so its output is the same as without the preemption.  (lucciola moves such a
    request to a queue that nothing reads again, src/scheduler.cc:33-40: the request is lost.)
  * A request that could never fit the pool on its own is refused when it is added.
  * With `share_prefixes` set, a request that is admitted while a running one begins with the same tokens takes over the whole pages
    of these that have been computed (all but its last token, at most) and starts behind them.  While the running one is still
    computing tokens that both begin with, the request waits for them, and those behind it that do not may pass.
  * With `token_tile` set, a portion that is not its prompt's last is shortened so that the step's tokens up to and
    including it are a multiple of the tile: the many-token products work on tiles of 128 tokens, and 32 decoded tokens
    beside a portion of 512 make them compute five tiles for 4.25 tiles of tokens.
"""
from __future__ import annotations

from collections import deque
from dataclasses import dataclass
from typing import Callable, Hashable, Iterable, Optional, Sequence

from ..cache.manager import CacheManager
from .prefixes import PrefixTree
from .request import Request, Status


@dataclass
class Scheduled:
    request: Request
    start: int             # position of the first token of this portion
    num_tokens: int
    sample: bool           # the portion reaches the request's last token: sample after the step


# Requests that a step may find to wait for a beginning that is being computed, before it looks no further.
_LOOK_PAST = 8


class Scheduler:
    def __init__(self, manager: CacheManager, max_tokens_per_step: int, max_num_seqs: int, max_model_len: int,
                 prefill_chunk: int = 0, eos_token_ids: Iterable[int] = (),
                 release: Optional[Callable[[Hashable], None]] = None, token_tile: int = 0, share_prefixes: bool = False):
        """`release(rid)` gives back all that a request holds; whoever keeps more per request than the cache
        manager does (the runner's converted block tables) passes its own."""
        self.manager = manager
        self._release_fn = release
        self.max_tokens_per_step = max_tokens_per_step
        self.max_num_seqs = min(max_num_seqs, manager.num_slots)
        self.max_model_len = max_model_len
        self.prefill_chunk = prefill_chunk
        self.token_tile = token_tile
        self.share_prefixes = share_prefixes
        self.eos_token_ids = frozenset(eos_token_ids)
        self.waiting: deque[Request] = deque()
        self.running: list[Request] = []
        self._admissions = 0
        self._prefixes = PrefixTree(manager.page_size)         # of the running requests, with share_prefixes
        self._changes = 0                      # requests that were admitted or ended, and portions that were computed
        self._awaited: dict[Hashable, tuple[Request, int, int]] = {}       # by request: the one that computes what it waits for, the
                                               # latter's admission, and how many pages that is
        self._blocked: Optional[tuple] = None  # the request that had to wait for pages, self._changes then, and how many it needs
        # counters
        self.num_preemptions = 0
        self.num_steps = 0
        self.num_scheduled_tokens = 0
        self.num_shared_tokens = 0             # tokens that were taken over instead of computed

    # ---- requests ----------------------------------------------------------
    def add_request(self, req: Request) -> None:
        req.params.validate()
        n = len(req.prompt)
        if n == 0:
            raise ValueError("a request needs at least one prompt token")
        if n >= self.max_model_len:
            raise ValueError(f"the prompt has {n} tokens; with max_model_len {self.max_model_len} nothing could be generated")
        most = min(n + req.params.max_new_tokens, self.max_model_len)
        for g, pool in enumerate(self.manager.pools):
            pages = self.manager.pages_for(g, most)
            if pages > pool.num_pages:
                raise ValueError(
                    f"the request may grow to {most} tokens = {pages} pages, the pool of cache group {g} has {pool.num_pages}")
        req.status = Status.WAITING
        self.waiting.append(req)

    def has_unfinished(self) -> bool:
        return bool(self.waiting or self.running)

    def abort(self, rid: int) -> bool:
        for r in list(self.running):
            if r.rid == rid:
                self._finish(r, "abort")
                return True
        for r in list(self.waiting):
            if r.rid == rid:
                self.waiting.remove(r)
                self._awaited.pop(rid, None)
                r.status, r.finish_reason = Status.FINISHED, "abort"
                return True
        return False

    # ---- pages, as they will be when the step takes them ----------------------
    def _pages_needed(self, r: Request, new_len: int) -> list[int]:
        if self.manager.has_request(r.rid):
            return self.manager.pages_needed(r.rid, new_len)
        return [self.manager.pages_for(g, new_len) for g in range(len(self.manager.pools))]

    def _fits(self, need: Sequence[int], reserved: Sequence[int]) -> bool:
        return all(p.num_free - reserved[g] >= need[g] for g, p in enumerate(self.manager.pools))

    def _largest_fit(self, r: Request, upto: int, reserved: Sequence[int]) -> int:
        """The largest length <= upto whose pages are free, given what the plan has reserved."""
        ps = self.manager.page_size
        best = upto
        for g, p in enumerate(self.manager.pools):
            have = len(self.manager.block_table(r.rid, g)) if self.manager.has_request(r.rid) else 0
            every = self.manager.groups[g].every       # a group with one entry for every `every` tokens
            best = min(best, (have + p.num_free - reserved[g]) * ps * every + (every - 1))
        return best

    def _release(self, rid: Hashable) -> None:
        if self._release_fn is not None:
            self._release_fn(rid)
        elif self.manager.has_request(rid):
            self.manager.release(rid)

    def _aligned(self, n: int, r: Request, budget: int) -> int:
        """The portion of n tokens, shortened so that the step's tokens so far plus the portion fill whole token tiles;
        unchanged when it is the prompt's last portion, or when less than half of it would be left."""
        tile = self.token_tile
        if tile <= 1 or n >= r.remaining:
            return n
        used = self.max_tokens_per_step - budget
        shorter = (used + n) // tile * tile - used
        return shorter if shorter >= max(1, n // 2) else n

    def _preempt(self, r: Request) -> None:
        self._release(r.rid)
        self.running.remove(r)
        self._forget(r)
        r.status = Status.WAITING
        r.num_computed = 0
        r.preemptions += 1
        self.num_preemptions += 1
        self.waiting.appendleft(r)

    def _finish(self, r: Request, reason: str) -> None:
        self._release(r.rid)
        if r in self.running:
            self.running.remove(r)
            self._forget(r)
        r.status, r.finish_reason = Status.FINISHED, reason

    # ---- requests that begin alike ---------------------------------------------
    def _forget(self, r: Request) -> None:
        """A request that does not run any more."""
        self._prefixes.remove(r.rid)
        self._changes += 1

    def _donor(self, r: Request) -> tuple[Optional[Request], int, bool]:
        """The running request with which r has the most whole pages in common that have been computed, how many, and whether another
        one is still computing more (self._awaited says which)."""
        ps = self.manager.page_size
        best, pages, awaited, more = None, 0, None, 0
        seen: set[Hashable] = set()
        for run, alike in reversed(self._prefixes.walk(r.tokens, (r.length - 1) // ps)):       # those with most in common first
            for d in run.holders.values():
                if d.rid in seen:
                    continue
                seen.add(d.rid)
                have = min(alike, d.num_computed // ps)
                if have > pages:
                    best, pages = d, have
                if d.remaining > 1 and alike > more:
                    awaited, more = d, alike
            if pages >= alike:
                break                          # nobody else has as much
        if more > pages:
            self._awaited[r.rid] = awaited, awaited.admitted_at, more
        return best, pages, more > pages

    def _waits(self, r: Request) -> bool:
        """Whether what r was found to wait for is still being computed."""
        if r.rid in self._awaited:
            d, admitted_at, pages = self._awaited[r.rid]
            if d.status is Status.RUNNING and d.admitted_at == admitted_at and d.remaining > 1 and d.num_computed // self.manager.page_size < pages:
                return True
            del self._awaited[r.rid]
        return False

    # ---- one step ------------------------------------------------------------
    def schedule(self) -> list[Scheduled]:
        """The batch of the next step.  Empty only when there is nothing to do."""
        while True:
            plan = self._schedule_once()
            if plan or not self.running:
                return plan
            # Every running request is stuck for pages: free the latest and try again.
            self._preempt(max(self.running, key=lambda r: r.admitted_at))

    def _schedule_once(self) -> list[Scheduled]:
        plan: list[Scheduled] = []
        # The common step of a running engine: nobody waits, everybody decodes, and there is a free page in every
        # group for each of them (more than they can need).  Nothing to weigh then.
        if not self.waiting and self.running and all(p.num_free >= len(self.running) for p in self.manager.pools) \
                and all(r.remaining == 1 for r in self.running):
            for r in sorted(self.running, key=lambda r: r.admitted_at):
                plan.append(Scheduled(r, r.num_computed, 1, True))
            self.num_steps += 1
            self.num_scheduled_tokens += len(plan)
            return plan
        reserved = [0] * len(self.manager.pools)
        budget = self.max_tokens_per_step

        def take(r: Request, n: int, need: Optional[Sequence[int]] = None) -> None:
            nonlocal budget
            if need is None:
                need = self._pages_needed(r, r.num_computed + n)
            for g, k in enumerate(need):
                reserved[g] += k
            plan.append(Scheduled(r, r.num_computed, n, r.num_computed + n == r.length))
            budget -= n

        preempted = False
        # 1. Requests that decode: one token each, whatever the budget says.
        for r in sorted((r for r in self.running if r.remaining == 1), key=lambda r: r.admitted_at):
            if r.status is not Status.RUNNING:
                continue                      # it was a victim a moment ago
            need = self._pages_needed(r, r.num_computed + 1)
            while not self._fits(need, reserved):
                scheduled = {s.request.rid for s in plan}
                victims = [v for v in self.running if v.rid not in scheduled]
                victim = max(victims, key=lambda v: v.admitted_at)
                self._preempt(victim)
                preempted = True
                if victim is r:
                    break
            if r.status is Status.RUNNING:
                take(r, 1, need)

        # 2. Prompts under way (and requests that are recomputed), oldest first.  After a preemption
        # nothing new starts in this step, or the victim would come straight back.
        blocked = preempted
        for r in sorted((r for r in self.running if r.remaining > 1), key=lambda r: r.admitted_at):
            if budget <= 0:
                break
            most = min(budget, self.prefill_chunk or budget, r.remaining)
            n = self._aligned(most, r, budget)
            n = min(n, self._largest_fit(r, r.num_computed + n, reserved) - r.num_computed)
            if n <= 0:
                blocked = True
                break
            take(r, n)
            if n < most and self.token_tile > 1:
                budget = 0                    # the step ends on a tile's edge: what is left of the budget stays unused

        # 3. New requests, first come first served, while there is budget and a slot.  A request is
        # admitted only when the pages for all it has to run (its prompt, and what it had generated
        # before a preemption) are free now: admitting it earlier would only get it preempted again.
        at = found_to_wait = 0
        while at < len(self.waiting) and not blocked and budget > 0 and len(self.running) < self.max_num_seqs and found_to_wait < _LOOK_PAST:
            r = self.waiting[at]
            donor, pages = None, 0
            if self.share_prefixes:
                # Whoever waits for a beginning lets the next ones pass.  These do not make it wait longer: one that has more in common with it
                # than has been computed would wait for the same.
                if self._waits(r):
                    at += 1
                    continue
                # It had to wait for pages, and since then nobody began, ended or computed what it could take over.
                if self._blocked is not None and self._blocked[:2] == (r.rid, self._changes) and not self._fits(self._blocked[2], reserved):
                    break
                donor, pages, more = self._donor(r)
                if more:
                    at += 1
                    found_to_wait += 1
                    continue
            need = self._pages_needed(r, r.length)
            if not self._fits([k - pages for k in need], reserved):
                self._blocked = r.rid, self._changes, [k - pages for k in need]
                break
            if donor is not None:
                self.manager.admit(r.rid)
                self.manager.share_prefix(r.rid, donor.rid, pages)
                r.num_computed = pages * self.manager.page_size
                self.num_shared_tokens += r.num_computed
            most = min(budget, self.prefill_chunk or budget, r.remaining)
            n = self._aligned(most, r, budget)
            del self.waiting[at]
            r.status = Status.RUNNING
            r.admitted_at = self._admissions
            self._admissions += 1
            self.running.append(r)
            if self.share_prefixes:
                self._prefixes.add(r)
                self._changes += 1
            take(r, n)
            if n < most:
                budget = 0

        self.num_steps += bool(plan)
        self.num_scheduled_tokens += sum(s.num_tokens for s in plan)
        return plan

    def update(self, plan: Sequence[Scheduled], sampled: Sequence[int]) -> list[tuple[Request, int, bool]]:
        """After the step: `sampled` holds one token for each plan entry with sample=True, in order.
        Returns (request, new token, finished) for those entries."""
        out = []
        it = iter(sampled)
        for s in plan:
            r = s.request
            r.num_computed += s.num_tokens
            if s.num_tokens > 1 or not s.sample:
                self._changes += 1
            if not s.sample:
                continue
            tok = int(next(it))
            r.append(tok)
            if self.share_prefixes and r.status is Status.RUNNING and r.length % self.manager.page_size == 0:
                self._prefixes.add(r)
            reason = None
            if tok in self.eos_token_ids and not r.params.ignore_eos:
                reason = "stop"
            elif len(r.output) >= r.params.max_new_tokens:
                reason = "length"
            elif r.length >= self.max_model_len:
                reason = "length"
            if reason:
                self._finish(r, reason)
            out.append((r, tok, reason is not None))
        return out
