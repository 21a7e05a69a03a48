"""The tree of running requests' pages, and what the scheduler asks of it: the answers of comparing every pair, at the cost of one comparison."""
import random

import pytest

from lucciola_b200.cache import CacheGroup, CacheManager
from lucciola_b200.engine.prefixes import PrefixTree
from lucciola_b200.engine.request import Request, Status
from lucciola_b200.engine.scheduler import Scheduler
from lucciola_b200.sampling.params import SamplingParams

PS = 4


class Token(int):
    """A token that counts how often it is compared."""
    compared = 0

    def __eq__(self, other):
        Token.compared += 1
        return int(self) == int(other)

    __hash__ = int.__hash__


def request(rid, tokens):
    return Request(rid, list(tokens), SamplingParams(max_new_tokens=1000))


def alike(a, b, most):
    """Whole pages with which both begin, at most `most`."""
    n = 0
    while n < most and a[n * PS:(n + 1) * PS] == b[n * PS:(n + 1) * PS] and (n + 1) * PS <= min(len(a), len(b)):
        n += 1
    return n


@pytest.mark.parametrize("seed", range(20))
def test_walks_of_a_changing_tree(seed):
    """Requests that come, grow and go: along the tree lie exactly the requests with as many pages in common, and nothing stays behind."""
    rng = random.Random(seed)
    tree, there = PrefixTree(PS), {}
    texts = [[rng.randrange(3) for _ in range(80)] for _ in range(4)]
    texts += [t[:rng.randrange(80)] + [rng.randrange(3) for _ in range(40)] for t in texts for _ in range(3)]
    for turn in range(400):
        what = rng.random()
        if what < 0.35 or not there:
            r = request(turn, rng.choice(texts)[:rng.randint(1, 80)])
            there[turn] = r
            tree.add(r)
        elif what < 0.75:
            r = there[rng.choice(list(there))]
            more = rng.choice(texts)[r.length:r.length + rng.randint(1, 9)]
            for t in more:
                r.append(t)
            tree.add(r)
        else:
            tree.remove(rid := rng.choice(list(there)))
            del there[rid]
        asked = rng.choice(texts)[:rng.randint(1, 80)]
        pages = rng.randint(0, len(asked) // PS)
        path = tree.walk(asked, pages)
        assert [n for _, n in path] == sorted({n for _, n in path})
        found = {}
        for run, n in path:
            for rid in run.holders:
                found[rid] = n
        assert found == {rid: n for rid, r in there.items() if (n := alike(r.tokens, asked, pages)) > 0}
        assert len(tree) == len(there) and tree.num_runs() <= 2 * len(there)
    for rid in list(there):
        tree.remove(rid)
    assert len(tree) == 0 and tree.num_runs() == 0
    tree.remove("nobody")


def run_step(s, m):
    plan = s.schedule()
    for e in plan:
        r = e.request
        if not m.has_request(r.rid):
            m.admit(r.rid)
        assert m.extend(r.rid, e.start + e.num_tokens)
    s.update(plan, [(sum(map(int, e.request.tokens[-3:])) * 7 + e.request.length) % 50 for e in plan if e.sample])
    return plan


@pytest.mark.parametrize("seed", range(6))
def test_donors_are_those_of_comparing_every_pair(seed):
    """Over the steps of a scheduler with prompts that begin alike in several ways, portions, preemptions and requests that are given up: for every
    waiting request as many pages are found, and whether more are being computed, as by comparing it with every running one."""
    rng = random.Random(seed)
    m = CacheManager([CacheGroup(2, 16, 0, (0,))], PS, 60, 8)
    s = Scheduler(m, 12, 8, 200, share_prefixes=True)
    base = [rng.randrange(50) for _ in range(40)]
    for i in range(30):
        s.add_request(Request(i, base[:rng.randrange(1, 40)] + [rng.randrange(50) for _ in range(rng.randrange(1, 10))],
                              SamplingParams(max_new_tokens=rng.randrange(1, 20))))
    steps = 0
    while s.has_unfinished():
        steps += 1
        assert steps < 1000
        for r in s.waiting:
            donor, pages, more = s._donor(r)
            most = (r.length - 1) // PS
            have = {d.rid: min(alike(d.tokens, r.tokens, most), d.num_computed // PS) for d in s.running}
            assert pages == max(have.values(), default=0) and (pages == 0 if donor is None else have[donor.rid] == pages)
            assert more == any(d.remaining > 1 and alike(d.tokens, r.tokens, most) > pages for d in s.running)
        run_step(s, m)
        m.check_invariants()
        if rng.random() < 0.1 and s.running:
            s.abort(rng.choice(s.running).rid)
    assert len(s._prefixes) == 0 and s._prefixes.num_runs() == 0


def test_a_request_that_waits_for_pages_is_not_compared_again():
    """24 requests behind 400 common tokens decode, and one that begins with these too waits for pages: over 30 steps its tokens are compared once
    when it comes first, and again only when something has changed that could help it."""
    m = CacheManager([CacheGroup(2, 16, 0, (0,))], PS, 100 + 24 * 20, 40)
    s = Scheduler(m, 1 << 20, 40, 1 << 20, share_prefixes=True)
    common = list(range(400))
    for i in range(24):
        s.add_request(Request(i, [Token(t) for t in common] + [Token(i), Token(7)], SamplingParams(max_new_tokens=40 + i)))
    Token.compared = 0
    while len(s.running) < 24:
        run_step(s, m)
    assert Token.compared <= 24 * 3 * 402                    # each along the tree when it is looked for and when it is put there
    s.add_request(Request(99, [Token(t) for t in common] + [Token(t) for t in range(1840)], SamplingParams(max_new_tokens=5)))
    Token.compared = 0
    for _ in range(30):
        run_step(s, m)
        assert len(s.waiting) == 1
    assert 0 < Token.compared <= 2 * 402
    for _ in range(60):
        run_step(s, m)
    assert not s.waiting and s.num_shared_tokens == 24 * 400         # 23 of the 24, and the one that waited


def test_requests_that_ended_leave_the_tree():
    m = CacheManager([CacheGroup(2, 16, 0, (0,))], PS, 200, 8)
    s = Scheduler(m, 64, 8, 200, share_prefixes=True)
    a, b = request(0, range(20)), request(1, range(21))
    for r in (a, b):
        s.add_request(r)
    run_step(s, m)
    assert s.abort(0)
    run_step(s, m)
    assert b.status is Status.RUNNING and len(s._prefixes) == 1
    s.abort(1)
    assert len(s._prefixes) == 0 and s._prefixes.num_runs() == 0


def test_requests_are_themselves():
    """Searching the running requests looks at no tokens: two requests of the same content are two."""
    a, b = request(0, [Token(1)] * 5), request(0, [Token(1)] * 5)
    Token.compared = 0
    assert a != b and a in [b, a] and a not in [b] and len({a, b}) == 2
    assert Token.compared == 0


def test_requests_that_grow_alike_stay_one_run():
    tree = PrefixTree(PS)
    rs = [request(i, range(10)) for i in range(3)]
    for n in range(10, 400):
        for r in rs:
            tree.add(r)
            r.append(n)
        assert tree.num_runs() == 1
    rs[0].append(-1)
    for n in range(8):
        for r in rs:
            r.append(n)
            tree.add(r)
    assert tree.num_runs() == 3
    assert tree.walk(rs[1].tokens, 90)[-1][1] == 90
    tree.remove(0)
    assert tree.num_runs() == 1
