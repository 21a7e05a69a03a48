"""Pages held by several requests: the pool's and the manager's bookkeeping, the scheduler that hands them over, the step function's groups."""
import random

import pytest
import torch

from lucciola_b200.cache import CacheGroup, CacheManager, PagePool, PagePoolError
from lucciola_b200.config import EngineOptions
from lucciola_b200.engine.request import Request
from lucciola_b200.engine.scheduler import Scheduler
from lucciola_b200.engine.step import StepEntry
from lucciola_b200.sampling.params import SamplingParams
from test_step_packing import HostRunner, StandInModel
import test_step_packing as packing

PS = 4


def manager(pages=64, slots=8, groups=1):
    return CacheManager([CacheGroup(2, 16, 0, (g,)) for g in range(groups)], PS, pages, slots)


def test_a_page_goes_back_when_its_last_holder_gives_it_up():
    pool = PagePool(3)
    a = pool.allocate()
    pool.share(a)
    assert pool.holders(a) == 2
    pool.free(a)
    assert pool.num_free == 2
    pool.free(a)
    assert pool.num_free == 3
    with pytest.raises(PagePoolError):
        pool.free(a)
    with pytest.raises(PagePoolError):
        pool.share(a)
    with pytest.raises(PagePoolError):
        pool.share(7)


def test_pages_are_taken_over_and_given_back():
    m = manager(groups=2)
    m.admit("a")
    m.extend("a", 18)                                        # five pages, four of them full
    m.admit("b")
    m.share_prefix("b", "a", 4)
    assert m.length("b") == 16 and all(m.block_table("b", g) == m.block_table("a", g)[:4] for g in range(2))
    assert m.pages_needed("b", 19) == [1, 1]
    m.extend("b", 19)
    m.check_invariants()
    assert m.pools[0].num_held == 6
    m.release("a")
    m.check_invariants()
    assert m.pools[0].num_held == 5
    m.admit("c")
    m.share_prefix("c", "b", 4)
    m.release("b")
    m.release("c")
    m.check_invariants()
    assert m.pools[0].num_held == 0


def test_what_cannot_be_taken_over_is_refused():
    m = manager()
    m.admit("a")
    m.extend("a", 10)
    m.admit("b")
    for rid, donor, pages in (("b", "a", 3), ("b", "a", 0), ("a", "a", 1)):
        with pytest.raises(PagePoolError):
            m.share_prefix(rid, donor, pages)
    m.extend("b", 1)
    with pytest.raises(PagePoolError):
        m.share_prefix("b", "a", 1)
    w = CacheManager([CacheGroup(2, 16, 8, (0,))], PS, 8, 2)
    w.admit("a")
    w.extend("a", 8)
    w.admit("b")
    assert not w.can_share()
    with pytest.raises(PagePoolError):
        w.share_prefix("b", "a", 1)


def test_groups_of_a_step():
    m = manager(pages=200, slots=12)
    m.admit("a")
    m.extend("a", 41)                                        # ten full pages
    for rid, donor, pages in (("b", "a", 10), ("c", "b", 10), ("d", "a", 3), ("e", "d", 3)):
        m.admit(rid)
        m.share_prefix(rid, donor, pages)
        m.extend(rid, m.length(rid) + 5)
    m.admit("x")
    m.extend("x", 9)
    assert m.prefix_groups(["x", "a"]) is None
    assert m.prefix_groups(["x", "b", "a"]) == ([-1, 1, 1], [0, 40, 0])
    assert m.prefix_groups(["d", "x", "e"]) == ([0, -1, 0], [12, 0, 0])
    assert m.prefix_groups(["a", "b", "c", "d", "e"]) == ([0, 0, 0, -1, -1], [40, 0, 0, 0, 0])      # 3 x 10 pages are more than 5 x 3
    assert m.prefix_groups(["b", "d"]) == ([0, 0], [12, 0])
    m.release("a")
    assert m.prefix_groups(["c", "b"]) == ([0, 0], [40, 0])
    assert m.prefix_groups([]) is None


def test_groups_name_pages_that_their_members_really_share():
    """Random families: every member's table begins with the pages that the group's row stands for, and its tokens lie behind them."""
    rng = random.Random(3)
    for _ in range(200):
        m = manager(pages=500, slots=16)
        alive = []
        for i in range(16):
            m.admit(i)
            if alive and rng.random() < 0.8:
                donor = rng.choice(alive)
                full = m.length(donor) // PS
                if full:
                    m.share_prefix(i, donor, rng.randint(1, full))
            m.extend(i, m.length(i) + rng.randint(1, 30))
            alive.append(i)
            if rng.random() < 0.2:
                m.release(alive.pop(rng.randrange(len(alive))))
        m.check_invariants()
        rng.shuffle(alive)
        groups = m.prefix_groups(alive)
        if groups is None:
            continue
        for i, leader in enumerate(groups[0]):
            if leader >= 0:
                n = groups[1][leader] // PS
                assert groups[0][leader] == leader and n > 0
                assert m.block_table(alive[i], 0)[:n] == m.block_table(alive[leader], 0)[:n]
                assert m.length(alive[i]) >= n * PS


def drive(s, m, steps=200):
    """Runs the scheduler as the engine does; the next token is a function of the tokens so far.  Checks what each step computes."""
    computed = 0
    while s.has_unfinished() and steps:
        steps -= 1
        plan = s.schedule()
        for e in plan:
            r = e.request
            if not m.has_request(r.rid):
                m.admit(r.rid)
            assert m.length(r.rid) == e.start == r.num_computed
            assert m.extend(r.rid, e.start + e.num_tokens)
            computed += e.num_tokens
        m.check_invariants()
        s.update(plan, [(sum(e.request.tokens) * 7 + len(e.request.tokens)) % 50 for e in plan if e.sample])
    assert not s.has_unfinished()
    assert m.pools[0].num_held == 0
    return computed


@pytest.mark.parametrize("pages", [200, 30])
def test_the_scheduler_computes_a_common_beginning_once(pages):
    """Eight answers to one prompt of 21 tokens, and two prompts that begin with half of it: the prompt is computed once, and the
    tokens are those of requests that share nothing, preemptions or not."""
    prompt = list(range(100, 121))
    prompts = [prompt] * 8 + [prompt[:10] + [7, 8, 9], prompt[:10] + [3]]

    def run(share):
        m = manager(pages=pages, slots=12)
        s = Scheduler(m, 64, 12, 200, share_prefixes=share)
        reqs = [Request(i, list(p), SamplingParams(max_new_tokens=12)) for i, p in enumerate(prompts)]
        for r in reqs:
            s.add_request(r)
        n = drive(s, m)
        return [r.output for r in reqs], n, s
    plain, n_plain, _ = run(False)
    shared, n_shared, s = run(True)
    assert shared == plain
    if pages == 200:
        assert s.num_shared_tokens == 7 * 20 + 2 * 8 and n_shared == n_plain - s.num_shared_tokens
        assert s.num_preemptions == 0
    else:
        assert n_shared < n_plain


def test_a_request_waits_for_a_beginning_that_is_being_computed():
    m = manager(slots=4)
    s = Scheduler(m, 8, 4, 200, share_prefixes=True)
    prompt = list(range(1, 30))
    for i in range(2):
        s.add_request(Request(i, list(prompt), SamplingParams(max_new_tokens=2)))
    seen = []
    for _ in range(5):
        plan = s.schedule()
        seen.append([(e.request.rid, e.start, e.num_tokens) for e in plan])
        for e in plan:
            if not m.has_request(e.request.rid):
                m.admit(e.request.rid)
            m.extend(e.request.rid, e.start + e.num_tokens)
        s.update(plan, [5] * sum(e.sample for e in plan))
    assert seen == [[(0, 0, 8)], [(0, 8, 8)], [(0, 16, 8)], [(0, 24, 5)], [(0, 29, 1), (1, 28, 1)]]


def test_others_pass_a_request_that_waits_for_a_beginning():
    """Behind a request that waits for a prompt that is being computed stand one that waits for the same and two that share nothing: these
    start at once, and the waiting ones as soon as the beginning is there."""
    m = manager(pages=200, slots=8)
    s = Scheduler(m, 16, 8, 200, prefill_chunk=8, share_prefixes=True)
    prompt = list(range(1, 30))
    for i, p in enumerate([prompt, prompt, [60, 61, 62], prompt[:25], [70, 71]]):
        s.add_request(Request(i, list(p), SamplingParams(max_new_tokens=9)))
    seen = []
    for _ in range(6):
        plan = s.schedule()
        seen.append([(e.request.rid, e.start, e.num_tokens) for e in plan])
        for e in plan:
            if not m.has_request(e.request.rid):
                m.admit(e.request.rid)
            m.extend(e.request.rid, e.start + e.num_tokens)
        s.update(plan, [5] * sum(e.sample for e in plan))
    assert seen[0] == [(0, 0, 8), (2, 0, 3), (4, 0, 2)]
    assert seen[1] == [(2, 3, 1), (4, 2, 1), (0, 8, 8)]
    assert seen[3] == [(2, 5, 1), (4, 4, 1), (0, 24, 5), (3, 24, 1)]         # what 3 waits for is there; 1 waits for one page more
    assert seen[4] == [(0, 29, 1), (2, 6, 1), (4, 5, 1), (3, 25, 1), (1, 28, 1)]


def test_many_that_wait_are_not_looked_for_in_every_step(monkeypatch):
    """A hundred requests that wait for the same prompt: each is looked for once while it is computed, a few a step."""
    m = manager(pages=400, slots=200)
    s = Scheduler(m, 4, 200, 200, share_prefixes=True)
    looked = []
    donor = Scheduler._donor
    monkeypatch.setattr(Scheduler, "_donor", lambda self, r: looked.append(r.rid) or donor(self, r))
    for i in range(100):
        s.add_request(Request(i, list(range(60)), SamplingParams(max_new_tokens=2)))
    steps = 0
    while s.running[0].num_computed < 56 if s.running else True:
        run = s.schedule()
        steps += 1
        assert [e.request.rid for e in run] == [0]
        for e in run:
            if not m.has_request(0):
                m.admit(0)
            m.extend(0, e.start + e.num_tokens)
        s.update(run, [])
    assert len(looked) == len(set(looked)) <= 8 * steps
    assert s.abort(99) and 99 not in s._awaited
    n = drive_on(s, m)
    assert n == 100 - 1


def drive_on(s, m):
    """To the end, with token 5 every time; how many requests ended."""
    ended = 0
    while s.has_unfinished():
        plan = s.schedule()
        for e in plan:
            if not m.has_request(e.request.rid):
                m.admit(e.request.rid)
            assert m.extend(e.request.rid, e.start + e.num_tokens)
        ended += sum(done for _, _, done in s.update(plan, [5] * sum(e.sample for e in plan)))
        m.check_invariants()
    assert not s._awaited
    return ended


def test_the_last_token_of_a_prompt_is_always_computed():
    m = manager()
    s = Scheduler(m, 64, 4, 200, share_prefixes=True)
    prompt = list(range(8))                                  # two whole pages
    s.add_request(Request(0, list(prompt), SamplingParams(max_new_tokens=4)))
    plan = s.schedule()
    m.admit(0)
    m.extend(0, 8)
    s.update(plan, [9])
    s.add_request(Request(1, list(prompt), SamplingParams(max_new_tokens=4)))
    plan = s.schedule()
    assert [(e.request.rid, e.start, e.num_tokens) for e in plan] == [(0, 8, 1), (1, 4, 4)]


class SharingModel(StandInModel):
    """Also hands out what the step says of its groups."""
    def forward(self, tok, step, caches, rows):
        out = super().forward(tok, step, caches, rows)
        self.groups = None if step.prefix_of is None else (step.prefix_of.tolist(), step.prefix_lens.tolist())
        return out


def runner(monkeypatch, **kw):
    monkeypatch.setattr(packing.step_mod, "_Staging", packing.HostStaging)
    from lucciola_b200.parts.base import Runtime
    monkeypatch.setattr(packing.step_mod, "DeviceCache", lambda *a, **k: type("C", (), {"states": {}, "views": []})())
    rt = Runtime("cpu", torch.bfloat16)
    return HostRunner(SharingModel(), rt, EngineOptions(max_blocks=100, max_num_seqs=8, use_cuda_graph=kw.pop("graph", False), share_prefixes=True, **kw))


def test_the_step_function_names_the_groups(monkeypatch):
    r = runner(monkeypatch)
    monkeypatch.setattr(packing.step_mod, "SHARED_ELEMENTS", 0)
    r.step([StepEntry("a", list(range(40)), (39,))])
    assert r.model.groups is None
    r.manager.admit("b")
    r.manager.share_prefix("b", "a", 2)
    r.step([StepEntry("x", [1, 2], (1,)), StepEntry("a", [5], (0,)), StepEntry("b", [1, 2, 3], (2,))])
    assert r.model.groups == ([-1, 1, 1], [0, 32, 0])
    r.step([StepEntry("b", [5], (0,))])
    assert r.model.groups is None


def test_recordings_of_steps_with_groups(monkeypatch):
    """A step with groups is recorded apart from one without, and a replay reads this step's groups; entries that pad belong to none."""
    r = runner(monkeypatch, graph=True)
    monkeypatch.setattr(packing.step_mod, "SHARED_ELEMENTS", 0)
    r.step([StepEntry("a", list(range(40)), (39,))])
    for rid in "bcde":
        r.manager.admit(rid)
        r.manager.share_prefix(rid, "a", 2)
        r.step([StepEntry(rid, [1, 2], (1,))])
    r.step([StepEntry(i, [3], (0,)) for i in "abc"])
    assert r.model.groups == ([0, 0, 0, -1], [32, 0, 0, 0])
    r.step([StepEntry("x", [3, 4], (1,))])
    before = r.graph_replays
    r.step([StepEntry(i, [3], (0,)) for i in ("x", "d", "b")])
    assert r.graph_replays == before + 1
    assert r.model.groups == ([-1, 1, 1, -1], [0, 32, 0, 0])
    assert sorted(len(k) for k in r._graphs if k[0] == 4) == [5]
    r.step([StepEntry(i, [3], (0,)) for i in ("x", "d")])
    assert r.model.groups is None


def test_models_that_keep_more_than_all_keys_refuse(monkeypatch):
    from lucciola_b200.parts.base import Runtime
    monkeypatch.setattr(packing.step_mod, "_Staging", packing.HostStaging)
    monkeypatch.setattr(packing.step_mod, "DeviceCache", lambda *a, **k: type("C", (), {"states": {}, "views": []})())
    with pytest.raises(ValueError, match="share_prefixes"):
        HostRunner(StandInModel(state=True), Runtime("cpu", torch.bfloat16), EngineOptions(max_blocks=10, max_num_seqs=2, share_prefixes=True))


def test_elements_that_groups_spare():
    from lucciola_b200.engine.step import _elements_saved
    assert _elements_saved([0, 0, -1, 3, 0, 3], [32, 0, 0, 16, 0, 0], 10) == (2 * 32 + 1 * 16) * 10
    assert _elements_saved([-1, -1], [0, 0], 10) == 0


def documents(m, first, docs, pages, each):
    """`docs` documents of `pages` pages that begin with the same `first` pages, `each` requests behind every one: (rid, document)."""
    out = []
    for d in range(docs):
        for i in range(each):
            rid = (d, i)
            m.admit(rid)
            if i:
                m.share_prefix(rid, (d, 0), pages)
            elif d and first:
                m.share_prefix(rid, (0, 0), first)
            m.extend(rid, pages * PS + 1 + i)
            out.append((rid, d))
    return out


@pytest.mark.parametrize("first", [0, 1, 4, 16, 50])
def test_documents_behind_a_common_beginning(first):
    """Requests on several long documents, all of which begin with the same system prompt: a group for every document, with all that its
    requests have in common."""
    m = manager(pages=4000, slots=40)
    rids = documents(m, first, 4, 64, 8)
    random.Random(first).shuffle(rids)
    of, lens = m.prefix_groups([r for r, _ in rids])
    for i, (_, d) in enumerate(rids):
        leader = of[i]
        assert leader >= 0 and rids[leader][1] == d and lens[leader] == 64 * PS
    assert sum(n > 0 for n in lens) == 4
    m.release((2, 0))
    of, lens = m.prefix_groups([r for r, _ in rids if r != (2, 0)])
    assert sorted(lens)[-4:] == [64 * PS] * 4 and of.count(-1) == 0


def test_what_deeper_groups_leave_over():
    """Two requests on a document each and six more behind the system prompt alone: these share the system prompt, if it is a block long."""
    for first, grouped in ((20, True), (15, False)):
        m = manager(pages=4000, slots=40)
        rids = [r for r, _ in documents(m, first, 2, 200, 2)]
        for i in range(6):
            m.admit(i)
            m.share_prefix(i, (0, 0), first)
            m.extend(i, first * PS + 3)
            rids.append(i)
        of, lens = m.prefix_groups(rids)
        assert of == [0, 0, 2, 2] + ([4] * 6 if grouped else [-1] * 6)
        assert lens == [200 * PS, 0, 200 * PS, 0] + ([first * PS] if grouped else [0]) + [0] * 5


def spared(m, rids, groups):
    of, lens = groups
    return sum((of.count(r) - 1) * n for r, n in enumerate(lens) if n)


def test_groups_of_nested_families():
    """Random trees of shared beginnings: groups name pages that their members share, and spare no less than one group of the best length would;
    the answer is the same when it is asked for again, and follows requests that end."""
    rng = random.Random(11)
    for turn in range(150):
        m = CacheManager([CacheGroup(2, 16, 0, (0,))], PS, 3000, 24)
        alive = []
        for i in range(24):
            m.admit(i)
            if alive and rng.random() < 0.85:
                donor = rng.choice(alive)
                full = m.length(donor) // PS
                m.share_prefix(i, donor, rng.choice([full, max(1, full // 2), rng.randint(1, full)]))
            m.extend(i, m.length(i) + rng.choice([rng.randint(PS, 30), rng.randint(100, 300)]))
            alive.append(i)
            if rng.random() < 0.1:
                m.release(alive.pop(rng.randrange(len(alive))))
            if rng.random() < 0.3:
                m.prefix_groups(alive)
        rng.shuffle(alive)
        groups = m.prefix_groups(alive)
        tables = [m.block_table(i, 0) for i in alive]
        one = 0
        for t in tables:
            for n in range(1, len(t) + 1):
                k = sum(u[:n] == t[:n] for u in tables)
                if k > 1:
                    one = max(one, (k - 1) * n * PS)
        assert (groups is None) == (one == 0)
        if groups is None:
            continue
        assert spared(m, alive, groups) >= one
        assert m.prefix_groups(list(alive)) == groups
        for i, leader in enumerate(groups[0]):
            if leader >= 0:
                n = groups[1][leader] // PS
                assert groups[0][leader] == leader and n > 0 and tables[i][:n] == tables[leader][:n]
                assert min(j for j, x in enumerate(groups[0]) if x == leader) == leader


@pytest.mark.parametrize("groups,members,prefix,heads,dim,single,faster", [
    # what was measured, see SHARED_ELEMENTS
    (1, 4, 2048, 8, 128, True, False), (1, 4, 4096, 8, 128, True, True), (1, 16, 512, 8, 128, True, False), (1, 16, 1024, 8, 128, True, True),
    (1, 32, 512, 8, 128, True, False), (1, 32, 1024, 8, 128, True, True), (1, 64, 512, 8, 128, True, True), (1, 32, 512, 8, 128, False, True),
    (16, 2, 1024, 8, 128, True, False), (16, 2, 2048, 8, 128, True, True), (8, 8, 256, 8, 128, True, False), (8, 8, 512, 8, 128, True, True),
    (128, 2, 512, 8, 128, True, False), (128, 2, 1024, 8, 128, True, True), (128, 2, 256, 16, 128, True, False), (16, 2, 1024, 8, 64, True, False),
    (16, 2, 4096, 8, 64, True, True), (1, 2, 8192, 8, 128, True, False)])
def test_steps_take_the_faster_way(groups, members, prefix, heads, dim, single, faster):
    from lucciola_b200.engine import step
    of = [s // members * members for s in range(groups * members)]
    lens = [0 if s % members else prefix for s in range(groups * members)]
    assert step._worth_sharing(of, lens, heads, heads * dim, single) == faster


def test_the_runner_asks_which_way_is_faster(monkeypatch):
    r = runner(monkeypatch)
    asked = []
    monkeypatch.setattr(packing.step_mod, "_worth_sharing", lambda *a: asked.append(a) or len(asked) > 1)
    r.rt.fast_kernels = True
    r.step([StepEntry("a", list(range(40)), (39,))])
    r.manager.admit("b")
    r.manager.share_prefix("b", "a", 2)
    r.step([StepEntry("b", [1, 2], (1,)), StepEntry("a", [3], (0,))])
    assert r.model.groups is None
    r.step([StepEntry("a", [3], (0,)), StepEntry("b", [1], (0,))])
    assert r.model.groups == ([0, 0], [32, 0])
    heads = r.groups[0].num_kv_heads
    assert asked == [([0, 0], [32, 0], heads, heads * r.groups[0].head_dim, False), ([0, 0], [32, 0], heads, heads * r.groups[0].head_dim, True)]
