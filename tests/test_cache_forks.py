"""Forked requests and compaction in the cache manager's books (no GPU), and what the engine makes of them."""

import random

import pytest

from llm_pipeline_b200.cache import CacheError, CacheManager, KV8PagesSpec, KVPagesSpec, PagePool, StateSpec
from llm_pipeline_b200.engine.scheduler import Request, Scheduler
from llm_pipeline_b200.sampling import SamplingConfig


def manager(num_pages=32, page_size=4, max_requests=6, window=None, state=False):
    specs = [(KVPagesSpec(2, 8), None), (KV8PagesSpec(2, 16, window), None)] + ([(None, StateSpec((3,)))] if state else [])
    return CacheManager(specs, page_size=page_size, num_pages=num_pages, max_requests=max_requests, max_request_tokens=64)


def begin(m, rid, length):
    m.admit(rid)
    assert m.reserve(rid, length)
    m.commit(rid, length)


def test_a_shared_page_is_free_when_its_last_holder_frees_it():
    pool = PagePool(4)
    a = pool.alloc(2)
    pool.share(a)
    pool.free(a)
    assert pool.num_free == 2 and pool.holders(a[0]) == 1
    pool.free(a)
    assert pool.num_free == 4
    with pytest.raises(CacheError, match="freed twice"):
        pool.free(a)
    with pytest.raises(CacheError, match="shared"):
        pool.share([a[0]])
    with pytest.raises(CacheError, match="shared"):
        pool.share([4])


@pytest.mark.parametrize("length", [0, 3, 4, 9, 10])
def test_a_fork_shares_full_pages_and_owns_the_last(length):
    m = manager()
    begin(m, "a", 10)
    used = m.groups[0].pool.num_used
    assert m.fork("a", ["b", "c"], length)
    m.check()
    full, part = divmod(length, 4)
    for g in (0, 1):
        a, b, c = (m.block_table(r, g) for r in "abc")
        assert a[:full] == b[:full] == c[:full] and len(b) == len(c) == full + (part > 0)
        if part:
            assert len({a[full], b[full], c[full]}) == 3
    assert m.groups[0].pool.num_used == used + 2 * (part > 0)
    assert m.length("b") == length and m.admission("b") != m.admission("a")
    for rid, n in (("b", length + 9), ("a", 15), ("c", length + 1)):           # each grows into pages of its own
        assert m.reserve(rid, n)
        m.commit(rid, n)
        m.check()
    m.free("a")
    m.check()
    m.free("c")
    m.free("b")
    m.check()
    assert all(g.pool.num_free == 32 for g in m.groups) and m.free_slots == 6


def test_forks_are_all_or_nothing_and_checked():
    m = manager(num_pages=5, max_requests=4)
    begin(m, "a", 10)                                                          # three pages, two are left
    before = m.stats()
    assert not m.fork("a", ["b", "c", "d"])                                    # three copies of the last page are too many
    assert m.stats() == before
    assert m.fork("a", ["b", "c"])
    assert not m.fork("a", ["d"]) and not m.fork("a", ["d", "e"], 8)           # no page; no slots
    assert m.fork("a", ["d"], 8)
    m.check()
    with pytest.raises(CacheError, match="not live"):
        m.fork("x", ["y"])
    with pytest.raises(CacheError, match="holds 10 tokens"):
        m.fork("a", ["y"], 11)
    with pytest.raises(CacheError, match="new request ids"):
        m.fork("a", ["b"])
    with pytest.raises(CacheError, match="new request ids"):
        m.fork("a", ["y", "y"])
    assert m.fork("a", [])


def test_state_is_forked_at_its_length_alone():
    m = manager(state=True)
    begin(m, "a", 8)
    with pytest.raises(CacheError, match="state"):
        m.fork("a", ["b"], 7)
    assert m.fork("a", ["b"])


def test_a_window_that_has_moved_on_cannot_be_forked_before_it():
    m = manager(window=6)
    begin(m, "a", 20)
    assert m.block_table("a", 1)[:3] == [-1, -1, -1]
    assert m.fork("a", ["b"], 20) and m.block_table("b", 1)[:3] == [-1, -1, -1]
    assert not m.fork("a", ["c"], 14)
    m.check()
    assert m.reserve("b", 30)
    m.commit("b", 30)                                                          # b lets go of shared pages that a still sees
    m.check()
    assert all(p >= 0 for p in m.block_table("a", 1)[3:])


def test_compaction_moves_as_few_pages_as_it_can():
    m = manager(num_pages=16, max_requests=4)
    for rid in "abcd":
        begin(m, rid, 10)                                                      # three pages each
    m.fork("d", [])
    m.free("a")
    m.free("c")
    admitted = m.admission("b")
    assert m.compact() == 2 * 3                                                # d's pages, in both groups
    m.check()
    assert m.admission("b") != admitted
    for g in m.groups:
        held = sorted(p for t in g.tables.values() for p in t)
        assert held == list(range(6))
        assert g.pool.alloc(2) == [6, 7]
        g.pool.free([6, 7])
    assert m.compact() == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_orders_of_forks_and_compactions_keep_the_books(seed):
    rng = random.Random(seed)
    m = manager(num_pages=40, max_requests=8, window=9 if seed % 2 else None)
    live, next_id = {}, 0
    for _ in range(800):
        action = rng.random()
        if action < 0.2 and m.free_slots:
            m.admit(next_id)
            live[next_id] = 0
            next_id += 1
        elif action < 0.6 and live:
            rid = rng.choice(list(live))
            want = live[rid] + rng.choice([1, 1, 2, 7])
            if want <= 64 and m.reserve(rid, want):
                m.commit(rid, want)
                live[rid] = want
        elif action < 0.75 and live:
            rid = rng.choice(list(live))
            new = [next_id + k for k in range(rng.choice([1, 2]))]
            length = live[rid] if rng.random() < 0.5 else rng.randint(0, live[rid])
            if m.fork(rid, new, length):
                live.update({n: length for n in new})
                next_id += len(new)
        elif action < 0.8:
            m.compact()
            for g in m.groups:
                assert g.pool.num_used == 0 or max(p for t in g.tables.values() for p in t) < g.pool.num_used
        elif live:
            rid = rng.choice(list(live))
            m.free(rid)
            del live[rid]
        m.check()
        assert all(m.length(rid) == n for rid, n in live.items())
    for rid in list(live):
        m.free(rid)
    m.check()
    assert all(g.pool.num_free == 40 for g in m.groups)


def test_a_forked_request_runs_at_once():
    m = manager()
    s = Scheduler(m, 4, 64, 64)
    first = Request("a", list(range(9)), SamplingConfig(), 4)
    s.add(first)
    plan = s.schedule()
    assert m.admit("a") is not None and m.reserve("a", 9)
    m.commit("a", 9)
    s.finish_step(plan, {"a": 5})
    other = Request("b", list(range(9)), SamplingConfig(), 4)
    s.check(other)
    assert m.fork("a", ["b"], 8)
    s.add_forked(other, 8)
    plan = s.schedule()
    assert [(e.request.req_id, e.start, e.count, e.samples) for e in plan.entries] == [("a", 9, 1, True), ("b", 8, 1, True)]
    assert plan.entries[1].token_ids == [8]
