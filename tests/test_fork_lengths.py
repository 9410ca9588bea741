"""Up to where the engine shares a prompt with those that wait for it (the books alone, no GPU)."""

from types import SimpleNamespace

import pytest

from llm_pipeline_b200.cache import CacheManager, KV8PagesSpec, KVPagesSpec
from llm_pipeline_b200.engine.generate import GenerationEngine
from llm_pipeline_b200.engine.scheduler import Scheduler, StepPlan
from llm_pipeline_b200.sampling import SamplingConfig


def engine(specs, num_pages=64, page_size=4, max_seqs=8, budget=64):
    e = object.__new__(GenerationEngine)
    e.cache = CacheManager([(s, None) for s in specs], page_size=page_size, num_pages=num_pages, max_requests=max_seqs, max_request_tokens=128)
    e.scheduler = Scheduler(e.cache, max_seqs, budget, 128)
    e.model, e.config = SimpleNamespace(spec=SimpleNamespace(vocab_size=1000)), None
    e.runner, e.sampler = SimpleNamespace(position_streams=1), SimpleNamespace(config=SamplingConfig())
    e._requests, e._forks = {}, {}
    return e


def step(e):
    """What the engine does around a plan, with a scripted token for every request that samples."""
    plan = e.scheduler.schedule()
    for r in plan.aborted:
        e._unfork(r)
    for entry in plan.entries:
        rid = entry.request.req_id
        if rid not in e.cache:
            e.cache.admit(rid)
        assert entry.start == e.cache.length(rid) and e.cache.reserve(rid, entry.start + entry.count)
        e.cache.commit(rid, entry.start + entry.count)
    if e._forks:
        e._fork(plan)
    e.scheduler.finish_step(plan, {x.request.req_id: 7 for x in plan.entries if x.samples})
    e.cache.check()
    return {x.request.req_id: (x.start, x.count) for x in plan.entries}


BF16, EIGHT = [KVPagesSpec(2, 16)], [KV8PagesSpec(2, 16)]


@pytest.mark.parametrize("specs", [BF16, EIGHT, BF16 + EIGHT])
@pytest.mark.parametrize("prompt", [2, 4, 5, 22])
def test_a_prompt_that_ends_with_its_request_is_shared_but_for_its_last_token(specs, prompt):
    e = engine(specs)
    e.add_request(range(prompt), 9, req_id="a")
    e.add_request(range(prompt), 9, req_id="b", same_prompt_as="a")
    assert step(e) == {"a": (0, prompt)}
    assert step(e) == {"a": (prompt, 1), "b": (prompt - 1, 1)}


@pytest.mark.parametrize("specs,shared", [(BF16, 21), (EIGHT, 20), (BF16 + EIGHT, 20)])
def test_what_a_preempted_request_has_sampled_is_not_in_what_it_shares(specs, shared):
    """A request that is read again after a preemption brings its prompt and what it has sampled in one portion. In 8 bits the page in which
    the prompt ends then has a scale, and values, that follow the sampled tokens: it is not shared."""
    e = engine(specs)
    e.add_request(range(22), 9, req_id="a")
    for _ in range(3):
        step(e)
    assert len(e._requests["a"].output) == 3
    e.scheduler._preempt_last(StepPlan())
    e.add_request(range(22), 9, req_id="b", same_prompt_as="a")
    assert step(e) == {"a": (0, 25)}
    assert e.cache.length("b") == shared
    assert step(e) == {"a": (25, 1), "b": (shared, 22 - shared)}
    while e.scheduler.has_unfinished():
        step(e)
    assert e._requests["b"].output == [7] * 9 and e.cache.num_live == 0


def test_a_short_prompt_of_a_preempted_request_is_computed_again():
    e = engine(EIGHT)
    e.add_request(range(3), 9, req_id="a")
    step(e), step(e)
    e.scheduler._preempt_last(StepPlan())
    e.add_request(range(3), 9, req_id="b", same_prompt_as="a")
    assert step(e) == {"a": (0, 5)}
    assert step(e) == {"a": (5, 1), "b": (0, 3)}


@pytest.mark.parametrize("specs", [BF16, EIGHT])
def test_as_many_share_a_prompt_as_there_are_pages_for(specs):
    """22 tokens are six pages, two tokens of the last. Six free pages are not enough for seven copies of that page: six requests share."""
    e = engine(specs, num_pages=12)
    e.add_request(range(22), 3, req_id="a")
    for i in range(7):
        e.add_request(range(22), 3, req_id=i, same_prompt_as="a")
    assert step(e) == {"a": (0, 22)}
    shared = [i for i in range(7) if i in e.cache]
    assert shared == [0, 1, 2, 3, 4, 5] and e.cache.groups[0].pool.num_free == 0
    computed = 22 + sum(n for _s, n in step(e).values())
    while e.scheduler.has_unfinished():
        computed += sum(n for _s, n in step(e).values())
    assert all(r.output == [7] * 3 for r in e._requests.values()) and e.cache.num_live == 0 and not e._forks
    assert computed < 4 * 22


def test_none_share_where_no_page_is_left():
    e = engine(EIGHT, num_pages=6)
    e.add_request(range(22), 2, req_id="a")
    e.add_request(range(22), 2, req_id="b", same_prompt_as="a")
    assert step(e) == {"a": (0, 22)}
    assert "b" not in e.cache
    while e.scheduler.has_unfinished():
        step(e)
    assert e._requests["b"].output == [7, 7] and e.cache.num_live == 0


def test_requests_that_wait_for_a_prompt_are_counted_as_waiting():
    e = engine(EIGHT, budget=8)
    e.steps = e.tokens_prefilled = e.tokens_decoded = 0
    e.runner.kernel_times = None
    e.add_request(range(22), 2, req_id="a")
    for i in range(3):
        e.add_request(range(22), 2, req_id=i, same_prompt_as="a")
    assert e.stats()["waiting"] == 4
    step(e)
    assert (e.stats()["waiting"], e.stats()["running"]) == (3, 1)
    step(e), step(e)
    assert (e.stats()["waiting"], e.stats()["running"]) == (0, 4)
