"""Calls around 8-bit pages that one user makes beside another's: two streams, two graphs, pages with values that are no number."""

import pytest
import torch

from test_gpu_kv8 import DEV, prompt

pytestmark = pytest.mark.gpu


def portions(starts, lens, seed, direct, case=(32, 8, 128, 16)):
    """(the result of a call alone, a call without arguments that gives it again, its plan)"""
    from llm_pipeline_b200.ops import kv8

    nq, nkv, d, ps = case
    host, tables, ctx, q, want = prompt(case, starts, lens, 0, torch.bfloat16, seed, direct=direct)
    N = sum(lens)
    dev = [q.to(DEV), host.raw.to(DEV), tables.to(DEV),
           torch.tensor([sum(lens[:r]) for r in range(len(lens) + 1)], dtype=torch.int32, device=DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV)]
    plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, 0, torch.bfloat16, torch.device(DEV))
    plan._direct = direct

    def call():
        out = torch.empty(N, nq * d, dtype=torch.bfloat16, device=DEV)
        return kv8.prompt_attention(plan, dev[0], q.stride(0), out, dev[1], dev[2], dev[3], dev[4], d ** -0.5)

    return want[:N], call, plan


@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("how", ["streams", "graphs"])
def test_portions_whose_keys_are_shared_run_beside_one_another(direct, how):
    """Two callers, tiles whose keys come in parts, many calls side by side: each gets what a call alone gives."""
    sets = [portions([4000], [40], 97, direct), portions([4500, 0], [70, 30], 98, direct)]
    for _want, call, plan in sets:
        call()
        places = plan.items()[2] if direct else plan.lists(next(iter(plan._lists)))[0][6]
        assert places > 1
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs, graphs = [[], []], []
    if how == "graphs":
        for i, (_want, call, _plan) in enumerate(sets):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs[i].append(call())
            graphs.append(graph)
    for _ in range(30):
        for i, (_want, call, _plan) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                if how == "graphs":
                    graphs[i].replay()
                else:
                    outs[i].append(call())
    torch.cuda.synchronize()
    for (want, _call, _plan), got in zip(sets, outs):
        assert all(torch.equal(out, want) for out in got)


@pytest.mark.parametrize("length", [13, 16, 29, 40])
def test_a_fork_at_the_length_that_is_offered_holds_its_own_tokens_alone(length):
    """The parent's later tokens are a thousand times larger: the fork, once it has stored its tokens, holds what a request that never shared
    anything holds."""
    from llm_pipeline_b200.cache import CacheManager, KV8PagesSpec
    from llm_pipeline_b200.ops import kernels

    nkv, d, ps, N = 2, 32, 16, 40
    cache = CacheManager([(KV8PagesSpec(nkv, d), None)], page_size=ps, num_pages=16, max_requests=4, max_request_tokens=64, device=torch.device(DEV))
    pages = cache.pages_tensor(0)
    x = torch.randn(64, 2 * nkv * d, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)

    def store(rid, begin, end, factor=1.0):
        assert cache.reserve(rid, end)
        table = cache.block_table(rid, 0)
        slots = torch.tensor([table[t // ps] * ps + t % ps for t in range(begin, end)], dtype=torch.int32, device=DEV)
        rows = x[begin:end] * factor
        kernels.kv8_store(rows[:, :nkv * d], rows[:, nkv * d:], slots, pages, nkv, d, ps)
        cache.commit(rid, end)

    cache.admit("parent")
    store("parent", 0, length)
    if length < N:
        store("parent", length, N, 1000.0)
    at = cache.fork_length("parent", length)
    assert at == (length if length == N else length - length % ps) and cache.fork("parent", ["child"], at)
    cache.admit("alone")
    for rid, begin in (("child", at), ("alone", 0)):
        store(rid, begin, length)
        store(rid, length, length + 2)
    body = 2 * nkv * ps * d
    for n, (a, b) in enumerate(zip(cache.block_table("child", 0), cache.block_table("alone", 0))):
        one, other = pages[a], pages[b]
        assert torch.equal(one[body:body + 2 * nkv], other[body:body + 2 * nkv])
        there = min(ps, length + 2 - n * ps)
        assert torch.equal(one[:body].view(2 * nkv, ps, d)[:, :there], other[:body].view(2 * nkv, ps, d)[:, :there])


@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.09])
@pytest.mark.parametrize("starts,lens", [([300, 0], [40, 150]), ([4000], [9])])
def test_the_kernel_that_reads_pages_takes_scales_of_any_sign(scale, starts, lens):
    """Called by itself; over unpacked pages a scale has to be positive, so that a step's portions refuse others."""
    import kv8_plain as plain
    from llm_pipeline_b200.ops import kernels, kv8
    from test_gpu_kv8 import bound

    nq, nkv, d, ps = 32, 8, 128, 16
    host, tables, ctx, q, _out = prompt((nq, nkv, d, ps), starts, lens, 0, torch.bfloat16, 55)
    plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, 0, torch.bfloat16, torch.device(DEV))
    items, shared, places = plan.items()
    N = sum(lens)
    out = torch.full((N + 2, nq * d), 9.0, dtype=torch.bfloat16, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)               # noqa: E731
    start, ct = i32([sum(lens[:r]) for r in range(len(lens) + 1)]), i32(ctx)
    kernels.kv8_prompt_attention(q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV), start, ct, items, shared, places, nq, nkv, ps, 0, scale)
    at = 0
    for r, n in enumerate(lens):
        k, v, there = host.request(tables[r], ctx[r])
        for i in sorted({0, n // 2, n - 1}):
            seen = slice(0, starts[r] + i + 1)
            row = q[at + i:at + i + 1, :nq * d].view(1, nq, d)
            want, size, top = plain.attend(row, k[seen], v[seen], [starts[r] + i], there[seen], scale, 0)
            # (`smallest` as for single tokens: weights times the values' scales in half precision)
            allowed = bound(want, size, top.abs(), torch.bfloat16, d) + plain.smallest(row[0], k[seen], v[seen], host.value_scales(tables[r], ctx[r])[seen],
                                                                                      starts[r] + i, there[seen], scale, 0)
            assert bool(((out[at + i].double().cpu().view(1, nq, d) - want).abs() <= allowed).all()), (r, i)
        at += n
    assert bool((out[N:] == 9).all())


@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("nq,nkv,d,ps,starts,lens,window", [(8, 2, 128, 16, [200], [300], 150), (32, 8, 128, 16, [5000, 0], [40, 200], 0), (9, 1, 128, 64, [700], [70], 0),
                                                            (16, 8, 128, 8, [3000], [3], 2500), (8, 8, 128, 128, [0], [257], 0), (6, 2, 80, 8, [100], [200], 0),
                                                            (6, 3, 256, 16, [100], [40], 0), (4, 4, 16, 4, [90], [90], 60)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_value_that_is_no_number_reaches_the_rows_that_see_its_token(nq, nkv, d, ps, starts, lens, window, dtype, direct):
    """A NaN among a head's values makes the rows of its group that see the token no numbers, and leaves all others, those of earlier
    tokens and of later windows in the same call among them, as they are to the bit: in every kernel that portions may go to."""
    from llm_pipeline_b200.ops import kernels, kv8

    if direct and not kernels.kv8_prompt_supports(dtype, nq, nkv, d, ps):
        pytest.skip("no kernel reads these pages as they are")
    G = nq // nkv
    host, tables, ctx, q, clean = prompt((nq, nkv, d, ps), starts, lens, window, dtype, 83, direct=direct)
    end = ctx[0] - 1
    # (token, key/value head, column, byte): both signs, first and last columns, tokens of one page and far apart
    values = [(end - 2, 0, 7, 127), (end - 2, 0, d - 1, 255), (end - 33, nkv - 1, 0, 127), (max(end - 140, starts[0] + 1), nkv - 1, d // 2, 255)]
    for t, h, c, byte in values:
        host.q[int(tables[0, t // ps]), 1, h, t % ps, c] = byte
    want = torch.zeros(sum(lens) + 2, nq, dtype=torch.bool)
    for i in range(lens[0]):
        pos = starts[0] + i
        for t, h, _c, _byte in values:
            if t <= pos and (not window or t > pos - window):
                want[i, h * G:(h + 1) * G] = True
    out = torch.full_like(clean, 9.0)
    plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, window, dtype, torch.device(DEV))
    plan._direct = direct
    kv8.prompt_attention(plan, q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV),
                         torch.tensor([sum(lens[:r]) for r in range(len(lens) + 1)], dtype=torch.int32, device=DEV),
                         torch.tensor(ctx, dtype=torch.int32, device=DEV), d ** -0.5)
    got = out.view(-1, nq, d).cpu()
    assert bool(want.any()) and not bool(want[:lens[0]].all())
    assert torch.equal(got.isnan().all(-1), want)
    assert torch.equal(got[~want], clean.view(-1, nq, d).cpu()[~want])


@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("nq,nkv,d,ps,starts,lens", [(32, 8, 128, 16, [5000], [40]), (32, 8, 128, 16, [0, 100], [70, 5]), (6, 2, 80, 8, [100], [60]),
                                                     (6, 3, 256, 16, [100], [40])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_and_keys_that_are_no_numbers_do_not_come_out_as_zeros(nq, nkv, d, ps, starts, lens, dtype, direct):
    """A query with a NaN: its own row. A key with one: the rows that see it. Whatever else the row sees, nothing at all included."""
    from llm_pipeline_b200.ops import kernels, kv8

    if direct and not kernels.kv8_prompt_supports(dtype, nq, nkv, d, ps):
        pytest.skip("no kernel reads these pages as they are")
    G, N = nq // nkv, sum(lens)
    host, tables, ctx, q, clean = prompt((nq, nkv, d, ps), starts, lens, 0, dtype, 84, direct=direct)
    q[3, (nq - 1) * d + 5] = float("nan")
    q[N - 1, 2] = float("nan")
    token = starts[0] + 20 if starts[0] else 0                                   # the first token of all: its row sees nothing else
    host.q[int(tables[0, token // ps]), 0, 1, token % ps, d - 1] = 127
    want = torch.zeros(N + 2, nq, dtype=torch.bool)
    want[3, nq - 1] = want[N - 1, 0] = True
    for i in range(lens[0]):
        if starts[0] + i >= token:
            want[i, G:2 * G] = True
    out = torch.full_like(clean, 9.0)
    plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, 0, dtype, torch.device(DEV))
    plan._direct = direct
    kv8.prompt_attention(plan, q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV),
                         torch.tensor([sum(lens[:r]) for r in range(len(lens) + 1)], dtype=torch.int32, device=DEV),
                         torch.tensor(ctx, dtype=torch.int32, device=DEV), d ** -0.5)
    got = out.view(-1, nq, d).cpu()
    assert torch.equal(got.isnan().all(-1), want)
    assert torch.equal(got[~want], clean.view(-1, nq, d).cpu()[~want])


@pytest.mark.parametrize("nkv,d,ps", [(2, 128, 16), (3, 48, 24), (1, 256, 8), (8, 16, 4), (2, 80, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_storing_many_rows_of_ragged_portions(nkv, d, ps, dtype):
    """A thousand rows and more: portions that begin and end anywhere in a page and in a block's rows, single tokens between them, rows without a
    slot, first, last, inside runs and many of them together."""
    import kv8_plain as plain
    from llm_pipeline_b200.ops import kernels
    from test_gpu_kv8 import filled, same_bytes

    gen = torch.Generator().manual_seed(ps + d)
    pick = lambda low, high: int(torch.randint(low, high + 1, (1,), generator=gen))      # noqa: E731
    slots, page = [-1, -1], 0
    while len(slots) < 1300:
        kind, offset = pick(0, 5), pick(0, ps - 1)
        if kind == 0:
            slots += [-1] * pick(1, 40)
        elif kind == 1:
            slots.append(page * ps + offset)
            page += 1
        else:
            n = pick(1, 5 * ps)
            run = [page * ps + offset + i for i in range(n)]
            if kind == 2:
                run.insert(n // 2, -1)
            slots += run
            page = run[-1] // ps + 1
    slots += [-1] * 35
    host = filled(page + 1, nkv, ps, d, 6)
    pages = host.raw.to(DEV)
    x = (torch.randn(len(slots), 2 * nkv * d, generator=gen) * torch.exp(2.0 * torch.randn(len(slots), 1, generator=gen))).to(dtype)
    host.store(x[:, :nkv * d], x[:, nkv * d:], slots)
    on = x.to(DEV)
    kernels.kv8_store(on[:, :nkv * d], on[:, nkv * d:], torch.tensor(slots, dtype=torch.int32, device=DEV), pages, nkv, d, ps)
    same_bytes(pages, host.raw)
    assert plain.page_bytes(nkv, ps, d) == pages.shape[1]
