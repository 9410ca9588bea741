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
