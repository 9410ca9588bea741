"""What the calls around 8-bit keys and values and copies of pages refuse, without a GPU: every check is made before anything is
launched, so tensors on the CPU reach it."""

import pytest
import torch

import kv8_plain as plain
from llm_pipeline_b200.cache import KV8PagesSpec, KVPagesSpec
from llm_pipeline_b200.ops import kernels, kv8

NKV, D, PS = 2, 32, 8


def pages(n=4, nkv=NKV, ps=PS, d=D):
    return torch.zeros(n, plain.page_bytes(nkv, ps, d), dtype=torch.uint8)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


STORE = dict(k=torch.zeros(3, NKV * D), v=torch.zeros(3, NKV * D), slots=i32(0, 1, 2), pages=pages(), num_kv_heads=NKV, head_dim=D, page_size=PS)


@pytest.mark.parametrize("change,message", [
    (dict(pages=pages().to(torch.int8)), "uint8"), (dict(pages=pages(ps=16)), "uint8"), (dict(pages=pages()[:, ::2]), "uint8"), (dict(pages=pages(0)), "uint8"),
    (dict(head_dim=24), "multiples of 16"), (dict(num_kv_heads=0), "at least one head"), (dict(page_size=0), "at least one head"),
    (dict(k=torch.zeros(2, NKV * D)), "one row per slot"), (dict(k=torch.zeros(3, NKV * D).bfloat16()), "one type"),
    (dict(k=torch.zeros(NKV * D, 3).t()), "neighbours"), (dict(v=torch.zeros(3, NKV * D + 1)), "one row per slot"), (dict(slots=torch.arange(3)), "int32"),
    (dict(k=torch.zeros(3, NKV * D).half(), v=torch.zeros(3, NKV * D).half()), "float32 and bfloat16"), ({}, "not on a CUDA device"),
])
def test_store(change, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.kv8_store(**{**STORE, **change})


GATHER = dict(pages=pages(), block_tables=torch.zeros(2, 3, dtype=torch.int32), ctx_len=i32(5, 6), index=i32(0, 1), out=torch.zeros(2, 2, NKV, PS, D))


@pytest.mark.parametrize("change,message", [
    (dict(out=torch.zeros(3, 2, NKV, PS, D)), "one index"), (dict(out=torch.zeros(2, 2, NKV, PS, 16)), "uint8"), (dict(ctx_len=i32(5)), "requests"),
    (dict(index=torch.zeros(2)), "int32"), (dict(out=torch.zeros(2, 2, NKV, PS, D).half()), "float32 and bfloat16"),
    (dict(out=torch.zeros(2, 2, NKV, D, PS).transpose(3, 4)), "contiguous"), ({}, "not on a CUDA device"),
])
def test_gather(change, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.kv8_gather(**{**GATHER, **change})


DECODE = dict(q=torch.zeros(2, 4 * D), q_stride=4 * D, out=torch.zeros(2, 4 * D), pages=pages(), block_tables=torch.zeros(2, 3, dtype=torch.int32),
              ctx_len=i32(5, 6), max_ctx=24, num_heads=4, num_kv_heads=NKV, head_dim=D, page_size=PS, window=0, scale=1.0)


@pytest.mark.parametrize("change,message", [
    (dict(num_heads=3), "cannot share"), (dict(q=torch.zeros(1, 4 * D)), "query rows"), (dict(q=torch.zeros(2, 4 * D).bfloat16()), "query rows"),
    (dict(q_stride=7), "query rows"), (dict(out=torch.zeros(2, 5 * D)), "decode output"), (dict(block_tables=torch.zeros(1, 3, dtype=torch.int32)), "block tables"),
    (dict(max_ctx=0), "positive"), (dict(window=-1), "negative"), (dict(ctx_len=torch.zeros(2)), "int32"), (dict(pages=pages(d=48)), "uint8"),
])
def test_decode(change, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.kv8_decode_attention(**{**DECODE, **change})


@pytest.mark.parametrize("tensors,src,dst,message", [
    ([torch.zeros(4, 3)], [0], [1, 2], "as many"), ([torch.zeros(4, 3)], [0], [4], "outside"), ([torch.zeros(4, 3)], [-1], [0], "outside"),
    ([torch.zeros(4, 3)], [0, 1], [2, 2], "twice"), ([torch.zeros(4, 3)], [0, 1], [1, 2], "twice"), ([torch.zeros(4, 3), torch.zeros(4, 2)], [0], [1], "one page size"),
    ([torch.zeros(4, 3), torch.zeros(4, 3).half()], [0], [1], "one type"), ([torch.zeros(4, 6)[:, ::2]], [0], [1], "contiguous"),
    ([torch.zeros(4, 3), torch.zeros(3, 3)], [3], [1], "outside"), ([torch.zeros(4, 3)], [0], [1], "not on a CUDA device"),
])
def test_copy_pages(tensors, src, dst, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.copy_pages(tensors, src, dst)


def test_copy_pages_of_many():
    t = torch.zeros(400, 3)
    for src, dst, message in (([0] * 100, list(range(1, 100)) + [400], "outside"), ([0] * 100, [-1] + list(range(1, 100)), "outside"),
                              ([0] * 100, [5] * 2 + list(range(6, 104)), "twice"), (list(range(100)), list(range(99, 199)), "twice"),
                              (list(range(100)), list(range(100, 200)), "not on a CUDA device")):
        with pytest.raises(kernels.KernelError, match=message):
            kernels.copy_pages([t], src, dst)


def test_nothing_to_copy():
    kernels.copy_pages([], [1], [2])
    kernels.copy_pages([torch.zeros(4, 3)], [], [])


def test_plans():
    make = lambda starts, lens, **kw: kv8.PromptPlan(starts, lens, 4, NKV, D, kw.pop("ps", PS), kw.pop("window", 0), torch.float32, torch.device("cpu"), **kw)  # noqa: E731
    for bad in (lambda: make([1], [1, 2]), lambda: make([-1], [1]), lambda: make([1], [-1]), lambda: make([1], [1], ps=0), lambda: make([1], [1], window=-1),
                lambda: make([1], [1], first_request=2)):
        with pytest.raises(kernels.KernelError):
            bad()
    plan = make([100, 0, 7], [20, 0, 1], window=30)
    assert plan.groups == [[0, 2]] and plan.pages_of(0) == (8, 15) and plan.pages_of(2) == (0, 1)
    assert make([100, 3], [20, 1], first_request=1).groups == [[1]]
    with pytest.raises(kernels.KernelError, match="plan is for queries"):
        kv8.prompt_attention(plan, torch.zeros(21, 4 * D).bfloat16(), 4 * D, torch.zeros(21, 4 * D), pages(), torch.zeros(3, 15, dtype=torch.int32), i32(0, 20, 20, 21),
                             i32(120, 0, 8), 1.0)
    with pytest.raises(kernels.KernelError, match="plan's requests"):
        kv8.prompt_attention(plan, torch.zeros(21, 4 * D), 4 * D, torch.zeros(21, 4 * D), pages(), torch.zeros(2, 15, dtype=torch.int32), i32(0, 20, 20, 21),
                             i32(120, 0, 8), 1.0)
    with pytest.raises(kernels.KernelError, match="more rows"):
        kv8.prompt_attention(plan, torch.zeros(20, 4 * D), 4 * D, torch.zeros(21, 4 * D), pages(), torch.zeros(3, 15, dtype=torch.int32), i32(0, 20, 20, 21),
                             i32(120, 0, 8), 1.0)
    for scale in (0.0, -0.5, float("nan"), float("inf")):
        with pytest.raises(kernels.KernelError, match="positive and finite"):
            kv8.prompt_attention(plan, torch.zeros(21, 4 * D), 4 * D, torch.zeros(21, 4 * D), pages(), torch.zeros(3, 15, dtype=torch.int32),
                                 i32(0, 20, 20, 21), i32(120, 0, 8), scale)


def test_the_workspace_holds_a_few_requests_at_a_time(monkeypatch):
    monkeypatch.setattr(kv8, "WORKSPACE_BYTES", 3 * 2 * NKV * PS * D * 4)
    plan = kv8.PromptPlan([0, 0, 0, 40, 0], [8, 16, 1, 8, 3], 4, NKV, D, PS, 0, torch.float32, torch.device("cpu"))
    assert plan.groups == [[0, 1], [2], [3], [4]]


def test_specs():
    spec = KV8PagesSpec(8, 128)
    assert spec.page_shape(16) == (32896,) and spec.bytes_per_page(16, torch.bfloat16) == 32896 and spec.dtype == torch.uint8
    assert KVPagesSpec(8, 128).bytes_per_page(16, torch.bfloat16) == 65536
    assert spec.group_key() != KVPagesSpec(8, 128).group_key() and spec.group_key() != KV8PagesSpec(8, 128, 4096).group_key()
    assert spec.bytes_per_token(torch.bfloat16) == 2048


def test_models():
    from llm_pipeline_b200.config import resolve_config
    from llm_pipeline_b200.models import build_model

    tiny = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", vocab_size=64, hidden_size=32, num_hidden_layers=2, num_attention_heads=4,
                num_key_value_heads=2, head_dim=16, intermediate_size=48)
    model = build_model(resolve_config(tiny))
    assert [pages for pages, _s in model.cache_specs("e4m3")] == [KV8PagesSpec(2, 16)] * 2
    assert [pages for pages, _s in model.cache_specs()] == [KVPagesSpec(2, 16)] * 2
    with pytest.raises(ValueError, match="not 'int8'"):
        model.cache_specs("int8")


def test_a_model_without_such_layers_refuses():
    import zasudra_cases as Z
    from llm_pipeline_b200.config import resolve_config
    from llm_pipeline_b200.models import build_model

    with pytest.raises(ValueError, match="8 bits"):
        build_model(resolve_config(Z.CONFIGS["wkv_only"])).cache_specs("e4m3")


def test_items_cover_every_key_tile_of_every_token_once():
    import random

    rng = random.Random(1)
    for _ in range(200):
        R = rng.randint(1, 5)
        starts, lens = [rng.choice([0, rng.randint(0, 9000)]) for _ in range(R)], [rng.choice([0, 1, rng.randint(1, 2000)]) for _ in range(R)]
        tokens, window, first, nkv = rng.choice([64, 128, 32, 256]), rng.choice([0, 0, 50, 1000]), rng.randint(0, R), rng.choice([1, 8])
        items, shared, places = kv8.plan_items(starts, lens, first, tokens, nkv, window, 148, rng.choice([0, 100, 10000]))
        seen, used = set(), set()
        for r, t, x, place in items:
            part, parts = x & 0xffff, x >> 16
            tiles = dict(((a, b), n) for n, a, b in kv8.tiles_of(starts, lens, first, tokens, window))[r, t]
            assert 0 <= part < parts <= tiles and (r, t, part) not in seen
            seen.add((r, t, part))
            if parts > 1:
                assert place not in used
                used.add(place)
        assert {(r, t) for r, t, _part in seen} == {(r, t) for r in range(first, R) for t in range(0, lens[r], tokens)}
        assert used == set(range(places)) and sum(s[2] for s in shared) == places
        if any(x >> 16 > 1 for _r, _t, x, _p in items):
            assert len(items) * nkv <= 148


def test_which_kernel_portions_take():
    take = lambda starts, lens, nq=32: kv8.reads_pages_directly(starts, lens, 0, nq, 8, 0, 148)         # noqa: E731
    assert take([8003], [40]) and take([2000], [128]) and take([2000], [8]) and take([8000], [512]) and take([0], [2048])
    assert not take([14000], [2048]) and not take([500], [64]) and not take([0], [1000]) and not take([0], [8000]) and not take([], []) and not take([5], [0])
