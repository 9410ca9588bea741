"""Keys and values in 8 bits, forked prompts and compaction through the engine."""

import pytest
import torch

import helpers as H
import kv8_plain as plain8
import plain_qwen3 as plain
from test_gpu_generate import engine_for
from test_gpu_kv8 import bound

pytestmark = pytest.mark.gpu
DTYPES = [pytest.param(torch.float32, id="f32"), pytest.param(torch.bfloat16, id="bf16")]
# head size 128: the streaming kernel and the tensor cores' attention
WIDE = dict(plain.TINY_A, head_dim=128, num_attention_heads=8, num_key_value_heads=2)
CONFIGS = [pytest.param(plain.TINY_A, id="tiny"), pytest.param(WIDE, id="wide")]


def runner_for(folder, dtype, num_pages=96, use_graphs=True, page_size=8):
    from llm_pipeline_b200.cache import CacheManager
    from llm_pipeline_b200.engine import ModelRunner
    from llm_pipeline_b200.models import load_model

    _config, model = load_model(folder, "cuda:0", dtype)
    cache = CacheManager(model.cache_specs("e4m3"), page_size=page_size, num_pages=num_pages, max_requests=8, max_request_tokens=512, device=model.device,
                         dtype=dtype)
    return ModelRunner(model, cache, use_graphs=use_graphs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("config", CONFIGS)
def test_every_layer_of_every_step_is_the_plain_form(tmp_path, config, dtype, monkeypatch):
    """Portions, single tokens and both in one step: what each layer stores is what the plain form makes of the keys and values of
    its rows, and what it attends to is what the pages hold."""
    from llm_pipeline_b200.ops import kernels
    from llm_pipeline_b200.parts import attention

    folder, _weights = H.make_case(tmp_path, config, 3, dtype, std=0.08)
    runner = runner_for(folder, dtype, use_graphs=False)
    nq, nkv, d, ps = config["num_attention_heads"], config["num_key_value_heads"], config["head_dim"], 8
    hosts, checked = {}, {"stores": 0, "rows": 0}
    store = kernels.kv8_store

    def checked_store(k, v, slots, pages, *sizes):
        store(k, v, slots, pages, *sizes)
        host = hosts.setdefault(pages.data_ptr(), plain8.Pages(pages.shape[0], nkv, ps, d))
        host.store(k, v, slots.tolist())
        assert torch.equal(pages.cpu()[:, :host.body + 2 * nkv], host.raw[:, :host.body + 2 * nkv])
        checked["stores"] += 1

    attend = attention.PagedAttention.attend

    def checked_attend(self, ctx, qkv, out, cache):
        attend(self, ctx, qkv, out, cache)
        host, at = hosts[cache.pages.data_ptr()], 0
        for r, n in enumerate(ctx.q_lens):
            k, v, there = host.request(ctx.block_tables[cache.group][r].tolist(), ctx.starts[r] + n)
            rows = sorted({0, n // 3, n // 2, n - 1})
            q = qkv[[at + i for i in rows], :nq * d].view(-1, nq, d)
            want, size, top = plain8.attend(q, k, v, [ctx.starts[r] + i for i in rows], there, self.scale, 0)
            allowed = bound(want, size, top, dtype, d) + (2.0 ** -8 * size if dtype == torch.bfloat16 else 0)
            assert bool(((out[[at + i for i in rows]].double().cpu().view(-1, nq, d) - want).abs() <= allowed).all())
            checked["rows"] += len(rows)
            at += n

    monkeypatch.setattr(kernels, "kv8_store", checked_store)
    monkeypatch.setattr(attention.PagedAttention, "attend", checked_attend)
    requests = {f"r{i}": H.random_tokens(config["vocab_size"], n, 60 + i) for i, n in enumerate((1, 40, 17, 90, 33))}
    H.replay(runner, H.cut_mixed(requests, [7, 30, 16, 64], decode_tail=5))
    assert checked["stores"] > 20 and checked["rows"] > 80


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("config", CONFIGS)
def test_replayed_steps_give_what_eager_ones_give(tmp_path, config, dtype):
    folder, _weights = H.make_case(tmp_path, config, 4, dtype, std=0.08)
    requests = {f"r{i}": H.random_tokens(config["vocab_size"], n, 70 + i) for i, n in enumerate((60, 41, 77))}
    got = []
    for graphs in (False, True):
        runner = runner_for(folder, dtype, use_graphs=graphs)
        # all together: prompts, then single tokens of all three for many steps
        steps, at = [([(rid, toks[:-30], [0]) for rid, toks in requests.items()], [])], 30
        for k in range(30):
            steps.append(([(rid, [toks[len(toks) - 30 + k]], [0]) for rid, toks in requests.items()], list(requests) if k == 29 else []))
        got.append(H.replay(runner, steps))
        assert (runner.graph_replays > 20) == graphs
    for rid in requests:
        # single tokens add partial sums in splits of a bound on the context that only a captured step rounds up: float32's last bits, and
        # what they make of the model's other roundings
        assert torch.allclose(got[0][rid], got[1][rid], atol=H.TOL[dtype])


@pytest.mark.parametrize("config", CONFIGS)
def test_generation_with_8_bits_is_seeded_and_ends_clean(tmp_path, config):
    folder, _weights = H.make_case(tmp_path, config, 5, torch.bfloat16, std=0.08)
    engine = engine_for(folder, torch.bfloat16, kv_cache_dtype="e4m3")
    assert engine.engine.cache.groups[0].tensors[0].dtype == torch.uint8
    prompts = [H.random_tokens(config["vocab_size"], n, 80 + n) for n in (3, 25, 70)]
    first = engine.generate(prompts, max_tokens=12, temperature=0.8, ignore_eos=True)
    assert [len(t) for t in first] == [12] * 3
    assert engine.generate(prompts, max_tokens=12, temperature=0.8, ignore_eos=True) == first
    engine.engine.cache.check()
    assert engine.engine.cache.num_live == 0
    ordinary = engine_for(folder, torch.bfloat16)
    eight, sixteen = engine.estimate_memory_usage()["kv_cache_bytes_per_token"], ordinary.estimate_memory_usage()["kv_cache_bytes_per_token"]
    body = 2 * config["num_key_value_heads"] * 8 * config["head_dim"]
    assert eight == config["num_hidden_layers"] * plain8.page_bytes(config["num_key_value_heads"], 8, config["head_dim"]) // 8
    assert sixteen == config["num_hidden_layers"] * 2 * body // 8 and eight < sixteen


@pytest.mark.parametrize("kind", [None, "e4m3"])
@pytest.mark.parametrize("prompt", [1, 8, 9, 45])
def test_several_samples_of_a_prompt_share_its_pages(tmp_path, kind, prompt):
    """Greedy samples are all the same tokens as a request of its own gives (float32: no near ties at these sizes), seeded ones differ; the
    prompt is computed once."""
    folder, _weights = H.make_case(tmp_path, plain.TINY_A, 6, torch.float32, std=0.08)
    engine = engine_for(folder, torch.float32, kv_cache_dtype=kind)
    ids = H.random_tokens(plain.TINY_A["vocab_size"], prompt, 90)
    alone = engine.generate(ids, max_tokens=9, temperature=0.0, ignore_eos=True)
    before = dict(engine.get_stats())
    got = engine.generate([ids], max_tokens=9, temperature=0.0, ignore_eos=True, num_return_sequences=4)
    assert len(got) == 4 and all(t == alone for t in got)
    after = engine.get_stats()
    computed = after["tokens_prefilled"] - before["tokens_prefilled"]
    assert computed == (prompt + 3 if prompt > 1 else 4)                        # the prompt, and its last token again for each of the others
    engine.engine.cache.check()
    assert engine.engine.cache.num_live == 0 and not engine.engine._forks
    drawn = engine.generate([ids], max_tokens=9, temperature=1.5, top_k=0, top_p=1.0, ignore_eos=True, num_return_sequences=4)
    assert len({tuple(t) for t in drawn}) > 1


def test_samples_that_find_no_room_are_computed_on_their_own(tmp_path):
    folder, _weights = H.make_case(tmp_path, plain.TINY_A, 6, torch.float32, std=0.08)
    ids = H.random_tokens(plain.TINY_A["vocab_size"], 45, 90)
    alone = engine_for(folder, torch.float32).generate(ids, max_tokens=20, temperature=0.0, ignore_eos=True)
    for kw in (dict(max_batch_size=2), dict(num_blocks=12), dict(max_num_batched_tokens=16)):
        engine = engine_for(folder, torch.float32, **kw)
        got = engine.generate([ids, ids[:30]], max_tokens=20, temperature=0.0, ignore_eos=True, num_return_sequences=3)
        assert got[:3] == [alone] * 3 and got[3] == got[4] == got[5]
        engine.engine.cache.check()
        assert engine.engine.cache.num_live == 0
    # the request whose prompt the others wait for is aborted
    core = engine_for(folder, torch.float32, max_num_batched_tokens=16).engine
    first = core.add_request(ids, 5, ignore_eos=True)
    others = [core.add_request(ids, 5, ignore_eos=True, same_prompt_as=first) for _ in range(2)]
    core.step()
    assert core.abort(others[1]).finish_reason == "abort"
    core.abort(first)
    while core.has_unfinished():
        core.step()
    assert len(core._requests[others[0]].output) == 5 and core._requests[others[1]].status == "finished" and core.cache.num_live == 0
    # one that waits for another that waits: the middle one goes, then the first
    first = core.add_request(ids, 5, ignore_eos=True)
    middle = core.add_request(ids, 5, ignore_eos=True, same_prompt_as=first)
    last = core.add_request(ids, 5, ignore_eos=True, same_prompt_as=middle)
    core.step()
    core.abort(middle)
    while core.has_unfinished():
        core.step()
    assert core._requests[first].output == core._requests[last].output and len(core._requests[last].output) == 5 and not core._forks
    with pytest.raises(ValueError, match="another prompt"):
        core.add_request(ids[:-1], 5, same_prompt_as=others[0])


def test_samples_of_a_model_with_state(tmp_path):
    import zasudra_cases as Z
    from llm_pipeline_b200.engine.generate import GenerationEngine
    from llm_pipeline_b200.weights import write_random_model

    folder = write_random_model(Z.CONFIGS["wkv_only"], 0, str(tmp_path / "m"))
    core = GenerationEngine.from_folder(folder, dtype=torch.float32, num_pages=64, max_num_seqs=8, max_model_len=256)
    ids = H.random_tokens(core.model.spec.vocab_size, 20, 7)
    alone = core.generate([ids], max_tokens=8, temperature=0.0, ignore_eos=True)[0].token_ids
    got = core.generate([ids], max_tokens=8, temperature=0.0, ignore_eos=True, samples_per_prompt=3)
    assert [r.token_ids for r in got] == [alone] * 3


@pytest.mark.parametrize("kind", [None, "e4m3"])
def test_compaction_between_steps_changes_nothing(tmp_path, kind):
    """Requests of different lengths end while others go on, in replayed steps too; the pool is compacted every few steps."""
    folder, _weights = H.make_case(tmp_path, WIDE, 8, torch.bfloat16, std=0.08)
    prompts = [H.random_tokens(WIDE["vocab_size"], n, 100 + n) for n in (5, 60, 21, 44, 33, 12)]
    got, moved = [], 0
    for compact in (False, True):
        core = engine_for(folder, torch.bfloat16, kv_cache_dtype=kind).engine
        ids = [core.add_request(p, 6 + 9 * i, ignore_eos=True) for i, p in enumerate(prompts)]
        step = 0
        while core.has_unfinished():
            core.step()
            step += 1
            if compact and step % 3 == 0:
                moved += core.cache.compact()
                core.cache.check()
        got.append([core._requests[i].output for i in ids])
        assert core.runner.graph_replays > 10
    assert moved > 10 and got[0] == got[1]


def test_forked_pages_hold_what_was_forked(tmp_path):
    """Two requests go on differently from one prompt: each one's logits are those of a request that was never forked."""
    folder, _weights = H.make_case(tmp_path, plain.TINY_A, 9, torch.float32, std=0.08)
    from llm_pipeline_b200.engine import StepEntry

    ids = H.random_tokens(plain.TINY_A["vocab_size"], 29, 110)
    tails = [H.random_tokens(plain.TINY_A["vocab_size"], 12, 111 + k) for k in range(2)]
    for make in (lambda: runner_for(folder, torch.float32), lambda: H.make_runner(folder, torch.float32, 8, 96)):
        want = []
        for tail in tails:
            runner = make()
            runner.step([StepEntry("x", ids, [])])
            want.append(torch.cat([runner.step([StepEntry("x", [t], [0])]).cpu() for t in tail]))
        runner = make()
        runner.step([StepEntry("x", ids, [])])
        assert runner.cache.fork("x", ["y"])
        rows = [[], []]
        for a, b in zip(*tails):
            logits = runner.step([StepEntry("x", [a], [0]), StepEntry("y", [b], [0])]).cpu()
            rows[0].append(logits[:1])
            rows[1].append(logits[1:])
            runner.cache.check()
        for got, ref in zip(rows, want):
            assert torch.allclose(torch.cat(got), ref, atol=1e-4)


def test_cli_with_8_bits(tmp_path, capsys):
    from llm_pipeline_b200 import cli

    folder, _weights = H.make_case(tmp_path, plain.TINY_A, 0, torch.bfloat16, std=0.08)
    assert cli.main(["infer", "--model", folder, "--prompt-ids", "5 17 3", "--max-new-tokens", "6", "--temperature", "0", "--num-blocks", "64",
                     "--max-sequence-length", "128", "--kv-cache-dtype", "e4m3"]) == 0
    assert len(capsys.readouterr().out.split()) >= 1
