"""Keys and values in 8 bits: storing, unpacking, attention of single tokens and of prompt portions, against plain forms in 64
bits (``kv8_plain.py``)."""

import math

import pytest
import torch

import kv8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [pytest.param(torch.float32, id="f32"), pytest.param(torch.bfloat16, id="bf16")]
SIZES = [(32, 8, 128, 16), (16, 8, 128, 8), (64, 8, 128, 32), (9, 1, 128, 64), (6, 2, 80, 8), (5, 5, 48, 4), (12, 1, 256, 16), (40, 2, 128, 16),
         (4, 4, 16, 1), (2, 1, 128, 128), (8, 4, 64, 24)]


def K():
    from llm_pipeline_b200.ops import kernels
    return kernels


def same_bytes(got, want, where=""):
    got, want = got.cpu(), want.cpu()
    assert got.shape == want.shape
    bad = (got != want).nonzero()
    assert bad.numel() == 0, f"{where}: {bad.shape[0]} bytes differ, the first at {bad[0].tolist()}: {got[tuple(bad[0])]} and not {want[tuple(bad[0])]}"


def filled(P, nkv, ps, d, seed, wild=True):
    """Host pages with scales of their own in every block, as bytes."""
    gen = torch.Generator().manual_seed(seed)
    host = plain.Pages(P, nkv, ps, d)
    host.q.copy_(torch.randint(0, 256, host.q.shape, generator=gen, dtype=torch.int32).to(torch.uint8))
    host.q[(host.q & 127) == 127] -= 1                                           # numbers alone
    host.e.copy_((torch.randint(117, 123, host.e.shape, generator=gen) if wild else torch.full(host.e.shape, 119)).to(torch.uint8))
    return host


# ---- storing and unpacking -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,ps", SIZES)
def test_store_matches_the_plain_form_to_the_bit(dtype, nq, nkv, d, ps):
    """Three calls one after another: rows at the start of pages, in their middle, over several pages, one by one; rows of very
    different sizes, so that scales rise; rows of a strided matrix."""
    gen = torch.Generator().manual_seed(ps * d + nkv)
    P = 9
    host = filled(P, nkv, ps, d, 1)
    pages = host.raw.to(DEV)
    steps = [list(range(3 * ps, 3 * ps + 2 * ps + ps // 2 + 1)) + [7 * ps],                    # two pages and a part, another request's first token
             [7 * ps + 1] if ps > 1 else [8 * ps],
             list(range(5 * ps + ps // 2 + 1, 6 * ps)) + list(range(1 * ps, 2 * ps)) + [-1] + [2 * ps + ps // 3]]
    for n, slots in enumerate(steps):
        N = len(slots)
        qkv = torch.randn(N, (nq + 2 * nkv) * d, generator=gen) * torch.exp(2.0 * torch.randn(N, 1, generator=gen)) * 10.0 ** n
        qkv = qkv.to(dtype)
        k, v = qkv[:, nq * d:(nq + nkv) * d], qkv[:, (nq + nkv) * d:]
        host.store(k, v, slots)
        on = qkv.to(DEV)
        K().kv8_store(on[:, nq * d:(nq + nkv) * d], on[:, (nq + nkv) * d:], torch.tensor(slots, dtype=torch.int32, device=DEV), pages, nkv, d, ps)
        same_bytes(pages, host.raw, f"step {n}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_store_of_unusual_numbers(dtype):
    """Zeros, the largest and the smallest numbers, infinities and NaN, a page that only gets zeros, a duplicate slot, slots beyond the
    pages, values on the border between two scales and on ties."""
    nkv, d, ps = 2, 32, 8
    host = filled(4, nkv, ps, d, 2)
    pages = host.raw.to(DEV)
    top = torch.finfo(dtype).max
    rows = torch.zeros(14, 2 * nkv * d)
    rows[1, :] = 448.0
    rows[1, 3] = -448.0
    rows[2, ::2] = 450.0
    rows[3, 5] = math.inf
    rows[3, 6] = -math.inf
    rows[3, 7] = math.nan
    rows[3, 40] = 1e-3
    rows[4, :] = top
    rows[5, :] = torch.finfo(dtype).tiny
    rows[6, ::3] = torch.finfo(dtype).tiny / 64
    rows[7, :] = torch.linspace(-20, 20, 2 * nkv * d)
    rows[8, :] = (torch.arange(2 * nkv * d) % 33) / 16.0 + 1.0                   # halves between steps: ties
    rows[9, :] = math.nan
    rows[10, :] = math.inf
    rows[11, :] = -0.0
    rows[12, :] = 2.0 ** -9 * 1.5
    rows[12, 0] = 448.0
    rows[13, :] = 5.0
    rows = rows.to(dtype)
    for slots in ([0, 1, 2, 3, 4], [8, 9, 10, 11, 12, 13, 14], [16, 17], [24, 25, 26, 27, 28]):
        first = {0: 0, 8: 5, 16: 9, 24: 9}[slots[0]]
        part = rows[first:first + len(slots)]
        k, v = part[:, :nkv * d], part[:, nkv * d:]
        host.store(k, v, slots)
        on = part.to(DEV)
        K().kv8_store(on[:, :nkv * d], on[:, nkv * d:], torch.tensor(slots, dtype=torch.int32, device=DEV), pages, nkv, d, ps)
        same_bytes(pages, host.raw, str(slots))
    # the same slot twice (the later row stays), rows without a slot inside a run, slots beyond the pages
    slots = [16, -1, 17, 18, 18, 32, 19, 1 << 30]
    part = rows[4:12]
    k, v = part[:, :nkv * d], part[:, nkv * d:]
    host.store(k, v, slots)
    on = part.to(DEV)
    K().kv8_store(on[:, :nkv * d], on[:, nkv * d:], torch.tensor(slots, dtype=torch.int32, device=DEV), pages, nkv, d, ps)
    same_bytes(pages, host.raw, "twice")


@pytest.mark.parametrize("dtype", DTYPES)
def test_store_cut_into_any_steps_holds_the_same_but_for_the_smallest_values(dtype):
    """A prompt in one call, in portions and token by token: the same scales, and values that differ by at most one rounding
    below the new scale's normal numbers (half of 2^-9)."""
    nkv, d, ps, N = 2, 64, 16, 41
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(N, 2 * nkv * d, generator=gen) * torch.exp(1.5 * torch.randn(N, 1, generator=gen))).to(dtype).to(DEV)
    got = []
    for cut in ([N], [5, 16, 16, 4], [1] * N):
        pages = torch.zeros(3, plain.page_bytes(nkv, ps, d), dtype=torch.uint8, device=DEV)
        at = 0
        for n in cut:
            part = x[at:at + n]
            K().kv8_store(part[:, :nkv * d], part[:, nkv * d:], torch.arange(at, at + n, dtype=torch.int32, device=DEV), pages, nkv, d, ps)
            at += n
        got.append(plain.Pages(3, nkv, ps, d, pages))
    whole = got[0]
    for other in got[1:]:
        assert torch.equal(whole.e, other.e)
        far = (whole.values([0, 1, 2]) - other.values([0, 1, 2])).abs()
        assert bool((far <= 2.0 ** -9 * plain.power(whole.e.int() - 127)[..., None, None]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nkv,d,ps", [(8, 128, 16), (1, 16, 1), (3, 80, 24), (2, 256, 128)])
def test_gather_is_exact_and_zeros_what_is_not_there(dtype, nkv, d, ps):
    P = 7
    host = filled(P, nkv, ps, d, 5)
    host.q[3, :, :, ps // 2 + 1:] = 127                                          # NaN behind the end of request 0
    tables = torch.tensor([[5, 3, 2], [1, -1, 99]], dtype=torch.int32)
    ctx = [ps + ps // 2 + 1, 3 * ps]
    index = [1, 0, 3, 4, 5, 2, 17, -1]
    want = torch.zeros(len(index), 2, nkv, ps, d, dtype=torch.float64)
    for i, entry in enumerate(index):
        if not 0 <= entry < 6 or not 0 <= int(tables.flatten()[entry]) < P:
            continue
        there = ctx[entry // 3] - entry % 3 * ps
        if there > 0:
            want[i, :, :, :there] = host.values([int(tables.flatten()[entry])])[0][:, :, :there]
    out = torch.full((len(index), 2, nkv, ps, d), 7.0, dtype=dtype, device=DEV)
    K().kv8_gather(host.raw.to(DEV), tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV),
                   torch.tensor(index, dtype=torch.int32, device=DEV), out)
    assert torch.equal(out.double().cpu(), want)


@pytest.mark.parametrize("d,ps", [(16, 64), (128, 16), (256, 8)])
def test_store_of_slots_twice_and_out_of_order_keeps_the_last_row(d, ps):
    gen = torch.Generator().manual_seed(8)
    host = filled(3, 1, ps, d, 9)
    pages = host.raw.to(DEV)
    slots = [ps + 2, ps + 1, ps + 5, ps + 5, ps + 1, ps + 3] + [-1] * 40 + [ps + 5, ps + 2] + [s for s in range(2 * ps, 3 * ps)] + [3 * ps - 1]
    x = torch.randn(len(slots), 2 * d, generator=gen)
    host.store(x[:, :d], x[:, d:], slots)
    on = x.to(DEV)
    K().kv8_store(on[:, :d], on[:, d:], torch.tensor(slots, dtype=torch.int32, device=DEV), pages, 1, d, ps)
    same_bytes(pages, host.raw)


# ---- attention -----------------------------------------------------------------------------------------------------------

def scattered(ctx, ps, P, seed):
    """Block tables of requests of ``ctx`` tokens over shuffled pages; one entry more than the longest needs, -1 where there is none."""
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randperm(P, generator=gen).tolist()
    width = max(1, max(-(-c // ps) for c in ctx)) + 1
    tables = torch.full((len(ctx), width), -1, dtype=torch.int32)
    for r, c in enumerate(ctx):
        for j in range(-(-c // ps)):
            tables[r, j] = ids.pop()
    return tables


def spoil(host, tables, ctx, ps):
    """NaN in every slot behind the contexts and in every page that no table names."""
    named = set(int(p) for p in tables.flatten() if p >= 0)
    for p in range(host.q.shape[0]):
        if p not in named:
            host.q[p] = 127
            host.e[p] = 255
    for r, c in enumerate(ctx):
        if c % ps:
            host.q[int(tables[r, c // ps]), :, :, c % ps:] = 127


def bound(out, size, top, dtype, d):
    """How far a row may be off. The result is rounded once. In bfloat16 the weights are rounded to half precision at best, to 2^-11
    of themselves on either side, and their sum is not: 2^-10 of sum w |v| takes both. In either type a score of d products of
    magnitude sum |q||k| scale = top is off by at most (d + 4) 2^-24 top, which moves weights by that much, twice (weight and sum);
    sums of weights and values in tiles, splits and warps add 2^-24 for every of at most 64 terms in a row of additions."""
    half = torch.finfo(dtype).eps / 2
    weights = 2.0 ** -10 if dtype == torch.bfloat16 else 0.0
    return half * out.abs() + size * (weights + 2 * (d + 4) * 2.0 ** -24 * top + 128 * 2.0 ** -24) + 1e-30


CONTEXTS = {"short": [1, 0, 15, 16, 17, 2], "mixed": [129, 700, 1, 256, 31, 64, 333], "long": [2100, 5, 1024, 1500]}


def decode_case(nq, nkv, d, ps, ctx, dtype, seed, wild=True):
    gen = torch.Generator().manual_seed(seed)
    P = sum(-(-c // ps) for c in ctx) + 3
    host = filled(P, nkv, ps, d, seed, wild)
    tables = scattered(ctx, ps, P, seed)
    q = torch.randn(len(ctx), nq * d + 32, generator=gen).to(dtype)
    return host, tables, q


def check_decode(host, tables, q, ctx, nq, nkv, d, ps, window, dtype, out, scale):
    for r, c in enumerate(ctx):
        k, v, there = host.request(tables[r], c)
        want, size, top = plain.attend(q[r:r + 1, :nq * d].view(1, nq, d), k, v, [c - 1], there, scale, window)
        got = out[r].double().cpu().view(1, nq, d)
        far = (got - want).abs()
        allowed = bound(want, size, top, dtype, d)
        if dtype == torch.bfloat16:
            # weights times the scales of their values are held in half precision relative to the largest of them, which is not below
            # the largest of any part of the keys: a factor below 2^-14 of it is off by up to 2^-25 of it, whatever its own size, and so its
            # key's share of an entry by 2^-25 max_j(w_j s_j) |b_j|; this passes 2^-10 sum w |v| only in an entry in which the values of
            # the large factors are (nearly) zeros
            allowed = allowed + plain.smallest(q[r, :nq * d].view(nq, d), k, v, host.value_scales(tables[r], c), c - 1, there, scale, window)
        assert bool((far <= allowed).all()), f"request {r} of {c} keys: {float((far / allowed).max())} times what it may be off"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("lengths", sorted(CONTEXTS))
@pytest.mark.parametrize("nq,nkv,d,ps", SIZES)
def test_single_tokens(dtype, nq, nkv, d, ps, lengths, window):
    ctx = CONTEXTS[lengths]
    host, tables, q = decode_case(nq, nkv, d, ps, ctx, dtype, len(ctx) + d)
    spoil(host, tables, ctx, ps)
    if window:                                                                   # pages that have left the window are gone
        for r, c in enumerate(ctx):
            tables[r, :max(0, c - window) // ps] = -1
    out = torch.full((len(ctx), nq * d), 9.0, dtype=dtype, device=DEV)
    K().kv8_decode_attention(q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV),
                             max(ctx) + 100, nq, nkv, d, ps, window, d ** -0.5)
    check_decode(host, tables, q, ctx, nq, nkv, d, ps, window, dtype, out, d ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,ps", [(32, 8, 128, 16), (6, 2, 80, 8)])
def test_single_tokens_over_blocks_of_very_different_scales(dtype, nq, nkv, d, ps):
    """Value blocks from 2^-60 to 2^60, blocks of zeros whose scale byte is 0 among them: every key has its weight, whatever its
    value's scale; a page missing in the middle has no keys."""
    ctx = [300, 64, 17]
    host, tables, q = decode_case(nq, nkv, d, ps, ctx, dtype, 11)
    gen = torch.Generator().manual_seed(4)
    host.e[:, 1] = torch.randint(67, 188, host.e[:, 1].shape, generator=gen).to(torch.uint8)
    empty = torch.rand(host.e[:, 1].shape, generator=gen) < 0.3
    host.e[:, 1][empty] = 0
    host.q[:, 1][empty] = 0
    tables[0, 3] = -1
    tables[1, 1] = 1000
    out = torch.empty((len(ctx), nq * d), dtype=dtype, device=DEV)
    K().kv8_decode_attention(q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV),
                             max(ctx), nq, nkv, d, ps, 0, d ** -0.5)
    check_decode(host, tables, q, ctx, nq, nkv, d, ps, 0, dtype, out, d ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,ps", [(32, 8, 128, 16), (6, 2, 80, 8)])
def test_single_tokens_with_sharp_and_flat_scores(dtype, nq, nkv, d, ps):
    """Queries of very different sizes in one group: weights from one-hot to even; a query of zeros; what is no number in a query or
    in a seen key makes its rows no number and no others."""
    ctx = [200, 90]
    host, tables, q = decode_case(nq, nkv, d, ps, ctx, torch.float32, 12, wild=False)
    q[:, :nq * d].view(2, nq, d).mul_(torch.logspace(-6, 0.6, nq)[None, :, None])
    q[0, :d] = 0
    q = q.to(dtype)
    out = torch.empty((len(ctx), nq * d), dtype=dtype, device=DEV)
    call = lambda pages, qq: K().kv8_decode_attention(qq.to(DEV), q.stride(0), out, pages.to(DEV), tables.to(DEV),      # noqa: E731
                                                      torch.tensor(ctx, dtype=torch.int32, device=DEV), max(ctx), nq, nkv, d, ps, 0, 1.0)
    call(host.raw, q)
    check_decode(host, tables, q, ctx, nq, nkv, d, ps, 0, dtype, out, 1.0)
    clean = out.clone()
    host.q[int(tables[0, 1]), 0, 0, 0, 5] = 127                                  # one key of head 0 of request 0
    bad = q.clone()
    bad[1, d + 3] = math.nan
    call(host.raw, bad)
    nan = out.view(2, nq, d).isnan()
    G = nq // nkv
    assert bool(nan[0, :G].all()) and not bool(nan[0, G:].any())
    assert bool(nan[1, 1].all()) and int(nan[1].sum()) == d
    assert torch.equal(out.view(2, nq, d)[~nan], clean.view(2, nq, d)[~nan])


def test_more_requests_than_a_launch_takes_and_a_negative_scale():
    """700 requests: two launches of the streaming kernel on one set of counters; scores with their signs turned, and of no size at all."""
    nq, nkv, d, ps = 8, 2, 128, 16
    ctx = [(37 * r) % 90 for r in range(700)]
    host, tables, q = decode_case(nq, nkv, d, ps, ctx, torch.bfloat16, 17)
    spoil(host, tables, ctx, ps)
    for scale in (-0.1, 0.0, 0.09):
        out = torch.full((700, nq * d), 9.0, dtype=torch.bfloat16, device=DEV)
        K().kv8_decode_attention(q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV), 90, nq, nkv,
                                 d, ps, 0, scale)
        for r in (0, 1, 2, 300, 511, 512, 513, 600, 699):
            k, v, there = host.request(tables[r], ctx[r])
            want, size, top = plain.attend(q[r:r + 1, :nq * d].view(1, nq, d), k, v, [ctx[r] - 1], there, scale, 0)
            assert bool(((out[r].double().cpu().view(1, nq, d) - want).abs() <= bound(want, size, top.abs(), torch.bfloat16, d)).all()), (scale, r)


def test_portions_captured_and_replayed():
    """A plan that has been used is captured; one that has not is refused inside a capture, and the stream goes on."""
    from llm_pipeline_b200.ops import kernels, kv8

    nq, nkv, d, ps, starts, lens = 32, 8, 128, 16, [3000], [40]
    for direct in (True, False):
        host, tables, ctx, q, want = prompt((nq, nkv, d, ps), starts, lens, 0, torch.bfloat16, 95, direct=direct)
        dev = [q.to(DEV), host.raw.to(DEV), tables.to(DEV), torch.tensor([0, 40], dtype=torch.int32, device=DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV)]
        out = torch.full_like(want, 9.0)
        plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, 0, torch.bfloat16, torch.device(DEV))
        plan._direct = direct
        call = lambda p: kv8.prompt_attention(p, dev[0], q.stride(0), out, dev[1], dev[2], dev[3], dev[4], d ** -0.5)       # noqa: E731
        call(plan)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(plan)
            fresh = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, 0, torch.bfloat16, torch.device(DEV))
            fresh._direct = direct
            with pytest.raises(kernels.KernelError, match="before a graph"):
                call(fresh)
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(32, 8, 128, 16), (12, 2, 64, 16), (5, 5, 48, 8)])
def test_portions_of_one_token_each(case, dtype):
    """They go where single tokens go, also behind requests that are left out, and give what that gives."""
    nq, nkv, d, ps = case
    starts, lens, window = [10, 300, 77, 9000], [5, 1, 1, 1], 0
    host, tables, ctx, q, out = prompt(case, starts, lens, window, dtype, 44, first=1)
    want = torch.empty(3, nq * d, dtype=dtype, device=DEV)
    K().kv8_decode_attention(q[5:8].to(DEV), q.stride(0), want, host.raw.to(DEV), tables[1:].to(DEV), torch.tensor(ctx[1:], dtype=torch.int32, device=DEV), 9001,
                             nq, nkv, d, ps, window, d ** -0.5)
    assert torch.equal(out[5:8], want) and bool((out[:5] == 9).all()) and bool((out[8:] == 9).all())
    check_decode(host, tables[1:], q[5:8], ctx[1:], nq, nkv, d, ps, window, dtype, out[5:8], d ** -0.5)


@pytest.mark.parametrize("direct", [True, False])
def test_one_plan_on_two_streams(direct):
    from llm_pipeline_b200.ops import kv8

    nq, nkv, d, ps, starts, lens = 32, 8, 128, 16, [500, 0], [40, 9]
    host, tables, ctx, q, want = prompt((nq, nkv, d, ps), starts, lens, 0, torch.bfloat16, 96, direct=direct)
    dev = [q.to(DEV), host.raw.to(DEV), tables.to(DEV), torch.tensor([0, 40, 49], dtype=torch.int32, device=DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV)]
    plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, 0, torch.bfloat16, torch.device(DEV))
    plan._direct = direct
    torch.cuda.synchronize()
    outs = []
    for stream in (torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.current_stream()):
        with torch.cuda.stream(stream):
            outs.append(torch.full((49, nq * d), 9.0, dtype=torch.bfloat16, device=DEV))
            kv8.prompt_attention(plan, dev[0], q.stride(0), outs[-1], dev[1], dev[2], dev[3], dev[4], d ** -0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[:49]) for out in outs)


def test_single_tokens_in_a_page_pool_beyond_four_gigabytes():
    """Pages whose bytes begin beyond 32-bit offsets."""
    nq, nkv, d, ps = 32, 8, 128, 64
    size = plain.page_bytes(nkv, ps, d)
    P = (1 << 32) // size + 9
    pages = torch.zeros(P, size, dtype=torch.uint8, device=DEV)
    ctx = [150]
    host, _t, q = decode_case(nq, nkv, d, ps, ctx, torch.bfloat16, 21)
    last = [P - 1, P - 3, P - 2]
    pages[last] = host.raw[:3].to(DEV)
    tables = torch.tensor([last], dtype=torch.int32)
    x = torch.randn(1, 2 * nkv * d, generator=torch.Generator().manual_seed(1)).bfloat16()
    K().kv8_store(x[:, :nkv * d].to(DEV), x[:, nkv * d:].to(DEV), torch.tensor([(P - 2) * ps + 21], dtype=torch.int32, device=DEV), pages, nkv, d, ps)
    host.store(x[:, :nkv * d], x[:, nkv * d:], [2 * ps + 21])
    same_bytes(pages[last], host.raw[:3])
    out = torch.empty(1, nq * d, dtype=torch.bfloat16, device=DEV)
    K().kv8_decode_attention(q.to(DEV), q.stride(0), out, pages, tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV), 150, nq, nkv, d, ps,
                             0, d ** -0.5)
    check_decode(host, torch.tensor([[0, 1, 2]]), q, ctx, nq, nkv, d, ps, 0, torch.bfloat16, out, d ** -0.5)


def prompt(case, starts, lens, window, dtype, seed, first=0, direct=True):
    """``direct``: through the kernel that reads 8-bit pages, where it takes the sizes."""
    from llm_pipeline_b200.ops import kv8

    nq, nkv, d, ps = case
    ctx = [s + n for s, n in zip(starts, lens)]
    P = sum(-(-c // ps) for c in ctx) + 3
    host = filled(P, nkv, ps, d, seed)
    tables = scattered(ctx, ps, P, seed)
    spoil(host, tables, ctx, ps)
    N = sum(lens)
    q = torch.randn(N + 2, (nq + 2 * nkv) * d, generator=torch.Generator().manual_seed(seed)).to(dtype)
    out = torch.full((N + 2, nq * d), 9.0, dtype=dtype, device=DEV)
    plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, window, dtype, torch.device(DEV), first_request=first)
    plan._direct = direct and K().kv8_prompt_supports(dtype, nq, nkv, d, ps)
    dev = dict(pages=host.raw.to(DEV), tables=tables.to(DEV), ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV), q=q.to(DEV),
               start=torch.tensor([sum(lens[:r]) for r in range(len(lens) + 1)], dtype=torch.int32, device=DEV))
    kv8.prompt_attention(plan, dev["q"], q.stride(0), out, dev["pages"], dev["tables"], dev["start"], dev["ctx"], d ** -0.5)
    return host, tables, ctx, q, out


PORTIONS = [([0], [1]), ([0], [300]), ([37, 0, 500], [129, 1, 70]), ([1000, 3], [2, 40])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("portions", range(len(PORTIONS)))
@pytest.mark.parametrize("direct", [True, False])
@pytest.mark.parametrize("nq,nkv,d,ps", [(32, 8, 128, 16), (6, 2, 80, 8), (5, 5, 48, 4), (9, 1, 128, 64)])
def test_prompt_portions(dtype, nq, nkv, d, ps, direct, portions, window):
    starts, lens = PORTIONS[portions]
    host, tables, ctx, q, out = prompt((nq, nkv, d, ps), starts, lens, window, dtype, 31 + portions, direct=direct)
    at = 0
    for r, n in enumerate(lens):
        rows = sorted({0, 1, n // 2, n - 1} & set(range(n)))
        k, v, there = host.request(tables[r], ctx[r])
        want, size, top = plain.attend(q[[at + i for i in rows], :nq * d].view(-1, nq, d), k, v, [starts[r] + i for i in rows], there, d ** -0.5, window)
        far = (out[[at + i for i in rows]].double().cpu().view(-1, nq, d) - want).abs()
        # the kernel over unpacked pages rounds the weights to bfloat16 (2^-8 of themselves, and their sum is not rounded)
        allowed = bound(want, size, top, dtype, d) + (2.0 ** -8 * size if dtype == torch.bfloat16 else 0)
        assert bool((far <= allowed).all()), f"request {r}: {float((far / allowed).max())}"
        at += n
    assert bool((out[at:] == 9).all())                                           # rows behind the last request's


@pytest.mark.parametrize("nq,nkv,d,ps,starts,lens", [(32, 8, 128, 16, [5000], [40]), (32, 8, 128, 8, [3001, 0], [3, 200]), (8, 8, 128, 32, [700, 2000], [1, 300]),
                                                     (40, 2, 128, 16, [4000], [17]), (9, 1, 128, 64, [6000], [5]), (32, 8, 128, 128, [0], [1111])])
@pytest.mark.parametrize("window", [0, 2000])
def test_prompt_portions_on_the_tensor_cores(nq, nkv, d, ps, starts, lens, window):
    """Few new tokens over many keys (their keys come in parts), odd groups, pages of every size, values of very different scales."""
    host, tables, ctx, q, out = prompt((nq, nkv, d, ps), starts, lens, window, torch.bfloat16, 61)
    check_prompt(host, tables, ctx, q, out, starts, lens, nq, nkv, d, window)


def check_prompt(host, tables, ctx, q, out, starts, lens, nq, nkv, d, window, skip=()):
    at = 0
    for r, n in enumerate(lens):
        k, v, there = host.request(tables[r], ctx[r])
        for i in sorted({0, 1, n // 3, n // 2, n - 2, n - 1} & set(range(n)) - set(skip)):
            row, pos = q[at + i:at + i + 1, :nq * d].view(1, nq, d), starts[r] + i
            seen = slice(max(0, pos - window + 1) if window else 0, pos + 1)
            kk, vv, tt = k[seen], v[seen], there[seen]
            want, size, top = plain.attend(row, kk, vv, [len(kk) - 1], tt, d ** -0.5, 0)
            allowed = bound(want, size, top, torch.bfloat16, d) + plain.smallest(row[0], kk, vv, host.value_scales(tables[r], ctx[r])[seen], len(kk) - 1, tt,
                                                                                d ** -0.5, 0)       # as for single tokens
            far = (out[at + i].double().cpu().view(1, nq, d) - want).abs()
            assert bool((far <= allowed).all()), f"request {r} row {i}: {float((far / allowed).max())}"
        at += n
    assert bool((out[at:] == 9).all())


def test_prompt_portions_over_blocks_of_very_different_scales():
    """Value blocks from 2^-60 to 2^60 and blocks of zeros; keys of very different sizes; queries of zeros and of 1e-30."""
    from llm_pipeline_b200.ops import kv8

    nq, nkv, d, ps, starts, lens = 32, 8, 128, 16, [333, 0], [100, 150]
    gen = torch.Generator().manual_seed(3)
    ctx = [433, 150]
    P = 40
    host = filled(P, nkv, ps, d, 71)
    host.e[:, 1] = torch.randint(67, 188, host.e[:, 1].shape, generator=gen).to(torch.uint8)
    empty = torch.rand(host.e[:, 1].shape, generator=gen) < 0.3
    host.e[:, 1][empty] = 0
    host.q[:, 1][empty] = 0
    host.e[::5, 0] = 0
    host.q[::5, 0] = 0
    tables = scattered(ctx, ps, P, 5)
    q = torch.randn(250, nq * d, generator=gen)
    q[3] = 0
    q[100] *= 1e-30
    q = q.bfloat16()
    out = torch.full((250, nq * d), 9.0, dtype=torch.bfloat16, device=DEV)
    plan = kv8.PromptPlan(starts, lens, nq, nkv, d, ps, 0, torch.bfloat16, torch.device(DEV))
    plan._direct = True
    kv8.prompt_attention(plan, q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV), torch.tensor([0, 100, 250], dtype=torch.int32, device=DEV),
                         torch.tensor(ctx, dtype=torch.int32, device=DEV), d ** -0.5)
    check_prompt(host, tables, ctx, q, out, starts, lens, nq, nkv, d, 0)


@pytest.mark.parametrize("dim,ps", [(128, 16)])
def test_what_a_row_cannot_see_does_not_matter_to_it(dim, ps):
    """Keys and values that are no number, of tokens that come after a row or before its window, leave the row as it is; rows that see them
    are no number; a query that is none is its own row's matter."""
    nq, nkv, starts, lens, window = 8, 2, [200], [300], 150
    host, tables, ctx, q, clean = prompt((nq, nkv, dim, ps), starts, lens, window, torch.bfloat16, 81)
    from llm_pipeline_b200.ops import kv8

    at = 320                                                                     # a token of the portion: rows 120 .. 269 see it
    host.q[int(tables[0, at // ps]), 1, 0, at % ps, 7] = 127                     # a value of head 0
    host.q[int(tables[0, at // ps]), 0, 1, at % ps, 9] = 255                     # a key of head 1
    q[5, 3 * dim] = float("nan")
    out = torch.full_like(clean, 9.0)
    plan = kv8.PromptPlan(starts, lens, nq, nkv, dim, ps, window, torch.bfloat16, torch.device(DEV))
    plan._direct = True
    kv8.prompt_attention(plan, q.to(DEV), q.stride(0), out, host.raw.to(DEV), tables.to(DEV), torch.tensor([0, 300], dtype=torch.int32, device=DEV),
                         torch.tensor(ctx, dtype=torch.int32, device=DEV), dim ** -0.5)
    nan = out[:300].view(300, nq, dim).isnan()
    sees = torch.zeros(300, dtype=torch.bool, device=DEV)
    sees[120:270] = True
    assert bool(nan[sees].all(-1).all()) or bool(nan[sees][:, 4:].all())
    assert bool(nan[sees].any(-1).all())
    assert not bool(nan[~sees].sum() - nan[5, 3].sum()) and bool(nan[5, 3].all())
    rest = ~sees[:, None].expand(300, nq).clone()
    rest[5, 3] = False
    assert torch.equal(out[:300].view(300, nq, dim)[rest], clean[:300].view(300, nq, dim)[rest])


def test_prompt_portions_in_turns_of_a_small_workspace(monkeypatch):
    from llm_pipeline_b200.ops import kv8

    case, starts, lens = (32, 8, 128, 16), [37, 0, 500, 20], [129, 1, 70, 33]
    whole = prompt(case, starts, lens, 0, torch.bfloat16, 41, direct=False)[-1]
    direct = prompt(case, starts, lens, 0, torch.bfloat16, 41, first=2)[-1]
    monkeypatch.setattr(kv8, "WORKSPACE_BYTES", 1 << 20)
    assert torch.equal(prompt(case, starts, lens, 0, torch.bfloat16, 41, direct=False)[-1], whole)
    # the first requests left to another kernel
    part = prompt(case, starts, lens, 0, torch.bfloat16, 41, first=2, direct=False)[-1]
    assert bool((part[:130] == 9).all()) and torch.equal(part[130:], whole[130:])
    assert bool((direct[:130] == 9).all()) and not bool((direct[130:-2] == 9).any())
    # without places for sums the kernel that reads 8-bit pages takes every tile's keys whole (other sums, so by the plain form)
    host, tables, ctx, q, out = prompt(case, starts, lens, 0, torch.bfloat16, 41)
    check_prompt(host, tables, ctx, q, out, starts, lens, 32, 8, 128, 0)


def test_a_step_in_a_graph_and_on_two_streams():
    """Store and attention captured, replayed over other contents; two such calls at once on two streams."""
    nq, nkv, d, ps = 32, 8, 128, 16
    ctx = [333, 40, 1000]
    sets = []
    for seed in (51, 52):
        host, tables, q = decode_case(nq, nkv, d, ps, ctx, torch.bfloat16, seed)
        x = torch.randn(3, 2 * nkv * d, generator=torch.Generator().manual_seed(seed)).bfloat16()
        slots = [int(tables[r, (c - 1) // ps]) * ps + (c - 1) % ps for r, c in enumerate(ctx)]
        sets.append((host, tables, q, x, slots))
    dev = [[host.raw.to(DEV), tables.to(DEV), q.to(DEV), x.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV),
            torch.tensor(ctx, dtype=torch.int32, device=DEV), torch.empty(3, nq * d, dtype=torch.bfloat16, device=DEV)]
           for host, tables, q, x, slots in sets]

    def call(t):
        pages, tables, q, x, slots, n, out = t
        K().kv8_store(x[:, :nkv * d], x[:, nkv * d:], slots, pages, nkv, d, ps)
        K().kv8_decode_attention(q, q.stride(0), out, pages, tables, n, 1024, nq, nkv, d, ps, 0, d ** -0.5)

    fresh = [t[0].clone() for t in dev]
    call(dev[0])
    graphs = []
    for t in dev:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(t)
        graphs.append(g)
    for host, tables, q, x, slots in sets:
        host.store(x[:, :nkv * d], x[:, nkv * d:], slots)
    for how in ("graphs", "streams"):
        for t, raw in zip(dev, fresh):
            t[0].copy_(raw)
            t[-1].zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(20):
            for t, g, s in zip(dev, graphs, streams):
                with torch.cuda.stream(s):
                    g.replay() if how == "graphs" else call(t)
        torch.cuda.synchronize()
        for t, (host, tables, q, x, slots) in zip(dev, sets):
            same_bytes(t[0], host.raw, how)
            check_decode(host, tables, q, ctx, nq, nkv, d, ps, 0, torch.bfloat16, t[-1], d ** -0.5)


def test_empty_calls_do_nothing():
    nkv, d, ps = 2, 32, 8
    pages = torch.full((2, plain.page_bytes(nkv, ps, d)), 3, dtype=torch.uint8, device=DEV)
    none = torch.empty(0, nkv * d, device=DEV)
    i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device=DEV)             # noqa: E731
    K().kv8_store(none, none, i32(0), pages, nkv, d, ps)
    K().kv8_gather(pages, i32(0, 3), i32(0), i32(0), torch.empty(0, 2, nkv, ps, d, device=DEV))
    K().kv8_decode_attention(torch.empty(0, 4 * d, device=DEV), 4 * d, torch.empty(0, 4 * d, device=DEV), pages, i32(0, 3), i32(0), 5, 4, nkv, d, ps, 0, 1.0)
    assert bool((pages == 3).all())


# ---- copies ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape,dtype", [((2, 8, 16, 128), torch.bfloat16), ((33024,), torch.uint8), ((7,), torch.uint8), ((5, 3), torch.float32)])
@pytest.mark.parametrize("tensors,pairs", [(1, 1), (50, 3), (2, 900)])
def test_copy_pages(shape, dtype, tensors, pairs):
    gen = torch.Generator(device=DEV).manual_seed(5)
    P = 2 * pairs + 3
    if tensors * P * math.prod(shape) > 1 << 28:
        tensors = 1
    caches = [torch.randint(0, 200, (P,) + shape, generator=gen, device=DEV).to(dtype) for _ in range(tensors)]
    order = torch.randperm(P, generator=torch.Generator().manual_seed(6)).tolist()
    src, dst = order[:pairs], order[pairs:2 * pairs]
    if pairs > 1:
        src[1] = src[0]                                                          # one page to two places
    want = [t.clone() for t in caches]
    for t in want:
        t[dst] = t[src]
    K().copy_pages(caches, src, dst)
    for got, t in zip(caches, want):
        assert torch.equal(got, t)
