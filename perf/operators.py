"""Cases of the 8-bit cache: storing keys and values with a scale for each page and head, attention of single tokens and of
prompt portions over such pages, and copies of pages of any cache (forks, compaction).

A page of a cache in 8 bits is a row of bytes: ``[2 (keys, values)][kv heads][page size][head size]`` in e4m3, then
``[2][kv heads]`` bytes of scales (byte e stands for 2^(e - 127), 0 for 0), padded to a multiple of 128 bytes. Heads and
head sizes are those of ``bench.py``'s shapes (0.6B: 16 query and 8 key/value heads, 8B: 32 and 8, 32B: 64 and 8, head size
128) and of the kernels' tests."""

import math

import torch

own = False                                  # True: the framework's calls instead of the plain form

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _case(name, kind, heads=32, kv=8, dim=128, page=16, dtype="bfloat16", requests=1, new=1, context=0, spread="even", window=0,
          layers=0, count=0):
    return {"name": name, "kind": kind, "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "requests": requests,
            "new": new, "context": context, "spread": spread, "window": window, "layers": layers, "count": count}


def listed():
    return [
        # a decode step of eight requests leaves one token of each in the cache
        _case("store, 8 single tokens", "store", requests=8, context=2041),
        # prompts of several users go into the cache in one step, one of them behind a page that is partly filled
        _case("store, prompts ragged", "store", requests=3, new=1500, context=37, spread="ragged"),
        # one short chat takes a token on the small model: latency
        _case("decode, 1 short", "decode", heads=16, context=300),
        # the serving step of the benchmark: eight requests at 2,048 tokens
        _case("decode, 8 at 2,048", "decode", requests=8, context=2047),
        # a full server: many requests of very different lengths
        _case("decode, 64 ragged", "decode", requests=64, context=4001, spread="ragged"),
        # a document beside short chats on the large model
        _case("decode, one long of 8", "decode", heads=64, requests=8, context=16390, spread="one long"),
        # the exact path on a layer with a window and a head size of its own
        _case("decode, float32 window", "decode", heads=6, kv=2, dim=80, page=8, dtype="float32", requests=4, context=700, spread="ragged",
              window=333),
        # a document is read
        _case("prompt, 2,048 tokens", "prompt", new=2048),
        # three users' prompts in one step, two of them going on behind what is cached
        _case("prompt, ragged", "prompt", requests=3, new=900, context=1100, spread="ragged"),
        # a question of 40 tokens behind a long document that several requests share
        _case("prompt, 40 behind 8,000", "prompt", new=40, context=8003),
        # eight requests fork: the partly filled page of each, in every layer of the small model
        _case("pages, 8 in 28 layers", "pages", requests=1, layers=28, count=8),
        # a pool is compacted
        _case("pages, 1,500 in 4 layers", "pages", requests=1, layers=4, count=1500),
    ]


def draw(rng):
    """One more case: steps of single tokens and prompt portions of 1 to 2,048 tokens over up to 16,000 cached ones, 1 to 64
    requests, pages of 8 to 64 tokens, the heads of the three shapes and of a few odd layers, some windows, some float32."""
    kind = rng.choice(["store", "decode", "decode", "decode", "prompt", "prompt", "pages"])
    spread = rng.choice(["even", "ragged", "ragged", "one long"])
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    page = rng.choice([8, 16, 16, 16, 32, 64])
    if kind == "pages":
        layers = rng.choice([1, 4, 28])
        return _case("", kind, page=page, layers=layers, count=log(1, 6000 * 16 // (layers * page)))
    heads, kv, dim = rng.choice([(16, 8, 128), (32, 8, 128), (32, 8, 128), (64, 8, 128), (12, 2, 64), (5, 5, 48), (9, 1, 128)])
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    window = log(40, 3000) if rng.random() < 0.2 else 0
    case = _case("", kind, heads, kv, dim, page, dtype, spread=spread, window=window)
    if kind == "store":
        case.update(requests=log(1, 64), window=0, context=log(1, 3000))
        if rng.random() < 0.5:
            case.update(requests=rng.randint(1, 4), new=log(2, 1000))
        case["context"] = min(case["context"], 30000 // case["requests"])
    elif kind == "decode":
        case["requests"] = log(1, 64)
        case["context"] = min(log(1, 16000), (160000 if dtype == "bfloat16" else 12000) // case["requests"])
    else:
        case.update(requests=rng.choice([1, 1, 2, 3, 4]), new=log(1, 2048 if dtype == "bfloat16" else 300))
        case["new"] = max(1, case["new"] // case["requests"])
        case["context"] = min(log(1, 8000), 2500000 // (case["new"] * case["requests"]))
    case.pop("name")
    return case


# ---- sizes of a case ---------------------------------------------------------------------------------------------------

def _lengths(case):
    """(new tokens, cached tokens) of every request: the first is the longest, with "ragged" the last a small part of it, with
    "one long" the others a 32nd."""
    R, new, context = case["requests"], case["new"], case["context"]
    if case["spread"] == "even" or R == 1:
        return [new] * R, [context] * R
    if case["spread"] == "one long":
        return [new] + [max(1, new // 3)] * (R - 1), [context] + [context // 32] * (R - 1)
    part = [1.0 - 0.9 * r / (R - 1) for r in range(R)]
    return [max(1, int(new * f)) for f in part], [int(context * f) for f in part]


def _page_bytes(case):
    body = 2 * case["kv"] * case["page"] * case["dim"]
    return -(-(body + 2 * case["kv"]) // 128) * 128, body


def _views(pages, case):
    """(e4m3 values [pages, 2, kv, page, dim], scale bytes [pages, 2, kv]) of a cache, as views."""
    body = _page_bytes(case)[1]
    shape = (pages.shape[0], 2, case["kv"], case["page"], case["dim"])
    values = pages.as_strided((pages.shape[0], body), (pages.stride(0), 1)).view(torch.float8_e4m3fn).unflatten(1, shape[1:])
    return values, pages[:, body:body + 2 * case["kv"]].unflatten(1, shape[1:3])


def _needed(amax):
    """The scale byte that values up to ``amax`` need: the smallest e in 1..247 with amax <= 448 * 2^(e - 127); 0 for zeros."""
    mantissa, exponent = torch.frexp(amax)                      # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent + 118 + (mantissa > 0.875).int()               # 448 = 0.875 * 2^9
    return torch.where(amax > 0, e.clamp(1, 247), torch.zeros_like(e))


def _power(e):
    """2^e for whole numbers e in -126..127, made of the bits of a float32."""
    return ((e + 127) << 23).view(torch.float32)


def _scales(byte):
    return (byte.int() << 23).view(torch.float32)               # byte 0: 0.0


# ---- a state -------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=device)

    kv, d, ps, dtype = case["kv"], case["dim"], case["page"], DTYPES[case["dtype"]]
    if case["kind"] == "pages":
        # bfloat16 pages [layers][pages, 2, kv, page, dim]; half of the pages are sources or destinations
        count, L = case["count"], case["layers"]
        total = 2 * count + 5
        order = torch.randperm(total, generator=g, device=device).tolist()
        pool = torch.empty((L, total, 2, kv, ps, d), dtype=torch.bfloat16, device=device).normal_(generator=g)
        src, dst = order[:count], order[count:2 * count]
        return {"case": case, "pool": pool, "tensors": list(pool.unbind(0)), "src": src, "dst": dst,
                "src_dev": torch.tensor(src, device=device), "dst_dev": torch.tensor(dst, device=device)}
    lens, starts = _lengths(case)
    total = [n + s for n, s in zip(lens, starts)]
    R, N = len(lens), sum(lens)
    held = [-(-t // ps) for t in total]
    width = max(held)
    P = sum(held) + 3
    ids = torch.randperm(P, generator=g, device=device)[:sum(held)].tolist()
    rows, at = [], 0
    for n in held:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    tables = torch.tensor(rows, dtype=torch.int32, device=device)
    # keys with channels of different sizes, values of even ones, pages of different sizes
    channel = torch.exp(0.8 * randn(kv, 1, d))
    pages = torch.zeros((P, _page_bytes(case)[0]), dtype=torch.uint8, device=device)
    values, scale = _views(pages, case)
    for first in range(0, P, 4096):
        part = slice(first, min(first + 4096, P))
        x = randn(part.stop - first, 2, kv, ps, d)
        x[:, 0] *= channel
        x *= torch.exp(0.5 * randn(part.stop - first, 2, kv, 1, 1))
        e = _needed(x.abs().amax((-2, -1)))
        scale[part] = e.to(torch.uint8)
        values[part] = (x * _power(127 - e)[..., None, None]).to(torch.float8_e4m3fn)
    state = {"case": case, "pages": pages, "tables": tables, "lens": lens, "starts": starts,
             "ctx_len": torch.tensor(total, dtype=torch.int32, device=device),
             "q_start": torch.tensor([sum(lens[:r]) for r in range(R + 1)], dtype=torch.int32, device=device)}
    request = torch.repeat_interleave(torch.arange(R, device=device), torch.tensor(lens, device=device))
    first_row = torch.tensor([sum(lens[:r]) for r in range(R)], device=device)
    start = torch.tensor(starts, device=device)
    position = torch.arange(N, device=device) - first_row[request] + start[request]
    state.update(request=request, position=position)
    # the rows of one product: queries, keys and values of a token side by side
    qkv = randn(N, (case["heads"] + 2 * kv) * d).to(dtype)
    state["qkv"] = qkv
    if case["kind"] == "store":
        page = tables.long()[request, position // ps]
        state["slots"] = (page * ps + position % ps).int()
        entries = sorted({r * width + t // ps for r in range(R) for t in range(starts[r], total[r])})
        state["index"] = torch.tensor(entries, dtype=torch.int32, device=device)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------

def _store(state):
    """Keys and values of the step's rows into their pages; the values of every page that was written, zeros behind the
    request's last token."""
    case, pages = state["case"], state["pages"]
    kv, d, ps, heads = case["kv"], case["dim"], case["page"], case["heads"]
    k, v = state["qkv"][:, heads * d:(heads + kv) * d], state["qkv"][:, (heads + kv) * d:]
    if own:
        from llm_pipeline_b200.ops import kernels

        kernels.kv8_store(k, v, state["slots"], pages, kv, d, ps)
        out = torch.empty((state["index"].numel(), 2, kv, ps, d), dtype=k.dtype, device=k.device)
        return kernels.kv8_gather(pages, state["tables"], state["ctx_len"], state["index"], out)
    values, scale = _views(pages, case)
    x = torch.stack([k, v], 1).unflatten(2, (kv, d)).float()                     # [N, 2, kv, d]
    finite = x.isfinite()
    slots = state["slots"].long()
    page, offset = slots // ps, slots % ps
    P = pages.shape[0]
    amax = torch.zeros((P, 2, kv), device=x.device).index_reduce_(0, page, torch.where(finite, x, torch.zeros_like(x)).abs().amax(-1), "amax")
    first = torch.full((P,), ps, device=x.device).index_reduce_(0, page, offset, "amin")        # offset of a page's first new token
    touched = state["tables"].flatten()[state["index"].long()].long()
    need, first = _needed(amax[touched]), first[touched]
    old = scale[touched].int()
    e = torch.where(first[:, None, None] > 0, torch.maximum(need, old), need)
    earlier = torch.arange(ps, device=x.device) < first[:, None]                                # [touched, ps]
    held = values[touched]
    moved = (held.float() * _power((old - e).clamp(min=-126))[..., None, None]).to(torch.float8_e4m3fn)
    held = torch.where((earlier[:, None, None, :] & (e > old)[..., None])[..., None], moved.view(torch.uint8), held.view(torch.uint8))
    values.view(torch.uint8)[touched] = held
    scale[touched] = e.to(torch.uint8)
    up = _power(127 - scale[page].int())[..., None]
    q = torch.where(finite, x * up, torch.full_like(x, math.nan)).to(torch.float8_e4m3fn)
    values.view(torch.uint8)[page, :, :, offset] = q.view(torch.uint8)
    index, width = state["index"].long(), state["tables"].shape[1]
    there = index[:, None] % width * ps + torch.arange(ps, device=x.device) < state["ctx_len"][index // width][:, None]
    now = values[touched].float() * _scales(scale[touched])[..., None, None]
    return torch.where(there[:, None, None, :, None], now, torch.zeros_like(now)).to(k.dtype)


def _attend(state):
    """Causal attention of the step's rows over the keys and values of their requests' pages."""
    case = state["case"]
    heads, kv, d, ps, window = case["heads"], case["kv"], case["dim"], case["page"], case["window"]
    q, lens, starts = state["qkv"], state["lens"], state["starts"]
    N, scale = q.shape[0], d ** -0.5
    if own:
        from llm_pipeline_b200.ops import kernels, kv8

        out = torch.empty((N, heads * d), dtype=q.dtype, device=q.device)
        if case["kind"] == "decode":
            return kernels.kv8_decode_attention(q, q.stride(0), out, state["pages"], state["tables"], state["ctx_len"], max(starts) + 1,
                                                heads, kv, d, ps, window, scale)
        if "plan" not in state:                       # one for all layers of a step
            state["plan"] = kv8.PromptPlan(starts, lens, heads, kv, d, ps, window, q.dtype, q.device)
        return kv8.prompt_attention(state["plan"], q, q.stride(0), out, state["pages"], state["tables"], state["q_start"],
                                    state["ctx_len"], scale)
    values, scales = _views(state["pages"], case)
    tables = state["tables"].long()
    R, width = tables.shape
    there = tables.clamp(min=0)
    T, most = width * ps, max(lens)
    held = values[there].float() * _scales(scales[there])[..., None, None]       # [R, width, 2, kv, ps, d]
    k, v = held.permute(2, 0, 3, 1, 4, 5).reshape(2, R, kv, T, d).unbind(0)
    place = state["position"] - torch.tensor(starts, device=q.device)[state["request"]]
    rows = torch.zeros((R, most, heads * d), device=q.device)
    rows[state["request"], place] = q[:, :heads * d].float()
    rows = rows.view(R, most, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(R, kv, heads // kv * most, d)
    s = (rows @ k.transpose(2, 3)).view(R, kv, heads // kv, most, T) * scale
    at = torch.tensor(starts, device=q.device)[:, None] + torch.arange(most, device=q.device)   # [R, most]
    j = torch.arange(T, device=q.device)
    seen = (j <= at[..., None]) & (j < state["ctx_len"][:, None, None])
    if window:
        seen &= j > at[..., None] - window
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    w = torch.exp_(s.sub_(s.amax(-1, keepdim=True).clamp_(min=-3e38)))
    w = w.div_(w.sum(-1, keepdim=True).clamp_(min=1e-30))
    o = (w.view(R, kv, -1, T) @ v).view(R, kv, heads // kv, most, d).permute(0, 3, 1, 2, 4).reshape(R, most, heads * d)
    return o[state["request"], place].to(q.dtype)


def _copy(state):
    """Pages ``src`` of every layer's cache to ``dst``; the caches."""
    if own:
        from llm_pipeline_b200.ops import kernels

        kernels.copy_pages(state["tensors"], state["src"], state["dst"])
    else:
        state["pool"][:, state["dst_dev"]] = state["pool"][:, state["src_dev"]]
    return state["tensors"]


@torch.no_grad()
def run(state):
    kind = state["case"]["kind"]
    if kind == "store":
        return {"values": _store(state)}
    if kind == "pages":
        return {"pages": _copy(state)}
    return {"rows": _attend(state)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def work(case):
    kv, d, ps, size = case["kv"], case["dim"], case["page"], DTYPES[case["dtype"]].itemsize
    if case["kind"] == "pages":
        return {"bytes": 2 * case["count"] * case["layers"] * 2 * kv * ps * d * 2, "flops": 0}
    lens, starts = _lengths(case)
    N = sum(lens)
    if case["kind"] == "store":
        # rows in, their 8 bits out; the written pages in (what they held before, then as they are) and their values out
        touched = sum(-(-(s + n) // ps) - s // ps for n, s in zip(lens, starts))
        return {"bytes": 2 * kv * d * (N * (size + 1) + touched * ps * (1 + size)), "flops": 0}
    window = case["window"] or 1 << 40
    pairs = keys = 0
    for n, s in zip(lens, starts):
        pairs += sum(min(p + 1, window) for p in range(s, s + n))
        keys += s + n - max(0, s - window + 1)
    return {"bytes": keys * 2 * kv * (d + 1 / ps) + 2 * N * case["heads"] * d * size, "flops": 4.0 * pairs * case["heads"] * d}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------------

def _two_to(n):
    """2^n in 64 bits for whole numbers n (a power function may miss the last bit, which decides what a tie rounds to)."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _decode_bytes(byte):
    """What bytes in e4m3 stand for: sign, four bits of exponent (bias 7, 0: subnormal), three of mantissa; 0x7f: no number."""
    byte = byte.long()
    exponent, mantissa = byte >> 3 & 15, (byte & 7).double()
    value = torch.where(exponent > 0, (8 + mantissa) * _two_to(exponent - 10), mantissa * 2.0 ** -9)
    value = torch.where((byte & 127) == 127, torch.full_like(value, math.nan), value)
    return torch.where(byte >= 128, -value, value)


def _nearest(y):
    """The nearest value in e4m3 (ties to an even mantissa) of numbers of at most 448."""
    step = _two_to(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return torch.round(y / step) * step


def _exact_pages(pages, ids, case):
    """Values [ids, 2, kv, page, dim] of pages in 64 bits."""
    body, kv = _page_bytes(case)[1], case["kv"]
    raw = pages[ids]
    e = raw[:, body:body + 2 * kv].long().view(len(ids), 2, kv, 1, 1)
    scale = torch.where(e > 0, _two_to(e - 127), torch.zeros_like(e).double())
    return _decode_bytes(raw[:, :body]).view(len(ids), 2, kv, case["page"], case["dim"]) * scale


def _exact_store(state):
    case = state["case"]
    kv, d, ps, heads = case["kv"], case["dim"], case["page"], case["heads"]
    x = state["qkv"][:, heads * d:].double().view(-1, 2, kv, d)
    tables, out, row = state["tables"].tolist(), [], 0
    for r, (n, s) in enumerate(zip(state["lens"], state["starts"])):
        for first in range(s // ps * ps, s + n, ps):
            id_ = torch.tensor([tables[r][first // ps]], device=x.device)
            held = _exact_pages(state["pages"], id_, case)[0]
            lo, hi = max(first, s), min(first + ps, s + n)
            new = x[row:row + hi - lo].permute(1, 2, 0, 3)                       # [2, kv, tokens, d]
            row += hi - lo
            top = new.abs().amax((-2, -1))
            e = torch.ceil(torch.log2(top / 448.0)).clamp(-126, 120)             # in 64 bits exact enough to be checked below
            e = torch.where(top <= 448 * _two_to(e - 1), e - 1, torch.where(top > 448 * _two_to(e), e + 1, e)).clamp(-126, 120)
            if lo > first:
                body = _page_bytes(case)[1]
                old = state["pages"][id_, body:body + 2 * kv].double().view(2, kv) - 127
                e = torch.maximum(e, old)
            scale = _two_to(e)[..., None, None]
            if lo > first:
                held[:, :, :lo - first] = _nearest(held[:, :, :lo - first] / scale) * scale
            held[:, :, lo - first:hi - first] = _nearest(new / scale) * scale
            held[:, :, hi - first:] = 0
            out.append(held)
    return torch.stack(out)


def _exact_attend(state):
    case = state["case"]
    heads, kv, d, ps = case["heads"], case["kv"], case["dim"], case["page"]
    q = state["qkv"][:, :heads * d].double().view(-1, kv, heads // kv, d)
    out, row = [], 0
    for r, (n, s) in enumerate(zip(state["lens"], state["starts"])):
        T = s + n
        held = _exact_pages(state["pages"], state["tables"][r, :-(-T // ps)].long(), case)
        k, v = held.permute(1, 2, 0, 3, 4).reshape(2, kv, -1, d)[:, :, :T].unbind(0)
        j = torch.arange(T, device=q.device)
        for at in range(0, n, 256):
            m = min(256, n - at)
            i = s + at + torch.arange(m, device=q.device)[:, None]
            scores = torch.einsum("mkgd,ktd->kgmt", q[row + at:row + at + m], k) / math.sqrt(d)
            hidden = j > i
            if case["window"]:
                hidden = hidden | (j <= i - case["window"])
            w = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
            out.append(torch.einsum("kgmt,ktd->mkgd", w, v).reshape(m, heads * d))
        row += n
    return torch.cat(out)


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "store":
        return {"values": _exact_store(state)}
    if case["kind"] == "pages":
        moved = dict(zip(state["dst"], state["src"]))
        where = torch.tensor([moved.get(p, p) for p in range(state["pool"].shape[1])], device=state["pool"].device)
        return {"pages": [t[where] for t in state["tensors"]]}
    return {"rows": _exact_attend(state)}
