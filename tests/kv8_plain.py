"""Pages of 8-bit keys and values in plain form, in 64 bits and row by row, for the tests."""

import math

import torch


def page_bytes(nkv, page_size, d):
    return -(-(2 * nkv * (page_size * d + 1)) // 128) * 128


def power(n):
    """2^n in 64 bits, exactly, for whole numbers (a tensor or a number)."""
    n = torch.as_tensor(n)
    return torch.ldexp(torch.ones(n.shape, dtype=torch.float64), n.to(torch.int32)) if n.device.type == "cpu" else power(n.cpu()).to(n.device)


# e4m3 from its definition: a sign, four bits of exponent (bias 7; 0: subnormal), three of mantissa; 0x7f: no number
E4M3 = torch.tensor([math.nan if b & 127 == 127 else
                     (-1.0 if b & 128 else 1.0) * ((8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10) if b >> 3 & 15 else (b & 7) * 2.0 ** -9)
                     for b in range(256)], dtype=torch.float64)


def nearest(y):
    """Bytes of the e4m3 values nearest to y (magnitudes up to 448; ties to an even mantissa); NaN to 0x7f."""
    y = y.double().cpu()
    steps = E4M3[:127]
    a = y.abs().clamp(max=448.0)
    hi = torch.searchsorted(steps, a.nan_to_num(0.0)).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = steps[hi] - a, a - steps[lo]
    take_lo = (down < up) | ((down == up) & (lo % 2 == 0))
    byte = torch.where(take_lo, lo, hi)
    byte = torch.where(a == steps[hi], hi, byte)
    byte = torch.where(torch.signbit(y), byte | 128, byte)
    return torch.where(y.isnan(), torch.full_like(byte, 127), byte).to(torch.uint8)


def needed(amax):
    """The smallest e in 1..247 with amax <= 448 * 2^(e - 127); 0 for 0. A python number."""
    if amax == 0:
        return 0
    e = 1
    while e < 247 and amax > math.ldexp(448.0, e - 127):
        e += 1
    return e


class Pages:
    """A cache on the host: bytes [P, 2, nkv, page_size, d] and scale bytes [P, 2, nkv]."""

    def __init__(self, P, nkv, page_size, d, raw=None):
        self.sizes = (P, nkv, page_size, d)
        self.body = 2 * nkv * page_size * d
        self.raw = torch.zeros(P, page_bytes(nkv, page_size, d), dtype=torch.uint8) if raw is None else raw.cpu().clone()
        self.q = self.raw[:, :self.body].view(P, 2, nkv, page_size, d)
        self.e = self.raw[:, self.body:self.body + 2 * nkv].view(P, 2, nkv)

    def store(self, k, v, slots):
        P, nkv, ps, d = self.sizes
        rows = [(i, int(s)) for i, s in enumerate(slots) if 0 <= int(s) < P * ps]
        x = torch.stack([k.double().cpu().view(-1, nkv, d), v.double().cpu().view(-1, nkv, d)], 1)
        at = 0
        while at < len(rows):
            page = rows[at][1] // ps
            end = at
            while end < len(rows) and rows[end][1] // ps == page:
                end += 1
            run, first = rows[at:end], min(s % ps for _i, s in rows[at:end])
            at = end
            new = x[[i for i, _s in run]]                                        # [run, 2, nkv, d]
            for kv in range(2):
                for h in range(nkv):
                    y = new[:, kv, h]
                    finite = y.isfinite()
                    e = needed(float(torch.where(finite, y, torch.zeros_like(y)).abs().max()))
                    old = int(self.e[page, kv, h])
                    if first > 0 and old >= e:
                        e = old
                    elif first > 0:
                        held = E4M3[self.q[page, kv, h, :first].long()]
                        self.q[page, kv, h, :first] = nearest(held * power(max(old - e, -126)))
                    self.e[page, kv, h] = e
                    for (_i, s), row, ok in zip(run, y, finite):
                        self.q[page, kv, h, s % ps] = nearest(torch.where(ok, row * power(127 - e), torch.full_like(row, math.nan)))

    def values(self, ids):
        """float64 [ids, 2, nkv, page_size, d]"""
        e = self.e[ids].int()
        scale = torch.where(e > 0, power(e - 127), torch.zeros(e.shape, dtype=torch.float64))
        return E4M3[self.q[ids].long()] * scale[..., None, None]

    def value_scales(self, table, ctx):
        """[ctx, nkv]: what the bytes of a request's values are to be multiplied by (1 for blocks of zeros and missing pages)."""
        P, nkv, ps, d = self.sizes
        ids = [int(p) if 0 <= int(p) < P else -1 for p in table[:-(-ctx // ps)]]
        if not ids:
            return torch.zeros(0, nkv, dtype=torch.float64)
        e = self.e[[max(i, 0) for i in ids], 1].int()
        e = torch.where((e > 0) & (torch.tensor(ids)[:, None] >= 0), e, torch.full_like(e, 127))
        return power(e - 127).repeat_interleave(ps, 0)[:ctx]

    def request(self, table, ctx):
        """Keys and values [ctx, nkv, d] of a request and which of its keys are there (a page may be missing)."""
        P, nkv, ps, d = self.sizes
        table = [int(p) for p in table[:-(-ctx // ps)]]
        there = torch.tensor([0 <= p < P for p in table], dtype=torch.bool).repeat_interleave(ps)[:ctx]
        held = self.values([p if 0 <= p < P else 0 for p in table]) if table else torch.zeros(0, 2, nkv, ps, d, dtype=torch.float64)
        k, v = held.permute(1, 0, 3, 2, 4).reshape(2, -1, nkv, d)[:, :ctx].unbind(0)
        return k, v, there


def smallest(q, k, v, v_scales, position, there, scale, window):
    """[nq, d]: 2^-25 max_j(w_j s_j) sum_j |b_j| of one row, with v_j = s_j b_j: what weights times the values' scales may be off by where
    they are held in half precision relative to the largest of them (numbers below 2^-14 are 2^-24 apart)."""
    nq, d = q.shape
    T, nkv, _ = k.shape
    j = torch.arange(T)
    seen = there & (j <= position) & ((j > position - window) if window else (j >= 0))
    if not bool(seen.any()):
        return torch.zeros(nq, d, dtype=torch.float64)
    G = nq // nkv
    kk, s = k[seen].repeat_interleave(G, 1), v_scales[seen].repeat_interleave(G, 1)
    w = torch.softmax(torch.einsum("hd,thd->ht", q.double().cpu(), kk) * scale, -1)
    b = (v[seen] / v_scales[seen][..., None]).abs().sum(0).repeat_interleave(G, 0)
    return 2.0 ** -25 * (w * s.t()).amax(-1, keepdim=True) * b


def attend(q, k, v, positions, there, scale, window):
    """q [n, nq, d] at ``positions`` over k, v [T, nkv, d]: (rows [n, nq, d], the same with magnitudes of the values: sum w |v|,
    the largest sum of magnitudes scale * sum |q| |k| of a row's keys). Keys that are not there, later ones and those before the window are
    left out before anything is computed with them; rows without keys are zeros."""
    n, nq, d = q.shape
    T, nkv, _ = k.shape
    q = q.double().cpu()
    out, size, top = torch.zeros(n, nq, d, dtype=torch.float64), torch.zeros(n, nq, d, dtype=torch.float64), torch.zeros(n, nq, 1, dtype=torch.float64)
    for i in range(n):
        j = torch.arange(T)
        seen = there & (j <= positions[i]) & ((j > positions[i] - window) if window else (j >= 0))
        if not bool(seen.any()):
            continue
        kk, vv = k[seen].repeat_interleave(nq // nkv, 1), v[seen].repeat_interleave(nq // nkv, 1)
        s = torch.einsum("hd,thd->ht", q[i], kk) * scale
        w = torch.softmax(s, -1)
        out[i] = torch.einsum("ht,thd->hd", w, vv)
        size[i] = torch.einsum("ht,thd->hd", w, vv.abs())
        top[i, :, 0] = (torch.einsum("hd,thd->ht", q[i].abs(), kk.abs()) * scale).amax(-1)
    return out, size, top
