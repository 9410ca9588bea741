"""Attention of prompt portions over pages of 8-bit keys and values (``cache.spec.KV8PagesSpec``).

bfloat16 queries of head size 128 go to a kernel that reads the pages as they are (``kernels.kv8_prompt_attention``) where that is
faster: few queries over many keys above all (``reads_pages_directly``). For all others the pages that a step's portions see are
unpacked into a workspace of the query's type, laid out as ordinary pages, and the attention kernels of ordinary pages run over it
(``kernels.paged_attention``): a page's values are exact in either type (the scales are powers of two), so the result is exactly what
they give for a cache that holds these values, their weights in bfloat16 included (2^-8 of sum w |v|; the kernel that reads the pages has
them in half precision, 2^-11). A value that is no number makes the whole rows of its head's group that see its token no
numbers either way, and no others (single tokens: the entries of its column)."""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import kernels

WORKSPACE_BYTES = 1 << 30            # unpacked pages, and sums of items: requests (or parts of tiles) that pass this together take turns (or are not cut)
KEY_TILE = 128                       # keys of a tile of the kernel that reads 8-bit pages
# Key tiles of a part at least where a tile's keys are shared among items, which costs a launch and the sums' way through memory.
PART_TILES = 4


def tiles_of(starts: Sequence[int], q_lens: Sequence[int], first_request: int, tokens: int, window: int) -> List[Tuple[int, int, int]]:
    """(key tiles, request, first token) of every ``tokens`` new tokens of a request."""
    tiles = []
    for r in range(first_request, len(q_lens)):
        for t in range(0, q_lens[r], tokens):
            last = starts[r] + min(t + tokens, q_lens[r]) - 1
            low = max(starts[r] + t - window + 1, 0) if window else 0
            tiles.append((last // KEY_TILE + 1 - low // KEY_TILE, r, t))
    return tiles


def plan_items(starts: Sequence[int], q_lens: Sequence[int], first_request: int, tokens: int, num_kv_heads: int, window: int, sms: int,
               most_places: int) -> Tuple[List[List[int]], List[List[int]], int]:
    """(items, shared, places) for ``kernels.kv8_prompt_attention``: every ``tokens`` new tokens of a request are a tile, whose keys come
    in parts, as many as still give every part and key/value head an SM of its own (few new tokens over many keys). The items that
    see most keys come first."""
    tiles = tiles_of(starts, q_lens, first_request, tokens, window)
    parts = [1] * len(tiles)
    if tiles and len(tiles) * num_kv_heads <= sms:
        low, high = PART_TILES, max(PART_TILES, max(n for n, _r, _t in tiles))
        while low < high:                            # the fewest key tiles a part for which all parts run side by side
            share = (low + high) // 2
            if sum(-(-n // share) for n, _r, _t in tiles) * num_kv_heads <= sms:
                high = share
            else:
                low = share + 1
        parts = [-(-n // low) for n, _r, _t in tiles]
        if sum(k for k in parts if k > 1) > most_places:
            parts = [1] * len(tiles)
    items, shared, places = [], [], 0
    for i in sorted(range(len(tiles)), key=lambda i: (-tiles[i][0] / parts[i], tiles[i][1:])):
        _n, r, t = tiles[i]
        for k in range(parts[i]):
            items.append([r, t, k | parts[i] << 16, places + k if parts[i] > 1 else 0])
        if parts[i] > 1:
            shared.append([r, t, parts[i], places])
            places += parts[i]
    return items, shared, places


def reads_pages_directly(starts: Sequence[int], q_lens: Sequence[int], first_request: int, num_heads: int, num_kv_heads: int, window: int,
                         sms: int) -> bool:
    """Whether a step's portions are better served by the kernel that reads 8-bit pages (256 query rows an item, its bytes unpacked in
    every one) than by unpacking the pages once and the attention kernel of ordinary pages (128 rows, two of them on an SM; keys
    shared by at most 8 items of at least 16 tiles). By what each takes, in us on a B200 (head size 128, 8 key/value heads):
    18 and the longer of 2.75 a key tile of the longest part and 3.2 for every key tile an SM has, against 8, 1.9 for every 1,000 tokens of
    the pages, and the longer of 2.8 a key tile of the longest item and 1.3 for every key tile an SM has, with up to 18 for the end. Measured
    (direct, unpacked), 32 query heads: 40 new tokens behind 8,000 31, 71; 128 behind 2,000 29, 48; 512 behind 8,000 113, 131; 1,024 behind
    8,000 206, 209; 2,048 new ones 65, 66; 64 behind 500 24, 21; 1,000 new ones 34, 30; 4,000 new ones 195, 179; 2,048 behind 14,000 644, 638. Other
    groups (8, 16 and 64 heads on 8, 32 on 4, 9 and 16 on 1), the worst of nine mixes of lengths each: 64 behind 500 on 16 and 8 heads 18.5, 21.9 (taken:
    unpacked), 512 behind 8,000 on 32 and 4 110, 125 (unpacked), 1,000 new ones on 9 and 1 29.6, 26.3 (direct)."""
    group = num_heads // num_kv_heads
    wide = tiles_of(starts, q_lens, first_request, max(1, 256 // group), window)
    if not wide:
        return False
    longest, places = 0, plan_items(starts, q_lens, first_request, max(1, 256 // group), num_kv_heads, window, sms, 1 << 30)[1]
    cut = {(r, t): k for r, t, k, _p in places}
    for n, r, t in wide:
        longest = max(longest, -(-n // cut.get((r, t), 1)))
    direct = 2.75 * longest
    if len(wide) * num_kv_heads > sms:
        direct = max(direct, 3.2 * sum(n for n, _r, _t in wide) * num_kv_heads / sms)
    narrow = tiles_of(starts, q_lens, first_request, max(1, 128 // group), window)
    blocks, most = len(narrow) * num_kv_heads, max(n for n, _r, _t in narrow)
    segments = min(8, 4 * sms // blocks, most // 16) if blocks <= sms else 1
    tokens = sum(s + n - (max(0, s - window + 1) if window else 0) for s, n in zip(starts[first_request:], q_lens[first_request:]) if n)
    unpacked = max(2.8 * -(-most // max(1, segments)), 1.3 * sum(n for n, _r, _t in narrow) * num_kv_heads / sms + min(1.1 * most, 18))
    return 18 + direct < 8 + 1.9e-3 * tokens * num_kv_heads / 8 + unpacked


class PromptPlan:
    """What a step's prompt attention needs besides its tensors. One plan serves every layer of a step with the same heads, head size,
    page size and window. ``starts`` and ``q_lens``: cached tokens and new tokens of every request, as host numbers; the requests
    before ``first_request`` are left out (their rows of the output are not written). Its lists are made on the stream that is
    current when it is first used; a call on another stream waits for that one. A captured call needs a plan that was used before with
    tables of the same width, and the plan has to live as long as the graph."""

    def __init__(self, starts: Sequence[int], q_lens: Sequence[int], num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                 window: int, dtype: torch.dtype, device: torch.device, first_request: int = 0):
        if len(starts) != len(q_lens) or any(n < 0 for n in q_lens) or any(s < 0 for s in starts):
            raise kernels.KernelError("a plan needs the cached and the new tokens of every request")
        if num_kv_heads <= 0 or num_heads <= 0 or num_heads % num_kv_heads:
            raise kernels.KernelError(f"{num_heads} query heads cannot share {num_kv_heads} key/value heads")
        if page_size <= 0 or window < 0 or not 0 <= first_request <= len(q_lens):
            raise kernels.KernelError("a plan needs a positive page size, a window of at least 0 and a first request of the step")
        self.starts, self.q_lens = [int(s) for s in starts], [int(n) for n in q_lens]
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.page_size, self.window, self.dtype, self.device = page_size, window, dtype, torch.device(device)
        self.first_request = first_request
        self.rows = sum(self.q_lens)
        # The first row where all portions are single tokens: the kernel for those takes them (behind 4,934 tokens, 3 requests of 12 and 2
        # heads of 64: 132 us as portions, whose keys only some sizes share among blocks, 14 as single tokens). A step of the engine has its
        # single tokens in front, where `first_request` leaves them out.
        self.single = sum(self.q_lens[:first_request]) if all(n == 1 for n in self.q_lens[first_request:]) else None
        self.longest = max((s + n for s, n in zip(self.starts, self.q_lens)), default=0)
        self.page_bytes = 2 * num_kv_heads * page_size * head_dim * dtype.itemsize
        self.groups = self._groups()
        self._lists: Dict[int, list] = {}            # by the width of the block tables
        self._items = None
        self._direct = None
        self._made: Optional[torch.cuda.Stream] = None          # the stream the lists were made on

    def direct(self) -> bool:
        """Whether the portions go to the kernel that reads 8-bit pages (sizes it takes, and ``reads_pages_directly``)."""
        if self._direct is None:                     # (asked once a plan, that is once a step)
            self._direct = kernels.kv8_prompt_supports(self.dtype, self.num_heads, self.num_kv_heads, self.head_dim, self.page_size) and \
                reads_pages_directly(self.starts, self.q_lens, self.first_request, self.num_heads, self.num_kv_heads, self.window, kernels.sm_count())
        return self._direct

    def pages_of(self, r: int) -> Tuple[int, int]:
        """The pages (first, end) of request r that its new tokens see."""
        first = max(0, self.starts[r] - self.window + 1) if self.window else 0
        return first // self.page_size, -(-(self.starts[r] + self.q_lens[r]) // self.page_size)

    def _groups(self) -> List[List[int]]:
        """The requests with new tokens, in runs whose unpacked pages fit the workspace together (a request alone may pass it)."""
        groups: List[List[int]] = []
        room = 0
        for r in range(self.first_request, len(self.q_lens)):
            if self.q_lens[r] == 0:
                continue
            first, end = self.pages_of(r)
            size = (end - first) * self.page_bytes
            if not groups or size > room:
                groups.append([])
                room = WORKSPACE_BYTES
            groups[-1].append(r)
            room -= size
        return groups

    def _on_device(self, lists: Sequence[torch.Tensor]) -> List[torch.Tensor]:
        """The int32 lists through one pinned copy, each from a multiple of 16 bytes on."""
        if kernels._capturing():
            raise kernels.KernelError("a plan's lists must exist before a graph is captured: call it once with this step's tables before")
        padded = [torch.nn.functional.pad(t.flatten(), (0, -t.numel() % 4)) for t in lists]
        stream = torch.cuda.current_stream(self.device)
        if self._made is not None and self._made != stream:
            stream.wait_stream(self._made)           # this stream's work then comes behind all lists, whichever it waits for later
        self._made = stream
        dev, at, out = torch.cat(padded).pin_memory().to(self.device, non_blocking=True), 0, []
        for t, room in zip(lists, padded):
            out.append(dev[at:at + t.numel()].view(t.shape))
            at += room.numel()
        return out

    def _for_this_stream(self, lists: Sequence[Optional[torch.Tensor]]) -> None:
        """Before work on another stream than the lists' own: it comes behind them, and their memory is not given away before its end."""
        if kernels._stream() == self._made.cuda_stream or kernels._capturing():      # (a capture begins with an idle device)
            return
        stream = torch.cuda.current_stream(self.device)
        stream.wait_stream(self._made)
        for t in lists:
            if t is not None:
                t.record_stream(stream)

    def items(self):
        """(items, shared, places) on the device for the kernel that reads 8-bit pages."""
        if self._items is None:
            tokens, floats = kernels.kv8_prompt_sizes(self.num_heads, self.num_kv_heads)
            items, shared, places = plan_items(self.starts, self.q_lens, self.first_request, tokens, self.num_kv_heads, self.window,
                                               kernels.sm_count(), WORKSPACE_BYTES // (4 * floats))
            lists = [torch.tensor(rows, dtype=torch.int32).reshape(len(rows), 4) for rows in (items, shared)]
            self._items = (*self._on_device(lists), places)
        return self._items

    def lists(self, table_width: int) -> list:
        """Per group: (entries of the block tables to unpack, block tables of the workspace, tile_req, tile_tok0, tile_seg, tile_slot,
        places, tokens per tile), on the device."""
        made = self._lists.get(table_width)
        if made is not None:
            return made
        from ..parts.attention import AttentionPolicy

        R, made = len(self.q_lens), []
        sizes = (self.num_heads, self.num_kv_heads, self.dtype, self.head_dim, self.page_size)
        tokens, segments = kernels.tokens_per_attention_tile(*sizes), kernels.attention_max_segments(*sizes)
        for group in self.groups:
            width = max(self.pages_of(r)[1] for r in group)
            index: List[int] = []
            tables = torch.full((R, width), -1, dtype=torch.int32)
            for r in group:
                first, end = self.pages_of(r)
                tables[r, first:end] = torch.arange(len(index), len(index) + end - first, dtype=torch.int32)
                index.extend(range(r * table_width + first, r * table_width + end))
            mine = set(group)
            alone = [n if r in mine else 0 for r, n in enumerate(self.q_lens)]
            req, tok0, seg, slot, places = AttentionPolicy.plan_items(self.starts, alone, tokens, 0, segments, self.num_kv_heads,
                                                                      kernels.sm_count())
            lists = [torch.tensor(index, dtype=torch.int32), tables] + [torch.tensor(x, dtype=torch.int32) for x in (req, tok0, seg, slot)]
            made.append((*self._on_device(lists)[:4 if not places else 6], *(() if places else (None, None)), places, tokens))
        self._lists[table_width] = made
        return made


def prompt_attention(plan: PromptPlan, q: torch.Tensor, q_stride: int, out: torch.Tensor, pages: torch.Tensor, block_tables: torch.Tensor,
                     q_start: torch.Tensor, ctx_len: torch.Tensor, scale: float) -> torch.Tensor:
    """Causal attention of the step's query rows over 8-bit pages, any portion sizes: as ``kernels.paged_attention`` over pages
    that hold the same values in q's type. ``q_start`` and ``ctx_len`` are the plan's lengths on the device. Every page that the new
    tokens see has to be there."""
    nq, nkv, d, ps = plan.num_heads, plan.num_kv_heads, plan.head_dim, plan.page_size
    kernels._kv8_pages(pages, nkv, d, ps)
    if q.dtype != plan.dtype:
        raise kernels.KernelError(f"the plan is for queries in {plan.dtype}")
    R = len(plan.q_lens)
    if not (block_tables.dim() == 2 and block_tables.shape[0] == R == ctx_len.numel() and q_start.numel() == R + 1):
        raise kernels.KernelError("block tables, q_start and ctx_len must be those of the plan's requests")
    if not (q.dim() == 2 and q.shape[1] >= nq * d and (q.shape[0] <= 1 or (q.stride(1) == 1 and q.stride(0) == q_stride))):
        raise kernels.KernelError("query rows must hold the plan's heads and lie q_stride apart")
    if q.shape[0] < plan.rows or out.shape[0] < plan.rows:
        raise kernels.KernelError("the plan has more rows than the queries or the output")
    if block_tables.shape[1] * ps < plan.longest:
        raise kernels.KernelError(f"a request sees {plan.longest} tokens, its block table has room for {block_tables.shape[1] * ps}")
    if not 0.0 < scale < float("inf"):                 # (the kernel over ordinary pages takes a row's largest score before it scales it)
        raise kernels.KernelError(f"the scale of a prompt's scores must be positive and finite, not {scale}")
    if not plan.groups:
        return out
    if plan.single is not None:
        at, r = plan.single, plan.first_request
        kernels.kv8_decode_attention(q[at:plan.rows], q_stride, out[at:plan.rows], pages, block_tables[r:], ctx_len[r:], plan.longest, nq, nkv, d, ps, plan.window,
                                     scale)
        return out
    if plan.direct() and (q.data_ptr() | 2 * q_stride | out.data_ptr()) % 16 == 0:
        items, shared, places = plan.items()
        plan._for_this_stream((items, shared))
        return kernels.kv8_prompt_attention(q, q_stride, out, pages, block_tables, q_start, ctx_len, items, shared, places, nq, nkv, ps,
                                            plan.window, scale)
    kernels._on_current_device(q, out, pages, block_tables, q_start, ctx_len)
    for index, tables, req, tok0, seg, slot, places, tokens in plan.lists(block_tables.shape[1]):
        plan._for_this_stream((index, tables, req, tok0, seg, slot))
        held = torch.empty((index.numel(), 2, nkv, ps, d), dtype=q.dtype, device=q.device)
        kernels.kv8_gather(pages, block_tables, ctx_len, index, held, hide=True)
        kernels.paged_attention(q, q_stride, out, held, tables, q_start, ctx_len, req, tok0, nq, nkv, d, ps, plan.window, scale, tokens,
                                seg, slot, places)
    return out
