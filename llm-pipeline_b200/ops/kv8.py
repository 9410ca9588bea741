"""Attention of prompt portions over pages of 8-bit keys and values (``cache.spec.KV8PagesSpec``).

A page's values are exact in bfloat16 and float32 (the scales are powers of two), and the row tiles of a portion read the
same pages many times. So the pages that a step's portions see are unpacked once per layer into a workspace of the
query's type, laid out as ordinary pages, and the attention kernels of ordinary pages run over it
(``kernels.paged_attention``): the result is exactly what they give for a cache that holds these values. Unpacking moves
three bytes a value; 2,048 new tokens of a group of four heads compute 16,384 products with it."""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import kernels

WORKSPACE_BYTES = 1 << 30            # requests whose unpacked pages pass this together take turns in the workspace


class PromptPlan:
    """What a step's prompt attention needs besides its tensors: which pages are unpacked to where, and the work list of the
    attention kernel. One plan serves every layer of a step with the same heads, head size, page size and window.
    ``starts`` and ``q_lens``: cached tokens and new tokens of every request, as host numbers; the requests before ``first_request``
    are left out (their rows of the output are not written). Its lists are made on the stream that is current when it is first used."""

    def __init__(self, starts: Sequence[int], q_lens: Sequence[int], num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                 window: int, dtype: torch.dtype, device: torch.device, first_request: int = 0):
        if len(starts) != len(q_lens) or any(n < 0 for n in q_lens) or any(s < 0 for s in starts):
            raise kernels.KernelError("a plan needs the cached and the new tokens of every request")
        if page_size <= 0 or window < 0 or not 0 <= first_request <= len(q_lens):
            raise kernels.KernelError("a plan needs a positive page size, a window of at least 0 and a first request of the step")
        self.starts, self.q_lens = [int(s) for s in starts], [int(n) for n in q_lens]
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.page_size, self.window, self.dtype, self.device = page_size, window, dtype, torch.device(device)
        self.first_request = first_request
        self.page_bytes = 2 * num_kv_heads * page_size * head_dim * dtype.itemsize
        self.groups = self._groups()
        self._lists: Dict[int, list] = {}            # by the width of the block tables

    def pages_of(self, r: int) -> Tuple[int, int]:
        """The pages (first, end) of request r that its new tokens see."""
        first = max(0, self.starts[r] - self.window + 1) if self.window else 0
        return first // self.page_size, -(-(self.starts[r] + self.q_lens[r]) // self.page_size)

    def _groups(self) -> List[List[int]]:
        """The requests with new tokens, in runs whose pages fit the workspace together (a request alone may pass it)."""
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
            kernels._need(width <= table_width, f"a request sees {width} pages, its block table has {table_width}")
            index: List[int] = []
            tables = torch.full((R, width), -1, dtype=torch.int32)
            for r in group:
                first, end = self.pages_of(r)
                tables[r, first:end] = torch.arange(len(index), len(index) + end - first, dtype=torch.int32)
                index.extend(range(r * table_width + first, r * table_width + end))
            alone = [n if r in set(group) else 0 for r, n in enumerate(self.q_lens)]
            req, tok0, seg, slot, places = AttentionPolicy.plan_items(self.starts, alone, tokens, 0, segments, self.num_kv_heads,
                                                                      kernels.sm_count())
            rows = [req, tok0] + ([seg, slot] if places else [])
            flat = torch.cat([torch.tensor(index, dtype=torch.int32), tables.flatten(), torch.tensor(rows, dtype=torch.int32).flatten()])
            dev = flat.pin_memory().to(self.device, non_blocking=True)
            at = len(index)
            items = dev[at + R * width:].view(len(rows), len(req))
            made.append((dev[:at], dev[at:at + R * width].view(R, width), items[0], items[1], items[2] if places else None,
                         items[3] if places else None, places, tokens))
        self._lists[table_width] = made
        return made


def prompt_attention(plan: PromptPlan, q: torch.Tensor, q_stride: int, out: torch.Tensor, pages: torch.Tensor, block_tables: torch.Tensor,
                     q_start: torch.Tensor, ctx_len: torch.Tensor, scale: float) -> torch.Tensor:
    """Causal attention of the step's query rows over 8-bit pages, any portion sizes: as ``kernels.paged_attention`` over pages
    that hold the same values in q's type. ``q_start`` and ``ctx_len`` are the plan's lengths on the device."""
    nq, nkv, d, ps = plan.num_heads, plan.num_kv_heads, plan.head_dim, plan.page_size
    kernels._kv8_pages(pages, nkv, d, ps)
    kernels._need(q.dtype == plan.dtype, f"the plan is for queries in {plan.dtype}")
    kernels._need(block_tables.dim() == 2 and block_tables.shape[0] == len(plan.q_lens) == ctx_len.numel() and
                  q_start.numel() == len(plan.q_lens) + 1, "block tables, q_start and ctx_len must be those of the plan's requests")
    kernels._need(q.dim() == 2 and q.stride(1) == 1 and q.stride(0) == q_stride or q.shape[0] <= 1, "query rows must lie q_stride apart")
    kernels._need(q.shape[0] >= sum(plan.q_lens) and out.shape[0] >= sum(plan.q_lens), "the plan has more rows than the queries or the output")
    kernels._on_current_device(q, out, pages, block_tables, q_start, ctx_len)
    for index, tables, req, tok0, seg, slot, places, tokens in plan.lists(block_tables.shape[1]):
        held = torch.empty((index.numel(), 2, nkv, ps, d), dtype=q.dtype, device=q.device)
        kernels.kv8_gather(pages, block_tables, ctx_len, index, held)
        kernels.paged_attention(q, q_stride, out, held, tables, q_start, ctx_len, req, tok0, nq, nkv, d, ps, plan.window, scale, tokens,
                                seg, slot, places)
    return out
