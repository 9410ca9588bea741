"""What the call of the kernel that reads 8-bit pages for prompt portions refuses, and what a plan refuses (no GPU: every check is made before
anything is launched)."""

import pytest
import torch

import kv8_plain as plain
from llm_pipeline_b200.ops import kernels, kv8

NQ, NKV, D, PS = 4, 2, 128, 16


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def rows(n, width=NQ * D, **kw):
    return torch.zeros(n, width, dtype=torch.bfloat16, **kw)


GOOD = dict(q=rows(6), q_stride=NQ * D, out=rows(6), pages=torch.zeros(4, plain.page_bytes(NKV, PS, D), dtype=torch.uint8), block_tables=i32(2, 3),
            q_start=i32(3), ctx_len=i32(2), items=i32(3, 4), shared=i32(1, 4), places=2, num_heads=NQ, num_kv_heads=NKV, page_size=PS, window=0, scale=0.1)


@pytest.mark.parametrize("change,message", [
    (dict(q=rows(6, NQ * D - 8), q_stride=NQ * D - 8), "query rows"), (dict(q_stride=NQ * D + 8), "query rows"), (dict(q=rows(6 * NQ * D, 1)[:, 0]), "query rows"),
    (dict(q=torch.zeros(NQ * D, 6, dtype=torch.bfloat16).t()), "query rows"), (dict(q=torch.zeros(6, NQ * D)), "bfloat16"),
    (dict(out=rows(6, NQ * D + 8)), "bfloat16"), (dict(out=rows(12)[::2]), "bfloat16"), (dict(out=rows(6 * NQ * D, 1)[:, 0]), "bfloat16"),
    (dict(block_tables=i32(3, 3)), "block tables"), (dict(block_tables=i32(2)), "block tables"), (dict(block_tables=i32(2, 0)), "block tables"),
    (dict(q_start=i32(2)), "block tables"), (dict(ctx_len=i32(3)), "block tables"), (dict(ctx_len=torch.zeros(2)), "int32"),
    (dict(items=i32(3, 3)), "lists"), (dict(items=i32(4)), "lists"), (dict(shared=i32(4)), "lists"), (dict(places=0), "places"), (dict(places=-1), "places"),
    (dict(shared=i32(0, 4)), "places"), (dict(num_heads=0), "does not serve"), (dict(num_heads=3), "does not serve"), (dict(num_heads=1), "does not serve"),
    (dict(num_kv_heads=0), "does not serve"), (dict(page_size=24), "does not serve"), (dict(page_size=0), "does not serve"), (dict(window=-1), "window"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(pages=GOOD["pages"][:, :-1]), "uint8"), ({}, "not on a CUDA device"),
])
def test_the_kernel_that_reads_pages(change, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.kv8_prompt_attention(**{**GOOD, **change})


@pytest.mark.parametrize("heads,kv", [(0, 2), (3, 2), (1, 2), (-4, 2), (4, 0), (4, -2)])
def test_plans_of_heads_that_do_not_fit(heads, kv):
    with pytest.raises(kernels.KernelError, match="heads"):
        kv8.PromptPlan([5], [3], heads, kv, D, PS, 0, torch.bfloat16, torch.device("cpu"))


def test_sizes_that_no_kernel_takes():
    """Asked of the library itself, which divides by the group's size."""
    for nq, nkv in ((0, 8), (-8, 8), (4, 8), (8, 0), (8, -8)):
        assert not kernels.kv8_prompt_supports(torch.bfloat16, nq, nkv, D, PS)
        assert not kernels.kv8_stream_supports(torch.bfloat16, nq, nkv, D, PS)
    assert kernels.kv8_prompt_supports(torch.bfloat16, 8, 8, D, PS) and kernels.kv8_stream_supports(torch.bfloat16, 8, 8, D, PS)
