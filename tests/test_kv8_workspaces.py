"""Scratch and counters of the attention kernels around 8-bit pages, by stream, capture and thread: the books alone, without a GPU."""

import threading
import time

import pytest
import torch

from llm_pipeline_b200.ops import kernels

COUNT = 8


class SlowSlab(list):
    """[tensor, entries given away]; whoever writes to it lets the other threads run before going on."""

    def __setitem__(self, i, value):
        super().__setitem__(i, value)
        time.sleep(0.005)


@pytest.fixture
def books(monkeypatch):
    monkeypatch.setattr(kernels, "_kv8_workspaces", {})
    monkeypatch.setattr(kernels, "_kv8_stream_sizes", lambda: (16, COUNT))
    monkeypatch.setattr(kernels, "_device", lambda: 0)
    monkeypatch.setattr(kernels, "_stream", lambda: 7)
    return kernels._kv8_workspaces


def in_threads(n, work):
    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert not any(t.is_alive() for t in threads)


def test_threads_that_capture_at_once_get_counters_of_their_own(books, monkeypatch):
    monkeypatch.setattr(kernels, "_capturing", lambda: True)
    books[0, "slab"] = SlowSlab([torch.zeros(64 * COUNT, dtype=torch.int32), 0])
    got = [None] * 24
    in_threads(24, lambda i: got.__setitem__(i, kernels.kv8_workspace(torch.device("cpu"))))
    assert len({counters.data_ptr() for _scratch, counters in got}) == 24 and all(c.numel() == COUNT for _s, c in got)
    assert books[0, "slab"][1] == 24 * COUNT


def test_a_used_up_slab_gives_way_to_counters_of_the_graph(books, monkeypatch):
    monkeypatch.setattr(kernels, "_capturing", lambda: True)
    books[0, "slab"] = [torch.zeros(2 * COUNT + 3, dtype=torch.int32), 0]
    slab = books[0, "slab"][0]
    got = [kernels.kv8_workspace(torch.device("cpu"))[1] for _ in range(4)]
    inside = [slab.data_ptr() <= c.data_ptr() < slab.data_ptr() + 4 * slab.numel() for c in got]
    assert inside == [True, True, False, False] and all(not bool(c.any()) for c in got)


def test_threads_that_start_at_once_make_one_slab(books, monkeypatch):
    """The slab's memory is held by the books alone: a second one in its place would free what captured graphs use."""
    made = []

    def zeros(n, **kwargs):
        time.sleep(0.005)
        made.append(n)
        return torch.empty(n, dtype=torch.int32).zero_()

    monkeypatch.setattr(kernels, "_capturing", lambda: False)
    monkeypatch.setattr(kernels.torch, "zeros", zeros)
    monkeypatch.setattr(kernels.torch.cuda, "current_stream", lambda *a: type("S", (), {"synchronize": lambda self: None})())
    in_threads(8, lambda i: kernels.kv8_workspace(torch.device("cpu")))
    assert made.count(kernels.KV8_CAPTURED_CALLS * COUNT) == 1


def paged_call(monkeypatch, places):
    """The pointer of the counters that one call with ``places`` shared places of 2 heads hands to its kernel."""
    seen = {}
    monkeypatch.setattr(kernels, "_ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(kernels, "_call", lambda name, *args: seen.update(name=name, counters=args[16]))
    monkeypatch.setattr(kernels, "error_flag", lambda: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(kernels, "attention_place_floats", lambda: 4)
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32)                  # noqa: E731
    items = (i32(places), i32(places)) if places else (None, None)
    kernels.paged_attention(torch.zeros(4, 32), 32, torch.zeros(4, 32), torch.zeros(2, 2, 2, 4, 8), i32(1, 2), i32(2), i32(1), i32(max(places, 1)),
                            i32(max(places, 1)), 4, 2, 8, 4, 0, 1.0, 1, *items, places)
    assert seen["name"] == "llmp_paged_attention"
    return seen["counters"]


def test_prompt_tiles_whose_keys_are_shared_count_by_stream(books, monkeypatch):
    """Calls on two streams, and captured ones, may run at the same time: what one counts on is not another's."""
    monkeypatch.setattr(kernels, "_attention_counters", {})
    capturing = False
    monkeypatch.setattr(kernels, "_capturing", lambda: capturing)
    monkeypatch.setattr(kernels.torch.cuda, "is_current_stream_capturing", lambda: capturing)
    kept, got = [], {}
    for stream in (7, 8, 7, 0):
        monkeypatch.setattr(kernels, "_stream", lambda: stream)                  # noqa: B023
        got.setdefault(stream, set()).add(paged_call(monkeypatch, 6))
    assert all(len(v) == 1 for v in got.values()) and len(set.union(*got.values())) == 3
    assert paged_call(monkeypatch, 0) is None
    # captured: counters of its own each time
    zeros = torch.zeros
    monkeypatch.setattr(kernels.torch, "zeros", lambda *a, **k: kept.append(zeros(*a, **k)) or kept[-1])
    capturing = True
    books[0, "slab"] = [zeros(20, dtype=torch.int32), 0]
    captured = [paged_call(monkeypatch, 6) for _ in range(3)]                    # 12 counters a call: one from the slab, two of the graph
    assert len(set(captured) | set.union(*got.values())) == 6
