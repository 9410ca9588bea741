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
