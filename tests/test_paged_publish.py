"""Publishing the page table of a paged cache: what a call reads is the table as it was when the
call was made, whatever the host changes afterwards, on any stream, and never by way of a graph."""

from __future__ import annotations

import pytest
import torch

from qweninfer_b200 import _lib
from qweninfer_b200.engine.kv_cache import KVCache, PagedKv8Cache, PagedKVCache
from qweninfer_b200.models.config import qwen2_0p5b

CFG = qwen2_0p5b(num_hidden_layers=1)


class Device:
    """The device's part of `sync`, recorded: copies as (source, stream), waits as (stream, event)."""

    device = torch.device("cuda", 0)

    def __init__(self, monkeypatch):
        self.stream, self.capturing, self.copies, self.waits = 1, False, [], []
        dev = self

        class Event:
            def record(self):
                self.at = dev.stream

        class Stream:
            def wait_event(self, e):
                dev.waits.append((dev.stream, e.at))

        class Guard:
            def __init__(self, d):
                assert d == dev.device

            def __enter__(self):
                pass

            def __exit__(self, kind, value, trace):
                pass

        for name, f in (("Event", Event), ("current_stream", Stream), ("device", Guard),
                        ("is_current_stream_capturing", lambda: self.capturing)):
            monkeypatch.setattr(torch.cuda, name, f)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: self.stream, raising=False)
        monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t.clone())

    def copy_(self, src, non_blocking=False):
        self.copies.append((src, self.stream))


@pytest.fixture
def paged(monkeypatch):
    c = PagedKVCache(CFG, 3, 512, device="cpu")
    c.table = Device(monkeypatch)
    return c


def test_a_published_table_is_not_written_again(paged):
    """An asynchronous copy reads its source later: every publish has one of its own."""
    paged.reserve(0, 300)
    paged.sync()
    want = paged.table_host.clone()
    paged.release(0)
    paged.reserve(1, 500)
    paged.sync()
    (first, _), (second, _) = paged.table.copies
    assert torch.equal(first, want) and torch.equal(second, paged.table_host)
    paged.sync()
    assert len(paged.table.copies) == 2


def test_other_streams_wait_for_the_copy(paged):
    paged.sync()
    assert not paged.table.copies and not paged.table.waits
    paged.reserve(0, 10)
    paged.sync()
    paged.table.stream = 2
    paged.sync()
    paged.sync()
    assert paged.table.waits == [(2, 1)]
    paged.table.stream = 3
    paged.reserve(1, 10)
    paged.sync()  # a copy behind the first one
    assert paged.table.waits == [(2, 1), (3, 1)] and paged.table.copies[-1][1] == 3
    paged.table.stream = 1
    paged.sync()
    assert paged.table.waits[-1] == (1, 3)


def test_a_capture_does_not_publish(paged):
    paged.reserve(0, 10)
    paged.table.capturing = True
    with pytest.raises(_lib.QiError, match="sync"):
        paged.sync()
    assert paged.dirty and not paged.table.copies
    paged.table.capturing = False
    paged.sync()
    paged.table.capturing, paged.table.stream = True, 7
    paged.sync()  # nothing to publish, and nothing that a captured call could wait for
    assert len(paged.table.copies) == 1 and not paged.table.waits


# ---------------------------------------------------------------------------- GPU


def filled(cls=PagedKVCache, n=200, rows=2):
    """A packed cache and a paged one with the same keys in rows 0 .. rows - 1."""
    g = torch.Generator("cuda").manual_seed(0)
    paged = cls(CFG, 3, 512, device="cuda")
    packed = KVCache(CFG, 3, 512, device="cuda")
    packed.k.copy_(torch.randn(packed.k.shape, generator=g, device="cuda"))
    packed.v.copy_(torch.randn(packed.v.shape, generator=g, device="cuda"))
    for r in range(rows):
        paged.reserve(r, n)
        for b in range(-(-n // 128)):
            pg = int(paged.table_host[r, b])
            if cls is PagedKVCache:
                paged.k[0, pg], paged.v[0, pg] = packed.k[0, r, :, 128 * b:128 * b + 128], packed.v[0, r, :, 128 * b:128 * b + 128]
    return packed, paged


@pytest.mark.gpu
def test_pages_released_behind_a_call():
    """The row's pages go back while the call that reads them still waits for work before it."""
    packed, paged = filled()
    q = torch.randn(40, 14, 64, device="cuda")
    rows, pos = torch.zeros(40, dtype=torch.int32).cuda(), torch.arange(160, 200, dtype=torch.int32).cuda()
    want = packed.attend(0, q, rows, pos)
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)
    got = paged.attend(0, q, rows, pos)
    paged.release(0)
    paged.reserve(2, 500)
    assert torch.equal(got, want)
    paged.check()


@pytest.mark.gpu
def test_appends_on_two_streams():
    """Two rows get their pages together; one stream's call publishes them behind work of its
    own, the other's comes at once."""
    g = torch.Generator("cuda").manual_seed(1)
    k = torch.randn(2, 100, 2, 64, generator=g, device="cuda")
    paged = PagedKv8Cache(CFG, 3, 512, device="cuda")
    pos = torch.arange(100, dtype=torch.int32).cuda()
    row = [torch.full((100,), r, dtype=torch.int32).cuda() for r in range(2)]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    paged.reserve(0, 100)
    paged.reserve(1, 100)
    with torch.cuda.stream(a):
        torch.cuda._sleep(20_000_000)
        paged.append(0, k[0], k[0], row[0], pos)
    with torch.cuda.stream(b):
        paged.append(0, k[1], k[1], row[1], pos)
    torch.cuda.synchronize()
    paged.check()
    got = paged.values(0)[0]
    for r in range(2):
        step = k[r].abs().max() / 63.5
        assert float((got[r, :, :100] - k[r].transpose(0, 1)).abs().max()) <= float(step) / 2


@pytest.mark.gpu
def test_captured_calls_read_the_published_table():
    packed, paged = filled()
    q = torch.randn(4, 14, 64, device="cuda")
    rows, pos = torch.tensor([0, 1, 0, 1], dtype=torch.int32).cuda(), torch.tensor([199, 150, 3, 0], dtype=torch.int32).cuda()
    want = packed.attend(0, q, rows, pos, query_run=1)
    graph = torch.cuda.CUDAGraph()
    paged.dirty = True
    with pytest.raises(_lib.QiError, match="sync"):
        with torch.cuda.graph(graph):
            paged.attend(0, q, rows, pos, query_run=1)
    paged.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.attend(0, q, rows, pos, query_run=1)
    graph.replay()
    assert torch.equal(out, want)
    paged.move_row(0, 2, 200)  # the replay goes by the table of its time
    paged.sync()
    rows.copy_(torch.tensor([2, 1, 2, 1]))
    graph.replay()
    assert torch.equal(out, want)
    paged.check()
