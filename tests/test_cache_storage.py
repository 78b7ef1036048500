"""Pages of a windowed paged cache that go back behind the window (`trim`) and are mapped
again when a row starts over (`reserve`)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qweninfer_b200 import synthetic
from qweninfer_b200.engine.generate import generate
from qweninfer_b200.engine.kv_cache import PagedKv8Cache, PagedKVCache
from qweninfer_b200.models.config import qwen2_0p5b
from qweninfer_b200.models.qwen2 import Qwen2

CFG = qwen2_0p5b(num_hidden_layers=2, vocab_size=4096)


def windowed(window=100, sinks=0, device="cpu", cls=PagedKVCache, max_len=1024, rows=2, **kw):
    return cls(CFG, rows, max_len, device=device, attn_window=window, attn_sinks=sinks, **kw)


def decode(c, row, lo, hi):
    """The storage calls of decode steps at positions lo .. hi - 1."""
    for q in range(lo, hi):
        c.trim(row, q)
        c.reserve(row, q + 1, q)
        seen = {q} | set(range(max(0, q - c.attn_window + 1), q)) | set(range(min(c.attn_sinks, q)))
        assert all(c.table_host[row, p // 128] >= 0 for p in seen), q


@pytest.mark.parametrize("sinks", [0, 3, 200])
@pytest.mark.parametrize("again", [60, 300, 1000])
def test_a_trimmed_row_starts_over(sinks, again):
    c = windowed(sinks=sinks)
    c.reserve(0, 200)
    decode(c, 0, 200, 900)
    assert (c.table_host[0, :6] < 0).any()
    for _ in range(2):
        c.reserve(0, again)
        assert (c.table_host[0, :-(-again // 128)] >= 0).all()
        decode(c, 0, again, min(1024, again + 500))
        assert len(set(c.table_host[c.table_host >= 0].tolist())) == c.pages_in_use()
    assert c.pages_in_use() <= 3 + -(-sinks // 128)
    c.release(0)
    assert c.pages_in_use() == 0 and sorted(c.free) == list(range(c.n_pages))


def test_a_trimmed_row_moves():
    c = windowed()
    c.reserve(0, 200)
    decode(c, 0, 200, 700)
    c.move_row(0, 1, 700)
    decode(c, 1, 700, 800)
    c.reserve(0, 300)
    c.reserve(1, 300)
    assert (c.table_host[:, :3] >= 0).all()


def test_going_back_behind_the_window_is_refused():
    """Positions that a query would see have gone back: refused, and nothing is changed."""
    c = windowed(window=300)
    c.reserve(0, 200)
    decode(c, 0, 200, 900)  # 0 .. 511 went back
    table = c.table_host.clone()
    for start in (1, 128, 500, 512, 513, 700, 810):
        with pytest.raises(RuntimeError, match="went back"):
            c.reserve(0, start + 1, start)
    assert torch.equal(c.table_host, table)
    decode(c, 0, 811, 950)  # sees 512 .. 810 of what is there
    with pytest.raises(IndexError):
        c.reserve(0, 5, 6)


# ---------------------------------------------------------------------------- GPU


@pytest.fixture(scope="module")
def model():
    return Qwen2.from_pretrained(synthetic.checkpoint_dir(CFG, seed=0, dtype=torch.bfloat16), dtype=torch.bfloat16,
                                 device="cuda")


def text(n, seed):
    return np.random.default_rng(seed).integers(0, CFG.vocab_size, (1, n))


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [PagedKVCache, PagedKv8Cache])
def test_generate_twice_on_a_windowed_paged_cache(model, cls):
    """The second text in a row whose pages went back gives what a new cache gives, and so
    does a forward over it afterwards."""
    used = windowed(sinks=3, device="cuda", cls=cls, rows=1)
    generate(model, torch.tensor(text(200, 1)), 600, cache=used)
    assert int((used.table_host[0] >= 0).sum()) <= 3
    for n in (400, 150):
        new = windowed(sinks=3, device="cuda", cls=cls, rows=1)
        ids = torch.tensor(text(n, n))
        assert generate(model, ids, 200, cache=used) == generate(model, ids, 200, cache=new)
    ids = torch.tensor(text(330, 9))
    new = windowed(sinks=3, device="cuda", cls=cls, rows=1)
    assert torch.equal(model(ids, cache=used), model(ids, cache=new))
    generate(model, ids, 300, cache=used)
    model.check()
    with pytest.raises(RuntimeError, match="went back"):
        model(ids[:, :1], positions=torch.tensor([400]), cache=used)
