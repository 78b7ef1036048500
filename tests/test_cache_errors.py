"""The error word of a cache's operators: there from the start, and kept."""

from __future__ import annotations

import pytest
import torch

from qweninfer_b200 import _lib
from qweninfer_b200.engine.kv_cache import Kv8Cache, KVCache, PagedKv8Cache, PagedKVCache
from qweninfer_b200.models.config import qwen2_0p5b

CFG = qwen2_0p5b(num_hidden_layers=1)
CACHES = [KVCache, PagedKVCache, Kv8Cache, PagedKv8Cache]


@pytest.mark.parametrize("cls", CACHES)
def test_error_word_is_made_with_the_cache(cls):
    c = cls(CFG, 2, 256, device="cpu")
    assert "_err" in c.__dict__ and c._errors() is c._err and not c._err.any()
    c.check()
    c._err.fill_(_lib.QI_ERR_INDEX)
    with pytest.raises(_lib.QiError):
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("cls", CACHES)
def test_a_first_call_that_is_captured(cls):
    """Nothing is recorded before the replay, and what a replay records stays through others."""
    c = cls(CFG, 2, 256, device="cuda")
    q = torch.zeros(1, 14, 64, device="cuda")
    row, pos = torch.zeros(1, dtype=torch.int32).cuda(), torch.full((1,), 256, dtype=torch.int32).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(0, q, row, pos)
    c.check()
    graph.replay()
    with pytest.raises(_lib.QiError):
        c.check()
    pos.fill_(-1)
    graph.replay()
    with pytest.raises(_lib.QiError):
        c.check()
