"""Workspaces that `Qwen2.score` keeps: a few, whatever the lengths of the texts."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qweninfer_b200 import synthetic
from qweninfer_b200.engine.kv_cache import Kv8Cache, KVCache
from qweninfer_b200.models.config import qwen2_0p5b
from qweninfer_b200.models.logprobs import token_logprobs
from qweninfer_b200.models.qwen2 import Qwen2

pytestmark = pytest.mark.gpu

CFG = qwen2_0p5b(num_hidden_layers=2, vocab_size=4096)


@pytest.fixture(scope="module")
def model():
    return Qwen2.from_pretrained(synthetic.checkpoint_dir(CFG, seed=0, dtype=torch.bfloat16), dtype=torch.bfloat16,
                                 device="cuda")


def text(n, rows=1, seed=0):
    return torch.tensor(np.random.default_rng(seed).integers(0, CFG.vocab_size, (rows, n)))


def test_texts_of_all_lengths_share_workspaces(model):
    """20 lengths, chunks that leave rests of all sizes: sizes are powers of two, so at most one
    workspace for each pair of (tokens 64..128, length 64..512)."""
    for n in range(2, 402, 20):
        model.score(text(n), chunk=100)
    assert len(model._workspaces) <= 2 * 4
    assert all(t & (t - 1) == 0 and n & (n - 1) == 0 for t, n in model._workspaces)
    model.check()


@pytest.mark.parametrize("n,rows,chunk", [(2, 1, 512), (130, 3, 50), (700, 1, 512), (1500, 2, 1100)])
def test_scores_are_those_of_a_forward(model, n, rows, chunk):
    """Chunk by chunk in a shared workspace, against one forward of the whole text (the same arithmetic
    in another order of sums: 5e-3, the bar of the model's tests)."""
    ids = text(n, rows, n)
    got = model.score(ids, top=3, chunk=chunk)
    logits = model(ids[:, :-1], logits_dtype=torch.float32)
    want = token_logprobs(logits.reshape(rows * (n - 1), -1), ids[:, 1:].reshape(-1), 3)
    assert float((got.logprob.reshape(-1) - want.logprob).abs().max()) <= 5e-3
    assert float((got.entropy.reshape(-1) - want.entropy).abs().max()) <= 5e-3
    model.check()


def test_a_given_cache_and_its_rows(model):
    ids = text(300, 2, 5)
    for cls in (KVCache, Kv8Cache):
        cache = cls(CFG, 5, 333, device="cuda")
        cache.row_start = 2
        a = model.score(ids, cache=cache, chunk=70)
        b = model.score(ids, cache=cls(CFG, 2, 299, device="cuda"), chunk=70)
        assert float((a.logprob - b.logprob).abs().max()) <= 5e-3
    model.check()
