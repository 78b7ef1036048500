"""The model on 8-bit and windowed caches, and log probabilities of its tokens: forward,
generate, Engine and score against a 64-bit restatement of the model (two layers) whose
cache rounds and whose attention sees what the options say.

Bars: the framework's parity bar (conftest.LOGIT_ATOL, LOGIT_MIN_COS) against the
restatement. A code next to a rounding border may differ by one step, since keys are known
to ~16 bits before they are rounded; the bar covers that. Runs of the same arithmetic in
another order (chunks, splits, batches) agree within 5e-3, the bar of the smoke test."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from conftest import LOGIT_ATOL, LOGIT_MIN_COS, logit_report
from qweninfer_b200 import synthetic
from qweninfer_b200.engine.engine import Engine, Request
from qweninfer_b200.engine.generate import generate
from qweninfer_b200.engine.kv_cache import Kv8Cache, KVCache, PagedKv8Cache, PagedKVCache
from qweninfer_b200.engine.runner import DecodeRunner
from qweninfer_b200.models.config import qwen2_0p5b
from qweninfer_b200.models.qwen2 import Qwen2, build_rope_cache
from test_cache_ops_gpu import Oracle8

pytestmark = pytest.mark.gpu

CFG = qwen2_0p5b(num_hidden_layers=2, vocab_size=4096)
SAME = 5e-3
OPTIONS = [("bf16", 0, 0), ("bf16", 24, 4), ("int8", 0, 0), ("int8", 40, 0), ("e4m3", 0, 0), ("e4m3", 17, 3)]


@pytest.fixture(scope="module")
def model():
    return Qwen2.from_pretrained(synthetic.checkpoint_dir(CFG, seed=0, dtype=torch.bfloat16), dtype=torch.bfloat16,
                                 device="cuda")


@pytest.fixture(scope="module")
def weights():
    return {k: v.to(torch.bfloat16).double() for k, v in synthetic.synthetic_state(CFG, 0).items()}


class Reference:
    """One row of the model in 64 bits; `step` runs the next tokens and returns their logits."""

    def __init__(self, w, fmt, window, sinks, max_len=512, block=32):
        self.w, self.fmt, self.window, self.sinks = w, fmt, window, sinks
        cos, sin = build_rope_cache(64, max_len, CFG.rope_theta)
        self.cos, self.sin = cos.double(), sin.double()
        self.n = 0
        L = CFG.num_hidden_layers
        if fmt == "bf16":
            self.kv = [[torch.zeros(2, max_len, 64, dtype=torch.float64) for _ in range(2)] for _ in range(L)]
        else:
            self.kv = [[Oracle8(1, 2, max_len, 64, fmt, block) for _ in range(2)] for _ in range(L)]

    def p(self, name):
        return self.w[name if name in self.w else "model." + name]

    def norm(self, x, name):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + CFG.rms_norm_eps) * self.p(name)

    def rope(self, x, pos):  # (tokens, heads, 64)
        half = torch.cat([-x[..., 32:], x[..., :32]], -1)
        return x * self.cos[pos][:, None] + half * self.sin[pos][:, None]

    def store(self, layer, which, x, pos):  # (tokens, 2, 64) -> values (2, length, 64)
        c = self.kv[layer][which]
        if self.fmt == "bf16":
            c[:, pos] = x.transpose(0, 1).to(torch.bfloat16).double()
            return c
        c.append(x.float(), [0] * len(pos), list(pos))
        return c.values()[0]

    def step(self, tokens):
        pos = list(range(self.n, self.n + len(tokens)))
        self.n += len(tokens)
        x = self.p("embed_tokens.weight")[tokens]
        for i in range(CFG.num_hidden_layers):
            n = f"layers.{i}."
            h = self.norm(x, n + "input_layernorm.weight")
            q, k, v = (h @ self.p(f"{n}self_attn.{c}_proj.weight").T + self.p(f"{n}self_attn.{c}_proj.bias") for c in "qkv")
            q = self.rope(q.view(-1, 14, 64), pos)
            k = self.store(i, 0, self.rope(k.view(-1, 2, 64), pos), pos)
            v = self.store(i, 1, v.view(-1, 2, 64), pos)
            j, at = torch.arange(k.shape[1]), torch.tensor(pos)[:, None]
            seen = j <= at
            if self.window:
                seen &= (j > at - self.window) | (j < self.sinks)
            s = torch.einsum("tghd,gjd->tghj", q.view(-1, 2, 7, 64), k) / 8
            a = torch.softmax(s.masked_fill(~seen[:, None, None], -math.inf), -1)
            o = torch.einsum("tghj,gjd->tghd", a, torch.where(seen.any(0)[None, :, None], v, 0.0)).reshape(-1, 896)
            x = x + o @ self.p(n + "self_attn.o_proj.weight").T
            h = self.norm(x, n + "post_attention_layernorm.weight")
            g = h @ self.p(n + "mlp.gate_proj.weight").T
            x = x + (g * torch.sigmoid(g) * (h @ self.p(n + "mlp.up_proj.weight").T)) @ self.p(n + "mlp.down_proj.weight").T
        return self.norm(x, "norm.weight") @ self.p("embed_tokens.weight").T


def make_cache(fmt, window, sinks, rows, max_len, paged=False, **kw):
    extra = dict(attn_window=window, attn_sinks=sinks, device="cuda", **kw)
    if fmt == "bf16":
        return (PagedKVCache if paged else KVCache)(CFG, rows, max_len, **extra)
    return (PagedKv8Cache if paged else Kv8Cache)(CFG, rows, max_len, format=fmt, **extra)


def prompt(n, seed):
    return np.random.default_rng(seed).integers(0, CFG.vocab_size, n).tolist()


@pytest.mark.parametrize("fmt,window,sinks", OPTIONS)
@pytest.mark.parametrize("paged", [False, True])
def test_forward_matches_the_restatement(model, weights, fmt, window, sinks, paged):
    """A prompt in one forward, a chunk behind it and single tokens, in a row of its own."""
    ids = prompt(70 + 33 + 5, 1)
    ref = Reference(weights, fmt, window, sinks)
    cache = make_cache(fmt, window, sinks, 2, 200, paged)
    cache.row_start = 1
    for lo, hi in [(0, 70), (70, 103)] + [(i, i + 1) for i in range(103, 108)]:
        want = ref.step(ids[lo:hi])
        got = model(torch.tensor([ids[lo:hi]]), positions=torch.arange(lo, hi), cache=cache, logits_dtype=torch.float32)[0]
        for t in range(hi - lo):
            err, cos = logit_report(got[t].cpu().numpy(), want[t].numpy())
            assert err <= LOGIT_ATOL and cos >= LOGIT_MIN_COS, (lo + t, err, cos)
    model.check()


@pytest.mark.parametrize("fmt,window,sinks,paged", [("bf16", 2700, 4, False), ("int8", 0, 0, True)])
def test_long_prompt_matches_the_restatement(model, weights, fmt, window, sinks, paged):
    """A prompt whose attention shares keys in tiles (400 tokens x 2 x 64 x window or length is
    above 2^27), and a token behind it."""
    ids = prompt(401, 2)
    ref = Reference(weights, fmt, window, sinks)
    cache = make_cache(fmt, window, sinks, 2, 4096, paged)
    cache.row_start = 1
    for lo, hi in [(0, 400), (400, 401)]:
        want = ref.step(ids[lo:hi])
        got = model(torch.tensor([ids[lo:hi]]), positions=torch.arange(lo, hi), cache=cache, logits_dtype=torch.float32)[0]
        for t in range(hi - lo):
            err, cos = logit_report(got[t].cpu().numpy(), want[t].numpy())
            assert err <= LOGIT_ATOL and cos >= LOGIT_MIN_COS, (lo + t, err, cos)
    model.check()


@pytest.mark.parametrize("fmt,window,sinks", OPTIONS)
@pytest.mark.parametrize("page_size", [0, 128])
def test_engine_matches_solo_generation(model, fmt, window, sinks, page_size):
    """Requests of all lengths through slots, row moves, batched prefill and graphs give the
    tokens and log probabilities that each has alone, as far as its choices are not ties."""
    reqs = [Request(i, prompt(5 + 23 * i % 150, 100 + i), 3 + 7 * (i % 4)) for i in range(7)]
    eng = Engine(model, max_slots=3, max_len=256, page_size=page_size, kv_format=None if fmt == "bf16" else fmt,
                 attn_window=window, attn_sinks=sinks, logprobs=3)
    done = eng.run(reqs)
    eng.runner.check()
    for r in done:
        assert len(r.output) == r.max_new_tokens == len(r.logprobs)
        cache = make_cache(fmt, window, sinks, 1, 256)
        toks, infos = generate(model, torch.tensor([r.prompt]), r.max_new_tokens, cache=cache, logprobs=2)
        for a, b, x, y in zip(r.output, toks, r.logprobs, infos):
            assert x.token == a and x.top[0][0] == a and len(x.top) == 3
            assert x.logprob == x.top[0][1] >= x.top[1][1] and 0 < x.entropy <= math.log(CFG.vocab_size) + 1e-4
            if a != b:
                assert y.top[0][1] - y.top[1][1] < 2 * SAME  # a tie: the rest may differ
                break
            assert abs(x.logprob - y.logprob) <= 2 * SAME and abs(x.entropy - y.entropy) <= 2 * SAME
    if page_size:
        assert eng.cache.pages_in_use() == 0


def test_windowed_pages_go_back(model):
    """A long generation under a window holds the pages of the window and the first tokens."""
    cache = make_cache("int8", 100, 3, 1, 1024, paged=True, n_pages=4)
    runner = DecodeRunner(model, cache, 1)
    tok = runner.prefill(0, prompt(200, 5))
    for p in range(200, 900):
        tok = int(runner.decode([tok], [p])[0])
        assert cache.pages_in_use() <= 3
    runner.check()
    cache.release(0)
    assert cache.pages_in_use() == 0


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_score(model, weights, fmt):
    ids = torch.tensor([prompt(90, 7), prompt(90, 8)])
    caches = [make_cache(fmt, 0, 0, 2, 89) for _ in range(2)]
    r = model.score(ids, top=4, cache=caches[0], chunk=32)
    one = model.score(ids, top=4, cache=caches[1])
    assert r.logprob.shape == r.entropy.shape == (2, 89) and r.top_ids.shape == (2, 89, 4)
    if fmt == "bf16":  # (chunks of an 8-bit cache round a growing block more than once)
        assert float((r.logprob - one.logprob).abs().max()) <= SAME
    for b in range(2):
        lp = torch.log_softmax(Reference(weights, fmt, 0, 0).step(ids[b, :89].tolist()), -1)
        want = lp.gather(1, ids[b, 1:, None])[:, 0]
        assert float((one.logprob[b].cpu().double() - want).abs().max()) <= 2 * LOGIT_ATOL
        assert float((one.entropy[b].cpu().double() + (lp.exp() * lp).sum(-1)).abs().max()) <= 2 * LOGIT_ATOL
    with pytest.raises(ValueError):
        model.score(ids[:, :1])
    with pytest.raises(ValueError):
        model.score(ids, chunk=0)


def test_launches_of_an_8_bit_step(model):
    runner = DecodeRunner(model, make_cache("int8", 0, 0, 2, 64), 2)
    runner.prefill(0, prompt(10, 9))
    kinds = [k for k, _ in runner.launch_times([1, 2], [10, 0])]
    assert kinds.count("kv_append") == kinds.count("attention") == 2 and len(kinds) == runner.kernels_per_forward(2)


def test_paged_codes_match_packed_ones():
    g = torch.Generator("cuda").manual_seed(3)
    packed = Kv8Cache(CFG, 3, 400, device="cuda", format="e4m3", block_tokens=64)
    paged = PagedKv8Cache(CFG, 3, 400, device="cuda", format="e4m3", block_tokens=64, n_pages=12)
    for b in range(4):
        for r in (1, 2, 0):  # scattered pages
            paged.reserve(r, min(400, 128 * (b + 1)))
    n = 200
    for lo, hi in ((0, 150), (150, 151), (151, 200)):
        k, v = (torch.randn(3 * (hi - lo), 2, 64, generator=g, device="cuda") * (1 + lo) for _ in range(2))
        rows = torch.tensor([0, 1, 2], dtype=torch.int32).repeat_interleave(hi - lo).cuda()
        pos = torch.arange(lo, hi, dtype=torch.int32).repeat(3).cuda()
        for c in (packed, paged):
            c.append(1, k, v, rows, pos)
    for a, b in zip(packed.values(1), paged.values(1)):
        assert torch.equal(a[:, :, :n], b[:, :, :n])
    q = 2 * torch.randn(100, 14, 64, generator=g, device="cuda")
    rows, pos = torch.full((100,), 1, dtype=torch.int32).cuda(), torch.arange(100, 200, dtype=torch.int32).cuda()
    for run in (1, 100):
        for window, sinks in ((0, 0), (50, 2)):
            assert torch.equal(packed.attend(1, q, rows, pos, window, sinks, run),
                               paged.attend(1, q, rows, pos, window, sinks, run))
    packed.check()
    paged.check()
    paged.release(2)
    assert not paged.values(1)[0][2].any()


def test_refusals(model):
    with pytest.raises(ValueError):
        Engine(model, 2, 64, kv_format="int4")
    with pytest.raises(ValueError):
        Engine(model, 2, 64, attn_window=-1)
    with pytest.raises(ValueError):
        Engine(model, 2, 64, logprobs=33)
    cache = make_cache("int8", 0, 0, 1, 64)
    cache._native = None
    with pytest.raises(IndexError):
        model(torch.tensor([[1]]), positions=torch.tensor([[64]]), cache=cache)
