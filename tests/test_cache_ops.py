"""Refusals of the cache-layer and log-probability operators, on the CPU: the C ABI's argument
checks and the Python entry points'."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from qweninfer_b200 import _lib
from qweninfer_b200.engine.kv_cache import Kv8Cache, KVCache
from qweninfer_b200.models.config import qwen2_0p5b
from qweninfer_b200.models.logprobs import token_logprobs

E = _lib.QI_ERR_ARG


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def layer(**kw):
    base = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, format=_lib.QI_KV_INT8, block=32, cache_rows=2, kv_heads=2,
                max_len=256, head_dim=64, page_table=None, page_size=0, pages_per_row=0, n_pages=0)
    base.update(kw)
    return _lib.QiKvLayer(*base.values())


BAD_LAYERS = [dict(k=None), dict(v=None), dict(k=4104), dict(k_scale=None), dict(v_scale=None), dict(format=3),
              dict(format=-1), dict(block=0), dict(block=48), dict(block=256), dict(cache_rows=0), dict(kv_heads=0),
              dict(max_len=0), dict(head_dim=96),
              dict(page_table=1, page_size=64, pages_per_row=4, n_pages=4),
              dict(page_table=1, page_size=128, pages_per_row=1, n_pages=4),
              dict(page_table=1, page_size=128, pages_per_row=2, n_pages=0)]


def append(lib, d, k=1, v=1, dt=0, rows=1, pos=1, M=1):
    return lib.qi_kv8_append(d if d is None else C.byref(d), k, 128, 64, v, 128, 64, dt, rows, pos, M, None, None)


def attend(lib, d, q=1, dt=0, heads=14, rows=1, pos=1, M=1, window=0, sinks=0, run=0, out=16, part=8):
    return lib.qi_cache_attention(d if d is None else C.byref(d), q, 896, 64, dt, heads, rows, pos, M, window, sinks, run,
                                  out, part, 0, 1, 0, None, None)


@pytest.mark.parametrize("bad", BAD_LAYERS, ids=str)
def test_bad_layers(lib, bad):
    d = layer(**bad)
    a, b = C.c_longlong(), C.c_longlong()
    assert append(lib, d) == E and attend(lib, d) == E
    assert lib.qi_kv8_values(C.byref(d), 16, 16, None) == E
    assert lib.qi_cache_attention_scratch(C.byref(d), 14, 1, 0, 0, 1, C.byref(a), C.byref(b)) == E


def test_bad_calls(lib):
    assert append(lib, None) == E and attend(lib, None) == E
    bf = layer(format=_lib.QI_KV_BF16, k_scale=None, v_scale=None, block=0)
    assert append(lib, bf) == E and lib.qi_kv8_values(C.byref(bf), 16, 16, None) == E
    d = layer()
    for kw in (dict(k=None), dict(v=None), dict(dt=3), dict(rows=None), dict(pos=None), dict(M=0)):
        assert append(lib, d, **kw) == E, kw
    for kw in (dict(q=None), dict(dt=-1), dict(heads=0), dict(heads=15), dict(heads=18), dict(rows=None),
               dict(pos=None), dict(M=0), dict(window=-1), dict(sinks=-1), dict(run=-1), dict(out=None), dict(out=8),
               dict(M=2**31 - 1), dict(part=4)):
        assert attend(lib, d, **kw) == E, kw
    assert lib.qi_kv8_values(C.byref(d), 16, 8, None) == E

    def logprobs(x=1, dt=0, ld=100, M=1, V=100, top=0, ids=1, lps=1, scratch=0):
        return lib.qi_token_logprobs(x, dt, ld, None, 0, M, V, top, None, 1, ids, lps, scratch, 0, 1, None)
    for kw in (dict(x=None), dict(dt=3), dict(ld=99), dict(M=0), dict(V=0), dict(top=-1), dict(top=33), dict(top=101),
               dict(top=1, ids=None), dict(top=1, lps=None), dict(scratch=8), dict(V=3, ld=3, top=4),
               dict(M=2**30, V=2**20, ld=2**20)):
        assert logprobs(**kw) == E, kw


def test_misaligned_pointers(lib):
    d = layer()
    for kw in (dict(k=2), dict(v=6), dict(k=1, dt=1), dict(v=3, dt=2), dict(rows=2), dict(pos=6)):
        assert append(lib, d, **{"k": 16, "v": 16, "rows": 16, "pos": 16, **kw}) == E, kw
    for kw in (dict(q=2), dict(q=1, dt=1), dict(rows=2), dict(pos=1), dict(out=4), dict(part=4)):
        assert attend(lib, d, **{"q": 16, "rows": 16, "pos": 16, **kw}) == E, kw
    assert append(lib, layer(k_scale=2), k=16, v=16, rows=16, pos=16) == E
    for i, x in ((0, 2), (3, 4), (8, 2), (9, 1), (10, 2), (11, 2), (14, 2)):
        args = [16, 0, 100, 16, 1, 1, 100, 1, 16, 16, 16, 16, 16, 0, 16, None]
        args[i] = x
        assert lib.qi_token_logprobs(*args) == E, (i, x)


def test_scratch_of_runs_in_tiles(lib):
    """QI_RUN_TILES belongs to the run's length: no other check takes it for one."""
    a, b = C.c_longlong(-1), C.c_longlong(-1)
    run = _lib.QI_RUN_TILES | 77
    assert lib.qi_cache_attention_scratch(C.byref(layer(max_len=64)), 14, 77, 0, 0, run, C.byref(a), C.byref(b)) == 0
    assert a.value == b.value == 0


def test_scratch_sizes(lib):
    a, b = C.c_longlong(-1), C.c_longlong(-1)
    assert lib.qi_cache_attention_scratch(C.byref(layer(max_len=64)), 14, 4, 0, 0, 1, C.byref(a), C.byref(b)) == 0
    assert (a.value, b.value) == (0, 0)  # short rows: one split
    assert lib.qi_cache_attention_scratch(C.byref(layer(max_len=100000)), 14, 1, 0, 0, 1, C.byref(a), C.byref(b)) == 0
    assert a.value % (14 * 66) == 0 and a.value >= 2 * 14 * 66 and b.value == 2
    assert lib.qi_cache_attention_scratch(C.byref(layer(max_len=100000)), 14, 1, 64, 4, 1, C.byref(a), C.byref(b)) == 0
    assert (a.value, b.value) == (0, 0)  # short windows too
    assert 0 < lib.qi_token_logprobs_scratch(1, 151936, 0) <= lib.qi_token_logprobs_scratch(4000, 151936, 1) < 2**20


def test_cache_arguments():
    cfg = qwen2_0p5b(1)
    with pytest.raises(ValueError):
        Kv8Cache(cfg, 1, 64, device="cpu", format="int4")
    with pytest.raises(ValueError):
        Kv8Cache(cfg, 1, 64, device="cpu", block_tokens=24)
    with pytest.raises(ValueError):
        Kv8Cache(cfg, 1, 64, dtype=torch.int8, device="cpu")
    c = Kv8Cache(cfg, 3, 65, device="cpu", format="e4m3", block_tokens=16)
    assert c.k.dtype == torch.float8_e4m3fn and c.k_scale.shape == (1, 3, 2, 5)
    assert c.memory_bytes() == 2 * (3 * 2 * 65 * 64 + 4 * 3 * 2 * 5)
    z = torch.zeros(2, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: c.append(0, z, z, i, i), lambda: c.attend(0, torch.zeros(2, 14, 64), i, i),
              lambda: c.values(0), lambda: KVCache(cfg, 1, 64, device="cpu").attend(0, torch.zeros(2, 14, 64), i, i)):
        with pytest.raises(_lib.QiError):
            f()
    with pytest.raises(IndexError):
        c.append(1, z, z, i, i)


def test_row_moves_of_an_8_bit_cache():
    c = Kv8Cache(qwen2_0p5b(2), 3, 100, device="cpu", block_tokens=32)
    g = torch.Generator().manual_seed(0)
    c.k.copy_(torch.randint(-127, 128, c.k.shape, generator=g))
    c.v.copy_(torch.randint(-127, 128, c.v.shape, generator=g))
    c.k_scale.copy_(torch.rand(c.k_scale.shape, generator=g))
    c.v_scale.copy_(torch.rand(c.v_scale.shape, generator=g))
    old = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    c.move_row(2, 0, 70)
    for t, o, n in zip((c.k, c.v, c.k_scale, c.v_scale), old, (70, 70, 3, 3)):
        assert torch.equal(t[:, 0, :, :n], o[:, 2, :, :n]) and torch.equal(t[:, 0, :, n:], o[:, 0, :, n:])
        assert torch.equal(t[:, 1:], o[:, 1:])
    with pytest.raises(IndexError):
        c.move_row(3, 0, 5)


def test_logprobs_arguments():
    with pytest.raises(_lib.QiError):
        token_logprobs(torch.zeros(1, 10))


@pytest.mark.gpu
def test_python_refusals():
    cfg = qwen2_0p5b(1)
    c = Kv8Cache(cfg, 2, 64, device="cuda")
    q = torch.zeros(3, 14, 64, device="cuda")
    kv = torch.zeros(3, 2, 64, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    bad = [
        lambda: c.attend(0, q[0], i, i), lambda: c.attend(0, q[..., :32], i, i), lambda: c.attend(0, q[:, :13], i, i),
        lambda: c.attend(0, torch.zeros(3, 18, 64, device="cuda"), i, i),
        lambda: c.attend(0, q.to(torch.float64), i, i), lambda: c.attend(0, q.transpose(1, 2)[:, :, :14], i, i),
        lambda: c.attend(0, q, i[:2], i), lambda: c.attend(0, q, i.long(), i), lambda: c.attend(0, q, i, i, window=-1),
        lambda: c.attend(0, q, i, i, sinks=-1), lambda: c.attend(0, q, i, i, out=q[:2]), lambda: c.attend(0, q, i, i, out=q),
        lambda: c.attend(0, q, torch.tensor([0, 1, 2]), i), lambda: c.attend(0, q, i, torch.tensor([0, 64, 2])),
        lambda: c.attend(0, q, i, torch.tensor([0, -2, 2])), lambda: c.append(0, kv, kv[:2], i, i),
        lambda: c.append(0, kv, kv.bfloat16(), i, i), lambda: c.append(0, kv[:, :1], kv[:, :1], i, i),
        lambda: c.append(0, kv, kv, i, torch.tensor([0, 1, 64])), lambda: c.attend(1, q, i, i),
        lambda: token_logprobs(torch.zeros(10, device="cuda")), lambda: token_logprobs(torch.zeros(2, 10, device="cuda"), top=11),
        lambda: token_logprobs(torch.zeros(2, 100, device="cuda"), top=33),
        lambda: token_logprobs(torch.zeros(10, 2, device="cuda").t()),
        lambda: token_logprobs(torch.zeros(1, 10, device="cuda").expand(4, 10)),
        lambda: token_logprobs(torch.zeros(2, 10, device="cuda"), torch.tensor([0, 10])),
        lambda: token_logprobs(torch.zeros(2, 10, device="cuda"), torch.tensor([0.0, 1.0])),
        lambda: token_logprobs(torch.zeros(2, 10, device="cuda", dtype=torch.float64)),
    ]
    for n, f in enumerate(bad):
        with pytest.raises((ValueError, IndexError)):
            f()
            print(n)
    c.check()
    assert c.attend(0, q[:0], i[:0], i[:0]).shape == (0, 14, 64)
    c.append(0, kv[:0], kv[:0], i[:0], i[:0])
    assert token_logprobs(torch.zeros(0, 10, device="cuda"), top=2).top_ids.shape == (0, 2)
