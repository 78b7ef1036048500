"""Attention over cache layers in tiles: what keys next to a token's own may do to it, and the
bits that each type of caller gets, against the formula in 64 bits.

Tolerance of an output element. A score is off by ds: q and k keep 22 bits (2^-22 each of the
absolute dot product), the product of D <= 128 terms is summed in fp32 (D + 3 roundings and
three of the scaling: 134 2^-24), and the difference to the maximum is rounded to 2^-23 of
itself. Weights move by 2 ds in sum, so the output by 2 ds sum w |v|. Of each term w v: the value
keeps 22 bits, the weight p_bits; four exponentials of 2^-22 (the weight, the two factors of a
tile's scale, the rescaling); of sums of n terms in parts of 32 numerator and denominator
(n + 32) 2^-24 each, the last division 2 2^-24 of them. The output is rounded once. Keys that their errors
cannot raise to 2^-60 of the largest weight have no say in ds, and none has where that leaves one; where ds is
above 0.1 the output may be any average of the values that have one."""

from __future__ import annotations

import math

import pytest
import torch

from test_cache_ops_gpu import filled, gen, i32, randn, seen_mask

pytestmark = pytest.mark.gpu


def exact(q, k, v, row, pos, window=0, sinks=0, p_bits=22):
    """(out, tolerance) in 64 bits of tokens of one row"""
    M, H, D = q.shape
    G = H // k.shape[1]
    mask = seen_mask(i32(pos), k.shape[2], window, sinks)
    out, tol = (torch.zeros(M, H, D, dtype=torch.float64, device="cuda") for _ in range(2))
    for h in range(H):
        x = q[:, h].double()
        kk, vv = k[row, h // G].double(), v[row, h // G].double()
        s = (x @ kk.T / math.sqrt(D)).masked_fill(~mask, -torch.inf)
        w = torch.softmax(s, -1)
        out[:, h] = w @ vv
        mag = x.abs() @ kk.abs().T / math.sqrt(D) * (2 * 2.0 ** -22 + 134 * 2.0 ** -24 + 2.0 ** -23)
        mag = mag.masked_fill(~mask, 0)
        top, at = s.max(-1, keepdim=True)
        say = mask & (top - s <= 42 + mag + mag.gather(1, at))
        ds = mag.masked_fill(~say, 0).amax(-1) + 2.0 ** -23 * (top - s).masked_fill(~say, 0).amax(-1)
        ds = torch.where(say.sum(-1) == 1, 0.0, ds)
        c = 5 * 2.0 ** -22 + 2.0 ** -p_bits + 2 * (mask.sum(-1) + 32) * 2.0 ** -24
        some = torch.stack([vv.abs().masked_fill(~y[:, None], 0).amax(0) for y in say])
        tol[:, h] = torch.where((ds > 0.1)[:, None], 2 * some, (w @ vv.abs()) * (2 * ds + c)[:, None] * 1.01)
    return out, tol + out.abs() * (torch.finfo(q.dtype).eps / 2) + 1e-30


def check(cache, k, v, q, row, pos, tiles=True, p_bits=22, **kw):
    got = cache.attend(0, q, i32([row] * len(pos)), i32(pos), query_run=len(pos) if tiles else 1, tiles=tiles, **kw)
    out, tol = exact(q, k, v, row, pos, p_bits=p_bits, **kw)
    err = (got.double() - out).abs()
    assert (err <= tol).all(), (f"off by {float((err / tol).nan_to_num(1e9).max()):.3f} of the bound at "
                                f"{(~(err <= tol)).nonzero()[0].tolist()}")
    return got


# (which tensor, factor on the late key's values)
OUTLIERS = [("v", 2.0 ** 30), ("v", 1e30), ("v", 2.0 ** 12), ("k", 2.0 ** 12), ("kv", 2.0 ** 18),
            ("k", 2.0 ** 30), ("k", 1e30), ("kv", 2.0 ** 40)]


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("which,factor", OUTLIERS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_large_later_key_does_not_reach_earlier_tokens(heads, kv, dim, which, factor, dtype):
    """A key at the end of 16 (and one in the middle of others) with values far above its
    neighbours': the tokens before it, in whose tile it lies, do not change beyond rounding,
    and those behind it see it."""
    cache, (k, v) = filled("bf16", heads, kv, dim, 1, 260, 40)
    for p in (15, 77, 200):
        for name, t in (("k", k), ("v", v)):
            if name in which:
                t[0, :, p] *= factor
    q = (2 * randn(gen(41), 260, heads, dim)).to(dtype)
    check(cache, k, v, q, 0, list(range(260)), p_bits=22 if dtype == torch.float32 else 11)
    check(cache, k, v, q[:150], 0, list(range(60, 210)), window=50, sinks=16, p_bits=22 if dtype == torch.float32 else 11)
    cache.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_large_value_without_weight(dim, dtype):
    """A key that every token sees, with a score far below the others' and values far above."""
    cache, (k, v) = filled("bf16", 8, 2, dim, 1, 200, 42)
    q = (randn(gen(43), 190, 8, dim) + 3).to(dtype)
    k[0, :, 5] = -60.0
    v[0, :, 5] = 1e30
    check(cache, k, v, q, 0, list(range(10, 200)), p_bits=22 if dtype == torch.float32 else 11)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spread", [5, 9, 40, 100])
def test_keys_of_all_sizes_together(dim, spread):
    """Every key with values of its own size, 2^-spread .. 2^spread: each keeps its bits. Scores
    are kept alike, so that small values show."""
    cache, (k, v) = filled("bf16", 6, 2, dim, 1, 180, 44)
    e = torch.linspace(-spread, spread, 180, device="cuda")[torch.randperm(180, generator=gen(45), device="cuda")].round()
    v[0] = (v[0].float() * torch.exp2(e)[:, None]).to(v.dtype)
    k[0] = (k[0].float() * torch.exp2(-e.abs())[:, None]).to(k.dtype)
    q = randn(gen(46), 170, 6, dim)
    check(cache, k, v, q, 0, list(range(10, 180)))


def test_a_late_key_that_is_not_finite():
    """NaN and infinities at the end of 16 keys: the tokens before it match the kernel that reads
    only what it sees."""
    for bad in (float("nan"), float("inf")):
        cache, (k, v) = filled("bf16", 14, 2, 64, 1, 200, 47)
        q = 2 * randn(gen(48), 200, 14, 64)
        v[0, 0, 79, 3] = bad
        k[0, 1, 111, 5] = float("nan")
        pos = list(range(200))
        check(cache, k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), q[:79], 0, pos[:79])
        one = cache.attend(0, q, i32([0] * 200), i32(pos), query_run=1)
        all_ = cache.attend(0, q, i32([0] * 200), i32(pos), query_run=200, tiles=True)
        assert torch.equal(one.isfinite(), all_.isfinite())
        fine = one.isfinite()
        assert float((one[fine] - all_[fine]).abs().max()) <= 1e-4


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 24, 2.0 ** 30, 2.0 ** 60])
def test_scores_far_from_zero(fmt, dim, tiles, size):
    """Queries so large that scores reach 2^20 to 2^66: the largest has all the weight, up to
    ties that 22 bits cannot tell apart."""
    cache, (k, v) = filled(fmt, 8, 2, dim, 1, 200, 51)
    q = randn(gen(52), 150, 8, dim) * size
    q[:, ::2] = q[:, ::2].abs()  # (of one sign: every score is far from zero)
    q[:, 4:6] *= -1
    check(cache, k, v, q, 0, list(range(50, 200)), tiles=tiles)
    check(cache, k, v, q, 0, list(range(50, 200)), tiles=tiles, window=33, sinks=2)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tiles", [False, True])
def test_half_precision_outputs_are_rounded_once(fmt, dim, tiles):
    """fp16 callers: the error is the output's own rounding. Its norm, of the 64-bit result
    rounded to fp16, is within 5 % the same for any result as near as 2^-18 (roundings are as good as random over
    10^5 elements); what comes before it adds at most 2^-18 of the norm, the bar of fp32 callers."""
    cache, vals = filled(fmt, 8, 2, dim, 1, 420, 49)
    q = randn(gen(50), 200, 8, dim).to(torch.float16)
    pos = list(range(220, 420))
    got = cache.attend(0, q, i32([0] * 200), i32(pos), query_run=200 if tiles else 1, tiles=tiles)
    out, _ = exact(q, *vals, 0, pos)
    own = float((out.to(torch.float16).double() - out).norm())
    assert float((got.double() - out).norm()) <= 1.05 * own + 2.0 ** -18 * float(out.norm())


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("low", [-60, -150, -1500])
def test_scores_far_below_zero(fmt, heads, kv, dim, dtype, low):
    """All scores of a row around `low`, in tiles of keys of which some rows see nothing: prompts of
    several cache rows next to each other, and the first tokens of a prompt that runs on into the
    next keys."""
    from test_cache_ops_gpu import config
    from qweninfer_b200.engine.kv_cache import Kv8Cache, KVCache
    g, n = gen(53), 300
    k = randn(g, 3, kv, n, dim) * 0.5 + low / math.sqrt(dim)
    v = randn(g, 3, kv, n, dim)
    if fmt == "bf16":
        cache = KVCache(config(heads, kv, dim), 3, n, device="cuda")
        cache.k[0].copy_(k)
        cache.v[0].copy_(v)
        k, v = cache.k[0], cache.v[0]
    else:
        cache = Kv8Cache(config(heads, kv, dim), 3, n, device="cuda", format=fmt)
        for r in range(3):
            cache.append(0, k[r].transpose(0, 1), v[r].transpose(0, 1), i32([r] * n), i32(range(n)))
        k, v = cache.values(0)
    runs = [(0, 110, 30), (2, 0, 3), (1, 250, 50), (0, 5, 9), (2, 120, 150)]  # row, first position, tokens
    rows = [r for r, a, m in runs for _ in range(m)]
    pos = [p for r, a, m in runs for p in range(a, a + m)]
    q = (1 + 0.05 * randn(g, len(pos), heads, dim)).to(dtype)
    bits = 11 if dtype == torch.bfloat16 else 22
    for window, sinks in ((0, 0), (20, 2)):
        got = cache.attend(0, q, i32(rows), i32(pos), window=window, sinks=sinks, query_run=150, tiles=True)
        for r in range(3):
            at = [i for i, x in enumerate(rows) if x == r]
            out, tol = exact(q[at], k, v, r, [pos[i] for i in at], window, sinks, bits)
            assert ((got[at].double() - out).abs() <= tol).all()
    cache.check()
