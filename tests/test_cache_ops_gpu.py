"""Operators of a cache layer on the GPU, against their formulas in 64 bits: the 8-bit
append (`Kv8Cache.append`, `values`) and attention with window and sinks (`attend`) over
bf16, int8 and e4m3 layers, packed and paged.

Tolerances. The append is defined to the bit. For attention the errors are bounded step by
step (`attention_bound`): parts of q, fp32 dot products, exponentials, parts of p, sums and
the output's own rounding."""

from __future__ import annotations

import math
import random

import pytest
import torch

from qweninfer_b200 import _lib
from qweninfer_b200.engine.kv_cache import Kv8Cache, KVCache, PagedKVCache
from qweninfer_b200.models.config import Qwen2Config

pytestmark = pytest.mark.gpu

TOP = {"int8": 127.0, "e4m3": 448.0}


def config(heads=14, kv_heads=2, dim=64, layers=1):
    return Qwen2Config(vocab_size=1024, hidden_size=heads * dim, intermediate_size=4864, num_hidden_layers=layers,
                       num_attention_heads=heads, num_key_value_heads=kv_heads, max_position_embeddings=4096,
                       rms_norm_eps=1e-6, rope_theta=1e6, tie_word_embeddings=True)


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


# ------------------------------------------------------------------ append oracle

def nearest(x, fmt, s):
    """The code nearest to x whose value, code * s, is finite in fp32."""
    if fmt == "int8":
        return torch.round(x).clamp(-63 if s == 2.0 ** 122 else -127, 63 if s == 2.0 ** 122 else 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-240 if s == 2.0 ** 120 else -448, 240 if s == 2.0 ** 120 else 448)


def least_scale(amax, fmt):
    s = 2.0 ** -126
    while TOP[fmt] * s < amax:
        s *= 2
    return s


class Oracle8:
    """codes and scales of one of K and V, by the definition, in float64 on the CPU"""

    def __init__(self, rows, heads, length, dim, fmt, block):
        self.fmt, self.block = fmt, block
        self.c = torch.zeros(rows, heads, length, dim, dtype=torch.float64)
        self.s = torch.zeros(rows, heads, -(-length // block), dtype=torch.float64)

    def append(self, x, rows, pos):
        x = x.double().cpu()
        cells = {}
        for t, (r, p) in enumerate(zip(rows, pos)):
            if p >= 0:
                cells.setdefault((r, p // self.block), {})[p] = t  # a later token replaces an earlier one
        for (r, b), toks in cells.items():
            f = min(toks)
            for h in range(self.c.shape[1]):
                s = least_scale(max(float(x[t, h].abs().max()) for t in toks.values()), self.fmt)
                if f > b * self.block:
                    old = float(self.s[r, h, b])
                    s = max(s, old)
                    at = slice(b * self.block, f)
                    self.c[r, h, at] = nearest(self.c[r, h, at] * old / s, self.fmt, s)
                for p, t in toks.items():
                    self.c[r, h, p] = nearest(x[t, h] / s, self.fmt, s)
                self.s[r, h, b] = s

    def values(self):
        at = torch.arange(self.c.shape[2]) // self.block
        return self.c * self.s[:, :, at, None]


def same_values(cache, oracles, rows_len):
    for got, want in zip(cache.values(0), oracles):
        want = want.values()
        for r, n in rows_len.items():
            assert torch.equal(got[r, :, :n].double().cpu(), want[r, :, :n]), f"row {r}"


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_append_one_by_one_and_together(fmt, block, dtype):
    """A row grown token by token (its scales grow: every value is a little larger than the
    last), a prompt at once whose last token comes first, and both continued."""
    g = gen(block)
    cache = Kv8Cache(config(), 4, 200, device="cuda", format=fmt, block_tokens=block)
    want = [Oracle8(4, 2, 200, 64, fmt, block) for _ in range(2)]

    def append(k, v, rows, pos):
        cache.append(0, k, v, i32(rows), i32(pos))
        want[0].append(k, rows, pos)
        want[1].append(v, rows, pos)

    for p in range(40):
        k, v = ((randn(g, 2, 2, 64) * 1.25 ** p * 1e-3).to(dtype) for _ in range(2))
        append(k, v, [3, 0], [p, p])
    same_values(cache, want, {3: 40, 0: 40})
    n = 131
    k, v = ((3 * randn(g, n, 2, 64)).to(dtype) for _ in range(2))
    append(k, v, [1] * n, [n - 1] + list(range(n - 1)))
    append(k[:50], v[:50], [3] * 50, list(range(40, 90)))
    same_values(cache, want, {3: 90, 0: 40, 1: n})
    # shorter again, from the middle of a block on
    append(k[:20], v[:20], [1] * 20, list(range(77, 97)))
    same_values(cache, want, {3: 90, 0: 40, 1: 97})
    cache.check()


def test_append_head_layouts_and_strides():
    g = gen(5)
    for heads, kv, dim in ((8, 8, 64), (16, 2, 128), (3, 3, 128)):
        cache = Kv8Cache(config(heads, kv, dim), 2, 70, device="cuda", format="int8", block_tokens=32)
        want = [Oracle8(2, kv, 70, dim, "int8", 32) for _ in range(2)]
        fused = randn(g, 33, (heads + 2 * kv) * dim + 3)  # odd row stride: unaligned slices
        k = fused[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
        v = fused[:, (heads + kv) * dim + 1:(heads + 2 * kv) * dim + 1].unflatten(1, (kv, dim))
        rows, pos = [1] * 33, list(range(20, 53))
        cache.append(0, k, v, i32(rows), i32(pos))
        want[0].append(k, rows, pos)
        want[1].append(v, rows, pos)
        assert torch.equal(cache.values(0)[0][1, :, 20:53].double().cpu(), want[0].values()[1, :, 20:53])
        assert torch.equal(cache.values(0)[1][1, :, 20:53].double().cpu(), want[1].values()[1, :, 20:53])


def test_append_same_position_twice_idle_and_outside():
    g = gen(6)
    cache = Kv8Cache(config(), 2, 64, device="cuda")
    want = [Oracle8(2, 2, 64, 64, "int8", 32) for _ in range(2)]
    k, v = randn(g, 6, 2, 64), randn(g, 6, 2, 64)
    rows, pos = [0, 0, 1, 0, 1, 0], [4, 5, -1, 4, 63, 5]
    cache.append(0, k, v, i32(rows), i32(pos))
    for o, x in zip(want, (k, v)):
        o.append(x, rows, pos)
        assert torch.equal(cache.values(0)[0 if o is want[0] else 1][0, :, 4:6].double().cpu(), o.values()[0, :, 4:6])
    cache.check()
    before = [t.clone() for t in (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)]
    cache.append(0, k[:3], v[:3], i32([0, 2, -1]), i32([64, 0, 0]))
    after = (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    with pytest.raises(_lib.QiError):
        cache.check()


@pytest.mark.parametrize("fmt,block,dtype", [("int8", 16, torch.float32), ("e4m3", 128, torch.bfloat16)])
def test_append_many_tokens_in_any_order(fmt, block, dtype):
    """Enough tokens that a CTA takes several: whole prompts, then the same rows' next tokens
    shuffled among idle slots, tokens outside the cache and positions that come twice."""
    g, r = gen(8), random.Random(8)
    n, length = 9, 400
    cache = Kv8Cache(config(), n, length, device="cuda", format=fmt, block_tokens=block)
    want = [Oracle8(n, 2, length, 64, fmt, block) for _ in range(2)]

    def append(cells):
        rows, pos = [c[0] for c in cells], [c[1] for c in cells]
        k, v = (randn(g, len(cells), 2, 64).to(dtype) for _ in range(2))
        cache.append(0, k, v, i32(rows), i32(pos))
        inside = [i for i, c in enumerate(cells) if 0 <= c[0] < n and 0 <= c[1] < length]
        for o, x in zip(want, (k, v)):
            o.append(x[inside], [rows[i] for i in inside], [pos[i] for i in inside])

    lengths = [r.randrange(100, 250) for _ in range(n)]
    append([(i, p) for i in range(n) for p in range(lengths[i])])
    same_values(cache, want, dict(enumerate(lengths)))
    cache.check()
    more = [r.randrange(1, 120) for _ in range(n)]
    cells = [(i, lengths[i] + p) for i in range(n) for p in range(more[i])]
    cells += r.choices(cells, k=40) + [(r.randrange(n), -1) for _ in range(60)]
    cells += [(n, 3), (-1, 5), (2, length), (4, -2)]
    r.shuffle(cells)
    append(cells)
    same_values(cache, want, {i: lengths[i] + more[i] for i in range(n)})
    with pytest.raises(_lib.QiError):
        cache.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_extreme_values(fmt):
    """Zeros, the smallest and the largest finite values, and values that are not finite."""
    cache = Kv8Cache(config(2, 2), 1, 64, device="cuda", format=fmt, block_tokens=16)
    want = Oracle8(1, 2, 64, 64, fmt, 16)
    k = torch.zeros(4, 2, 64, device="cuda")
    k[1] = 1e-45
    k[2] = 3.4028234663852886e38
    k[2, :, ::2] *= -1
    k[3, 0, 5] = float("nan")
    k[3, 1, 7] = float("-inf")
    pos = [0, 16, 32, 48]
    cache.append(0, k, k, i32([0] * 4), i32(pos))
    want.append(k[:3], [0] * 3, pos[:3])
    for got in cache.values(0):
        assert torch.equal(got[0, :, [0, 16, 32]].double().cpu(), want.values()[0, :, [0, 16, 32]])
        assert got[0, :, 48].isnan().all()
    # the block stays poisoned while it is kept, and starts over with its first position
    cache.append(0, k[:1], k[:1], i32([0]), i32([49]))
    assert cache.values(0)[0][0, :, 48:50].isnan().all()
    one = torch.ones(1, 2, 64, device="cuda")
    cache.append(0, one, one, i32([0]), i32([48]))
    assert torch.equal(cache.values(0)[0][0, :, 48], one[0])


# --------------------------------------------------------------- attention oracle

def seen_mask(pos, length, window, sinks):
    j = torch.arange(length, device="cuda")
    p = pos.long()[:, None]
    m = j <= p
    if window:
        m &= (j > p - window) | (j < sinks)
    return m


def reference(q, k, v, rows, pos, window, sinks):
    """(out, scores' absolute dot products, largest |v|, keys) in 64 bits; k, v are the
    cache's values (rows, kv_heads, length, dim)"""
    M, H, D = q.shape
    hkv = k.shape[1]
    out = torch.zeros(M, H, D, dtype=torch.float64, device="cuda")
    mags = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    vmax = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    mask = seen_mask(pos, k.shape[2], window, sinks)
    for t in range(M):
        if int(pos[t]) < 0:
            continue
        m = mask[t]
        for h in range(H):
            kk, vv = k[rows[t], h // (H // hkv)][m].double(), v[rows[t], h // (H // hkv)][m].double()
            s = kk @ q[t, h].double() / math.sqrt(D)
            out[t, h] = torch.softmax(s, 0) @ vv
            mags[t, h] = (kk.abs() @ q[t, h].double().abs()).max() / math.sqrt(D)
            vmax[t, h] = vv.abs().max()
    return out, mags, vmax


def attention_bound(out, mags, vmax, keys, dtype, bits):
    """Largest error of an element. q and p keep `bits` bits in their parts, so each of their
    products is off by 2^-bits; a dot product of D <= 128 terms in fp32 by at most (D + 3)
    2^-24 of the absolute sum, the scaling to log2 units by two roundings and the scale's
    own (3 2^-24). A score off by ds moves the weights by at most 2 ds in sum; exponentials
    are good to 2^-22 and their differences' rounding to 2^-23 |score|; fp32 sums over n
    terms to n 2^-24, in numerator and denominator."""
    ds = mags * (2.0 ** -bits + 134 * 2.0 ** -24 + 2 * 2.0 ** -23)
    tol = vmax * (2 * ds + 2.0 ** -bits + 2 * (2.0 ** -22 + keys * 2.0 ** -24) + 2.0 ** -22)
    return tol[..., None] * 1.01 + out.abs() * (torch.finfo(dtype).eps / 2)


def check_attend(cache, values, q, rows, pos, window, sinks, run, bits):
    got = cache.attend(0, q, i32(rows), i32(pos), window=window, sinks=sinks, query_run=run, tiles=run > 1)
    assert got.dtype == q.dtype and got.shape == q.shape
    pos_t = torch.as_tensor(pos).cuda()
    out, mags, vmax = reference(q, *values, rows, pos_t, window, sinks)
    tol = attention_bound(out, mags, vmax, max(pos) + 1, q.dtype, bits)
    err = (got.double() - out).abs()
    assert (err <= tol).all(), f"off by {float((err / tol).max()):.3f} of the bound"
    if q.dtype == torch.float32:  # far inside it on average: roundings are random
        assert float((got.double() - out).norm()) <= 4e-6 * max(float(out.norm()), 1e-30)
    return got


def filled(fmt, heads, kv, dim, rows, length, seed, block=32):
    g = gen(seed)
    cfg = config(heads, kv, dim)
    k = randn(g, rows, kv, length, dim) + 2 * randn(g, kv, 1, dim)
    v = randn(g, rows, kv, length, dim)
    if fmt == "bf16":
        cache = KVCache(cfg, rows, length, dtype=torch.bfloat16, device="cuda")
        cache.k[0].copy_(k)
        cache.v[0].copy_(v)
        return cache, (cache.k[0], cache.v[0])
    cache = Kv8Cache(cfg, rows, length, device="cuda", format=fmt, block_tokens=block)
    for r in range(rows):
        cache.append(0, k[r].transpose(0, 1), v[r].transpose(0, 1), i32([r] * length), i32(range(length)))
    return cache, cache.values(0)


def bits_of(fmt, dtype):
    return 21 if fmt != "bf16" else 22 if dtype == torch.float32 else 15


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 3), (100, 4), (64, 70), (300, 1), (10**9, 10**9)])
def test_attend_decode(fmt, dtype, window, sinks):
    cache, values = filled(fmt, 14, 2, 64, 5, 700, 1)
    rows = [3, 0, 4, 1, 2, 0, 3]
    pos = [699, 0, 31, 32, 333, -1, 1]
    q = (2 * randn(gen(2), len(rows), 14, 64)).to(dtype)
    got = check_attend(cache, values, q, rows, pos, window, sinks, 1, bits_of(fmt, dtype))
    assert not got[5].any()
    cache.check()


@pytest.mark.parametrize("fmt,block", [("bf16", 0), ("int8", 16), ("int8", 128), ("e4m3", 64)])
@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 64), (8, 1, 128), (12, 3, 64), (4, 2, 128)])
def test_attend_head_layouts(fmt, block, heads, kv, dim):
    cache, values = filled(fmt, heads, kv, dim, 3, 450, 3, block)
    rows, pos = [1, 2, 0, 1], [449, 17, 200, 60]
    fused = 2 * randn(gen(4), 4, heads * dim + 5)
    q = fused[:, 3:3 + heads * dim].unflatten(1, (heads, dim))  # strided and unaligned
    for window, sinks in ((0, 0), (37, 2)):
        check_attend(cache, values, q, rows, pos, window, sinks, 1, bits_of(fmt, torch.float32))
    cache.check()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
def test_attend_long_rows_split(fmt):
    """One long row over many key splits, and rows of all lengths in one call."""
    cache, values = filled(fmt, 14, 2, 64, 2, 9000, 5)
    q = 2 * randn(gen(6), 1, 14, 64)
    check_attend(cache, values, q, [1], [8999], 0, 0, 1, bits_of(fmt, torch.float32))
    pos = [0, 255, 256, 257, 511, 512, 4000, 8998, -1]
    q = 2 * randn(gen(7), len(pos), 14, 64)
    check_attend(cache, values, q, [0, 1] * 4 + [0], pos, 0, 0, 1, bits_of(fmt, torch.float32))
    check_attend(cache, values, q, [0, 1] * 4 + [0], pos, 3000, 33, 1, bits_of(fmt, torch.float32))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,start,window,sinks", [(2, 0, 0, 0), (77, 0, 0, 0), (64, 130, 0, 0), (150, 40, 32, 4),
                                                  (130, 0, 50, 0), (33, 200, 1, 1)])
def test_attend_prompts(fmt, dtype, n, start, window, sinks):
    """Prompts, and chunks of prompts behind earlier tokens, over two rows; with the other
    rows' single tokens behind them (a batched prefill's order)."""
    cache, values = filled(fmt, 14, 2, 64, 4, 260, 8)
    rows = [2] * n + [0] * n + [1, 3]
    pos = [start + i for i in range(n)] * 2 + [100, 3]
    q = (2 * randn(gen(9), len(rows), 14, 64)).to(dtype)
    for run in (n, 0, 1):
        check_attend(cache, values, q, rows, pos, window, sinks, run, bits_of(fmt, dtype))
    cache.check()


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 64), (5, 5, 128), (16, 2, 128), (3, 1, 64)])
def test_attend_prompts_head_layouts(fmt, heads, kv, dim):
    cache, values = filled(fmt, heads, kv, dim, 2, 300, 26)
    q = 2 * randn(gen(27), 180, heads, dim)
    check_attend(cache, values, q, [1] * 130 + [0] * 50, list(range(170, 300)) + list(range(50)), 0, 0, 130,
                 bits_of(fmt, torch.float32))
    check_attend(cache, values, q, [1] * 130 + [0] * 50, list(range(170, 300)) + list(range(50)), 90, 7, 130,
                 bits_of(fmt, torch.float32))


@pytest.mark.parametrize("n", [511, 513])
def test_attend_prompts_by_size(n):
    """A run on either side of the work from which tiles are taken (2^27)."""
    cache, values = filled("e4m3", 14, 2, 64, 1, 2048, 28)
    q = 2 * randn(gen(29), n, 14, 64)
    check = dict(bits=bits_of("e4m3", torch.float32), window=0, sinks=0)
    got = cache.attend(0, q, i32([0] * n), i32(range(300, 300 + n)), query_run=n)
    tiles = check_attend(cache, values, q, [0] * n, list(range(300, 300 + n)), run=n, **check)
    single = check_attend(cache, values, q, [0] * n, list(range(300, 300 + n)), run=1, **check)
    assert torch.equal(got, tiles if n * 2 * 64 * 2048 >= 2 ** 27 else single)


def test_attend_dead_positions_are_not_read():
    """NaN, infinities and wild scales behind the rows' ends and before the window change
    nothing."""
    for fmt in ("bf16", "int8", "e4m3"):
        cache, _ = filled(fmt, 14, 2, 64, 2, 400, 10)
        q = 2 * randn(gen(11), 40, 14, 64)
        rows, pos = i32([0] * 39 + [1]), i32(list(range(170, 209)) + [5])
        clean = [cache.attend(0, q, rows, pos, window=60, sinks=5, query_run=r, tiles=r > 1) for r in (1, 39)]
        lo, hi = 111, 208  # seen by row 0's tokens: the window's union, and the sinks
        for t in (cache.k, cache.v):
            if fmt == "bf16":
                for a, b in ((5, lo), (hi + 1, 400)):
                    t[0, 0, :, a:b] = float("nan")
                t[0, 1, :, 6:] = float("inf")
            elif fmt == "e4m3":
                bad = t.view(torch.uint8)
                bad[0, 0, :, 5:lo] = 0x7F
                bad[0, 0, :, hi + 1:] = 0xFF
                bad[0, 1, :, 6:] = 0x7F
        if fmt != "bf16":
            for s in (cache.k_scale, cache.v_scale):
                s[0, 0, :, 32 // 32:lo // 32] = float("nan")
                s[0, 0, :, hi // 32 + 1:] = float("inf")
                s[0, 1, :, 1:] = float("nan")
        for r, want in zip((1, 39), clean):
            assert torch.equal(cache.attend(0, q, rows, pos, window=60, sinks=5, query_run=r, tiles=r > 1), want)


def test_attend_values_that_are_seen_show():
    """A NaN that a token does see reaches its output, and only its."""
    cache, _ = filled("bf16", 14, 2, 64, 1, 100, 12)
    q = 2 * randn(gen(13), 3, 14, 64)
    rows, pos = i32([0, 0, 0]), i32([9, 10, 99])
    clean = cache.attend(0, q, rows, pos, query_run=1)
    cache.v[0, 0, 0, 10, 3] = float("nan")
    got = cache.attend(0, q, rows, pos, query_run=1)
    assert torch.equal(got[0], clean[0])
    assert got[1:, :7, 3].isnan().all() and torch.equal(got[1:, 7:], clean[1:, 7:])


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e4])
def test_attend_ranges(scale):
    """Queries and values far from 1; scores that differ by hundreds."""
    cache, values = filled("int8", 14, 2, 64, 1, 300, 14)
    q = randn(gen(15), 2, 14, 64) * scale
    got = cache.attend(0, q, i32([0, 0]), i32([299, 10]), query_run=1)
    out, _, _ = reference(q, *values, [0, 0], torch.tensor([299, 10]).cuda(), 0, 0)
    # a score of size 1e5 is known to 2^-21 of itself (0.05): weights of near-ties shift
    tol = 2e-5 if scale < 1 else 0.5
    assert float((got.double() - out).abs().max()) <= tol * float(values[1].abs().max())


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_offsets_beyond_32_bits(fmt):
    """A row whose last heads lie more than 2^32 elements into the layer, against a short one
    with the same keys: positions apart by a multiple of every block and tile."""
    long, short, n = 2 ** 22 + 2 ** 18, 256, 200
    base = long - short
    g, cfg = gen(31), config(8, 8, 128)
    k, v = (randn(g, n, 8, 128) for _ in range(2))
    q = 2 * randn(g, 40, 8, 128)
    pos = list(range(n - 40, n))

    def make(length, at):
        if fmt == "int8":
            c = Kv8Cache(cfg, 1, length, device="cuda")
            c.append(0, k, v, i32([0] * n), i32(range(at, at + n)))
            return c
        c = KVCache(cfg, 1, length, dtype=torch.bfloat16, device="cuda")
        c.k[0, 0, :, at:at + n], c.v[0, 0, :, at:at + n] = k.transpose(0, 1), v.transpose(0, 1)
        return c

    near, far = make(short, 0), make(long, base)
    assert far.k[0].numel() > 2 ** 32
    values = near.values(0) if fmt == "int8" else (near.k[0], near.v[0])
    for window in (1, 100):
        out, mags, vmax = reference(q, *values, [0] * 40, i32(pos), window, 0)
        tol = attention_bound(out, mags, vmax, n, q.dtype, bits_of(fmt, q.dtype))
        for tiles in (False, True):
            got = far.attend(0, q, i32([0] * 40), i32([base + p for p in pos]), window=window, query_run=40, tiles=tiles)
            assert ((got.double() - out).abs() <= tol).all()
    far.check()


def test_attend_paged_matches_packed():
    g = gen(16)
    cfg = config()
    packed = KVCache(cfg, 3, 500, dtype=torch.bfloat16, device="cuda")
    paged = PagedKVCache(cfg, 3, 500, device="cuda", page_size=128, n_pages=14)
    packed.k.copy_(randn(g, *packed.k.shape))
    packed.v.copy_(randn(g, *packed.v.shape))
    order = [(r, b) for b in range(4) for r in (2, 0, 1)]
    for r, b in order:  # scattered pages
        paged.reserve(r, min(500, 128 * (b + 1)))
    for r in range(3):
        for b in range(4):
            pg, n = int(paged._t[r, b]), min(128, 500 - 128 * b)
            paged.k[0, pg, :, :n] = packed.k[0, r, :, 128 * b:128 * b + n]
            paged.v[0, pg, :, :n] = packed.v[0, r, :, 128 * b:128 * b + n]
    q = 2 * randn(g, 130, 14, 64)
    rows, pos = i32([2] * 127 + [0, 1, 1]), i32(list(range(300, 427)) + [499, 128, -1])
    for run in (1, 127):
        for window, sinks in ((0, 0), (70, 3)):
            assert torch.equal(paged.attend(0, q, rows, pos, window, sinks, run, tiles=run > 1),
                               packed.attend(0, q, rows, pos, window, sinks, run, tiles=run > 1))
    paged.check()
    # a window's released pages are not touched; a page that is seen and missing is reported
    paged._t[2, 0] = -1
    paged.dirty = True
    assert torch.equal(paged.attend(0, q[:127], rows[:127], pos[:127], 100, 0, 127, tiles=True),
                       packed.attend(0, q[:127], rows[:127], pos[:127], 100, 0, 127, tiles=True))
    paged.check()
    paged.attend(0, q[:127], rows[:127], pos[:127], 100, 4, 127, tiles=True)
    with pytest.raises(_lib.QiError):
        paged.check()


def test_attend_outside_the_cache_is_reported():
    cache, values = filled("int8", 14, 2, 64, 2, 64, 17)
    q = randn(gen(18), 5, 14, 64)
    for run in (1, 5):
        cache._errors().zero_()
        got = cache.attend(0, q, i32([0, 0, 2, -1, 1]), i32([64, -2, 3, 3, 63]), query_run=run, tiles=run > 1)
        assert not got[:4].any() and got[4].any()
        with pytest.raises(_lib.QiError):
            cache.check()


def test_streams_graphs_and_reuse():
    """Calls on two streams at once, a captured step replayed over changing inputs next to
    an eager call of another size, and the same call twice give the same bits."""
    cache, _ = filled("int8", 14, 2, 64, 4, 4000, 19)
    q = [2 * randn(gen(20 + i), 4, 14, 64) for i in range(2)]
    rows, pos = i32([0, 1, 2, 3]), i32([3999, 100, 2500, -1])
    want = [cache.attend(0, x, rows, pos, query_run=1) for x in q]
    one = cache.attend(0, q[0][:1], rows[:1], pos[:1], query_run=1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attend(0, q[i], rows, pos, query_run=1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    buf = q[0].clone()
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed at once on two streams
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, cache.attend(0, buf, rows, pos, query_run=1)))
    for i in range(2):
        buf.copy_(q[i])
        torch.cuda.synchronize()
        for (gr, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        eager = cache.attend(0, q[0][:1], rows[:1], pos[:1], query_run=1)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[i]) for _, out in graphs) and torch.equal(eager, one)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_captured_prompts(fmt):
    """A prompt with another row's single token behind it, captured and replayed over changing
    queries and positions while eager calls run on another stream: the eager calls' bits."""
    cache, _ = filled(fmt, 14, 2, 64, 3, 700, 32)
    q = [2 * randn(gen(33 + i), 151, 14, 64) for i in range(2)]
    rows = i32([1] * 150 + [2])
    pos = [i32(list(range(a, a + 150)) + [a]) for a in (400, 17)]
    want = [cache.attend(0, q[i], rows, pos[i], query_run=150, tiles=True) for i in range(2)]
    qb, pb = q[0].clone(), pos[0].clone()
    side, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        out = cache.attend(0, qb, rows, pb, query_run=150, tiles=True)
    for i in (0, 1, 0):
        qb.copy_(q[i])
        pb.copy_(pos[i])
        gr.replay()
        with torch.cuda.stream(side):
            eager = cache.attend(0, q[1 - i], rows, pos[1 - i], query_run=150, tiles=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(eager, want[1 - i])
    cache.check()


def test_append_then_attend_as_a_server_does():
    """A prompt and decode steps through append and attend, against attention over what the
    cache stands for; a row move keeps a row's outputs; rows behind the last are untouched."""
    g = gen(30)
    cache = Kv8Cache(config(), 4, 160, device="cuda", format="e4m3", block_tokens=16)
    n = 70
    k, v = randn(g, n, 2, 64), randn(g, n, 2, 64)
    q = 2 * randn(g, n, 14, 64)
    rows = [2] * n
    cache.append(0, k, v, i32(rows), i32(range(n)))
    check_attend(cache, cache.values(0), q, rows, list(range(n)), 0, 0, n, 21)
    for p in range(n, n + 20):
        k, v = randn(g, 2, 2, 64), randn(g, 2, 2, 64)
        cache.append(0, k, v, i32([2, 0]), i32([p, p - n]))
        q = 2 * randn(g, 2, 14, 64)
        check_attend(cache, cache.values(0), q, [2, 0], [p, p - n], 40, 4, 1, 21)
    before = cache.attend(0, q, i32([2, 0]), i32([n + 19, 19]), query_run=1)
    cache.move_row(2, 1, n + 20)
    assert torch.equal(cache.attend(0, q, i32([1, 0]), i32([n + 19, 19]), query_run=1), before)
    assert not cache.k[0, 3].view(torch.int8).any() and not cache.k_scale[0, 3].any()
    cache.check()
