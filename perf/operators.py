"""Operators of the bounded-memory serving path, as cases to measure.

Three kinds of call, each in its plain form (elementary torch operations in fp32) and as a
user of qweninfer_b200 makes it (`own`):

* `append`: new keys and values into a cache of 8-bit codes with one scale for each block
  of tokens and KV head, and the values that the cache then stands for;
* `attend`: grouped-query attention over a cache (bf16, int8 or e4m3), optionally with a
  sliding window and first tokens that stay visible;
* `logprobs`: log probabilities of given tokens, entropy and top alternatives from logits.

Shapes: 14 query and 2 KV heads of 64 dimensions and a vocabulary of 151936 are this
package's model; the drawn cases add other head layouts and vocabularies.

The 8-bit cache. A block is `block` consecutive positions of one cache row and KV head (K
and V apart). Its scale is a power of two, the least 2^e with top * 2^e >= every absolute
value appended to it (top = 127 for int8, 448 for e4m3), and a value x is held as the
nearest code to x / 2^e, ties to even. Appending at position p keeps the positions before
p: where they share a block with p, a larger scale rounds their codes again (code * old /
new), and a block whose first position is appended starts over. Positions after the last
appended one are dead.

Attention. The query at position p of its row sees key j if 0 <= j <= p and either no
window is set, or j > p - window, or j < sinks. p = -1 marks an idle slot: nothing is
seen and the output is zero.
"""

import math

import torch

own = False

VOCAB = 151936
TOP_CODE = {"int8": 127.0, "e4m3": 448.0}
CODE_DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ESIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------ cases

def listed():
    model = {"heads": 14, "kv_heads": 2, "dim": 64}
    return [
        # one decode step of 32 slots: one token per row into an int8 cache
        {"name": "append_step", "op": "append", **model, "rows": 32, "tokens": 1, "max_len": 256,
         "format": "int8", "block": 32, "dtype": "fp32"},
        # four prompts admitted together, K and V as slices of one fused projection output
        {"name": "append_prompts", "op": "append", **model, "rows": 4, "tokens": 1000, "max_len": 1100,
         "format": "e4m3", "block": 64, "dtype": "bf16"},
        # interactive decode: a single short row, where the call's latency is all there is
        {"name": "kv8_step", "op": "attend", **model, "rows": 1, "tokens": 1, "max_len": 1024, "context": 700,
         "idle": 0, "format": "int8", "block": 32, "window": 0, "sinks": 0, "dtype": "fp32"},
        # a full decode batch: 64 slots of ragged lengths up to 4096, two of them idle
        {"name": "kv8_batch", "op": "attend", **model, "rows": 64, "tokens": 1, "max_len": 4096, "context": 4096,
         "idle": 2, "format": "int8", "block": 32, "window": 0, "sinks": 0, "dtype": "fp32"},
        # two long documents: few rows, the key axis carries the work
        {"name": "kv8_long", "op": "attend", **model, "rows": 2, "tokens": 1, "max_len": 131072,
         "context": 131071, "idle": 0, "format": "e4m3", "block": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
        # the last chunk of a long prompt over the 8-bit cache
        {"name": "kv8_prompt", "op": "attend", **model, "rows": 1, "tokens": 1024, "max_len": 4096,
         "context": 4096, "idle": 0, "format": "int8", "block": 32, "window": 0, "sinks": 0, "dtype": "bf16"},
        # a decode batch over the bf16 cache with a window and four first tokens
        {"name": "window_batch", "op": "attend", **model, "rows": 64, "tokens": 1, "max_len": 4096, "context": 4096,
         "idle": 0, "format": "bf16", "block": 0, "window": 1024, "sinks": 4, "dtype": "fp32"},
        # a whole prompt under a window, as the model's forward runs it (fp32 activations)
        {"name": "window_prompt", "op": "attend", **model, "rows": 1, "tokens": 4000, "max_len": 4096,
         "context": 4000, "idle": 0, "format": "bf16", "block": 0, "window": 1024, "sinks": 4, "dtype": "fp32"},
        # window and 8-bit cache together on long rows
        {"name": "kv8_window", "op": "attend", **model, "rows": 8, "tokens": 1, "max_len": 32768, "context": 32768,
         "idle": 0, "format": "e4m3", "block": 32, "window": 8000, "sinks": 64, "dtype": "fp32"},
        # one sampled token of one sequence with its five best alternatives
        {"name": "logprobs_step", "op": "logprobs", "tokens": 1, "vocab": VOCAB, "top": 5, "dtype": "fp32"},
        # a decode batch's logits with the twenty best alternatives
        {"name": "logprobs_batch", "op": "logprobs", "tokens": 64, "vocab": VOCAB, "top": 20, "dtype": "bf16"},
        # scoring a text of a thousand tokens
        {"name": "logprobs_score", "op": "logprobs", "tokens": 1000, "vocab": VOCAB, "top": 1, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([VOCAB, _log_int(rng, 1000, VOCAB), 32 * _log_int(rng, 32, 4700)])
        return {"op": op, "tokens": _log_int(rng, 1, 1000), "vocab": vocab,
                "top": rng.choice([0, 1, 5, _log_int(rng, 1, 20)]), "dtype": rng.choice(["fp32", "bf16"])}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (14, 2, 64), (8, 8, 64), (12, 3, 64), (16, 2, 128), (8, 2, 128)])
    model = {"heads": heads, "kv_heads": kv_heads, "dim": dim}
    if op == "append":
        tokens = rng.choice([1, _log_int(rng, 1, 1000)])
        rows = _log_int(rng, 1, 64) if tokens == 1 else _log_int(rng, 1, 4)
        return {"op": op, **model, "rows": rows, "tokens": tokens, "max_len": tokens + rng.randint(1, 200),
                "format": rng.choice(["int8", "e4m3"]), "block": rng.choice([16, 32, 64, 128]),
                "dtype": rng.choice(["fp32", "bf16"])}
    tokens = rng.choice([1, 1, _log_int(rng, 2, 1000)])
    if tokens == 1:
        rows = _log_int(rng, 1, 64)
        context = _log_int(rng, 1, min(65536, 262144 // rows))
    else:
        rows = _log_int(rng, 1, 4)
        context = tokens + rng.randint(0, 1024)
    fmt = rng.choice(["bf16", "int8", "e4m3"])
    window, sinks = (0, 0)
    if fmt == "bf16" or rng.random() < 0.5:
        window, sinks = _log_int(rng, 1, max(2, context)), rng.choice([0, 1, 4, rng.randint(0, 100)])
    return {"op": op, **model, "rows": rows, "tokens": tokens, "max_len": context + rng.randint(0, 100),
            "context": context, "idle": 0 if rows < 4 or tokens > 1 else rng.choice([0, 1]), "format": fmt,
            "block": 0 if fmt == "bf16" else rng.choice([16, 32, 64, 128]), "window": window, "sinks": sinks,
            "dtype": rng.choice(["fp32", "bf16"])}


# ---------------------------------------------------------------------- prepare

def _config(case):
    from qweninfer_b200.models.config import Qwen2Config
    return Qwen2Config(vocab_size=VOCAB, hidden_size=case["heads"] * case["dim"], intermediate_size=4864,
                       num_hidden_layers=1, num_attention_heads=case["heads"],
                       num_key_value_heads=case["kv_heads"], max_position_embeddings=case["max_len"],
                       rms_norm_eps=1e-6, rope_theta=1000000.0, tie_word_embeddings=True)


def _scale_of(amax, fmt):
    """The least power of two s with TOP_CODE * s >= amax (2^-126 for amax = 0)."""
    m, e = torch.frexp(amax)
    top_m, top_e = math.frexp(TOP_CODE[fmt])
    return torch.ldexp(torch.ones_like(amax), (e - top_e + (m > top_m)).clamp(min=-126).where(amax > 0, -126))


def _codes(x, fmt):
    """x (in units of the scale) as the codes' values, ties to even."""
    return torch.round(x) if fmt == "int8" else x.to(torch.float8_e4m3fn).to(torch.float32)


def _quantised(x, fmt, block):
    """A filled cache (rows, kv_heads, len, dim) as codes and scales."""
    r, h, n, d = x.shape
    nb = -(-n // block)
    pad = torch.nn.functional.pad(x, (0, 0, 0, nb * block - n)).view(r, h, nb, block, d)
    s = _scale_of(pad.abs().amax((-1, -2)), fmt)
    c = _codes(pad / s[..., None, None], fmt).view(r, h, nb * block, d)[:, :, :n]
    return c.to(CODE_DTYPE[fmt]).contiguous(), s


def _values(codes, scale, block):
    """Codes and scales as the fp32 values that they stand for."""
    return codes.to(torch.float32) * scale.repeat_interleave(block, 2)[:, :, :codes.shape[2], None]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dev = torch.device("cuda")

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "logprobs":
        # a peaked distribution: unit noise with a few thousand raised candidates
        m, v = case["tokens"], case["vocab"]
        x = randn(m, v)
        x *= 2.5
        hot = torch.randint(0, v, (m, max(1, v // 50)), generator=g, device=dev)
        x.scatter_add_(1, hot, 3 * randn(m, hot.shape[1]))
        return {"case": case, "logits": x.to(DTYPE[case["dtype"]]),
                "targets": torch.randint(0, v, (m,), generator=g, device=dev).to(torch.int32)}

    rows, n, length = case["rows"], case["tokens"], case["max_len"]
    hq, hkv, d, fmt = case["heads"], case["kv_heads"], case["dim"], case["format"]
    dt = DTYPE[case["dtype"]]
    cache_rows = rows + 1
    # the call's rows, in an order of their own
    row = torch.randperm(cache_rows, generator=g, device=dev)[:rows]
    # keys with the channel offsets that a projection bias gives them
    k = randn(cache_rows, hkv, length, d) + 2 * randn(hkv, 1, d)
    v = randn(cache_rows, hkv, length, d)
    st = {"case": case}
    if case["op"] == "append":
        start = torch.randint(0, length - n + 1, (rows,), generator=g, device=dev)
        fused = torch.cat([randn(rows * n, hq * d), randn(rows * n, hkv * d) + 2 * randn(hkv * d),
                           randn(rows * n, hkv * d)], 1).to(dt)
        # as a fused projection leaves them: slices with a longer row stride
        st["k"] = fused[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        st["v"] = fused[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        # the earlier tokens are in the cache; what lies behind them is dead
        live = (torch.arange(length, device=dev) < torch.zeros(cache_rows, 1, device=dev, dtype=torch.long)
                .index_copy(0, row, start[:, None]))[:, None, :, None]
        k, v = k * live, v * live
        pos = start[:, None] + torch.arange(n, device=dev)
        st["start"] = start
    else:
        # ragged contexts: the first row has the longest, the others between a half and all of it
        last = torch.randint((case["context"] + 1) // 2, case["context"] + 1, (rows,), generator=g, device=dev)
        last[0] = case["context"]
        last = last.clamp(min=n)
        pos = last[:, None] - n + torch.arange(n, device=dev)
        if case["idle"]:
            pos[rows - case["idle"]:] = -1
        st["q"] = (2 * randn(rows * n, hq, d)).to(dt)
    if fmt == "bf16":
        st["kc"], st["vc"] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    else:
        st["kc"], st["ks"] = _quantised(k, fmt, case["block"])
        st["vc"], st["vs"] = _quantised(v, fmt, case["block"])
    st["row"], st["pos2"] = row, pos
    st["rows"] = row.repeat_interleave(n).to(torch.int32)
    st["pos"] = pos.reshape(-1).to(torch.int32)
    if own:
        from qweninfer_b200.engine.kv_cache import Kv8Cache, KVCache
        cfg = _config(case)
        if fmt == "bf16":
            cache = KVCache(cfg, cache_rows, length, dtype=torch.bfloat16, device=dev)
        else:
            cache = Kv8Cache(cfg, cache_rows, length, device=dev, format=fmt, block_tokens=case["block"])
            cache.k_scale[0].copy_(st["ks"])
            cache.v_scale[0].copy_(st["vs"])
        cache.k[0].copy_(st["kc"])
        cache.v[0].copy_(st["vc"])
        st["cache"] = cache
        for name in ("kc", "vc", "ks", "vs"):
            st.pop(name, None)
    return st


# -------------------------------------------------------------------------- run

def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state)
    return {"append": _append, "attend": _attend, "logprobs": _logprobs}[op](state)


def _run_own(st):
    c = st["case"]
    if c["op"] == "logprobs":
        from qweninfer_b200.models.logprobs import token_logprobs
        r = token_logprobs(st["logits"], st["targets"], top=c["top"])
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if c["top"]:
            out.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs)
        return out
    cache = st["cache"]
    if c["op"] == "append":
        cache.append(0, st["k"], st["v"], st["rows"], st["pos"])
        k, v = cache.values(0)
        return {"k": k, "v": v}
    return cache.attend(0, st["q"], st["rows"], st["pos"], window=c["window"], sinks=c["sinks"],
                        query_run=c["tokens"])


def _append(st):
    c = st["case"]
    k = _appended(st, st["k"], st["kc"], st["ks"])
    v = _appended(st, st["v"], st["vc"], st["vs"])
    return {"k": _values(*k, c["block"]), "v": _values(*v, c["block"])}


def _appended(st, x, codes, scale):
    """One of K and V with the call's tokens in it: codes and scales are updated in place."""
    c = st["case"]
    fmt, block, r, n = c["format"], c["block"], c["rows"], c["tokens"]
    h, d, length, nb = c["kv_heads"], c["dim"], c["max_len"], scale.shape[2]
    row, pos, start = st["row"], st["pos2"], st["start"]
    # the rows' new values by position, in whole blocks
    new = torch.zeros(r, nb * block, h, d, device=x.device)
    new.scatter_(1, pos[:, :, None, None].expand(r, n, h, d), x.reshape(r, n, h, d).float())
    new = new.permute(0, 2, 1, 3).reshape(r, h, nb, block, d)
    at = torch.arange(nb * block, device=x.device).view(1, nb, block)
    is_new = (at >= start[:, None, None]) & (at < start[:, None, None] + n)
    is_old = at < start[:, None, None]
    touched = is_new.any(-1)
    kept = touched & is_old.any(-1)  # blocks that hold earlier positions too
    s_old = scale[row]
    s = torch.where(kept[:, None], torch.maximum(s_old, _scale_of(new.abs().amax((-1, -2)), fmt)),
                    _scale_of(new.abs().amax((-1, -2)), fmt))
    old = torch.nn.functional.pad(codes[row].float(), (0, 0, 0, nb * block - length)).view(r, h, nb, block, d)
    again = _codes(old * (s_old / s)[..., None, None].where(kept[:, None, :, None, None], 1.0), fmt)
    now = torch.where(is_new[:, None, ..., None], _codes(new / s[..., None, None], fmt),
                      torch.where((kept[..., None] & is_old)[:, None, ..., None], again, old))
    codes[row] = now.view(r, h, nb * block, d)[:, :, :length].to(codes.dtype)
    scale[row] = torch.where(touched[:, None], s, s_old)
    return codes, scale


def _attend(st):
    c = st["case"]
    r, n, hkv, d = c["rows"], c["tokens"], c["kv_heads"], c["dim"]
    if c["format"] == "bf16":
        k, v = st["kc"][st["row"]].float(), st["vc"][st["row"]].float()
    else:
        k = _values(st["kc"][st["row"]], st["ks"][st["row"]], c["block"])
        v = _values(st["vc"][st["row"]], st["vs"][st["row"]], c["block"])
    q = st["q"].float().view(r, n, hkv, -1, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, -1, d)  # (heads of a group, tokens)
    s = q @ k.transpose(-1, -2)
    s *= 1 / math.sqrt(d)
    j = torch.arange(k.shape[2], device=q.device)
    p = st["pos2"][..., None]
    seen = j <= p
    if c["window"]:
        seen &= (j > p - c["window"]) | (j < c["sinks"])
    s = s.view(r, hkv, -1, n, s.shape[-1]).masked_fill_(~seen[:, None, None], -torch.inf)
    top = s.amax(-1, keepdim=True)
    s -= top.where(top > -torch.inf, 0.0)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    o = (s.view(r, hkv, -1, s.shape[-1]) @ v).view(r, hkv, -1, n, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(r * n, -1, d).to(st["q"].dtype)


def _logprobs(st):
    x = st["logits"].float()
    top = x.amax(-1, keepdim=True)
    z = x - top
    e = z.exp()
    total = e.sum(-1)
    lse = total.log()
    out = {"logprob": z.gather(1, st["targets"].long()[:, None])[:, 0] - lse,
           "entropy": lse - (e * z).sum(-1) / total}
    n = st["case"]["top"]
    if n:
        # the order of floats as integers, then the lower index: ties are decided
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = key * 2**20 + (2**20 - 1 - torch.arange(x.shape[1], device=x.device))
        best = key.topk(n, dim=-1).indices
        out["top_ids"] = best.to(torch.int32)
        out["top_logprobs"] = z.gather(1, best) - lse[:, None]
    return out


# ------------------------------------------------------------------------- work

def _visible(case):
    """Keys that the call's queries can see, each counted once, and query-key pairs (the
    rows' mean context is three quarters of the longest)."""
    n, w, k = case["tokens"], case["window"], case["sinks"]
    keys = pairs = 0
    for i in range(case["rows"] - case["idle"]):
        end = max(n, case["context"] if i == 0 else round(0.75 * case["context"]))
        if not w:
            keys += end
            pairs += n * end - n * (n - 1) // 2
            continue
        lo = max(0, end - n - w + 1)  # the first query's first key under the window
        keys += end - lo + min(k, lo)
        pairs += sum(min(p + 1, w) + min(k, max(0, p + 1 - w)) for p in range(end - n, end))
    return keys, pairs


def work(case):
    if case["op"] == "logprobs":
        m, v = case["tokens"], case["vocab"]
        return {"bytes": m * v * ESIZE[case["dtype"]] + m * (12 + 8 * case["top"]), "flops": 6 * m * v}
    hkv, d, es = case["kv_heads"], case["dim"], ESIZE[case["dtype"]]
    t = case["rows"] * case["tokens"]
    if case["op"] == "append":
        cells = (case["rows"] + 1) * hkv * case["max_len"] * d
        scales = 4 * (case["rows"] + 1) * hkv * -(-case["max_len"] // case["block"])
        # K and V each: the tokens read, their codes written; all codes read, their values written
        return {"bytes": 2 * (t * hkv * d * (es + 1) + cells * 5 + scales) + 8 * t, "flops": 4 * t * hkv * d + 2 * cells}
    keys, pairs = _visible(case)
    per = 2 * d * (2 if case["format"] == "bf16" else 1) + (8 / case["block"] if case["block"] else 0)
    return {"bytes": keys * hkv * per + t * (2 * case["heads"] * d * es + 8), "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------------ exact

def _nearest_code(x, fmt):
    """The code nearest to x, ties to even: e4m3 has steps of 2^(e - 3) in [2^e, 2^(e + 1)),
    e >= -6."""
    if fmt == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(st, x, codes, scale):
    """Block by block, as the module's text says it."""
    c = st["case"]
    fmt, block, n = c["format"], c["block"], c["tokens"]
    codes, scale, x = codes.double().cpu(), scale.double().cpu(), x.double().cpu()
    for i, r in enumerate(st["row"].tolist()):
        first = int(st["start"][i])
        for b in range(first // block, (first + n - 1) // block + 1):
            lo, hi = max(b * block, first), min((b + 1) * block, first + n)
            new = x[i * n + lo - first:i * n + hi - first].transpose(0, 1)  # (kv_heads, positions, dim)
            for h in range(c["kv_heads"]):
                amax = float(new[h].abs().max())
                s = 2.0 ** -126
                while TOP_CODE[fmt] * s < amax:
                    s *= 2
                if lo > b * block:
                    old = float(scale[r, h, b])
                    s = max(s, old)
                    codes[r, h, b * block:lo] = _nearest_code(codes[r, h, b * block:lo] * old / s, fmt)
                codes[r, h, lo:hi] = _nearest_code(new[h] / s, fmt)
                scale[r, h, b] = s
    at = torch.arange(codes.shape[2]) // block
    return codes * scale[:, :, at, None]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        out = {"logprob": [], "entropy": [], "top_ids": None, "top_logprobs": []}
        for i in range(case["tokens"]):
            x = st["logits"][i].double()
            lp = x - torch.logsumexp(x, 0)
            out["logprob"].append(lp[st["targets"][i].long()])
            out["entropy"].append(-(lp.exp() * lp).sum())
            out["top_logprobs"].append(lp.topk(case["top"]).values)
        out = {k: None if v is None else torch.stack(v) for k, v in out.items()}
        if not case["top"]:
            del out["top_ids"], out["top_logprobs"]
        return out
    if case["op"] == "append":
        return {"k": _exact_append(st, st["k"], st["kc"], st["ks"]),
                "v": _exact_append(st, st["v"], st["vc"], st["vs"])}
    hkv, d, n = case["kv_heads"], case["dim"], case["tokens"]
    group = case["heads"] // hkv
    q = st["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i, r in enumerate(st["row"].tolist()):
        side = []
        for c, s in ((st["kc"], st.get("ks")), (st["vc"], st.get("vs"))):
            x = c[r].double()
            if s is not None:
                x = x * s[r].double()[:, torch.arange(x.shape[1], device=x.device) // case["block"], None]
            side.append(x)
        for first in range(0, n, 256):  # queries of one row, some at a time
            at = st["pos2"][i, first:first + 256]
            if int(at[0]) < 0:
                continue
            key = torch.arange(case["max_len"], device=q.device)
            hidden = key[None] > at[:, None]
            if case["window"]:
                hidden |= (key[None] <= at[:, None] - case["window"]) & (key[None] >= case["sinks"])
            for h in range(case["heads"]):
                lo = i * n + first
                s = q[lo:lo + at.numel(), h] @ side[0][h // group].T / math.sqrt(d)
                w = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
                out[lo:lo + at.numel(), h] = w @ side[1][h // group]
    return out
