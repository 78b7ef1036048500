"""Log probabilities of tokens from a model's logits, with entropy and alternatives.

The reference only takes the argmax of its logits (qweninfer/engine/engine.py:129,155);
`token_logprobs` is what a caller needs to score given text or to report how sure a
generated token was. One kernel (qi_token_logprobs) reads the logits once.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from qweninfer_b200 import _lib

MAX_TOP = 32


@dataclass
class TokenLogprobs:
    """`logprob`, `entropy` (M,) fp32; `top_ids` (M, top) int32 and `top_logprobs` (M, top)
    fp32, largest first (None for top = 0). Natural logarithms."""
    logprob: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


@dataclass
class TokenInfo:
    """A generated token: its log probability, the entropy of the distribution it was taken
    from, and the best alternatives as (id, log probability), itself first (greedy)."""
    token: int
    logprob: float
    entropy: float
    top: list[tuple[int, float]]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, top: int = 0) -> TokenLogprobs:
    """Per row of `logits` (M, V) (float32, bfloat16 or float16; rows may be strided):
    log softmax at targets[t], the entropy of the distribution, and its `top` (0..32, at
    most V) largest entries, equal logits in the order of their index.

    targets: (M,) int32 or int64 on the logits' device, or on the host, where they are
    checked; a negative target has no log probability and gives 0, one outside the
    vocabulary NaN. A logit of -inf has probability 0. A row with a NaN or +inf logit, or of
    -inf alone, has NaN results. Exponentials and sums are fp32. Enqueued on the current
    stream."""
    key = (logits.shape, logits.stride(), logits.dtype, logits.device, top)
    plan = _plans.get(key)
    if plan is None:
        plan = _plan(logits, top)
        if len(_plans) >= 4096:
            _plans.clear()
        _plans[key] = plan
    M, V, dtype, ld, nbytes = plan
    dev = logits.device
    if targets is not None and not (targets.dtype in _INTS and targets.device == dev and targets.shape == (M,)
                                    and targets.is_contiguous()):
        targets = _targets(targets, M, V, dev)
    f32, new = torch.float32, torch.empty_strided  # (the cheapest of the ways to allocate)
    ent = new((M,), (1,), dtype=f32, device=dev)
    lp = new((M,), (1,), dtype=f32, device=dev) if targets is not None else None
    ids = new((M, top), (top, 1), dtype=torch.int32, device=dev) if top else None
    lps = new((M, top), (top, 1), dtype=f32, device=dev) if top else None
    r = TokenLogprobs(lp, ent, ids, lps)
    if M == 0:
        return r
    if _lib.ready(dev.index):
        code = _call(logits, plan, targets, top, r)
    else:
        with _lib.on_device(dev):
            code = _call(logits, plan, targets, top, r)
    if code:
        _lib.check(code, "qi_token_logprobs")
    return r


def _call(logits: torch.Tensor, plan: tuple, targets: torch.Tensor | None, top: int, r: TokenLogprobs) -> int:
    M, V, dtype, ld, nbytes = plan
    dev = logits.device
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    data, counters, _keep = _lib.scratch(dev, stream, nbytes, _lib.LOGPROBS_COUNTERS)
    y, wide = (None, 0) if targets is None else (targets.data_ptr(), targets.dtype is torch.int64)
    return _lib.lib().qi_token_logprobs(
        logits.data_ptr(), dtype, ld, y, wide, M, V, top, y and r.logprob.data_ptr(), r.entropy.data_ptr(),
        r.top_ids.data_ptr() if top else None, r.top_logprobs.data_ptr() if top else None, data, nbytes, counters, stream)


_INTS = (torch.int32, torch.int64)
_plans: dict[tuple, tuple] = {}


def _plan(logits: torch.Tensor, top: int) -> tuple:
    """What the shapes of a call decide, checked: (M, V, element type, row stride, scratch)."""
    if logits.device.type != "cuda":
        raise _lib.QiError(f"token_logprobs: qweninfer_b200 computes on CUDA (sm_100) tensors only, got {logits.device}")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be (tokens, vocabulary), got {tuple(logits.shape)}")
    if logits.dtype not in _lib.DTYPES:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    M, V = logits.shape
    if logits.stride(1) != 1 or (M > 1 and logits.stride(0) < V):
        raise ValueError("a row of logits must be contiguous and rows must not overlap")
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be 0..{min(MAX_TOP, V)}, got {top}")
    dtype = _lib.DTYPES[logits.dtype]
    with _lib.on_device(logits.device):
        nbytes = _lib.lib().qi_token_logprobs_scratch(M, V, dtype)
    return M, V, dtype, logits.stride(0) if M > 1 else V, nbytes


def _targets(targets: torch.Tensor, M: int, V: int, dev: torch.device) -> torch.Tensor:
    """Targets as (M,) integers on the logits' device; those given on the host are checked."""
    if targets.dim() != 1 or targets.shape[0] != M or targets.dtype not in _INTS:
        raise ValueError(f"targets must be ({M},) int32 or int64, got {tuple(targets.shape)} {targets.dtype}")
    if targets.device.type == "cpu":
        if M and int(targets.max()) >= V:
            raise IndexError("target outside the vocabulary")
        targets = targets.to(dev)
    elif targets.device != dev:
        raise ValueError(f"targets on {targets.device}, logits on {dev}")
    return targets.contiguous()
