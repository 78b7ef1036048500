"""token_logprobs on the GPU against log softmax in 64 bits.

Tolerances: with z = x - max (one rounding), exponentials good to 2^-22 plus 2^-23 |z| for
the rounding of z log2(e), sums of V terms over lanes, warps and slices of at most V / 32
terms each in fp32: Z is known to 2^-21 + 64 2^-24 + log2-sized factors, log Z and z to one
rounding of their size; 2e-6 + 2^-22 |value| covers a log probability, and for the entropy
the weighted sum doubles it."""

from __future__ import annotations

import pytest
import torch

from qweninfer_b200.models.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def logits_of(M, V, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (3 * torch.randn(M, V, generator=g, device="cuda")).to(dtype)


def check(x, targets, top):
    r = token_logprobs(x, targets, top)
    lp = torch.log_softmax(x.double(), -1)
    ent = -(torch.where(lp > -torch.inf, lp.exp() * lp, 0.0)).sum(-1)
    if targets is not None:
        want = lp.gather(1, targets.long().cuda().clamp(min=0)[:, None])[:, 0]
        want = torch.where(targets.cuda() < 0, 0.0, want)
        same = r.logprob.double() == want  # -inf too
        err = torch.where(same, 0.0, (r.logprob.double() - want).abs())
        assert (err <= 2e-6 + 2.0 ** -22 * want.abs()).all(), float(err.max())
    else:
        assert r.logprob is None
    assert ((r.entropy.double() - ent).abs() <= 4e-6 + 2.0 ** -21 * ent).all()
    if top:
        # equal logits in the order of their index: a stable sort
        ids = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids.long(), ids)
        want = lp.gather(1, ids)
        err = torch.where(r.top_logprobs.double() == want, 0.0, (r.top_logprobs.double() - want).abs())
        assert (err <= 2e-6 + 2.0 ** -22 * want.abs()).all()
    else:
        assert r.top_ids is None and r.top_logprobs is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,V", [(1, 1), (1, 31), (3, 33), (2, 1000), (5, 4099), (1, 151936), (7, 32003), (40, 151936)])
def test_sizes(dtype, M, V):
    x = logits_of(M, V, dtype, M + V)
    t = torch.randint(0, V, (M,), generator=torch.Generator().manual_seed(1))
    for top in {0, 1, min(V, 5), min(V, 32)}:
        check(x, t.to(torch.int32).cuda(), top)
    check(x, t, min(V, 3))  # targets on the host, int64
    check(x, None, min(V, 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_and_orders(dtype):
    """Equal logits everywhere, rising and falling rows, all candidates at one end."""
    V = 20011
    ramp = torch.linspace(-30, 30, V, device="cuda")
    x = torch.stack([torch.zeros(V, device="cuda"), ramp, ramp.flip(0), torch.full((V,), -5.0, device="cuda"),
                     (ramp * 0.2).round(), ramp.abs()]).to(dtype)
    x[3, -40:] = 2.0
    check(x, torch.tensor([0, V - 1, 5, V - 1, 77, 3]), 32)


def test_strided_and_unaligned_rows():
    x = logits_of(6, 5003, torch.bfloat16)
    for a, b in ((0, 5003), (1, 5000), (3, 4999), (7, 4103)):
        check(x[:, a:b], torch.tensor([0, 1, 2, 3, 4, -1]), 8)
    check(x[::2, :777], torch.tensor([776, 0, 5]), 8)
    y = logits_of(1, 9001, torch.float32)
    check(y[:, 1:], torch.tensor([8999]), 20)


def test_masked_vocabulary_and_rows_without_a_distribution():
    x = logits_of(7, 6000, torch.float32)
    x[0, 100:] = -torch.inf
    x[1, :] = -torch.inf
    x[1, 5999] = -1e30
    x[2] = torch.finfo(torch.float32).min
    x[2, 17] = 0
    x[3] = torch.finfo(torch.float32).min
    check(x[:4], torch.tensor([5, 5999, 17, 0]), 20)
    r = token_logprobs(x[:1], torch.tensor([200]), 0)
    assert float(r.logprob[0]) == -torch.inf
    x[4] = -torch.inf
    x[5, 3000] = torch.nan
    x[6, 4] = torch.inf
    r = token_logprobs(x[4:], torch.tensor([0, 1, 2]), 4)
    assert r.logprob.isnan().all() and r.entropy.isnan().all() and r.top_logprobs[0].isnan().all()
    assert r.top_ids[0].tolist() == [0, 1, 2, 3] and r.top_ids[2, 0] == 4 and 3000 not in r.top_ids[1].tolist()


def test_targets_outside_on_the_device_give_nan():
    x = logits_of(3, 500, torch.float32)
    r = token_logprobs(x, torch.tensor([500, -1, 2**31], device="cuda"), 0)
    assert r.logprob[0].isnan() and r.logprob[1] == 0 and r.logprob[2].isnan()


def test_streams_and_graphs():
    xs = [logits_of(2, 151936, torch.float32, i) for i in range(2)]
    t = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    want = [token_logprobs(x, t, 5) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(token_logprobs(xs[i], t, 5))
    torch.cuda.synchronize()

    def equal(a, b):
        return all(torch.equal(getattr(a, n), getattr(b, n)) for n in ("logprob", "entropy", "top_ids", "top_logprobs"))
    assert all(equal(r, want[i]) for i in range(2) for r in got[i])
    buf = xs[0].clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, token_logprobs(buf, t, 5)))
    for i in range(2):
        buf.copy_(xs[i])
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(equal(r, want[i]) for _, r in graphs)
