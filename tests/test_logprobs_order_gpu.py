"""Order of the alternatives of `token_logprobs` where it goes by index, or past NaN."""

from __future__ import annotations

import pytest
import torch

from qweninfer_b200.models.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def best(x, top):
    """Indices of the `top` largest, equal ones (zeros of either sign are) in order, NaN none."""
    x = x.double() + 0.0
    ids = torch.sort(x.nan_to_num(-torch.inf), dim=-1, descending=True, stable=True).indices[:, :top]
    return torch.where(x.gather(1, ids).isnan(), -1, ids)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [2, 40, 3001, 151936])
def test_zeros_of_either_sign_are_equal(dtype, V):
    g = torch.Generator("cuda").manual_seed(V)
    x = -torch.rand(6, V, generator=g, device="cuda") - 1
    at = torch.randint(0, V, (6, 60), generator=g, device="cuda")
    x.scatter_(1, at, torch.where(torch.rand(6, 60, generator=g, device="cuda") < 0.5, -0.0, 0.0))
    x[0, :2] = torch.tensor([-0.0, 0.0])
    x[1] = torch.where(torch.rand(V, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    x = x.to(dtype)
    for top in (1, min(V, 5), min(V, 32)):
        r = token_logprobs(x, None, top)
        assert torch.equal(r.top_ids.long(), best(x, top))
        assert torch.equal(r.top_logprobs[0, 0], token_logprobs(x[:1] + 0.0, None, 1).top_logprobs[0, 0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [8, 200, 5000, 40000])
def test_rows_that_begin_with_nan(dtype, n):
    """Lanes whose first values are all NaN: the alternatives are those of the other values."""
    V = 60000
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.randn(5, V, generator=g, device="cuda")
    x[0, :n] = torch.nan
    x[1, torch.randperm(V, generator=g, device="cuda")[:n]] = torch.nan
    x[2, :n] = torch.nan
    x[2, n:] = x[2, n:].round()
    for t in range(n // 256 + 1):  # 8 values of every 256
        x[3, 256 * t:256 * t + 8] = torch.nan
    x[4] = torch.nan
    x[4, -3:] = torch.tensor([1.0, 2.0, 1.0])
    x = x.to(dtype)
    for top in (1, 7, 32):
        r = token_logprobs(x, None, top)
        want = best(x, top)
        want[4, 3:] = -1
        assert torch.equal(r.top_ids.long(), want), [int((a != b).sum()) for a, b in zip(r.top_ids.long(), want)]
        assert r.entropy.isnan().all()
