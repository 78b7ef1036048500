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
