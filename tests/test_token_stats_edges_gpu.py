"""Token statistics at the edges of what they promise (csrc/token_stats.cu): NaN
among the alternatives, and the gradient of rows far from zero."""
import math

import pytest
import torch

from chessdecoder_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error():
    K.get_error()
    yield
    assert K.get_error() == 0


def best(x, k):
    """The k best classes: NaN above every number, equal values in order of their index."""
    x = x.cpu().float()
    rank = torch.where(x.isnan(), math.inf, torch.where(x == math.inf, torch.finfo(x.dtype).max, x)).double()
    rank = torch.where(x == torch.finfo(x.dtype).max, torch.finfo(x.dtype).max * 0.5, rank)  # below +inf
    return torch.sort(rank, dim=1, descending=True, stable=True)[1][:, :k]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [1, 2, 5, 32, 41, 1924, 20001, 131071])
def test_nan_comes_first_wherever_it_is(V, bf16):
    """In class 0, in the last, in several, everywhere; every class asked where there are few."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(6, V, generator=g)
    x[0, 0] = math.nan
    x[1, V - 1] = math.nan
    x[2, ::3] = math.nan
    x[3] = math.nan
    x[4, 0], x[4, V // 2] = -math.nan, math.inf
    x[5, V // 2:] = math.nan
    x = (x.to(torch.bfloat16) if bf16 else x).to(DEV)
    t = torch.zeros(6, dtype=torch.int32, device=DEV)
    for k in {1, min(V, 3), min(V, 32)}:
        lp, ent, lse = (torch.zeros(6, device=DEV) for _ in range(3))
        ids = torch.full((6, k), -9, dtype=torch.int32, device=DEV)
        top = torch.zeros(6, k, device=DEV)
        K.token_logprobs(x, t, lp, entropy=ent, lse=lse, top_ids=ids, top_lp=top)
        assert torch.equal(ids.cpu().long(), best(x, k)), (ids.cpu(), best(x, k))
        assert top.isnan().all() and lp.isnan().all() and ent.isnan().all() and lse.isnan().all()
