"""Token statistics at the edges of what they promise (csrc/token_stats.cu): NaN
among the alternatives, and the gradient of rows far from zero."""
import math

import pytest
import torch

from chessdecoder_b200 import kernels as K

from test_token_stats_gpu import U, reference

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


def grid(R, V, seed):
    """fp32 logits on a grid of 2^-6, so that a shift by a whole number is exact."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, V, generator=g) * 3 * 64).round() / 64
    t = torch.randint(0, V, (R,), generator=g)
    t[1] = -100
    dlp, dent = torch.randn(2, R, generator=g)
    return x, t.to(torch.int32).to(DEV), dlp.to(DEV), dent.to(DEV)


@pytest.mark.parametrize("shift", [0, 100, -1000, 10000, 100000])
@pytest.mark.parametrize("V", [41, 1924, 20001])
def test_gradient_of_rows_far_from_zero(V, shift):
    """A constant added to a row changes no probability: the gradient keeps the bound of
    the row whose maximum is 0 (tests/test_token_stats_gpu.py; log s and x - m are what it
    is computed from), through the op and through the kernels, and sums to as little."""
    import chessdecoder_b200.ops  # noqa: F401
    x, t, dlp, dent = grid(8, V, V)
    want = reference(x - x.amax(1, keepdim=True), t, dlp, dent)
    x = (x + shift).to(DEV)
    lp, ent, lse, low = (torch.empty(8, device=DEV) for _ in range(4))
    K.token_logprobs(x, t, lp, entropy=ent, lse=lse, lse_low=low)
    dx = torch.empty_like(x)
    K.token_logprobs_bwd(x, t, lse, ent, dlp, dent, dx, lse_low=low)
    tol = want["dx_tol"] + U * (want["dx"].abs() + want["dx_tol"]) + 2.0 ** -126
    off = (dx.cpu().double() - want["dx"]).abs()
    assert (off <= tol).all(), (off / tol).max()
    assert (dx.cpu().double().sum(1).abs() <= tol.sum(1)).all()
    exact = x.cpu().double().logsumexp(1)
    assert ((lse.cpu().double() + low.cpu().double() - exact).abs() <= want["lse_tol"]).all()
    assert torch.equal(lse, (lse.double() + low.double()).float())
    y = x.clone().requires_grad_(True)
    a, b, c, _, _ = torch.ops.cdk.token_logprobs(y, t.long(), 0)
    assert torch.equal(a, lp) and torch.equal(b, ent) and torch.equal(c, lse)
    torch.autograd.backward([a, b], [dlp, dent])
    assert torch.equal(y.grad, dx)


def test_lse_low_of_rows_without_a_sum():
    """Nothing above -inf: 0 beside -inf, and a gradient of zeros; NaN and +inf: NaN."""
    x = torch.full((3, 50), -math.inf, device=DEV)
    x[1, 7], x[2, 7] = math.nan, math.inf
    t = torch.zeros(3, dtype=torch.int32, device=DEV)
    lp, ent, lse, low = (torch.full((3,), 5.0, device=DEV) for _ in range(4))
    K.token_logprobs(x, t, lp, entropy=ent, lse=lse, lse_low=low)
    assert lse[0] == -math.inf and low[0] == 0 and lse[1:].isnan().all() and low[1:].isnan().all()
    dx = torch.full_like(x, 5.0)
    K.token_logprobs_bwd(x, t, lse, ent, torch.ones(3, device=DEV), torch.ones(3, device=DEV), dx, lse_low=low)
    assert (dx[0] == 0).all() and dx[1:].isnan().all()
    one = torch.empty(3, device=DEV)
    K.token_logprobs(x, t, lp, lse_low=one)  # alone
    assert torch.equal(one.nan_to_num(9), low.nan_to_num(9))
