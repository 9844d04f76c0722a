"""Arguments of the token statistics that are refused or converted, without a GPU."""
import pytest
import torch

from chessdecoder_b200 import _lib
from chessdecoder_b200 import kernels as K
from chessdecoder_b200.ops import _stat_rows


def _top(rows, k, dtype, kind):
    if kind == "spread":  # a step between the columns
        return torch.zeros(rows, 2 * k, dtype=dtype)[:, ::2]
    if kind == "tail":  # the last of them at the end of the storage
        return torch.zeros(rows, 3 * k, dtype=dtype)[:, 2::3]
    return torch.zeros(k, rows + 1, dtype=dtype).t()[:rows]


@pytest.mark.parametrize("rows,k,kind", [(r, k, kind) for r, k in ((1, 2), (1, 5), (3, 2), (3, 1))
                                         for kind in ("spread", "tail", "turned") if k > 1 or kind != "turned"])
@pytest.mark.parametrize("which", ["top_ids", "top_lp"])
def test_alternatives_that_are_not_contiguous_are_refused(which, kind, rows, k):
    """One row too: the kernel writes k neighbours, which a view with a step does not own."""
    dtypes = dict(top_ids=torch.int32, top_lp=torch.float32)
    kw = {n: torch.zeros(rows, k, dtype=d) for n, d in dtypes.items()}
    kw[which] = _top(rows, k, dtypes[which], kind)
    with pytest.raises(RuntimeError, match="contiguous"):
        K.token_logprobs(torch.zeros(rows, 10), torch.zeros(rows, dtype=torch.int32), torch.zeros(rows), **kw)


@pytest.mark.parametrize("rows,k", [(1, 1), (1, 4), (3, 1), (3, 4), (3, 0)])
def test_contiguous_alternatives_are_taken(rows, k):
    """Views of one row or column whose strides do not matter pass the check (and stop at the device's)."""
    ids, top = torch.zeros(rows, 9, dtype=torch.int32), torch.zeros(rows, 9)
    pairs = [(torch.zeros(rows, k, dtype=torch.int32), torch.zeros(rows, k))]
    if rows == 1:
        pairs.append((ids[:, 2:2 + k], top[:, 2:2 + k]))
    for i, t in pairs:
        with pytest.raises(RuntimeError, match="need CUDA tensors"):
            K.token_logprobs(torch.zeros(rows, 10), torch.zeros(rows, dtype=torch.int32), torch.zeros(rows), top_ids=i,
                             top_lp=t)


@pytest.mark.parametrize("V", [100, 200, 1924, 70000])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8, torch.bool])
def test_targets_of_every_integer_type_keep_their_meaning(dtype, V):
    """Targets inside the classes stay, those outside stay outside, whatever the type holds."""
    low, high = (0, 1) if dtype == torch.bool else (torch.iinfo(dtype).min, torch.iinfo(dtype).max)
    given = [v for v in (0, 1, 99, 100, 127, 156, 200, 250, 255, 1923, 32767, 69999, 2 ** 31 - 1, 2 ** 32 + 5, 2 ** 40,
                         -1, -100, -128, -2 ** 31, -2 ** 40) if low <= v <= high]
    t = torch.tensor(given, dtype=dtype)
    got = _stat_rows(torch.zeros(len(given), V), t)[1]
    assert got.dtype == torch.int32
    for v, g in zip(given, got.tolist()):
        assert g == v if 0 <= v < V else not 0 <= g < V, (v, g)
    wide = torch.stack([t, t], 1)  # every second one of a wider tensor
    assert torch.equal(_stat_rows(torch.zeros(len(given), V), wide[:, 0])[1], got)
    assert _stat_rows(torch.zeros(len(given), V), wide[:, 0])[1].is_contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.complex64, torch.uint16, torch.uint64])
def test_targets_of_other_types_are_refused(dtype):
    with pytest.raises(ValueError, match="integer targets"):
        _stat_rows(torch.zeros(3, 10), torch.zeros(3, dtype=dtype))


def test_the_second_part_of_the_sum_is_checked_like_the_first():
    x, t, f = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    for bad in (torch.zeros(2), torch.zeros(3, dtype=torch.float64), torch.zeros(6)[::2]):
        with pytest.raises(RuntimeError, match="lse_low"):
            K.token_logprobs(x, t, f, lse_low=bad)
        with pytest.raises(RuntimeError, match="lse_low"):
            K.token_logprobs_bwd(x, t, f, f, f, f, x, lse_low=bad)
    lib = _lib.load()  # the addresses are never followed: the host refuses before it launches
    f = lambda x=64, V=10, R=3: lib.cdk_token_logprobs_split(  # noqa: E731
        x, 0, 10, R, V, 64, 64, None, None, 64, None, None, 0, None)
    b = lambda dx=128, lse=64, R=3: lib.cdk_token_logprobs_bwd_split(  # noqa: E731
        64, 0, 10, R, 10, 64, lse, 64, 64, 64, 64, dx, 10, None)
    assert f(x=None) == -1 and f(V=11) == -3 and f(R=0) == 0
    assert b(dx=None) == -1 and b(lse=None) == -1 and b(dx=130) == -4 and b(R=0) == 0


def test_op_has_five_outputs_and_is_the_forward_with_both_parts():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 50, device="cuda", requires_grad=True)
        out = torch.ops.cdk.token_logprobs(x, torch.empty(3, dtype=torch.long, device="cuda"), 2)
        both = torch.ops.cdk.token_logprobs_forward(x, torch.empty(3, dtype=torch.long, device="cuda"), 2)
        assert len(out) == 5 and len(both) == 6
        assert [o.requires_grad for o in both] == [True, True, False, False, False, False]
        dx = torch.ops.cdk.token_logprobs_backward(x, torch.empty(3, dtype=torch.long, device="cuda"), both[2], both[1],
                                                   both[0], None, both[3])
        assert dx.shape == x.shape
