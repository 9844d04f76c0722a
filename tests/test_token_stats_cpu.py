"""Refusals of the token statistics' entry points without a GPU: the wrappers'
checks on CPU tensors and the C entries' host checks."""
import pytest
import torch

from chessdecoder_b200 import _lib
from chessdecoder_b200 import kernels as K

F32, I32 = torch.float32, torch.int32


def _z(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kw,why", [
    (dict(logits=_z(3, 10, dtype=torch.float16)), "logits"), (dict(logits=_z(10, 3).t()), "logits"),
    (dict(logits=_z(3, 0)), "ncls"), (dict(ncls=11), "ncls"), (dict(ncls=0), "ncls"),
    (dict(logits=_z(1, 10).expand(3, 10)), "overlap"), (dict(target=_z(3, dtype=torch.int64)), "target32"),
    (dict(target=_z(2, dtype=I32)), "target32"), (dict(lp=_z(3, dtype=torch.float64)), "lp"),
    (dict(entropy=_z(2)), "entropy"), (dict(lse=_z(6)[::2]), "lse"), (dict(top_ids=_z(3, 2, dtype=I32)), "together"),
    (dict(top_ids=_z(3, 11, dtype=I32), top_lp=_z(3, 11)), "k <="),
    (dict(logits=_z(3, 50), top_ids=_z(3, 33, dtype=I32), top_lp=_z(3, 33)), "k <="),
    (dict(top_ids=_z(3, 2, dtype=I32), top_lp=_z(3, 3)), "k <="),
    (dict(top_ids=_z(3, 2, dtype=torch.int64), top_lp=_z(3, 2)), "k <="), (dict(), "need CUDA tensors"),
])
def test_forward_refuses(kw, why):
    a = dict(logits=_z(3, 10), target=_z(3, dtype=I32), lp=_z(3))
    a.update(kw)
    with pytest.raises(RuntimeError, match=why):
        K.token_logprobs(a.pop("logits"), a.pop("target"), a.pop("lp"), **a)


@pytest.mark.parametrize("kw,why", [
    (dict(entropy=None), "needs the forward's entropy"), (dict(dlogits=_z(3, 10, dtype=torch.bfloat16)), "dlogits"),
    (dict(dlogits=_z(3, 9)), "dlogits"), (dict(dlogits=_z(1, 10).expand(3, 10)), "overlap"), (dict(dlp=_z(4)), "dlp"),
    (dict(lse=_z(3, dtype=torch.float64)), "lse"), (dict(), "need CUDA tensors"),
])
def test_backward_refuses(kw, why):
    a = dict(lse=_z(3), entropy=_z(3), dlp=_z(3), dent=_z(3), dlogits=_z(3, 10))
    a.update(kw)
    with pytest.raises(RuntimeError, match=why):
        K.token_logprobs_bwd(_z(3, 10), _z(3, dtype=I32), a["lse"], a["entropy"], a["dlp"], a["dent"], a["dlogits"])


def test_c_entries_refuse():
    """The addresses are never followed: the host refuses before it launches."""
    lib = _lib.load()
    f = lambda x=64, dt=0, ldl=10, R=3, V=10, t=64, lp=64, ids=None, top=None, k=0: lib.cdk_token_logprobs(  # noqa: E731
        x, dt, ldl, R, V, t, lp, None, None, ids, top, k, None)
    assert f(R=0) == 0 and f(x=None) == -1 and f(t=None) == -1 and f(lp=None) == -1 and f(R=-1) == -1
    assert f(dt=2) == -2 and f(V=0) == -3 and f(V=11) == -3 and f(V=2 ** 31, ldl=2 ** 31) == -3 and f(x=66) == -4
    assert f(ids=64) == -5 and f(ids=64, top=64, k=33) == -6 and f(ids=64, top=64, k=11) == -6
    b = lambda x=64, dt=0, ldl=10, R=3, V=10, lse=64, ent=64, h=64, dx=128, ldd=10: lib.cdk_token_logprobs_bwd(  # noqa: E731
        x, dt, ldl, R, V, 64, lse, ent, 64, h, dx, ldd, None)
    assert b(R=0) == 0 and b(lse=None) == -1 and b(dx=None) == -1 and b(dt=3) == -2 and b(ldd=9) == -3
    assert b(dx=130) == -4 and b(ent=None) == -5 and b(dx=64, ldd=12) == -6


def test_op_under_fake_tensors():
    """cdk::token_logprobs has a fake implementation: shapes, types and what carries a gradient."""
    import chessdecoder_b200.ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 4, 50, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        t = torch.empty(3, 4, device="cuda", dtype=torch.long)
        lp, ent, lse, ids, top = torch.ops.cdk.token_logprobs(x, t, 5)
        assert lp.shape == ent.shape == lse.shape == (3, 4) and ids.shape == top.shape == (3, 4, 5)
        assert (lp.dtype, ids.dtype, top.dtype) == (F32, I32, F32)
        assert lp.requires_grad and ent.requires_grad and not (lse.requires_grad or top.requires_grad)
        dx = torch.ops.cdk.token_logprobs_backward(x, t, lse, ent, lp, None)
        assert dx.shape == x.shape and dx.dtype == x.dtype
