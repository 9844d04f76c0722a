"""cdk::token_logprobs (chessdecoder_b200/ops.py) under autograd, and
GRPOStep.score, against 64 bits; tolerances of tests/test_token_stats_gpu.py."""
import pytest
import torch

import chessdecoder_b200.ops  # noqa: F401
from chessdecoder_b200 import kernels as K

from test_token_stats_gpu import U, alternatives, inputs, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def loss_of(lp, ent, c):
    return (lp * c).sum() - 0.3 * ent.mean()


@pytest.mark.parametrize("bf16", [False, True])
def test_gradients_through_the_op(bf16):
    """Shared leading dimensions, padded int64 targets, a loss whose incoming gradients are broadcast."""
    B, S, V = 3, 5, 777
    x, _, c, _ = inputs(B * S, V, bf16)
    g = torch.Generator().manual_seed(3)
    t = torch.randint(0, V, (B, S), generator=g)
    t[0, 0], t[1, 2], t[2, 4] = -100, 2 ** 40, V
    x = x.view(B, S, V).requires_grad_(True)
    c = c.view(B, S)
    lp, ent, lse, ids, top = torch.ops.cdk.token_logprobs(x, t.to(DEV), 4)
    assert not (lse.requires_grad or ids.requires_grad or top.requires_grad) and lp.requires_grad
    loss_of(lp, ent, c).backward()
    assert x.grad.dtype == x.dtype and x.grad.shape == x.shape
    flat = x.detach().view(-1, V)
    dent = torch.full((B * S,), -0.3 / (B * S))
    ref = reference(flat, t.view(-1), c.reshape(-1), dent)
    half = 2.0 ** -8 if bf16 else U
    tol = ref["dx_tol"] + half * (ref["dx"].abs() + ref["dx_tol"]) + 2.0 ** -126 + 4 * U * ref["dx"].abs()
    assert ((x.grad.view(-1, V).cpu().double() - ref["dx"]).abs() <= tol).all()
    assert torch.equal(ids.view(-1, 4).cpu().long(), alternatives(flat, 4))
    # only one of the two outputs used; an expanded gradient
    y = x.detach().clone().requires_grad_(True)
    torch.ops.cdk.token_logprobs(y, t.to(DEV), 0)[1].sum().backward()
    ref = reference(flat, t.view(-1), None, torch.ones(B * S))
    tol = ref["dx_tol"] + half * (ref["dx"].abs() + ref["dx_tol"]) + 2.0 ** -126
    assert ((y.grad.view(-1, V).cpu().double() - ref["dx"]).abs() <= tol).all()


def test_op_on_views_and_empty_batches():
    x, t, _, _ = inputs(12, 300, pitch=20)
    want = torch.ops.cdk.token_logprobs(x.contiguous(), t.long(), 3)
    for got in (torch.ops.cdk.token_logprobs(x, t, 3), torch.ops.cdk.token_logprobs(x.t().contiguous().t(), t.long(), 3)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    same = x[:1].expand(4, 300)
    got = torch.ops.cdk.token_logprobs(same, t[:1].expand(4), 2)
    assert all(torch.equal(a[0], a[3]) for a in got)
    e = torch.zeros(0, 300, device=DEV, requires_grad=True)
    out = torch.ops.cdk.token_logprobs(e, torch.zeros(0, dtype=torch.long, device=DEV), 2)
    assert out[3].shape == (0, 2)
    out[0].sum().backward()
    assert e.grad.shape == e.shape
    with pytest.raises(ValueError):
        torch.ops.cdk.token_logprobs(x.half(), t, 0)
    with pytest.raises(ValueError):
        torch.ops.cdk.token_logprobs(x, t[:3], 0)
    with pytest.raises(RuntimeError, match="k <="):
        torch.ops.cdk.token_logprobs(x, t, 33)


def test_op_forward_and_backward_in_a_graph():
    x, t, c, _ = inputs(64, 1924)
    x.requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            lp, ent, *_ = torch.ops.cdk.token_logprobs(x, t, 0)
            x.grad = torch.autograd.grad(loss_of(lp, ent, c), x)[0]
    torch.cuda.current_stream().wait_stream(s)
    eager = x.grad.clone()
    del lp, ent  # no eager graph of the leaf lives during the capture
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lp, ent, *_ = torch.ops.cdk.token_logprobs(x, t, 0)
        dx = torch.autograd.grad(loss_of(lp, ent, c), x)[0]
    g.replay()
    assert torch.equal(dx, eager)
    with torch.no_grad():
        x.mul_(0.5)
    g.replay()
    lp, ent, *_ = torch.ops.cdk.token_logprobs(x, t, 0)
    assert torch.equal(dx, torch.autograd.grad(loss_of(lp, ent, c), x)[0])


def test_grpo_score():
    """GRPOStep.score: the log-probabilities are those of log_probs (another kernel:
    1e-5, as tests/test_rl_gpu.py holds two passes to), the statistics those of the
    oracle's logits within its tolerance there (5e-2)."""
    from test_rl_gpu import SMALL, _rl_batch

    from chessdecoder_b200.engine import ModelConfig
    from chessdecoder_b200.rl import GRPOStep, prepare_rl_batch
    from oracle.model import OracleChessDecoder
    torch.manual_seed(0)
    oracle = OracleChessDecoder(ModelConfig().vocab_size, **SMALL)
    sd = {k: v.detach().clone() for k, v in oracle.state_dict().items()}
    batch = _rl_batch(2, SMALL["max_seq_len"], seed=9)
    step = GRPOStep(ModelConfig(**SMALL), device=DEV, state_dict=sd)
    rb = prepare_rl_batch(batch, DEV)
    lp, mask = step.log_probs(rb)
    got = step.score(rb, top_k=3)
    assert torch.equal(got["mask"], mask) and torch.allclose(got["log_probs"], lp, atol=1e-5)
    with torch.no_grad():
        h = oracle(batch["input_ids"], mask_type="prefix", block_id=batch["block_id"],
                   wl_positions=batch["wl_positions"], d_positions=batch["d_positions"],
                   **dict(zip(("wl_values", "d_values"), _snapped(oracle, batch))))
    for name, (flat, ids, top) in got["heads"].items():
        logits = getattr(oracle, name)(h.reshape(-1, h.shape[-1])[flat.cpu()]).double()
        logp = torch.log_softmax(logits, 1)
        ent = -(logp.exp() * logp).sum(1)
        assert (got["entropy"].reshape(-1)[flat].cpu() - ent).abs().max() < 5e-2
        assert (top.cpu() - logp.gather(1, ids.cpu().long())).abs().max() < 5e-2
        assert (logp.amax(1) - logp.gather(1, ids[:, :1].cpu().long())[:, 0]).max() < 5e-2
    assert (got["entropy"][~mask] == 0).all()
    assert K.get_error() == 0


def _snapped(model, b):
    """The placeholder values at their nearest bucket centres."""
    out = []
    for v, c, at in ((b["wl_values"], model.wl_bucket_centers, b["wl_positions"]),
                     (b["d_values"], model.d_bucket_centers, b["d_positions"])):
        near = c[(v[..., None] - c).abs().argmin(-1)]
        out.append(torch.where(at, near, 0.0))
    return out
