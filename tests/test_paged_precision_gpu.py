"""Paged attention where its weights' precision and range show: differences
between scores that are one step of fp32, weights that nearly cancel, many small
weights beside a large one, and every scale that a float8_e8m0fnu pool may hold.
Against the plain 64-bit statement of tests/paged_reference.py."""
import math

import pytest
import torch

from chessdecoder_b200 import kernels as K

from paged_reference import D

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error():
    K.get_error()
    yield
    assert K.get_error() == 0


def attend(q, k, v, fp8, p=32, scale=1.0, kbyte=127, vbyte=127):
    """Attention of q [H, 64] over keys and values [n, 64] of one kv head (numbers
    that bf16 or, with the scale bytes, e4m3 hold exactly) in pages of p rows."""
    n, H = k.shape[0], q.shape[0]
    pages = -(-n // p)
    pools, scales = [], []
    for x, byte in ((k, kbyte), (v, vbyte)):
        pool = torch.zeros(pages * p, D)
        pool[:n] = x
        pool = pool.view(pages, 1, p, D)
        kept = pool.to(torch.float8_e4m3fn if fp8 else torch.bfloat16)
        assert torch.equal(kept.float(), pool)
        pools.append(kept.to(DEV))
        b = torch.full((pages, 1, p), 127, dtype=torch.uint8)
        b.view(-1)[:n] = torch.as_tensor(byte, dtype=torch.uint8)
        scales.append(b.view(torch.float8_e8m0fnu).to(DEV) if fp8 else None)
    out = torch.full((1, H * D), float("nan"), dtype=torch.bfloat16, device=DEV)
    K.paged_attn(q.to(torch.bfloat16).reshape(1, -1).to(DEV), *pools,
                 torch.arange(pages, dtype=torch.int32, device=DEV)[None],
                 torch.tensor([n], dtype=torch.int32, device=DEV), out, k_scale=scales[0], v_scale=scales[1], scale=scale)
    return out.cpu().double().view(H, D)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("more", [1, 2, 3])
def test_scores_one_step_apart(more, fp8):
    """Scores of 2^27 + 16 i (base 2), 16 being a step of fp32 there: the weight of
    the key that is a step or more above is 2^16 times the others', neither infinite
    nor lost.  scale = ln 2 makes the base-2 scale 1; products and sums are exact in
    fp32, and the output is rounded once (2^-8), its sums by n * 2^-24 before that.
    (520 keys: a warp has more than one tile of them.)"""
    n = 520
    q, k, v = torch.zeros(1, D), torch.zeros(n, D), torch.ones(n, D)
    q[0, 0], q[0, 1] = 2.0 ** 19, 16.0
    k[:, 0], k[:, 1] = 256.0, 1.0
    k[40, 1], v[40] = 1.0 + more, -2.0
    got = attend(q, k, v, fp8, scale=math.log(2))
    w = 2.0 ** (16 * more)
    want = (n - 1 - 2 * w) / (n - 1 + w)
    assert ((got - want).abs() <= (2.0 ** -8 + n * 2.0 ** -24) * abs(want)).all(), got[0, 0]
