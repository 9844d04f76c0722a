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


# Scores with one product each: exact but for the scale's rounding, its product and the
# difference to the reference, 2 * 3 * 2^-24 |s| + 2^-24 |s - m| with |s| <= 8 and |s - m| <= 24
# in base 2, so 2^-18 of a weight at most; the exponential 2^-22; sums of 64 terms 2^-18; a
# weight in two bf16 2^-17 (in two fp16 2^-22).
WEIGHTS = {fp8: 2.0 ** -18 + 2.0 ** -22 + 2.0 ** -18 + 2.0 ** (-22 if fp8 else -17) for fp8 in (False, True)}


def held_to_the_weights(got, s, v, fp8):
    """got [H, 64] against softmax(s [H, n]) @ v with values of magnitude 1: the output's
    own rounding and WEIGHTS.  One rounding of the weights to the products' type is
    outside that somewhere."""
    w = torch.exp(s - s.amax(-1, keepdim=True))
    want = (w @ v.double()) / w.sum(-1, keepdim=True)
    tol = 2.0 ** -8 * want.abs() + WEIGHTS[fp8]
    once = w.float().to(torch.float16 if fp8 else torch.bfloat16).double()
    assert (((once @ v.double()) / w.sum(-1, keepdim=True) - want).abs() > 1.5 * tol).any()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H", [1, 7, 12])
@pytest.mark.parametrize("p", [8, 16, 64])
def test_weights_that_nearly_cancel(p, H, fp8):
    """Values of +-1 whose weighted sum is next to nothing: what the weights lose shows."""
    g = torch.Generator().manual_seed(100 * H + p)
    n = 64
    q, k = torch.zeros(H, D), torch.zeros(n, D)
    q[:, 0] = torch.rand(1, generator=g).add(0.5).to(torch.bfloat16).float()
    k[:, 0] = torch.randint(-16, 17, (n,), generator=g) / 8.0
    s = q[:, :1].double() * k[:, 0].double() * 1.1
    w = torch.softmax(s, -1).mean(0)
    v, left = torch.zeros(n, D), torch.zeros(D, dtype=torch.float64)
    for i, j in enumerate(w.argsort(descending=True).tolist()):  # at random, then against what is left
        side = torch.randint(0, 2, (D,), generator=g) * 2.0 - 1 if i < 12 else torch.where(left > 0, -1.0, 1.0)
        v[j], left = side, left + side.double() * w[j]
    held_to_the_weights(attend(q, k, v, fp8, p=p, scale=1.1), s, v, fp8)


@pytest.mark.parametrize("fp8", [False, True])
def test_many_equal_weights_beside_a_large_one(fp8):
    """Two tiles of one key with weight 1 and 31 with r 2^-5 each, r next to the middle
    between two numbers of the products' type, so that all round the same way."""
    r = 1 + 0.98 * (2.0 ** -11 if fp8 else 2.0 ** -8)
    scale = (5 - math.log2(r)) * math.log(2)
    q, k, v = torch.zeros(1, D), torch.zeros(64, D), -torch.ones(64, D)
    q[0, 0] = 1.0
    k[:, 0] = -1.0
    k[::32, 0], v[::32] = 0.0, 1.0
    held_to_the_weights(attend(q, k, v, fp8, scale=scale), k[:, 0].double()[None] * scale, v, fp8)


@pytest.mark.parametrize("p", [8, 16, 64])
def test_the_smallest_scale(p):
    """Keys at scale byte 0 (2^-127) under queries of 2^122: ordinary scores, products
    of four numbers each (as WEIGHTS has them, to 2^-17 with three more); values at byte 0
    beside others."""
    n = 64
    q, k, v = torch.zeros(2, D), torch.zeros(n, D), torch.ones(n, D)
    q[:, 0] = torch.tensor([2.0 ** 122, -1.5 * 2.0 ** 122])
    k[:, 0] = torch.arange(n) % 9.0 * 8 - 32
    v[1::2] = -1.75
    byte = torch.full((n,), 127)
    byte[::5] = 0
    got = attend(q, k, v, True, p=p, kbyte=0, vbyte=byte)
    w = torch.softmax(q[:, :1].double() * 2.0 ** -127 * k[:, 0].double(), -1)
    seen = v.double() * torch.pow(2.0, byte.double() - 127)[:, None]
    assert ((got - w @ seen).abs() <= 2.0 ** -8 * (w @ seen).abs() + 2.0 ** -16 * (w @ seen.abs())).all()


@pytest.mark.parametrize("which", ["key", "value"])
def test_a_scale_that_is_not_a_number(which):
    """Scale byte 255: the row is NaNs, as in the read-back, and so is what attends to it."""
    n = 70
    byte = torch.full((n,), 127)
    byte[66] = 255
    kw = dict(kbyte=byte) if which == "key" else dict(vbyte=byte)
    assert attend(torch.ones(3, D), torch.ones(n, D), torch.ones(n, D), True, **kw).isnan().all()
    out = torch.zeros(1, 1, 32, D, dtype=torch.bfloat16, device=DEV)
    pool = torch.ones(1, 1, 32, D, device=DEV).to(torch.float8_e4m3fn)
    s = torch.full((1, 1, 32), 127, dtype=torch.uint8, device=DEV)
    s[0, 0, 3], s[0, 0, 4] = 255, 0
    K.paged_gather(pool, pool, torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                   torch.tensor([32], dtype=torch.int32, device=DEV), out, out.clone(), k_scale=s, v_scale=s)
    assert out[0, 0, 3].isnan().all() and (out[0, 0, 4] == 2.0 ** -127).all() and (out[0, 0, 5:] == 1).all()
