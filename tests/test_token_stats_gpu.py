"""Token statistics on the GPU (csrc/token_stats.cu): log-probability of given
tokens, entropy, best alternatives, and the gradient, against 64 bits.

Tolerances.  u = 2^-24.  With x exact, z = x - m is off by u |z|, its exponential
by (|z| + 4) 2 u of itself, a sum of V terms in at least 32 partial sums by
(V / 32 + 64) u of the sum of the magnitudes.  So with zbar = sum e |z| / sum e,
  ds = (2 zbar + 8 + V / 32 + 64) u                relative, of s and of t
  lp: ds + 4 u (|x| + |m| + |log s| + 1)           absolute
  entropy: 2 ds (1 + zbar) + 4 u (1 + log V)
A gradient inherits d(log p) = lp's bound as the relative error of p, and is
rounded once to the logits' type (2^-8 for bf16, 2^-24 for fp32)."""
import math

import pytest
import torch

from chessdecoder_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _no_device_error():
    K.get_error()
    yield
    assert K.get_error() == 0


def reference(x, t, dlp=None, dent=None):
    """In 64 bits: lp, entropy, logp, the bounds of lp and entropy, and the gradient with its bound."""
    x = x.cpu().double()
    R, V = x.shape
    t = t.cpu().long()
    logp = torch.log_softmax(x, 1)
    p = logp.exp()
    fin = x.masked_fill(x == -math.inf, 0.0)
    m = x.amax(1)
    z = torch.where(p > 0, (x - m[:, None]).abs(), 0.0)
    zbar = (p * z).sum(1)
    ds = (2 * zbar + 8 + V / 32 + 64) * U
    lse = torch.logsumexp(x, 1)
    dlogp = ds[:, None] + 4 * U * (fin.abs() + m.abs()[:, None] + (lse - m).abs()[:, None] + 1)
    ent = -torch.where(p > 0, p * logp, 0.0).sum(1)
    dent_tol = 2 * ds * (1 + zbar) + 4 * U * (1 + math.log(V))
    given = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1)[:, None]
    lp = torch.where(given, logp.gather(1, at)[:, 0], 0.0)
    out = dict(lp=lp, lp_tol=dlogp.gather(1, at)[:, 0], ent=ent, ent_tol=dent_tol, logp=logp, logp_tol=dlogp, lse=lse,
               lse_tol=ds + 4 * U * (m.abs() + lse.abs()))
    if dlp is not None or dent is not None:
        g = torch.zeros(R, 1).double() if dlp is None else (dlp.cpu().double() * given)[:, None]
        h = torch.zeros(R, 1).double() if dent is None else dent.cpu().double()[:, None]
        hit = torch.zeros(R, V).double().scatter_(1, at, given.double()[:, None])
        slog = torch.where(p > 0, logp, 0.0)
        out["dx"] = g * (hit - p) - h * p * (slog + ent[:, None])
        out["dx_tol"] = (g.abs() * p + h.abs() * p * (slog + ent[:, None]).abs()) * (dlogp + 8 * U) \
            + h.abs() * p * (dlogp + dent_tol[:, None] + 4 * U * (slog.abs() + ent[:, None])) + 4 * U * g.abs() * hit
    return out


def alternatives(x, k):
    return torch.sort(x.cpu().float(), dim=1, descending=True, stable=True)[1][:, :k]


def run(x, t, k=0, dlp=None, dent=None, ncls=None, check=True):
    R, V = x.shape[0], x.shape[1] if ncls is None else ncls
    lp, ent, lse = (torch.full((R,), 77.0, device=DEV) for _ in range(3))
    ids = torch.full((R, k), -9, dtype=torch.int32, device=DEV)
    top = torch.full((R, k), 77.0, device=DEV)
    K.token_logprobs(x, t, lp, entropy=ent, lse=lse, top_ids=ids, top_lp=top, ncls=ncls)
    dx = None
    if dlp is not None or dent is not None:
        dx = torch.full_like(x, 77.0)
        K.token_logprobs_bwd(x, t, lse, ent, dlp, dent, dx, ncls=ncls)
    if check:
        want = reference(x[:, :V], t, dlp, dent)

        def near(got, ref, tol, what):
            got, both = got.cpu().double(), torch.isfinite(ref)
            assert torch.equal(got[~both], ref[~both]), what
            bad = ((got - ref).abs() > tol)[both]
            assert not bad.any(), (what, ((got - ref).abs() / tol)[both].max().item())
        near(lp, want["lp"], want["lp_tol"], "lp")
        near(ent, want["ent"], want["ent_tol"], "entropy")
        near(lse, want["lse"], want["lse_tol"], "lse")
        if k:
            order = alternatives(x[:, :V], k)
            assert torch.equal(ids.cpu().long(), order)
            near(top, want["logp"].gather(1, order), want["logp_tol"].gather(1, order), "top_lp")
        if dx is not None:
            half = 2.0 ** -8 if x.dtype == torch.bfloat16 else U
            low = 2.0 ** -134 if x.dtype == torch.bfloat16 else 2.0 ** -126  # below the normal range
            near(dx[:, :V], want["dx"], want["dx_tol"] + half * (want["dx"].abs() + want["dx_tol"]) + low, "dx")
            assert (dx[:, V:] == 77).all()
    return lp, ent, lse, ids, top, dx


def inputs(R, V, bf16=False, masked=0.0, seed=0, pitch=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V + pitch, generator=g) * spread
    t = torch.randint(0, V, (R,), generator=g)
    if masked:
        gone = torch.rand(R, V + pitch, generator=g) < masked
        gone.scatter_(1, t[:, None], False)
        x.masked_fill_(gone, -math.inf)
    t[torch.rand(R, generator=g) < 0.2] = -100
    x = (x.to(torch.bfloat16) if bf16 else x).to(DEV)
    dlp, dent = torch.randn(2, R, generator=g).to(DEV)
    return x[:, :V] if pitch else x, t.to(torch.int32).to(DEV), dlp.contiguous(), dent.contiguous()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [1, 2, 3, 31, 32, 33, 41, 100, 255, 257, 1000, 1924, 2049, 4097, 8191, 32003, 131071])
def test_sizes(V, bf16):
    R = 5 if V > 5000 else 37
    x, t, dlp, dent = inputs(R, V, bf16, seed=V)
    run(x, t, min(5, V), dlp, dent)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("k", [0, 1, 2, 7, 20, 31, 32])
@pytest.mark.parametrize("V", [32, 1924, 20001])
def test_alternatives(V, k, bf16):
    x, t, _, _ = inputs(9, V, bf16, masked=0.5, seed=k)
    run(x, t, k)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [160, 480, 1924, 3934])
def test_as_many_alternatives_as_lanes(V, bf16):
    """Many rows of a warp each: the least of its lanes' maxima admits more candidates than there is room for in some."""
    x, t, _, _ = inputs(2400, V, bf16, seed=V)
    x[::3] = x[::3].sort(dim=1, descending=True)[0]
    x[1::3] = 0.25
    run(x, t, 32)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("R,V", [(2400, 1029), (2400, 3999), (2400, 8003), (2400, 16001), (600, 20001), (600, 33001)])
def test_many_long_rows(R, V, bf16):
    """A warp's rows in one part and more, a block's with fewer and more threads, equal and masked ones among them."""
    x, t, _, _ = inputs(R, V, bf16, seed=V, pitch=1)
    x[7::11] = -math.inf
    x[7::11, V // 3] = 2.0
    x[8::11] = -1e4
    x[9::11, :40] = 30.0
    order = x.float().sort(dim=1, descending=True, stable=True)[1]
    want = reference(x[:33], t[:33])
    for k in (1, 12, 13, 32):
        lp, ent, lse, ids, top, _ = run(x, t, k, check=False)
        assert torch.equal(ids.long(), order[:, :k])
        assert ((lp[:33].cpu() - want["lp"]).abs() <= want["lp_tol"])[want["lp"] > -math.inf].all()
        assert ((ent[:33].cpu() - want["ent"]).abs() <= want["ent_tol"]).all()
        assert ((lse[:33].cpu() - want["lse"]).abs() <= want["lse_tol"]).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [41, 1924, 20001, 131071])
def test_alternatives_of_masked_and_equal_rows(V, bf16):
    """Fewer logits than alternatives above the mask (-inf, the type's lowest, the lowest fp32), and rows of few values."""
    dtype = torch.bfloat16 if bf16 else torch.float32
    masks = [-math.inf, torch.finfo(dtype).min, -1e4]
    x, t, _, _ = inputs(12, V, bf16, seed=V, pitch=3)
    g = torch.Generator().manual_seed(V)
    for r in range(9):
        few = torch.randperm(V, generator=g)[:(0, 3, 31)[r // 3]].to(DEV)
        keep = x[r, few].clone()
        x[r] = masks[r % 3]
        x[r, few] = keep
    x[0, V // 2] = 1.0  # (a row of -inf alone has its test)
    x[9] = 0.0
    x[10] = torch.randint(0, 2, (V,), generator=g).to(DEV)
    x[11] = torch.arange(V, device=DEV) // 7 % 50
    for k in (1, 5, 20, 32):
        lp, _, lse, ids, top, _ = run(x, t, k, check=False)
        assert torch.equal(ids.cpu().long(), alternatives(x, k))
        want = torch.log_softmax(x.cpu().double(), 1).gather(1, ids.cpu().long())
        # 1e-3: ds <= (2 zbar + 72 + 131071 / 32) u < 3e-4 (zbar < 50), the other terms 4 u * 200;
        # x - m is 0 in the rows of one value.
        some = want > -1e4  # of the others the fp32 differences are as large as the mask
        assert ((top.cpu() - want).abs() <= 1e-3)[some].all() and (top.cpu()[~some] <= -9e3).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("descending", [False, True])
@pytest.mark.parametrize("threads", [1, 3, 40])
def test_best_logits_in_few_threads(threads, descending, bf16):
    """The best are all in every 256th vector from a few on, in either order."""
    V, n = 131072, 8 if bf16 else 4
    x, t, _, _ = inputs(2, V, bf16, seed=threads)
    part = x.view(2, V // (256 * n), 256, n)[:, :, :threads]
    rise = torch.arange(part[0].numel(), device=DEV).view(part[0].shape) * 2.0 ** -6 + 20.0
    part.copy_(rise.flip(0) if descending else rise)
    run(x, t, 32)
    run(x, t, 3)


@pytest.mark.parametrize("R", [1, 2, 147, 149, 1000, 5000])
def test_rows(R):
    x, t, dlp, dent = inputs(R, 131, seed=R)
    run(x, t, 3, dlp, dent)
    if R < 200:
        x, t, dlp, dent = inputs(R, 30011, True, seed=R)
        run(x, t, 3, dlp, dent)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V,pitch", [(41, 3), (1924, 4), (1923, 1), (9001, 7), (100, 28)])
def test_pitches_and_column_limits(V, pitch, bf16):
    """Rows with a pitch (aligned and not), a first column that is not aligned, and ncls below the columns."""
    x, t, dlp, dent = inputs(11, V, bf16, pitch=pitch)
    run(x, t, 4, dlp, dent)
    x, t, dlp, dent = inputs(11, V + pitch, bf16, seed=1)
    run(x[:, 1:], (t - 1).clamp(max=V - 1), 4, dlp, dent, ncls=V - 1)


@pytest.mark.parametrize("V", [40, 1924, 20000])
def test_order_of_equal_values(V):
    """Ties go to the lowest index: all equal, two values, zeros of both signs, sorted both ways."""
    rows = [torch.zeros(V), torch.arange(V) % 2.0, torch.where(torch.arange(V) % 3 == 0, -0.0, 0.0),
            torch.arange(V, dtype=torch.float32) / 64, -torch.arange(V, dtype=torch.float32) / 64,
            torch.full((V,), -3.0e38), (torch.arange(V) // 7 % 5).float()]
    x = torch.stack(rows).to(DEV)
    t = torch.zeros(len(rows), dtype=torch.int32, device=DEV)
    run(x, t, 32)
    run(x.to(torch.bfloat16), t, 20)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V,threads", [(1924, 32), (131071, 256), (70003, 256)])
def test_best_logits_crowded_into_few_columns(V, threads, bf16):
    """The best classes all lie in a few strided groups of columns (16-byte pieces, every
    32nd or 256th of them), hundreds to thousands of them: more than a selection by
    per-thread maxima keeps."""
    n = 8 if bf16 else 4
    x = torch.rand(3, V, generator=torch.Generator().manual_seed(V))
    crowd = (torch.arange(V) // n) % threads < 20
    x[:, crowd] += 5
    x[2, crowd] = 7.0
    x = (x.to(torch.bfloat16) if bf16 else x).to(DEV)
    t = torch.zeros(3, dtype=torch.int32, device=DEV)
    for k in (5, 21, 32):
        run(x, t, k)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [33, 1924, 40001])
def test_masked_rows(V, bf16):
    """Almost everything -inf, the type's lowest value, one legal class, none, infinities and NaN."""
    dt = torch.bfloat16 if bf16 else torch.float32
    x = torch.full((6, V), -math.inf)
    x[0, V - 1] = 2.0
    x[1, ::7] = torch.linspace(-3, 3, len(x[1, ::7]))
    x[2] = torch.finfo(dt).min
    x[2, 5] = 0.0
    t = torch.tensor([V - 1, 7, 5, 4, 4, 4], dtype=torch.int32, device=DEV)
    dlp, dent = torch.ones(6, device=DEV), torch.ones(6, device=DEV)
    x = x.to(dt)
    run(x[:3].to(DEV), t[:3], 5, dlp[:3], dent[:3])
    x[4, 3], x[4, 4] = math.inf, 1.0
    x[5] = 0.0
    x[5, 8], x[5, 9] = math.nan, math.inf
    lp, ent, lse, ids, top, dx = run(x.to(DEV), t, 3, dlp, dent, check=False)
    # nothing legal
    assert lp[3] == -math.inf and lse[3] == -math.inf and ent[3] == 0 and (dx[3] == 0).all()
    assert ids[3].tolist() == [0, 1, 2] and (top[3] == -math.inf).all()
    for r in (4, 5):
        assert lp[r].isnan() and ent[r].isnan() and lse[r].isnan() and top[r].isnan().all()
    assert ids[4].tolist() == [3, 4, 0] and ids[5].tolist() == [8, 9, 0]
    # a target that is masked
    lp, _, _, _, _, dx = run(x[1:2].to(DEV), torch.tensor([1], dtype=torch.int32, device=DEV), 0, dlp[:1], dent[:1],
                             check=False)
    assert lp[0] == -math.inf and dx.isfinite().all() and dx[0, 1] == 1


@pytest.mark.parametrize("target", [-1, -100, 2 ** 31 - 1, -2 ** 31, 50])
def test_targets_outside_the_classes(target):
    x, _, dlp, dent = inputs(4, 50)
    run(x, torch.full((4,), target, dtype=torch.int32, device=DEV), 2, dlp, dent)


def test_outputs_are_optional_and_gradients_may_overwrite():
    x, t, dlp, dent = inputs(40, 777)
    lp, ent, lse, _, _, dx = run(x, t, 0, dlp, dent)
    lp2 = torch.empty_like(lp)
    K.token_logprobs(x, t, lp2)
    assert torch.equal(lp, lp2)
    run(x, t, 0, dlp, None)
    run(x, t, 0, None, dent)
    only = torch.empty_like(x)
    K.token_logprobs_bwd(x, t, lse, None, dlp, None, only)
    want = reference(x, t, dlp, None)
    assert ((only.cpu().double() - want["dx"]).abs() <= want["dx_tol"] + U * want["dx"].abs() + 2.0 ** -126).all()
    K.token_logprobs_bwd(x, t, lse, ent, dlp, dent, x)
    assert torch.equal(x, dx)


@pytest.mark.parametrize("bf16", [False, True])
def test_gradient_against_differences(bf16):
    """sum(dlp lp + dent H) along a direction: central differences of the 64-bit
    definition (step 1e-5: off by about 1e-9) and of the kernel's own forward
    (step 2^-4: its truncation is h^2 / 6 of the third derivative, which is below
    6 (|dlp| + 4 |dent| log V) per row for a direction of unit length)."""
    R, V, h = 6, 500, 2.0 ** -4
    x, t, dlp, dent = inputs(R, V, bf16, spread=1.0)
    dx = run(x, t, 0, dlp, dent)[5].cpu().double()
    d = torch.randn(R, V, generator=torch.Generator().manual_seed(5)).double()
    d /= d.norm(dim=1, keepdim=True)
    x64 = x.cpu().double()

    def f(y):
        r = reference(y, t)
        return dlp.cpu().double() * r["lp"] + dent.cpu().double() * r["ent"]
    num = (f(x64 + 1e-5 * d) - f(x64 - 1e-5 * d)) / 2e-5
    want = reference(x, t, dlp, dent)
    half = 2.0 ** -8 if bf16 else U
    tol = ((want["dx_tol"] + half * want["dx"].abs()) * d.abs()).sum(1) + 1e-8
    assert ((dx * d).sum(1) - num).abs().le(tol).all()
    if not bf16:
        ys = [(x64 + s * h * d).float().to(DEV) for s in (1, -1)]
        out = [run(y, t)[:2] for y in ys]
        fs = [(dlp * lp + dent * e).cpu().double() for lp, e in out]
        size = dlp.abs().cpu().double() + 4 * dent.abs().cpu().double() * math.log(V)
        assert (((fs[0] - fs[1]) / (2 * h) - (dx * d).sum(1)).abs() <= h * h * size + 40 * V / 32 * U * size / h).all()


def test_streams_and_graphs():
    x, t, dlp, dent = inputs(64, 1924)
    lp, ent, lse = (torch.zeros(64, device=DEV) for _ in range(3))
    ids, top = torch.zeros(64, 5, dtype=torch.int32, device=DEV), torch.zeros(64, 5, device=DEV)
    dx = torch.zeros_like(x)

    def step():
        K.token_logprobs(x, t, lp, entropy=ent, lse=lse, top_ids=ids, top_lp=top)
        K.token_logprobs_bwd(x, t, lse, ent, dlp, dent, dx)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for seed in (3, 4):
        y, t2, _, _ = inputs(64, 1924, seed=seed)
        x.copy_(y)
        t.copy_(t2)
        g.replay()
        a = run(x, t, 5, dlp, dent)
        for got, want in zip((lp, ent, lse, ids, top, dx), a):
            assert torch.equal(got, want)
