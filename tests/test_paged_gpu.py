"""The paged KV cache on the GPU (csrc/paged.cu) against a plain 64-bit
statement (tests/paged_reference.py).

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value, to e4m3 by
2^-4 of it or 2^-10 of the row's unit, one fp32 operation by 2^-24.
* Append: a rotated value is two products and a sum: 3 * 2^-24 (|u c| + |w s|)
  before its rounding.  Unrotated rows are exact up to the rounding, so their
  codes and scales must be equal.
* Read-back: the values that the codes stand for have at most 4 significant
  bits and the scale is a power of two, so bf16 holds them: equality.
* Attention: with c = the relative error of a weight, |out - ref| <=
  2^-8 |ref| + c * sum p|v|.  A score is 64 products and sums and a scaling
  (68 * 2^-24 * scale * sum|q k|, twice: its own and the maximum's), the
  exponential 2^-20, the running sums n * 2^-24 at worst, and the weight is
  rounded to bf16 (2^-8) for bf16 pages, to fp16 (2^-11, and 2^-25 of the largest
  weight below its normal range) for e4m3 pages."""
import pytest
import torch

from chessdecoder_b200 import kernels as K

from paged_reference import D, attention, quantise, rope_table, rotate, rows_of, values

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error():
    K.get_error()
    yield
    assert K.get_error() == 0


def pool(n, h, p, fp8, seed=0, fill=None, layers=None, layer=0):
    """k, v, k_scale, v_scale of n pages; layers: a view of one layer of a pool that holds several per page."""
    g = torch.Generator().manual_seed(seed)
    shape = (n, h, p, D) if layers is None else (n, layers, h, p, D)
    got, scales = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g) * torch.exp(0.7 * torch.randn(shape[-1], generator=g))
        if fp8:
            v, e = quantise(x)
            unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]
            x, s = (v / unit).float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
            s = s.to(DEV)
            scales.append(s if layers is None else s[:, layer])
        else:
            x = x.to(torch.bfloat16)
        x = x.to(DEV)
        got.append(x if layers is None else x[:, layer])
    return got + (scales if fp8 else [None, None])


def table_of(lens, p, seed=0, width=None, spare=2):
    """Random distinct pages for sequences of the given lengths; unused entries -1."""
    need = [(max(n, 0) + p - 1) // p for n in lens]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    t = torch.full((len(lens), max(need + [1]) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t.to(DEV), sum(need) + spare


def check_attn(out, q, kp, vp, ks, vs, table, lens, H, scale):
    ref, mag, big = attention(q, values(kp, ks), values(vp, vs), table, lens, H, scale)
    n = torch.tensor(lens, dtype=torch.float64)[:, None, None]
    c = 2 * 68 * 2.0 ** -24 * big[..., None] + 2.0 ** -20 + n * 2.0 ** -24
    if ks is None:
        tol = 2.0 ** -8 * ref.abs() + (c + 2.0 ** -8) * mag
    else:
        top = torch.stack([rows_of(values(vp, vs), table, b, m).abs().amax() if m > 0 else torch.tensor(0.0).double()
                           for b, m in enumerate(lens)])[:, None, None]
        tol = 2.0 ** -8 * ref.abs() + (c + 2.0 ** -11) * mag + n * 2.0 ** -25 * top
    got = out.cpu().double().view(len(lens), H, D)
    assert got.isfinite().all()
    worst = ((got - ref).abs() / tol.clamp_min(1e-30))
    worst[(got - ref) == 0] = 0
    assert worst.max().item() <= 1.0, (worst.max().item(), lens)


def run_attn(lens, H, Hkv, p, fp8, seed=0, scale=0.125, **kw):
    table, n = table_of(lens, p, seed)
    kp, vp, ks, vs = pool(n, Hkv, p, fp8, seed, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(len(lens), H * D, generator=g) * 1.5).to(torch.bfloat16).to(DEV)
    out = torch.full((len(lens), H * D), float("nan"), dtype=torch.bfloat16, device=DEV)
    K.paged_attn(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), out, k_scale=ks, v_scale=vs,
                 scale=scale)
    check_attn(out, q, kp, vp, ks, vs, table, lens, H, scale)
    return out


# -- append -------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("B,S,H,Hkv,p,rot", [(1, 1, 1, 1, 16, True), (3, 1, 8, 2, 64, True), (2, 37, 3, 3, 16, True),
                                             (4, 5, 6, 2, 1, False), (2, 70, 16, 16, 64, False), (5, 3, 7, 1, 8, True)])
def test_append(B, S, H, Hkv, p, rot, f32, fp8):
    g = torch.Generator().manual_seed(B * 100 + S)
    start = [(13 * b) % 29 for b in range(B)]
    count = [S - (b % 3) if S > 2 else S for b in range(B)]
    caps = [a + c for a, c in zip(start, count)]
    table, n = table_of(caps, p, 3)
    kp, vp, ks, vs = pool(n, Hkv, p, fp8, 5)
    before = [values(kp, ks), values(vp, vs)]
    x = torch.randn(B * S, (H + 2 * Hkv) * D + 24, generator=g) * 3
    x = x if f32 else x.to(torch.bfloat16)
    qkv = x.to(DEV)
    rope = rope_table(128, DEV) if rot else None
    pos = torch.randint(0, 128, (B * S,), generator=g).to(torch.int32)
    q_out = torch.full((B * S, H * D + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    K.paged_append(qkv, B, S, H, kp, vp, table, torch.tensor(start, dtype=torch.int32, device=DEV),
                   num_new=torch.tensor(count, dtype=torch.int32, device=DEV), k_scale=ks, v_scale=vs,
                   pos=pos.to(DEV) if rot else None, rope=rope, q_out=q_out)
    heads = x[:, :(H + 2 * Hkv) * D].double().view(B, S, H + 2 * Hkv, D)
    err = torch.zeros_like(heads)
    if rot:
        cs = rope.cpu()[pos.long()].view(B, S, 1, D // 2, 2)
        turned = rotate(heads[:, :, :H + Hkv], cs)
        err[:, :, :H + Hkv] = 3 * 2.0 ** -24 * 2 * heads[:, :, :H + Hkv].abs().amax(-1, keepdim=True)
        heads = torch.cat([turned, heads[:, :, H + Hkv:]], 2)
    got_q = q_out.cpu().double()
    assert (got_q[:, H * D:] == 7).all()
    got_q = got_q[:, :H * D].reshape(B, S, H, D)
    after = [values(kp, ks), values(vp, vs)]
    for b in range(B):
        m = count[b]
        assert (got_q[b, m:] == 7).all()  # padding is left alone
        ref = heads[b, :m, :H]
        assert ((got_q[b, :m] - ref).abs() <= 2.0 ** -8 * ref.abs() + 2 * err[b, :m, :H]).all()
        for i, now in enumerate(after):
            at = H + i * Hkv
            ref, e0 = heads[b, :m, at:at + Hkv], err[b, :m, at:at + Hkv]
            rows = rows_of(now, table, b, caps[b])[:, start[b]:].transpose(0, 1)
            if fp8:
                want, e = quantise(ref)
                unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]
                if not rot or i == 1:
                    assert torch.equal(rows, want)
                else:  # the rotation's last bits can move a maximum over 448 * 2^e: one unit more
                    assert ((rows - ref).abs() <= 2.0 ** -4 * ref.abs() + 2.0 ** -9 * unit + 2 * e0).all()
            else:
                assert ((rows - ref).abs() <= 2.0 ** -8 * ref.abs() + 2 * e0).all()
    written = torch.zeros(n, p, dtype=torch.bool)
    for b in range(B):
        j = torch.arange(start[b], caps[b])
        written[table[b].cpu().long()[j // p], j % p] = True
    keep = ~written[:, None, :, None].expand_as(before[0])
    for a, c in zip(before, after):
        assert torch.equal(a[keep], c[keep])  # every other row as it was


def test_append_scale_edges():
    """Rows at the borders of a scale: 448 * 2^e exactly, just above it, zeros, the
    smallest and largest numbers, an infinity, a NaN."""
    tiny = torch.finfo(torch.float32).tiny
    tops = [448.0, 448.0 * (1 + 2.0 ** -23), 447.9, 0.0, tiny, tiny / 4, 1.0, 3.3e38, 448 * 2.0 ** -126]
    x = torch.zeros(len(tops) + 2, 3 * D)
    x[:len(tops)] = torch.linspace(-1, 1, 3 * D)[None] * torch.tensor(tops)[:, None]
    x[:len(tops), D:2 * D][:, 5] = torch.tensor(tops)
    x[:len(tops), 2 * D:][:, 7] = -torch.tensor(tops)
    x[-2, D + 3], x[-2, D + 4] = float("inf"), 2.0
    x[-1, D + 3], x[-1, D + 4] = float("nan"), 448.0
    T = x.shape[0]
    table = torch.arange(T, dtype=torch.int32, device=DEV)[:, None].contiguous()
    kp, vp, ks, vs = pool(T, 1, 1, True)
    K.paged_append(x.to(DEV), T, 1, 1, kp, vp, table, torch.zeros(T, dtype=torch.int32, device=DEV), k_scale=ks,
                   v_scale=vs)
    got = [values(kp, ks)[:, 0, 0], values(vp, vs)[:, 0, 0]]
    n = len(tops)
    for i in range(2):
        rows = x[:n, (i + 1) * D:(i + 2) * D]
        want, e = quantise(rows)
        assert torch.equal((ks, vs)[i].cpu().view(torch.uint8)[:n, 0, 0].long(), e.long() + 127)
        assert torch.equal(got[i][:n], want)
    assert got[0][-2][3] == 448 * 2.0 ** 120 and got[0][-2].float()[3] == float("inf")
    assert got[0][-1][3].isnan() and got[0][-1][4] == 448 and got[0][-1].isnan().sum() == 1


# -- read back ----------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("p,lens", [(16, [1, 0, 33, 16, 17]), (64, [200]), (1, [3, 5]), (256, [255, 256, 257])])
def test_gather(p, lens, fp8):
    table, n = table_of(lens, p, 1)
    kp, vp, ks, vs = pool(n, 3, p, fp8, 2)
    B, S = len(lens), max(lens) + 2
    # [B, S, heads, 64] storage seen as [B, heads, S, 64]: strides other than the contiguous ones
    outs = [torch.full((B, S, 3, D), 9.0, dtype=torch.bfloat16, device=DEV).transpose(1, 2) for _ in range(2)]
    K.paged_gather(kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), *outs, k_scale=ks, v_scale=vs)
    for o, vals in zip(outs, (values(kp, ks), values(vp, vs))):
        for b, m in enumerate(lens):
            assert torch.equal(o[b, :, :m].cpu().double(), rows_of(vals, table, b, m))
            assert (o[b, :, m:] == 9).all()


def test_gather_keeps_every_scale():
    """All scale bytes that an append writes, with every finite code, come back as
    the fp32 product rounds to bf16."""
    codes = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8)
    byte = torch.arange(1, 249, dtype=torch.uint8)
    x = codes.repeat(4)[:D * 15].view(15, D)
    kp = x[None, None].expand(248, 1, 15, D).contiguous()
    kp = torch.cat([kp, kp[:, :, :1]], 2).view(torch.float8_e4m3fn).to(DEV)
    ks = byte[:, None, None].expand(248, 1, 16).contiguous().view(torch.float8_e8m0fnu).to(DEV)
    table = torch.arange(248, dtype=torch.int32, device=DEV)[:, None].contiguous()
    lens = torch.full((248,), 16, dtype=torch.int32, device=DEV)
    ko, vo = (torch.zeros(248, 1, 16, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    K.paged_gather(kp, kp, table, lens, ko, vo, k_scale=ks, v_scale=ks)
    want = values(kp, ks)[:, 0].float().to(torch.bfloat16)  # the largest products are beyond fp32: infinity on both sides
    assert torch.equal(ko.cpu()[:, 0], want) and torch.equal(vo.cpu()[:, 0], want)


# -- attention ----------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (16, 16), (6, 2), (8, 1), (9, 1), (14, 2), (16, 1), (12, 4)])
def test_attn_heads(H, Hkv, fp8):
    run_attn([1, 100, 0, 257], H, Hkv, 16, fp8, seed=H)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("p", [1, 2, 8, 16, 32, 64, 128, 512])
def test_attn_pages_and_lengths(p, fp8):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 511, 513]
    run_attn(lens, 4, 2, p, fp8, seed=p)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens", [[20011], [1, 9000, 3], [4096] * 3, [0, 0, 0], [1] * 700, [50] * 300 + [3000]])
def test_attn_uneven_batches(lens, fp8):
    run_attn(lens, 4, 2, 64, fp8, seed=len(lens))


# a warp per item; eight; four, with one to many waves of blocks; the deal
WAYS = [[i * 7 % 61 for i in range(320)], [i * 37 % 257 for i in range(640)], [700, 0, 33, 1000, 129],
        [i * 331 % 1001 for i in range(160)], [0, 1, 1500, 40, 3000], [i * 331 % 1201 for i in range(150)]]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,p", [(2, 16), (16, 64), (18, 16), (32, 32)])
@pytest.mark.parametrize("lens", WAYS, ids=["warp", "warp8", "eight", "four", "deal", "deal150"])
def test_attn_ways(lens, H, p, fp8):
    run_attn(lens, H, 2, p, fp8, seed=H)


@pytest.mark.parametrize("fp8", [False, True])
def test_attn_sharp_and_flat_scores(fp8):
    for scale in (0.0, 1.0, -2.0, 8.0):
        run_attn([70, 1000], 4, 4, 32, fp8, scale=scale)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("qe,ke,se", [(125, -113, -12), (-120, 100, 20), (0, -126, 126), (60, 60, -120)])
def test_attn_far_magnitudes(qe, ke, se, fp8):
    """Queries and keys near the ends of the number range whose scores are ordinary,
    values of 2^-90 and rows of zeros among them."""
    lens, H, p = [70, 33], 4, 16
    table, n = table_of(lens, p, 3)
    kp, vp, ks, vs = pool(n, 2, p, fp8, 3)
    if fp8:
        ks = (ks.view(torch.uint8).int() + ke).clamp(1, 247).to(torch.uint8).view(torch.float8_e8m0fnu)
        vs = (vs.view(torch.uint8).int() - 90).to(torch.uint8).view(torch.float8_e8m0fnu)
        vp.view(torch.uint8)[:, :, ::3] = 0
        vs.view(torch.uint8)[:, :, ::3] = 1
    else:
        kp, vp = (kp.float() * 2.0 ** ke).to(torch.bfloat16), (vp.float() * 2.0 ** -90).to(torch.bfloat16)
        vp[:, :, ::3] = 0
    g = torch.Generator().manual_seed(2)
    q = (torch.randn(2, H * D, generator=g).clamp(-3, 3) * 2.0 ** qe).to(torch.bfloat16).to(DEV)
    out = torch.empty(2, H * D, dtype=torch.bfloat16, device=DEV)
    scale = 0.125 * 2.0 ** se
    K.paged_attn(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), out, k_scale=ks, v_scale=vs,
                 scale=scale)
    check_attn(out, q, kp, vp, ks, vs, table, lens, H, scale)


@pytest.mark.parametrize("fp8", [False, True])
def test_attn_strides_and_layer_views(fp8):
    lens, H, Hkv, p = [90, 0, 17], 6, 3, 16
    table, n = table_of(lens, p, 4, width=None)
    wide = torch.full((3, table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    kp, vp, ks, vs = pool(n, Hkv, p, fp8, 4, layers=3, layer=1)
    base = torch.randn(3, H * D + 64).to(torch.bfloat16).to(DEV)
    q = base[:, 8:8 + H * D]
    hold = torch.full((3, H * D + 16), 5.0, dtype=torch.bfloat16, device=DEV)
    out = hold[:, 8:8 + H * D]
    K.paged_attn(q, kp, vp, wide[:, :table.shape[1]], torch.tensor(lens, dtype=torch.int32, device=DEV), out,
                 k_scale=ks, v_scale=vs)
    check_attn(out, q, kp, vp, ks, vs, table, lens, H, 0.125)
    assert (hold[:, :8] == 5).all() and (hold[:, 8 + H * D:] == 5).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_attn_ignores_what_is_behind_a_sequence(fp8):
    """Rows behind a length and pages that no sequence holds: NaN, infinities, NaN scales."""
    lens, H, Hkv, p = [5, 64, 70, 0], 4, 2, 64
    table, n = table_of(lens, p, 6)
    kp, vp, ks, vs = pool(n, Hkv, p, fp8, 6)
    used = torch.zeros(n, p, dtype=torch.bool)
    for b, m in enumerate(lens):
        j = torch.arange(m)
        used[table[b].cpu().long()[j // p], j % p] = True
    dead = ~used.to(DEV)
    for x, s in ((kp, ks), (vp, vs)):
        if fp8:
            x.view(torch.uint8).transpose(1, 2)[dead] = 0x7F
            s.view(torch.uint8).transpose(1, 2)[dead] = 0xFF
        else:
            x.transpose(1, 2)[dead] = float("nan")
            x[:, 0, -1][dead[:, -1]] = float("inf")
    q = torch.randn(4, H * D).to(torch.bfloat16).to(DEV)
    out = torch.full((4, H * D), float("nan"), dtype=torch.bfloat16, device=DEV)
    K.paged_attn(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), out, k_scale=ks, v_scale=vs)
    assert out.isfinite().all() and (out[3] == 0).all()
    clean = [kp.clone(), vp.clone()]
    for x in clean:
        x.view(torch.uint8 if fp8 else torch.bfloat16).transpose(1, 2)[dead] = 0
    cs = [None, None]
    if fp8:
        cs = [ks.clone(), vs.clone()]
        for s in cs:
            s.view(torch.uint8).transpose(1, 2)[dead] = 127
    check_attn(out, q, clean[0], clean[1], cs[0], cs[1], table, lens, H, 0.125)


def test_attn_nan_in_a_key_that_counts_stays_in_its_head():
    lens, H = [40], 4
    table, n = table_of(lens, 16, 6)
    kp, vp, _, _ = pool(n, 4, 16, False, 6)
    kp[table[0, 1], 2, 3, 5] = float("nan")
    q = torch.randn(1, H * D).to(torch.bfloat16).to(DEV)
    out = torch.zeros(1, H * D, dtype=torch.bfloat16, device=DEV)
    K.paged_attn(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), out)
    bad = out.view(4, D).isnan().all(1)
    assert bad.tolist() == [False, False, True, False] and out.view(4, D)[~bad].isfinite().all()


def test_attn_shared_pages_and_repeats():
    """Two sequences over the same pages give what one gives; the same call twice gives the same bits."""
    table, n = table_of([300], 16, 2)
    kp, vp, ks, vs = pool(n, 2, 16, True, 2)
    q = torch.randn(1, 8 * D).to(torch.bfloat16).to(DEV).repeat(3, 1)
    lens = torch.tensor([300, 300, 300], dtype=torch.int32, device=DEV)
    outs = [torch.empty(3, 8 * D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for o in outs:
        K.paged_attn(q, kp, vp, table.repeat(3, 1), lens, o, k_scale=ks, v_scale=vs)
    assert torch.equal(outs[0], outs[1])
    check_attn(outs[0], q, kp, vp, ks, vs, table.repeat(3, 1), [300] * 3, 8, 0.125)


def test_bad_pages_set_the_error_bit_and_are_skipped():
    """A table entry that no pool has, or a length past the table: the rows there are
    masked, not written, left alone, and the index error bit is set."""
    p, H = 16, 2
    kp, vp, _, _ = pool(4, H, p, False, 1)
    table = torch.tensor([[0, 99, 2], [1, -3, 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([40, 100], dtype=torch.int32, device=DEV)
    q = torch.randn(2, H * D).to(torch.bfloat16).to(DEV)
    out = torch.empty(2, H * D, dtype=torch.bfloat16, device=DEV)
    K.paged_attn(q, kp, vp, table, lens, out)
    assert K.get_error() == 2
    # what is left: rows 0..15 and 32..39 of the first, 0..15 and 32..47 of the second
    t2 = torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device=DEV)
    check_attn(out, q, kp, vp, None, None, t2, [24, 32], H, 0.125)
    ko, vo = (torch.full((2, H, 48, D), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    K.paged_gather(kp, vp, table, lens, ko, vo)
    assert K.get_error() == 2
    assert (ko[:, :, 16:32] == 3).all() and torch.equal(ko[0, :, 32:40], kp[2, :, :8]) and (ko[0, :, 40:] == 3).all()
    assert torch.equal(vo[1, :, 32:48], vp[3])
    before = kp.clone()
    qkv = torch.randn(2, 3 * H * D, device=DEV)
    K.paged_append(qkv, 2, 1, H, kp, vp, table, torch.tensor([17, 48], dtype=torch.int32, device=DEV))
    assert K.get_error() == 2 and torch.equal(kp, before)
    K.paged_append(qkv, 2, 1, H, kp, vp, table, torch.tensor([-1, 0], dtype=torch.int32, device=DEV),
                   pos=torch.tensor([0, 8], dtype=torch.int32, device=DEV), rope=rope_table(8, DEV))
    assert K.get_error() == 2 and torch.equal(kp, before)  # row -1; position 8 of 8


def test_long_cache_offsets_past_32_bits():
    """A pool of more than 2^32 bytes whose last pages are used."""
    p, Hkv = 64, 8
    n = (1 << 32) // (Hkv * p * D * 2) + 9  # bf16 bytes per page
    kp = torch.zeros(n, Hkv, p, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros(n, Hkv, p, D, dtype=torch.bfloat16, device=DEV)
    table = torch.tensor([[n - 1, 2, n - 5]], dtype=torch.int32, device=DEV)
    qkv = torch.randn(150, 3 * Hkv * D, device=DEV)
    K.paged_append(qkv, 1, 150, Hkv, kp, vp, table, torch.zeros(1, dtype=torch.int32, device=DEV))
    ko, vo = (torch.zeros(1, Hkv, 150, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    lens = torch.tensor([150], dtype=torch.int32, device=DEV)
    K.paged_gather(kp, vp, table, lens, ko, vo)
    want = qkv[:, Hkv * D:2 * Hkv * D].view(150, Hkv, D).transpose(0, 1).to(torch.bfloat16)
    assert torch.equal(ko[0], want)
    q = torch.randn(1, Hkv * D, device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    K.paged_attn(q, kp, vp, table, lens, out)
    small = torch.cat([kp[n - 1:], kp[2:3], kp[n - 5:n - 4]]), torch.cat([vp[n - 1:], vp[2:3], vp[n - 5:n - 4]])
    check_attn(out, q, small[0], small[1], None, None, torch.arange(3, dtype=torch.int32)[None], [150], Hkv, 0.125)


# -- how it is called -----------------------------------------------------------
def test_streams_graphs_and_workspaces():
    """A side stream; a captured step (append, attention) replayed while its inputs
    change, with a workspace of its own; two graphs that share a workspace, one after
    the other; two streams at once with a workspace each."""
    B, H, p = 3, 4, 16
    lens = [20, 200, 64]
    table, n = table_of([m + 8 for m in lens], p, 9)
    kp, vp, ks, vs = pool(n, H, p, True, 9)
    rope = rope_table(512, DEV)
    qkv = torch.randn(B, 3 * H * D, device=DEV)
    start = torch.tensor(lens, dtype=torch.int32, device=DEV)
    after = start + 1
    q16 = torch.zeros(B, H * D, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros(B, H * D, dtype=torch.bfloat16, device=DEV)
    ws = torch.empty(K.paged_attn_workspace(B, H, H), dtype=torch.uint8, device=DEV)

    def step(o, w=ws):
        K.paged_append(qkv, B, 1, H, kp, vp, table, start, k_scale=ks, v_scale=vs, pos=start, rope=rope, q_out=q16)
        K.paged_attn(q16, kp, vp, table, after, o, k_scale=ks, v_scale=vs, workspace=w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out)
    torch.cuda.current_stream().wait_stream(side)
    check_attn(out, q16, kp, vp, ks, vs, table, [m + 1 for m in lens], H, 0.125)
    outs = [torch.zeros_like(out) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, o in zip(graphs, outs):
        with torch.cuda.graph(g):
            step(o)
    for k in range(3):
        qkv.copy_(torch.randn(B, 3 * H * D, device=DEV))
        graphs[0].replay()
        check_attn(outs[0], q16, kp, vp, ks, vs, table, [m + 1 + k for m in lens], H, 0.125)
        graphs[1].replay()  # the same step again into another output
        assert torch.equal(outs[0], outs[1])
        start += 1
        after += 1
    both = [torch.zeros_like(out) for _ in range(2)]
    spaces = [torch.empty_like(ws) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, o, w in zip(streams, both, spaces):
            with torch.cuda.stream(st):
                K.paged_attn(q16, kp, vp, table, start, o, k_scale=ks, v_scale=vs, workspace=w)
    torch.cuda.synchronize()
    assert torch.equal(both[0], both[1])
    check_attn(both[0], q16, kp, vp, ks, vs, table, start.tolist(), H, 0.125)


def test_workspace_needs_no_clearing():
    lens = [3000, 1, 700]
    table, n = table_of(lens, 64, 5)
    kp, vp, _, _ = pool(n, 2, 64, False, 5)
    q = torch.randn(3, 4 * D).to(torch.bfloat16).to(DEV)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = torch.empty(K.paged_attn_workspace(3, 4, 2), dtype=torch.uint8, device=DEV)
    outs = []
    for fill in (0, 0xFF, 0x7F):
        ws.fill_(fill)
        outs.append(torch.empty(3, 4 * D, dtype=torch.bfloat16, device=DEV))
        K.paged_attn(q, kp, vp, table, ln, outs[-1], workspace=ws)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_empty_batches_launch_nothing():
    kp, vp, _, _ = pool(2, 2, 16, False)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    t = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    K.paged_attn(torch.zeros(0, 128, dtype=torch.bfloat16, device=DEV), kp, vp, t, none,
                 torch.zeros(0, 128, dtype=torch.bfloat16, device=DEV))
    K.paged_append(torch.zeros(0, 384, device=DEV), 0, 4, 2, kp, vp, t, none)
    K.paged_gather(kp, vp, t, none, *(torch.zeros(0, 2, 5, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)))
    # a table without pages: every sequence is empty
    t = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    out = torch.ones(2, 128, dtype=torch.bfloat16, device=DEV)
    K.paged_attn(torch.ones_like(out), kp, vp, t, torch.zeros(2, dtype=torch.int32, device=DEV), out)
    assert (out == 0).all()
