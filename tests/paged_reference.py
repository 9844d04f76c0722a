"""Plain 64-bit statements of the paged cache's operators, for the tests."""
import torch

D = 64


def rope_table(n, dev="cpu"):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return torch.stack([a.cos(), a.sin()], -1).float().to(dev)


def rotate(x, cs):
    """x [..., 64], cs [..., 32, 2] (broadcast): interleaved pairs, 64 bits."""
    x, cs = x.double(), cs.double()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1).flatten(-2)


def scale_exponent(rows):
    """The least e >= -126 with max|row| <= 448 * 2^e."""
    mant, e = torch.frexp(rows.double().abs().amax(-1) / 448.0)
    return torch.where(mant == 0.5, e - 1, torch.where(mant == 0, -126, e)).clamp(min=-126)


def e4m3(x):
    """x rounded to the nearest e4m3 value, ties to even, in 64 bits (|x| <= 448)."""
    mag = x.abs()
    _, e = torch.frexp(mag)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 4).clamp(min=-9).double())
    return torch.sign(x) * torch.round(mag / step) * step


def quantise(rows):
    """(values that the codes stand for, exponents) of rows of 64."""
    e = scale_exponent(rows)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]
    return e4m3(rows.double() / unit) * unit, e


def values(pages, scale):
    """What a pool's rows stand for, in 64 bits, [pages, heads, page_size, 64]."""
    x = pages.cpu().float().double()
    if scale is not None:
        e = scale.cpu().view(torch.uint8).double() - 127
        x = x * torch.pow(torch.full_like(e, 2.0), e)[..., None]
    return x


def rows_of(vals, table, b, n):
    """The first n rows of sequence b, [kv_heads, n, 64]."""
    p = vals.shape[2]
    j = torch.arange(n)
    return vals[table[b].cpu().long()[j // p], :, j % p].transpose(0, 1)


def attention(q, kv, vv, table, lens, H, scale):
    """(out, sum p|v|, largest scale * sum|q k|) per sequence and head; empty sequences give zeros."""
    B, G = len(lens), H // kv.shape[1]
    out, mag = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    big = torch.zeros(B, H, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        qb = q[b].cpu().double().view(-1, G, D)
        k, v = rows_of(kv, table, b, n), rows_of(vv, table, b, n)
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", qb, k) * scale, -1)
        out[b] = torch.einsum("hgn,hnd->hgd", p, v).reshape(H, D)
        mag[b] = torch.einsum("hgn,hnd->hgd", p, v.abs()).reshape(H, D)
        big[b] = (torch.einsum("hgd,hnd->hgn", qb.abs(), k.abs()).amax(-1) * abs(scale)).reshape(H)
    return out, mag, big
