"""Cases of the paged key-value cache and of the token statistics, for timing.

Four operators: rows of a projection rotated and written into a paged cache
(bf16, or e4m3 with a power-of-two scale a row), the pages read back as dense
bf16 rows, the attention of one new token a sequence over its pages, and the
log-probability of given tokens with the entropy, the top alternatives and the
gradient.  Heads are 64 wide, as everywhere in this framework.

Where ``own`` is false, ``run`` computes the plain form in elementary torch
operations; where it is true, it calls the framework's kernels.
"""
import math

import torch

own = False

D = 64


def listed():
    return [
        # one decode step of a batch of games: every sequence's new key and value
        dict(name="append_step", op="append", B=64, S=1, H=16, G=1, P=64, fp8=False, f32=True, rope=True),
        # the same step of a few grouped-query sequences into an 8-bit cache
        dict(name="append_step_fp8", op="append", B=7, S=1, H=32, G=8, P=16, fp8=True, f32=True, rope=True),
        # padded prompts, already rotated by the projection's epilogue, quantised as they are written
        dict(name="append_prompt_fp8", op="append", B=24, S=1000, H=16, G=1, P=64, fp8=True, f32=False, rope=False),
        # a few short sequences taken out of the pool
        dict(name="gather_short", op="gather", B=5, lo=1, hi=300, H=16, G=1, P=16, fp8=False),
        # long 8-bit sequences read back for a many-token pass
        dict(name="gather_long_fp8", op="gather", B=16, lo=500, hi=8191, H=16, G=1, P=64, fp8=True),
        # the smallest step: one game of a few moves, where latency counts
        dict(name="attn_one", op="attn", B=1, lo=137, hi=137, H=16, G=1, P=64, fp8=False),
        # a batch of games in mid-rollout, one of them just begun
        dict(name="attn_step", op="attn", B=64, lo=0, hi=2000, H=16, G=1, P=64, fp8=False),
        # few long sequences with grouped heads and an 8-bit cache
        dict(name="attn_long_fp8", op="attn", B=6, lo=9001, hi=65536, H=32, G=8, P=64, fp8=True),
        # the largest: a full serving batch
        dict(name="attn_batch", op="attn", B=256, lo=1, hi=4095, H=16, G=1, P=64, fp8=False),
        # the tokens that a decode step chose, with five alternatives (legal moves only)
        dict(name="stats_step", op="stats", R=64, V=1924, k=5, bf16=False, grad=False, masked=0.9),
        # the move rows of a policy-gradient batch with an entropy bonus, padding among them
        dict(name="stats_train", op="stats", R=16384, V=1924, k=0, bf16=False, grad=True, masked=0.0),
        # a large vocabulary of odd size, with the alternatives that an interface returns at most
        dict(name="stats_vocab", op="stats", R=509, V=131071, k=20, bf16=True, grad=True, masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "attn", "attn", "stats"])
    heads = dict(P=rng.choice([16, 32, 64, 128]), fp8=rng.random() < 0.5)
    heads["G"] = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16])
    heads["H"] = heads["G"] * rng.choice([1, 2, 4, 8, 16] if heads["G"] < 5 else [1, 2, 4])
    kv = heads["H"] // heads["G"]
    if op == "append":
        S = rng.choice([1, 1, _log_int(rng, 2, 2000)])
        B = _log_int(rng, 1, max(1, min(256, 1_000_000 // (S * (heads["H"] + 2 * kv)))))
        return dict(op=op, B=B, S=S, **heads, f32=rng.random() < 0.5, rope=rng.random() < 0.7)
    if op == "stats":
        V = _log_int(rng, 41, 131071)
        R = _log_int(rng, 1, max(1, min(20000, 60_000_000 // V)))
        return dict(op=op, R=R, V=V, k=rng.choice([0, 1, 5, 20, 32]), bf16=rng.random() < 0.5, grad=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.0, 0.5, 0.9]))
    B = _log_int(rng, 1, 256)
    most = min(131072 if op == "attn" else 16384, (8_000_000 if op == "attn" else 1_000_000) // (B * kv))
    hi = _log_int(rng, 1, max(1, most))
    return dict(op=op, B=B, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, **heads)


def _lens(case):
    """Ragged lengths spread over [lo, hi], the first at hi, the second at lo."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi if b == 0 else lo if b == 1 else lo + int((hi - lo) * (b * 0.6180339887 % 1.0)) for b in range(B)]


def _counts(case):
    """New tokens of each sequence of an append: all of S, or ragged prompts."""
    B, S = case["B"], case["S"]
    return [S if S == 1 or b == 0 else S - int(S * 0.5 * (b * 0.6180339887 % 1.0)) for b in range(B)]


def work(case):
    op = case["op"]
    if op == "stats":
        one = case["R"] * case["V"] * (2 if case["bf16"] else 4)
        return {"bytes": one * (3 if case["grad"] else 1), "flops": case["R"] * case["V"] * (12 if case["grad"] else 5)}
    H, kv = case["H"], case["H"] // case["G"]
    row = kv * (2 * (D + 1) if case["fp8"] else 4 * D)  # key and value of one token in the cache
    if op == "append":
        n, elt = sum(_counts(case)), 4 if case["f32"] else 2
        q = H * D * (elt + 2) if case["rope"] else 0
        return {"bytes": n * (2 * kv * D * elt + row + q), "flops": n * (H + 2 * kv) * D * 4}
    n = sum(_lens(case))
    if op == "gather":
        return {"bytes": n * (row + kv * 4 * D), "flops": n * kv * 2 * D}
    return {"bytes": n * row + case["B"] * H * D * 4, "flops": 4 * n * H * D}


def _codes(x):
    """(e4m3 codes, scale bytes) of rows of 64: the least power of two 2^e, e >= -126, with max|x| <= 448 * 2^e."""
    bits = x.abs().amax(-1).view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=1)
    inv = ((254 - byte) << 23).view(torch.float32)
    return (x * inv.unsqueeze(-1)).to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _pool(case, g, pages, dev):
    """A pool as a long-running program has it: earlier keys and values in every row, some channels larger."""
    kv, P = case["H"] // case["G"], case["P"]
    amp = torch.exp(0.7 * torch.randn(2, kv, 1, D, generator=g, device=dev))
    out = []
    for i in range(2):
        x = torch.empty(pages, kv, P, D, dtype=torch.float8_e4m3fn if case["fp8"] else torch.bfloat16, device=dev)
        s = torch.empty(pages, kv, P, dtype=torch.uint8, device=dev) if case["fp8"] else None
        for a in range(0, pages, 4096):
            r = torch.randn(min(4096, pages - a), kv, P, D, generator=g, device=dev) * amp[i]
            if case["fp8"]:
                x[a:a + 4096], s[a:a + 4096] = _codes(r)
            else:
                x[a:a + 4096] = r
        out.append((x, None if s is None else s.view(torch.float8_e8m0fnu)))
    return out


def _table(caps, P, g, dev):
    """Page tables in a pool whose pages were taken in random order; unused entries are -1."""
    need = [(n + P - 1) // P for n in caps]
    total, width = sum(need), max(max(need), 1)
    pages = total + 3
    order = torch.randperm(pages, generator=g, device=dev)[:total].to(torch.int32)
    table = torch.full((len(caps), width), -1, dtype=torch.int32, device=dev)
    used = torch.arange(width, device=dev)[None] < torch.tensor(need, device=dev)[:, None]
    table[used] = order
    return table, pages


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "stats":
        R, V = case["R"], case["V"]
        x = torch.randn(R, V, generator=g, device=dev) * 2.5
        t = torch.randint(0, V, (R,), generator=g, device=dev)
        if case["masked"]:
            gone = torch.rand(R, V, generator=g, device=dev) < case["masked"]
            gone.scatter_(1, t[:, None], False)
            x.masked_fill_(gone, -math.inf)
        s["logits"] = x.to(torch.bfloat16) if case["bf16"] else x
        pad = torch.rand(R, generator=g, device=dev) < 0.05
        s["target"] = torch.where(pad, -100, t).to(torch.int32)
        if case["grad"]:
            s["dlp"] = torch.where(pad, 0.0, torch.randn(R, generator=g, device=dev)) / R
            s["dent"] = torch.where(pad, 0.0, -0.01 / R * torch.ones(R, device=dev))
        return s
    B, H, kv, P = case["B"], case["H"], case["H"] // case["G"], case["P"]
    perm = torch.randperm(B, generator=g, device=dev).cpu().tolist()
    if case["op"] == "append":
        count = [_counts(case)[i] for i in perm]
        start = [37 * i % 400 for i in perm]  # what each sequence holds already
        caps = [a + n for a, n in zip(start, count)]
        T = B * case["S"]
        qkv = torch.randn(T, (H + 2 * kv) * D, generator=g, device=dev)
        qkv *= torch.exp(0.5 * torch.randn((H + 2 * kv) * D, generator=g, device=dev))
        s["qkv"] = qkv if case["f32"] else qkv.to(torch.bfloat16)
        s["start"] = torch.tensor(start, dtype=torch.int32, device=dev)
        s["count"] = torch.tensor(count, dtype=torch.int32, device=dev)
        if case["rope"]:
            at = torch.arange(4096, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2) / D)
            s["rope"] = torch.stack([at.cos(), at.sin()], -1).float().to(dev)
            pos = s["start"][:, None] + torch.arange(case["S"], dtype=torch.int32, device=dev)[None]
            s["pos"] = pos.reshape(-1).to(torch.int32)
            s["q_out"] = torch.zeros(T, H * D, dtype=torch.bfloat16, device=dev)
    else:
        caps = [_lens(case)[i] for i in perm]
        s["lens"] = torch.tensor(caps, dtype=torch.int32, device=dev)
    s["table"], pages = _table(caps, P, g, dev)
    (s["k"], s["ks"]), (s["v"], s["vs"]) = _pool(case, g, pages, dev)
    if case["op"] == "gather":
        for n in ("k_out", "v_out"):
            s[n] = torch.zeros(B, kv, max(max(caps), 1), D, dtype=torch.bfloat16, device=dev)
    elif case["op"] == "attn":
        s["q"] = (torch.randn(B, H * D, generator=g, device=dev) * 1.5).to(torch.bfloat16)
        s["out"] = torch.empty(B, H * D, dtype=torch.bfloat16, device=dev)
    return s


def run(state):
    return globals()["_" + state["case"]["op"]](state)


def _append(s):
    case = s["case"]
    B, S, H, P = case["B"], case["S"], case["H"], case["P"]
    if own:
        from chessdecoder_b200 import kernels as K
        K.paged_append(s["qkv"], B, S, H, s["k"], s["v"], s["table"], s["start"], num_new=s["count"],
                       k_scale=s["ks"], v_scale=s["vs"], pos=s.get("pos"), rope=s.get("rope"), q_out=s.get("q_out"))
        return _written(s)
    kv = H // case["G"]
    x = s["qkv"].float().view(B * S, H + 2 * kv, D)
    qk, v = x[:, :H + kv], x[:, H + kv:]
    off = torch.arange(S, device=x.device)[None]
    real = (off < s["count"][:, None]).reshape(-1)
    slot = s["start"][:, None].long() + off
    if case["rope"]:
        cs = s["rope"][s["pos"].long().clamp(max=s["rope"].shape[0] - 1)][:, None]
        a, b = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1).reshape(qk.shape)
        s["q_out"].copy_(torch.where(real[:, None], qk[:, :H].reshape(B * S, H * D), s["q_out"].float()))
    page = s["table"].gather(1, (slot // P).clamp(max=s["table"].shape[1] - 1)).reshape(-1)[real].long()
    at = (slot % P).reshape(-1)[real]
    for rows, pool, scale in ((qk[:, H:], s["k"], s["ks"]), (v, s["v"], s["vs"])):
        if case["fp8"]:
            codes, byte = _codes(rows[real].contiguous())
            pool.view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
            scale.view(torch.uint8)[page, :, at] = byte
        else:
            pool[page, :, at] = rows[real].to(torch.bfloat16)
    return _written(s)


def _written(s):
    return {n: s[n] for n in ("q_out", "k", "v", "ks", "vs") if s.get(n) is not None}


def _dense(s, n):
    """Keys or values of every sequence as fp32 [B, kv, width * P, D], rows of unused pages zero."""
    t = s["table"]
    x = s[n][t.clamp(min=0).long()].float()
    if s[n + "s"] is not None:
        x = x * s[n + "s"][t.clamp(min=0).long()].float().unsqueeze(-1)
    x = x.transpose(1, 2).flatten(2, 3)
    here = torch.arange(x.shape[2], device=x.device)[None] < s["lens"][:, None]
    return torch.where(here[:, None, :, None], x, 0.0), here


def _gather(s):
    if own:
        from chessdecoder_b200 import kernels as K
        K.paged_gather(s["k"], s["v"], s["table"], s["lens"], s["k_out"], s["v_out"], k_scale=s["ks"], v_scale=s["vs"])
        return s["k_out"], s["v_out"]
    for n in ("k", "v"):
        x, here = _dense(s, n)
        out = s[n + "_out"]
        S = out.shape[2]
        out.copy_(torch.where(here[:, None, :S, None], x[:, :, :S].to(torch.bfloat16), out))
    return s["k_out"], s["v_out"]


def _attn(s):
    if own:
        from chessdecoder_b200 import kernels as K
        K.paged_attn(s["q"], s["k"], s["v"], s["table"], s["lens"], s["out"], k_scale=s["ks"], v_scale=s["vs"],
                     scale=D ** -0.5)
        return s["out"]
    case = s["case"]
    B, H, G = case["B"], case["H"], case["G"]
    k, here = _dense(s, "k")
    q = s["q"].float().view(B, H // G, G, D)
    score = (q @ k.transpose(2, 3)) * D ** -0.5
    del k
    score = score.masked_fill(~here[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    v, _ = _dense(s, "v")
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(B, H * D).to(torch.bfloat16)


def _stats(s):
    case, x, t = s["case"], s["logits"], s["target"]
    R, V, k = case["R"], case["V"], min(case["k"], case["V"])
    if own:
        from chessdecoder_b200 import kernels as K
        dev = x.device
        lp, ent = torch.empty(R, device=dev), torch.empty(R, device=dev)
        lse = torch.empty(R, device=dev) if case["grad"] else None
        ids = torch.empty(R, k, dtype=torch.int32, device=dev) if k else None
        top = torch.empty(R, k, device=dev) if k else None
        K.token_logprobs(x, t, lp, entropy=ent, lse=lse, top_ids=ids, top_lp=top)
        got = [lp, ent]
        if k:
            got += [ids, top]
        if case["grad"]:
            dx = torch.empty_like(x)
            K.token_logprobs_bwd(x, t, lse, ent, s["dlp"], s["dent"], dx)
            got.append(dx)
        return got
    f = x.float()
    m = f.amax(1, keepdim=True)
    z = f - m
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logp = z - torch.log(total)
    p = e / total
    given = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1).long()[:, None]
    lp = torch.where(given, logp.gather(1, at)[:, 0], 0.0)
    ent = torch.log(total)[:, 0] - (e * torch.where(e > 0, z, 0.0)).sum(1) / total[:, 0]
    got = [lp, ent]
    if k:
        order = torch.sort(f, dim=1, descending=True, stable=True)[1][:, :k]
        got += [order.to(torch.int32), logp.gather(1, order)]
    if case["grad"]:
        dx = -p * (s["dlp"][:, None] * given[:, None] + s["dent"][:, None] * (torch.where(p > 0, logp, 0.0) + ent[:, None]))
        dx.scatter_add_(1, at, (s["dlp"] * given)[:, None])
        got.append(dx.to(x.dtype))
    return got


# ---------------------------------------------------------------------------
# 64 bits, sequence by sequence and row by row, from the definitions
# ---------------------------------------------------------------------------
def _exact_rows(s, b, n, which):
    """The first n cached rows of sequence b, [kv, n, D] in 64 bits."""
    P = s["case"]["P"]
    j = torch.arange(n, device="cuda")
    page = s["table"][b, j // P].long()
    x = s[which].view(torch.uint8 if s["case"]["fp8"] else torch.bfloat16)[page, :, j % P]
    if s["case"]["fp8"]:
        e = s[which + "s"].view(torch.uint8)[page, :, j % P].double() - 127
        x = x.view(torch.float8_e4m3fn).double() * torch.pow(torch.full_like(e, 2.0), e)[..., None]
    return x.double().transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](case, s)


def _exact_append(case, s):
    B, S, H, P = case["B"], case["S"], case["H"], case["P"]
    kv = H // case["G"]
    x = s["qkv"].double().view(B, S, H + 2 * kv, D)
    out = {n: None if s.get(n) is None else s[n].double() for n in ("q_out", "k", "v", "ks", "vs")}
    if case["rope"]:
        pair = torch.view_as_complex(x[:, :, :H + kv].reshape(B, S, H + kv, D // 2, 2).contiguous())
        turn = torch.view_as_complex(s["rope"].double())[s["pos"].long().clamp(max=4095)].view(B, S, 1, D // 2)
        x = torch.cat([torch.view_as_real(pair * turn).reshape(B, S, H + kv, D), x[:, :, H + kv:]], 2)
    for b in range(B):
        n, first = int(s["count"][b]), int(s["start"][b])
        j = torch.arange(first, first + n, device="cuda")
        page = s["table"][b, j // P].long()
        if case["rope"]:
            out["q_out"].view(B, S, H * D)[b, :n] = x[b, :n, :H].reshape(n, H * D)
        for name, rows in (("k", x[b, :n, H:H + kv]), ("v", x[b, :n, H + kv:])):
            if case["fp8"]:
                mant, e = torch.frexp(rows.abs().amax(-1) / 448.0)
                e = torch.where(mant == 0.5, e - 1, torch.where(mant == 0, -126, e)).clamp(min=-126)
                unit = torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), e.double())
                out[name + "s"][page, :, j % P] = unit
                rows = (rows / unit[..., None]).float().to(torch.float8_e4m3fn).double()
            out[name][page, :, j % P] = rows
    return {n: v for n, v in out.items() if v is not None}


def _exact_gather(case, s):
    got = []
    for n in ("k", "v"):
        out = s[n + "_out"].double()
        for b, length in enumerate(s["lens"].tolist()):
            out[b, :, :length] = _exact_rows(s, b, length, n)
        got.append(out)
    return tuple(got)


def _exact_attn(case, s):
    B, H, G = case["B"], case["H"], case["G"]
    out = torch.zeros(B, H * D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        if n:
            q = s["q"][b].double().view(H // G, G, D)
            w = torch.softmax(torch.einsum("hgd,hnd->hgn", q, _exact_rows(s, b, n, "k")) / math.sqrt(D), -1)
            out[b] = torch.einsum("hgn,hnd->hgd", w, _exact_rows(s, b, n, "v")).reshape(-1)
    return out


def _exact_stats(case, s):
    R, V, k = case["R"], case["V"], min(case["k"], case["V"])
    grad = case["grad"]
    parts = []
    for a in range(0, R, 4096):
        x, t = s["logits"][a:a + 4096].double(), s["target"][a:a + 4096].long()
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        plogp = torch.where(p > 0, p * logp, 0.0)
        ent = -plogp.sum(1)
        given = (t >= 0) & (t < V)
        hit = torch.nn.functional.one_hot(t.clamp(0, V - 1), V) * given[:, None]
        part = [torch.where(given, torch.gather(logp, 1, t.clamp(0, V - 1)[:, None])[:, 0], 0.0), ent]
        if k:
            part += [torch.sort(logp, dim=1, descending=True, stable=True)[0][:, :k]]
        if grad:
            dlp, dent = s["dlp"][a:a + 4096].double()[:, None], s["dent"][a:a + 4096].double()[:, None]
            part.append(dlp * given[:, None] * (hit - p) - dent * (plogp + p * ent[:, None]))
        parts.append(part)
    got = [torch.cat(c) for c in zip(*parts)]
    return got[:2] + ([None] + got[2:3] if k else []) + (got[-1:] if grad else [])
