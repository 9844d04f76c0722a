"""PagedBackbone (chessdecoder_b200/paged.py): prompts of different lengths, steps
with some sequences idle, sequences that end and make room for others, and
generation with its statistics, against the oracle (one sequence at a time, so
that nothing of the paging is shared with it).

Tolerance: as tests/test_decode_gpu.py, a relative Frobenius error of 3e-2 and a
per-row cosine of 0.998.  For an e4m3 cache the rounding of a key changes scores
and so on through the layers, by more than a tolerance of the result could tell
from a mistake; so there the oracle's attention takes the rows that the cache
holds (read from its pages, as tests/paged_reference.py says what they stand
for), the hidden states are held to the same tolerance, and the cached rows are
compared with the oracle's own: they are projections of hidden states that agree
to 3e-2, rounded by at most 2^-4 of a value (and 2^-10 of a row's unit, below
2^-4 of the row's norm)."""
import numpy as np
import pytest
import torch

from chessdecoder_b200 import kernels as K
from chessdecoder_b200 import vocab as V
from chessdecoder_b200.engine import ModelConfig, init_reference_weights
from chessdecoder_b200.paged import PagedBackbone
from oracle import decode as OD

from paged_reference import rows_of, values

pytestmark = pytest.mark.gpu
CFG = dict(num_layers=3)


@pytest.fixture(autouse=True)
def _no_device_error():
    K.get_error()
    yield
    assert K.get_error() == 0


def weights(cfg, seed, head=1.0):
    sd = init_reference_weights(cfg, seed)
    for i in range(cfg.num_layers):
        for n in ("q_proj", "k_proj"):
            sd[f"layers.{i}.attn.{n}.weight"] = sd[f"layers.{i}.attn.{n}.weight"] * 4.0
    sd["board_head.weight"] = sd["board_head.weight"] * head
    return sd


class _CachedRows:
    """numpy for the oracle's module, but its joining of past and new keys and
    values (one pair per layer) gives what the product's cache holds."""

    def __init__(self, rows):
        self.rows, self.calls = rows, 0

    def __getattr__(self, name):
        return getattr(np, name)

    def concatenate(self, arrays, axis=0):
        if axis != 2:
            return np.concatenate(arrays, axis=axis)
        held = self.rows[self.calls // 2][self.calls % 2]
        self.calls += 1
        new = arrays[1][0]
        mine = held[:, held.shape[1] - new.shape[1]:]
        assert np.linalg.norm(mine - new) <= (2.0 ** -4 + 3e-2) * np.linalg.norm(new)
        return held[None]


class Ones:
    """The oracle, a cache of one sequence each; bb: a backbone whose cached rows
    its attention takes (after the backbone's own call), or None."""

    def __init__(self, sd, cfg, B, max_len, bb=None):
        w = {k: v.float().numpy() for k, v in sd.items()}
        self.w, self.bb, self.layers = w, bb, cfg.num_layers
        self.new = lambda: OD.Batched(w, dict(num_layers=cfg.num_layers, num_heads=cfg.num_heads,  # noqa: E731
                                              embed_dim=cfg.embed_dim, max_seq_len=cfg.max_seq_len), 1, max_len)
        self.seq = [self.new() for _ in range(B)]

    def run(self, b, call):
        if self.bb is None:
            return call()
        c = self.bb.cache
        rows = [[rows_of(values(x[i], s[i]), c.table, b, c.lengths[b]).float().numpy()
                 for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))] for i in range(self.layers)]
        OD.np = _CachedRows(rows)
        try:
            return call()
        finally:
            OD.np = np

    def prefill(self, b, ids, ov=None, om=None):
        o, S = self.seq[b], len(ids)
        z = np.zeros((1, S), np.float32) if ov is None else ov[None]
        m = np.zeros((1, S), bool) if om is None else om[None]
        return self.run(b, lambda: o.causal_forward(ids[None], np.arange(S)[None], z, m, np.ones(1, bool),
                                                    np.array([S])))[0]

    def step(self, b, tok, ov=0.0, om=False):
        o = self.seq[b]
        return self.run(b, lambda: o.causal_incremental(
            np.array([[tok]]), np.array([[o.causal_len]]), np.full((1, 1), ov, np.float32), np.full((1, 1), om),
            np.ones(1, bool)))[0, 0]


def near(h, ref, what):
    h, ref = h.detach().float().cpu().reshape(-1, h.shape[-1]), torch.as_tensor(ref).float().reshape(-1, h.shape[-1])
    rel = ((h - ref).norm() / ref.norm()).item()
    cos = torch.nn.functional.cosine_similarity(h, ref, dim=1).min().item()
    assert rel < 3e-2 and cos > 0.998, (what, rel, cos)


@pytest.mark.parametrize("use_graphs", [True, False])
@pytest.mark.parametrize("fp8", [False, True])
def test_prompts_steps_and_replacement(fp8, use_graphs):
    cfg = ModelConfig(**CFG)
    B, max_len, p = 4, 96, 16
    sd = weights(cfg, 3)
    pages = 16  # fewer than all four at full length need (24)
    bb = PagedBackbone(cfg, B, max_len, num_pages=pages, page_size=p, state_dict=sd, use_graphs=use_graphs,
                       kv_dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16)
    o = Ones(sd, cfg, B, max_len, bb if fp8 else None)
    rng = np.random.default_rng(4)
    real = [37, 0, 5, 64]
    ids = rng.integers(0, cfg.vocab_size, (B, 64))
    ov, om = np.zeros((B, 64), np.float32), np.zeros((B, 64), bool)
    om[0, 7], ov[0, 7] = True, 0.4
    h = bb.prefill(torch.from_numpy(ids), real, torch.from_numpy(ov), torch.from_numpy(om))
    assert bb.lengths == real and bb.cache.lens.tolist() == real
    for b, n in enumerate(real):
        if n:
            near(h[b, :n], o.prefill(b, ids[b, :n], ov[b, :n], om[b, :n]), ("prefill", b))
    # a second prompt while the others keep theirs
    more = rng.integers(0, cfg.vocab_size, (B, 20))
    h = bb.prefill(torch.from_numpy(more), torch.tensor([0, 20, 0, 0]))
    near(h[1], o.prefill(1, more[1]), "second prompt")
    for k in range(6):
        act = [True, k != 2, k % 2 == 0, True]
        tok = rng.integers(0, cfg.vocab_size, (B, 1))
        o1, m1 = np.zeros((B, 1), np.float32), np.zeros((B, 1), bool)
        if k == 3:
            m1[3], o1[3] = True, -0.7
        h = bb.step(torch.from_numpy(tok), torch.from_numpy(o1), torch.from_numpy(m1), active=act)
        for b in range(B):
            if act[b]:
                near(h[b, 0], o.step(b, tok[b, 0], o1[b, 0], m1[b, 0]), ("step", k, b))
    assert bb.lengths == bb.cache.lens.tolist() == [43, 25, 8, 70]
    # the longest game ends; another takes its place (and pages)
    free = bb.cache.free_pages
    bb.release([3])
    assert bb.cache.free_pages == free + 5 and bb.lengths == [43, 25, 8, 0]
    o.seq[3] = o.new()
    new = rng.integers(0, cfg.vocab_size, (B, 33))
    h = bb.prefill(torch.from_numpy(new), [0, 0, 0, 33])
    near(h[3], o.prefill(3, new[3]), "replacement")
    for k in range(2):
        tok = rng.integers(0, cfg.vocab_size, (B, 1))
        h = bb.step(torch.from_numpy(tok))
        for b in range(B):
            near(h[b, 0], o.step(b, tok[b, 0]), ("after", k, b))
    # a pool too small, a sequence too long: refused, nothing taken
    free, lens = bb.cache.free_pages, bb.lengths
    with pytest.raises(ValueError, match="cache full"):
        bb.cache.reserve([60, 0, 0, 0])
    with pytest.raises(ValueError, match="out of pages"):
        bb.cache.reserve([50, 60, 80, 60])
    with pytest.raises(ValueError, match="empty sequence"):
        bb.prefill(torch.from_numpy(new), [0, 3, 0, 0])
    assert (bb.cache.free_pages, bb.lengths) == (free, lens)


@pytest.mark.parametrize("use_graphs", [True, False])
def test_generation_and_its_statistics(use_graphs):
    """Greedy generation from prompts of different lengths, fed back
    teacher-forced into the oracle: each token is the oracle's argmax unless its
    top-2 margin is a near-tie (as in tests/test_decode_gpu.py); the statistics are
    those of the loop's own logits (64 bits; the tolerances of
    tests/test_token_stats_gpu.py for 41 classes are below 1e-5 here) and close to
    the oracle's."""
    cfg = ModelConfig(**CFG)
    B, max_len, n = 3, 64, 10
    sd = weights(cfg, 13, head=30.0)
    bb = PagedBackbone(cfg, B, max_len, page_size=8, state_dict=sd, use_graphs=use_graphs)
    o = Ones(sd, cfg, B, max_len)
    rng = np.random.default_rng(8)
    real = [12, 30, 3]
    ids = rng.integers(0, cfg.vocab_size, (B, 30))
    bb.prefill(torch.from_numpy(ids), real)
    for b in range(B):
        o.prefill(b, ids[b, :real[b]])
    lut = V.board_idx_to_full_idx
    first = torch.zeros(B, 1, dtype=torch.long)
    act = [True, True, False]
    got = bb.generate(first, n, lut=lut, active=act, top_k=5)
    assert bb.lengths == bb.cache.lens.tolist() == [22, 40, 3]
    assert got["ids"].shape == (n, B) and got["top_ids"].shape == (n, B, 5)
    inv = {t: i for i, t in enumerate(lut)}
    wt = o.w["board_head.weight"], o.w["board_head.bias"]
    near_ties = 0
    for b in (0, 1):
        tok = 0
        for k in range(n):
            logits = torch.from_numpy(o.step(b, tok) @ wt[0].T + wt[1]).double()
            tok = int(got["ids"][k, b])
            margin = (logits.max() - logits[inv[tok]]).item()
            assert margin < 0.02 * logits.std().item()
            near_ties += margin > 0
            logp = torch.log_softmax(logits, 0)
            # the logits agree to 3e-2 of their norm (above): so do these, to twice that of their largest
            tol = 6e-2 * logits.abs().max().item()
            assert abs(got["log_probs"][k, b].item() - logp[inv[tok]].item()) < tol
            assert abs(got["entropy"][k, b].item() + (logp.exp() * logp).sum().item()) < tol
            assert int(got["top_ids"][k, b, 0]) == tok  # greedy: the choice is the best alternative
            assert torch.equal(got["top_log_probs"][k, b, 0], got["log_probs"][k, b])
            assert (got["top_log_probs"][k, b].diff() <= 0).all()
            assert len(set(got["top_ids"][k, b].tolist())) == 5
    assert near_ties <= 2
    # the same loop again continues where it stopped
    a = bb.generate(got["ids"][-1].view(B, 1), 4, lut=lut, active=act, temperature=1.0, seed=5)
    assert "top_ids" not in a and bb.lengths == [26, 44, 3]
    # sampled: a choice has the log-probability that the alternatives give it, or is none of them.  (The
    # same seed need not give the same game: the projections' split sums are added by atomics, so logits
    # differ in their last bits from run to run.)
    bb.release([0, 1])
    bb.prefill(torch.from_numpy(ids), [12, 30, 0])
    x = bb.generate(first, 6, lut=lut, active=act, temperature=0.7, seed=9, top_k=32)
    for k in range(6):
        for b in (0, 1):
            at = (x["top_ids"][k, b] == x["ids"][k, b]).nonzero().reshape(-1)
            lp = x["log_probs"][k, b]
            assert len(at) <= 1 and int(x["ids"][k, b]) in inv
            assert lp == x["top_log_probs"][k, b, at[0]] if len(at) else lp <= x["top_log_probs"][k, b, -1]
    assert bb.generate(first, 0)["ids"].shape == (0, B)


def test_value_heads_on_a_step():
    cfg = ModelConfig(**CFG)
    sd = weights(cfg, 2)
    bb = PagedBackbone(cfg, 2, 32, page_size=16, state_dict=sd, use_graphs=False)
    bb.prefill(torch.randint(0, cfg.vocab_size, (2, 9)))
    bb.step(torch.randint(0, cfg.vocab_size, (2, 1)))
    idx, value, lp, logits = bb.value_head("wl_head")
    assert idx.shape == (2,) and logits.shape == (2, cfg.n_buckets) and torch.equal(idx, logits.argmax(1))


def test_pages_read_back_into_a_dense_cache():
    """A paged prompt read back gives the rows that the dense cache holds, up to the
    bf16 rounding of a rotation computed in another order (2^-8 of a value, and
    3 * 2^-24 * 2 of its row's largest before it)."""
    from chessdecoder_b200.decode import BatchedBackbone
    cfg = ModelConfig(num_layers=2)
    sd = weights(cfg, 6)
    ids = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(1))
    pb = PagedBackbone(cfg, 2, 64, page_size=16, state_dict=sd)
    db = BatchedBackbone(cfg, 2, 64, state_dict=sd)
    pb.prefill(ids)
    db.causal_forward(ids, torch.arange(40).repeat(2, 1), None, None, None, torch.tensor([40, 40]))
    k, v = (torch.zeros(2, 16, 64, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    K.paged_gather(lens=pb.cache.lens, k_out=k, v_out=v, **pb.cache.layer(0))
    for got, want in ((k, db.causal.k[0]), (v, db.causal.v[0])):
        got, want = got[:, :, :40].float(), want[:, :, :40].float()
        # both are roundings of values that the split sums of the projection (order of its atomics) leave
        # 2^-16 of the row's largest apart at most
        tol = 2.0 ** -7 * want.abs() + 2.0 ** -16 * want.abs().amax(-1, keepdim=True)
        assert ((got - want).abs() <= tol).all()
