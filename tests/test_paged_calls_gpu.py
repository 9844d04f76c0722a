"""PagedBackbone around its calls: what a failed one leaves behind, and that a
backbone ends with its last reference.  Hidden states are held to the tolerance of
tests/test_paged_backbone_gpu.py between two backbones of the same weights."""
import gc
import weakref

import pytest
import torch

from chessdecoder_b200 import kernels as K
from chessdecoder_b200.engine import ModelConfig
from chessdecoder_b200.paged import PagedBackbone

from test_paged_backbone_gpu import near, weights

pytestmark = pytest.mark.gpu
CFG = dict(num_layers=2)


@pytest.fixture(autouse=True)
def _no_device_error():
    K.get_error()
    yield
    assert K.get_error() == 0


@pytest.mark.parametrize("use_graphs", [True, False])
def test_what_follows_a_failed_call(monkeypatch, use_graphs):
    """Prompts, steps and a generation that raise half-way, some of their kernels
    launched: the next calls answer as on a backbone that never failed."""
    cfg = ModelConfig(**CFG)
    sd = weights(cfg, 5, head=30.0)
    bb, ok = (PagedBackbone(cfg, 3, 64, page_size=16, state_dict=sd, use_graphs=use_graphs) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, cfg.vocab_size, (3, 40), generator=g)
    tok = torch.randint(0, cfg.vocab_size, (3, 1), generator=g)
    real = [12, 40, 3]

    def fail(name, after, call):
        calls, fn = [0], getattr(K, name)

        def cut(*a, **k):
            calls[0] += 1
            if calls[0] > after:
                raise MemoryError
            return fn(*a, **k)
        before = bb.lengths
        with monkeypatch.context() as m:
            m.setattr(K, name, cut)
            with pytest.raises(MemoryError):
                call()
        assert bb.lengths == bb.cache.lens.tolist() == before

    fail("attn_fwd", 1, lambda: bb.prefill(ids, real))
    fail("fourier_features", 0, lambda: bb.prefill(ids, real))
    a, b = bb.prefill(ids, real), ok.prefill(ids, real)
    for i, n in enumerate(real):
        near(a[i, :n], b[i, :n].cpu(), ("prompt", i))
    fail("paged_attn", 1, lambda: bb.step(tok))
    near(bb.step(tok), ok.step(tok).cpu(), "step")
    if use_graphs:
        fail("paged_attn", 1, lambda: bb.step(tok))  # within the capture
    near(bb.step(tok, active=[1, 0, 1]), ok.step(tok, active=[1, 0, 1]).cpu(), "second step")
    near(bb.step(tok), ok.step(tok).cpu(), "third step")
    fail("head_select", 1, lambda: bb.generate(tok, 5))  # the second step, within the capture or not
    assert bb.lengths == bb.cache.lens.tolist() == ok.lengths == [15, 42, 6]
    x, y = (c.generate(tok, 4, top_k=3) for c in (bb, ok))
    # the first choice is of one hidden state; the logits' scale is the head's
    assert (x["top_log_probs"][0] - y["top_log_probs"][0]).abs().max() < 6e-2 * y["top_log_probs"][0].abs().max() + 0.1
    assert bb.lengths == bb.cache.lens.tolist() == ok.lengths


def test_value_heads_after_prompts_of_different_lengths():
    """By default on the last token of each prompt: what its own hidden state gives."""
    cfg = ModelConfig(**CFG)
    bb = PagedBackbone(cfg, 3, 32, page_size=16, state_dict=weights(cfg, 2))
    ids = torch.randint(0, cfg.vocab_size, (3, 9), generator=torch.Generator().manual_seed(3))
    real = [9, 2, 5]
    bb.prefill(ids, real)
    mine = torch.stack([bb.last_hidden16[b, n - 1] for b, n in enumerate(real)])
    for head in ("wl_head", "d_head"):
        for got, want in zip(bb.value_head(head), bb.value_head(head, h16=mine)):
            assert torch.equal(got, want)
    bb.step(ids[:, :1])
    assert torch.equal(bb.value_head("wl_head")[3], bb.value_head("wl_head", h16=bb.last_hidden16[:, 0])[3])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("p", [16, 32, 64])
@pytest.mark.parametrize("B,Hkv,keys", [(1, 16, 137), (3, 2, 3000), (64, 16, 2000), (150, 2, 1500), (700, 2, 60),
                                        (700, 2, 200), (1600, 2, 4000), (2, 1, 0)])
def test_launches_are_counted_as_they_are(B, Hkv, keys, p, fp8):
    """One kernel where items are whole, two where partial results are joined: those
    write the workspace, the others leave it as it was, also where one is given."""
    width = -(-keys // p)  # the way goes by the table's size: sequences of 200 keys on the same pages
    n = max(min(width, 4), 1)
    table = (torch.arange(width, dtype=torch.int32, device="cuda") % n).repeat(B, 1)
    pool = torch.zeros(n, Hkv, p, 64, dtype=torch.uint8 if fp8 else torch.bfloat16, device="cuda")
    pool = pool.view(torch.float8_e4m3fn) if fp8 else pool
    s = torch.full((n, Hkv, p), 127, dtype=torch.uint8, device="cuda") if fp8 else None
    q = torch.zeros(B, Hkv * 64, dtype=torch.bfloat16, device="cuda")
    lens = torch.full((B,), min(keys, 200), dtype=torch.int32, device="cuda")
    ws = torch.full((K.paged_attn_workspace(B, Hkv, Hkv),), 0x5A, dtype=torch.uint8, device="cuda")
    before = K.LAUNCHES[0]
    K.paged_attn(q, pool, pool, table, lens, torch.empty_like(q), k_scale=s, v_scale=s, workspace=ws)
    assert K.LAUNCHES[0] - before == 1 + int((ws != 0x5A).any())


def test_a_backbone_ends_with_its_last_reference():
    """What it keeps of its graphs does not point back at it: a collection that came
    later could end a graph while another is being captured."""
    cfg = ModelConfig(**CFG)
    bb = PagedBackbone(cfg, 2, 32, page_size=16, state_dict=weights(cfg, 2))
    tok = torch.zeros(2, 1, dtype=torch.long)
    bb.prefill(torch.zeros(2, 5, dtype=torch.long), [5, 2])
    for _ in range(3):
        bb.step(tok)
    bb.generate(tok, 4, top_k=2)
    assert bb._step is not None and all(st.graph is not None for st in bb._gen.values())
    ends = [weakref.ref(x) for x in (bb, bb.cache, bb._step, *bb._gen.values())]
    gc.collect()
    gc.disable()
    try:
        del bb
        assert [r() for r in ends] == [None] * len(ends)
    finally:
        gc.enable()
