"""What the KV-cache backbones refuse, and what a refused or failed call leaves
behind, without a GPU: the weights are set up on the CPU and every call ends
before, or at, its first kernel."""
import pytest
import torch

from chessdecoder_b200 import engine
from chessdecoder_b200 import kernels as K
from chessdecoder_b200.decode import BatchedBackbone
from chessdecoder_b200.engine import ModelConfig
from chessdecoder_b200.paged import PagedBackbone, PagedKVCache

CFG = dict(num_layers=1)
B, S = 2, 5
IDS = torch.zeros(B, S, dtype=torch.long)


@pytest.fixture(autouse=True)
def _no_kernels(monkeypatch):
    monkeypatch.setattr(engine.K, "cast_bf16", lambda src, dst: dst.copy_(src))

    def reached(*a, **kw):
        raise MemoryError("the first kernel of a pass")
    monkeypatch.setattr(K, "fourier_features", reached)


def paged(**kw):
    return PagedBackbone(ModelConfig(**CFG), B, 32, page_size=16, device="cpu", **kw)


#: shapes that do not have a value for each of the B * S tokens
WRONG = [(B, 1), (1, S), (S,), (), (B, S - 1), (B, S + 1), (B, S, 2), (0,)]


@pytest.mark.parametrize("shape", WRONG)
@pytest.mark.parametrize("which", ["ov", "om"])
def test_prompts_refuse_overrides_of_another_size(which, shape):
    bb = paged()
    with pytest.raises(ValueError, match=which):
        bb.prefill(IDS, [S, S - 1], **{which: torch.zeros(shape)})
    assert bb.cache.lens.tolist() == bb.lengths == [0, 0] and bb.cache.free_pages == 4


@pytest.mark.parametrize("shape", [(), (1,), (B, 2), (0,), (B + 1,)])
@pytest.mark.parametrize("which", ["ov", "om"])
def test_steps_refuse_overrides_of_another_size(which, shape):
    bb = paged()
    with pytest.raises(ValueError, match=which):
        bb.step(IDS[:, :1], **{which: torch.zeros(shape)})
    assert bb.cache.lens.tolist() == bb.lengths == [0, 0] and bb.cache.free_pages == 4


@pytest.mark.parametrize("kw", [dict(ov=torch.zeros(B, 1)), dict(om=torch.zeros(B, 1)), dict(om=torch.zeros(B, S + 1)),
                                dict(pos=torch.zeros(1, S, dtype=torch.int32)), dict(pos=torch.zeros(1))])
def test_dense_backbone_refuses_arguments_shorter_than_the_tokens(kw):
    a = dict(pos=torch.arange(S).repeat(B, 1), ov=None, om=None)
    a.update(kw)
    bb = BatchedBackbone(ModelConfig(**CFG), B, 32, device="cpu")
    for call in (lambda: bb.causal_forward(IDS, a["pos"], a["ov"], a["om"], None, None),
                 lambda: bb.causal_probe(IDS, a["pos"], a["ov"], a["om"])):
        with pytest.raises(ValueError, match="tokens need as many"):
            call()
    assert bb.causal_len == 0


def test_the_right_sizes_reach_the_kernels():
    for ov, om in ((None, None), (torch.zeros(B, S), torch.zeros(B, S, dtype=torch.bool)), (torch.zeros(B * S), None)):
        with pytest.raises(MemoryError):
            paged().prefill(IDS, None, ov, om)
        with pytest.raises(MemoryError):
            BatchedBackbone(ModelConfig(**CFG), B, 32, device="cpu").causal_probe(IDS, torch.arange(S).repeat(B, 1), ov, om)
    with pytest.raises(MemoryError):
        paged().step(IDS[:, :1], torch.zeros(B), torch.zeros(B, 1))


def _passes(monkeypatch, bb):
    """The pass without its kernels, for the bookkeeping around it."""
    monkeypatch.setattr(bb, "_embed", lambda ids, ov, om: torch.zeros(ids.numel(), bb.cfg.embed_dim))
    monkeypatch.setattr(bb, "_layers_forward", lambda x, b, s, attend: x.view(b, s, -1))


def _books(bb):
    c = bb.cache
    return c.lengths, c.lens.tolist(), c.start.tolist(), c.table.tolist(), sorted(c._free), c._held


@pytest.mark.parametrize("error", [MemoryError, KeyboardInterrupt])
@pytest.mark.parametrize("times", [1, 3])
def test_a_call_that_fails_leaves_the_lengths(monkeypatch, times, error):
    """The device's lengths are moved before the pass; a pass that raises (memory that
    runs out is the ordinary way) must not leave them so: what follows is what a
    backbone without the failure does."""
    def reached(*a, **kw):
        raise error
    monkeypatch.setattr(K, "fourier_features", reached)
    bb, fresh = paged(), paged()
    tok = IDS[:, :1]

    def fail(call):
        before = _books(bb)[:2]
        for _ in range(times):
            with pytest.raises(error):
                call()
            assert _books(bb)[:2] == before
    fail(lambda: bb.prefill(IDS, [S, S - 1]))
    with monkeypatch.context() as m:
        for b in (bb, fresh):
            _passes(m, b)
            b.prefill(IDS, [S, S - 1])
        assert _books(bb) == _books(fresh) and bb.cache.lens.tolist() == [S, S - 1]
        # a replaced prompt while the other sequence keeps its tokens
        for b in (bb, fresh):
            b.release([1])
    fail(lambda: bb.prefill(IDS, [0, 3]))
    fail(lambda: bb.step(tok, active=[True, False]))
    fail(lambda: bb.generate(tok, 4, active=[True, False]))
    with monkeypatch.context() as m:
        for b in (bb, fresh):
            _passes(m, b)
            b.prefill(IDS, [0, 3])
            b.step(tok, active=[True, False])
            b.step(tok)
        assert _books(bb)[:5] == _books(fresh)[:5] and bb.cache.lens.tolist() == [S + 2, 4]


def test_a_generation_that_fails_on_its_way_counts_for_nothing(monkeypatch):
    bb = paged()
    _passes(monkeypatch, bb)
    bb.prefill(IDS, [S, 2])
    left = [2]

    def body(self, b):
        b._step_body(self.ids, None, None)
        left[0] -= 1
        if left[0] < 0:
            raise MemoryError
    from chessdecoder_b200 import paged as P
    monkeypatch.setattr(P._GenLoop, "body", body)
    with pytest.raises(MemoryError):
        bb.generate(IDS[:, :1], 6)
    assert bb.lengths == bb.cache.lens.tolist() == [S, 2]
    with pytest.raises(RuntimeError):
        bb.generate(IDS, 6)  # not one token per sequence: refused before pages are taken
    assert bb.cache.free_pages == 2


def test_a_call_that_is_cut_short_by_its_capture_can_be_made_again(monkeypatch):
    """A capture that raises leaves no half-made graph behind to be replayed."""
    from chessdecoder_b200 import paged as P
    bb = paged()
    st = P._GenLoop(bb, "board_head", None, 0.0, 0)

    class Graph:
        def replay(self):
            raise AssertionError("replayed before it was captured")

    class Capture:
        def __init__(self, graph):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *a):
            return False
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", Capture)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda dev=None: None)
    for _ in range(2):
        with pytest.raises(MemoryError):
            st.replay(bb)
        assert st.graph is None


def test_the_last_rows_are_each_sequences_own(monkeypatch):
    """value_head's default rows: a prompt's last token, not the padding behind it."""
    bb = paged()

    def run(x, b, s, attend):
        bb.last_hidden16 = torch.arange(float(b * s)).view(b, s, 1).to(torch.bfloat16)
        return bb.last_hidden16.float()
    monkeypatch.setattr(bb, "_embed", lambda ids, ov, om: None)
    monkeypatch.setattr(bb, "_layers_forward", run)
    rows = lambda: bb._last_rows().flatten().tolist()  # noqa: E731
    bb.prefill(IDS, [2, S])
    assert rows() == [1, S + S - 1]
    bb.release([0])
    bb.prefill(IDS, [4, 0])
    assert rows()[0] == 3
    bb.step(IDS[:, :1])
    assert rows() == [0, 1]
    bb.release([0, 1])
    bb.prefill(IDS)
    assert rows() == [S - 1, 2 * S - 1]
    bb.release([0, 1])
    bb.prefill(IDS, torch.tensor([1, 1]))
    assert rows() == [0, S]


def test_attention_launches_go_with_the_workspace():
    """No workspace, one kernel; and what the C entry refuses."""
    from chessdecoder_b200 import _lib
    lib = _lib.load()

    def cache(page_size=64, width=10, kv_heads=2, dtype=0, **kw):
        row = kv_heads * page_size
        c = dict(k=256, v=256, k_scale=256, v_scale=256, table=256, ldt=width, width=width, num_pages=4,
                 ld_page=row * 64, ld_scale=row, kv_heads=kv_heads, page_size=page_size, dtype=dtype, reserved=0)
        return _lib.PAGED_CACHE.pack(*{**c, **kw}.values())
    seen = set()
    for b in (1, 5, 64, 300, 700, 1600, 16384):
        for width in (1, 4, 16, 63, 128, 400):
            for p in (16, 32, 64):
                for dtype in (0, 1):
                    n = lib.cdk_paged_attn_launches(cache(p, width, dtype=dtype), b, 4)
                    need = lib.cdk_paged_attn_workspace(b, 4, 2, width * p)
                    assert n == 1 if need == 0 else n in (1, 2)
                    seen.add((n, need > 0))
    assert seen == {(1, False), (1, True), (2, True)}
    assert lib.cdk_paged_attn_launches(cache(), 0, 4) == 0 and lib.cdk_paged_attn_launches(cache(), 3, 5) == -11
    assert lib.cdk_paged_attn_launches(cache(page_size=12), 3, 4) == -4 and lib.cdk_paged_attn_launches(None, 3, 4) == -1


@pytest.mark.parametrize("seqs", [[0, 7], [2, -4], [1, 0, 3], [3]])
def test_releasing_a_sequence_that_is_not_there_releases_none(seqs):
    """The host's books and the device's table and lengths say the same afterwards."""
    c = PagedKVCache(1, 8, 3, 16, 1, page_size=4, device="cpu")
    c.reserve([4, 5, 4])
    c.advance([4, 5, 4])
    c.lens.copy_(torch.tensor([4, 5, 4]))
    before = (c.lengths, c.lens.tolist(), c.table.tolist(), c.free_pages)
    with pytest.raises(IndexError):
        c.release(seqs)
    assert (c.lengths, c.lens.tolist(), c.table.tolist(), c.free_pages) == before
    c.release([-1, 0, 0])
    assert c.lengths == c.lens.tolist() == [0, 5, 0] and c.free_pages == 6 and torch.equal(c.table, c._table)
