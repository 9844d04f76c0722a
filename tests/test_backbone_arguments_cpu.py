"""What the KV-cache backbones refuse, and what a refused or failed call leaves
behind, without a GPU: the weights are set up on the CPU and every call ends
before, or at, its first kernel."""
import pytest
import torch

from chessdecoder_b200 import engine
from chessdecoder_b200 import kernels as K
from chessdecoder_b200.decode import BatchedBackbone
from chessdecoder_b200.engine import ModelConfig
from chessdecoder_b200.paged import PagedBackbone

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
