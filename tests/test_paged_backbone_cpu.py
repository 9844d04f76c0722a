"""The page allocator (PagedKVCache) on the CPU, and PagedBackbone's refusals."""
import random

import pytest
import torch

from chessdecoder_b200.engine import ModelConfig
from chessdecoder_b200.paged import PagedBackbone, PagedKVCache


def test_allocator_never_shares_or_loses_a_page():
    c = PagedKVCache(1, 23, 5, 40, 2, page_size=4, device="cpu")
    r = random.Random(0)
    for _ in range(500):
        if r.random() < 0.3:
            b = r.randrange(5)
            c.release([b])
        else:
            new = [r.choice([0, 0, 1, 3, 9]) for _ in range(5)]
            before = (c.lengths, c.free_pages, c._table.clone())
            try:
                c.reserve(new)
            except ValueError:
                assert before[0] == c.lengths and before[1] == c.free_pages and torch.equal(before[2], c._table)
                continue
            c.advance(new)
        held = [[p for p in row if p >= 0] for row in c.table.tolist()]
        flat = [p for h in held for p in h]
        assert sorted(flat + c._free) == list(range(23))
        assert torch.equal(c.table, c._table)
        for b in range(5):
            assert len(held[b]) * 4 >= c.lengths[b]


def test_cache_types_and_refusals():
    c = PagedKVCache(2, 3, 1, 100, 2, page_size=16, dtype=torch.float8_e4m3fn, device="cpu")
    assert c.k.shape == (2, 3, 2, 16, 64) and c.k_scale.shape == (2, 3, 2, 16) and c.table.shape == (1, 7)
    assert set(c.layer(1)) == {"k_pages", "v_pages", "table", "k_scale", "v_scale"}
    with pytest.raises(ValueError, match="out of pages"):
        c.reserve([49])
    with pytest.raises(ValueError, match="cache full"):
        c.reserve([101])
    with pytest.raises(ValueError, match="counts"):
        c.reserve([1, 2])
    for kw in (dict(page_size=12), dict(dtype=torch.float16), dict(page_size=0)):
        with pytest.raises(ValueError):
            PagedKVCache(1, 2, 1, 8, 1, device="cpu", **kw)
    with pytest.raises(ValueError):
        PagedKVCache(1, 0, 1, 8, 1, device="cpu")
    for cfg in (ModelConfig(moe_experts=4), ModelConfig(embed_dim=256, num_heads=2)):
        with pytest.raises(ValueError):
            PagedBackbone(cfg, 2, device="cpu")


def test_captured_steps_form_no_cycle():
    """What a backbone keeps of its graphs does not point back at it, so that it
    (and its graphs) end with its last reference, not in a later collection."""
    import inspect

    from chessdecoder_b200 import paged
    for cls in (paged._Captured, paged._GenLoop):
        source = inspect.getsource(cls)
        assert "self.bb" not in source and "= bb\n" not in source
