"""Which models a cache in 8 bits is for, and what becomes of the option where it has no effect."""
import dataclasses

import pytest
import torch

from art_b200.engine.factory import build_runner
from art_b200.models.config import resolve_config

CFG = dataclasses.replace(resolve_config("qwen2.5-7b"), num_heads=32, num_kv_heads=2, head_dim=128)


@pytest.mark.parametrize("kw,block_size,says", [
    (dict(num_heads=34), 16, "17 query heads to a kv head"),
    (dict(head_dim=80), 16, "head dim 80"),
    ({}, 24, "multiple of 16"),
])
@pytest.mark.parametrize("name", ["fp8", "int8", torch.int8])
def test_refused_when_the_engine_is_built(kw, block_size, says, name, monkeypatch):
    """Not at the first decode step, nor with the cache's memory taken."""
    import art_b200.engine.factory as factory

    monkeypatch.setattr(factory, "KVCache", lambda *a, **k: pytest.fail("the cache is there already"))
    with pytest.raises(ValueError, match=says):
        build_runner(dataclasses.replace(CFG, **kw), None, num_blocks=4, block_size=block_size, device="cpu", kv_dtype=name)
