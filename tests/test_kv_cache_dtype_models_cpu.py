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


ARCH = dict(name="tiny", vocab_size=512, hidden_size=64, num_layers=1, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128)


@pytest.mark.parametrize("name,says", [(None, None), ("auto", None), ("bfloat16", None), ("fp8", "head dim 16"), ("fp8_e5m2", "fp8_e5m2"), ("float16", "float16"),
                                       (["fp8"], "supported are")])
def test_a_service_runs_whatever_the_option_says(name, says, tmp_path, caplog):
    """Configurations name formats of other engines, and models that a cache in 8 bits does not take: a warning, as before the option
    had an effect."""
    import art_b200 as art
    from art_b200.local.service import ModelState

    config = art.dev.get_model_config("random:tiny", str(tmp_path), {"init_args": {"architecture": ARCH}, "engine_args": {"kv_cache_dtype": name}})
    with caplog.at_level("WARNING"):
        state = ModelState("random:tiny", config, str(tmp_path))
    told = [r.getMessage() for r in caplog.records if "kv_cache_dtype" in r.getMessage()]
    assert not told if says is None else len(told) == 1 and says in told[0]
    state.close()


@pytest.mark.skipif(torch.cuda.is_available(), reason="what becomes of it without a GPU")
def test_no_cache_on_the_cpu(tmp_path, caplog):
    import art_b200 as art
    from art_b200.local.service import ModelState

    config = art.dev.get_model_config("random:tiny", str(tmp_path), {"init_args": {"architecture": {**ARCH, "head_dim": 32}}, "engine_args": {"kv_cache_dtype": "fp8"}})
    with caplog.at_level("WARNING"):
        state = ModelState("random:tiny", config, str(tmp_path))
    assert any("keep no cache" in r.getMessage() for r in caplog.records)
    state.close()
