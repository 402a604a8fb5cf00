"""The choice of the cache's number format: names, sizes, refusals."""
import pytest
import torch

from art_b200.engine.factory import build_runner, cache_bytes
from art_b200.engine.kv_cache import KV_CACHE_DTYPES, KVCache, kv_cache_dtype
from art_b200.models.config import ModelConfig, resolve_config

CPU = torch.device("cpu")


def test_names():
    assert kv_cache_dtype(None) == kv_cache_dtype("auto") == kv_cache_dtype("bfloat16") == torch.bfloat16
    assert kv_cache_dtype("fp8") == kv_cache_dtype("fp8_e4m3") == torch.float8_e4m3fn and kv_cache_dtype("int8") == torch.int8
    assert all(kv_cache_dtype(t) == t for t in KV_CACHE_DTYPES.values())
    for name in ("fp8_e5m2", "int4", "", torch.float16):
        with pytest.raises(ValueError, match="kv_cache_dtype|supported"):
            kv_cache_dtype(name if name != "" else "none")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn, torch.int8])
def test_layout_and_sleep(dtype):
    kv = KVCache(2, 6, 32, 3, 64, CPU, dtype)
    assert kv.shape == (6, 32, 3, 64) and kv.resident and kv.quantised == (dtype != torch.bfloat16)
    layers = list(zip(kv.k, kv.v, kv.k_scale, kv.v_scale)) if kv.quantised else list(zip(kv.k, kv.v))
    assert sum(t.nbytes for layer in layers for t in layer) == 6 * KVCache.bytes_per_block(2, 32, 3, 64, dtype.itemsize)
    for i, t in enumerate(t for layer in layers for t in layer):
        t.copy_(torch.full(t.shape, float(i + 1)).to(t.dtype))
    kv.offload()
    assert not kv.resident
    kv.restore()
    layers = list(zip(kv.k, kv.v, kv.k_scale, kv.v_scale)) if kv.quantised else list(zip(kv.k, kv.v))
    assert [float(t.float().mean()) for layer in layers for t in layer] == [float(i + 1) for i in range(len(layers) * len(layers[0]))]
    kv.discard()
    kv.restore()
    assert not any(t.float().any() for t in kv.k + kv.v + kv.k_scale + kv.v_scale)


def test_memory_of_a_block():
    cfg = resolve_config("qwen2.5-7b")
    bf, _ = cache_bytes(cfg, 16)
    for name in ("fp8", "int8"):
        q8, _ = cache_bytes(cfg, 16, kv_dtype=name)
        assert q8 == bf // 2 + 2 * cfg.num_layers * cfg.num_kv_heads * 4 and q8 < 0.502 * bf


def test_refusals():
    with pytest.raises(ValueError, match="multiple of 16"):
        KVCache(1, 4, 8, 2, 64, CPU, torch.int8)
    with pytest.raises(ValueError, match="head dim 80"):
        KVCache(1, 4, 16, 2, 80, CPU, torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="hybrid models"):
        build_runner(resolve_config("gaborax-tiny"), None, num_blocks=4, device="cpu", kv_dtype="fp8")
    with pytest.raises(ValueError, match="fp8_e5m2"):
        build_runner(ModelConfig(), None, num_blocks=4, device="cpu", kv_dtype="fp8_e5m2")


def test_engine_argument_is_acted_on():
    from art_b200.dev.engine import split_engine_args

    assert "kv_cache_dtype" in split_engine_args({"kv_cache_dtype": "fp8"})[0]
