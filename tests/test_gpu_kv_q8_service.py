"""A model service whose engine_args ask for a cache in 8 bits: its engine, its budget, sleep and training steps between rollouts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ARCH = dict(name="small", vocab_size=2048, hidden_size=512, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=128, intermediate_size=1024)


def service(tmp_path, **engine_args):
    import art_b200 as art
    from art_b200.local.service import ModelState

    config = art.dev.get_model_config("random:small", str(tmp_path), {"init_args": {"architecture": ARCH, "max_seq_length": 2048}, "engine_args": engine_args})
    return ModelState("random:small", config, str(tmp_path))


def greedy(state, prompts, tokens=24):
    from art_b200.engine.engine import SamplingParams

    seqs = [state.engine.add_request(p, SamplingParams(max_tokens=tokens, temperature=0.0, ignore_eos=True), None) for p in prompts]
    while not all(s.finished for s in seqs):
        state.engine.step()
    return [s.output_ids for s in seqs]


@pytest.mark.parametrize("name,dtype", [("fp8", torch.float8_e4m3fn), ("int8", torch.int8), ("auto", torch.bfloat16), ("fp8_e5m2", torch.bfloat16)])
def test_the_option_reaches_the_cache(name, dtype, tmp_path):
    from art_b200.engine.kv_cache import KVCache

    state = service(tmp_path, kv_cache_dtype=name, num_gpu_blocks_override=256, enable_sleep_mode=True)
    assert state.kv.dtype == dtype and state.kv.shape == (256, 16, 2, 128)
    layers = [t for layer in zip(state.kv.k, state.kv.v, *((state.kv.k_scale, state.kv.v_scale) if state.kv.quantised else ())) for t in layer]
    assert sum(t.nbytes for t in layers) == 256 * KVCache.bytes_per_block(2, 16, 2, 128, dtype.itemsize)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (200, 37, 5)]
    first = greedy(state, prompts)
    assert all(len(o) == 24 for o in first) and (not state.kv.quantised or any(bool(s.any()) for s in state.kv.k_scale))
    for level in (1, 2):
        state.engine.sleep(level)
        state.engine.wake_up()
        again = greedy(state, [p[:-1] + [7] for p in prompts])
        assert all(len(o) == 24 for o in again)
    state.close()


def test_twice_the_tokens_in_the_same_memory(tmp_path, monkeypatch):
    blocks = {}
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a, **k: (1 << 30, 1 << 30))
    for name in ("auto", "fp8", "int8"):
        state = service(tmp_path / name, kv_cache_dtype=name, gpu_memory_utilization=0.5)
        blocks[name] = state.kv.shape[0]
        assert sum(t.nbytes for t in state.kv.k + state.kv.v + state.kv.k_scale + state.kv.v_scale) <= 1 << 28
        assert all(len(o) == 24 for o in greedy(state, [list(range(30))]))
        state.close()
    assert blocks["fp8"] == blocks["int8"] and 1.99 * blocks["auto"] < blocks["fp8"] <= 2 * blocks["auto"]
