"""Engines with a cache in 8 bits whose results hang on what is cached: logits and attention rows beside an engine whose bf16 cache holds
the same values, and, so that the comparison is one, beside the same engine with something wrong in its cache."""
import pytest
import torch

from .test_gpu_kv_q8_engine import DEV, KINDS, runner, slots_of, views

pytestmark = pytest.mark.gpu

# Products of two layers with about eight roundings of bf16 each, 2^-8 of a value at most, that fall differently where sums have another
# order: 16 * 2^-8.  A decode step's own token is cached in 8 bits too, off by 2^-4 of a value at most.
SAME, STEP = 2.0 ** -4, 2.0 ** -3


def weights(moe=False):
    """Attention is most of a row: values and outputs are large beside the embedding, scores far apart."""
    from art_b200.models.config import ModelConfig
    from art_b200.models.weights import init_base_weights

    kw = dict(num_experts=8, num_experts_per_tok=2, moe_intermediate_size=256, norm_topk_prob=True, qkv_bias=False) if moe else {}
    cfg = ModelConfig(name="small", vocab_size=2048, hidden_size=512, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=128,
                      intermediate_size=1024, **kw)
    base = init_base_weights(cfg, seed=2)
    for k, w in base.items():
        for name, size in (("q_proj.weight", 3), ("k_proj.weight", 3), ("v_proj.weight", 8), ("o_proj.weight", 8)):
            if k.endswith(name):
                w *= size
    return cfg, {k: v.to(torch.bfloat16) for k, v in base.items()}


def copy_cache(kv_bf, kv):
    """The values of the 8-bit cache into the bf16 cache."""
    for plain, codes, scale in zip(kv_bf.k + kv_bf.v, kv.k + kv.v, kv.k_scale + kv.v_scale):
        plain.copy_((codes.float() * scale[..., None, None]).transpose(1, 2))


def wrong(kv, how):
    """Something else in the cache's codes."""
    if how == "values":              # of other tokens of their block
        for c in kv.v:
            c.copy_(c.view(torch.uint8).flip(2).view(c.dtype))
    for c, s in zip(kv.k + kv.v, kv.k_scale + kv.v_scale):
        if how == "zeros":
            c.view(torch.uint8).zero_()
        elif how == "heads":
            c.copy_(c.view(torch.uint8).flip(1).view(c.dtype))
            s.copy_(s.flip(1))


def off(a, b):
    """Largest relative distance of two rows."""
    a, b = a.float(), b.float()
    return float(((a - b).norm(dim=-1) / b.norm(dim=-1)).max())


@KINDS
@pytest.mark.parametrize("moe", [False, True], ids=["dense", "experts"])
@pytest.mark.parametrize("lens,cached", [([60, 40], [48, 32]), ([900, 700], [608, 688]), ([48, 900, 20], [32, 640, 16])])
def test_portions(kind, moe, lens, cached):
    """The rest of prompts whose beginning is cached."""
    from dataclasses import replace

    cfg, base = weights(moe)
    bf, kv_bf = runner(cfg, dict(base), "auto")
    q8, kv = runner(cfg, dict(base), kind)
    seqs = views(lens, cached)
    q8.step_logits([replace(s, num_cached=0, upto=s.num_cached) for s in seqs], [[] for _ in seqs])
    copy_cache(kv_bf, kv)
    held = [t.clone() for t in kv.k + kv.v + kv.k_scale + kv.v_scale]
    want = [[len(s.tokens) - s.num_cached - 1] for s in seqs]
    a, b = bf.step_logits(seqs, want), q8.step_logits(seqs, want)
    assert off(b, a) <= SAME
    for how in ("zeros", "heads", "values"):
        for t, h in zip(kv.k + kv.v + kv.k_scale + kv.v_scale, held):
            t.copy_(h)
        wrong(kv, how)
        assert off(q8.step_logits(seqs, want), a) >= 4 * SAME, how
    for r in (bf, q8):
        r.close()


@KINDS
@pytest.mark.parametrize("way", ["finish", "separate", "unfused"])
@pytest.mark.parametrize("n", [3, 40])
def test_decode_steps(kind, way, n, monkeypatch):
    """Decode steps over a cache of prompts, in each of the ways that keys and values get into it: eager, captured, replayed."""
    from art_b200.ops import kv_q8

    if way == "separate":
        monkeypatch.setattr(kv_q8, "finalize_covers", lambda Hq, Hkv: False)
    if way == "unfused":
        monkeypatch.setenv("ARTB_DECODE_FUSED", "0")
    cfg, base = weights()
    bf, kv_bf = runner(cfg, dict(base), "auto", blocks=1024)
    q8, kv = runner(cfg, dict(base), kind, blocks=1024)
    lens = [33 + (13 * i) % 150 for i in range(n)]
    seqs = views(lens, blocks=1024)
    q8.prefill(seqs)
    for s in seqs:
        s.tokens = s.tokens + [(7 * s.tokens[-1] + 1) % 2048]
    copy_cache(kv_bf, kv)
    held, held_bf = ([t.clone() for t in ts] for ts in (kv.k + kv.v + kv.k_scale + kv.v_scale, kv_bf.k + kv_bf.v))

    def step(r, tensors, before, change=None):
        for t, h in zip(tensors, before):
            t.copy_(h)
        if change:
            wrong(kv, change)
        r.decode(seqs, 1)
        return next(iter(r._dstate.values()))["attn_out"][:n].clone()

    a = step(bf, kv_bf.k + kv_bf.v, held_bf)
    for _ in range(3):
        assert off(step(q8, kv.k + kv.v + kv.k_scale + kv.v_scale, held), a) <= STEP
    # the step's keys and values of the first layer are those of the bf16 engine, rounded
    at = torch.tensor([slots_of(s, len(s.tokens))[-1] for s in seqs], device=DEV)
    for plain, codes, scale in ((kv_bf.k[0], kv.k[0], kv.k_scale[0]), (kv_bf.v[0], kv.v[0], kv.v_scale[0])):
        x = plain.flatten(0, 1)[at].float()
        y = codes.view(torch.uint8)[at // 16, :, at % 16].view(codes.dtype).float() * scale[at // 16][..., None]
        assert off(y.flatten(1), x.flatten(1)) <= 2.0 ** -4 + 2.0 ** -7
    for how in ("zeros", "heads", "values"):
        assert off(step(q8, kv.k + kv.v + kv.k_scale + kv.v_scale, held, how), a) >= 4 * STEP, how
    for r in (bf, q8):
        r.close()


@KINDS
def test_prefix_hits(kind):
    """A prompt whose beginning another request left in the cache has the probabilities that it has without a prefix cache."""
    from art_b200.engine.engine import Engine, SamplingParams
    from art_b200.engine.factory import build_runner
    from art_b200.engine.kv_cache import BlockManager

    cfg, base = weights()
    g = torch.Generator().manual_seed(1)
    prefix = torch.randint(0, 2048, (208,), generator=g).tolist()
    prompt = prefix + torch.randint(0, 2048, (5,), generator=g).tolist()

    def distribution(prefix_caching, spoil=False):
        run, kv = build_runner(cfg, dict(base), num_blocks=256, device=DEV, max_loras=2, kv_dtype=kind)
        eng = Engine(run, BlockManager(256, 16, prefix_caching), eos_token_id=None, max_loras=2, kv_cache=kv)

        def go(tokens):
            seq = eng.add_request(tokens, SamplingParams(max_tokens=1, temperature=0.0, top_logprobs=20), None)
            while not seq.finished:
                eng.step()
            return seq

        go(prefix + [1])
        if spoil:
            wrong(kv, "zeros")
        seq = go(prompt)
        assert seq.prefix_hit_tokens == (208 if prefix_caching else 0)
        run.close()
        return dict(seq.top_logprobs[0])

    want, got, bad = distribution(False), distribution(True), distribution(True, spoil=True)
    # logits near the top are about 3 of their spread above the mean: a relative error of SAME + 2^-4 of a row is 2^-3 of the spread
    spread = 0.02 * 512 ** 0.5
    far = lambda d: max(abs(d[t] - want[t]) if t in d else float("inf") for t in sorted(want, key=want.get)[-5:])      # noqa: E731
    assert far(got) <= 2.0 ** -3 * 4 * spread
    assert far(bad) > far(got) * 4
