"""Engines whose cache is held in 8 bits, beside engines with a bf16 cache of the same weights."""
import pytest
import torch

from .kv_q8_oracle import Cache, attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = pytest.mark.parametrize("kind", ["fp8", "int8"])


def weights(hd=128, qk_norm=False, layers=2):
    from art_b200.models.config import ModelConfig
    from art_b200.models.weights import init_base_weights

    cfg = ModelConfig(name="small", vocab_size=2048, hidden_size=512, num_layers=layers, num_heads=4, num_kv_heads=2, head_dim=hd,
                      intermediate_size=1024, qk_norm=qk_norm, qkv_bias=not qk_norm)
    base = {k: v.to(torch.bfloat16) for k, v in init_base_weights(cfg, seed=0).items()}
    # a token's embedding is most of its hidden row and the head points from it to the next token: draws are decided
    emb = torch.randn(cfg.vocab_size, cfg.hidden_size, generator=torch.Generator().manual_seed(5))
    base["model.embed_tokens.weight"] = (emb * 4).bfloat16()
    base["lm_head.weight"] = (emb.roll(1, 0) * 20 / cfg.hidden_size).bfloat16()
    return cfg, base


def runner(cfg, base, kind, blocks=256, bs=16):
    from art_b200.engine.factory import build_runner

    return build_runner(cfg, base, num_blocks=blocks, block_size=bs, device=DEV, max_loras=2, kv_dtype=kind)


def views(lens, cached=None, bs=16, seed=3, extra=2, blocks=256):
    from art_b200.engine.runner import SeqView

    g = torch.Generator().manual_seed(seed)
    order = iter(torch.randperm(blocks, generator=g).tolist())
    out = []
    for i, n in enumerate(lens):
        toks = torch.randint(0, 2048, (n,), generator=g).tolist()
        out.append(SeqView(toks, cached[i] if cached else 0, [next(order) for _ in range((n + 16 * extra) // bs + 1)], -1, 0.0, 0, 0))
    return out


def slots_of(s, n, bs=16):
    return [s.blocks[t // bs] * bs + t % bs for t in range(n)]


@KINDS
@pytest.mark.parametrize("lens,hd,qk_norm", [([37, 5, 64], 128, False), ([700, 33], 128, False), ([300, 17], 64, True)])
def test_prompts_fill_the_cache(kind, lens, hd, qk_norm):
    """Whole prompts: every layer's cache is the bf16 engine's, rounded.  Both engines' products are the same up to the order of
    their partial sums, which turns some bf16 roundings: one step, 2^-7 of a value, and what later layers make of it."""
    cfg, base = weights(hd, qk_norm)
    bf, kv_bf = runner(cfg, dict(base), "auto")
    q8, kv = runner(cfg, dict(base), kind)
    seqs = views(lens)
    t0, t1 = bf.prefill(seqs)[0], q8.prefill(seqs)[0]
    assert t0 == t1 == [(s.tokens[-1] + 1) % 2048 for s in seqs]
    for li in range(cfg.num_layers):
        for plain, codes, scale in ((kv_bf.k[li], kv.k[li], kv.k_scale[li]), (kv_bf.v[li], kv.v[li], kv.v_scale[li])):
            c = Cache(codes, scale)
            for s, n in zip(seqs, lens):
                slots = slots_of(s, n)
                x = plain.flatten(0, 1)[torch.tensor(slots, device=DEV)].double().cpu()
                y = c.tokens(slots)
                step = c.scale[torch.tensor(slots) // 16][..., None]
                half = step * 0.5 if kind == "int8" else torch.maximum(x.abs() * 2 ** -4, step * 2 ** -10)
                if li == 0:
                    assert ((y - x).abs() <= half * 1.02 + x.abs() * 2 ** -7 + 1e-9).all()
                assert (y - x).norm() <= half.norm() * 1.02 + 2 ** -6 * x.norm()
    for r in (bf, q8):
        r.close()


@KINDS
@pytest.mark.parametrize("lens,cached", [([60, 40], [32, 16]), ([900, 700], [304, 16]), ([48, 900, 20], [32, 0, 16])])
def test_portions_attend_to_the_cache_as_it_is(kind, lens, cached):
    """The second portion of a prompt: the same logits as those of the bf16 engine whose cache holds the 8-bit cache's values."""
    cfg, base = weights()
    bf, kv_bf = runner(cfg, dict(base), "auto")
    q8, kv = runner(cfg, dict(base), kind)
    seqs = views(lens, cached)
    first = [s for s in seqs if s.num_cached]
    from dataclasses import replace

    q8.step_logits([replace(s, num_cached=0, upto=s.num_cached) for s in first], [[] for _ in first])
    for li in range(cfg.num_layers):
        for plain, codes, scale in ((kv_bf.k[li], kv.k[li], kv.k_scale[li]), (kv_bf.v[li], kv.v[li], kv.v_scale[li])):
            plain.copy_((codes.float() * scale[..., None, None]).transpose(1, 2))
    want = [[len(s.tokens) - s.num_cached - 1, 0] for s in seqs]
    a, b = bf.step_logits(seqs, want), q8.step_logits(seqs, want)
    # where the bf16 engine reads its new keys and values back they are the same numbers; sums in any order turn bf16 roundings
    assert (a - b).norm() <= 2 ** -6 * a.norm()
    for r in (bf, q8):
        r.close()


@KINDS
@pytest.mark.parametrize("finish", [True, False], ids=["finish", "separate"])
@pytest.mark.parametrize("n,hd,qk_norm", [(5, 128, False), (40, 64, True), (200, 128, False)])
def test_decode_steps(kind, n, hd, qk_norm, finish, monkeypatch):
    """A decode step quantises the keys and values it computes into the cache, and its last layer's attention is that of its queries
    over that cache; eager, captured and replayed.  Longer runs draw the tokens that the bf16 engine draws."""
    from art_b200.ops import kv_q8

    if not finish:       # as with an odd number of heads: rows are finished in bf16 and quantised by a launch of their own
        monkeypatch.setattr(kv_q8, "finalize_covers", lambda Hq, Hkv: False)
    cfg, base = weights(hd, qk_norm, layers=2)
    lens = [3 + (7 * i) % 60 for i in range(n)]
    q8, kv = runner(cfg, dict(base), kind, blocks=2048)
    bf, kv_bf = runner(cfg, dict(base), "auto", blocks=2048)
    seqs = views(lens, blocks=2048)
    for r in (bf, q8):
        r.prefill(seqs)
    toks = [s.tokens for s in seqs]
    for s, t in zip(seqs, toks):
        s.tokens = t + [(t[-1] + 1) % 2048]
    held = [t.clone() for t in kv.k + kv.v + kv.k_scale + kv.v_scale]
    for use in range(3):
        for t, h in zip(kv.k + kv.v + kv.k_scale + kv.v_scale, held):
            t.copy_(h)
        ids, _ = q8.decode(seqs, 1)
        assert ids[0] == [(s.tokens[-1] + 1) % 2048 for s in seqs]
        st = next(iter(q8._dstate.values()))
        li, w = cfg.num_layers - 1, cfg.kv_size
        slots = [s.blocks[(len(s.tokens) - 1) // 16] * 16 + (len(s.tokens) - 1) % 16 for s in seqs]
        caches = []
        for j, (codes, scale, before) in enumerate(((kv.k[li], kv.k_scale[li], (held[li], held[4 + li])),
                                                     (kv.v[li], kv.v_scale[li], (held[2 + li], held[6 + li])))):
            now = Cache(codes, scale)
            if not finish:
                o = Cache(*before)
                o.write(st["kv_rows"][:n, j * w:(j + 1) * w], slots)
                assert torch.equal(now.codes, o.codes) and torch.equal(now.scale, o.scale)
            caches.append(now)
        for i in range(0, n, max(1, n // 10)):
            at = slots_of(seqs[i], len(seqs[i].tokens))
            ref, bound = attend(st["q"][i].double().cpu().view(cfg.num_heads, hd), caches[0].tokens(at), caches[1].tokens(at), caches[0].dtype)
            assert ((st["attn_out"][i].double().cpu().view(cfg.num_heads, hd) - ref).abs() <= bound).all()
    a, b = q8.decode(seqs, 16)[0], bf.decode(seqs, 16)[0]
    assert a == b
    for r in (bf, q8):
        r.close()


def test_unfused_steps(monkeypatch):
    """The path of replicas that the finish kernels do not cover."""
    monkeypatch.setenv("ARTB_DECODE_FUSED", "0")
    cfg, base = weights()
    q8, kv = runner(cfg, dict(base), "fp8")
    seqs = views([37, 5, 64])
    assert q8.prefill(seqs)[0] == [(s.tokens[-1] + 1) % 2048 for s in seqs]
    for s in seqs:
        s.tokens = s.tokens + [(s.tokens[-1] + 1) % 2048]
    for _ in range(3):
        ids = q8.decode(seqs, 4)[0]
        assert ids == [[(s.tokens[-1] + 1 + k) % 2048 for s in seqs] for k in range(4)]
    q8.close()


@KINDS
@pytest.mark.parametrize("use_arena", [True, False])
def test_engine_with_prefix_hits_and_sleep(kind, use_arena):
    from art_b200.engine.engine import Engine, SamplingParams
    from art_b200.engine.kv_cache import BlockManager
    from art_b200.engine.factory import build_runner

    cfg, base = weights()
    run, kv = build_runner(cfg, base, num_blocks=256, device=DEV, max_loras=2, use_arena=use_arena, kv_dtype=kind)
    eng = Engine(run, BlockManager(256, 16, True), eos_token_id=None, max_loras=2, num_scheduler_steps=4, kv_cache=kv,
                 max_num_batched_tokens=64)                      # prompts come in portions
    p = SamplingParams(max_tokens=20, temperature=0.0)
    prompts = [list(range(5, 205)), list(range(100, 117)), [7, 8, 9]]

    def go(prs):
        seqs = [eng.add_request(pr, p, None) for pr in prs]
        while not all(s.finished for s in seqs):
            eng.step()
        eng.step()
        assert [s.output_ids for s in seqs] == [[(pr[-1] + 1 + k) % 2048 for k in range(20)] for pr in prs]

    go(prompts)
    go(prompts)
    assert eng.bm.stats()["prefix_hits"] >= 1
    ptrs = [t.data_ptr() for t in kv.k + kv.v + kv.k_scale + kv.v_scale]
    for level in (1, 2):
        live = eng.add_request(list(range(200, 240)), p, None)
        eng.step()
        before = [t.clone() for t in kv.k + kv.v + kv.k_scale + kv.v_scale]
        eng.sleep(level)
        assert not kv.resident and not kv.k_scale
        eng.wake_up()
        torch.cuda.synchronize()
        if use_arena:
            assert [t.data_ptr() for t in kv.k + kv.v + kv.k_scale + kv.v_scale] == ptrs
        if level == 1:
            assert all(torch.equal(a.double(), b.double()) for a, b in zip(before, kv.k + kv.v + kv.k_scale + kv.v_scale))
        while not live.finished:
            eng.step()
        assert live.output_ids == [240 + k for k in range(20)]
        go(prompts)
    run.close()
