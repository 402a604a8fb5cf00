"""Operators of a paged cache of keys and values held in 8 bits, as cases to time.

A cache holds codes ``[blocks, kv heads, block size, head dim]`` (``e4m3`` or ``int8``) and a scale ``[blocks, kv heads]``, a
power of two, for keys and for values; a value is its code times the scale of its block and head.  Three operators:

``write``   the keys and values of new tokens are quantised into the cache.  The scale of a block and head is the least power of
            two that holds the largest value written to it; a token at a block's first place starts the block anew, a later
            token can only raise the scale, and then the codes that the block holds already are rounded to the new one.
``rows``    cached tokens are read back as bf16 beside the new tokens of a prompt.
``decode``  attention of one new token per sequence over the cache.

``run`` computes them from elementary operations; with ``own`` it makes the calls of :mod:`art_b200.ops.kv_q8`.  Head layouts
are those of the package's presets; lengths are those of its rollouts, conversations and long documents.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
MOST = {"e4m3": 448.0, "int8": 127.0}
LEAST = -126                # exponent of the smallest scale: a normal fp32 number
LAYOUTS = [(14, 2, 64), (16, 2, 128), (28, 4, 128), (32, 4, 128), (32, 8, 128), (40, 8, 128), (8, 8, 128), (12, 12, 64), (4, 2, 32), (16, 1, 128), (20, 2, 64)]


def listed():
    return [
        # one user of a small model: latency
        {"name": "decode-one", "op": "decode", "cache": "e4m3", "heads": 16, "kv": 2, "dim": 128, "block": 16, "seqs": 1, "lo": 777, "hi": 777},
        # the first steps of a few short chats on the smallest preset
        {"name": "decode-short", "op": "decode", "cache": "int8", "heads": 14, "kv": 2, "dim": 64, "block": 16, "seqs": 24, "lo": 1, "hi": 905},
        # many rollouts that have only begun
        {"name": "decode-begun", "op": "decode", "cache": "e4m3", "heads": 32, "kv": 4, "dim": 128, "block": 32, "seqs": 509, "lo": 1, "hi": 300},
        # the rollouts of the headline benchmark: prompts of 512 and up to 1536 new tokens
        {"name": "decode-batch", "op": "decode", "cache": "e4m3", "heads": 28, "kv": 4, "dim": 128, "block": 16, "seqs": 256, "lo": 512, "hi": 2032},
        # agents with long contexts
        {"name": "decode-agents", "op": "decode", "cache": "int8", "heads": 32, "kv": 8, "dim": 128, "block": 16, "seqs": 48, "lo": 2000, "hi": 6000},
        # three readers of documents near the longest context of the larger presets
        {"name": "decode-document", "op": "decode", "cache": "e4m3", "heads": 40, "kv": 8, "dim": 128, "block": 64, "seqs": 3, "lo": 31007, "hi": 32767},
        # the keys and values of one decode step, a token each
        {"name": "write-step", "op": "write", "cache": "e4m3", "heads": 28, "kv": 4, "dim": 128, "block": 16, "seqs": 256, "lo": 1, "hi": 1, "held": True},
        {"name": "write-one", "op": "write", "cache": "int8", "heads": 16, "kv": 2, "dim": 128, "block": 16, "seqs": 1, "lo": 1, "hi": 1, "held": True},
        # prompts of a rollout group as they arrive
        {"name": "write-prompts", "op": "write", "cache": "e4m3", "heads": 28, "kv": 4, "dim": 128, "block": 16, "seqs": 24, "lo": 130, "hi": 1100, "held": False},
        # portions of long prompts that begin and end inside blocks
        {"name": "write-portions", "op": "write", "cache": "int8", "heads": 40, "kv": 8, "dim": 128, "block": 32, "seqs": 4, "lo": 3000, "hi": 4093, "held": True},
        # the next turn of a conversation: the earlier turns from the cache, 203 new tokens
        {"name": "rows-turn", "op": "rows", "cache": "int8", "heads": 32, "kv": 8, "dim": 128, "block": 16, "seqs": 1, "lo": 1504, "hi": 1504, "new": 203},
        # a batch of turns over long prefixes
        {"name": "rows-prefixes", "op": "rows", "cache": "e4m3", "heads": 28, "kv": 4, "dim": 128, "block": 16, "seqs": 9, "lo": 1000, "hi": 6001, "new": 77},
    ]


def draw(rng: random.Random):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["decode", "decode", "decode", "write", "write", "rows"])
    heads, kv, dim = rng.choice(LAYOUTS)
    case = {"op": op, "cache": rng.choice(["e4m3", "int8"]), "heads": heads, "kv": kv, "dim": dim, "block": rng.choice([16, 16, 16, 32, 48, 64, 128])}
    token = kv * dim            # bytes of a token's keys
    if op == "decode":          # up to the bytes of the largest listed case
        most = 190_000_000 // token
        seqs = log(1, 640)
        hi = log(2, max(3, min(32768, most // seqs)))
        return {**case, "seqs": seqs, "lo": max(0, int(hi * rng.random()) - 5), "hi": hi}
    if op == "write":
        most = min(30_000, 14_000_000 // token)
        seqs = log(1, 300)
        hi = 1 if rng.random() < 0.4 else log(2, max(3, min(5000, most // seqs)))
        return {**case, "seqs": seqs, "lo": max(1, int(hi * rng.random())), "hi": hi, "held": rng.random() < 0.7}
    most = 16_000_000 // token
    seqs = log(1, 40)
    hi = log(16, max(17, min(8000, most // seqs)))
    return {**case, "seqs": seqs, "lo": max(1, int(hi * rng.random())), "hi": hi, "new": log(1, 400)}


def lengths(case) -> list[int]:
    """Lengths of the case's sequences, evenly from ``lo`` to ``hi``."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def held(case) -> list[int]:
    """Tokens that each sequence of a write has in its first blocks already."""
    return [(11 * i + 5) % (2 * case["block"]) if case["held"] else 0 for i in range(case["seqs"])]


def work(case):
    token = case["kv"] * case["dim"]
    lens = lengths(case)
    if case["op"] == "decode":
        blocks = sum(-(-n // case["block"]) for n in lens)
        size = sum(lens) * token * 2 + blocks * (case["kv"] * 8 + 4) + len(lens) * (case["heads"] * case["dim"] * 4 + 4)
        return {"bytes": size, "flops": 4 * sum(lens) * case["heads"] * case["dim"]}
    if case["op"] == "write":
        blocks = sum(-(-(h % case["block"] + n) // case["block"]) for h, n in zip(held(case), lens))
        return {"bytes": sum(lens) * (token * 6 + 4) + blocks * case["kv"] * 8, "flops": 2 * sum(lens) * token}
    rows = sum(lens) + case["seqs"] * case["new"]
    blocks = sum(-(-n // case["block"]) for n in lens)
    return {"bytes": sum(lens) * token * 2 + rows * (token * 4 + 4) + blocks * case["kv"] * 8, "flops": 2 * sum(lens) * token}


# ---------------------------------------------------------------------------------- inputs
def power_of_two(amax: torch.Tensor, most: float) -> torch.Tensor:
    """Least power of two that takes ``amax`` to ``most`` or below."""
    m, e = torch.frexp(amax)
    mm, me = math.frexp(most)
    e = torch.where(amax > 0, e - me + (m > mm).to(e.dtype), torch.full_like(e, LEAST)).clamp(min=LEAST)
    return torch.ldexp(torch.ones_like(amax), e)


def coded(x: torch.Tensor, kind: str) -> torch.Tensor:
    """``x`` rounded to codes, to the nearest, ties to even; it lies in their range."""
    return x.to(torch.float8_e4m3fn) if kind == "e4m3" else x.round().to(torch.int8)


def rows_like_keys(shape, kv: int, dim: int, g) -> torch.Tensor:
    """Values with channels of different size, as keys after a rotation have; ``shape`` ends in [kv, dim]."""
    size = torch.exp(0.5 * torch.randn(kv, dim, generator=g, device=DEV))
    return torch.randn(*shape, kv, dim, generator=g, device=DEV) * size


def cache_of(blocks: int, case, g):
    """Codes and scales of a cache whose blocks are full."""
    x = rows_like_keys((blocks, case["block"]), case["kv"], case["dim"], g).transpose(1, 2)
    x *= torch.exp(0.3 * torch.randn(blocks, case["kv"], 1, 1, generator=g, device=DEV))       # blocks of different size
    scale = power_of_two(x.abs().amax((2, 3)), MOST[case["cache"]])
    return coded(x / scale[..., None, None], case["cache"]).contiguous(), scale


def tables(lens, case, g):
    """Blocks of the sequences, in random order in a cache with a few more: ``(block table [n, width], blocks in the cache)``."""
    need = [-(-n // case["block"]) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    width = max(1, max(need))
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEV)
    at = torch.arange(width, device=DEV)[None, :]
    bt = order[(first[:, None] + at).clamp(max=total - 1)]
    return torch.where(at < torch.tensor(need, device=DEV)[:, None], bt, torch.zeros_like(bt)).contiguous(), total


def slots_of(bt, which, place, block: int) -> torch.Tensor:
    """Cache slots of the tokens ``place`` of the sequences ``which``."""
    return (bt[which, place // block] * block + place % block).to(torch.int32)


def flat_places(starts, counts):
    """``(sequence, place)`` of every token of ``counts[i]`` tokens from ``starts[i]`` on."""
    which = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    place = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, counts)])
    return which.to(DEV), place.to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = lengths(case)
    heads, kv, dim, bs = case["heads"], case["kv"], case["dim"], case["block"]
    s = {"case": case}
    if case["op"] == "decode":
        order = torch.randperm(len(lens), generator=g, device=DEV).tolist()
        lens = [lens[i] for i in order]
        s["table"], total = tables(lens, case, g)
        s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["qkv"] = torch.randn(len(lens), (heads + 2 * kv) * dim, generator=g, device=DEV).bfloat16()
        s["out"] = torch.empty(len(lens), heads * dim, dtype=torch.bfloat16, device=DEV)
        if own:
            from art_b200.ops import kv_q8

            s["workspace"] = kv_q8.decode_q8_workspace(len(lens), heads, kv, dim, DEV)
    elif case["op"] == "write":
        before = held(case)
        s["table"], total = tables([h + n for h, n in zip(before, lens)], case, g)
        which, place = flat_places(before, lens)
        s["slot"] = slots_of(s["table"], which, place, bs)
        x = torch.randn(len(place), (heads + 2 * kv) * dim, generator=g, device=DEV)
        x[:, heads * dim:(heads + kv) * dim] = rows_like_keys((len(place),), kv, dim, g).flatten(1)
        s["qkv"] = (x * torch.exp(0.4 * torch.randn(len(place), 1, generator=g, device=DEV))).bfloat16()
    else:
        s["table"], total = tables(lens, case, g)
        which, place = flat_places([0] * len(lens), [n + case["new"] for n in lens])
        limit = torch.tensor(lens, device=DEV)[which]
        slot = slots_of(s["table"], which, torch.minimum(place, limit - 1), bs)
        s["slot"] = torch.where(place < limit, slot, torch.full_like(slot, -1))
        s["rows"] = torch.zeros(len(place), (heads + 2 * kv) * dim, dtype=torch.bfloat16, device=DEV)
    s["k"], s["ks"] = cache_of(total, case, g)
    s["v"], s["vs"] = cache_of(total, case, g)
    return s


# ---------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    k_col, v_col = heads * dim, (heads + kv) * dim
    if own:
        from art_b200.ops import kv_q8

        if case["op"] == "decode":
            return kv_q8.paged_decode_q8(s["qkv"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["ctx"], heads, kv, dim, s["out"], s["workspace"])
        if case["op"] == "write":
            kv_q8.kv_write_q8(s["qkv"], k_col, v_col, s["slot"], s["k"], s["v"], s["ks"], s["vs"])
            return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}
        kv_q8.kv_rows_q8(s["k"], s["v"], s["ks"], s["vs"], s["slot"], s["rows"], k_col, v_col)
        return s["rows"][:, k_col:]
    if case["op"] == "decode":
        return plain_decode(s)
    if case["op"] == "write":
        plain_write(s["qkv"][:, k_col:v_col], s["slot"], s["k"], s["ks"], case["cache"])
        plain_write(s["qkv"][:, v_col:], s["slot"], s["v"], s["vs"], case["cache"])
        return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}
    s["rows"][:, k_col:v_col] = plain_rows(s["k"], s["ks"], s["slot"])
    s["rows"][:, v_col:] = plain_rows(s["v"], s["vs"], s["slot"])
    return s["rows"][:, k_col:]


def plain_decode(s):
    case = s["case"]
    heads, kv, dim, bs = case["heads"], case["kv"], case["dim"], case["block"]
    table, ctx = s["table"].long(), s["ctx"].long()
    n, width = table.shape

    def pages(codes, scale):        # [n, kv, tokens, dim]
        x = codes.float() * scale[..., None, None]
        return x[table].transpose(1, 2).reshape(n, kv, width * bs, dim)

    q = s["qkv"][:, :heads * dim].float().view(n, kv, heads // kv, dim) / math.sqrt(dim)
    score = q @ pages(s["k"], s["ks"]).transpose(2, 3)
    there = torch.arange(width * bs, device=q.device) < ctx[:, None]
    score = score.masked_fill(~there[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    o = (w @ pages(s["v"], s["vs"])) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    s["out"].copy_(o.reshape(n, heads * dim))
    return s["out"]


def plain_rows(codes, scale, slot):
    nb, kv, bs, dim = codes.shape
    at = slot.long().clamp(min=0)
    x = codes.view(torch.uint8)[at // bs, :, at % bs].view(codes.dtype).float() * scale[at // bs][..., None]
    return torch.where((slot >= 0)[:, None, None], x, torch.zeros_like(x)).reshape(len(slot), kv * dim).bfloat16()


def plain_write(x, slot, codes, scale, kind):
    """Quantises rows ``x`` [M, kv * dim] into ``codes`` and ``scale``, in place."""
    nb, kv, bs, dim = codes.shape
    there = slot >= 0
    x, at = x.float().view(-1, kv, dim)[there], slot.long()[there]
    block, row = torch.unique(at // bs, return_inverse=True)
    place = at % bs
    amax = torch.zeros(len(block), kv, device=x.device).index_reduce_(0, row, x.abs().amax(-1), "amax")
    new = torch.zeros(len(block), bs, dtype=torch.bool, device=x.device)
    new[row, place] = True
    anew = new[:, :1]
    old = scale[block]
    to = power_of_two(amax, MOST[kind])
    to = torch.where(anew, to, torch.maximum(to, old))
    c = codes.view(torch.uint8)[block].view(codes.dtype)                       # [touched, kv, bs, dim]
    kept = torch.where(anew, torch.ones_like(to), old / to)[..., None, None]
    c = coded(c.float() * kept, kind)
    mine = coded(x / to[row][..., None], kind).view(torch.uint8)
    c = c.view(torch.uint8)
    c[row, :, place] = mine
    codes.view(torch.uint8)[block] = c
    scale[block] = to


# ---------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    heads, kv, dim, bs = case["heads"], case["kv"], case["dim"], case["block"]
    if case["op"] == "decode":
        out = torch.zeros(case["seqs"], heads, dim, dtype=torch.float64, device=DEV)
        for i, n in enumerate(s["ctx"].tolist()):
            if n == 0:
                continue
            blocks = s["table"][i, :-(-n // bs)].long()
            take = lambda c, f: (c.view(torch.uint8)[blocks].view(c.dtype).double() * f[blocks].double()[..., None, None]).transpose(0, 1).reshape(kv, -1, dim)[:, :n]  # noqa: E731
            q = s["qkv"][i, :heads * dim].double().view(kv, heads // kv, dim)
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, take(s["k"], s["ks"])) / dim ** 0.5, -1)
            out[i] = torch.einsum("hgn,hnd->hgd", p, take(s["v"], s["vs"])).reshape(heads, dim)
        return out.flatten(1)
    if case["op"] == "rows":
        slot = s["slot"].tolist()
        have = torch.tensor([i for i, t in enumerate(slot) if t >= 0], device=DEV)
        t = torch.tensor([t for t in slot if t >= 0], device=DEV)
        out = torch.zeros(len(slot), 2, kv, dim, dtype=torch.float64, device=DEV)
        for j, (c, f) in enumerate(((s["k"], s["ks"]), (s["v"], s["vs"]))):
            out[have, j] = c.double().permute(0, 2, 1, 3).reshape(-1, kv, dim)[t] * f.double().repeat_interleave(bs, 0)[t][..., None]
        return out.flatten(1)
    of = {}
    for row, t in enumerate(s["slot"].tolist()):
        of.setdefault(t // bs, []).append((row, t % bs))
    found = {}
    for j, name in enumerate("kv"):
        codes, scale = s[name].double().cpu(), s[name + "s"].double().cpu()
        x = s["qkv"][:, (heads + j * kv) * dim:(heads + (j + 1) * kv) * dim].double().cpu().view(-1, kv, dim)
        for b, members in of.items():
            rows, places = [r for r, _ in members], [p for _, p in members]
            top = x[rows].abs().amax((0, 2))
            f = torch.tensor([2.0 ** max(LEAST, math.ceil(math.log2(t / MOST[case["cache"]]))) if t > 0 else 2.0 ** LEAST for t in top.tolist()], dtype=torch.float64)
            if 0 not in places:
                f = torch.maximum(f, scale[b])
                codes[b] = nearest(codes[b] * (scale[b] / f)[:, None, None], case["cache"])
            codes[b][:, places] = nearest(x[rows] / f[:, None], case["cache"]).transpose(0, 1)
            scale[b] = f
        found[name], found[name + "_scale"] = codes if case["cache"] == "e4m3" else codes.to(torch.int8), scale
    return found


def nearest(x: torch.Tensor, kind: str) -> torch.Tensor:
    """Nearest number of the format, ties to even, in 64 bits."""
    if kind == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)          # 3 bits of fraction, none below 2^-9
    return torch.round(x / step) * step
