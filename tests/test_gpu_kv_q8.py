"""A paged cache in 8 bits on the GPU: writes, read-back and decode attention against their definitions in 64 bits."""
import random

import pytest
import torch

from .kv_q8_oracle import Cache, attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4, I8 = torch.float8_e4m3fn, torch.int8
KINDS = pytest.mark.parametrize("dtype", [E4, I8], ids=["e4m3", "int8"])


def empty(nb, kv, bs, hd, dtype, dev=DEV):
    c = lambda: torch.zeros(nb, kv, bs, hd, dtype=dtype, device=dev)      # noqa: E731
    return c(), c(), torch.zeros(nb, kv, device=dev), torch.zeros(nb, kv, device=dev)


def same(cache, k: Cache, v: Cache):
    for c, s, o in ((cache[0], cache[2], k), (cache[1], cache[3], v)):
        assert torch.equal(s.double().cpu().nan_to_num(nan=-1.0), o.scale.nan_to_num(nan=-1.0))
        assert torch.equal(c.double().cpu(), o.codes)


def keys(M, kv, hd, g, spread=0.7, extra=0):
    """bf16 [M, (extra | k | v)] with rows and channels of different size."""
    x = torch.randn(M, extra + 2 * kv * hd, generator=g, device=DEV)
    x *= torch.exp(spread * torch.randn(M, 1, generator=g, device=DEV)) * torch.exp(spread * torch.randn(1, x.shape[1], generator=g, device=DEV))
    return x.bfloat16()


def write(x, extra, slots, cache, oracles, kv, hd):
    from art_b200.ops import kv_q8

    w = kv * hd
    kv_q8.kv_write_q8(x, extra, extra + w, torch.tensor(slots, dtype=torch.int32, device=DEV), *cache)
    oracles[0].write(x[:, extra:extra + w], slots)
    oracles[1].write(x[:, extra + w:extra + 2 * w], slots)


def oracles_of(cache):
    return Cache(cache[0], cache[2]), Cache(cache[1], cache[3])


@KINDS
@pytest.mark.parametrize("kv,hd,bs,portions", [
    (2, 64, 16, [1]),
    (2, 128, 16, [16, 16, 1]),
    (4, 128, 16, [5, 11, 3, 40, 1, 1]),            # portions that begin and end inside blocks
    (1, 32, 16, [33, 31, 1, 62]),
    (3, 64, 48, [47, 2, 95, 1]),                   # blocks that are no power of two, more than one batch of rows
    (8, 128, 128, [130, 7, 250]),
    (5, 128, 32, [1] * 37),                        # token by token
])
def test_writes_of_one_sequence(dtype, kv, hd, bs, portions):
    g = torch.Generator(device=DEV).manual_seed(kv * hd + bs)
    nb = sum(portions) // bs + 3
    order = torch.randperm(nb, generator=torch.Generator().manual_seed(3)).tolist()
    cache = empty(nb, kv, bs, hd, dtype)
    o = oracles_of(cache)
    at = 0
    for n in portions:
        x = keys(n, kv, hd, g, extra=16)
        write(x, 16, [order[(at + i) // bs] * bs + (at + i) % bs for i in range(n)], cache, o, kv, hd)
        at += n
    same(cache, *o)


@KINDS
def test_writes_of_a_batch(dtype):
    """Several sequences' portions beside rows that are not written, over blocks that others have used."""
    g = torch.Generator(device=DEV).manual_seed(1)
    kv, hd, bs, nb = 4, 64, 16, 40
    cache = empty(nb, kv, bs, hd, dtype)
    o = oracles_of(cache)
    full = keys(nb * bs, kv, hd, g)
    write(full, 0, list(range(nb * bs)), cache, o, kv, hd)
    same(cache, *o)
    slots = []
    for blocks, start, n in (([3, 9, 4], 5, 30), ([7], 0, 1), ([11, 2], 16, 9), ([30, 31, 32], 0, 48), ([5], 15, 1), ([6], 3, 12)):
        slots += [-1] * (n % 3) + [blocks[(start + i) // bs] * bs + (start + i) % bs for i in range(n)]
    for scale in (0.01, 30.0):                     # into blocks of larger and of smaller values
        write((keys(len(slots), kv, hd, g).float() * scale).bfloat16(), 0, slots, cache, o, kv, hd)
        same(cache, *o)
    # a decode step: one token per sequence, each at its own place of its own block
    step = [b * bs + (7 * b) % bs for b in range(20)] + [-1] * 4
    write(keys(len(step), kv, hd, g, extra=64), 64, step, cache, o, kv, hd)
    same(cache, *o)
    # the same step again changes nothing
    before = [t.clone() for t in cache]
    x = keys(len(step), kv, hd, g)
    write(x, 0, step, cache, o, kv, hd)
    write(x, 0, step, cache, o, kv, hd)
    same(cache, *o)
    assert not torch.equal(cache[0].double(), before[0].double())
    assert torch.equal(cache[0][36:].double(), before[0][36:].double())        # blocks that no row names


@KINDS
@pytest.mark.parametrize("kv,hd,bs", [(2, 128, 48), (3, 64, 64), (1, 32, 128), (2, 128, 160), (2, 64, 32), (1, 128, 32)])
@pytest.mark.parametrize("many", [False, True])
def test_writes_of_long_runs(dtype, kv, hd, bs, many):
    """More rows than a step has, into long blocks: runs of every length beside one another, from any place of a block on, that begin
    at any row of the call, rows that are not written between them, and a second call that goes on in the same blocks with values
    that raise the scales of some."""
    g = torch.Generator(device=DEV).manual_seed(kv * hd + bs)
    r = random.Random(bs + hd)
    lens = [1, 2, 15, 16, 17, 18, 31, 32, 33, 47, 48, 49, 63, 64, 65, 1, 1, 1, 96, 127, 128, 129, 160]
    lens = [min(n, bs) for n in lens] + ([bs] * (2300 // bs) if many else [])
    r.shuffle(lens)
    nb = len(lens) + 2
    cache = empty(nb, kv, bs, hd, dtype)
    o = oracles_of(cache)
    full = keys(nb * bs, kv, hd, g, spread=0.2)
    write(full, 0, list(range(nb * bs)), cache, o, kv, hd)
    for size in (0.02, 1.0, 40.0):
        slots, blocks = [], list(range(len(lens)))
        r.shuffle(blocks)
        for b, n in zip(blocks, lens):
            at = r.choice([0, bs - n, r.randint(0, bs - n)])
            slots += [-1] * r.choice([0, 0, 1, 3]) + [b * bs + at + i for i in range(n)]
        assert len(slots) > (2048 if many else 256)
        write((keys(len(slots), kv, hd, g, extra=8).float() * size).bfloat16(), 8, slots, cache, o, kv, hd)
        same(cache, *o)


@KINDS
def test_a_step_into_long_blocks(dtype):
    """A token each of more sequences than a warp per row is for."""
    g = torch.Generator(device=DEV).manual_seed(5)
    kv, hd, bs, n = 2, 64, 64, 301
    cache = empty(n + 2, kv, bs, hd, dtype)
    o = oracles_of(cache)
    write(keys((n + 2) * bs, kv, hd, g, spread=0.2), 0, list(range((n + 2) * bs)), cache, o, kv, hd)
    step = [b * bs + (7 * b) % bs for b in range(n)]
    write(keys(n, kv, hd, g), 0, step, cache, o, kv, hd)
    same(cache, *o)


@KINDS
def test_long_rows_of_a_prompt(dtype):
    g = torch.Generator(device=DEV).manual_seed(2)
    kv, hd, bs, M = 2, 128, 16, 5003
    cache = empty(M // bs + 2, kv, bs, hd, dtype)
    o = oracles_of(cache)
    write(keys(M, kv, hd, g), 0, [i + 5 for i in range(M)], cache, o, kv, hd)
    same(cache, *o)


@KINDS
def test_extreme_values(dtype):
    """Zeros, the largest and smallest numbers of bf16, the borders between two scales and of rounding."""
    kv, hd, bs = 1, 64, 16
    big = torch.finfo(torch.bfloat16).max
    rows = [0.0, 2.0 ** -133, 2.0 ** -126, 1.75, 1.7578125, 1.984375, 1.9921875, 448.0, 450.0, 127.0, 127.5, big, -big, 2.0 ** -120]
    cache = empty(len(rows), kv, bs, hd, dtype)
    o = oracles_of(cache)
    x = torch.zeros(len(rows), 2 * hd, device=DEV)
    x[:, ::3] = torch.tensor(rows, device=DEV)[:, None]
    x[:, 1::3] = torch.tensor(rows, device=DEV)[:, None] * torch.linspace(-1, 1, len(x[0, 1::3]), device=DEV)
    write(x.bfloat16(), 0, [b * bs for b in range(len(rows))], cache, o, kv, hd)
    same(cache, *o)
    write((x * 2).clamp(-big, big).bfloat16(), 0, [b * bs + 1 for b in range(len(rows))], cache, o, kv, hd)
    same(cache, *o)


@KINDS
def test_values_that_are_not_finite(dtype):
    """A block and head that received one reads as NaN until it starts anew; other heads and blocks do not notice."""
    from art_b200.ops import kv_q8

    kv, hd, bs = 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(5)
    cache = empty(4, kv, bs, hd, dtype)
    o = oracles_of(cache)
    write(keys(40, kv, hd, g), 0, list(range(40)), cache, o, kv, hd)
    x = keys(2, kv, hd, g)
    x[0, 3], x[1, kv * hd + hd + 1] = float("inf"), float("nan")       # key head 0 of the first row, value head 1 of the second
    write(x, 0, [40, 41], cache, o, kv, hd)
    same(cache, *o)
    write(keys(1, kv, hd, g), 0, [42], cache, o, kv, hd)               # stays
    same(cache, *o)
    dst = torch.zeros(43, 2 * kv * hd, dtype=torch.bfloat16, device=DEV)
    kv_q8.kv_rows_q8(*cache, torch.arange(43, dtype=torch.int32, device=DEV), dst, 0, kv * hd)
    nan = dst.isnan().view(43, 2, kv, hd)
    assert nan[32:, 0, 0].all() and nan[32:, 1, 1].all() and not nan[:32].any() and not nan[:, 0, 1].any() and not nan[:, 1, 0].any()
    write(keys(3, kv, hd, g), 0, [32, 33, 34], cache, o, kv, hd)       # the block starts anew
    same(cache, *o)
    assert not cache[2].isnan().any() and not cache[3].isnan().any()


@KINDS
@pytest.mark.parametrize("kv,hd,bs", [(2, 64, 16), (4, 128, 16), (3, 32, 48), (8, 128, 64)])
def test_rows(dtype, kv, hd, bs):
    from art_b200.ops import kv_q8

    g = torch.Generator(device=DEV).manual_seed(7)
    nb, w = 9, kv * hd
    cache = empty(nb, kv, bs, hd, dtype)
    o = oracles_of(cache)
    write(keys(nb * bs, kv, hd, g), 0, list(range(nb * bs)), cache, o, kv, hd)
    slots = torch.randint(-3, nb * bs, (77,), generator=torch.Generator().manual_seed(1)).tolist() + [0, nb * bs - 1, -1]
    wide = torch.full((len(slots) + 2, 24 + 2 * w + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    dst = wide[:, :24 + 2 * w]
    kv_q8.kv_rows_q8(*cache, torch.tensor(slots, dtype=torch.int32, device=DEV), dst, 24 + w, 24)      # values first
    for col, c in ((24 + w, o[0]), (24, o[1])):
        assert torch.equal(dst[:len(slots), col:col + w].double().cpu(), c.tokens(slots).flatten(1))     # a code fits bf16
    assert (wide[:, :24] == 5).all() and (wide[:, 24 + 2 * w:] == 5).all() and (wide[len(slots):] == 5).all()


def pages(lens, bs, spare=3, seed=1):
    need = [(n + bs - 1) // bs for n in lens]
    nb = sum(need) + spare
    order = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    bt = torch.full((len(lens), max(need) + 1), -7, dtype=torch.int32)          # entries behind a sequence's end are not read
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = order[at:at + n]
        at += n
    return bt, nb


def filled(nb, kv, bs, hd, dtype, g):
    cache = empty(nb, kv, bs, hd, dtype)
    from art_b200.ops import kv_q8

    kv_q8.kv_write_q8(keys(nb * bs, kv, hd, g, spread=0.3), 0, kv * hd, torch.arange(nb * bs, dtype=torch.int32, device=DEV), *cache)
    return cache


def check_decode(out, q, cache, bt, lens, Hq, hd, some=16):
    k, v = oracles_of(cache)
    bs = cache[0].shape[2]
    for i in list(range(len(lens)))[:: max(1, len(lens) // some)]:
        n = lens[i]
        t = torch.arange(n)
        slots = bt[i].cpu().long()[t // bs] * bs + t % bs
        ref, bound = attend(q[i, :Hq * hd].double().cpu().view(Hq, hd), k.tokens(slots), v.tokens(slots), k.dtype)
        off = (out[i, :Hq * hd].double().cpu().view(Hq, hd) - ref).abs()
        assert (off <= bound).all(), (i, n, float((off - bound).max()))


DECODE = [
    ([1], 2, 1, 64, 16),
    ([777], 16, 2, 128, 16),                                  # one context in many shares
    ([0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 0], 8, 8, 128, 16),    # edges of a block and of tiles; empty contexts
    ([5000, 3, 0, 2111], 28, 4, 128, 16),
    ([33] * 700, 14, 2, 64, 16),                              # more pairs than CTAs
    ([257, 64, 1], 32, 2, 32, 48),                            # 16 query heads per kv head, blocks that are no power of two
    ([100, 1, 900], 20, 2, 128, 32),                          # 10
    ([1500] * 64, 8, 8, 64, 32),
    ([19, 4001], 9, 1, 128, 128),
    ([0, 0, 0], 4, 2, 32, 16),
    ([(5 * i) % 70 for i in range(1500)], 4, 2, 64, 16),          # more sequences than a CTA lists one by one
    ([0] * 2000 + [40, 0, 300] + [0] * 1500 + [1], 4, 1, 128, 16),
    ([3] * 1024, 4, 4, 32, 16),
    ([90] * 40, 128, 64, 64, 16),                                 # many kv heads
    ([70, 900], 600, 600, 32, 16),                                # more than CTAs
    ([300, 0, 0, 0, 0, 2, 0, 64], 6, 2, 128, 64),
]


@KINDS
@pytest.mark.parametrize("lens,Hq,Hkv,hd,bs", DECODE, ids=[f"{len(c[0])}x{max(c[0])}-{c[1]}/{c[2]}x{c[3]}-{c[4]}" for c in DECODE])
def test_decode(dtype, lens, Hq, Hkv, hd, bs):
    from art_b200.ops import kv_q8

    g = torch.Generator(device=DEV).manual_seed(len(lens) + hd)
    bt, nb = pages(lens, bs)
    bt = bt.to(DEV)
    cache = filled(nb, Hkv, bs, hd, dtype, g)
    q = torch.randn(len(lens), (Hq + 2 * Hkv) * hd, generator=g, device=DEV).bfloat16()
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = kv_q8.decode_q8_workspace(len(lens), Hq, Hkv, hd, DEV)
    wide = torch.full((len(lens), Hq * hd + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    out = wide[:, :Hq * hd]
    kv_q8.paged_decode_q8(q, *cache, bt, ctx, Hq, Hkv, hd, out, ws)
    again = torch.empty_like(out)
    kv_q8.paged_decode_q8(q, *cache, bt, ctx, Hq, Hkv, hd, again, ws)          # the workspace is as the first call found it
    assert torch.equal(out, again) and (wide[:, Hq * hd:] == 5).all()
    check_decode(out, q, cache, bt, lens, Hq, hd)


@KINDS
def test_decode_sharp_and_large_scores(dtype):
    """Scores far apart, so that the running maximum moves often, queries near the ends of bf16's range, and values whose blocks
    differ in size by many powers of two."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs, lens = 8, 2, 64, 16, [1000, 37]
    g = torch.Generator(device=DEV).manual_seed(11)
    bt, nb = pages(lens, bs)
    bt = bt.to(DEV)
    cache = empty(nb, Hkv, bs, hd, dtype)
    x = torch.randn(nb * bs, 2 * Hkv * hd, generator=g, device=DEV)
    x[:, Hkv * hd:] *= torch.exp2(torch.randint(-30, 30, (nb, 1), generator=g, device=DEV).float()).repeat_interleave(bs, 0)
    kv_q8.kv_write_q8(x.bfloat16(), 0, Hkv * hd, torch.arange(nb * bs, dtype=torch.int32, device=DEV), *cache)
    ctx, ws = torch.tensor(lens, dtype=torch.int32, device=DEV), kv_q8.decode_q8_workspace(2, Hq, Hkv, hd, DEV)
    base = torch.randn(2, Hq * hd, generator=g, device=DEV)
    for size in (0.0, 1e-30, 1e-3, 12.0):
        q = (base * size).bfloat16()
        q[0, 5] *= 2.0 ** -20
        out = kv_q8.paged_decode_q8(q, *cache, bt, ctx, Hq, Hkv, hd, torch.empty_like(q), ws)
        check_decode(out, q, cache, bt, lens, Hq, hd)


@KINDS
@pytest.mark.parametrize("least,most", [(-110, 110), (-110, -90), (90, 110)])
def test_decode_values_of_any_size(dtype, least, most):
    """Blocks of values from bf16's smallest to its largest in one context, and blocks of zeros, whose scale is the least there is."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs, lens = 8, 2, 64, 16, [3000, 37, 160]
    g = torch.Generator(device=DEV).manual_seed(31)
    bt, nb = pages(lens, bs)
    bt = bt.to(DEV)
    cache = empty(nb, Hkv, bs, hd, dtype)
    x = torch.randn(nb * bs, 2 * Hkv * hd, generator=g, device=DEV)
    size = torch.exp2(torch.randint(least, most + 1, (nb, 1), generator=g, device=DEV).float())
    size[torch.rand(nb, generator=g, device=DEV) < 0.2] = 0
    x[:, Hkv * hd:] *= size.repeat_interleave(bs, 0)
    kv_q8.kv_write_q8(x.bfloat16(), 0, Hkv * hd, torch.arange(nb * bs, dtype=torch.int32, device=DEV), *cache)
    ctx, ws = torch.tensor(lens, dtype=torch.int32, device=DEV), kv_q8.decode_q8_workspace(3, Hq, Hkv, hd, DEV)
    for sharp in (1.0, 20.0):
        q = (sharp * torch.randn(3, Hq * hd, generator=g, device=DEV)).bfloat16()
        out = kv_q8.paged_decode_q8(q, *cache, bt, ctx, Hq, Hkv, hd, torch.empty_like(q), ws)
        check_decode(out, q, cache, bt, lens, Hq, hd)


@KINDS
@pytest.mark.parametrize("Hq,Hkv,hd", [(4, 2, 32), (6, 2, 64), (28, 4, 128), (16, 1, 128)])
def test_decode_queries_of_uneven_size(dtype, Hq, Hkv, hd):
    """Queries of one value among zeros, of values from the largest a head's scaling leaves to bits below its last, of all the same
    largest magnitude, of bf16's smallest numbers, and of zeros: the rounding of a query is relative to its head."""
    from art_b200.ops import kv_q8

    bs, lens = 16, [700, 33, 64, 90, 500]
    g = torch.Generator(device=DEV).manual_seed(21)
    bt, nb = pages(lens, bs)
    cache = filled(nb, Hkv, bs, hd, dtype, g)
    q = torch.randn(len(lens), Hq, hd, generator=g, device=DEV)
    q[0] = 0
    q[0, :, 5] = torch.linspace(-3, 3, Hq, device=DEV)
    q[1] *= torch.exp2(-(torch.arange(hd, device=DEV) % 24).float())
    q[2] = q[2].sign() * 255 * 2.0 ** -10
    q[3] *= 2.0 ** -130
    q[4, ::2] = 0
    q = q.bfloat16().view(len(lens), Hq * hd)
    table, ctx = bt.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = kv_q8.decode_q8_workspace(len(lens), Hq, Hkv, hd, DEV)
    out = kv_q8.paged_decode_q8(q, *cache, table, ctx, Hq, Hkv, hd, torch.empty_like(q), ws)
    check_decode(out, q, cache, bt, lens, Hq, hd)


def test_decode_keeps_what_is_masked_out():
    """What lies behind a context in its last block is not seen, whatever it holds."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs, lens = 8, 2, 128, 32, [50, 1, 33]
    g = torch.Generator(device=DEV).manual_seed(4)
    bt, nb = pages(lens, bs)
    bt = bt.to(DEV)
    cache = filled(nb, Hkv, bs, hd, E4, g)
    q = torch.randn(3, Hq * hd, generator=g, device=DEV).bfloat16()
    ctx, ws = torch.tensor(lens, dtype=torch.int32, device=DEV), kv_q8.decode_q8_workspace(3, Hq, Hkv, hd, DEV)
    out = kv_q8.paged_decode_q8(q, *cache, bt, ctx, Hq, Hkv, hd, torch.empty_like(q), ws)
    for i, n in enumerate(lens):
        b = int(bt[i, (n - 1) // bs])
        for c in cache[:2]:
            c.view(torch.uint8)[b, :, (n - 1) % bs + 1:] = 0x7f        # NaN
    again = kv_q8.paged_decode_q8(q, *cache, bt, ctx, Hq, Hkv, hd, torch.empty_like(q), ws)
    assert torch.equal(out, again)
    check_decode(again, q, cache, bt, lens, Hq, hd)


@KINDS
def test_decode_shows_what_is_not_a_number(dtype):
    """A scale that is NaN, as a key or value that was not finite leaves it, and a query that is none: the heads that meet it are NaN,
    wherever in the context it lies; others are as without it."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs, lens = 6, 2, 64, 16, [3000, 40, 9]
    g = torch.Generator(device=DEV).manual_seed(14)
    bt, nb = pages(lens, bs)
    cache = filled(nb, Hkv, bs, hd, dtype, g)
    q = torch.randn(3, Hq * hd, generator=g, device=DEV).bfloat16()
    table, ctx = bt.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = kv_q8.decode_q8_workspace(3, Hq, Hkv, hd, DEV)
    good = kv_q8.paged_decode_q8(q, *cache, table, ctx, Hq, Hkv, hd, torch.empty_like(q), ws).clone()
    cache[2][bt[0, 100], 1] = float("nan")         # a key scale amid the first context, kv head 1
    cache[3][bt[1, 2], 0] = float("nan")           # a value scale at the end of the second, kv head 0
    q[2, 5 * hd + 7] = float("nan")                # the last query head of the third
    out = kv_q8.paged_decode_q8(q, *cache, table, ctx, Hq, Hkv, hd, torch.empty_like(q), ws)
    bad = torch.zeros(3, Hq, dtype=torch.bool, device=DEV)
    bad[0, 3:] = bad[1, :3] = bad[2, 5] = True
    out, good = out.view(3, Hq, hd), good.view(3, Hq, hd)
    assert out[bad].isnan().all() and torch.equal(out[~bad], good[~bad])


@KINDS
def test_a_sequence_from_prompt_to_decoding(dtype):
    """The calls in the order of a rollout: a prompt in two portions, the first read back for the second, then tokens one by one."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs = 6, 2, 128, 16
    g = torch.Generator(device=DEV).manual_seed(21)
    lens, first, more = [37, 5, 64], [20, 5, 48], 20
    bt, nb = pages([n + more for n in lens], bs)
    table = bt.to(DEV)
    cache = empty(nb, Hkv, bs, hd, dtype)
    o = oracles_of(cache)
    slot = lambda i, t: int(bt[i, t // bs]) * bs + t % bs      # noqa: E731
    q0, w = Hq * hd, Hkv * hd
    for lo, hi in (([0, 0, 0], first), (first, lens)):
        s = [slot(i, t) for i in range(3) for t in range(lo[i], hi[i])]
        write(keys(len(s), Hkv, hd, g, extra=q0), q0, s, cache, o, Hkv, hd)
        old = [slot(i, t) if t < lo[i] else -1 for i in range(3) for t in range(hi[i])]
        dst = torch.empty(len(old), q0 + 2 * w, dtype=torch.bfloat16, device=DEV)
        kv_q8.kv_rows_q8(*cache, torch.tensor(old, dtype=torch.int32, device=DEV), dst, q0, q0 + w)
        assert torch.equal(dst[:, q0:q0 + w].double().cpu(), o[0].tokens(old).flatten(1))
    ws = kv_q8.decode_q8_workspace(4, Hq, Hkv, hd, DEV)
    for step in range(more):
        x = keys(4, Hkv, hd, g, spread=0.4, extra=q0)
        x[:, :q0] = torch.randn(4, q0, generator=g, device=DEV)
        at = [n + step for n in lens]
        write(x, q0, [slot(i, at[i]) for i in range(3)] + [-1], cache, o, Hkv, hd)       # a padded batch
        ctx = torch.tensor([t + 1 for t in at] + [0], dtype=torch.int32, device=DEV)
        tab = torch.cat([table, torch.zeros_like(table[:1])])
        out = kv_q8.paged_decode_q8(x, *cache, tab, ctx, Hq, Hkv, hd, torch.empty(4, q0, dtype=torch.bfloat16, device=DEV), ws)
        same(cache, *o)
        assert not out[3].any()
        check_decode(out, x, cache, tab, [t + 1 for t in at] + [0], Hq, hd)


@KINDS
def test_graphs_and_streams(dtype):
    """A captured step replayed on other inputs, and two streams with a workspace each."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs, lens = 14, 2, 64, 16, [600, 1, 90, 0]
    g = torch.Generator(device=DEV).manual_seed(8)
    bt, nb = pages(lens, bs)
    table = bt.to(DEV)
    cache = filled(nb, Hkv, bs, hd, dtype, g)
    spare = [t.clone() for t in cache]
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    w, q0 = Hkv * hd, Hq * hd
    slots = torch.tensor([int(bt[i, (n - 1) // bs]) * bs + (n - 1) % bs if n else -1 for i, n in enumerate(lens)], dtype=torch.int32, device=DEV)
    xs = [keys(4, Hkv, hd, g, spread=0.3, extra=q0) for _ in range(2)]

    def step(x, c, out, ws):
        kv_q8.kv_write_q8(x, q0, q0 + w, slots, *c)
        kv_q8.paged_decode_q8(x, *c, table, ctx, Hq, Hkv, hd, out, ws)
        kv_q8.kv_rows_q8(*c, slots, x, q0, q0 + w)

    def fresh():
        return torch.zeros(4, q0, dtype=torch.bfloat16, device=DEV), kv_q8.decode_q8_workspace(4, Hq, Hkv, hd, DEV)

    want = []
    for x in xs:
        y, (out, ws) = x.clone(), fresh()
        step(y, cache, out, ws)
        want.append((out, y))
    for a, b in zip(cache, spare):
        a.copy_(b)
    x, (out, ws) = xs[0].clone(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(x, cache, out, ws)
    for i in range(2):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i][0]) and torch.equal(x, want[i][1])
    # two streams at once
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    caches = [[t.clone() for t in spare] for _ in streams]
    torch.cuda.synchronize()
    for s, c in zip(streams, caches):
        with torch.cuda.stream(s):
            x, (out, ws) = xs[0].clone(), fresh()
            for _ in range(20):
                step(x, c, out, ws)
                x.copy_(xs[0])
            step(x, c, out, ws)
            got.append((out, x))
    torch.cuda.synchronize()
    for out, x in got:
        assert torch.equal(out, want[0][0]) and torch.equal(x, want[0][1])


@KINDS
@pytest.mark.parametrize("M,Hq,Hkv,hd,bs,lora,norm,bias", [
    (5, 14, 2, 64, 16, True, False, True),
    (200, 28, 4, 128, 16, True, False, True),          # two rows to a multiprocessor
    (33, 32, 8, 128, 48, False, True, False),
    (1, 3, 1, 32, 16, False, False, True),
    (64, 4, 2, 32, 32, True, True, False),
])
def test_finish_kernel(dtype, M, Hq, Hkv, hd, bs, lora, norm, bias):
    """The finish kernel into the 8-bit cache: the numbers of the bf16 finish kernel and a write of its rows."""
    from art_b200.ops import kv_q8, paged

    g = torch.Generator(device=DEV).manual_seed(M + hd)
    N, kpad, cols, w = (Hq + 2 * Hkv) * hd, 64, 24, Hkv * hd
    ws = torch.randn(M + 3, N + kpad + 8, generator=g, device=DEV) * torch.exp(0.7 * torch.randn(M + 3, 1, generator=g, device=DEV))
    kw = dict(bias=torch.randn(N, generator=g, device=DEV) if bias else None, cols=cols,
              adapter=torch.randint(-1, 2, (M,), generator=g, device=DEV).int() if lora else None,
              B_all=(0.1 * torch.randn(kpad, N, generator=g, device=DEV)).bfloat16() if lora else None,
              q_norm=torch.rand(hd, generator=g, device=DEV).bfloat16() if norm else None,
              k_norm=(torch.rand(hd, generator=g, device=DEV) * 3).bfloat16() if norm else None)
    pos = torch.randint(0, 5000, (M,), generator=g, device=DEV).int()
    nb = M + 4
    block = torch.randperm(nb, generator=g, device=DEV)[:M]
    slot = (block * bs + torch.randint(0, bs, (M,), generator=g, device=DEV)).int()
    slot[M // 2] = -1 if M > 1 else slot[0]
    cache = filled(nb, Hkv, bs, hd, dtype, g)
    other = [t.clone() for t in cache]
    args = (M, Hq, Hkv, hd, kpad, pos, 1e6)
    q1, q2 = (torch.zeros(M, Hq * hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ws1, ws2 = ws.clone(), ws.clone()
    kv_q8.decode_finalize_qkv_q8(ws1, *args, slot, *cache, q1, **kw)
    rows = torch.zeros(M, 2 * w, dtype=torch.bfloat16, device=DEV)
    at = torch.arange(0, 2 * M, 2, dtype=torch.int32, device=DEV)
    paged.decode_finalize_qkv(ws2, *args, at, rows.view(2 * M, 1, Hkv, hd), rows[:, w:], q2, **kw)
    kv_q8.kv_write_q8(rows, 0, w, slot, *other)
    assert torch.equal(q1, q2) and torch.equal(ws1, ws2) and not torch.equal(ws1, ws)
    for a, b in zip(cache, other):
        assert torch.equal(a.float(), b.float())


def order_case(g):
    """Calls whose inputs another launch, copy or stream writes just before: ``(fill, calls, want)``."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs, lens = 8, 2, 64, 16, [600, 33, 90, 1]
    bt, nb = pages(lens, bs)
    table = bt.to(DEV)
    cache = filled(nb, Hkv, bs, hd, E4, g)
    spare = [t.clone() for t in cache]
    w, q0 = Hkv * hd, Hq * hd
    slots = [int(bt[i, (n - 1) // bs]) * bs + (n - 1) % bs for i, n in enumerate(lens)]
    src = (keys(4, Hkv, hd, g, spread=0.3, extra=q0), torch.tensor(slots, dtype=torch.int32, device=DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    x, slot, ctx = (torch.zeros_like(t) for t in src)
    out, back = torch.zeros(4, q0, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 2 * w, dtype=torch.bfloat16, device=DEV)
    ws = kv_q8.decode_q8_workspace(4, Hq, Hkv, hd, DEV)

    def reset():
        for a, b in zip(cache, spare):
            a.copy_(b)
        slot.fill_(-1)
        for t in (x, ctx, out, back):
            t.zero_()

    def fill(copy=lambda a, b: a.copy_(b)):
        for a, b in zip((x, slot, ctx), src):
            copy(a, b)

    def calls():
        kv_q8.kv_write_q8(x, q0, q0 + w, slot, *cache)
        kv_q8.paged_decode_q8(x, *cache, table, ctx, Hq, Hkv, hd, out, ws)
        kv_q8.kv_rows_q8(*cache, slot, back, 0, w)

    def got():
        torch.cuda.synchronize()
        return [t.clone() for t in (out, back, *(c.float() for c in cache))]

    reset()
    fill()
    torch.cuda.synchronize()
    calls()
    return reset, fill, calls, got, got()


@pytest.mark.parametrize("how", ["kernel", "copy", "stream", "graph", "forked graph"])
def test_inputs_that_are_only_just_written(how):
    """Launches start ahead of what comes before them; what they read is there all the same."""
    g = torch.Generator(device=DEV).manual_seed(31)
    reset, fill, calls, got, want = order_case(g)
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()

    def same_as_wanted():
        for a, b in zip(got(), want):
            assert torch.equal(a, b)

    def forked():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000)
            fill()
        torch.cuda._sleep(1000)
        torch.cuda.current_stream().wait_stream(side)
        calls()

    for _ in range(3):
        reset()
        torch.cuda.synchronize()
        if how == "kernel":
            torch.cuda._sleep(200_000)
            fill(lambda a, b: torch.add(b, 0, out=a))
            calls()
        elif how == "copy":
            host = {}
            fill(lambda a, b: host.__setitem__(a.data_ptr(), b.cpu().pin_memory()))
            torch.cuda._sleep(200_000)
            fill(lambda a, b: a.copy_(host[a.data_ptr()], non_blocking=True))
            calls()
        elif how == "stream":
            forked()
        else:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                if how == "graph":
                    torch.cuda._sleep(200_000)
                    fill()
                    calls()
                else:
                    forked()
            reset()
            graph.replay()
        same_as_wanted()


def test_places_outside_the_cache_are_reported():
    """Slots, table entries and lengths that name no place are skipped or cut off, and the status word says so."""
    from art_b200.ops import _lib, kv_q8

    Hq, Hkv, hd, bs = 4, 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(8)
    cache = filled(6, Hkv, bs, hd, I8, g)
    before = [t.clone() for t in cache]
    x = keys(3, Hkv, hd, g)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)        # noqa: E731
    kv_q8.kv_write_q8(x, 0, Hkv * hd, i32(-1, 6 * bs, 2 ** 31 - 1), *cache)
    with pytest.raises(_lib.KernelStatusError):
        _lib.check_status()
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    dst = torch.ones(3, 2 * Hkv * hd, dtype=torch.bfloat16, device=DEV)
    kv_q8.kv_rows_q8(*cache, i32(6 * bs, 5, 2 ** 31 - 1), dst, 0, Hkv * hd)
    with pytest.raises(_lib.KernelStatusError):
        _lib.check_status()
    assert not dst[0].any() and dst[1].any() and not dst[2].any()
    q = torch.randn(3, Hq * hd, generator=g, device=DEV).bfloat16()
    ws = kv_q8.decode_q8_workspace(3, Hq, Hkv, hd, DEV)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=DEV)
    rope = torch.zeros(3, dtype=torch.int32, device=DEV)
    kv_q8.decode_finalize_qkv_q8(torch.randn(3, (Hq + 2 * Hkv) * hd, generator=g, device=DEV), 3, Hq, Hkv, hd, 0, rope, 1e6, i32(-5, 6 * bs, 2 ** 31 - 1),
                                 *cache, torch.empty_like(q))
    with pytest.raises(_lib.KernelStatusError):
        _lib.check_status()
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    good = kv_q8.paged_decode_q8(q, *cache, table, i32(32, 20, 32), Hq, Hkv, hd, torch.empty_like(q), ws)
    _lib.check_status()
    out = kv_q8.paged_decode_q8(q, *cache, table, i32(2 ** 31 - 1, 20, 33), Hq, Hkv, hd, torch.empty_like(q), ws)
    with pytest.raises(_lib.KernelStatusError):
        _lib.check_status()
    assert torch.equal(out, good)
    table[0, 1], table[2, 0] = 6, -1
    out = kv_q8.paged_decode_q8(q, *cache, table, i32(32, 20, 32), Hq, Hkv, hd, torch.empty_like(q), ws)
    with pytest.raises(_lib.KernelStatusError):
        _lib.check_status()
    assert torch.equal(out[1], good[1]) and out.isfinite().all()


def test_rows_of_a_block_that_are_not_in_order_are_refused():
    """A row after another of its block that is not at the next place: not written, and the status word says so."""
    from art_b200.ops import _lib, kv_q8

    Hkv, hd, bs = 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(8)
    for slots, written in (([5, 7], [5, -1]), ([5, 5], [5, -1]), ([5, 4], [5, -1]), ([3, 4, 20, 22, 21], [3, 4, 20, -1, -1])):
        cache = filled(3, Hkv, bs, hd, E4, g)
        o = oracles_of(cache)
        x = keys(len(slots), Hkv, hd, g)
        kv_q8.kv_write_q8(x, 0, Hkv * hd, torch.tensor(slots, dtype=torch.int32, device=DEV), *cache)
        with pytest.raises(_lib.KernelStatusError):
            _lib.check_status()
        for j in range(2):
            o[j].write(x[:, j * Hkv * hd:(j + 1) * Hkv * hd], written)
        same(cache, *o)


def test_caches_beyond_32_bits():
    """Offsets of more than 2^31 bytes."""
    from art_b200.ops import kv_q8

    Hq, Hkv, hd, bs = 8, 8, 128, 16
    nb = 2 ** 31 // (Hkv * bs * hd) + 70
    cache = empty(nb, Hkv, bs, hd, E4)
    g = torch.Generator(device=DEV).manual_seed(8)
    n = 1000
    first = nb - 63
    slots = torch.arange(first * bs, first * bs + n, dtype=torch.int32, device=DEV)
    x = keys(n, Hkv, hd, g, spread=0.3, extra=Hq * hd)
    kv_q8.kv_write_q8(x, Hq * hd, 2 * Hq * hd, slots, *cache)
    small = empty(63, Hkv, bs, hd, E4)
    kv_q8.kv_write_q8(x, Hq * hd, 2 * Hq * hd, slots - first * bs, *small)
    for a, b in zip(cache, small):
        assert torch.equal(a[first:].float(), b.float())
    dst, dst2 = torch.zeros_like(x), torch.zeros_like(x)
    kv_q8.kv_rows_q8(*cache, slots, dst, Hq * hd, 2 * Hq * hd)
    kv_q8.kv_rows_q8(*small, slots - first * bs, dst2, Hq * hd, 2 * Hq * hd)
    assert torch.equal(dst, dst2) and dst.any()
    table = torch.arange(first, nb, dtype=torch.int32, device=DEV)[None].contiguous()
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    ws = kv_q8.decode_q8_workspace(1, Hq, Hkv, hd, DEV)
    q = x[:1]
    a = kv_q8.paged_decode_q8(q, *cache, table, ctx, Hq, Hkv, hd, torch.empty(1, Hq * hd, dtype=torch.bfloat16, device=DEV), ws)
    b = kv_q8.paged_decode_q8(q, *small, table - first, ctx, Hq, Hkv, hd, torch.empty(1, Hq * hd, dtype=torch.bfloat16, device=DEV), ws)
    assert torch.equal(a, b) and a.any()


def test_workspace_of_another_size_is_refused():
    from art_b200.ops import kv_q8

    cache = empty(4, 2, 16, 64, E4)
    q = torch.zeros(300, 8 * 64, dtype=torch.bfloat16, device=DEV)
    bt, ctx = torch.zeros(300, 2, dtype=torch.int32, device=DEV), torch.zeros(300, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="needed"):
        kv_q8.paged_decode_q8(q, *cache, bt, ctx, 8, 2, 64, torch.empty_like(q), torch.zeros(8, dtype=torch.uint8, device=DEV))


def test_more_tiles_than_can_be_numbered_are_refused():
    from art_b200.ops import kv_q8

    cache = empty(1, 1, 1 << 20, 32, E4)
    q = torch.zeros(33, 32, dtype=torch.bfloat16, device=DEV)
    bt, ctx = torch.zeros(33, 2048, dtype=torch.int32, device=DEV), torch.ones(33, dtype=torch.int32, device=DEV)
    ws = kv_q8.decode_q8_workspace(33, 1, 1, 32, DEV)
    with pytest.raises(ValueError, match="beyond the supported maximum"):
        kv_q8.paged_decode_q8(q, *cache, bt, ctx, 1, 1, 32, torch.empty_like(q), ws)
    kv_q8.paged_decode_q8(q, *cache, bt[:, :1024].contiguous(), ctx, 1, 1, 32, torch.empty_like(q), ws)
