"""Writes into the 8-bit cache whose rows of one block are no neighbours: refused and reported, and none that are in order."""
import pytest
import torch

from .test_gpu_kv_q8 import DEV, E4, KINDS, empty, filled, keys, oracles_of, same

pytestmark = pytest.mark.gpu


def accepted(slots, bs):
    """The slots that are written: a run of neighbours begins where its block is not that of the last row before it that has a slot
    (of any row before it in a call of up to 256), and goes on while places follow one another."""
    out, last, before = [], -1, set()
    for i, s in enumerate(slots):
        if s < 0:
            out.append(-1)
            continue
        if i and slots[i - 1] == s - 1 and s % bs:
            out.append(s if out[-1] >= 0 else -1)
        else:
            again = s // bs in before if len(slots) <= 256 else last >= 0 and last // bs == s // bs
            out.append(-1 if again else s)
        last = s
        before.add(s // bs)
    return out


def runs(bs, *parts):
    """(block, first place, rows) or a number of rows that are not written, one after the other."""
    out = []
    for p in parts:
        out += [-1] * p if isinstance(p, int) else [p[0] * bs + p[1] + i for i in range(p[2])]
    return out


def gaps(bs, total, gap):
    """Runs in blocks of their own with rows that are not written before, between and behind them; every third run is cut by such."""
    parts, block, n = [gap], 0, gap
    while n < total:
        rows = 1 + (7 * block) % (bs - 3)
        parts += [(block, 1, rows), 1 + (gap * (block % 5)) // 4]
        if block % 3 == 2 and rows + 1 < bs:
            parts += [(block, 1 + rows, 1), 2]
        n = sum(p if isinstance(p, int) else p[2] for p in parts)
        block += 1
    return runs(bs, *parts)


CALLS = [
    (16, runs(16, (0, 5, 1), 1, (0, 6, 1))),
    (16, runs(16, (0, 5, 1), (2, 8, 1), (0, 6, 1))),
    (16, runs(16, (1, 0, 3), 2, (1, 3, 2), (0, 0, 1), (1, 5, 1), 1)),
    (16, runs(16, 3, (0, 0, 16), 1, (1, 0, 16), 40, (1, 15, 1))),
    (32, runs(32, (3, 4, 20), (1, 0, 32), (3, 24, 2), 100, (0, 0, 5), (3, 26, 1))),
    (64, runs(64, (0, 0, 40), 9, (0, 40, 20), (1, 0, 9))),
    (16, gaps(16, 300, 9)), (64, gaps(64, 300, 9)),               # 4 rows to a warp; a run to four warps
    (16, gaps(16, 2100, 31)), (16, gaps(16, 4000, 700)), (128, gaps(128, 4000, 600)),
    (16, runs(16, (0, 0, 1), 4000, (0, 1, 1))),
]


@KINDS
@pytest.mark.parametrize("bs,slots", CALLS, ids=[f"{len(c[1])}-{c[0]}-{i}" for i, c in enumerate(CALLS)])
@pytest.mark.parametrize("in_order", [False, True])
def test_writes(dtype, bs, slots, in_order):
    from art_b200.ops import _lib, kv_q8

    Hkv, hd, want = 2, 64, accepted(slots, bs)
    assert want != slots
    if in_order:                  # the same call without the rows that are refused is taken whole
        slots = want
    g = torch.Generator(device=DEV).manual_seed(len(slots))
    cache = filled(max(slots) // bs + 2, Hkv, bs, hd, dtype, g)
    o = oracles_of(cache)
    x = keys(len(slots), Hkv, hd, g)
    kv_q8.kv_write_q8(x, 0, Hkv * hd, torch.tensor(slots, dtype=torch.int32, device=DEV), *cache)
    if in_order:
        _lib.check_status()
    else:
        with pytest.raises(_lib.KernelStatusError):
            _lib.check_status()
    for j in range(2):
        o[j].write(x[:, j * Hkv * hd:(j + 1) * Hkv * hd], want)
    same(cache, *o)


def test_rows_above_in_no_block():
    """Slots beyond the cache share no block with others, and the largest of them name no row in reach."""
    from art_b200.ops import _lib, kv_q8

    Hkv, hd, bs = 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(3)
    for rows in (5, 300, 3000):
        slots = [2 ** 31 - 1, -2 ** 31, 3, -1, 2 ** 31 - 2] + [-1] * (rows - 6) + [16]
        cache = empty(4, Hkv, bs, hd, E4)
        o = oracles_of(cache)
        x = keys(len(slots), Hkv, hd, g)
        kv_q8.kv_write_q8(x, 0, Hkv * hd, torch.tensor(slots, dtype=torch.int32, device=DEV), *cache)
        with pytest.raises(_lib.KernelStatusError):
            _lib.check_status()
        for j in range(2):
            o[j].write(x[:, j * Hkv * hd:(j + 1) * Hkv * hd], [s if 0 <= s < 64 else -1 for s in slots])
        same(cache, *o)


@KINDS
@pytest.mark.parametrize("rows,twice", [(3, {2: 0}), (9, {3: 1, 8: 1, 6: 4}), (300, {299: 0, 270: 250, 256: 255})])
def test_finish(dtype, rows, twice):
    """Of two rows of one block the later is not written and reported; its query is there, and so are all others."""
    from art_b200.ops import _lib, kv_q8

    Hq, Hkv, hd, bs = 4, 2, 64, 32
    g = torch.Generator(device=DEV).manual_seed(rows)
    ws = torch.randn(rows, (Hq + 2 * Hkv) * hd, generator=g, device=DEV)
    pos = torch.randint(0, 500, (rows,), generator=g, device=DEV).int()
    slot = torch.randperm(rows + 2, generator=g, device=DEV)[:rows].int() * bs + torch.randint(0, bs, (rows,), generator=g, device=DEV).int()
    slot[rows // 2] = -1
    want = slot.clone()
    for later, first in twice.items():
        slot[later], want[later] = slot[first] // bs * bs + (slot[first] + 7) % bs, -1
    results = []
    for s in (slot, want):
        cache, q = filled(rows + 2, Hkv, bs, hd, dtype, torch.Generator(device=DEV).manual_seed(1)), torch.zeros(rows, Hq * hd, dtype=torch.bfloat16, device=DEV)
        kv_q8.decode_finalize_qkv_q8(ws.clone(), rows, Hq, Hkv, hd, 0, pos, 1e6, s, *cache, q)
        if s is slot:
            with pytest.raises(_lib.KernelStatusError):
                _lib.check_status()
        else:
            _lib.check_status()
        results.append([q, *(c.double() for c in cache)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
