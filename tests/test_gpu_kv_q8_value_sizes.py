"""Decode attention over the 8-bit cache where a warp reads many tiles of one context whose values differ in size from block to block:
what has been summed so far is carried from one block's scale to the next."""
import pytest
import torch

from .kv_q8_oracle import attend
from .test_gpu_kv_q8 import DEV, KINDS, empty, pages

pytestmark = pytest.mark.gpu


def zeros(blocks):
    """Blocks of zeros, two to five in a row, at a context's start, in its middle and at its end."""
    size = torch.ones(blocks)
    for at, run in ((0, 2), (blocks // 3, 3), (blocks // 2, 5), (blocks - 2, 2)):
        size[max(0, at):at + run] = 0
    return size


def ends_in_zeros(blocks):
    size = torch.ones(blocks)
    size[max(1, blocks - 4):] = 0
    return size


def falling(blocks):
    return torch.exp2(-60.0 * (torch.arange(blocks) // 2 % 3))


def rising(blocks):
    return torch.exp2(60.0 * (torch.arange(blocks) // 2 % 3) - 60)


def far(blocks):
    """The largest, the smallest and none, in turn."""
    size = torch.exp2(100 - 200.0 * (torch.arange(blocks) % 2))
    size[torch.arange(blocks) % 7 > 4] = 0
    return size


def any_size(blocks):
    g = torch.Generator().manual_seed(blocks)
    size = torch.exp2(torch.randint(-100, 101, (blocks,), generator=g).float())
    size[torch.rand(blocks, generator=g) < 0.2] = 0
    return size


# a warp's tiles are of one context in the first, of one to five contexts in the others: 2, 20, 8 and 14 tiles to a warp
SHAPES = [([6000], 32, 8, 128, 16), ([1500] * 64, 16, 8, 128, 32), ([(37 * i) % 400 for i in range(512)], 8, 4, 32, 16), ([1500] * 64, 96, 8, 64, 16)]


@KINDS
@pytest.mark.parametrize("sizes", [zeros, ends_in_zeros, falling, rising, far, any_size])
@pytest.mark.parametrize("lens,Hq,Hkv,hd,bs", SHAPES, ids=[f"{len(c[0])}x{max(c[0])}-{c[1]}/{c[2]}x{c[3]}" for c in SHAPES])
def test_values_of_uneven_blocks(dtype, sizes, lens, Hq, Hkv, hd, bs):
    from art_b200.ops import kv_q8

    g = torch.Generator(device=DEV).manual_seed(len(lens) + hd)
    bt, nb = pages(lens, bs)
    size = torch.ones(nb)
    first = torch.zeros(nb, dtype=torch.bool)
    for i, n in enumerate(lens):
        own = bt[i, :-(-n // bs)].long()
        size[own] = sizes(len(own))
        first[own[:1]] = True
    x = torch.randn(nb * bs, 2, Hkv, hd, generator=g, device=DEV)
    x[:, 1] *= size.to(DEV).repeat_interleave(bs)[:, None, None]
    # the first block's scores lie 7 powers of two below the others': weights are relative to the first of them
    x[:, 0, :, 0] = torch.where(first.to(DEV).repeat_interleave(bs), 0.0, 0.7 * hd ** 0.5)[:, None]
    cache = empty(nb, Hkv, bs, hd, dtype)
    for lo in range(0, nb * bs, 1 << 16):
        rows = x[lo:lo + (1 << 16)].bfloat16().flatten(1)
        kv_q8.kv_write_q8(rows, 0, Hkv * hd, torch.arange(lo, lo + len(rows), dtype=torch.int32, device=DEV), *cache)
    ctx, ws = torch.tensor(lens, dtype=torch.int32, device=DEV), kv_q8.decode_q8_workspace(len(lens), Hq, Hkv, hd, DEV)
    table = bt.to(DEV)
    for sharp in (0.1, 1.0):
        q = sharp * torch.randn(len(lens), Hq, hd, generator=g, device=DEV)
        q[:, ::2, 0] = 7.0
        q = q.flatten(1).bfloat16()
        out = kv_q8.paged_decode_q8(q, *cache, table, ctx, Hq, Hkv, hd, torch.empty_like(q), ws)
        assert out.isfinite().all()
        for i in range(0, len(lens), max(1, len(lens) // 8)):
            t = torch.arange(lens[i], device=DEV)
            at = table[i].long()[t // bs], t % bs
            k, v = (c.view(torch.uint8)[at[0], :, at[1]].view(dtype).double() * s[at[0]].double()[..., None] for c, s in (cache[::2], cache[1::2]))
            ref, bound = attend(q[i].double().view(Hq, hd), k, v, dtype)
            # Sums are in units of at most twice a block's scale: a weight below 2^-14 in these is off by 2^-24 of its own, where
            # `bound` has 2^-25.  Where sums of 2^118 units leave no room for a smaller unit a weight is off by 2^-25 units: times
            # codes below 2^9 and fewer than 2^13 keys, beside a sum of at most 2^8 of the values, 2^(-25 + 9 + 13 + 8 - 118).
            tiny = 2.0 ** -25 * v.abs().sum(0) + 2.0 ** -113 * v.abs().sum(0).amax(-1, keepdim=True)
            bound = bound + tiny.repeat_interleave(Hq // Hkv, 0)
            off = (out[i].double().view(Hq, hd) - ref).abs()
            assert (off <= bound).all(), (i, lens[i], float((off / bound).max()))
