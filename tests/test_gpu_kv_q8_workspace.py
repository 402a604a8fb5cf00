"""The workspace of decode attention over the 8-bit cache: one for calls of any lengths, its counters zero after each."""
import pytest
import torch

from .test_gpu_kv_q8 import DEV, KINDS, filled, pages

pytestmark = pytest.mark.gpu


@KINDS
@pytest.mark.parametrize("Hq,Hkv,hd,bs", [(8, 4, 32, 16), (28, 4, 128, 16), (24, 2, 64, 32)])
def test_one_workspace_for_calls_of_any_lengths(dtype, Hq, Hkv, hd, bs):
    from art_b200.ops import _lib, kv_q8

    calls = [[6000], [1, 0, 4001, 33], [700] * 300, [(37 * i) % 400 for i in range(512)], [9000, 9000], [40] * 1200, [31] * 3 + [8000]]
    most = max(map(len, calls))
    ws = kv_q8.decode_q8_workspace(most, Hq, Hkv, hd, DEV)
    counters = ws[ws.numel() - (most * Hkv + 3) // 4 * 16:]
    for lens in calls:
        g = torch.Generator(device=DEV).manual_seed(len(lens))
        bt, nb = pages(lens, bs)
        cache, table = filled(nb, Hkv, bs, hd, dtype, g), bt.to(DEV)
        ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
        q = torch.randn(len(lens), Hq * hd, generator=g, device=DEV).bfloat16()
        fresh = kv_q8.decode_q8_workspace(len(lens), Hq, Hkv, hd, DEV)
        want = kv_q8.paged_decode_q8(q, *cache, table, ctx, Hq, Hkv, hd, torch.empty_like(q), fresh)
        out = kv_q8.paged_decode_q8(q, *cache, table, ctx, Hq, Hkv, hd, torch.full_like(q, 7.0), ws)
        assert torch.equal(out, want) and not counters.any()
    _lib.check_status()
