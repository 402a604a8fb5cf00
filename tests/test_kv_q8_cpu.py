"""What the front-ends of the 8-bit cache refuse, before any kernel is loaded."""
import pytest
import torch

from art_b200.ops import kv_q8

E4, I8, BF = torch.float8_e4m3fn, torch.int8, torch.bfloat16


def cache(nb=4, kv=2, bs=16, hd=64, dtype=E4):
    c = lambda: torch.zeros(nb, kv, bs, hd, dtype=dtype)      # noqa: E731
    return c(), c(), torch.zeros(nb, kv), torch.zeros(nb, kv)


def write(c, qkv=None, k_col=128, v_col=256, slot=None):
    qkv = torch.zeros(3, 384, dtype=BF) if qkv is None else qkv
    kv_q8.kv_write_q8(qkv, k_col, v_col, torch.zeros(qkv.shape[0], dtype=torch.int32) if slot is None else slot, *c)


def rows(c, dst=None, slot=None, k_col=0, v_col=128):
    dst = torch.zeros(3, 256, dtype=BF) if dst is None else dst
    kv_q8.kv_rows_q8(*c, torch.zeros(3, dtype=torch.int32) if slot is None else slot, dst, k_col, v_col)


SAME, FUSED = torch.zeros(3, 256, dtype=BF), torch.zeros(4, 512, dtype=BF)


def decode(c, q=None, table=None, ctx=None, heads=(4, 2, 64), out=None, ws=None):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)         # noqa: E731
    q = torch.zeros(3, 256, dtype=BF) if q is None else q
    kv_q8.paged_decode_q8(q, *c, z(3, 2) if table is None else table, z(3) if ctx is None else ctx, *heads,
                          torch.zeros(3, 256, dtype=BF) if out is None else out, torch.zeros(64, dtype=torch.uint8) if ws is None else ws)


@pytest.mark.parametrize("call", [write, rows, decode])
@pytest.mark.parametrize("change,says", [
    (lambda c: (c[0], c[1].to(I8), *c[2:]), "differ"),
    (lambda c: (c[0][:, :, :8], c[1][:, :, :8], *c[2:]), "multiple of 16"),
    (lambda c: (c[0].to(torch.float8_e5m2), c[1].to(torch.float8_e5m2), *c[2:]), "float8_e4m3fn or int8"),
    (lambda c: (c[0].to(BF), c[1].to(BF), *c[2:]), "float8_e4m3fn or int8"),
    (lambda c: (c[0].view(4, 2, 32, 32).view(4, 2, 64, 16), c[1].view(4, 2, 64, 16), *c[2:]), "head dim 16"),
    (lambda c: (c[0], c[1], c[2][:3], c[3]), "k_scale"),
    (lambda c: (c[0], c[1], c[2], c[3].double()), "v_scale"),
    (lambda c: (c[0].transpose(0, 1).contiguous().transpose(0, 1), *c[1:]), "contiguous"),
    (lambda c: c, "one CUDA device"),                         # all else is in order: tensors of the CPU
])
def test_caches(call, change, says):
    with pytest.raises(ValueError, match=says):
        call(change(cache()))


@pytest.mark.parametrize("kw,says", [
    (dict(qkv=torch.zeros(3, 384)), "bf16"),
    (dict(qkv=torch.zeros(384, 3, dtype=BF).t()), "unit inner stride"),
    (dict(k_col=4), "multiples of 8"),
    (dict(v_col=264), "does not hold"),
    (dict(k_col=-8), "does not hold"),
    (dict(qkv=torch.zeros(3, 388, dtype=BF)[:, :384]), "16 bytes"),
    (dict(slot=torch.zeros(2, dtype=torch.int32)), "slot"),
    (dict(slot=torch.zeros(3, dtype=torch.int64)), "slot"),
    (dict(slot=torch.zeros(6, dtype=torch.int32)[::2]), "slot"),
])
def test_writes(kw, says):
    with pytest.raises(ValueError, match=says):
        write(cache(), **kw)


@pytest.mark.parametrize("kw,says", [
    (dict(v_col=64), "overlap"),
    (dict(dst=torch.zeros(1, 256, dtype=BF).expand(3, 256)), "overlap"),
    (dict(dst=torch.zeros(2, 256, dtype=BF)), "3 slots for 2 rows"),
    (dict(slot=torch.zeros(1, 3, dtype=torch.int32)), "slot"),
])
def test_rows(kw, says):
    with pytest.raises(ValueError, match=says):
        rows(cache(), **kw)


@pytest.mark.parametrize("kw,says", [
    (dict(heads=(5, 2, 64)), "query heads"),
    (dict(heads=(34, 2, 64)), "at most 16"),
    (dict(heads=(4, 4, 64)), "the cache has 2 of 64"),
    (dict(heads=(4, 2, 32)), "the cache has 2 of 64"),
    (dict(heads=(0, 2, 64)), "query heads"),
    (dict(q=torch.zeros(3, 128, dtype=BF)), "does not hold"),
    (dict(q=torch.zeros(3, 256)), "bf16"),
    (dict(out=torch.zeros(2, 256, dtype=BF)), "out must have 3 rows"),
    (dict(out=torch.zeros(1, 256, dtype=BF).expand(3, 256)), "overlap"),
    (dict(q=SAME, out=SAME), "nor lie where q does"),
    (dict(q=FUSED[:3, :256], out=FUSED[:3, 248:504]), "nor lie where q does"),
    (dict(q=FUSED[:3, 256:], out=FUSED[:3, 8:264]), "nor lie where q does"),
    (dict(q=FUSED[:3, :256], out=FUSED[1:, :256]), "nor lie where q does"),       # the next row's query
    (dict(q=FUSED[:3, :256], out=FUSED.view(8, 256)[1:4]), "nor lie where q does"),
    (dict(q=FUSED[:3, :256], out=FUSED[:3, 256:]), "one CUDA device"),            # beside it: in order
    (dict(q=FUSED[:3, 256:], out=FUSED[1:, :256]), "one CUDA device"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int32)), "block_table"),
    (dict(table=torch.zeros(3, 0, dtype=torch.int32)), "block_table"),
    (dict(table=torch.zeros(3, 2)), "block_table"),
    (dict(table=torch.zeros(3, 4, dtype=torch.int32)[:, ::2]), "block_table"),
    (dict(ctx=torch.zeros(2, dtype=torch.int32)), "ctx_len"),
    (dict(ctx=torch.zeros(3)), "ctx_len"),
])
def test_decode(kw, says):
    with pytest.raises(ValueError, match=says):
        decode(cache(), **kw)


def finish(c, M=3, heads=(4, 2, 64), pos=None, slot=None, q=None, ws=None, **kw):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)         # noqa: E731
    kv_q8.decode_finalize_qkv_q8(torch.zeros(4, 512) if ws is None else ws, M, *heads, 0, z(3) if pos is None else pos, 1e6, z(3) if slot is None else slot,
                                 *c, torch.zeros(3, 256, dtype=BF) if q is None else q, **kw)


@pytest.mark.parametrize("kw,says", [
    (dict(heads=(3, 2, 64)), "even"),
    (dict(heads=(4, 4, 64)), "the cache has 2 of 64"),
    (dict(heads=(4, 2, 32)), "the cache has 2 of 64"),
    (dict(M=4), "slot"),
    (dict(pos=torch.zeros(3)), "pos"),
    (dict(q=torch.zeros(2, 256, dtype=BF)), "q_out"),
    (dict(ws=torch.zeros(2, 512)), "ws must be"),
    (dict(ws=torch.zeros(4, 504)), "ws must be"),
    (dict(ws=torch.zeros(4, 512, dtype=BF)), "ws must be"),
    (dict(ws=torch.zeros(512, 4).t()), "ws must be"),
    (dict(bias=torch.zeros(512, dtype=BF)), "bias must be"),
    (dict(bias=torch.zeros(511)), "bias must be"),
    (dict(q_norm=torch.zeros(64), k_norm=torch.zeros(64, dtype=BF)), "q_norm must be"),
    (dict(q_norm=torch.zeros(64, dtype=BF), k_norm=torch.zeros(128, dtype=BF)[::2]), "k_norm must be"),
    (dict(adapter=torch.zeros(2, dtype=torch.int32)), "adapter must be"),
    (dict(adapter=torch.zeros(3, dtype=torch.int32)), "B_all must be"),
    (dict(adapter=torch.zeros(3, dtype=torch.int32), B_all=torch.zeros(8, 504, dtype=BF)), "B_all must be"),
    (dict(adapter=torch.zeros(3, dtype=torch.int32), B_all=torch.zeros(8, 512)), "B_all must be"),
    (dict(), "one CUDA device"),
])
def test_finish(kw, says):
    with pytest.raises(ValueError, match=says):
        finish(cache(), **kw)
