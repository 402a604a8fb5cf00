"""Front-ends of a paged cache of keys and values held in 8 bits: write, read-back, decode attention.

A cache is four tensors of a layer: codes ``k_cache`` and ``v_cache`` ``[blocks, Hkv, block_size, hd]`` (``torch.float8_e4m3fn``
or ``torch.int8``) and scales ``k_scale`` and ``v_scale`` ``[blocks, Hkv]`` fp32.  A value is its code times the scale of its
block and kv head; scales are powers of two (csrc/include/kv_q8.cuh).  A zeroed cache is an empty one.

Half the bytes of the bf16 cache (:mod:`.paged`), which is what bounds both the number of sequences that run at a time and decode
attention.  ``e4m3`` keeps 4 significant bits of every value, ``int8`` an absolute step of less than 1/63 of the largest value in
the block and head.  The reference has the choice as ``engine_args.kv_cache_dtype`` (src/art/dev/engine.py:24) of the engine it
serves through.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import _lib

vp, ci, cl = ctypes.c_void_p, ctypes.c_int, ctypes.c_long
# The launches that a layer makes take their arguments as one block of memory, laid out as the C structs of these names
# (csrc/include/kv_q8.cuh): ctypes takes 0.1 us for each argument that it converts, and the kernels take a few.
_blocks = {
    "artb_kv_write_q8": struct.Struct("PPPPPPP q iiiiiiii"),
    "artb_kv_rows_q8": struct.Struct("PPPPPPP q iiiiiiii"),
    "artb_paged_decode_q8": struct.Struct("PPPPPPPPPP q iiiiiiiii"),
}
_sigs = {
    **{name: [ctypes.c_char_p, vp] for name in _blocks},
    "artb_paged_decode_q8_bytes": [ci, ci, ci, ci],
    "artb_decode_finalize_qkv_q8": [vp, ci, ci, ci, ci, ci, ci, vp, vp, vp, ci, ci, vp, ctypes.c_float, vp, vp, ctypes.c_float, vp, vp,
                                    vp, vp, vp, ci, ci, vp, ci, cl, vp, vp],
}
_bound: dict[str, object] = {}

BF16, I32, F32 = torch.bfloat16, torch.int32, torch.float32
KINDS = {torch.float8_e4m3fn: 0, torch.int8: 1}
HEAD_DIMS = (32, 64, 128)


def _f(name: str):
    fn = _bound.get(name)
    if fn is None:
        fn = getattr(_lib.kernels(), name)
        fn.argtypes = _sigs[name]
        fn.restype = ci
        _bound[name] = fn
    return fn


MOST_HEADS = 16                 # query heads of a kv head


def check_geometry(dtype: torch.dtype, block_size: int, hd: int, group: int = 1) -> None:
    """Refuses what the kernels do not cover; ``group``: query heads of a kv head."""
    if dtype not in KINDS:
        raise ValueError(f"a cache of {dtype}: codes are float8_e4m3fn or int8")
    if block_size < 16 or block_size % 16:
        raise ValueError(f"blocks of {block_size} tokens: a cache in 8 bits has blocks of a multiple of 16")
    if hd not in HEAD_DIMS:
        raise ValueError(f"head dim {hd}: a cache in 8 bits takes {', '.join(map(str, HEAD_DIMS))}")
    if group > MOST_HEADS:
        raise ValueError(f"{group} query heads to a kv head: a cache in 8 bits takes at most {MOST_HEADS}")


def _check_cache(k_cache, v_cache, k_scale, v_scale) -> None:
    """Says what is wrong with a cache."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} {k_cache.dtype} and v_cache {tuple(v_cache.shape)} {v_cache.dtype} differ "
                         "or are not [blocks, Hkv, block_size, hd]")
    nb, hkv, bs, hd = k_cache.shape
    check_geometry(k_cache.dtype, bs, hd)
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s.shape != (nb, hkv) or s.dtype != torch.float32 or not s.is_contiguous():
            raise ValueError(f"{name} must be contiguous fp32 [{nb}, {hkv}]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache and v_cache must be contiguous")
    raise ValueError(f"a cache of {nb} blocks and {hkv} kv heads")


def _geometry(k_cache, v_cache, k_scale, v_scale) -> tuple[int, int, int, int, int]:
    """(blocks, Hkv, block_size, hd, kind) of a cache that is one.  These checks run before every launch, and a launch takes the
    GPU a few microseconds: what is in order is found so with as few calls as there are conditions."""
    shape, dtype = k_cache.shape, k_cache.dtype
    kind = KINDS.get(dtype)
    if len(shape) == 4 and kind is not None and v_cache.shape == shape and v_cache.dtype is dtype:
        nb, hkv, bs, hd = shape
        scales = (nb, hkv)
        if (nb > 0 and hkv > 0 and bs > 0 and bs % 16 == 0 and hd in HEAD_DIMS and k_scale.shape == scales and v_scale.shape == scales
                and k_scale.dtype is v_scale.dtype is F32 and k_cache.is_contiguous() and v_cache.is_contiguous()
                and k_scale.is_contiguous() and v_scale.is_contiguous()):
            return nb, hkv, bs, hd, kind
    _check_cache(k_cache, v_cache, k_scale, v_scale)


def _rows(name: str, x: torch.Tensor, lo: int, hi: int, width: int) -> tuple[int, int, int]:
    """(rows, row stride, address) of ``x`` [rows, ld] bf16 that holds ``width`` columns from ``lo`` and from ``hi`` on, in pieces of
    16 bytes."""
    shape, stride, at = x.shape, x.stride(), x.data_ptr()
    if len(shape) == 2 and x.dtype is BF16:
        n, cols = shape
        ld, inner = stride
        if n < 2:                              # a stride that leads nowhere
            ld = cols + -cols % 8
        if inner == 1 and not (lo | hi | ld) & 7 and not at & 15 and lo >= 0 and hi >= 0 and lo + width <= cols and hi + width <= cols:
            return n, ld, at
        if inner == 1:
            if lo < 0 or hi < 0 or lo % 8 or hi % 8 or max(lo, hi) + width > cols:
                raise ValueError(f"{name} [{n}, {cols}] does not hold {width} columns at {lo} and {hi}, multiples of 8")
            raise ValueError(f"{name}: rows must begin on 16 bytes")
    raise ValueError(f"{name} must be bf16 [rows, columns] with unit inner stride")


def _index(name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype is not I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{n}]")


def _device(*tensors: torch.Tensor) -> int:
    """Number of the CUDA device that all tensors lie on."""
    devices = {t.get_device() for t in tensors}
    dev = devices.pop()
    if devices or dev < 0:
        raise ValueError(f"tensors of one CUDA device are needed: {', '.join(sorted({str(t.device) for t in tensors}))}")
    return dev


def _launch(dev: int, name: str, *args) -> None:
    """On the current stream of device ``dev``, whichever device is current; ``args`` end before the status word."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _launch(dev, name, *args)
    fn, word, stream = _bound.get(name) or _f(name), _lib.status_word(dev).data_ptr(), _lib.raw_stream(dev)
    rc = fn(_blocks[name].pack(word, *args), stream) if name in _blocks else fn(*args, word, stream)
    if rc:
        _lib.check_rc(rc, name.removeprefix("artb_"))
    _lib.LAUNCHES += 1


def kv_write_q8(qkv: torch.Tensor, k_col: int, v_col: int, slot: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Quantises the keys and values of the rows of ``qkv`` (bf16 [M, >= ...], columns ``k_col`` and ``v_col`` on) into the cache.
    ``slot`` int32 [M]: block * block_size + place, negative: the row is not written.  The rows that go to one block are neighbours and
    go to consecutive places, as those of a prompt and of a decode step do.  A row that comes behind others of its block and is not
    their neighbour at the next place, rows that are not written between them or not, is not written and reported through the status
    word, as are slots beyond the cache.  Calls of up to 256 rows report it of blocks that take turns (5, 40, 6 in blocks of 16) too;
    in longer calls such blocks are not found, and what they then hold is undefined.

    The scale of a block and head is the least power of two that takes the largest value written to it into the range of the
    codes.  A row at a block's first place starts the block anew.  Rows at later places can only raise the scale, and then what
    the block holds already is rounded once more.  A value that is not finite makes the scale NaN until the block starts anew."""
    nb, hkv, bs, hd, kind = _geometry(k_cache, v_cache, k_scale, v_scale)
    n, ld, at = _rows("qkv", qkv, k_col, v_col, hkv * hd)
    _index("slot", slot, n)
    dev = qkv.get_device()
    if not (0 <= dev == slot.get_device() == k_cache.get_device() == v_cache.get_device() == k_scale.get_device() == v_scale.get_device()):
        _device(qkv, slot, k_cache, v_cache, k_scale, v_scale)
    _launch(dev, "artb_kv_write_q8", at, slot.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), nb, n, ld, k_col, v_col, hkv, hd, bs, kind)


def decode_finalize_qkv_q8(ws: torch.Tensor, M: int, Hq: int, Hkv: int, hd: int, kpad: int, pos: torch.Tensor, theta: float,
                           slot: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                           v_scale: torch.Tensor, q_out: torch.Tensor, *, bias: torch.Tensor | None = None,
                           adapter: torch.Tensor | None = None, B_all: torch.Tensor | None = None, cols: int = 0,
                           q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6) -> None:
    """:func:`~art_b200.ops.paged.decode_finalize_qkv` into a cache in 8 bits, the same numbers as that and :func:`kv_write_q8` of
    its bf16 rows in one launch.  No two of the ``M`` slots lie in one block, as in a decode step: the later row of
    such two is not written and reported through the status word.  ``Hq + Hkv`` is even (:func:`finalize_covers`)."""
    nb, hkv, bs, d, kind = _geometry(k_cache, v_cache, k_scale, v_scale)
    if hkv != Hkv or d != hd or not finalize_covers(Hq, Hkv):
        raise ValueError(f"{Hq} query heads and {Hkv} kv heads of {hd}: the cache has {hkv} of {d}, and the number of both must be even")
    _index("slot", slot, M)
    _index("pos", pos, M)
    n, ldq, to = _rows("q_out", q_out, 0, 0, Hq * hd)
    N = (Hq + 2 * Hkv) * hd
    if (ws.dtype is not F32 or ws.dim() != 2 or ws.shape[0] < M or ws.shape[1] < N + (kpad if adapter is not None else 0) or ws.stride(1) != 1
            or n != M):
        raise ValueError(f"ws must be fp32 [>= {M}, >= {N} and the low-rank columns], and q_out have {M} rows")
    given = []
    for name, t, dtype, size in (("bias", bias, F32, N), ("adapter", adapter, I32, M), ("q_norm", q_norm, BF16, hd), ("k_norm", k_norm, BF16, hd)):
        if t is not None:
            if t.dtype is not dtype or t.numel() < size or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dtype} of {size} numbers")
            given.append(t)
    if adapter is not None:
        if B_all is None or B_all.dtype is not BF16 or B_all.dim() != 2 or B_all.shape[1] < N or B_all.stride(1) != 1:
            raise ValueError(f"B_all must be bf16 [rows of all adapters, >= {N}]")
        given.append(B_all)
    dev = _device(ws, pos, slot, k_cache, v_cache, k_scale, v_scale, q_out, *given)
    ptr = lambda t: 0 if t is None else t.data_ptr()      # noqa: E731
    _launch(dev, "artb_decode_finalize_qkv_q8", ws.data_ptr(), ws.stride(0), M, Hq, Hkv, hd, kpad, ptr(bias), ptr(adapter), ptr(B_all),
            B_all.stride(0) if B_all is not None else 0, cols, pos.data_ptr(), theta, ptr(q_norm), ptr(k_norm), eps, slot.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), bs, kind, to, ldq, nb)


def finalize_covers(Hq: int, Hkv: int) -> bool:
    """Whether :func:`decode_finalize_qkv_q8` takes these numbers of heads."""
    return (Hq + Hkv) % 2 == 0 and Hkv <= 128


def kv_rows_q8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, slot: torch.Tensor,
               dst: torch.Tensor, k_col: int, v_col: int) -> None:
    """The cached keys and values at ``slot`` (int32 [n]) as bf16 into the k and v columns of ``dst[:n]``; zeros where negative."""
    nb, hkv, bs, hd, kind = _geometry(k_cache, v_cache, k_scale, v_scale)
    have, ld, to = _rows("dst", dst, k_col, v_col, hkv * hd)
    if abs(k_col - v_col) < hkv * hd or ld < max(k_col, v_col) + hkv * hd:
        raise ValueError("the columns of keys and values, or the rows of dst, overlap")
    n = slot.numel()
    _index("slot", slot, n)
    if n > have:
        raise ValueError(f"{n} slots for {have} rows")
    dev = dst.get_device()
    if not (0 <= dev == slot.get_device() == k_cache.get_device() == v_cache.get_device() == k_scale.get_device() == v_scale.get_device()):
        _device(dst, slot, k_cache, v_cache, k_scale, v_scale)
    _launch(dev, "artb_kv_rows_q8", to, slot.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), nb, n, ld, k_col, v_col, hkv, hd, bs, kind)


def _meet(a: int, lda: int, b: int, ldb: int, n: int, width: int) -> bool:
    """Whether ``n`` rows of ``width`` 16-bit numbers at address ``a`` and as many at ``b`` may share bytes; of rows of one stride
    that lie among each other, whether they do."""
    if b >= a + 2 * (lda * (n - 1) + width) or a >= b + 2 * (ldb * (n - 1) + width):
        return False
    return lda != ldb or not 2 * width <= (b - a) % (2 * ldb) <= 2 * (ldb - width)


@functools.lru_cache(maxsize=1024)
def _decode_bytes(n: int, Hq: int, Hkv: int, hd: int, device: int) -> int:
    with torch.cuda.device(device):
        return _f("artb_paged_decode_q8_bytes")(n, Hq, Hkv, hd)


def decode_q8_workspace(n: int, Hq: int, Hkv: int, hd: int, device) -> torch.Tensor:
    """Workspace of :func:`paged_decode_q8` for up to ``n`` sequences of these heads; one call at a time may use it."""
    dev = torch.device(device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    return torch.zeros(_decode_bytes(n, Hq, Hkv, hd, index), dtype=torch.uint8, device=dev)


def paged_decode_q8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                    block_table: torch.Tensor, ctx_len: torch.Tensor, Hq: int, Hkv: int, hd: int, out: torch.Tensor,
                    ws: torch.Tensor) -> torch.Tensor:
    """Attention of one token per sequence over the first ``ctx_len`` cached tokens: q bf16 [n, >= Hq*hd] (row stride arbitrary),
    ``block_table`` int32 [n, width], ``ctx_len`` int32 [n] (0: the row becomes zeros); out bf16 [n, >= Hq*hd].  Scales are as
    :func:`kv_write_q8` leaves them.  Values of 2^120 / ``ctx_len`` and more may overflow the fp32 sums.  Entries that are no block
    and lengths that the table cannot hold are reported through the status word; such keys are left out.  The same inputs give the
    same bits."""
    nb, hkv, bs, d, kind = _geometry(k_cache, v_cache, k_scale, v_scale)
    if hkv != Hkv or d != hd or Hq <= 0 or Hq % Hkv or Hq > MOST_HEADS * Hkv:
        raise ValueError(f"{Hq} query heads of {hd} over {Hkv} kv heads: the cache has {hkv} of {d}, and a kv head serves at most {MOST_HEADS}")
    n, ldq, at = _rows("q", q, 0, 0, Hq * hd)
    m, ldo, to = _rows("out", out, 0, 0, Hq * hd)
    if m != n or ldo < Hq * hd or (abs(to - at) < 2 * n * max(ldq, ldo) and _meet(at, ldq, to, ldo, n, Hq * hd)):
        raise ValueError(f"out must have {n} rows that do not overlap, nor lie where q does")
    _index("ctx_len", ctx_len, n)
    table = block_table.shape
    if block_table.dtype is not I32 or len(table) != 2 or table[0] != n or table[1] < 1 or not block_table.is_contiguous():
        raise ValueError(f"block_table must be contiguous int32 [{n}, width]")
    dev = q.get_device()
    if not (0 <= dev == k_cache.get_device() == v_cache.get_device() == k_scale.get_device() == v_scale.get_device()
            == block_table.get_device() == ctx_len.get_device() == out.get_device() == ws.get_device()):
        _device(q, k_cache, v_cache, k_scale, v_scale, block_table, ctx_len, out, ws)
    if n and (ws.nbytes < _decode_bytes(n, Hq, Hkv, hd, dev) or not ws.is_contiguous()):
        raise ValueError(f"workspace of {ws.nbytes} bytes, {_decode_bytes(n, Hq, Hkv, hd, dev)} needed in a row")
    _launch(dev, "artb_paged_decode_q8", at, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            block_table.data_ptr(), ctx_len.data_ptr(), to, ws.data_ptr(), nb, n, ldq, ldo, Hq, Hkv, hd, bs, table[1], kind)
    return out
