"""Addresses that the kernels of the 8-bit cache cannot load from are refused before a launch.  The addresses are made up: nothing here
may reach a GPU."""
import ctypes

import pytest
import torch

from art_b200.ops import kv_q8

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls with made-up addresses")
AT = 1 << 20
ALIGN = -2


def finish(**odd):
    a = {k: AT + odd.get(k, 0) for k in ("ws", "bias", "adapter", "B_all", "pos", "q_norm", "k_norm", "slot", "k", "v", "ks", "vs", "out")}
    args = (a["ws"], 576, 3, 4, 2, 64, 64, a["bias"], a["adapter"], a["B_all"], 512, 24, a["pos"], 1e6, a["q_norm"], a["k_norm"], 1e-6,
            a["slot"], a["k"], a["v"], a["ks"], a["vs"], 16, 0, a["out"], 256, 4, None, None)
    return kv_q8._f("artb_decode_finalize_qkv_q8")(*args)


@pytest.mark.parametrize("name", ["ws", "bias", "B_all", "q_norm", "k_norm", "k", "v", "out"])
@pytest.mark.parametrize("by", [4, 8])
def test_finish(name, by):
    assert finish(**{name: by}) == ALIGN


def packed(name, *args):
    return kv_q8._f(name)(kv_q8._blocks[name].pack(0, *args), ctypes.c_void_p())


@pytest.mark.parametrize("name", ["artb_kv_write_q8", "artb_kv_rows_q8"])
@pytest.mark.parametrize("which", [0, 2, 3])
def test_rows(name, which):
    at = [AT] * 6                            # rows, slots, codes, scales
    at[which] += 8
    assert packed(name, *at, 4, 3, 384, 128, 256, 2, 64, 16, 0) == ALIGN


@pytest.mark.parametrize("which", [0, 1, 2, 7, 8])
def test_decode(which):
    at = [AT] * 9                            # q, codes, scales, table, lengths, out, workspace
    at[which] += 8
    assert packed("artb_paged_decode_q8", *at, 4, 3, 256, 256, 4, 2, 64, 16, 2, 0) == ALIGN
