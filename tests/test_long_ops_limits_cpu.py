"""Sizes beyond what a launch holds (2^32 threads) are refused by name, without a GPU."""
import ctypes

import pytest
import torch

from tests.test_long_ops_cpu import Args
from vln_imagine_amd import _lib, ops


def _args(**kw):
    a = Args()
    a.dtype, a.B, a.Sq, a.Sk, a.nh, a.nkv, a.D, a.scale = 1, 2, 5, 7, 4, 2, 64, 0.125
    for n in ("q", "k", "v", "dout", "out", "stat", "work", "dq", "dk", "dv"):
        setattr(a, n, 4096)
    for n in ("q_stride", "k_stride", "v_stride", "do_stride"):
        setattr(a, n, (ctypes.c_long * 3)(64 * 64, 64 * 4, 64))
    a.work_floats = a.prep_floats = 1 << 50
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw", [dict(B=1 << 22, Sq=1, nh=8, nkv=8), dict(B=1 << 21, Sq=200, nh=8, nkv=1), dict(B=1 << 23, Sk=1, nkv=4), dict(B=128, Sq=1 << 24, Sk=1, nh=4, nkv=1),
                                dict(B=64, Sk=1 << 24, Sq=1, nh=2, nkv=2), dict(B=1 << 9, Sk=1 << 24, Sq=1, nh=1, nkv=1, kmask=4096, prep=4096)])
def test_more_blocks_than_a_launch_holds(kw):
    lib = _lib.load()
    a, sizes = _args(**kw), (ctypes.c_long * 3)()
    for rc in (lib.vlni_long_attn_sizes(ctypes.addressof(a), ctypes.addressof(sizes)), lib.vlni_long_attn_fwd(ctypes.addressof(a), 0), lib.vlni_long_attn_bwd(ctypes.addressof(a), 0)):
        assert rc < 0 and b"more than one launch holds" in lib.vlni_last_error()


def test_the_largest_that_fit():
    lib, sizes = _lib.load(), (ctypes.c_long * 3)()
    for kw in (dict(B=1 << 21, Sq=1, nh=4, nkv=4), dict(B=1, Sq=1 << 24, Sk=1 << 24, nh=2, nkv=2), dict(B=60, Sk=1 << 24, Sq=1, nh=2, nkv=2)):
        assert lib.vlni_long_attn_sizes(ctypes.addressof(_args(**kw)), ctypes.addressof(sizes)) == 0, kw


@pytest.mark.parametrize("rows,V", [(1 << 26, 40), (1 << 26, 2040), (1 << 24, 2041), (1 << 24, 2048), (1 << 24, 5000), ((1 << 31) - 1, 1)])
def test_more_rows_than_a_launch_holds(rows, V):
    with pytest.raises(ValueError, match="rows"):
        ops.token_logprobs(torch.empty(rows, V, device="meta"), torch.empty(rows, dtype=torch.int64, device="meta"))
    lib = _lib.load()
    assert lib.vlni_token_logprobs_fwd(1, 4096, V, 4096, -100, 4096, 4096, 4096, 0, 0, 0, rows, V, 0) < 0 and b"rows of" in lib.vlni_last_error()
    assert lib.vlni_token_logprobs_bwd(1, 4096, 4096, 4096, V, 4096, -100, 4096, 4096, V, rows, V, 0) < 0 and b"rows of" in lib.vlni_last_error()


def test_the_most_rows_reach_the_device_check():
    for rows, V in (((1 << 26) - 1, 40), ((1 << 24) - 1, 2041)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            ops.token_logprobs(torch.empty(rows, V, device="meta"), torch.empty(rows, dtype=torch.int64, device="meta"))
