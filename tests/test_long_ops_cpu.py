"""Refusals of ops.long_attention / ops.token_logprobs and of their C entry points, without a GPU; the bucket borders of the distance bias."""
import ctypes
import math

import pytest
import torch

from vln_imagine_amd import _lib, ops


class Args(ctypes.Structure):                # VlniLongAttnArgs (include/vlni.h)
    _fields_ = [(n, ctypes.c_int) for n in ("dtype", "B", "Sq", "Sk", "nh", "nkv", "D", "causal")] + \
               [("scale", ctypes.c_float), ("rel_n", ctypes.c_int), ("rel_sides", ctypes.c_int), ("rel_first", ctypes.c_void_p)] + \
               [(n, ctypes.c_void_p) for n in ("q", "k", "v", "dout")] + \
               [(n, ctypes.c_long * 3) for n in ("q_stride", "k_stride", "v_stride", "do_stride")] + \
               [(n, ctypes.c_void_p) for n in ("kmask", "rel_table", "out", "out_low", "stat")] + \
               [("prep", ctypes.c_void_p), ("prep_floats", ctypes.c_long), ("work", ctypes.c_void_p), ("work_floats", ctypes.c_long)] + \
               [(n, ctypes.c_void_p) for n in ("dq", "dk", "dv", "dtable")]


def test_packed_arguments_have_the_structures_layout():
    assert ops._LA_ARGS.size == ctypes.sizeof(Args)
    vals = list(range(1, 9)) + [0.5] + list(range(10, 42))
    a = Args.from_buffer_copy(ops._LA_ARGS.pack(*vals))
    assert (a.dtype, a.causal, a.scale, a.rel_sides, a.rel_first, a.q, a.dout) == (1, 8, 0.5, 11, 12, 13, 16)
    assert list(a.q_stride) == [17, 18, 19] and list(a.do_stride) == [26, 27, 28]
    assert (a.kmask, a.rel_table, a.out, a.out_low, a.stat, a.prep, a.prep_floats, a.work, a.work_floats, a.dq, a.dtable) == (29, 30, 31, 32, 33, 34, 35, 36, 37, 38, 41)


def _qkv(B=2, Sq=5, Sk=7, nh=4, nkv=2, D=64, dtype=torch.float32):
    return torch.zeros(B, Sq, nh, D, dtype=dtype), torch.zeros(B, Sk, nkv, D, dtype=dtype), torch.zeros(B, Sk, nkv, D, dtype=dtype)


def test_long_attention_refuses():
    q, k, v = _qkv()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.long_attention(q, k, v)
    bad = [
        ((q[0], k, v), {}), ((q, k[:1], v[:1]), {}), ((q, k, v[:, :6]), {}), (_qkv(nh=3, nkv=2), {}), (_qkv(D=12), {}), (_qkv(D=136), {}), (_qkv(D=4), {}),
        ((q, k, v), dict(kmask=torch.zeros(2, 5))), ((q, k, v), dict(kmask=torch.ones(2, 7, dtype=torch.bool))), ((q, k, v), dict(kmask=torch.zeros(1, 7))),
        ((q, k, v), dict(kmask=torch.zeros(2, 7, requires_grad=True))), ((q, k, v), dict(scale=0.0)), ((q, k, v), dict(scale=float("nan"))), ((q, k, v), dict(scale=-1.0)),
        ((q, k, v), dict(rel_table=torch.zeros(31, 4))), ((q, k, v), dict(rel_table=torch.zeros(32, 2))), ((q, k, v), dict(rel_table=torch.zeros(32, 4, dtype=torch.float16))),
        ((q, k, v), dict(rel_table=torch.zeros(32, 4), rel_max=8)), ((q, k, v), dict(rel_table=torch.zeros(32, 4), rel_max=1025)),
        ((q, k, v), dict(rel_table=torch.zeros(32, 4), rel_max=20.5)), ((q, k, v), dict(rel_table=torch.zeros(2, 4))), ((q, k, v), dict(rel_table=torch.zeros(130, 4))),
    ]
    for args, kw in bad:
        with pytest.raises(ValueError):
            ops.long_attention(*args, **kw)
    with pytest.raises(TypeError):
        ops.long_attention(q, k.half(), v)
    with pytest.raises(TypeError):
        ops.long_attention(q.double(), k.double(), v.double())


def test_token_logprobs_refuses():
    x, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.token_logprobs(x, t)
    for args, kw in (((x, t.int()), {}), ((x, t[:2]), {}), ((x, t[:, None]), {}), ((x, t), dict(top=11)), ((torch.zeros(3, 40), t), dict(top=17)), ((x, t), dict(top=-1)),
                     ((torch.zeros(3, 0), t), {}),
                     ((torch.empty(2, (1 << 28) + 1, device="meta"), torch.empty(2, dtype=torch.int64, device="meta")), {}),
                     ((torch.empty(1 << 31, 1, device="meta"), torch.empty(1 << 31, dtype=torch.int64, device="meta")), {})):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args, **kw)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.double(), t)


def test_c_entry_points_refuse():
    """Every argument the kernels' addressing depends on is looked at before a launch (pointers here are made up: nothing may be read through them)."""
    lib = _lib.load()

    def args(**kw):
        a = Args()
        a.dtype, a.B, a.Sq, a.Sk, a.nh, a.nkv, a.D, a.scale = 1, 2, 5, 7, 4, 2, 64, 0.125
        for n in ("q", "k", "v", "dout", "out", "stat", "work", "dq", "dk", "dv"):
            setattr(a, n, 4096)
        for n in ("q_stride", "k_stride", "v_stride", "do_stride"):
            setattr(a, n, (ctypes.c_long * 3)(64 * 64, 64 * 4, 64))
        a.work_floats = 1 << 40
        for n, v in kw.items():
            setattr(a, n, v)
        return a
    three = (ctypes.c_long * 3)
    first = (ctypes.c_int * 4)(0, 1, 2, 4)
    wrong = [dict(dtype=3), dict(B=0), dict(Sq=0), dict(Sk=-1), dict(nkv=3), dict(D=60), dict(D=192), dict(scale=0.0), dict(Sk=(1 << 24) + 1), dict(q=4104), dict(k=0), dict(v=4100),
             dict(k_stride=three(1, 64, 64)), dict(out=0), dict(out_low=4104), dict(stat=0), dict(kmask=4096), dict(prep=4096, prep_floats=3, kmask=4096),
             dict(rel_table=4096, rel_n=4, rel_sides=2), dict(rel_table=4096, rel_n=65, rel_sides=1, rel_first=ctypes.addressof(first)),
             dict(rel_table=4096, rel_n=3, rel_sides=3, rel_first=ctypes.addressof(first))]
    for kw in wrong:
        for fn in (lib.vlni_long_attn_fwd, lib.vlni_long_attn_bwd):
            assert fn(ctypes.addressof(args(**kw)), 0) < 0, kw
            assert lib.vlni_last_error()
    for kw in (dict(dout=8), dict(dq=0), dict(dv=4100), dict(work=0), dict(work_floats=3), dict(dtable=4096), dict(do_stride=three(4, 64, 64))):
        assert lib.vlni_long_attn_bwd(ctypes.addressof(args(**kw)), 0) < 0, kw
    bad_first = (ctypes.c_int * 4)(0, 3, 2, 4)
    far_first = (ctypes.c_int * 4)(0, 3, 5, 2000)
    for f in (bad_first, far_first):
        assert lib.vlni_long_attn_fwd(ctypes.addressof(args(rel_table=4096, rel_n=4, rel_sides=1, rel_first=ctypes.addressof(f))), 0) < 0
    sizes = three()
    assert lib.vlni_long_attn_sizes(ctypes.addressof(args(Sq=1, Sk=8191, nh=16, nkv=4)), ctypes.addressof(sizes)) == 0 and sizes[0] == 0 and sizes[1] > 0
    assert lib.vlni_long_attn_fwd(ctypes.addressof(args(Sq=1, Sk=8191, work_floats=16)), 0) < 0
    f, b = lib.vlni_token_logprobs_fwd, lib.vlni_token_logprobs_bwd
    good = [1, 4096, 10, 4096, -100, 4096, 4096, 4096, 4096, 4096, 2, 3, 10, 0]
    for i, v in ((0, 5), (1, 0), (2, 9), (3, 0), (5, 0), (7, 0), (8, 0), (10, 17), (10, 11), (10, -1), (11, 0), (12, 0)):
        assert f(*[v if n == i else x for n, x in enumerate(good)]) < 0, (i, v)
    good = [1, 4096, 4096, 4096, 10, 4096, -100, 4096, 4096, 10, 3, 10, 0]
    for i, v in ((0, -1), (3, 0), (4, 9), (5, 0), (7, 0), (8, 0), (9, 9), (10, 0), (11, 0)):
        assert b(*[v if n == i else x for n, x in enumerate(good)]) < 0, (i, v)


@pytest.mark.parametrize("n,rel_max", [(2, 5), (4, 16), (16, 128), (16, 37), (13, 300), (64, 1024), (64, 33), (5, 3)])
def test_bucket_borders(n, rel_max):
    """first[b] is the smallest distance whose bucket is >= b, by the definition floor((n - e) log(d / e) / log(rel_max / e)) with a margin for its rounding."""
    first, e = list(ops.rel_bucket_starts(n, rel_max)), n // 2
    assert len(first) == n and first[0] == 0 and first == sorted(first) and first[-1] <= rel_max

    def bucket(d):
        return d if d < e else min(n - 1, e + math.floor((n - e) * math.log(d / e) / math.log(rel_max / e) + 1e-9))
    for d in range(rel_max + 50):
        assert sum(d >= f for f in first) - 1 == bucket(d), d
