"""GPU: ops.long_attention (forward, backward, learned distance bias) against the formulas in float64.

Bounds are elementwise and follow from the arithmetic, with u = eps / 2 of the 16-bit type (0 for float32, whose products are exact to the accumulator):
  scores   |dt| <= 2^-24 (D scale <|q|,|k|> + 4 |t| + 4 |row maximum|), so P is off by at most epsP = 2 max|dt| + 2^-20 relative (the float32 exp2 and the sum's own
           rounding are inside 2^-20), sums of n terms by n 2^-24 of the sum of magnitudes;
  out      (u + epsP + n 2^-24) P|V| + u |out|            (P rounded once, out rounded once)
  delta    |dO| . (error of out, whose own rounding is kept beside it to u^2 |out| in 16 bits) + D 2^-24 |dO|.|out|
  dS       u |dS| + epsP |dS| + P (error of delta + D 2^-24 |dO|.|V|)
  dV, dQ, dK   the same sums over the errors of P and dS, and one rounding of the result; the table's gradient sums dS before it is rounded
           and with delta from the rows' own sums.
float16 adds half its smallest step (2^-25) wherever a P, a dS or a result below its normal range is rounded."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a MI355X"
    from vln_imagine_amd import ops as o
    return o


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def _bucket(rel, nb, rel_max, bidir):
    """From the definition, in floating point with a margin at the borders (the library finds them in whole numbers)."""
    n = nb // 2 if bidir else nb
    e = n // 2
    d = rel.abs() if bidir else (-rel).clamp(min=0)
    far = e + torch.floor((n - e) * torch.log(d.double().clamp(min=e) / e) / math.log(rel_max / e) + 1e-9).long()
    b = torch.where(d < e, d, far.clamp(max=n - 1))
    return b + n * (rel > 0).long() if bidir else b


def _reference(q, k, v, dout, kmask, causal, scale, table, rel_max, bidir):
    """float64 results and elementwise bounds: {name: (value, bound)}."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    up, tiny, e24 = (0.0 if dt == F32 else u), (2.0 ** -25 if dt == F16 else 0.0), 2.0 ** -24
    B, Sq, nh, D = q.shape
    Sk, nkv = k.shape[1], k.shape[2]
    G = nh // nkv
    f = lambda t: t.detach().double().transpose(1, 2)
    Q, K, V, dO = f(q), f(k).repeat_interleave(G, 1), f(v).repeat_interleave(G, 1), f(dout)
    i, j = torch.arange(Sq, device=q.device)[:, None], torch.arange(Sk, device=q.device)[None]
    seen = torch.ones((B, 1, Sq, Sk), dtype=torch.bool, device=q.device)
    add = torch.zeros((B, 1, 1, Sk), dtype=torch.float64, device=q.device)
    if kmask is not None:
        gone = (kmask == float("-inf"))[:, None, None]
        seen = seen & ~gone
        add = torch.where(gone, torch.zeros_like(add), kmask.double()[:, None, None])
        K, V = (torch.where(gone.transpose(2, 3), torch.zeros_like(t), t) for t in (K, V))
    if causal:
        seen = seen & (j <= i + Sk - Sq)
    t = scale * Q @ K.transpose(2, 3) + add
    mag = scale * Q.abs() @ K.abs().transpose(2, 3)
    if table is not None:
        which = _bucket(j - (i + Sk - Sq), table.shape[0], rel_max, bidir)
        t = t + table.detach().double().t()[:, which][None]
    t = torch.where(seen, t, torch.full_like(t, float("-inf")))
    some = seen.any(-1, keepdim=True)
    m = torch.where(some, t.amax(-1, keepdim=True), torch.zeros_like(t[..., :1]))
    P = torch.where(seen, torch.exp(t - m), torch.zeros_like(t))
    P = P / torch.where(some, P.sum(-1, keepdim=True), torch.ones_like(m))
    ab = torch.where(seen & (t > -1e20), t.abs(), torch.zeros_like(t)).amax()
    epsP = float(2 * e24 * (D * mag.amax() + 8 * ab) + 2.0 ** -20)
    nk, nq = (Sk + 8) * e24, (Sq * G + 8) * e24
    out = P @ V
    aV = P @ V.abs()
    eO = (up + epsP + nk) * aV + u * out.abs() + tiny * V.abs().sum(2, keepdim=True)
    res = {"out": (out, eO)}
    dP = dO @ V.transpose(2, 3)
    delta = (dO * out).sum(-1, keepdim=True)
    eD = eO if dt == F32 else eO - (u - u * u) * out.abs()
    edelta = (dO.abs() * (eD + D * e24 * out.abs())).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    eS = epsP * dS.abs() + P * (edelta + D * e24 * (dO.abs() @ V.abs().transpose(2, 3)) + 4 * e24 * (dP.abs() + delta.abs()))
    aS = dS.abs()
    eSr = up * aS + eS + tiny * seen
    dQ = scale * dS @ K
    res["dq"] = (dQ, scale * ((eSr + nk * aS) @ K.abs()) + u * dQ.abs())
    dK, eK = scale * dS.transpose(2, 3) @ Q, scale * ((eSr + nq * aS).transpose(2, 3) @ Q.abs())
    dV, eV = P.transpose(2, 3) @ dO, ((up + epsP + nq) * P + tiny * seen).transpose(2, 3) @ dO.abs()
    for n, g, e in (("dk", dK, eK), ("dv", dV, eV)):
        g, e = g.view(B, nkv, G, Sk, D).sum(2), e.view(B, nkv, G, Sk, D).sum(2)
        res[n] = (g, e + u * g.abs())
    res = {n: (a.transpose(1, 2), b.transpose(1, 2) + tiny + 1e-30) for n, (a, b) in res.items()}
    if table is not None:
        # the table's gradient takes every row's delta from the sum of its dS, not from the rounded out: no error of out in it
        row = ((epsP + nk) * (aS + P * edelta)).sum(-1, keepdim=True)
        eS = epsP * aS + P * (row + D * e24 * (dO.abs() @ V.abs().transpose(2, 3)) + 4 * e24 * (dP.abs() + delta.abs()))
        gt, et = torch.zeros_like(table, dtype=torch.float64), torch.zeros_like(table, dtype=torch.float64)
        for b in range(table.shape[0]):
            w = (which == b)
            gt[b] = (dS * w).sum((0, 2, 3))
            et[b] = ((eS + (B * Sq + Sk) * e24 * aS) * w).sum((0, 2, 3)) + e24 * gt[b].abs()
        res["dtable"] = (gt, et + 1e-30)
    return res


def _check(got, ref, what):
    for n, g in got.items():
        val, bound = ref[n]
        assert g.shape == val.shape, (what, n, g.shape, val.shape)
        assert torch.isfinite(g).all(), (what, n, "not finite")
        bad = (g.double() - val).abs() / bound
        assert bad.max().item() <= 1.0, (what, n, bad.max().item(), (g.double() - val).abs().max().item())


def _mask(kind, B, Sk, seed):
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, Sk + 1, (B,), generator=g)
    j = torch.arange(Sk)[None]
    if kind == "pad":
        m = torch.where(j < lens[:, None], 0.0, float("-inf"))
    elif kind == "empty":
        lens[-1] = 0
        m = torch.where(j < lens[:, None], 0.0, float("-inf"))
    elif kind == "neg":
        m = torch.where(j < lens[:, None], 0.0, -10000.0)
        m[-1] = -10000.0                                  # a sample whose every key is masked the finite way: plain softmax
    elif kind == "left":
        m = torch.where(j >= Sk - lens[:, None], 0.0, torch.finfo(F32).min)
    elif kind == "leftpad":
        m = torch.where(j >= Sk - lens[:, None], 0.0, float("-inf"))
    elif kind == "holes":
        m = torch.where(torch.rand((B, Sk), generator=g) < 0.3, float("-inf"), 0.0) + 0.5 * torch.randn((B, Sk), generator=g)
    return m.float().cuda()


def _run(ops, q, k, v, dout, kmask, causal, table, rel_max, bidir, scale=None):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    tb = None if table is None else table.detach().requires_grad_(True)
    out = ops.long_attention(*leaves, kmask=kmask, causal=causal, scale=scale, rel_table=tb, rel_max=rel_max, rel_bidirectional=bidir)
    gs = torch.autograd.grad(out, leaves + ([tb] if tb is not None else []), dout)
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *gs)))


def _case(ops, dtype, shape, causal=False, mask="none", rel=None, seed=0, scale=None, prepare=None):
    B, Sq, Sk, nh, nkv, D = shape
    q, k, v, dout = (_rand(s, dtype, seed + x) for x, s in enumerate([(B, Sq, nh, D), (B, Sk, nkv, D), (B, Sk, nkv, D), (B, Sq, nh, D)]))
    km = _mask(mask, B, Sk, seed + 7)
    table, rel_max, bidir = None, 128, True
    if rel:
        nb, rel_max, bidir = rel
        table = _rand((nb, nh), F32, seed + 9, 0.7)
    if prepare:
        prepare(q, k, v, km)
    got = _run(ops, q, k, v, dout, km, causal, table, rel_max, bidir, scale)
    _check(got, _reference(q, k, v, dout, km, causal, scale if scale is not None else D ** -0.5, table, rel_max, bidir), (dtype, shape, causal, mask, rel))
    return got


SHAPES = [  # B, Sq, Sk, nh, nkv, D
    (1, 1, 1, 1, 1, 8), (2, 3, 2, 2, 2, 64), (2, 1, 130, 4, 2, 64), (1, 33, 1, 2, 1, 16), (1, 32, 32, 1, 1, 64), (2, 65, 63, 2, 1, 40),
    (1, 128, 128, 2, 2, 64), (1, 200, 200, 3, 3, 64), (2, 129, 257, 4, 1, 128), (1, 257, 129, 2, 2, 96), (1, 1, 1025, 6, 2, 128), (3, 5, 700, 8, 2, 72),
    (1, 600, 70, 4, 1, 64), (1, 517, 517, 2, 2, 64),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(ops, dtype, causal, shape):
    _case(ops, dtype, shape, causal, seed=sum(shape))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("mask", ["pad", "empty", "neg", "left", "holes"])
@pytest.mark.parametrize("shape", [(3, 70, 70, 2, 1, 64), (2, 130, 333, 2, 2, 128), (3, 2, 400, 4, 1, 64)])
def test_masks(ops, dtype, causal, mask, shape):
    _case(ops, dtype, shape, causal, mask, seed=11)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("mask,shape", [("leftpad", (3, 300, 300, 2, 1, 64)), ("leftpad", (2, 130, 333, 2, 2, 128)), ("leftpad", (4, 1, 500, 4, 2, 64)), ("holes", (2, 65, 200, 2, 1, 40)),
                                        ("pad", (2, 100, 150, 2, 2, 96)), ("neg", (2, 100, 150, 2, 2, 32)), ("left", (2, 65, 200, 2, 1, 72)), ("leftpad", (2, 900, 900, 2, 2, 64))])
def test_masks_at_other_sizes(ops, dtype, causal, mask, shape):
    """Keys left out in front (whole tiles of them, rows that see none), and masks where head sizes are padded or rows are no power of two."""
    _case(ops, dtype, shape, causal, mask, seed=17)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,causal,mask,rel", [
    ((2, 70, 70, 2, 2, 64), False, "none", (32, 128, True)), ((1, 300, 300, 3, 3, 64), False, "pad", (8, 20, True)), ((1, 300, 300, 2, 2, 64), True, "none", (13, 37, False)),
    ((2, 50, 420, 4, 2, 128), True, "left", (16, 64, False)), ((1, 420, 50, 2, 1, 64), False, "empty", (10, 33, True)), ((1, 1, 700, 4, 2, 64), True, "none", (32, 128, False)),
    ((1, 3, 3, 1, 1, 8), False, "none", (4, 2, True)), ((1, 640, 640, 2, 2, 64), True, "holes", (32, 100, True)), ((1, 260, 260, 1, 1, 128), False, "none", (128, 1024, True)),
    ((1, 130, 130, 2, 2, 32), False, "none", (2, 5, False)), ((2, 900, 900, 2, 1, 64), True, "leftpad", (24, 256, False)), ((2, 330, 500, 2, 2, 72), False, "pad", (32, 128, True)),
    ((1, 500, 300, 2, 2, 96), True, "holes", (32, 128, True)),
])
def test_learned_distance_bias(ops, dtype, shape, causal, mask, rel):
    _case(ops, dtype, shape, causal, mask, rel, seed=23)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_excluded_keys_may_hold_anything(ops, dtype):
    def spoil(q, k, v, km):
        gone = km == float("-inf")
        k[gone] = float("nan")
        v[gone] = float("inf")
    got = _case(ops, dtype, (3, 70, 140, 2, 2, 64), mask="holes", seed=5, prepare=spoil)
    got2 = _case(ops, dtype, (3, 70, 140, 2, 2, 64), mask="empty", seed=5, prepare=spoil)
    assert (got["dk"] == 0).any() and (got2["out"][-1] == 0).all() and (got2["dv"][-1] == 0).all() and (got2["dq"][-1] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_zero_lengths(ops, dtype):
    for B, Sq, Sk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v = (torch.randn(B, S, 2, 64, device="cuda").to(dtype).requires_grad_(True) for S in (Sq, Sk, Sk))
        table = torch.randn(8, 2, device="cuda", requires_grad=True)
        out = ops.long_attention(q, k, v, rel_table=table)
        assert out.shape == q.shape and (out == 0).all()
        gs = torch.autograd.grad(out.float().sum(), [q, k, v, table])
        assert all((g == 0).all() and g.shape == t.shape for g, t in zip(gs, (q, k, v, table)))


def test_large_scores(ops):
    """Scores of hundreds: the running maximum carries the softmax."""
    _case(ops, F32, (1, 150, 300, 2, 2, 64), scale=8.0, seed=3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_alignment_and_orders(ops, dtype):
    """Views of a packed projection, [B, heads, S, D] storage, rows off the 16-byte grid, keys shared by the batch, an expanded output gradient."""
    B, S, nh, D = 2, 90, 3, 64
    packed = _rand((B, S, 3, nh, D), dtype, 1)
    dense = [packed[:, :, n].contiguous() for n in range(3)]
    dout = _rand((B, S, nh, D), dtype, 2)
    ref = _run(ops, *dense, dout, None, True, None, 0, True)
    other = {
        "packed": [packed[:, :, n] for n in range(3)],
        "heads first": [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dense],
        "off the grid": [torch.cat([t.flatten(), t.flatten()[:1]])[1:].view(t.shape).copy_(t) for t in dense],
        "last axis strided": [torch.stack([t, t], -1)[..., 0] for t in dense],
    }
    for what, ts in other.items():
        got = _run(ops, *ts, dout.transpose(1, 2).contiguous().transpose(1, 2), None, True, None, 0, True)
        for n in ref:
            assert torch.equal(got[n], ref[n]), (what, n)
    # one k, v for the whole batch and all heads
    k1, v1 = _rand((1, S, 1, D), dtype, 3).requires_grad_(True), _rand((1, S, 1, D), dtype, 4).requires_grad_(True)
    out = ops.long_attention(dense[0], k1.expand(B, S, nh, D), v1.expand(B, S, nh, D))
    gk, gv = torch.autograd.grad(out, [k1, v1], torch.ones((), dtype=dtype, device="cuda").expand(out.shape))
    k2, v2 = (t.detach().repeat(B, 1, nh, 1).requires_grad_(True) for t in (k1, v1))
    out2 = ops.long_attention(dense[0], k2, v2)
    assert torch.equal(out, out2)
    wk, wv = torch.autograd.grad(out2, [k2, v2], torch.ones_like(out2))
    u = torch.finfo(dtype).eps
    for g, w in ((gk, wk), (gv, wv)):
        s, a = w.double().sum((0, 2), keepdim=True), w.double().abs().sum((0, 2), keepdim=True)
        assert ((g.double() - s).abs() <= 3 * u * a).all()


def test_offsets_beyond_32_bits(ops):
    """A cache whose second sample lies more than 2^31 elements behind the first."""
    S, D, far = 300, 64, 2 ** 31 + 4096
    store = torch.empty(far + S * D, dtype=BF16, device="cuda")
    kv = torch.as_strided(store, (2, S, 1, D), (far, D, D, 1))
    small = _rand((2, S, 1, D), BF16, 1)
    kv.copy_(small)
    q, dout = _rand((2, 40, 2, D), BF16, 2), _rand((2, 40, 2, D), BF16, 3)
    a, b = _run(ops, q, kv, kv, dout, None, False, None, 0, True), _run(ops, q, small, small, dout, None, False, None, 0, True)
    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("rel", [None, (16, 64, True)])
def test_equal_calls_give_equal_bits_and_streams(ops, rel):
    B, S, nh, D = 2, 700, 2, 64
    q, k, v, dout = (_rand((B, S, nh, D), BF16, x) for x in range(4))
    km = _mask("pad", B, S, 3)
    table = _rand((rel[0], nh), F32, 9) if rel else None
    a = _run(ops, q, k, v, dout, km, False, table, 64, True)
    for _ in range(3):
        b = _run(ops, q, k, v, dout, km, False, table, 64, True)
        assert all(torch.equal(a[n], b[n]) for n in a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = _run(ops, q, k, v, dout, km, False, table, 64, True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a[n], c[n]) for n in a)


def test_two_captured_graphs_and_eager_work_between(ops):
    """Forward + backward recorded twice at different shapes, replayed in turn with eager calls in between: every replay equals the eager result."""
    made = []
    for B, S, seed in ((2, 300, 1), (1, 520, 5)):
        q, k, v, dout = (_rand((B, S, 2, 64), BF16, seed + x) for x in range(4))
        km, table = _mask("left", B, S, 3), _rand((16, 2), F32, 9)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _run(ops, q, k, v, dout, km, True, table, 64, True)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = _run(ops, q, k, v, dout, km, True, table, 64, True)
        made.append((g, res, q, k, v, dout, km, table))
    for r in range(3):
        for g, res, q, k, v, dout, km, table in made:
            q.copy_(_rand(q.shape, BF16, 50 + r))
            g.replay()
        for g, res, q, k, v, dout, km, table in made:
            eager = _run(ops, q, k, v, dout, km, True, table, 64, True)
            torch.cuda.synchronize()
            assert all(torch.equal(res[n], eager[n]) for n in eager), r


def test_gradients_against_differences(ops):
    """Central differences of the float32 forward pass. With a step of 2^-4 the difference quotient of a sum L = <out, dout> is off by h^2 / 6 |L'''| plus the
    forward's rounding over 2 h; along a random unit direction both stay under 2 % of |dout| |V| (checked as 0.02 against values of order one)."""
    q, k, v, dout = (_rand((1, 40, 2, 32), F32, x) for x in range(4))
    table = _rand((8, 2), F32, 9)
    got = _run(ops, q, k, v, dout, None, True, table, 16, True)
    args = {"dq": q, "dk": k, "dv": v, "dtable": table}
    for n, t in args.items():
        d = _rand(t.shape, F32, 77)
        d = d / d.norm()
        h = 2.0 ** -4
        val = []
        for s in (h, -h):
            moved = {m: (x + s * d if m == n else x) for m, x in args.items()}
            out = ops.long_attention(moved["dq"], moved["dk"], moved["dv"], causal=True, rel_table=moved["dtable"], rel_max=16)
            val.append((out.double() * dout.double()).sum())
        num, ana = ((val[0] - val[1]) / (2 * h)).item(), (got[n].double() * d.double()).sum().item()
        assert abs(num - ana) <= 0.02 * max(1.0, abs(ana)), (n, num, ana)


def test_frozen_inputs_and_no_grad(ops):
    q, k, v, dout = (_rand((1, 70, 2, 64), BF16, x) for x in range(4))
    ref = _run(ops, q, k, v, dout, None, False, None, 0, True)
    with torch.no_grad():
        assert torch.equal(ops.long_attention(q, k, v), ref["out"])
    q1 = q.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ops.long_attention(q1, k, v), q1, dout)[0], ref["dq"])
    k1 = k.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ops.long_attention(q, k1, v), k1, dout)[0], ref["dk"])
