"""GPU: corners of ops.long_attention and ops.token_logprobs where results went wrong, or could have, at unusual masks, ties and magnitudes."""
import pytest
import torch

from tests.test_long_attention_gpu import _bucket, _check, _reference, _run

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a MI355X"
    from vln_imagine_amd import ops as o
    return o


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


@pytest.mark.parametrize("rows,V", [(3, 2500), (40, 8000), (3, 70001), (17, 150000), (1100, 12000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_in_every_pass_of_long_rows(ops, dtype, rows, V):
    """More equal best entries than the candidates' list holds, in every pass over a row, between passes without any: the block's waves have to
    take the same branch each time (blocks of 256 and of 1024 threads). Constant rows, rows of few values, rows of -inf with one or twenty others, and values that rise along the row.
    logp's bound: the sums have at most 32 c + 16 additions (c passes), exp2 and its argument 2^-23 (2 + |x - m|) relative, |x - m| <= 4."""
    x = torch.randint(-2, 3, (rows, V), generator=torch.Generator().manual_seed(V)).float()
    x[0] = 1.0
    x[1] = -INF
    x[1, torch.randperm(V, generator=torch.Generator().manual_seed(1))[:20]] = 0.5
    x[2] = torch.arange(V).float().div(9000).floor() * 0.25        # a new best value every 9000 entries
    x = x.to(dtype).cuda()
    t = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(2)).cuda()
    top = 16
    logp, ent, tl, ti = ops.token_logprobs(x, t, top=top)
    ref = torch.log_softmax(x.double(), 1)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(ti, order)
    err = 2.0 ** -23 * (32 * (V // 8192 + 2) + 18 + 2 * 5)
    want = ref.gather(1, t[:, None])[:, 0]
    live = want > -INF
    assert torch.equal(logp > -INF, live) and ((logp.double() - want).abs()[live] <= err).all()
    w = ref.gather(1, order)
    fin = w > -INF
    assert torch.equal(tl > -INF, fin) and ((tl.double() - w).abs()[fin] <= err).all()
    H = torch.special.entr(ref.exp()).sum(1)
    assert ((ent.double() - H).abs() <= err * (3 + H)).all()
    again = ops.token_logprobs(x, t, top=top)
    assert all(torch.equal(a, b) for a, b in zip(again, (logp, ent, tl, ti)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("S,lens,rel,causal", [(1024, (200, 1024, 70), (16, 40, True), False), (1500, (1, 640), (32, 91, True), False), (1024, (300, 900), (13, 37, False), False),
                                               (900, (64, 500), (16, 40, False), True)])
def test_table_gradient_of_rows_whose_near_keys_are_all_masked(ops, dtype, S, lens, rel, causal):
    """Whole row blocks see valid keys beyond the last bucket's distance only: the band around them holds nothing but masked keys."""
    B, nh, D = len(lens), 2, 64
    q, k, v, dout = (_rand((B, S, nh, D), dtype, 31 + x) for x in range(4))
    km = torch.where(torch.arange(S)[None] < torch.tensor(lens)[:, None], 0.0, -INF).float().cuda()
    nb, rel_max, bidir = rel
    table = _rand((nb, nh), F32, 40, 0.7)
    got = _run(ops, q, k, v, dout, km, causal, table, rel_max, bidir)
    _check(got, _reference(q, k, v, dout, km, causal, D ** -0.5, table, rel_max, bidir), (dtype, S, lens, rel))
    again = _run(ops, q, k, v, dout, km, causal, table, rel_max, bidir)
    assert all(torch.equal(got[n], again[n]) for n in got)


def _left(B, S, low):
    """Keys in front of a sample's text carry `low`: S, S - S // 3, ... valid ones at the end."""
    lens = torch.tensor([max(1, S - b * (S // 3)) for b in range(B)])
    return torch.where(torch.arange(S)[None] >= S - lens[:, None], 0.0, low).float().cuda()


def _by_row(q, k, v, dout, kmask, causal, scale, table=None, rel_max=0, bidir=True):
    """float64 results with elementwise bounds as in test_long_attention_gpu, but with every row's own error of P: from the scores and the maximum among the keys
    that have a share in it. Masks (and entries of the table) of -1e8 and less absorb scores below 32 in float32 (half a step of 1.4e8 is 8 in units of log2 already at 2^28): such a key's t is the mask itself, and
    a row of nothing else has no rounding in its t at all.
    float16's smallest step: 2^-25 of a P in the forward pass and of a result; in the backward pass P is rounded times 2^12 and dS, whose size is
    at most 2 D max|dO| max|V| P, times 2^12 and the power of two that brings that bound between 2 and 4 (max|dO|: of the row for dQ, of the sample and key head for dK)."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    up, tiny, e24 = (0.0 if dt == F32 else u), (2.0 ** -25 if dt == F16 else 0.0), 2.0 ** -24
    B, Sq, nh, D = q.shape
    Sk, nkv = k.shape[1], k.shape[2]
    G = nh // nkv
    f = lambda t: t.detach().double().transpose(1, 2)
    Q, K, V, dO = f(q), f(k).repeat_interleave(G, 1), f(v).repeat_interleave(G, 1), f(dout)
    i, j = torch.arange(Sq, device=q.device)[:, None], torch.arange(Sk, device=q.device)[None]
    add = torch.zeros((B, 1, 1, Sk), dtype=torch.float64, device=q.device) if kmask is None else kmask.double()[:, None, None]
    bias = torch.zeros_like(add)
    seen = (add > -INF).expand(B, 1, Sq, Sk)
    if causal:
        seen = seen & (j <= i + Sk - Sq)
    t = scale * Q @ K.transpose(2, 3)
    mag = scale * Q.abs() @ K.abs().transpose(2, 3)
    if table is not None:
        which = _bucket(j - (i + Sk - Sq), table.shape[0], rel_max, bidir)
        bias = table.detach().double().t()[:, which][None]
    far, far_m, far_b = (add <= -1e8) | (bias <= -1e8), add <= -1e8, bias <= -1e8
    assert not far.any() or ((t + bias * ~far_b).abs().max() < 32 and (add * far_m + bias * far_b).where(far, -1e9).max() <= -1e9)
    t = torch.where(far, torch.where(far_m, add.clamp(min=-1e30), 0.0) + torch.where(far_b, bias, 0.0), t + add + bias)
    t = torch.where(seen, t, torch.full_like(t, -INF))
    some = seen.any(-1, keepdim=True)
    m = torch.where(some, t.amax(-1, keepdim=True), torch.zeros_like(t[..., :1]))
    P = torch.where(seen, torch.exp(t - m), torch.zeros_like(t))
    P = P / torch.where(some, P.sum(-1, keepdim=True), torch.ones_like(m))
    share = (P > 2.0 ** -40) & ~far
    zero = torch.zeros_like(t)
    epsP = 2 * e24 * (D * torch.where(share, mag, zero).amax(-1, keepdim=True) + 8 * torch.where(share, t.abs(), zero).amax(-1, keepdim=True)) + 2.0 ** -20
    nk, nq = (Sk + 8) * e24, (Sq * G + 8) * e24
    out, aV = P @ V, P @ V.abs()
    eO = (up + epsP + nk) * aV + u * out.abs() + tiny * V.abs().sum(2, keepdim=True)
    res = {"out": (out, eO)}
    dP, delta = dO @ V.transpose(2, 3), (dO * out).sum(-1, keepdim=True)
    eD = eO if dt == F32 else eO - (u - u * u) * out.abs()
    edelta = (dO.abs() * (eD + D * e24 * out.abs())).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    aS, prod = dS.abs(), D * e24 * (dO.abs() @ V.abs().transpose(2, 3)) + 4 * e24 * (dP.abs() + delta.abs())
    eS = up * aS + epsP * aS + P * (edelta + prod)
    rowmax, allmax = dO.abs().amax(-1, keepdim=True), dO.abs().reshape(B, nkv, -1).amax(-1).repeat_interleave(G, 1)[:, :, None, None]
    least = 2.0 ** -12 * tiny * D * V.abs().amax((2, 3), keepdim=True) * seen
    dQ = scale * dS @ K
    res["dq"] = (dQ, scale * ((eS + nk * aS + least * rowmax) @ K.abs()) + u * dQ.abs())
    dK, eK = scale * dS.transpose(2, 3) @ Q, scale * ((eS + nq * aS + least * allmax).transpose(2, 3) @ Q.abs())
    dV, eV = P.transpose(2, 3) @ dO, ((up + epsP + nq) * P + 2.0 ** -12 * tiny * seen).transpose(2, 3) @ dO.abs()
    for n, g, e in (("dk", dK, eK), ("dv", dV, eV)):
        g, e = g.view(B, nkv, G, Sk, D).sum(2), e.view(B, nkv, G, Sk, D).sum(2)
        res[n] = (g, e + u * g.abs())
    res = {n: (a.transpose(1, 2), b.transpose(1, 2) + tiny + 1e-30) for n, (a, b) in res.items()}
    if table is not None:
        row = ((epsP + nk) * (aS + P * edelta)).sum(-1, keepdim=True)
        eS = epsP * aS + P * (row + prod) + (B * Sq + Sk) * e24 * aS
        gt, et = torch.zeros_like(table, dtype=torch.float64), torch.zeros_like(table, dtype=torch.float64)
        for b in range(table.shape[0]):
            w = (which == b)
            gt[b], et[b] = (dS * w).sum((0, 2, 3)), (eS * w).sum((0, 2, 3))
        res["dtable"] = (gt, et + e24 * gt.abs() + 1e-30)
    return res


LOWS = [-1e4, -65504.0, -1e6, -1e9, -1e12, -1e19, -1e25, torch.finfo(F32).min]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("low", LOWS)
@pytest.mark.parametrize("shape,causal,all_,rel", [((2, 300, 300, 4, 2, 64), True, False, None), ((2, 130, 750, 2, 2, 128), False, True, None), ((3, 200, 200, 2, 1, 64), True, False, (16, 40, False)),
                                                   ((1, 1400, 1400, 1, 1, 32), True, True, None), ((2, 3, 900, 4, 1, 64), False, True, None)])
def test_finite_masks_of_any_size(ops, dtype, low, shape, causal, all_, rel):
    """Rows that see nothing but keys with a finite mask (every key of a sample, padding in front of a causal batch) are an ordinary softmax: the shares of a row add up to 1 in
    the backward pass too - with an output gradient of ones, dV summed over the keys counts the rows. Where the mask absorbs the scores, and for -1e4, each value is held as well.
    The sum's bound: P and its normalisation 2^-18 (m + log2(l) is kept in one float32 up to 64), n + rows additions of 2^-24, in 16 bits one rounding of P and one of dV."""
    B, Sq, Sk, nh, nkv, D = shape
    q, k, v, dout = (_rand(s, dtype, 3 + x) for x, s in enumerate([(B, Sq, nh, D), (B, Sk, nkv, D), (B, Sk, nkv, D), (B, Sq, nh, D)]))
    km = torch.full((B, Sk), low, device="cuda") if all_ else _left(B, Sk, low)
    nb, rel_max, bidir = rel or (0, 0, True)
    table = _rand((nb, nh), F32, 9, 0.7) if rel else None
    got = _run(ops, q, k, v, torch.ones_like(dout), km, causal, table, rel_max, bidir)
    rows = Sq * (nh // nkv)
    u = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    bound = rows * (2.0 ** -18 + (Sk + rows) * 2.0 ** -24 + 2 * u) + (2.0 ** -25 * Sk * (rows + 1) if dtype == F16 else 0)
    assert ((got["dv"].double().sum(1) - rows).abs() <= bound).all(), ((got["dv"].double().sum(1) - rows).abs().max().item(), bound)
    if low in (-65504.0, -1e6):
        return
    got = _run(ops, q, k, v, dout, km, causal, table, rel_max, bidir)
    _check(got, _by_row(q, k, v, dout, km, causal, D ** -0.5, table, rel_max, bidir), (dtype, low, shape, causal))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape,rel", [((3, 70, 70, 2, 1, 64), None), ((2, 130, 333, 2, 2, 128), None), ((3, 2, 400, 4, 1, 64), None), ((2, 300, 300, 2, 2, 64), (16, 40, True)), ((1, 900, 900, 1, 1, 40), None)])
def test_rows_beside_masked_keys_to_their_own_bounds(ops, dtype, causal, shape, rel):
    """-10000 on a sample's last keys: its rows' own scores are of order one, and so is their error."""
    B, Sq, Sk, nh, nkv, D = shape
    q, k, v, dout = (_rand(s, dtype, 13 + x) for x, s in enumerate([(B, Sq, nh, D), (B, Sk, nkv, D), (B, Sk, nkv, D), (B, Sq, nh, D)]))
    lens = torch.tensor([Sk - b * (Sk // 4) - 1 for b in range(B)])
    km = torch.where(torch.arange(Sk)[None] < lens[:, None], 0.0, -10000.0).float().cuda()
    nb, rel_max, bidir = rel or (0, 0, True)
    table = _rand((nb, nh), F32, 9, 0.7) if rel else None
    _check(_run(ops, q, k, v, dout, km, causal, table, rel_max, bidir), _by_row(q, k, v, dout, km, causal, D ** -0.5, table, rel_max, bidir), (dtype, causal, shape))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("factor", [8.0, 300.0])
def test_shares_add_up_at_large_scores(ops, dtype, factor):
    """Scores of hundreds to ten thousands without a mask: the row's maximum leaves no room for log2(l) beside it in a float32."""
    S, nh, D = 261, 16, 64
    q, k, v = (_rand((1, S, nh, D), dtype, 3 + x) for x in range(3))
    k[:, 1::3] = k[:, 2::3] = k[:, ::3]                              # every best key three times: shares of a third, and log2(3) beside the maximum
    row = 16 * torch.arange(nh) + 2                                  # one row of each head has an output gradient, of ones
    dout = torch.zeros_like(q)
    dout[0, row, torch.arange(nh)] = 1.0
    u = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    for causal in (False, True):
        got = _run(ops, q, k, v, dout, None, causal, None, 0, True, scale=factor)
        # (a tile at the causal border rounds its scores once more, before the maximum is off them: 2^-24 of a |score| below 64 factor, twice)
        bound = 2.0 ** -18 + 2 * S * 2.0 ** -24 + 2 * u + causal * 2 * 2.0 ** -24 * 64 * factor
        off = (got["dv"].double().sum(1) - 1).abs().max().item()
        assert off <= bound, (causal, off, bound)


def _spread(t, low):
    """Rows of a tensor [B, S, ...] times powers of two from 1 down to `low`."""
    n = torch.arange(t.shape[1], device=t.device) % 4
    return (t.float() * (low ** (n / 3.0)).log2().round().exp2().view(1, -1, 1, 1)).to(t.dtype)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape,rel", [((2, 1500, 1500, 2, 1, 64), None), ((1, 260, 3000, 2, 2, 128), None), ((3, 700, 700, 4, 2, 64), (16, 40, True)), ((2, 2, 2500, 4, 1, 64), None), ((2, 333, 333, 2, 2, 72), None)])
@pytest.mark.parametrize("size", [1e-4, 1.0, "rows", "samples"])
def test_float16_gradients_of_any_size(ops, causal, shape, rel, size):
    """Output gradients far from one, all alike or with small rows or samples beside large ones: P and dS below float16's normal range as they stand."""
    B, Sq, Sk, nh, nkv, D = shape
    q, k, v, dout = (_rand(s, F16, 61 + x) for x, s in enumerate([(B, Sq, nh, D), (B, Sk, nkv, D), (B, Sk, nkv, D), (B, Sq, nh, D)]))
    if size == "rows":
        dout = _spread(dout, 2.0 ** -12)
    elif size == "samples":
        dout = (dout.float() * torch.tensor([2.0 ** -12, 1.0, 2.0 ** -6])[:B].view(-1, 1, 1, 1).cuda()).half()
    else:
        dout = (dout.float() * size).half()
    km = _left(B, Sk, -INF) if not causal else None
    nb, rel_max, bidir = rel or (0, 0, True)
    table = _rand((nb, nh), F32, 9, 0.7) if rel else None
    got = _run(ops, q, k, v, dout, km, causal, table, rel_max, bidir)
    ref = _by_row(q, k, v, dout, km, causal, D ** -0.5, table, rel_max, bidir)
    _check(got, ref, (shape, causal, size))


def test_float16_gradients_beyond_its_range_inside(ops):
    """dS of 1e5 under results that float16 holds: not representable as it stands."""
    B, Sq, Sk, nh, D, scale = 1, 24, 90, 2, 64, 1 / 16
    q, k, v, dout = (_rand((B, S, nh, D), F16, 71 + x, c) for x, (S, c) in enumerate([(Sq, 2.0), (Sk, 2.0), (Sk, 8.0), (Sq, 3000.0)]))
    ref = _by_row(q, k, v, dout, None, False, scale)
    assert all(val.abs().max() < 6e4 for val, _ in ref.values())
    Q, K, V, dO = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    P, g = torch.softmax(scale * Q @ K.transpose(2, 3).contiguous(), -1), dO @ V.transpose(2, 3).contiguous()
    assert (P * (g - (P * g).sum(-1, keepdim=True))).abs().max() > 7e4
    _check(_run(ops, q, k, v, dout, None, False, None, 0, True, scale=scale), ref, "large")


@pytest.mark.parametrize("causal", [False, True])
def test_float16_excluded_keys_do_not_set_the_scale(ops, causal):
    """Keys left out hold infinities, NaN and the largest number; their values are no part of what the gradients are scaled by."""
    B, S, nh, D = 2, 400, 2, 64
    q, k, v, dout = (_rand((B, S, nh, D), F16, 81 + x) for x in range(4))
    dout = (dout.float() * 1e-3).half()
    km = torch.where(torch.rand((B, S), generator=torch.Generator().manual_seed(1)) < 0.3, -INF, 0.0)
    km[:, 0] = 0.0
    km = km.cuda()
    want = _run(ops, q, k, v, dout, km, causal, None, 0, True)
    gone = km == -INF
    k2, v2 = k.clone(), v.clone()
    k2[gone], v2[gone] = float("nan"), 65504.0
    v2[:, :, 1][gone] = INF
    got = _run(ops, q, k2, v2, dout, km, causal, None, 0, True)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("V", [37, 1500, 5000])
def test_large_entropy_gradients_beside_impossible_entries(ops, V):
    """A loss scale of 2^40 on the entropy term: entries of -inf have no gradient, whatever the factor."""
    x = _rand((4, V), F32, 5)
    x[:, ::3] = -INF
    t = torch.ones(4, dtype=torch.int64, device="cuda")
    def grad(c):
        lg = x.clone().requires_grad_(True)
        logp, ent, _, _ = ops.token_logprobs(lg, t)
        return torch.autograd.grad([logp, ent], [lg], [torch.full((4,), c, device="cuda"), torch.full((4,), -c, device="cuda")])[0]
    one, big = grad(1.0), grad(2.0 ** 40)
    assert torch.isfinite(big).all() and (big[:, ::3] == 0).all()
    assert torch.equal(big, one * 2.0 ** 40)                         # powers of two are exact


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masks_up_to_the_types_largest_value(ops, dtype):
    """A key with the largest mask of all takes the whole row; -inf beside it leaves its key out."""
    B, S, nh, D = 2, 130, 2, 64
    q, k, v, dout = (_rand((B, S, nh, D), dtype, 21 + x) for x in range(4))
    km = torch.zeros((B, S), device="cuda")
    km[:, 77], km[:, 3] = torch.finfo(F32).max, -INF
    got = _run(ops, q, k, v, dout, km, False, None, 0, True)
    assert torch.equal(got["out"], v[:, 77:78].expand_as(v))
    assert (got["dv"][:, :77] == 0).all() and (got["dv"][:, 78:] == 0).all()
    # one share of 1: dS = <dO, v> - <dO, out> with out = v, which differ by the roundings of two sums of D products, D 2^-24 of their magnitudes each
    # (out is exact), and the results by one rounding more
    off = 2 * D * 2.0 ** -24 * (dout.double().abs() * v.double()[:, 77:78].abs()).sum(-1, keepdim=True) * D ** -0.5 * (1 + 2 * torch.finfo(dtype).eps)
    assert (got["dq"].double().abs() <= off * k.double()[:, 77:78].abs()).all()
    rest = torch.arange(S, device="cuda") != 77
    assert (got["dk"][:, rest] == 0).all() and (got["dk"].double().abs()[:, 77] <= (off * q.double().abs()).sum(1)).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("S,D,rel,nh,nkv", [(300, 64, None, 2, 2), (200, 128, (16, 40, False), 2, 2), (70, 40, None, 2, 2), (2500, 64, None, 2, 1), (9, 64, None, 8, 2), (1800, 96, (32, 300, False), 2, 1)])
def test_rows_without_keys_may_hold_anything(ops, dtype, S, D, rel, nh, nkv):
    """Causal batch with keys left out in front: rows that see none come out as zeros, and send no gradient back, with NaN in their q and infinities in
    their output's gradient."""
    B = 2
    q, k, v, dout = (_rand((B, S, h, D), dtype, 91 + x) for x, h in enumerate((nh, nkv, nkv, nh)))
    km = _left(B, S, -INF)
    km[0, :S // 2 + 3] = -INF
    dead = (km == -INF).long().cumprod(1).bool()                     # rows before a sample's first key
    assert dead.any() and not dead.all()
    dout[dead] = 0
    nb, rel_max, bidir = rel or (0, 0, True)
    table = _rand((nb, nh), F32, 9, 0.7) if rel else None
    want = _run(ops, q, k, v, dout, km, True, table, rel_max, bidir)
    q2, dout2 = q.clone(), dout.clone()
    q2[dead], dout2[dead] = float("nan"), INF
    got = _run(ops, q2, k, v, dout2, km, True, table, rel_max, bidir)
    assert (got["out"][dead] == 0).all() and (got["dq"][dead] == 0).all()
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_out_of_range_targets_are_counted_on_the_counters_device_only(ops):
    """The counter lies on one device; the same call on another one must not write there, and one that follows on the first counts as before."""
    ops.watch_index_errors()
    ops.index_errors(raise_=False)
    x, t = _rand((6, 50), F32, 1), torch.tensor([50, -1, 3, 49, -100, 1 << 40]).cuda()
    want = ops.token_logprobs(x, t, top=3)
    assert ops.index_errors(raise_=False) == 3
    if torch.cuda.device_count() < 2:
        pytest.skip("one device: nothing to be kept apart")
    got = ops.token_logprobs(x.to("cuda:1"), t.to("cuda:1"), top=3)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want)) and ops.index_errors(raise_=False) == 0
    ops.token_logprobs(x, t)
    assert ops.index_errors(raise_=False) == 3


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("shape,rel", [((2, 700, 700, 4, 2, 64), (16, 40, False)), ((1, 3, 2000, 4, 1, 128), None)])
def test_captured_with_statistics_apart(ops, dtype, shape, rel):
    """Recorded forward and backward with padding of -1e9 in front (rows whose 1 / sum stays apart), float16's ranges among the launches; replayed on inputs of other sizes with
    eager calls between."""
    B, Sq, Sk, nh, nkv, D = shape
    sizes = [(B, Sq, nh, D), (B, Sk, nkv, D), (B, Sk, nkv, D), (B, Sq, nh, D)]
    q, k, v, dout = (_rand(s, dtype, 3 + x) for x, s in enumerate(sizes))
    km = _left(B, Sk, -1e9)
    nb, rel_max, bidir = rel or (0, 0, True)
    table = _rand((nb, nh), F32, 9, 0.7) if rel else None
    args = (q, k, v, dout, km, True, table, rel_max, bidir)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(ops, *args)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = _run(ops, *args)
    for r, c in enumerate((1.0, 1e-3, 30.0)):
        for t, s in zip((q, k, v, dout), sizes):
            t.copy_(_rand(s, dtype, 50 + r))
        dout.mul_(c)
        km.copy_(_left(B, Sk, -INF if r == 2 else -1e6))
        g.replay()
        eager = _run(ops, *args)
        torch.cuda.synchronize()
        assert all(torch.equal(res[n], eager[n]) for n in eager), r


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("S,lens,D,low", [(300, (300, 120), 64, -1e9), (700, (90, 700), 128, -1e9), (500, (200, 60), 40, -1e12)])
def test_rows_that_see_only_distances_the_table_forbids(ops, dtype, S, lens, D, low):
    """A window by the table (far buckets at -1e9) over a ragged batch: padded rows see nothing but far keys. Their scores are absorbed by the bias: every key has the same share."""
    B, nh = len(lens), 2
    q, k, v, dout = (_rand((B, S, nh, D), dtype, 41 + x) for x in range(4))
    km = torch.where(torch.arange(S)[None] < torch.tensor(lens)[:, None], 0.0, -INF).float().cuda()
    table = _rand((16, nh), F32, 9, 0.7)
    table[7] = table[15] = low
    got = _run(ops, q, k, v, dout, km, False, table, 30, True)
    _check(got, _by_row(q, k, v, dout, km, False, D ** -0.5, table, 30, True), (dtype, S, lens))


@pytest.mark.parametrize("dtype,size", [(F32, 3e3), (F32, 1e6), (BF16, 3e3), (BF16, 1e6), (F16, 3e3), (F16, 1e4)])
@pytest.mark.parametrize("causal", [False, True])
def test_scores_far_beyond_a_float32s_steps(ops, dtype, size, causal):
    """Scores of 1e7 to 1e14: the best key of a row takes it whole (rows whose two best lie closer than the scores' rounding, D 2^-24 of their magnitudes, are left out)."""
    S, nh, D = 200, 2, 64
    q, k, v, dout = (_rand((1, S, nh, D), dtype, 51 + x, c) for x, c in enumerate((size, size, 1.0, 1.0)))
    t = q.double().transpose(1, 2) @ k.double().permute(0, 2, 3, 1) * D ** -0.5
    if causal:
        t = t.masked_fill(torch.arange(S, device="cuda")[None] > torch.arange(S, device="cuda")[:, None], -INF)
    near = 4 * D * 2.0 ** -24 * (q.double().abs().transpose(1, 2) @ k.double().abs().permute(0, 2, 3, 1)).amax(-1) * D ** -0.5 + 60
    two, best = t.topk(2, -1)
    clear = two[..., 0] - two[..., 1] > near
    assert clear.double().mean() > 0.9
    got = _run(ops, q, k, v, dout, None, causal, None, 0, True)
    want = v.transpose(1, 2).gather(2, best[..., :1].expand(-1, -1, -1, D))
    assert torch.equal(got["out"].transpose(1, 2)[clear], want[clear])
    assert all(torch.isfinite(g).all() for g in got.values())
    # dS of such a row is <dO, v> - <dO, out>, the roundings of two equal sums, or 0
    off = 2 * D * 2.0 ** -24 * (dout.double().abs().transpose(1, 2) * want.double().abs()).sum(-1) * D ** -0.5 * k.double().abs().max() * 1.01
    assert (got["dq"].double().transpose(1, 2).abs()[clear] <= off[clear][:, None] + 2.0 ** -25).all()
