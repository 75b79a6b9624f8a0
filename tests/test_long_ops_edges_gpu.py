"""GPU: corners of ops.long_attention and ops.token_logprobs where results went wrong, or could have, at unusual masks, ties and magnitudes."""
import pytest
import torch

from tests.test_long_attention_gpu import _check, _reference, _run

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
