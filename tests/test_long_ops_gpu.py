"""GPU: ops.long_attention with a learned distance bias and ops.token_logprobs together, as a token policy uses them: embedded tokens through one
self-attention block to the log probabilities and the entropy of the next tokens, a policy-gradient loss, gradients of every weight, a captured training
step. And both operators where autograd hands back other tensors than it was given (checkpointing, offloading of saved tensors)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
V, H, NH, NKV, D, BUCKETS, REL_MAX = 700, 64, 4, 2, 32, 16, 64


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a MI355X"
    from vln_imagine_amd import ops as o
    return o


class Policy(torch.nn.Module):
    def __init__(self, seed):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        par = lambda *s: torch.nn.Parameter((torch.randn(s, generator=g) * s[-1] ** -0.5).cuda())
        self.embed, self.qkv, self.out = par(V, H), par((NH + 2 * NKV) * D, H), par(H, NH * D)
        self.table = par(BUCKETS, NH)

    def forward(self, ops, tok, kmask):
        B, S = tok.shape
        x = self.embed[tok]
        y = ops.linear(x, self.qkv).view(B, S, NH + 2 * NKV, D)
        q, k, v = y.split([NH, NKV, NKV], 2)                       # views of the packed projection, read in place
        a = ops.long_attention(q, k, v, kmask=kmask, causal=True, rel_table=self.table, rel_max=REL_MAX, rel_bidirectional=False)
        x = x + ops.linear(a.reshape(B, S, NH * D), self.out)
        return ops.linear(x, self.embed)


def _batch(B, S, seed):
    g = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, V, (B, S), generator=g)
    lens = torch.tensor([S, S - 37])[:B]
    pad = torch.arange(S)[None] >= lens[:, None]
    target = torch.where(torch.arange(S)[None] >= lens[:, None] - 1, torch.full_like(tok, -100), tok.roll(-1, 1))
    adv = torch.randn((B, S), generator=g)
    return tok.cuda(), torch.where(pad, float("-inf"), 0.0).float().cuda(), target.cuda(), adv.cuda()


def _loss(logp, ent, adv, live):
    return -(logp * adv).sum() - 0.01 * (ent * live).sum()


def _reference(model, tok, kmask, target, adv):
    """The same in float64 by torch's own gradients."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in model.named_parameters()}
    B, S = tok.shape
    x = p["embed"][tok]
    y = (x @ p["qkv"].t()).view(B, S, NH + 2 * NKV, D)
    q, k, v = (t.transpose(1, 2) for t in y.split([NH, NKV, NKV], 2))
    k, v = k.repeat_interleave(NH // NKV, 1), v.repeat_interleave(NH // NKV, 1)
    i, j = torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None]
    d, e = (i - j).clamp(min=0), BUCKETS // 2
    far = e + torch.floor((BUCKETS - e) * torch.log(d.double().clamp(min=e) / e) / torch.log(torch.tensor(REL_MAX / e).double()) + 1e-9).long()
    t = q @ k.transpose(2, 3) * D ** -0.5 + p["table"].t()[:, torch.where(d < e, d, far.clamp(max=BUCKETS - 1))] + kmask.double()[:, None, None]
    a = torch.softmax(torch.where(j <= i, t, torch.full_like(t, float("-inf"))), -1) @ v
    lp = torch.log_softmax((x + a.transpose(1, 2).reshape(B, S, NH * D) @ p["out"].t()) @ p["embed"].t(), -1)
    live = target != -100
    logp = torch.where(live, lp.gather(-1, target.clamp(min=0)[..., None])[..., 0], torch.zeros_like(lp[..., 0]))
    ent = -(lp.exp() * lp).sum(-1)
    loss = _loss(logp, ent, adv.double(), live)
    return loss, logp, ent, lp, dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def test_policy_gradient_through_both(ops):
    """The longest path adds up sums of 64 + 32 + 150 + 150 + 128 + 64 (to the logits), 64 (log probabilities), 700 + 64 + 150 + 150 + 128 and 300 (rows of
    the weights' gradients) terms: below 2200 roundings of 2^-24, 1.3e-4 of the magnitudes. Random signs leave a sum of n terms sqrt(n) of them, and its
    n roundings sqrt(n) as well, so 1.3e-4 is held with room against the L2 norm of each result."""
    model = Policy(1)
    tok, kmask, target, adv = _batch(2, 150, 2)
    live = target != -100
    logits = model(ops, tok, kmask)
    logp, ent, tl, ti = ops.token_logprobs(logits, target, top=5)
    loss = _loss(logp, ent, adv, live)
    grads = dict(zip((n for n, _ in model.named_parameters()), torch.autograd.grad(loss, list(model.parameters()))))
    rloss, rlogp, rent, rlp, rgrads = _reference(model, tok, kmask, target, adv)
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()
    bound = 2200 * 2.0 ** -24
    assert abs(loss.item() - rloss.item()) <= bound * (rlogp * adv).abs().sum().item()
    assert rel(logp.detach(), rlogp) <= bound and rel(ent.detach(), rent) <= bound
    assert rel(tl[live], rlp.topk(5, -1)[0][live]) <= bound
    assert torch.equal(tl, tl.sort(-1, descending=True)[0]) and rel(tl[live], rlp.gather(-1, ti)[live]) <= bound
    for n, g in grads.items():
        assert rel(g, rgrads[n]) <= bound, (n, rel(g, rgrads[n]))


def test_captured_training_step_follows_the_eager_one(ops):
    """FlatTrainer over both operators: graphs replayed on new batches against a twin that runs eagerly. Equal bits step by step is too much to ask of the
    optimizer's inputs (its norm is summed in any order), so the losses are held: four steps of lr 1e-3 change a weight by at most 4e-3, a
    relative gradient difference of 1e-6 moves that by at most 4e-9 where Adam's quotient is regular; the loss, a sum over 2 x 150 rows, is held to 1e-4."""
    from vln_imagine_amd.train import FlatTrainer
    twin = Policy(1)
    model = Policy(1)
    tr, tw = FlatTrainer(model, lr=1e-3), FlatTrainer(twin, lr=1e-3)
    batches = [_batch(2, 150, s) for s in range(4)]
    stage = [t.clone() for t in batches[0]]

    def step(m, b):
        tok, kmask, target, adv = b
        logp, ent, _, _ = ops.token_logprobs(m(ops, tok, kmask), target)
        loss = _loss(logp, ent, adv, target != -100)
        loss.backward()
        return loss.detach()
    try:
        graphed = tr.capture(lambda: step(model, stage))            # one real warm-up step on the first batch
        tw.zero_grad()
        step(twin, batches[0])
        tw.step()
        before = model.table.detach().clone()
        for b in batches:
            for s, t in zip(stage, b):
                s.copy_(t)
            a = graphed()
            tw.zero_grad()
            e = step(twin, b)
            tw.step()
            torch.cuda.synchronize()
            assert abs(a.item() - e.item()) <= 1e-4 * max(1.0, abs(e.item())), (a.item(), e.item())
        assert not torch.equal(model.table, before)                 # the bias is trained through the arena
    finally:
        tr.close()
        tw.close()


def _both(ops, run):
    """Gradients of both operators with `run` around the graph that saves their tensors."""
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g).cuda()
    y, table, x = rnd(2, 150, 8, 64).to(BF16), rnd(16, 4), rnd(40, 3, 5000).to(BF16)
    km = torch.where(torch.arange(150)[None] < torch.tensor([[150], [70]]), 0.0, float("-inf")).float().cuda()
    dout, dl = rnd(2, 150, 4, 64).to(BF16), rnd(40, 3)
    t = torch.randint(0, 5000, (40, 3), generator=g).cuda()
    leaves = [v.requires_grad_(True) for v in (y, table, x)]
    attend = lambda y, tb: ops.long_attention(y[:, :, :4], y[:, :, 4:6], y[:, :, 6:], kmask=km, rel_table=tb, rel_max=64)
    score = lambda x: ops.token_logprobs(x[:, 1], t[:, 1])[0]      # rows with gaps
    out, lp = run(attend, y, table), run(score, x)
    junk = [torch.full((2, 150, 4, 64), 7.0, dtype=BF16, device="cuda") for _ in range(8)]   # takes the place of what was let go
    gs = torch.autograd.grad([out, lp], leaves, [dout, dl[:, 1]])
    del junk
    return [out.detach(), lp.detach(), *gs]


def test_checkpointed_and_offloaded_tensors(ops):
    from torch.utils.checkpoint import checkpoint
    plain = _both(ops, lambda f, *a: f(*a))
    again = _both(ops, lambda f, *a: checkpoint(f, *a, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(plain, again))

    def offloaded(f, *a):
        with torch.autograd.graph.save_on_cpu():                   # comes back contiguous: in other strides than it was saved in
            return f(*a)
    assert all(torch.equal(a, b) for a, b in zip(plain, _both(ops, offloaded)))


def test_a_scale_on_the_device_counts_with_its_value_of_the_call(ops):
    q = torch.randn((1, 40, 2, 64), generator=torch.Generator().manual_seed(1)).cuda()
    scale = torch.tensor(0.125, device="cuda")
    a = ops.long_attention(q, q, q, scale=scale)
    scale.fill_(0.5)
    b = ops.long_attention(q, q, q, scale=scale)
    assert torch.equal(a, ops.long_attention(q, q, q, scale=0.125)) and torch.equal(b, ops.long_attention(q, q, q, scale=0.5)) and not torch.equal(a, b)


def _pass(ops, q, k, v, dout, table):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = ops.long_attention(*leaves[:3], causal=True, rel_table=leaves[3], rel_max=200, rel_bidirectional=False)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def _wide(seed, S):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(t).cuda() for s, t in (((1, S, 4, 128), BF16), ((1, S, 2, 128), BF16), ((1, S, 2, 128), BF16), ((1, S, 4, 128), BF16), ((24, 4), F32))]


def test_captured_heads_of_128(ops):
    """More than 64 KiB of LDS a block, split along the keys: recorded, and replayed with eager calls in between."""
    args = _wide(1, 1500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _pass(ops, *args)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = _pass(ops, *args)
    for r in range(3):
        for a, b in zip(args, _wide(5 + r, 1500)):
            a.copy_(b)
        g.replay()
        want = _pass(ops, *args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), r


def test_two_streams_at_once(ops):
    """Passes that overlap on two streams share nothing: the bits of each are those of a pass alone."""
    jobs = [_wide(1, 1500), _wide(2, 1100)]
    want = [_pass(ops, *j) for j in jobs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for j, st in zip(jobs, streams):
            with torch.cuda.stream(st):
                got.append(_pass(ops, *j))
    torch.cuda.synchronize()
    for i, res in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(res, want[i % 2])), i
