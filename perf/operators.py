"""Operators that are measured one by one: attention over long sequences with its recomputing backward pass, the same with a learned relative
position bias by buckets (and the gradient of its table), and log probabilities of given tokens with entropy and top alternatives.

`own = False`: the operators in elementary torch operations, in 32 bits. `own = True`: the calls of vln_imagine_amd.ops.

attention   t_ij = scale <q_i, k_j> + kmask_j + table[bucket(j - (i + Sk - Sq)), head];  P = softmax_j(t);  out = P v
            a key whose mask is -inf, and with `causal` a key j > i + Sk - Sq, takes no part; a row without keys gives zeros and no gradient
bucket      distances below half of a side's n buckets have one each, the others are spread over log(distance) up to rel_max, the last one takes
            everything beyond; bidirectional: the upper half of the table is for keys behind the query, otherwise those count as distance 0
log probs   logp = x_target - logsumexp(x);  H = -sum p log p;  the `top` largest log probabilities and their indices (ties: lowest index);
            ignored targets give logp 0; a row of -inf only: logp -inf, H 0, no gradient
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100


def _attn(name, B, Sq, Sk, nh, nkv, D, dtype="bf16", causal=False, mask="none", rel=0, rel_max=0, bidir=True, train=True):
    c = dict(op="attn", dtype=dtype, B=B, Sq=Sq, Sk=Sk, nh=nh, nkv=nkv, D=D, causal=causal, mask=mask, rel=rel, rel_max=rel_max, bidir=bidir, train=train)
    return dict(name=name, **c) if name else c


def _logp(name, rows, V, top, dtype="bf16", masked=0.0, train=True):
    c = dict(op="logp", dtype=dtype, rows=rows, V=V, top=top, masked=masked, train=train)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one 200-token instruction (DUET's --max_instr_len), 12 heads of 64: the smallest training call, latency
        _attn("attn_instruction", 1, 200, 200, 12, 12, 64, mask="neg"),
        # a batch of ragged multi-paragraph texts, padded to 1024 with excluded keys
        _attn("attn_text_batch", 8, 1024, 1024, 12, 12, 64, mask="pad"),
        # causal pass over a 4 k context, three query heads to a key head, float16
        _attn("attn_causal_4k", 2, 4096, 4096, 12, 4, 64, dtype="f16", causal=True),
        # the largest: 8 k context, heads of 128
        _attn("attn_causal_8k", 1, 8192, 8192, 16, 16, 128, causal=True),
        # the float32 parity path at an odd length, one sample of the batch empty
        _attn("attn_f32_odd", 4, 577, 577, 12, 12, 64, dtype="f32", mask="empty"),
        # one new token per sequence against a cache of 8191, four query heads to a key head
        _attn("attn_token", 16, 1, 8191, 16, 4, 128, causal=True, train=False),
        # text encoder with a learned bias over 2 k tokens, ragged batch, training
        _attn("rel_text_2k", 4, 2048, 2048, 12, 12, 64, mask="pad", rel=32, rel_max=128),
        # causal, one-sided buckets, odd length, left-padded batch whose mask holds the type's lowest value
        _attn("rel_causal_odd", 3, 1501, 1501, 8, 8, 64, dtype="f16", causal=True, mask="left", rel=24, rel_max=256, bidir=False),
        # action head of a rollout: 64 episodes x 15 steps, 37 views, impossible moves at -inf; policy gradient with entropy bonus
        _logp("logp_actions", 960, 37, 3, dtype="f32", masked=0.4),
        # masked-token head over the text vocabulary, 64 x 80 tokens, training
        _logp("logp_vocab", 5120, 30522, 0),
        # the same scored for reporting: forward only, with the eight best alternatives
        _logp("logp_vocab_top8", 2048, 30522, 8, train=False),
        # one answer token of eight sequences, float32 logits, five alternatives
        _logp("logp_token", 8, 30522, 5, dtype="f32", train=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["train", "train", "rel", "rel", "token", "logp", "logp", "score"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("train", "rel", "token"):
        D = rng.choice([32, 64, 64, 96, 128])
        nkv = rng.choice([1, 2, 3, 4, 8, 12])
        nh = nkv * rng.choice([g for g in (1, 1, 2, 3, 4) if g * nkv <= 16])
        causal = rng.random() < 0.5
        top = 2048 if dtype == "f32" else 6000
        if kind == "token":
            Sq, Sk = rng.choice([1, 1, 2, 5]), _log_int(rng, 16, 16000)
        else:
            Sq = _log_int(rng, 24, top)
            Sk = Sq if rng.random() < 0.7 else max(Sq, _log_int(rng, 24, top)) if causal else _log_int(rng, 24, top)
        most = 16 * 8192 * 8192 // (4 if dtype == "f32" else 2)
        B = min(_log_int(rng, 1, 32), max(1, most // (nh * Sq * Sk)), max(1, (1 << 28) // (nkv * Sk * D)))
        mask = rng.choice(["none", "pad", "neg", "empty"] if not causal else ["none", "pad", "left"])
        if kind == "rel":
            bidir = not causal or rng.random() < 0.3
            rel = 2 * rng.choice([4, 8, 16]) if bidir else rng.choice([8, 13, 32])
            return _attn(None, B, Sq, Sk, nh, nkv, D, dtype, causal, mask, rel, rng.choice([37, 64, 128, 300]), bidir)
        return _attn(None, B, Sq, Sk, nh, nkv, D, dtype, causal, mask, train=kind == "train")
    V = _log_int(rng, 2, 60000)
    rows = min(_log_int(rng, 1, 20000), max(1, 150_000_000 // V))
    return _logp(None, rows, V, min(V, rng.choice([0, 1, 3, 5, 8])), dtype, rng.choice([0.0, 0.0, 0.3]), train=kind == "logp")


# ------------------------------------------------------------------------------------------------ inputs
def _lens(case, seed):
    """Valid keys per sample: spread evenly over (Sk / 2, Sk], which sample gets which is the seed's choice."""
    B, Sk = case["B"], case["Sk"]
    lens = [max(1, Sk - (b * Sk) // (2 * B)) for b in range(B)]
    if case["mask"] == "empty":
        lens[-1] = 0
    g = torch.Generator().manual_seed(seed)
    return [lens[i] for i in torch.randperm(B, generator=g).tolist()]


def prepare(case, seed):
    dt = DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "logp":
        rows, V = case["rows"], case["V"]
        x = randn(rows, V) * 2.0
        target = torch.randint(0, V, (rows,), generator=g, device="cuda")
        x.scatter_add_(1, target[:, None], randn(rows, 1).abs() * 3.0)          # a trained head favours the target
        if case["masked"]:
            bad = torch.rand((rows, V), generator=g, device="cuda") < case["masked"]
            bad.scatter_(1, target[:, None], False)
            x.masked_fill_(bad, float("-inf"))
        target = torch.where(torch.rand((rows,), generator=g, device="cuda") < 0.1, IGNORE, target)     # finished episodes, unscored tokens
        st = dict(case=case, logits=x.to(dt).requires_grad_(case["train"]), target=target)
        if case["train"]:
            st["g_logp"], st["g_ent"] = randn(rows), 0.1 * randn(rows)
        return st
    B, Sq, Sk, nh, nkv, D = (case[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "D"))
    st = dict(case=case, kmask=None, table=None)
    for n, S, h in (("q", Sq, nh), ("k", Sk, nkv), ("v", Sk, nkv)):
        st[n] = randn(B, S, h, D).to(dt).requires_grad_(case["train"])
    if case["train"]:
        st["dout"] = randn(B, Sq, nh, D).to(dt)
    if case["mask"] != "none":
        lens = torch.tensor(_lens(case, seed), device="cuda")[:, None]
        pos = torch.arange(Sk, device="cuda")[None]
        if case["mask"] == "left":
            off, low = pos < Sk - lens, torch.finfo(torch.float32).min
        else:
            off, low = pos >= lens, -10000.0 if case["mask"] == "neg" else float("-inf")
        st["kmask"] = torch.zeros((B, Sk), device="cuda").masked_fill_(off, low)
    if case["rel"]:
        st["table"] = (0.5 * randn(case["rel"], nh)).requires_grad_(case["train"])
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "logp":
        return _run_logp_own(state, case) if own else _run_logp_plain(state, case)
    return _run_attn_own(state, case) if own else _run_attn_plain(state, case)


def _run_attn_own(st, case):
    from vln_imagine_amd import ops
    rel = {}
    if case["rel"]:
        rel = dict(rel_table=st["table"], rel_max=case["rel_max"], rel_bidirectional=case["bidir"])
    out = ops.long_attention(st["q"], st["k"], st["v"], kmask=st["kmask"], causal=case["causal"], **rel)
    if not case["train"]:
        return [out]
    leaves = [st["q"], st["k"], st["v"]] + ([st["table"]] if case["rel"] else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, st["dout"])]


def _run_logp_own(st, case):
    from vln_imagine_amd import ops
    logp, ent, top_logp, top_idx = ops.token_logprobs(st["logits"], st["target"], top=case["top"], ignore_index=IGNORE)
    outs = [logp.detach(), ent.detach()] + ([top_logp, top_idx] if case["top"] else [])
    if case["train"]:
        outs += torch.autograd.grad([logp, ent], [st["logits"]], [st["g_logp"], st["g_ent"]])
    return outs


def _buckets(case, device):
    """[Sq, Sk] bucket of every pair; the borders of the logarithmic ones are found in whole numbers."""
    Sq, Sk, nb, far = case["Sq"], case["Sk"], case["rel"], case["rel_max"]
    n = nb // 2 if case["bidir"] else nb
    e = n // 2
    border, d = [], e                       # border[b]: the smallest distance of bucket e + 1 + b:  (d / e)^(n - e) >= (far / e)^(b + 1)
    for b in range(1, n - e):
        while d ** (n - e) * e ** b < far ** b * e ** (n - e):
            d += 1
        border.append(d)
    rel = torch.arange(Sk, device=device)[None] - (torch.arange(Sq, device=device)[:, None] + Sk - Sq)
    dist = rel.abs() if case["bidir"] else (-rel).clamp_min(0)
    idx = dist.clamp_max(e)
    for d in border:
        idx = idx + (dist >= d)
    if case["bidir"]:
        idx = idx + n * (rel > 0)
    return idx


def _run_attn_plain(st, case):
    with torch.no_grad():
        B, Sq, Sk, nh, nkv, D = (case[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "D"))
        dt, dev, G, scale = st["q"].dtype, st["q"].device, nh // nkv, 1.0 / math.sqrt(D)
        q = st["q"].float().transpose(1, 2)                                                        # [B, nh, Sq, D]
        k = st["k"].float().transpose(1, 2).repeat_interleave(G, 1)
        v = st["v"].float().transpose(1, 2).repeat_interleave(G, 1)
        out_of = torch.zeros((1, 1, 1, 1), dtype=torch.bool, device=dev)
        t = torch.matmul(q, k.transpose(2, 3)) * scale
        if case["rel"]:
            idx = _buckets(case, dev)
            t += st["table"].float().t()[:, idx][None]
        if st["kmask"] is not None:
            km = st["kmask"][:, None, None]
            out_of = km == float("-inf")
            t += torch.where(out_of, 0.0, km)
        if case["causal"]:
            out_of = out_of | (torch.arange(Sk, device=dev)[None] > torch.arange(Sq, device=dev)[:, None] + Sk - Sq)[None, None]
        t.masked_fill_(out_of, float("-inf"))
        top = t.amax(-1, keepdim=True)
        p = t.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
        s = p.sum(-1, keepdim=True)
        p /= torch.where(s == 0, 1.0, s)
        o = torch.matmul(p, v)
        outs = [o.transpose(1, 2).to(dt)]
        if not case["train"]:
            return outs
        do = st["dout"].float().transpose(1, 2)
        ds = torch.matmul(do, v.transpose(2, 3))
        dv = torch.matmul(p.transpose(2, 3), do)
        ds -= (ds * p).sum(-1, keepdim=True)
        ds *= p
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(2, 3), q) * scale
        outs.append(dq.transpose(1, 2).to(dt))
        for g in (dk, dv):
            outs.append(g.view(B, nkv, G, Sk, D).sum(2).transpose(1, 2).to(dt))
        if case["rel"]:
            # per distance: rows turned round and padded by one column more than the next row needs, so that a diagonal is a column of the sheared view
            x = torch.nn.functional.pad(ds.sum(0).flip(1), (0, Sq)).view(nh, -1)[:, :Sq * (Sk + Sq - 1)].view(nh, Sq, Sk + Sq - 1)
            per = x.sum(1, dtype=torch.float64)                                                    # column c: j - i = c - (Sq - 1)
            first = torch.cat([idx[:, 0].flip(0), idx[0, 1:]])                                     # bucket of every distance
            hot = (first[:, None] == torch.arange(case["rel"], device=dev)[None]).double()
            outs.append(torch.matmul(per, hot).t().float())
        return outs


def _run_logp_plain(st, case):
    with torch.no_grad():
        x = st["logits"].float()
        rows, V, top = case["rows"], case["V"], case["top"]
        target, dev = st["target"], x.device
        keep = (target >= 0) & (target < V)
        m = x.amax(1, keepdim=True)
        empty = m == float("-inf")
        z = x - torch.where(empty, 0.0, m)
        e = z.exp()
        s = e.sum(1, keepdim=True)
        ls = torch.where(empty, 0.0, s).log()
        lp = z - torch.where(empty, 0.0, ls)
        p = e / torch.where(empty, 1.0, s)
        plp = p * torch.where(p == 0, 0.0, lp)
        ent = -plp.sum(1)
        safe = torch.where(keep, target, 0)
        logp = torch.where(keep, lp.gather(1, safe[:, None])[:, 0], 0.0)
        outs = [logp, ent]
        if top:
            idx = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top].contiguous()
            outs += [lp.gather(1, idx), idx]
        if case["train"]:
            g, h = torch.where(keep, st["g_logp"], 0.0)[:, None], st["g_ent"][:, None]
            dx = -p * g - h * (plp + p * ent[:, None])
            dx.scatter_add_(1, safe[:, None], torch.where(empty, 0.0, g))
            outs.append(dx.to(st["logits"].dtype))
        return outs


# ------------------------------------------------------------------------------------------------ work
def _pairs(case):
    """Query-key pairs of one head over the batch that take part (excluded keys do not; finite masks do)."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    lens = _lens(case, 0) if case["mask"] in ("pad", "empty") else [Sk] * B
    if not case["causal"]:
        return Sq * sum(lens)
    off, n = Sk - Sq, 0
    for L in lens:
        lo = max(0, min(Sq, L - off))                    # rows i < lo see i + off + 1 keys, the others L
        first = max(0, -off)
        if lo > first:
            n += (lo - first) * (off + 1) + (lo - 1 + first) * (lo - first) // 2
        n += (Sq - max(lo, first)) * L
    return n


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "logp":
        n = case["rows"] * case["V"]
        small = case["rows"] * (8 + 8 + 12 * case["top"] + (8 if case["train"] else 0))
        return {"bytes": n * es * (2 if case["train"] else 1) + small, "flops": n * (10 if case["train"] else 5)}
    B, Sq, Sk, nh, nkv, D = (case[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "D"))
    keys = sum(_lens(case, 0)) if case["mask"] in ("pad", "empty") else B * Sk
    qo, kv = B * Sq * nh * D * es, keys * nkv * D * es
    nbytes = 2 * qo + 2 * kv + (0 if case["mask"] == "none" else 4 * B * Sk) + 4 * case["rel"] * nh
    if case["train"]:
        nbytes += 2 * qo + 2 * B * Sk * nkv * D * es + 4 * case["rel"] * nh
    return {"bytes": nbytes, "flops": (14 if case["train"] else 4) * _pairs(case) * nh * D}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return _exact_logp(st, case) if case["op"] == "logp" else _exact_attn(st, case)


def _exact_attn(st, case):
    """One head at a time; the gradients follow from d(softmax) = diag(P) - P P^T."""
    B, Sq, Sk, nh, nkv, D = (case[n] for n in ("B", "Sq", "Sk", "nh", "nkv", "D"))
    dev, f8 = st["q"].device, torch.float64
    q, k, v = (st[n].detach().to(f8) for n in "qkv")
    out = torch.zeros((B, Sq, nh, D), dtype=f8, device=dev)
    if case["train"]:
        do = st["dout"].to(f8)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    at = torch.arange(Sq, device=dev)[:, None] + (Sk - Sq)
    key = torch.arange(Sk, device=dev)[None]
    if case["rel"]:
        n = case["rel"] // 2 if case["bidir"] else case["rel"]
        e, far = n // 2, case["rel_max"]
        d = (at - key).abs() if case["bidir"] else (at - key).clamp(min=0)
        spread = torch.floor((n - e) * torch.log(d.to(f8).clamp(min=e) / e) / math.log(far / e) + 1e-9).long()
        which = torch.where(d < e, d, (e + spread).clamp(max=n - 1)) + (n * (key > at).long() if case["bidir"] else 0)
        table = st["table"].detach().to(f8)
        dtable = torch.zeros_like(table)
    for b in range(B):
        seen = torch.ones((Sq, Sk), dtype=torch.bool, device=dev)
        add = torch.zeros((1, Sk), dtype=f8, device=dev)
        if st["kmask"] is not None:
            row = st["kmask"][b].to(f8)[None]
            seen = seen & ~torch.isinf(row)
            add = torch.where(torch.isinf(row), torch.zeros_like(row), row)
        if case["causal"]:
            seen = seen & (key <= at)
        some = seen.any(1, keepdim=True)
        for h in range(nh):
            c = h * nkv // nh
            t = q[b, :, h] @ k[b, :, c].t() / math.sqrt(D) + add
            if case["rel"]:
                t = t + table[:, h][which]
            t = torch.where(seen, t, torch.full_like(t, float("-inf")))
            p = torch.where(some, torch.softmax(torch.where(some, t, torch.zeros_like(t)), 1), torch.zeros_like(t))
            out[b, :, h] = p @ v[b, :, c]
            if case["train"]:
                g = do[b, :, h] @ v[b, :, c].t()
                g = p * (g - (do[b, :, h] * out[b, :, h]).sum(1, keepdim=True))
                dq[b, :, h] = g @ k[b, :, c] / math.sqrt(D)
                dk[b, :, c] += g.t() @ q[b, :, h] / math.sqrt(D)
                dv[b, :, c] += p.t() @ do[b, :, h]
                if case["rel"]:
                    for i in range(case["rel"]):
                        dtable[i, h] += g[which == i].sum()
    if not case["train"]:
        return [out]
    return [out, dq, dk, dv] + ([dtable] if case["rel"] else [])


def _exact_logp(st, case):
    V, top, f8 = case["V"], case["top"], torch.float64
    logp, ent, val, idx, dx = [], [], [], [], []
    step = max(1, (1 << 27) // V)
    for r in range(0, case["rows"], step):
        x, tg = st["logits"].detach()[r:r + step].to(f8), st["target"][r:r + step]
        ok = (tg >= 0) & (tg < V)
        lp = torch.log_softmax(x, 1)
        dead = torch.isinf(x).all(1)
        lp[dead] = float("-inf")
        p = lp.exp()
        info = torch.special.entr(p)
        H = info.sum(1)
        pick = torch.where(ok, tg, torch.zeros_like(tg))
        logp.append(torch.where(ok, lp.gather(1, pick[:, None])[:, 0], torch.zeros_like(H)))
        ent.append(H)
        if top:
            order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :top]
            idx.append(order)
            val.append(lp.gather(1, order))
        if case["train"]:
            a = torch.where(ok & ~dead, st["g_logp"][r:r + step].to(f8), torch.zeros_like(H))[:, None]
            one = torch.zeros_like(x).scatter_(1, pick[:, None], 1.0)
            dx.append(a * (one - p) + st["g_ent"][r:r + step].to(f8)[:, None] * (info - p * H[:, None]))
    res = [torch.cat(logp), torch.cat(ent)]
    if top:
        res += [torch.cat(val), torch.cat(idx)]
    if case["train"]:
        res.append(torch.cat(dx))
    return res
