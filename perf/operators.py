"""Measured cases of the post-training operators (``ops/losses.py``): log-probabilities of given tokens, the clipped policy loss with a KL term,
the paired preference loss, distillation from a teacher's top logits - each with the gradient of the logits - and the scoring of given tokens
straight from hidden states.

Vocabularies are those of the framework's own configurations: 260 (bytes), 32000 (llama-50m, 8b as it is scored here), 50257 (gpt2-small; rows of
an odd number of values), 50304 (the same, padded: the padding's logits are masked with -inf), 128256 (llama-3-8b).  Logits are those of a
model that has learnt something: the token that was taken stands out by more or less.  Sequences have a prompt in front, whose tokens are
not scored, and different lengths.

``exact`` states every operator in float64."""
from __future__ import annotations

import math

import torch

own = False                                     # True: the framework's operators, False: their plain forms

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    rows = lambda name, op, B, S, V, dtype="bf16", **kw: dict(name=name, op=op, batch=B, seq=S, vocab=V, dtype=dtype, **kw)
    return [
        rows("logprobs_bytes_1x17", "logprobs", 1, 17, 260, "fp32"),          # one short text of a byte model, in 32 bits: launches count
        rows("logprobs_gpt2_2x700", "logprobs", 2, 700, 50257),               # rows that start at any 2 bytes
        rows("policy_bytes_4x24", "policy", 4, 24, 260, "fp32", old=False, ref=False, clip="0.2", mean="sequences", kl="k3"),   # a first try on a toy model
        rows("policy_50m_8x544", "policy", 8, 544, 32000, old=False, ref=True, clip="0.2", mean="sequences", kl="k3"),          # a group of eight, on policy
        rows("policy_8b_4x2048", "policy", 4, 2048, 128256, old=True, ref=True, clip="0.2,0.28", mean="tokens", kl="k3"),       # long answers, several epochs on one rollout
        rows("preference_50m_4x160", "preference", 4, 160, 32000, loss="sigmoid", average=False),     # pairs of short answers
        rows("preference_8b_2x1000", "preference", 2, 1000, 128256, loss="squared", average=True),    # pairs of long ones
        rows("distill_gpt2_2x333", "distill", 2, 333, 50304, top=20, temperature=1.0, masked=47),     # stored top 20 of an API
        rows("distill_50m_8x1024", "distill", 8, 1024, 32000, top=64, temperature=2.0),               # a student's full batch
        rows("score_8b_1x61", "score", 1, 61, 128256, hidden=4096),           # one short answer under the reference model: the head's weight is what is read
        rows("score_50m_8x1024", "score", 8, 1024, 32000, hidden=512),        # rollouts of the small model
        rows("score_8b_2x2500", "score", 2, 2500, 128256, hidden=4096),       # perplexity of long texts
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "distill", "score"])
    V = rng.choice([260, 32000, 50257, 50304, 128256, _log_between(rng, 200, 130000), _log_between(rng, 200, 130000)])
    most = 4 * 2048 * 128256 // (2 if op == "preference" else 1)
    B = _log_between(rng, 1, 16)
    S = _log_between(rng, 2, min(4096, max(2, most // (B * V * (2 if op == "preference" else 1)))))
    case = dict(op=op, batch=B, seq=S, vocab=V, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if op == "score":
        case |= dict(dtype="bf16", hidden=8 * _log_between(rng, 8, 512))
        case["seq"] = max(2, min(S, int(5000 * 128256 * 4096 / (B * V * case["hidden"]))))
    elif case["dtype"] == "fp32":
        case["seq"] = max(2, S // 2)
    if op == "policy":
        case |= dict(old=rng.random() < 0.6, ref=rng.random() < 0.6, clip=rng.choice(["0.2", "0.2,0.28", "none"]), mean=rng.choice(["tokens", "sequences"]),
                     kl=rng.choice(["k3", "k3", "k1"]))
    elif op == "preference":
        case |= dict(loss=rng.choice(["sigmoid", "sigmoid", "hinge", "squared"]), average=rng.random() < 0.4)
    elif op == "distill":
        case |= dict(top=min(V // 2, _log_between(rng, 1, 256)), temperature=rng.choice([1.0, 2.0, 0.7]), masked=rng.choice([0, min(47, V // 4)]))
    return case


# ------------------------------------------------------------------------------------------------- inputs
def _spans(case):
    """(first, end) of the scored positions of every sequence: behind its prompt, up to its length."""
    S = case["seq"]
    n = case["batch"] * (2 if case["op"] == "preference" else 1)
    prompt = [(7919 * i + 3) % (S // 3 + 1) for i in range(n)]
    end = [S - 1 - (104729 * i) % (S // 4 + 1) for i in range(n)]              # the last position has no token behind it
    return [(min(a, b - 1) if b > 0 else 0, max(b, 1)) for a, b in zip(prompt, end)]


def _scored(case):
    return sum(b - a for a, b in _spans(case))


def _lse(z):
    m = z.max(-1, keepdim=True).values
    return (m + (z - m).exp().sum(-1, keepdim=True).log())[..., 0]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.rand(shape, generator=g, device="cuda")
    randn = lambda *shape, **kw: torch.randn(shape, generator=g, device="cuda", **kw)
    B, S, V, op = case["batch"] * (2 if case["op"] == "preference" else 1), case["seq"], case["vocab"], case["op"]
    dtype = DTYPES[case["dtype"]]
    live = V - case.get("masked", 0)
    targets = torch.randint(0, live, (B, S), generator=g, device="cuda")
    at = torch.arange(S, device="cuda")
    spans = torch.tensor(_spans(case), device="cuda")
    keep = (at >= spans[:, :1]) & (at < spans[:, 1:])
    st = dict(case=case, targets=torch.where(keep, targets, torch.full_like(targets, IGNORE)))
    if op == "score":
        H = case["hidden"]
        w = randn(V, H, dtype=torch.bfloat16) * 0.02                            # a head as it is initialised
        x = randn(B * S, H, dtype=torch.bfloat16) * (2.0 / (0.02 * math.sqrt(H))) * 0.5
        flat = st["targets"].reshape(-1)
        lean = (w[flat.clamp(min=0)].float() * (rand(B * S, 1) * 6 / (0.0004 * H))).to(torch.bfloat16)
        st |= dict(x=x + lean, weight=w, targets=flat)                          # states that lean to the token that follows
        return st
    z = randn(B, S, V, dtype=dtype).mul_(2.5)
    z.scatter_add_(2, targets[..., None], (rand(B, S, 1) * 14).to(dtype))
    if live < V:
        z[..., live:] = float("-inf")
    st["logits"] = z
    if op == "logprobs":
        st["dlogp"] = randn(B, S)
    elif op == "policy":
        st["advantages"] = 0.5 + (randn(B) if case["mean"] == "sequences" else randn(B, S))     # of an answer, or of every token
        lp = _taken(z, targets)
        if case["old"]:
            d = 0.12 * randn(B, S)                                              # an older policy; no ratio stands on a border of the clip
            lo, hi = _clip(case) or (0.2, 0.2)
            for edge in (math.log1p(-lo), math.log1p(hi)):
                d = torch.where((d - edge).abs() < 2e-3, torch.full_like(d, edge + 2e-3), d)
            st["old"] = lp - d
        if case["ref"]:
            st["ref"] = lp + 0.3 * randn(B, S) - 0.1
    elif op == "preference":
        lp = torch.where(keep, _taken(z, targets), torch.zeros((), device="cuda")).double().sum(1)
        gap = torch.where(rand(B // 2) < 0.3, 6.5 + 2 * rand(B // 2), 12 + 28 * rand(B // 2)) * torch.where(rand(B // 2) < 0.1, -1.0, 1.0)
        share = rand(B // 2)                                                    # of the chosen answer in the pair's margin
        ref = lp - torch.cat([gap * share, gap * (share - 1)])
        st["ref"] = (ref / keep.sum(1) if case["average"] else ref).float()
    elif op == "distill":
        K = case["top"]
        teacher = randn(B, S, K).mul_(2).sort(-1, descending=True).values
        ids = (targets[..., None] + torch.arange(K, device="cuda") * (live // K)) % live
        ids = torch.where(keep[..., None], ids, torch.full_like(ids, -1))       # positions that are not trained on have no entries
        if K > 4:
            short = rand(B, S, 1) < 0.1                                         # and some rows have fewer than K
            ids = torch.where(short & (torch.arange(K, device="cuda") >= K // 2), torch.full_like(ids, -1), ids)
        st |= dict(top_ids=ids, top_logits=teacher)
    return st


def _taken(z, targets):
    """log p of the targets, row block by row block (inputs only)."""
    out = []
    for rows, t in zip(z.flatten(0, 1).split(2048), targets.flatten().split(2048)):
        f = rows.float()
        out.append(f.gather(1, t[:, None])[:, 0] - torch.logsumexp(f, -1))
    return torch.cat(out).view(targets.shape)


def _clip(case):
    c = case["clip"]
    if c == "none":
        return None
    v = [float(x) for x in c.split(",")]
    return (v[0], v[-1])


KL_COEF, BETA, SMOOTH = 0.04, 0.1, 0.05


# ------------------------------------------------------------------------------------------------- one pass
def run(st):
    return _own(st) if own else _plain(st)


def _own(st):
    from transformers_fusion_b200.ops import losses as L
    case, op = st["case"], st["case"]["op"]
    if op == "logprobs":
        lp, lse = L.logprobs_fwd(st["logits"], st["targets"])
        return dict(logp=lp, dlogits=L.logprobs_bwd(st["dlogp"], st["logits"], st["targets"], lse))
    if op == "policy":
        o = L.policy_loss_fwd_bwd(st["logits"], st["targets"], st["advantages"], st.get("old"), st.get("ref"), clip=_clip(case),
                                  kl_coef=KL_COEF if case["ref"] else 0.0, kl=case["kl"], mean=case["mean"])
        return dict(loss=o.loss, kl=o.kl, logp=o.logp, dlogits=o.dlogits)
    if op == "preference":
        o = L.preference_loss_fwd_bwd(st["logits"], st["targets"], st["ref"], beta=BETA, kind=case["loss"], average=case["average"],
                                      label_smoothing=SMOOTH if case["loss"] == "sigmoid" else 0.0)
        return dict(loss=o.loss, margins=o.margins, logp=o.logp, dlogits=o.dlogits)
    if op == "distill":
        o = L.distill_loss_fwd_bwd(st["logits"], st["top_ids"], st["top_logits"], temperature=case["temperature"])
        return dict(loss=o.loss, kl=o.kl, dlogits=o.dlogits)
    lp, lse = L.linear_logprobs(st["x"], st["weight"], st["targets"])
    return dict(logp=lp, lse=lse)


def _plain(st):
    case, op = st["case"], st["case"]["op"]
    if op == "score":
        keep = st["targets"] != IGNORE
        z = st["x"].float() @ st["weight"].float().t()
        lse = _lse(z)
        lp = z.gather(1, st["targets"].clamp(min=0)[:, None])[:, 0] - lse
        zero = torch.zeros((), device="cuda")
        return dict(logp=torch.where(keep, lp, zero), lse=torch.where(keep, lse, zero))
    z, dtype = st["logits"].float(), st["logits"].dtype
    zero = torch.zeros((), device="cuda")
    if op == "distill":
        tau, ids = case["temperature"], st["top_ids"]
        have = ids >= 0
        keep = have.any(-1)
        q = torch.where(have, st["top_logits"].float() / tau, torch.full((), float("-inf"), device="cuda"))
        lq = torch.where(have, q - torch.where(keep, _lse(torch.where(keep[..., None], q, zero)), zero)[..., None], zero)
        q = torch.where(have, lq.exp(), zero)
        z = z / tau
        lse = _lse(z)
        lp = z.gather(2, ids.clamp(min=0)) - lse[..., None]
        kl = torch.where(keep, (q * torch.where(have, lq - lp, zero)).sum(-1), zero)
        w = tau / keep.sum().clamp(min=1)
        d = (z - lse[..., None]).exp_().mul_((w * keep)[..., None])
        d.scatter_add_(2, ids.clamp(min=0), -w * q)
        return dict(loss=kl.sum() * tau * w, kl=kl, dlogits=d.to(dtype))
    keep = st["targets"] != IGNORE
    tgt = st["targets"].clamp(min=0)
    lse = _lse(z.double() if op == "preference" else z)                         # a margin is the difference of two long sums
    lp = torch.where(keep, z.gather(2, tgt[..., None])[..., 0] - lse, zero)
    lse, out = lse.float(), {}
    if op == "logprobs":
        c = torch.where(keep, st["dlogp"], zero)
    elif op == "policy":
        A = st["advantages"] if st["advantages"].dim() == 2 else st["advantages"][:, None]
        clip = _clip(case)
        if clip is None and not case["old"]:
            s, ds = A * lp, A.expand_as(lp)
        else:
            r = (lp - st["old"]).exp() if case["old"] else torch.ones_like(lp)
            s = ds = r * A
            if clip is not None:
                c = r.clamp(1 - clip[0], 1 + clip[1]) * A
                ds = torch.where(s <= c, s, zero)
                s = torch.minimum(s, c)
        kl, dkl = zero.expand_as(lp), zero.expand_as(lp)
        if case["ref"]:
            x = st["ref"] - lp
            kl, dkl = (torch.expm1(x) - x, -torch.expm1(x)) if case["kl"] == "k3" else (x, -torch.ones_like(x))
        coef = KL_COEF if case["ref"] else 0.0
        w = keep / (keep.sum().clamp(min=1) if case["mean"] == "tokens" else len(lp) * keep.sum(1, keepdim=True).clamp(min=1))
        c = w * (coef * dkl - ds)
        out = dict(loss=(w * (coef * kl - s)).sum(), kl=(w * kl).sum(), logp=lp)
    else:
        n = keep.sum(1).clamp(min=1).float() if case["average"] else torch.ones(len(lp), device="cuda")
        L = lp.sum(1) / n
        d = L - st["ref"]
        N = len(L) // 2
        h = (d[:N] - d[N:]).float()
        if case["loss"] == "sigmoid":
            b = BETA * h
            soft = torch.log1p((-b.abs()).exp())                                # log(1 + exp(-|b|))
            l, dl = soft + (-b).clamp(min=0) + SMOOTH * b, BETA * (SMOOTH - 1 / (1 + b.exp()))
        elif case["loss"] == "hinge":
            l, dl = (1 - BETA * h).clamp(min=0), -BETA * (BETA * h < 1).float()
        else:
            l, dl = (h - 0.5 / BETA) ** 2, 2 * (h - 0.5 / BETA)
        c = torch.cat([dl, -dl])[:, None] / N / n[:, None] * keep
        out = dict(loss=l.mean(), margins=BETA * h, logp=L.float())
    d = (z - lse[..., None]).exp_().mul_(-c[..., None])
    d.scatter_add_(2, tgt[..., None], c[..., None])
    return dict(out, dlogits=d.to(dtype)) if out else dict(logp=lp, dlogits=d.to(dtype))


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    V, e = case["vocab"], 4 if case["dtype"] == "fp32" else 2
    T = case["batch"] * case["seq"] * (2 if case["op"] == "preference" else 1)
    live = _scored(case)
    if case["op"] == "score":
        H = case["hidden"]
        return {"bytes": (live + V) * H * e + T * 16, "flops": 2.0 * live * V * H}
    small = 8 * T + {"logprobs": 8 * T, "policy": 4 * T * (1 + case.get("old", False) + case.get("ref", False)), "preference": 8 * case["batch"],
                     "distill": T * case.get("top", 0) * 12}[case["op"]]
    return {"bytes": live * V * e + T * V * e + small, "flops": 6.0 * live * V}


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    f64, op = torch.float64, case["op"]
    y = st["targets"].flatten()
    on = y != IGNORE

    def blocks(n=1024):
        """(rows, logits in 64 bits) of every block of positions."""
        for a in range(0, y.numel(), n):
            rows = slice(a, min(y.numel(), a + n))
            yield rows, (st["x"][rows].to(f64) @ st["weight"].to(f64).T if op == "score" else st["logits"].flatten(0, 1)[rows].to(f64))
    if op == "distill":
        tau, kl, grads, K = case["temperature"], [], [], case["top"]
        ids, tl = st["top_ids"].view(-1, K), st["top_logits"].view(-1, K).to(f64)
        count = int((ids >= 0).any(1).sum())
        for rows, z in blocks():
            i, p = ids[rows], torch.softmax(z / tau, 1)
            e = torch.exp(tl[rows] / tau) * (i >= 0)
            q = e / e.sum(1, keepdim=True).clamp(min=1e-300)
            ratio = torch.where(q > 0, q.clamp(min=1e-300).log() - torch.log_softmax(z / tau, 1).gather(1, i.clamp(min=0)), torch.zeros((), dtype=f64, device="cuda"))
            kl.append((q * ratio).sum(1))
            p = p * (i >= 0).any(1, keepdim=True)
            for k in range(K):                                                  # one entry after the other: an id may come twice
                p[torch.arange(len(p), device="cuda"), i[:, k].clamp(min=0)] -= q[:, k]
            grads.append((p * tau / max(1, count)).float())
        kl = torch.cat(kl)
        return dict(loss=tau ** 2 * kl.sum() / max(1, count), kl=kl.view(st["targets"].shape), dlogits=torch.cat(grads).view(st["logits"].shape))
    lp, ls = torch.zeros(y.numel(), dtype=f64, device="cuda"), torch.zeros(y.numel(), dtype=f64, device="cuda")
    for rows, z in blocks():
        ls[rows] = torch.logsumexp(z, 1) * on[rows]
        lp[rows] = torch.log_softmax(z, 1)[torch.arange(len(z), device="cuda"), y[rows].clamp(min=0)] * on[rows]
    if op == "score":
        return dict(logp=lp, lse=ls)
    lp = lp.view(st["targets"].shape).requires_grad_(True)
    on2 = on.view(lp.shape).to(f64)
    out = {}
    if op == "logprobs":
        total = (lp * st["dlogp"].to(f64) * on2).sum()
        out = dict(logp=lp.detach())
    elif op == "policy":
        A = st["advantages"].to(f64)
        A = A if A.dim() == 2 else A[:, None].expand_as(lp)
        per = -A * lp                                                           # without an older policy and without a clip
        if case["old"] or case["clip"] != "none":
            r = torch.exp(lp - (st["old"].to(f64) if case["old"] else lp.detach()))
            lo, hi = _clip(case) or (1.0, math.inf)
            per = -torch.min(r * A, torch.clip(r, 1 - lo, 1 + hi) * A)
        kl = torch.zeros_like(lp)
        if case["ref"]:
            gap = st["ref"].to(f64) - lp
            kl = gap.exp() - gap - 1 if case["kl"] == "k3" else gap
            per = per + KL_COEF * kl
        if case["mean"] == "tokens":
            mean = lambda v: (v * on2).sum() / on2.sum().clamp(min=1)
        else:
            mean = lambda v: ((v * on2).sum(1) / on2.sum(1).clamp(min=1)).mean()
        total = mean(per)
        out = dict(loss=total.detach(), kl=mean(kl).detach(), logp=(lp * on2).detach())
    else:
        L = (lp * on2).sum(1)
        if case["average"]:
            L = L / on2.sum(1).clamp(min=1)
        a, b = (L - st["ref"].to(f64)).chunk(2)
        m = a - b
        if case["loss"] == "sigmoid":
            l = -(1 - SMOOTH) * torch.nn.functional.logsigmoid(BETA * m) - SMOOTH * torch.nn.functional.logsigmoid(-BETA * m)
        elif case["loss"] == "hinge":
            l = torch.relu(1 - BETA * m)
        else:
            l = (m - 1 / (2 * BETA)) ** 2
        total = l.mean()
        out = dict(loss=total.detach(), margins=(BETA * m).detach(), logp=L.detach())
    (c,) = torch.autograd.grad(total, lp)
    c, grads = c.flatten(), []
    for rows, z in blocks():
        d = -torch.softmax(z, 1)
        d[torch.arange(len(d), device="cuda"), y[rows].clamp(min=0)] += 1
        grads.append((d * (c[rows] * on[rows])[:, None]).float())
    return dict(out, dlogits=torch.cat(grads).view(st["logits"].shape))
