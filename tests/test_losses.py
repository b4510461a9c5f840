"""Losses of post-training on logits (``ops/losses.py``) against their definitions in float64 with autograd, on the CPU statements and on the kernels.

Tolerances.  Of a row with soft-max p and target y, a kernel's gradient is c (onehot(y) - p), rounded once: half a step of its type.  Before that,
relative to p: the exponent (z - m) log2 e is rounded to 32 bits (values of p above 2^-100: 100 * 2^-24 * ln 2 = 4.2e-6), ex2 is good to 2^-22,
the sum of V terms in at most V / 512 + 16 steps to 2^-24 each on its way (256 steps: 1.5e-5 at V = 131072, far less as they are of both signs), lse in 32 bits to
2^-24 * 32 = 2e-6; c follows lp with the same errors.  REL = 4e-5 holds them all.  lp itself: the sum's relative error, plus its own rounding."""
import math

import pytest
import torch

from transformers_fusion_b200.ops import _lib
from transformers_fusion_b200.ops import losses as L

REL = 4e-5
TINY = 1e-30          # below it values may be flushed to zero (2^-100)
IGN = -100
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF, F32 = torch.bfloat16, torch.float32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(device, seed=0):
    return torch.Generator(device=device).manual_seed(seed)


def make(device, lead, V, dtype, seed=0, ignored=0.3, idx=torch.int64):
    g = gen("cpu", seed)
    z = (3 * torch.randn(*lead, V, generator=g)).to(dtype)
    y = torch.randint(0, V, lead, generator=g)
    z.scatter_add_(-1, y[..., None], (8 * torch.rand(*lead, 1, generator=g)).to(dtype))
    keep = torch.rand(lead, generator=g) >= ignored
    return z.to(device), torch.where(keep, y, torch.full_like(y, IGN)).to(idx).to(device)


def rows64(z, y):
    """(kept rows, z in float64 with gradient, log p of the targets, zero on the others)."""
    keep = y != IGN
    z64 = torch.where(keep[..., None], z.double(), torch.zeros((), dtype=torch.float64, device=z.device)).requires_grad_(True)
    lp = torch.log_softmax(z64, -1).gather(-1, y.long().clamp(min=0)[..., None])[..., 0]
    return keep, z64, torch.where(keep, lp, torch.zeros((), dtype=torch.float64, device=z.device))


def near(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got - want).abs()[bad].max().item(), got[bad][:4].tolist(), want[bad][:4].tolist())


def lp_tol(lp):
    return REL / 2 + 2 ** -23 * lp.abs()


def grad_tol(want, c, p, hot, dtype):
    """Half a step of the type, and REL of what the gradient is the difference of."""
    return half(dtype) * want.abs() * (1 + REL) + REL * c.abs()[..., None] * (p + hot) + TINY


def check_grad(got, z, y, c, dtype):
    """got against c (onehot(y) - p), c in float64 (0 on ignored rows)."""
    keep = y != IGN
    p = torch.softmax(torch.where(keep[..., None], z.double(), torch.zeros((), dtype=torch.float64, device=z.device)), -1)
    hot = torch.zeros_like(p).scatter_(-1, y.long().clamp(min=0)[..., None], 1.0)
    want = torch.where(keep[..., None], c[..., None] * (hot - p), torch.zeros_like(p))
    near(got, want, torch.where(keep[..., None], grad_tol(want, c, p, hot, dtype), torch.zeros_like(p)), "dlogits")


SHAPES = [((1,), 1), ((1,), 2), ((3,), 7), ((2, 3), 64), ((17,), 260), ((5,), 513), ((2, 4), 1000), ((3,), 4096), ((3,), 4097), ((2, 3), 16385), ((3,), 32000),
          ((2,), 50257), ((2, 2), 65537), ((2,), 128256), ((2,), 131073), ((1,), 262149)]


# ------------------------------------------------------------------------------------------------- log-probabilities
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lead,V", SHAPES)
def test_logprobs(dev, dtype, lead, V):
    z, y = make(dev, lead, V, dtype, V, idx=torch.int32 if V % 3 == 0 else torch.int64)
    if len(lead) == 1 and lead[0] == 1:
        y = y.clamp(min=0)
    keep, z64, want = rows64(z, y)
    lp, stats = L.logprobs_fwd(z, y)
    assert lp.dtype == stats.dtype == F32
    near(lp, want.detach(), lp_tol(want.detach()), "logp")
    w_lse = torch.logsumexp(z64, -1).detach() * keep
    near(stats.sum(0), w_lse, lp_tol(w_lse), "lse")
    c = torch.randn(lead, generator=gen("cpu", 5)).to(dev)
    check_grad(L.logprobs_bwd(c, z, y, stats), z, y, c.double(), dtype)
    inside = z.clone().requires_grad_(True)                       # the autograd form
    (g,) = torch.autograd.grad(L.token_logprobs(inside, y), inside, c)
    assert torch.equal(g, L.logprobs_bwd(c, z, y, stats))
    again = z.clone()                                             # in place
    assert L.logprobs_bwd(c, again, y, stats, out=again) is again and torch.equal(again, g)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [33, 1000, 4099, 50257])
@pytest.mark.parametrize("kind", ["no_last", "no_first", "sequence_major", "offset", "expanded", "out_offset", "padded"])
def test_strides(dev, dtype, V, kind):
    B, S = 3, 4
    z, y = make(dev, (B, S + 1), V, dtype, V)
    c, out = torch.randn(B, S, generator=gen("cpu", 5)).to(dev), None
    if kind == "no_last":
        z, y = z[:, :-1], y[:, 1:]
    elif kind == "no_first":
        z, y = z[:, 1:], y[:, :-1]
    else:
        y = y[:, 1:]
        z0 = z[:, 1:].clone()
        z = z0
    if kind == "sequence_major":
        z = z.transpose(0, 1).contiguous().transpose(0, 1)
    elif kind == "offset":
        z = torch.cat([z0.new_zeros(1), z0.flatten()])[1:].view(B, S, V)
    elif kind == "expanded":
        z = z[:, :1].expand(B, S, V)
        out = torch.empty(B, S, V, dtype=dtype, device=dev)
    elif kind == "out_offset":
        out = torch.full((B * S * V + 3,), 7.0, dtype=dtype, device=dev)[3:].view(B, S, V)
    elif kind == "padded":
        z = torch.nn.functional.pad(z, (0, 5), value=float("nan"))[..., :V]
        out = torch.full((B, S, V + 3), 7.0, dtype=dtype, device=dev)[..., :V]
    keep, _, want = rows64(z, y)
    lp, stats = L.logprobs_fwd(z, y)
    near(lp, want.detach(), lp_tol(want.detach()))
    g = L.logprobs_bwd(c, z, y, stats, out=out)
    check_grad(g, z, y, c.double(), dtype)
    if kind == "padded":                                          # behind the rows nothing is written
        assert bool((out.as_strided((B, S, 3), (S * (V + 3), V + 3, 1), V) == 7).all())
    A = torch.randn(B, S, generator=gen("cpu", 6)).to(dev)
    o = L.policy_loss_fwd_bwd(z, y, A, clip=None, mean="sum", out=out)
    check_grad(o.dlogits, z, y, -A.double(), dtype)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [40, 3000, 40000, 100001])
def test_masked_values(dev, dtype, V):
    """Rows: 0 a masked tail, 1 all but the target masked, 2 the target masked, 3 everything masked, 4 masks of the type's lowest value, 5 everything at it,
    6 +inf, 7 NaN, 8 ignored with NaN and inf, 9 a target outside the vocabulary, 10 large values of both signs, 11 ordinary."""
    g = gen("cpu", V)
    z = (2 * torch.randn(12, V, generator=g)).to(dtype)
    y = torch.randint(0, V // 2, (12,), generator=g)
    low = torch.finfo(dtype).min
    z[0, V // 2:] = -math.inf
    z[1] = -math.inf
    z[1, y[1]] = 1.5
    z[2, y[2]] = -math.inf
    z[3] = -math.inf
    z[4, V // 2:] = low
    z[5] = low
    z[6, 3] = math.inf
    z[7, V - 1] = math.nan
    z[8, ::2], z[8, 1], y[8] = math.nan, math.inf, IGN
    y[9] = V
    z[10] *= 1e30
    z, y = z.to(dev), y.to(dev)
    c = torch.full((12,), 0.5, device=dev)
    A = torch.full((12,), -0.5, device=dev)
    lp, stats = L.logprobs_fwd(z, y)
    d = L.logprobs_bwd(c, z, y, stats)
    o = L.policy_loss_fwd_bwd(z, y, A, clip=None, mean="sum")
    for name, got_lp, got in (("logprobs", lp, d), ("policy", o.logp, o.dlogits)):
        for bad in (3, 6, 7, 9):
            assert got_lp[bad].isnan() and got[bad].isnan().any(), (name, bad)
        assert got_lp[8] == 0 and not got[8].any()
        assert got_lp[2] == -math.inf and got_lp[1].abs() < 1e-6
        for r in (0, 1, 2, 4, 5, 10, 11):
            check_grad(got[r:r + 1], z[r:r + 1], y[r:r + 1], c[r:r + 1].double(), dtype)
            want = torch.log_softmax(z[r].double(), -1)[y[r]]
            near(got_lp[r], want, REL / 2 + 2 ** -22 * abs(want.item()) if math.isfinite(want.item()) else 0.0, (name, r))
    assert o.loss.isnan()


# ------------------------------------------------------------------------------------------------- policy
def policy64(z, y, A, old, ref, clip, kl_coef, kl, mean, n_valid=None):
    keep, z64, lp = rows64(z, y)
    lp = lp.detach().requires_grad_(True)
    A = A.double()
    A = (A[:, None] if A.dim() < lp.dim() else A).expand(lp.shape)
    if old is None and clip is None:
        s = A * lp
    else:
        r = torch.exp(lp - (old.double() if old is not None else lp.detach()))
        s = r * A
        if clip is not None:
            s = torch.minimum(s, r.clamp(1 - clip[0], 1 + clip[1]) * A)
    k = torch.zeros_like(lp)
    if ref is not None:
        x = ref.double() - lp
        k = torch.exp(x) - 1 - x if kl == "k3" else x
    w = keep.double()
    if mean == "tokens":
        w = w / (n_valid if n_valid is not None else max(1, int(keep.sum())))
    elif mean == "sequences":
        w = w / (max(1, w.shape[0] if w.dim() == 2 else 1) * w.sum(-1, keepdim=True).clamp(min=1))
    l = -s + kl_coef * k
    loss = (w * l).sum()
    (c,) = torch.autograd.grad(loss, lp)
    slack = REL * (c.abs().sum() + (w * (s.abs() + kl_coef * k.abs())).sum()).item() + TINY
    kslack = REL * (w * (1 + k.abs() + (ref.double() - lp).abs().expm1() if ref is not None else k)).sum().item() + TINY
    return loss.detach(), (w * k).sum().detach(), lp.detach(), c, slack, kslack


POLICY = [dict(), dict(clip=None), dict(old=True), dict(old=True, clip=None), dict(old=True, clip=(0.1, 0.3), mean="sequences"), dict(ref=True, kl_coef=0.1),
          dict(old=True, ref=True, kl_coef=0.05, kl="k1", mean="sum"), dict(old=True, ref=True, kl_coef=0.3, mean="sequences", per_seq=True), dict(ref=True, clip=None, kl="k1"),
          dict(old=True, n_valid=37.0), dict(old=True, clip=0.0)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lead,V", [((1, 1), 5), ((3, 9), 260), ((2, 5), 9001), ((2, 3), 32000), ((1, 2), 50257), ((2, 1), 140000)])
@pytest.mark.parametrize("kw", POLICY, ids=lambda kw: "-".join(f"{k}={v}" for k, v in kw.items()) or "plain")
def test_policy(dev, dtype, lead, V, kw):
    kw = dict(kw)
    z, y = make(dev, lead, V, dtype, 3 + V)
    if lead[0] > 1:
        y[0] = IGN                                                # a sequence without tokens
    g = gen("cpu", 9)
    rand = lambda *s: torch.randn(*s, generator=g).to(dev)
    _, _, lp = rows64(z, y)
    lp = lp.detach()
    A = rand(lead[0]) if kw.pop("per_seq", False) else rand(*lead)
    clip = kw.get("clip", 0.2)
    bounds = None if clip is None else clip if isinstance(clip, tuple) else (clip, clip)
    old = ref = n_valid = None
    if kw.pop("old", False):
        d = 0.25 * rand(*lead)
        for edge in [math.log1p(-bounds[0]), math.log1p(bounds[1])] if bounds else []:      # no ratio within 1e-3 of a border
            d = torch.where((d - edge).abs() < 2e-3, torch.full_like(d, edge + 2e-3 * (1 if edge >= 0 else -1)), d)
        old = (lp - d).float()
    if kw.pop("ref", False):
        ref = (lp + 0.4 * rand(*lead)).float()
    if "n_valid" in kw:
        n_valid = kw["n_valid"]
        kw["n_valid"] = torch.tensor(n_valid, device=dev)
    loss, k, lp, c, slack, kslack = policy64(z, y, A, old, ref, bounds, kw.get("kl_coef", 0.0), kw.get("kl", "k3"), kw.get("mean", "tokens"), n_valid)
    o = L.policy_loss_fwd_bwd(z, y, A, old, ref, **kw)
    near(o.loss, loss, slack, "loss")
    near(o.kl, k, kslack, "kl")
    near(o.logp, lp, lp_tol(lp) * (y != IGN), "logp")
    check_grad(o.dlogits, z, y, c, dtype)
    quiet = L.policy_loss_fwd_bwd(z, y, A, old, ref, want_grad=False, **kw)
    assert quiet.dlogits is None
    near(quiet.loss, o.loss, 2 * slack, "loss without gradient")      # other groups of values are added up first: each of the two is within slack
    near(quiet.logp, o.logp, 2 * lp_tol(lp) * (y != IGN))
    w = z.clone()
    again = L.policy_loss_fwd_bwd(w, y, A, old, ref, out=w, **kw)     # in place, and bit for bit again
    assert again.dlogits is w and torch.equal(w, o.dlogits) and torch.equal(again.loss, o.loss)


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_clip_share_and_flat(dev):
    """Which tokens the clip takes is counted, and [T, V] logits are one sequence."""
    z, y = make(dev, (40,), 50, F32, 4, ignored=0.25)
    _, _, lp = rows64(z, y)
    r = torch.linspace(0.5, 1.5, 40, dtype=torch.float64, device=dev) + 0.003
    A = torch.where(torch.arange(40, device=dev) % 2 == 0, 1.0, -1.0)
    o = L.policy_loss_fwd_bwd(z, y, A, (lp.detach() - r.log()).float(), clip=(0.2, 0.3))
    keep = y != IGN
    lost = keep & (((r > 1.3) & (A > 0)) | ((r < 0.8) & (A < 0)))
    near(o.clipped, lost.double().sum() / keep.sum(), 1e-6)
    assert not o.dlogits[lost | ~keep].any() and bool(o.dlogits[keep & ~lost].any(-1).all())
    one = L.policy_loss_fwd_bwd(z[None], y[None], A[None], (lp.detach() - r.log()).float()[None], clip=(0.2, 0.3), mean="sequences")
    assert torch.equal(one.dlogits[0], o.dlogits) and torch.equal(one.loss, o.loss)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("shape", [(2, 3), (0, 3), (2, 0), (0,)])
def test_nothing_to_train_on(dev, shape):
    z = torch.full((*shape, 11), math.nan, device=dev)
    y = torch.full(shape, IGN, device=dev)
    o = L.policy_loss_fwd_bwd(z, y, torch.full(shape, math.nan, device=dev), mean="tokens")
    assert o.loss == 0 and o.kl == 0 and not o.dlogits.any() and o.dlogits.shape == z.shape
    lp, stats = L.logprobs_fwd(z, y)
    assert not lp.any() and not stats.any() and not L.logprobs_bwd(torch.ones(shape, device=dev), z, y, stats).any()
    d = L.distill_loss_fwd_bwd(z, torch.full((*shape, 4), -1, device=dev), torch.zeros(*shape, 4, device=dev))
    assert d.loss == 0 and not d.dlogits.any() and not d.kl.any()
    if len(shape) == 2:
        p = L.preference_loss_fwd_bwd(z, y, torch.arange(shape[0], device=dev).float())
        want = torch.nn.functional.softplus(torch.tensor(-0.1)) if shape[0] else torch.tensor(0.0)      # h = (0 - 0) - (0 - 1)
        near(p.loss.cpu(), want, 1e-6)
        assert not p.dlogits.any() and not p.logp.any()


# ------------------------------------------------------------------------------------------------- preferences
def preference64(z, y, ref, beta, kind, eps, average):
    keep, _, lp = rows64(z, y)
    lp = lp.detach().requires_grad_(True)
    n = keep.sum(1).clamp(min=1) if average else 1
    s = lp.sum(1) / n
    d = s - (ref.double() if ref is not None else 0)
    h = d[:len(d) // 2] - d[len(d) // 2:]
    if kind == "sigmoid":
        l = -(1 - eps) * torch.nn.functional.logsigmoid(beta * h) - eps * torch.nn.functional.logsigmoid(-beta * h)
    elif kind == "hinge":
        l = torch.relu(1 - beta * h)
    else:
        l = (h - 1 / (2 * beta)) ** 2
    (c,) = torch.autograd.grad(l.mean(), lp)
    return l.mean().detach(), (beta * h).detach(), s.detach(), c, keep


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,S,V", [(1, 1, 9), (3, 17, 260), (2, 5, 32000), (1, 3, 50257), (40, 2, 33)])
@pytest.mark.parametrize("kw", [dict(), dict(label_smoothing=0.1, beta=0.5), dict(kind="hinge", beta=0.02), dict(kind="squared", average=True, beta=1.0), dict(average=True)],
                         ids=["sigmoid", "smooth", "hinge", "squared", "average"])
def test_preference(dev, dtype, N, S, V, kw):
    z, y = make(dev, (2 * N, S), V, dtype, N + V)
    if N > 1:
        y[1] = IGN                                                # an empty answer
    ref = None if N == 40 else (rows64(z, y)[2].detach().sum(1) * 0.97).float()
    beta = kw.get("beta", 0.1)
    loss, x, s, c, keep = preference64(z, y, ref, beta, kw.get("kind", "sigmoid"), kw.get("label_smoothing", 0.0), kw.get("average", False))
    o = L.preference_loss_fwd_bwd(z, y, ref, **kw)
    per = REL / 2 * keep.sum(1).clamp(min=1)                      # of a sum of log-probabilities
    near(o.logp, s, per + 2 ** -23 * s.abs(), "logp")
    wide = beta * (per[:N] + per[N:])
    near(o.margins, x, wide + 2 ** -23 * x.abs(), "margins")
    steep = 1 if kw.get("kind") != "squared" else 2 * (x / beta - 0.5 / beta).abs().max().item() / beta + 1
    near(o.loss, loss, steep * wide.max().item() + 1e-6 * loss.abs().item(), "loss")
    # the coefficient moves with the margin: by at most beta/4 (sigmoid), 2 / beta... per unit of x, relative to c
    move = {"sigmoid": 1.0, "hinge": 0.0, "squared": 2.0 / beta ** 2}[kw.get("kind", "sigmoid")] * wide.max().item() * beta / N
    p = torch.softmax(torch.where(keep[..., None], z.double(), torch.zeros((), dtype=torch.float64, device=dev)), -1)
    hot = torch.zeros_like(p).scatter_(-1, y.long().clamp(min=0)[..., None], 1.0)
    want = c[..., None] * (hot - p) * keep[..., None]
    near(o.dlogits, want, grad_tol(want, c, p, hot, dtype) + move * (p + hot), "dlogits")
    assert not o.dlogits[~keep].any()
    again = L.preference_loss_fwd_bwd(z, y, ref, out=z, **kw)     # in place
    assert torch.equal(again.dlogits, o.dlogits) and again.dlogits is z and torch.equal(again.loss, o.loss)
    assert L.preference_loss_fwd_bwd(o.dlogits, y, ref, want_grad=False, **kw).dlogits is None


# ------------------------------------------------------------------------------------------------- distillation
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lead,V,K", [((1,), 1, 1), ((3,), 7, 9), ((2, 5), 260, 20), ((3,), 4098, 1), ((4,), 32000, 64), ((2,), 50257, 255), ((2, 2), 20000, 1024), ((2,), 150001, 7)])
@pytest.mark.parametrize("tau,kind", [(1.0, "distinct"), (2.0, "twice"), (0.5, "holes")])
def test_distill(dev, dtype, lead, V, K, tau, kind):
    g = gen("cpu", V + K)
    z = (3 * torch.randn(*lead, V, generator=g)).to(dtype)
    top = (2 * torch.randn(*lead, K, generator=g)).to(BF if kind == "holes" else F32)
    ids = torch.randint(0, V, (*lead, K), generator=g)                # ids may come more than once
    if kind == "distinct" and K <= V:
        ids = torch.rand(*lead, V, generator=g).argsort(-1)[..., :K]
    elif kind == "twice" and K > 1:
        ids[..., 1::2] = ids[..., :1]
    elif kind == "holes":
        ids[..., 1:][torch.rand(*lead, K - 1, generator=g) < 0.4] = -1
        ids[0] = -1                                                   # a row (a sequence) that is not trained on
    ids = ids.to(torch.int32 if kind == "twice" else torch.int64)
    z, top, ids = z.to(dev), top.to(dev), ids.to(dev)
    keep, have = ids[..., 0] >= 0, ids >= 0
    z64 = z.double().requires_grad_(True)
    t64 = torch.where(have, top.double() / tau, torch.full((), -math.inf, dtype=torch.float64, device=dev))
    lq = torch.log_softmax(torch.where(keep[..., None], t64, torch.zeros((), dtype=torch.float64, device=dev)), -1)
    q = torch.where(have, lq.exp(), torch.zeros_like(lq))
    lp = torch.log_softmax(z64 / tau, -1).gather(-1, ids.long().clamp(min=0))
    kl = torch.where(have & (q > 0), q * (lq - lp), torch.zeros_like(q)).sum(-1)
    n = max(1, int(keep.sum()))
    loss = tau ** 2 * kl.sum() / n
    (want,) = torch.autograd.grad(loss, z64)
    o = L.distill_loss_fwd_bwd(z, ids, top, temperature=tau)
    ktol = REL * (1 + torch.where(have & (q > 0), q * (lq.abs() + lp.abs()), torch.zeros_like(q)).sum(-1)).detach()
    near(o.kl, kl.detach(), ktol, "kl")
    near(o.loss, loss.detach(), tau ** 2 * ktol.sum().item() / n + 1e-6 * loss.item(), "loss")
    p, back = torch.softmax(z64.detach() / tau, -1) * keep[..., None], torch.zeros(*lead, V, dtype=torch.float64, device=dev)
    back.scatter_add_(-1, ids.long().clamp(min=0), q.detach())
    near(o.dlogits, want, half(dtype) * want.abs() * (1 + REL) + REL * tau / n * (p + back) + TINY, "dlogits")
    assert not o.dlogits[~keep].any()
    part = L.distill_loss_fwd_bwd(z, ids, top, temperature=tau, n_valid=torch.tensor([4.0 * n], device=dev), want_grad=False)
    near(part.loss * 4, o.loss, 1e-6 * o.loss.abs().item())
    again = L.distill_loss_fwd_bwd(z, ids, top, temperature=tau, out=z)
    assert torch.equal(again.dlogits, o.dlogits) and torch.equal(again.loss, o.loss)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [50, 40001])
def test_distill_masked(dev, V):
    """Rows: 0 a teacher's token that the student has masked (KL is infinite, its gradient is not), 1 the student's mask elsewhere, 2 a teacher's mask, 3 all of it,
    4 an id outside the vocabulary, 5 ordinary."""
    g = gen("cpu", V)
    z = torch.randn(6, V, generator=g)
    ids = torch.randint(0, V // 2, (6, 3), generator=g) // 3 * 3 + torch.arange(3)
    top = torch.randn(6, 3, generator=g)
    z[0, ids[0, 1]] = -math.inf
    z[1, V - 5:] = -math.inf
    top[2, 1] = -math.inf
    top[3] = -math.inf
    ids[4, 2] = V
    z, ids, top = z.to(dev), ids.to(dev), top.to(dev)
    o = L.distill_loss_fwd_bwd(z, ids, top, n_valid=torch.ones(1, device=dev))
    assert o.kl[0] == math.inf and o.kl[3].isnan() and o.kl[4].isnan() and o.loss.isnan()
    assert o.dlogits[3].isnan().any() and o.dlogits[4].isnan().any()
    q = torch.softmax(top.double(), -1)
    for r in (0, 1, 2, 5):
        want = torch.softmax(z[r].double(), -1)
        tol = REL * want
        want = want.index_add(0, ids[r], -q[r])
        near(o.dlogits[r], want, half(F32) * want.abs() + tol.index_add(0, ids[r], REL * q[r]) + TINY)
        kl = torch.where(q[r] > 0, q[r] * (q[r].log() - torch.log_softmax(z[r].double(), -1)[ids[r]]), torch.zeros((), dtype=torch.float64, device=dev)).sum()
        near(o.kl[r], kl, REL * (1 + kl.abs().item()) if r else 0)


# ------------------------------------------------------------------------------------------------- scoring
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("lead,H,V", [((1,), 8, 1), ((3, 5), 64, 260), ((2,), 72, 1001), ((1, 129), 128, 2000), ((300,), 64, 517), ((257,), 512, 4000), ((2, 200), 256, 32000), ((61,), 1024, 50257),
                                       ((513,), 136, 777)])
def test_linear_logprobs(dev, lead, H, V):
    g = gen("cpu", V)
    x = torch.randn(*lead, H, generator=g).to(BF).to(dev)
    w = (torch.randn(V, H, generator=g) * 2 / math.sqrt(H)).to(BF).to(dev)
    y = torch.randint(0, V, lead, generator=g)
    y = torch.where(torch.rand(lead, generator=g) < 0.2, torch.full_like(y, IGN), y).to(dev)
    keep = y != IGN
    z = x.double() @ w.double().t()
    # a product of H terms in 32 bits: H * 2^-24 of the sum of their sizes at worst, and the statistics' own error
    size = (x.double().abs() @ w.double().abs().t()).max().item()
    lse = torch.logsumexp(z, -1) * keep
    lp = (z.gather(-1, y.clamp(min=0)[..., None])[..., 0] * keep - lse)
    got, got_lse = L.linear_logprobs(x, w, y)
    tol = REL / 2 + 2 * H * 2 ** -24 * size
    near(got, lp, tol * keep)
    near(got_lse, lse, tol * keep)
    xs = torch.nn.functional.pad(x, (0, 3))[..., :H]                  # rows of another pitch
    ws = torch.nn.functional.pad(w, (1, 0))[:, 1:]
    near(L.linear_logprobs(xs, ws, y.int())[0], lp, tol * keep)


@pytest.mark.parametrize("dev", DEVICES)
def test_linear_logprobs_special(dev):
    """A target outside the vocabulary gives NaN, ignored rows of NaN and empty inputs give nothing."""
    x, w = torch.randn(200, 64).to(BF).to(dev), torch.randn(300, 64).to(BF).to(dev)
    y = torch.arange(200, device=dev)
    y[5], y[6], y[7] = 300, -3, IGN
    x[7] = math.nan
    lp, lse = L.linear_logprobs(x, w, y)
    assert lp[5].isnan() and lp[6].isnan() and lp[7] == 0 and lse[7] == 0
    rest = torch.ones(200, dtype=torch.bool, device=dev)
    rest[5:8] = False
    assert lp[rest].isfinite().all() and lse[[5, 6]].isfinite().all()
    assert L.linear_logprobs(x[:0], w, y[:0])[0].shape == (0,)
    w[3] = math.inf * torch.ones(64, device=dev)
    assert L.linear_logprobs(x[:5].abs(), w, y[:5])[0].isnan().all()


# ------------------------------------------------------------------------------------------------- gradients by differences
@pytest.mark.parametrize("dev", DEVICES)
def test_gradients_by_differences(dev):
    """Central differences of the loss along random directions.  h = 2^-5, |d| = 1 in every row: the third derivative of a row's loss is below 8 |c|
    (h^2 / 6 * 8 = 1.3e-3 |c|), and a loss in 32 bits is off by 2^-23 of its terms (over 2 h: 2e-6)."""
    B, S, V, h = 2, 4, 12, 2.0 ** -5
    z, y = make(dev, (B, S), V, F32, 1, ignored=0.2)
    g = gen("cpu", 2)
    rand = lambda *s: torch.randn(*s, generator=g).to(dev)
    A, ref = rand(B, S), rows64(z, y)[2].detach().float() + 0.3 * rand(B, S)
    ids = torch.rand(B, S, V, generator=g).argsort(-1)[..., :5].to(dev)
    top = rand(B, S, 5)
    kept = int((y != IGN).sum())
    losses = [(lambda t: L.policy_loss_fwd_bwd(t, y, A, None, ref, clip=None, kl_coef=0.2), 3.0),
              (lambda t: L.preference_loss_fwd_bwd(t, y, None, beta=0.5), 2.0 * kept),
              (lambda t: L.distill_loss_fwd_bwd(t, ids, top, temperature=1.5), 1.5)]
    for f, c in losses:
        d = rand(B, S, V)
        d = d / d.norm(dim=-1, keepdim=True)
        o = f(z)
        want = (f(z + h * d).loss - f(z - h * d).loss) / (2 * h)
        near((o.dlogits.double() * d.double()).sum(), want.double(), 1.3e-3 * c + 2e-5 * (1 + o.loss.abs().item()))


# ------------------------------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    z, y = torch.zeros(2, 3, 8, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev)
    A, f = torch.zeros(2, 3, device=dev), torch.zeros(2, 3, device=dev)
    st = torch.zeros(2, 2, 3, device=dev)
    ids, top = torch.zeros(2, 3, 4, dtype=torch.int64, device=dev), torch.zeros(2, 3, 4, device=dev)
    P, Q, D, W = L.policy_loss_fwd_bwd, L.preference_loss_fwd_bwd, L.distill_loss_fwd_bwd, L.linear_logprobs
    x, w, yy = torch.zeros(6, 16, dtype=BF, device=dev), torch.zeros(8, 16, dtype=BF, device=dev), torch.zeros(6, dtype=torch.int64, device=dev)
    bad = [
        lambda: L.logprobs_fwd(z.half(), y), lambda: L.logprobs_fwd(z.double(), y), lambda: L.logprobs_fwd(z[0, 0], y[0, 0]), lambda: L.logprobs_fwd(z, y[:1]),
        lambda: L.logprobs_fwd(z, y.float()), lambda: L.logprobs_fwd(z[..., ::2], y), lambda: L.logprobs_fwd(z[..., :0], y),
        lambda: L.logprobs_fwd(z[None], y[None]), lambda: L.logprobs_bwd(f.double(), z, y, st), lambda: L.logprobs_bwd(f, z, y, f),
        lambda: L.logprobs_bwd(f, z, y, st, out=torch.zeros(2, 3, 8, dtype=BF, device=dev)), lambda: L.logprobs_bwd(f, z, y, st, out=z[:, :1].expand(2, 3, 8)),
        lambda: L.logprobs_bwd(f[:, :2], z[:, :2], y[:, :2], st[..., :2], out=z[:, 1:]), lambda: L.logprobs_bwd(f, z, y, st, out=torch.zeros(2, 3, 16, device=dev)[..., ::2]),
        lambda: P(z, y, A[0]), lambda: P(z, y, A[:, :2]), lambda: P(z, y, A.double()), lambda: P(z, y, A, f[:1]), lambda: P(z, y, A, None, f[:1]),
        lambda: P(z, y, A, kl="k2"), lambda: P(z, y, A, mean="rows"), lambda: P(z, y, A, clip=-0.1), lambda: P(z, y, A, kl_coef=0.1),
        lambda: P(z, y, A, mean="sum", n_valid=torch.ones(1, device=dev)), lambda: P(z, y, A, n_valid=torch.ones(2, device=dev)), lambda: P(z, y, A, want_grad=False, out=z),
        lambda: Q(z[0], y[0]), lambda: Q(z[:1], y[:1]), lambda: Q(z, y, f[0]), lambda: Q(z, y, beta=0.0), lambda: Q(z, y, kind="dpo"),
        lambda: Q(z, y, label_smoothing=0.5), lambda: Q(z, y, kind="hinge", label_smoothing=0.1),
        lambda: D(z, ids[0], top[0]), lambda: D(z, ids[..., :0], top[..., :0]), lambda: D(z, ids, top[..., :2]), lambda: D(z, ids.float(), top), lambda: D(z, ids, top.double()),
        lambda: D(z, ids, top, temperature=0.0), lambda: D(z, ids, top, temperature=math.inf), lambda: D(z, ids.repeat(1, 1, 300), top.repeat(1, 1, 300)),
        lambda: W(x, w[:, :8], yy), lambda: W(x, w.float(), yy), lambda: W(x, w, yy[:2]), lambda: W(x.requires_grad_(True), w, yy), lambda: W(x.detach(), w[:0], yy),
    ]
    if dev == "cuda":
        bad += [lambda: L.logprobs_fwd(z, y.cpu()), lambda: P(z, y, A.cpu()), lambda: D(z, ids, top.cpu()), lambda: W(x.detach(), w.cpu(), yy),
                lambda: W(x.detach().float(), w.float(), yy), lambda: W(x.detach()[:, :9], w[:, :9], yy)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was taken")


# ------------------------------------------------------------------------------------------------- GPU: streams, graphs, far rows
@pytest.mark.gpu
def test_streams_and_graphs():
    """Two captured graphs replayed on two streams at once, beside eager calls, give what one call alone gives."""
    z, y = make("cuda", (4, 50), 32000, BF, 3)
    A, old = torch.randn(4, 50, device="cuda"), torch.randn(4, 50, device="cuda") - 8
    ids, top = torch.randint(0, 32000, (4, 50, 20), device="cuda"), torch.randn(4, 50, 20, device="cuda")
    x, w = torch.randn(200, 256, device="cuda").to(BF), (torch.randn(32000, 256, device="cuda") / 16).to(BF)

    def everything():
        p = L.policy_loss_fwd_bwd(z, y, A, old, old, kl_coef=0.1)
        q = L.preference_loss_fwd_bwd(z, y)
        d = L.distill_loss_fwd_bwd(z, ids, top)
        s = L.linear_logprobs(x, w, y.view(-1))
        return [p.loss, p.kl, p.clipped, p.logp, p.dlogits, q.loss, q.margins, q.logp, q.dlogits, d.loss, d.kl, d.dlogits, *s]
    want = [t.clone() for t in everything()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for s in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            everything()
            s.synchronize()
            with torch.cuda.graph(graph, stream=s):
                out = everything()
        graphs.append((graph, out))
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = everything()
    torch.cuda.synchronize()
    for got in (eager, graphs[0][1], graphs[1][1]):
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    _lib.check_status()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows behind 2^31 values of bfloat16 logits, in place."""
    V, T = 128256, 16800
    z = torch.empty(T, V, dtype=BF, device="cuda").normal_(generator=gen("cuda", 1))
    y = torch.full((T,), IGN, device="cuda")
    y[::700] = torch.arange(24, device="cuda") * 5000
    y[-1] = V - 1
    rows = (y != IGN).nonzero()[:, 0]
    keep, A = z[rows].clone(), torch.randn(T, device="cuda")
    o = L.policy_loss_fwd_bwd(z, y, A, clip=None, mean="sum", out=z)
    check_grad(z[rows], keep, y[rows], -A[rows].double(), BF)
    near(o.logp[rows], torch.log_softmax(keep.double(), -1).gather(1, y[rows, None])[:, 0], 1e-4)
    assert not z[1:700].any() and not z[-5:-1].any()


# ------------------------------------------------------------------------------------------------- calls that few make
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [50, 20001])
def test_reported_kl_and_infinite_margins(dev, V):
    """A target that the model has masked: its KL estimate is infinite, and has no part in a loss that only reports it; an answer with it is infinitely
    unlikely, which the sigmoid loss takes without a gradient that is not a number."""
    z, y = make(dev, (2, 3), V, F32, 1, ignored=0.0)
    z[0, 1, y[0, 1]] = -math.inf
    A, ref = torch.ones(2, 3, device=dev), torch.zeros(2, 3, device=dev)
    old = torch.full((2, 3), -3.0, device=dev)
    with_ref, without = L.policy_loss_fwd_bwd(z, y, A, old, ref), L.policy_loss_fwd_bwd(z, y, A, old)
    assert with_ref.kl == math.inf and with_ref.loss.isfinite() and torch.equal(with_ref.loss, without.loss) and torch.equal(with_ref.dlogits, without.dlogits)
    o = L.preference_loss_fwd_bwd(z, y)                       # the chosen answer is impossible
    assert o.margins[0] == -math.inf and o.loss == math.inf and o.dlogits.isfinite().all()
    o = L.preference_loss_fwd_bwd(z.flip(0), y.flip(0))       # the rejected one is
    assert o.margins[0] == math.inf and o.loss == 0 and not o.dlogits.any()


@pytest.mark.parametrize("dev", DEVICES)
def test_inputs_with_a_graph(dev):
    """Raw calls take no part in autograd: logits that want a gradient may be given, and may be written over."""
    z, y = make(dev, (2, 4), 40, F32, 2)
    A = torch.ones(2, 4, device=dev)
    leaf = z.clone().requires_grad_(True)
    want = [L.policy_loss_fwd_bwd(z, y, A), L.preference_loss_fwd_bwd(z, y), L.distill_loss_fwd_bwd(z, y[..., None].clamp(min=0), A[..., None])]
    got = [L.policy_loss_fwd_bwd(leaf, y, A), L.preference_loss_fwd_bwd(leaf, y), L.distill_loss_fwd_bwd(leaf, y[..., None].clamp(min=0), A[..., None])]
    for a, b in zip(got, want):
        assert not a.loss.requires_grad and torch.equal(a.loss, b.loss) and torch.equal(a.dlogits, b.dlogits)
    assert L.policy_loss_fwd_bwd(leaf, y, A, out=leaf).dlogits is leaf and torch.equal(leaf.detach(), want[0].dlogits)
    hidden = torch.randn(3, 5, 8, device=dev, requires_grad=True)
    logits = hidden @ torch.randn(8, 40, device=dev)
    o = L.policy_loss_fwd_bwd(logits, torch.zeros(3, 5, dtype=torch.int64, device=dev), torch.ones(3, 5, device=dev))
    logits.backward(o.dlogits)
    assert hidden.grad.isfinite().all() and hidden.grad.any()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,K", [(260, 200), (5001, 3), (40003, 50), (300000, 1000)])
def test_distill_into_rows_of_another_alignment(dev, dtype, V, K):
    """Gradient rows that start elsewhere in a vector than the logits'; many entries for short rows; long rows with many entries."""
    g = gen("cpu", V)
    z = (2 * torch.randn(3, V, generator=g)).to(dtype).to(dev)
    ids, top = torch.randint(0, V, (3, K), generator=g).to(dev), torch.randn(3, K, generator=g).to(dev)
    a = L.distill_loss_fwd_bwd(z, ids, top, temperature=1.5)
    out = torch.full((3 * (V + 1) + 3,), 9.0, dtype=dtype, device=dev)[3:].view(3, V + 1)[:, :V]
    b = L.distill_loss_fwd_bwd(z, ids, top, temperature=1.5, out=out)
    z64 = z.double().requires_grad_(True)
    q = torch.softmax(top.double() / 1.5, -1)
    kl = (q * (q.log() - torch.log_softmax(z64 / 1.5, -1).gather(-1, ids))).sum(-1)
    loss = 1.5 ** 2 * kl.mean()
    (want,) = torch.autograd.grad(loss, z64)
    back = torch.zeros_like(want).scatter_add_(-1, ids, q)
    tol = half(dtype) * want.abs() * (1 + REL) + REL * 0.5 * (torch.softmax(z64.detach() / 1.5, -1) + back) + TINY
    for o in (a, b):
        near(o.dlogits, want, tol)
        near(o.loss, loss.detach(), 2e-5 * (1 + loss.item()))
    assert bool((out.as_strided((3, 1), (V + 1, 1), out.storage_offset() + V) == 9).all())


@pytest.mark.gpu
def test_scoring_of_many_rows():
    """More rows than one launch takes, most of them not scored."""
    M, H, V = L.SCORE_ROWS + 300, 64, 500
    g = gen("cuda", 3)
    x, w = torch.randn(M, H, generator=g, device="cuda").to(BF), torch.randn(V, H, generator=g, device="cuda").to(BF)
    y = torch.randint(0, V, (M,), generator=g, device="cuda")
    y[torch.rand(M, generator=g, device="cuda") < 0.9] = IGN
    y[-1], y[0] = 7, IGN
    lp, lse = L.linear_logprobs(x, w, y)
    z = x.double() @ w.double().t()
    keep = y != IGN
    near(lp, torch.log_softmax(z, -1).gather(1, y.clamp(min=0)[:, None])[:, 0] * keep, 1e-4 * keep)
    near(lse, torch.logsumexp(z, -1) * keep, 1e-4 * keep)
    again = L.linear_logprobs(x, w, y)
    assert torch.equal(again[0], lp) and torch.equal(again[1], lse)
    for m in (1, 61, 100, 2000):                              # few rows, and the same twice
        a, b = L.linear_logprobs(x[:m], w, y[:m].clamp(min=0)), L.linear_logprobs(x[:m], w, y[:m].clamp(min=0))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("V,T", [(32000, 600), (50257, 400), (128256, 300), (3000, 900), (260, 3000)])
def test_repeats_bit_for_bit(V, T):
    """Rings, exchanges between blocks and sums in the same order: ten calls beside other work on another stream give the same bits."""
    z, y = make("cuda", (T,), V, BF, V)
    A, old = torch.randn(T, device="cuda"), torch.randn(T, device="cuda") - 9
    ids, top = torch.randint(0, V, (T, 12), device="cuda"), torch.randn(T, 12, device="cuda")
    side, noise = torch.cuda.Stream(), torch.empty(1 << 26, device="cuda")
    first = None
    for _ in range(10):
        with torch.cuda.stream(side):
            noise.add_(1)
        lp, st = L.logprobs_fwd(z, y)
        p, d = L.policy_loss_fwd_bwd(z, y, A, old, old, kl_coef=0.1), L.distill_loss_fwd_bwd(z, ids, top)
        got = [lp, st, p.loss, p.kl, p.clipped, p.logp, p.dlogits, d.loss, d.kl, d.dlogits]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    _lib.check_status()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,apart", [(40, False), (20001, False), (20001, True)], ids=["warp", "pipeline", "block"])
@pytest.mark.parametrize("kw", [dict(), dict(mean="sum"), dict(ref=True), dict(ref=True, kl_coef=0.1)], ids=["clip", "sum", "reported", "kl"])
def test_bad_rows_of_a_clipped_policy(dev, dtype, V, apart, kw):
    """On the policy's own tokens the ratio is 1 whatever their log-probability is, but a row that has none (a NaN, an infinity, nothing left by the mask, a target that is masked
    or outside the vocabulary) makes the loss NaN, as its gradient is; the other rows keep theirs."""
    kw = dict(kw)
    z, y = make("cpu", (3,), V, dtype, V, ignored=0.0)
    ref = torch.full((3,), -2.0, device=dev) if kw.pop("ref", False) else None
    A = torch.tensor([0.7, -0.4, 0.2], device=dev)

    def call(z, y):
        z, y = z.to(dev), y.to(dev)
        out = torch.empty(3 * V + 1, dtype=dtype, device=dev)[1:].view(3, V) if apart else None      # rows that start elsewhere in a vector
        return L.policy_loss_fwd_bwd(z, y, A, None, ref, out=out, **kw)
    good = call(z, y)
    assert good.loss.isfinite() and good.dlogits.isfinite().all()
    for kind in ("nan", "inf", "empty", "outside", "before", "masked"):
        b, t = z.clone(), y.clone()
        if kind in ("nan", "inf"):
            b[1, (t[1] + 1) % V] = math.nan if kind == "nan" else math.inf
        elif kind == "empty":
            b[1] = -math.inf
        elif kind == "masked":
            b[1, t[1]] = -math.inf
        else:
            t[1] = V if kind == "outside" else -3
        o = call(b, t)
        assert o.loss.isnan() and o.dlogits[1].isnan().all(), kind
        assert torch.equal(o.dlogits[[0, 2]], good.dlogits[[0, 2]]), kind


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M,H,V", [(1, 64, 300), (7, 72, 1), (9, 512, 4000), (61, 1024, 50257), (65, 256, 1001), (100, 512, 32000), (100, 2048, 4001), (128, 1024, 777), (129, 64, 260),
                                   (300, 256, 1001), (1500, 512, 8000)])
def test_scoring_of_nearly_certain_tokens(dev, M, H, V):
    """Targets whose probability is 0.5 to 1 - 1e-12.  With e the errors of the products (each H 2^-24 of the sum of its terms' sizes at most) lp is off by (1 - p) times two of them,
    by REL of 1 - p from the statistics, and by its own rounding: what a nearly certain token's is off by shrinks with it, down to what 64 bits hold next to 1 (2^-53 a sum, 2^-44 in all)."""
    g = gen("cpu", H + V)
    w = (torch.randn(V, H, generator=g) * 2 / math.sqrt(H)).to(BF)
    y = torch.randint(0, V, (M,), generator=g)
    x = (w[y].float() * (10 + 30 * torch.rand(M, 1, generator=g)) / 4).to(BF)
    y[torch.rand(M, generator=g) < 0.2] = IGN
    x, w, y = x.to(dev), w.to(dev), y.to(dev)
    keep = y != IGN
    z = x.double() @ w.double().t()
    zy = z.gather(1, y.clamp(min=0)[:, None])
    others = torch.logsumexp(z.scatter(1, y.clamp(min=0)[:, None], -math.inf), 1) - zy[:, 0]      # log((1 - p) / p)
    lp, q = -torch.nn.functional.softplus(others) * keep, torch.sigmoid(others)
    size = (x.double().abs() @ w.double().abs().t()).max(1).values
    tol = q * (2 * H * 2 ** -24 * size + REL) + 2 ** -23 * lp.abs() + 2 ** -44
    got, lse = L.linear_logprobs(x, w, y)
    near(got, lp, tol * keep, "logp")
    near(lse, torch.logsumexp(z, 1) * keep, (H * 2 ** -24 * size + REL / 2 + 2 ** -23 * z.abs().max(1).values) * keep, "lse")
    assert (got <= 0).all()


def exact_products(M, H, V, g, dev):
    """States and a head whose products are exact in 32 bits, in any order: multiples of 1/4 up to 1/2, so that sums are multiples of 1/16 below H / 4 < 2^20."""
    x, w = (torch.randint(-2, 3, (n, H), generator=g, device=g.device).mul(0.25).to(BF).to(dev) for n in (M, V))
    y = torch.randint(0, V, (M,), generator=g, device=g.device)
    return x, w, torch.where(torch.rand(M, generator=g, device=g.device) < 0.3, torch.full_like(y, IGN), y).to(dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M,H,V", [(1, 512, 4001), (61, 512, 50257), (64, 64, 33), (65, 256, 1001), (100, 512, 50257), (128, 1024, 777), (128, 64, 129), (100, 2048, 4001), (128, 2048, 513),
                                   (129, 256, 1001), (400, 512, 9000)])
def test_scoring_of_exact_products(dev, M, H, V):
    """What is left is the statistics' own error, a hundredth of one column's part in most of these: every column and row is in its place, in each form of the product."""
    x, w, y = exact_products(M, H, V, gen("cpu", M + V), dev)
    keep, lsm = y != IGN, torch.log_softmax(x.double() @ w.double().t(), -1)
    want = lsm.gather(1, y.clamp(min=0)[:, None])[:, 0] * keep
    lp, lse = L.linear_logprobs(x, w, y)
    near(lp, want, lp_tol(want) * keep)
    want = torch.logsumexp(x.double() @ w.double().t(), -1) * keep
    near(lse, want, lp_tol(want) * keep)


@pytest.mark.gpu
@pytest.mark.parametrize("last", [1, 100, 129])
def test_scoring_of_a_short_last_launch(last):
    """The rows behind a launch's most take another form of the product, in the workspace of the first."""
    M, H, V = L.SCORE_ROWS + last, 64, 700
    x, w, y = exact_products(M, H, V, gen("cuda", last), "cuda")
    y[-1] = 3
    keep, z = y != IGN, x.double() @ w.double().t()
    lp, lse = L.linear_logprobs(x, w, y)
    want = torch.log_softmax(z, -1).gather(1, y.clamp(min=0)[:, None])[:, 0] * keep
    near(lp, want, lp_tol(want) * keep)
    want = torch.logsumexp(z, -1) * keep
    near(lse, want, lp_tol(want) * keep)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [37, 16400])
def test_kl_of_the_policys_tokens_and_of_the_references(dev, V):
    """A uniform policy's tokens are every token once: over them log_ratio and k3 have the mean KL(policy || reference), k1 its negative.  The reference's tokens, when that is the
    uniform one: k1 has the mean KL(reference || policy).  With a coefficient the gradient is the derivative of that mean."""
    T = min(V, 400)                                               # a vocabulary whose first T tokens are all that is not masked
    q = torch.log_softmax(torch.randn(T, generator=gen("cpu", V), dtype=torch.float64), 0)
    z = torch.full((T, V), -math.inf)
    z[:, :T] = 0.0
    y, A, flat = torch.arange(T), torch.zeros(T), torch.full((T,), -math.log(T))
    z, y, A, other, flat = z.to(dev), y.to(dev), A.to(dev), q.float().to(dev), flat.to(dev)
    kl_p = (-math.log(T) - q).mean().item()                       # KL(uniform || other) = KL(other || policy) of the second call's roles
    got = {k: L.policy_loss_fwd_bwd(z, y, A, None, other, clip=None, kl=k, kl_coef=0.5) for k in ("k3", "log_ratio", "k1")}
    tol = REL * (1 + q.abs().max().item())
    for k, sign in (("k3", 1), ("log_ratio", 1), ("k1", -1)):
        assert abs(got[k].kl.item() - sign * kl_p) <= tol and abs(got[k].loss.item() - 0.5 * sign * kl_p) <= tol, k
    p = torch.softmax(z.double(), -1)
    hot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    for k, c in (("log_ratio", 0.5 / T), ("k1", -0.5 / T)):
        c = torch.full((T,), c, dtype=torch.float64, device=dev)
        check_grad(got[k].dlogits, z, y, c, F32)
    zq = z.clone()
    zq[:, :T] = other
    o = L.policy_loss_fwd_bwd(zq, y, A, None, flat, clip=None, kl="k1", kl_coef=0.5)
    assert abs(o.kl.item() - kl_p) <= tol


@pytest.mark.gpu
def test_launches_of_several_kernels_and_cluster_sizes_in_turn():
    """What is remembered of a launch belongs to its kernel and its size of cluster: calls that alternate between losses, types and vocabularies give what each gives alone."""
    calls = []
    for V, dtype in ((9001, BF), (50257, F32), (128256, BF), (140000, F32)):
        z, y = make("cuda", (40,), V, dtype, V)
        A, ids = torch.randn(40, generator=gen("cpu", V)).cuda(), torch.randint(0, V, (40, 300), generator=gen("cpu", V)).cuda()
        top = torch.randn(40, 300, generator=gen("cpu", V)).cuda()
        calls += [lambda z=z, y=y: L.logprobs_fwd(z, y), lambda z=z, y=y, A=A: L.policy_loss_fwd_bwd(z, y, A)[3:], lambda z=z, ids=ids, top=top: L.distill_loss_fwd_bwd(z, ids, top)[1:],
                  lambda z=z, y=y, A=A: L.policy_loss_fwd_bwd(z, y, A, want_grad=False)[:1]]
    alone = [[c() for _ in range(2)][1] for c in calls]
    for order in (range(len(calls)), reversed(range(len(calls))), list(range(0, len(calls), 3)) * 2):
        for i in order:
            assert all(torch.equal(a, b) for a, b in zip(calls[i](), alone[i])), i
    _lib.check_status()


@pytest.mark.filterwarnings("ignore")      # operations that torch maps over one by one
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [9, 300])
def test_transformations_of_token_logprobs(dev, V):
    """Second derivatives, forward mode, batched gradients and the transformations of torch.func, against the same of the formula in float64.  Every value is made of at most two sums of
    V terms in 32 bits and products of three numbers up to 8: V 2^-24 * 64 holds them."""
    g = gen("cpu", V)
    z, y = make("cpu", (2, 3), V, F32, V, ignored=0.0)
    y[0, 1], y[1, 2] = IGN, V                                     # an ignored row, and a target outside the vocabulary in the last one
    v, d = torch.randn(2, 3, V, generator=g), torch.randn(5, 2, 3, generator=g)
    z, y, v, d = z.to(dev), y.to(dev), v.to(dev), d.to(dev)
    ok = torch.ones(2, 3, dtype=torch.bool, device=dev)
    ok[1, 2] = False                                              # its results are NaN in all of them
    f = lambda t: L.token_logprobs(t, y)
    f64 = lambda t: torch.log_softmax(t, -1).gather(-1, y.clamp(0, V - 1)[..., None])[..., 0] * (y != IGN)
    z64, tol = z.double(), 64 * V * 2 ** -24

    def same(got, want, rows):
        at = (..., rows, slice(None)) if want.shape[-1] == V else (..., rows)
        near(got[at], want[at], tol)
    a, b = z.clone().requires_grad_(True), z64.clone().requires_grad_(True)
    (ga,), (gb,) = torch.autograd.grad(f(a), a, d[0], create_graph=True), torch.autograd.grad(f64(b), b, d[0].double(), create_graph=True)
    same(ga.detach(), gb.detach(), ok)
    (ha,), (hb,) = torch.autograd.grad((ga * v)[ok].sum(), a), torch.autograd.grad((gb * v)[ok].sum(), b)
    same(ha, hb, ok)
    w = torch.ones(2, 3, device=dev, requires_grad=True)          # and of the gradient that is handed in
    (gw,) = torch.autograd.grad(f(a), a, w, create_graph=True)
    (dw,) = torch.autograd.grad((gw * v)[ok].sum(), w)
    w64 = torch.ones(2, 3, device=dev, dtype=torch.float64, requires_grad=True)
    (dw64,) = torch.autograd.grad((torch.autograd.grad(f64(b), b, w64, create_graph=True)[0] * v)[ok].sum(), w64)
    same(dw, dw64, ok)
    many, many64 = torch.autograd.grad(f(a), a, d, is_grads_batched=True)[0], torch.autograd.grad(f64(b), b, d.double(), is_grads_batched=True)[0]
    same(many, many64, ok)
    along = torch.func.jvp(f64, (z64,), (v.double(),))[1]
    same(torch.func.jvp(f, (z,), (v,))[1], along, ok)
    with torch.autograd.forward_ad.dual_level():
        same(torch.autograd.forward_ad.unpack_dual(f(torch.autograd.forward_ad.make_dual(z, v))).tangent, along, ok)
    stack = torch.stack([z, z + v])
    same(torch.func.vmap(f)(stack), torch.stack([f64(t) for t in stack.double()]), ok)
    same(torch.func.vmap(torch.func.grad(lambda t: (f(t) * d[0])[ok].sum()))(stack),
         torch.stack([torch.func.grad(lambda t: (f64(t) * d[0])[ok].sum())(t) for t in stack.double()]), ok)
    rows = torch.func.vmap(L.token_logprobs)(stack.flatten(0, 1), torch.cat([y, y]))      # targets that are mapped over too
    same(rows.view(2, 2, 3), torch.stack([f64(t) for t in stack.double()]), ok)
    for got in (f(z), ga.detach()[..., 0], torch.func.vmap(f)(stack)[0]):
        assert got[~ok].isnan().all()
    with pytest.raises(ValueError):
        torch.func.vmap(L.token_logprobs)(stack.flatten(0, 1), torch.cat([y, y])[:, :2])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("call", ["logprobs", "policy", "preference", "distill"])
@pytest.mark.parametrize("other", [False, True], ids=["logits", "tensor"])
def test_a_graph_that_needs_what_is_written_over(dev, call, other):
    """A tensor that takes the gradient counts as changed: a graph that has saved it raises in its backward pass, whatever the device."""
    hidden = torch.randn(2, 3, 8, device=dev, requires_grad=True)
    logits = hidden @ torch.randn(8, 40, device=dev)
    buffer = hidden.new_zeros(2, 3, 40)
    saved = buffer if other else logits
    loss = (logits * saved).sum() if other else (saved * saved).sum()
    lp = L.token_logprobs(logits, torch.zeros(2, 3, dtype=torch.int64, device=dev))
    z, y = logits.detach(), torch.ones(2, 3, dtype=torch.int64, device=dev)
    ids, c, out = torch.zeros(2, 3, 2, dtype=torch.int64, device=dev), torch.ones(2, 3, device=dev), buffer if other else z
    before = saved._version
    {"logprobs": lambda: L.logprobs_bwd(c, z, y, L.logprobs_fwd(z, y)[1], out=out), "policy": lambda: L.policy_loss_fwd_bwd(z, y, c, out=out),
     "preference": lambda: L.preference_loss_fwd_bwd(z, y, out=out), "distill": lambda: L.distill_loss_fwd_bwd(z, ids, torch.zeros(2, 3, 2, device=dev), out=out)}[call]()
    assert saved._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    if other:
        lp.sum().backward()                                       # the logits are as they were
    else:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            lp.sum().backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_out_that_is_another_input(dev):
    """A gradient is not written over what its own call still reads: the teacher's logits, the tokens' numbers, the statistics."""
    V = 6
    buf = torch.randn(3, 2, V, generator=gen("cpu", 1)).to(dev)
    z, top = buf[:2], buf[1:]                                     # the teacher's rows are the student's, one further
    y, ids = torch.zeros(2, 2, dtype=torch.int64, device=dev), torch.arange(V, device=dev).expand(2, 2, V)
    c = torch.ones(2, 2, device=dev)
    _, stats = L.logprobs_fwd(z, y)
    space = torch.zeros(2 * 2 * V + 4, device=dev)
    out, tail = space[:2 * 2 * V].view(2, 2, V), space[2 * 2 * V - 2:][:4].view(2, 2)
    apart, whole = space[4:].view(2, 2, V), space[:4].view(2, 2)
    n = space[3:4]
    bad = [lambda: L.distill_loss_fwd_bwd(z, ids, top, out=z), lambda: L.distill_loss_fwd_bwd(z, ids, top, n_valid=n, out=out),
           lambda: L.policy_loss_fwd_bwd(z, y, tail, out=out), lambda: L.policy_loss_fwd_bwd(z, y, c, tail, out=out), lambda: L.policy_loss_fwd_bwd(z, y, c, None, tail, out=out),
           lambda: L.policy_loss_fwd_bwd(z, y, c, n_valid=n, out=out), lambda: L.preference_loss_fwd_bwd(z, y, tail[0], out=out),
           lambda: L.logprobs_bwd(tail, z, y, stats, out=out), lambda: L.logprobs_bwd(c, z, y, space[20:].view(2, 2, 2), out=out),
           lambda: L.logprobs_bwd(c, z, space.view(torch.int64)[:4].view(2, 2), stats, out=out)]
    before = (buf.clone(), space.clone())
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was taken")
    assert torch.equal(buf, before[0]) and torch.equal(space, before[1])
    own = L.distill_loss_fwd_bwd(z, ids, z)                       # a teacher that is the student
    copy = z.clone()
    assert torch.equal(L.distill_loss_fwd_bwd(copy, ids, copy, out=copy).dlogits, own.dlogits) and own.loss.abs() < 1e-6
    want = L.policy_loss_fwd_bwd(z, y, c).dlogits                 # next to each other is apart
    whole.fill_(1.0)
    assert torch.equal(L.policy_loss_fwd_bwd(z, y, whole, out=apart).dlogits, want) and torch.equal(whole, c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M,H,V", [(200, 64, 1), (70, 64, 2), (3, 64, 300001), (140, 8, 300001)])
def test_scoring_of_one_column_and_of_many(dev, M, H, V):
    """A vocabulary of one token, whose log-probability is 0 and whose row has no other columns, and one that no cluster's shared memory holds."""
    x, w, y = exact_products(M, H, V, gen("cpu", M), dev)
    y[0] = V - 1
    keep, z = y != IGN, x.double() @ w.double().t()
    lp, lse = L.linear_logprobs(x, w, y)
    want = torch.log_softmax(z, -1).gather(1, y.clamp(min=0)[:, None])[:, 0] * keep
    near(lp, want, lp_tol(want) * keep)
    want = torch.logsumexp(z, -1) * keep
    near(lse, want, lp_tol(want) * keep)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M", [3, 90, 200])
def test_scoring_of_infinite_logits(dev, M):
    """Rows: 0 a target whose logit is +inf, 1 another column at +inf, 2 a target at -inf, 3 ordinary, 4 all but the target at -inf."""
    H, V = 8, 40
    x, w = torch.zeros(max(M, 5), H), torch.zeros(V, H)
    w[:, 0] = torch.linspace(-1, 1, V)
    x[:, 0] = 2.0
    # a logit is infinite where a state of 3e38 meets a weight of 3e38, with the sign of the weight; the other states are 0 there
    big = 3e38
    x[0, 1] = x[1, 2] = x[2, 3] = x[4, 4] = big
    y = torch.full((max(M, 5),), 7)
    w[7, 1], w[9, 2], w[7, 3] = big, big, -big
    w[:, 4], w[7, 4] = -big, 0.0
    x, w, y = x.to(BF).to(dev)[:M], w.to(BF).to(dev), y.to(dev)[:M]
    lp, lse = L.linear_logprobs(x, w, y)
    z = x[:, :1].double() @ w[:, :1].double().t()
    lsm, other = torch.log_softmax(z, -1)[:, 7], torch.logsumexp(torch.cat([z[:, :7], z[:, 8:]], 1), 1)
    tol = REL + 2 ** -22
    want = [(math.nan, math.nan), (math.nan, math.nan), (-math.inf, other[2].item()), None, (0.0, None)]
    for r in range(M):
        l, s = want[r] if r < 5 and want[r] else (lsm[r].item(), torch.logsumexp(z[r], 0).item())
        s = z[r, 7].item() if s is None else s
        near(lp[r].cpu(), torch.tensor(l), tol, ("logp", r))
        near(lse[r].cpu(), torch.tensor(s), tol, ("lse", r))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 100])
def test_scoring_of_few_rows_in_graphs(M):
    """Two graphs captured on two streams, replayed at once beside eager calls on a third, each with inputs of its own that change between replays."""
    H, V = 512, 20000
    x, w, y = exact_products(3 * M, H, V, gen("cuda", M), "cuda")
    want = L.linear_logprobs(x, w, y)
    want64 = torch.log_softmax(x.double() @ w.double().t(), -1).gather(1, y.clamp(min=0)[:, None])[:, 0] * (y != IGN)
    near(want[0], want64, lp_tol(want64))
    streams, graphs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams[:2]:
        xs, ys = torch.zeros_like(x[:M]), torch.zeros_like(y[:M])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            L.linear_logprobs(xs, w, ys)
            s.synchronize()
            with torch.cuda.graph(graph, stream=s):
                out = L.linear_logprobs(xs, w, ys)
        graphs.append((graph, xs, ys, out))
    torch.cuda.synchronize()
    for turn in range(4):
        got = []
        for i, (s, (graph, xs, ys, out)) in enumerate(zip(streams, graphs)):
            part = slice((turn + i) % 3 * M, (turn + i) % 3 * M + M)
            with torch.cuda.stream(s):
                xs.copy_(x[part])
                ys.copy_(y[part])
                graph.replay()
                got.append((part, [t.clone() for t in out]))
        with torch.cuda.stream(streams[2]):
            part = slice((turn + 2) % 3 * M, (turn + 2) % 3 * M + M)
            got.append((part, L.linear_logprobs(x[part], w, y[part])))
        torch.cuda.synchronize()
        for part, (lp, lse) in got:
            near(lp, want64[part], lp_tol(want64[part]))
            near(lse, want[1][part], 2 * lp_tol(want[1][part].double()))
    _lib.check_status()
