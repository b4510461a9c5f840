"""Trainers on the losses of ``ops/losses.py``: what one step does to the weights' gradients against plain autograd of the same formulas, the
operators one after the other as a training run uses them, and scoring without logits.

The gradients of a whole model are compared in fp32 on the CPU (two orders of the same 32-bit sums: 1e-5 of the largest entry), and on the GPU, where model and gradient are
bfloat16, by the angle between them: every logit gradient is rounded to 2^-9 of itself in both, at different places, as are the products behind it."""
import threading

import pytest
import torch

from transformers_fusion_b200.engines import dense as ED
from transformers_fusion_b200.models.config import TransformerConfig
from transformers_fusion_b200.models.dense import DenseModel
from transformers_fusion_b200.models.moe import MoEAllConfig, create_moe_variant
from transformers_fusion_b200.ops import functional as F
from transformers_fusion_b200.ops import losses as L
from transformers_fusion_b200.trainer import rl

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def model(dev, seed=0, V=96):
    cfg = TransformerConfig(vocab_size=V, hidden_size=128, num_layers=2, num_heads=2, ffn_hidden_size=192, max_seq_len=64, init_std=0.1)
    return DenseModel(cfg, device=dev, dtype=torch.float32 if dev == "cpu" else torch.bfloat16, seed=seed)


def stepped_gradients(trainer, step):
    """The flat gradient that a train_step hands to its optimizer, and what it returned."""
    seen = {}

    def take():
        seen["g"] = trainer.flat.grads.clone()
        trainer.flat.grads.zero_()
    trainer.opt.step = take
    out = step()
    return seen["g"], out


def plain_gradients(m, f):
    m.flat.grads.zero_()
    loss = f()
    loss.backward()
    for p in m.flat.params_list:
        if p.grad is not None:
            p.main_grad.add_(p.grad.float())
            p.grad = None
    g = m.flat.grads.clone()
    m.flat.grads.zero_()
    return g, float(loss.detach())


def same(g, want, dev):
    if dev == "cpu":
        assert (g - want).abs().max() <= 1e-5 * want.abs().max()
    else:
        assert torch.nn.functional.cosine_similarity(g.double(), want.double(), dim=0) > 0.999
        assert abs(g.norm() / want.norm() - 1) < 0.02


def batch(dev, n=4, S=17, V=96, seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (n, S), generator=g)
    mask = torch.zeros(n, S)
    for i in range(n):
        mask[i, 3 + i:S - i] = 1
    return ids.to(dev), mask.to(dev), g


def lp64(m, ids):
    lp = torch.log_softmax(m(ids).float()[:, :-1], -1)
    return lp.gather(-1, ids[:, 1:, None])[..., 0]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("clip,kl", [(0.0, 0.0), (0.2, 0.0), (0.0, 0.1), (0.2, 0.1)])
def test_grpo_step(dev, clip, kl):
    m = model(dev)
    t = rl.GRPOTrainer(m, group_size=4, beta=0.04, clip_eps=clip, kl_coef=kl)
    if kl:
        t.ref_model = model(dev, seed=7).eval()
    ids, mask, g = batch(dev)
    rewards = torch.tensor([1.0, 0.2, -0.5, 0.7])
    got, loss = stepped_gradients(t, lambda: t.train_step(ids, mask, rewards))
    adv = t.advantages(rewards).to(dev)[:, None]

    def plain():
        lp, k = lp64(m, ids), mask[:, 1:]
        n = k.sum(-1).clamp(min=1)
        per = -torch.exp(lp - lp.detach()) * adv if clip else -adv * lp
        out = ((per * k).sum(-1) / n).mean()
        if kl:
            with torch.no_grad():
                r = lp64(t.ref_model, ids)
            out = out + kl * (((torch.exp(r - lp) - (r - lp) - 1) * k).sum(-1) / n).mean()
        return out
    want, wloss = plain_gradients(m, plain)
    same(got, want * (1 - 0.01 * 0.04), dev)
    assert loss == pytest.approx(wloss, rel=1e-4, abs=1e-4)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("given", [False, True])
def test_ppo_step(dev, given):
    m = model(dev)
    t = rl.PPOTrainer(m)
    ids, mask, g = batch(dev)
    old = None
    if given:
        with torch.no_grad():
            old = lp64(m, ids) + 0.1 * torch.randn(4, 16, generator=g).to(dev)
    seen = []
    t.set_log_callback(lambda *a: seen.append(a))
    real = t.values
    coef = t.kl_coef
    v = real(ids).detach()
    got, (loss, vloss, kl) = stepped_gradients(t, lambda: t.train_step(ids, mask, torch.tensor([1.0, 0.0, -1.0, 0.5]), old))
    k = mask[:, 1:]
    advs = []
    for b, r1 in enumerate([1.0, 0.0, -1.0, 0.5]):
        r = torch.zeros(16)
        r[int(k[b].nonzero().max())] = r1
        advs.append(rl.gae(r, torch.cat([v[b, :16].cpu(), torch.zeros(1)]), 0.99, 0.95)[0])
    adv = torch.stack(advs).to(dev)
    adv = (adv - (adv * k).sum() / k.sum()) / (adv[k > 0].std() + 1e-8)

    def plain():
        lp = lp64(m, ids)
        o = lp.detach() if old is None else old
        r = torch.exp(lp - o)
        pol = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv)
        return (pol * k).sum() / k.sum() + coef * ((o - lp) * k).sum() / k.sum()
    want, wloss = plain_gradients(m, plain)
    same(got, want, dev)
    assert loss == pytest.approx(wloss, rel=1e-3, abs=1e-3) and seen[0][0] == pytest.approx(loss)


@pytest.mark.parametrize("dev", DEVICES)
def test_dpo_step_of_answers_of_two_lengths(dev):
    m, ref = model(dev), model(dev, seed=3)
    t = rl.DPOTrainer(m, ref, beta=0.3)
    c, cm, _ = batch(dev, S=17)
    r, rm, _ = batch(dev, S=12, seed=5)
    got, (loss, acc) = stepped_gradients(t, lambda: t.train_step(c, r, cm, rm))

    def plain():
        f = lambda q, i, k: (lp64(q, i) * k[:, 1:]).sum(-1)
        with torch.no_grad():
            rc, rr = f(ref, c, cm), f(ref, r, rm)
        x = 0.3 * ((f(m, c, cm) - rc) - (f(m, r, rm) - rr))
        return -torch.nn.functional.logsigmoid(x).mean()
    want, wloss = plain_gradients(m, plain)
    same(got, want, dev)
    assert loss == pytest.approx(wloss, rel=1e-4 if dev == "cpu" else 2e-2)
    again = rl.DPOTrainer(model(dev, seed=9), beta=0.3)               # the reference is a copy: every margin is 0 before the first step
    assert again.train_step(c, r, cm, rm)[0] == pytest.approx(0.6931472, rel=1e-6)


@pytest.mark.parametrize("dev", DEVICES)
def test_distill_step(dev):
    m, teacher = model(dev), model(dev, seed=11)
    t = rl.DistillTrainer(m, temperature=2.0)
    ids, mask, _ = batch(dev)
    top = t.teacher_top(teacher, ids, k=10)
    assert top[0].dtype == torch.int32 and top[0].shape == (4, 17, 10)
    got, loss = stepped_gradients(t, lambda: t.train_step(ids, mask, *top))

    def plain():
        keep = torch.nn.functional.pad(mask[:, 1:], (0, 1)) > 0
        lq = torch.log_softmax(top[1] / 2, -1)
        lp = torch.log_softmax(m(ids).float() / 2, -1).gather(-1, top[0].long())
        kl = (lq.exp() * (lq - lp)).sum(-1)
        return 4 * kl[keep].mean()
    want, wloss = plain_gradients(m, plain)
    same(got, want, dev)
    assert loss == pytest.approx(wloss, rel=1e-4) and t.last_loss() == loss


class Squashed(torch.nn.Module):
    """A model whose last operation keeps what it returned: its logits must not be written over."""

    def __init__(self, inner):
        super().__init__()
        self.inner, self.cfg, self.flat = inner, inner.cfg, inner.flatten()

    tok_embeddings = property(lambda self: self.inner.tok_embeddings)

    def flatten(self):
        return self.flat

    def forward(self, ids):
        return 5 * torch.tanh(self.inner(ids).float() / 5)


@pytest.mark.parametrize("dev", DEVICES)
def test_logits_that_the_backward_pass_reads_stay(dev):
    m = Squashed(model(dev))
    t = rl.GRPOTrainer(m, group_size=4)
    ids, mask, _ = batch(dev)
    rewards = torch.tensor([1.0, 0.2, -0.5, 0.7])
    got, _ = stepped_gradients(t, lambda: t.train_step(ids, mask, rewards))
    adv = t.advantages(rewards).to(dev)[:, None]
    want, _ = plain_gradients(m, lambda: (-(adv * lp64(m, ids)) * mask[:, 1:]).sum(-1).div(mask[:, 1:].sum(-1)).mean())
    same(got, want * (1 - 0.01 * 0.04), dev)


@pytest.mark.gpu
def test_first_work_of_a_thread():
    """A product is the first GPU work of a new thread, as of autograd's when the logits' gradient is handed to it."""
    x = torch.randn(192, 256, device="cuda").bfloat16()
    w = torch.randn(320, 256, device="cuda").bfloat16()
    out, errors = torch.zeros(192, 320, device="cuda", dtype=torch.bfloat16), []
    torch.cuda.synchronize()

    def work():
        try:
            F.gemm(x, w, out=out)
        except Exception as e:      # the thread's own
            errors.append(e)
    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert not errors, errors
    torch.cuda.synchronize()
    want = x.double() @ w.double().t()
    assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -20 * (x.double().abs() @ w.double().abs().t())).all()


class Capped(DenseModel):
    """A model of the framework's class with a forward pass of its own, whose backward reads the logits that it returned."""

    def forward(self, ids):
        return torch.tanh(super().forward(ids))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["forward", "hook"])
def test_forward_passes_of_other_kinds_keep_their_logits(dev, kind):
    cfg = model("cpu").cfg
    m = (Capped if kind == "forward" else DenseModel)(cfg, device=dev, dtype=torch.float32 if dev == "cpu" else torch.bfloat16, seed=0)
    seen = []
    if kind == "hook":
        m.register_forward_hook(lambda mod, args, out: seen.append((out.detach(), out.detach().clone())))
    t = rl.GRPOTrainer(m, group_size=4, beta=0.0, clip_eps=0.0)
    ids, mask, g = batch(dev)
    rewards = torch.tensor([1.0, 0.2, -0.5, 0.7])
    got, loss = stepped_gradients(t, lambda: t.train_step(ids, mask, rewards))
    adv, w = t.advantages(rewards).to(dev)[:, None], mask[:, 1:]
    want, wloss = plain_gradients(m, lambda: -(((adv * lp64(m, ids)) * w).sum(-1) / w.sum(-1).clamp(min=1)).mean())
    same(got, want, dev)
    assert all(torch.equal(a, b) for a, b in seen)
    # and are scored as they are (by a pass without a graph, which rounds at other places)
    with torch.no_grad():
        lp = torch.log_softmax(m(ids[:1, :9]).float(), -1)[0, 4:8].gather(-1, ids[0, 5:9, None]).mean()
    assert abs(ED.EvalHarness(m)._seq_logp(ids[0, :5].tolist(), ids[0, 5:9].tolist()) - lp.item()) <= 1e-5 * abs(lp.item())


@pytest.mark.parametrize("dev", DEVICES)
def test_score_tokens(dev):
    m = model(dev)
    ids, mask, _ = batch(dev)
    targets = rl.next_tokens(ids, mask)
    lp = m.score_tokens(ids, targets)
    z = m.hidden_states(ids).view(4, 17, -1).double() @ m.lm_head.double().t()
    want = torch.log_softmax(z, -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0] * (targets != -100)
    assert lp.shape == ids.shape and not lp.requires_grad and (lp - want).abs().max() < 1e-4
    assert (rl.score_tokens(m, ids, targets) - want).abs().max() < (1e-4 if dev == "cpu" else 0.1)      # from logits, which are bfloat16 on the GPU
    h = ED.EvalHarness(m)
    a, b = ids[0].tolist()[:6], ids[0].tolist()[6:11]
    assert h._seq_logp(a, b) == pytest.approx(float(m.score_tokens(ids[:1, :11], rl.next_tokens(ids[:1, :11]))[0, 5:10].mean()), rel=1e-5)


@pytest.mark.parametrize("dev", DEVICES)
def test_engine_losses(dev):
    g = torch.Generator().manual_seed(0)
    z = torch.randn(4, 6, 30, generator=g).to(dev)
    y = torch.randint(0, 30, (4, 6), generator=g).to(dev)
    y[:, 0] = -100
    ids, top = torch.rand(4, 6, 30, generator=g).argsort(-1)[..., :5].to(dev), torch.randn(4, 6, 5, generator=g).to(dev)
    ids[0, 0] = -1
    adv = torch.randn(24, generator=g).to(dev)
    for f, plain in (
            (lambda t: ED.policy_grad_loss(t, y, adv), lambda t: -(adv.view(4, 6) * lp_of(t, y) * (y != -100)).sum() / (y != -100).sum()),
            (lambda t: ED.distill_top_loss(t, ids, top, 1.5), lambda t: top_loss(t, ids, top, 1.5)),
            (lambda t: ED.preference_loss(t, y, beta=0.5), lambda t: -torch.nn.functional.logsigmoid(
                0.5 * ((lp_of(t, y) * (y != -100)).sum(1)[:2] - (lp_of(t, y) * (y != -100)).sum(1)[2:])).mean())):
        loss, d = f(z)
        t = z.double().requires_grad_(True)
        want = plain(t)
        want.backward()
        assert float(getattr(loss, "loss", loss)) == pytest.approx(float(want.detach()), rel=1e-5)
        assert d.shape == z.shape and (d - t.grad).abs().max() < 1e-6


def lp_of(t, y):
    return torch.log_softmax(t, -1).gather(-1, y.clamp(min=0)[..., None])[..., 0]


def top_loss(t, ids, top, tau):
    keep = ids[..., 0] >= 0
    lq = torch.log_softmax(top.double() / tau, -1)
    lp = torch.log_softmax(t / tau, -1).gather(-1, ids.clamp(min=0))
    return tau ** 2 * (lq.exp() * (lq - lp)).sum(-1)[keep].mean()


@pytest.mark.parametrize("dev", DEVICES)
def test_a_run_of_them(dev):
    """One round of post-training as it is put together: old log-probabilities by scoring, several policy steps on one rollout in micro-batches, a
    preference step, a distillation step - eagerly, and on the GPU with the losses of the policy steps in a captured graph; twice, with the same result from the same weights."""
    def run(graph):
        m, teacher = model(dev, seed=2), model(dev, seed=4)
        m.flatten()
        ids, mask, g = batch(dev, n=8)
        targets = rl.next_tokens(ids, mask)
        adv = torch.randn(8, generator=g).to(dev)
        old = rl.score_tokens(m, ids, targets)
        ref = teacher.score_tokens(ids, targets)
        count = (targets != -100).sum().float().reshape(1)
        z_in = torch.empty(4, 17, 96, dtype=m.tok_embeddings.dtype, device=dev)
        t_in, a_in, o_in, r_in = targets[:4].clone(), adv[:4].clone(), old[:4].clone(), ref[:4].clone()
        call = lambda: L.policy_loss_fwd_bwd(z_in, t_in, a_in, o_in, r_in, clip=(0.2, 0.3), kl_coef=0.05, n_valid=count)
        replay = None
        if graph:
            call()
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                res = call()
            replay = lambda: (gr.replay(), res)[1]
        losses = []
        for step in range(3):
            for half in (slice(0, 4), slice(4, 8)):
                logits = m(ids[half])
                for dst, src in ((z_in, logits.detach()), (t_in, targets[half]), (a_in, adv[half]), (o_in, old[half]), (r_in, ref[half])):
                    dst.copy_(src)
                o = replay() if replay else call()
                logits.backward(o.dlogits.clone())
                losses.append(o.loss.clone())
            with torch.no_grad():
                m.flat.params.sub_((0.05 * m.flat.grads).to(m.flat.params.dtype))
                m.flat.grads.zero_()
        d = rl.DPOTrainer(m, teacher)
        losses.append(torch.tensor(d.train_step(ids[:4], ids[4:], mask[:4], mask[4:])[0]))
        k = rl.DistillTrainer(m)
        losses.append(torch.tensor(k.train_step(ids, mask, *k.teacher_top(teacher, ids, 8))))
        return torch.stack([l.float().cpu() for l in losses]), m.flat.params.clone()
    first, second = run(False), run(dev == "cuda")
    assert first[0].isfinite().all() and torch.equal(first[0][:2], second[0][:2])
    if dev == "cpu":
        assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    else:                       # the embedding's gradient is added up in no fixed order: a weight may round to its neighbour (2^-8)
        assert ((first[0] - second[0]).abs() <= 2e-2 * first[0].abs() + 2e-2).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["dense", "other"])
def test_harness_without_a_context(dev, kind):
    """An empty context: the continuation's first token is scored by the last position, the others by the one before them."""
    m = model(dev)
    ids = batch(dev)[0][0, :6].tolist()
    with torch.no_grad():
        lp = torch.log_softmax(m(torch.tensor([ids], device=dev)).double(), -1)[0]
        if kind == "other":
            m = Squashed(m)
            lp = torch.log_softmax(m(torch.tensor([ids], device=dev)).double(), -1)[0]
    for ctx in range(4):
        at = [(ctx - 1 + i) % 6 for i in range(6 - ctx)]
        want = lp[at, ids[ctx:]].mean().item()
        # logits of the dense model are bfloat16 on the GPU and rounded nowhere in its scoring: 2^-9 of values below 8
        assert abs(ED.EvalHarness(m)._seq_logp(ids[:ctx], ids[ctx:]) - want) <= (2 * 8 * 2 ** -9 if dev == "cuda" else 1e-5 * abs(want)), ctx


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("scope", ["model", "global"])
def test_hooks_on_what_a_model_is_called_with(dev, scope):
    """A hook in front of the forward pass changes what is scored, and sees every call of a trainer."""
    m = model(dev)
    ids = batch(dev)[0][:1, :9]
    plain = ED.EvalHarness(m)._seq_logp(ids[0, :5].tolist(), ids[0, 5:].tolist())
    swapped = (ids + 1) % 96
    swapped[0, 5:] = ids[0, 5:]
    want = ED.EvalHarness(m)._seq_logp(swapped[0, :5].tolist(), ids[0, 5:].tolist())
    assert abs(plain - want) > 1e-2

    def hook(mod, args):
        return (torch.cat([(args[0][:, :5] + 1) % 96, args[0][:, 5:]], 1),) if mod is m else None
    handle = m.register_forward_pre_hook(hook) if scope == "model" else torch.nn.modules.module.register_module_forward_pre_hook(hook)
    try:
        got = ED.EvalHarness(m)._seq_logp(ids[0, :5].tolist(), ids[0, 5:].tolist())
    finally:
        handle.remove()
    assert abs(got - want) <= (2 * 8 * 2 ** -9 if dev == "cuda" else 1e-5 * abs(want))
    assert ED.EvalHarness(m)._seq_logp(ids[0, :5].tolist(), ids[0, 5:].tolist()) == plain


@pytest.mark.parametrize("dev", DEVICES)
def test_logits_of_other_layouts(dev):
    """Logits whose last dimension is not dense, of a type that the losses do not take, and of more rows and positions than there are tokens."""
    g = torch.Generator().manual_seed(2)
    z = torch.randn(4, 9, 30, generator=g).to(dev)
    ids = torch.randint(0, 30, (3, 7), generator=g).to(dev)
    f = rl.GRPOTrainer.compute_log_probs
    want = torch.log_softmax(z.double()[:3, :6], -1).gather(-1, ids[:, 1:, None])[..., 0]
    apart = z.transpose(1, 2).contiguous().transpose(1, 2)
    assert apart.stride(-1) != 1
    # 2^-24 of a sum of 30 terms on its way, and half a step of values below 16
    for t, tol in ((z, 4e-6), (apart, 4e-6), (apart[:3, :7], 4e-6), (z.double(), 4e-6), (apart.half(), 2 ** -11 * 16)):
        assert (f(t, ids) - want).abs().max() <= tol
    leaf = apart.clone(memory_format=torch.preserve_format).requires_grad_(True)
    f(leaf, ids).sum().backward()
    p = torch.softmax(z.double(), -1)
    grad = torch.zeros_like(p)
    grad[:3, :6] = torch.zeros_like(p[:3, :6]).scatter_(-1, ids[:, 1:, None], 1.0) - p[:3, :6]
    assert leaf.stride() == apart.stride() and (leaf.grad - grad).abs().max() <= 4e-6
    with pytest.raises(ValueError):
        f(z[:2], ids)

    class Fixed(torch.nn.Module):
        def forward(self, ids):
            return apart[:3, :7]
    assert (rl.token_logprobs(Fixed(), ids) - want).abs().max() <= 4e-6
    assert (rl.score_tokens(Fixed(), ids, rl.next_tokens(ids))[:, :-1] - want).abs().max() <= 4e-6


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_grad_loss_of_other_arguments(dev):
    """Logits whose last dimension is not dense, one advantage for all rows, advantages of other types, labels below 0 that are not the ignored one (they count as 0)."""
    g = torch.Generator().manual_seed(3)
    z = torch.randn(7, 10, generator=g).to(dev).t()
    y = torch.randint(0, 7, (10,), generator=g).to(dev)
    y[2], y[5] = -100, -1
    keep = y != -100
    for adv in (torch.randn(10, generator=g).to(dev), torch.randn(1, generator=g).to(dev), torch.tensor(2.0, device=dev), torch.arange(10, device=dev)):
        loss, d = ED.policy_grad_loss(z, y, adv)
        t = z.double().requires_grad_(True)
        want = -(adv.double() * torch.log_softmax(t, -1).gather(1, y.clamp(min=0)[:, None])[:, 0] * keep).sum() / keep.sum()
        want.backward()
        assert loss == pytest.approx(float(want.detach()), rel=1e-5, abs=1e-6) and (d - t.grad).abs().max() < 1e-5 * adv.abs().max().item() + 1e-6
    ids, top = torch.rand(10, 7, generator=g).argsort(-1)[:, :3].to(dev), torch.randn(10, 3, generator=g).to(dev)
    assert torch.equal(ED.distill_top_loss(z, ids, top)[1], ED.distill_top_loss(z.contiguous(), ids, top)[1])
    pairs, labels = torch.randn(2, 7, 5, generator=g).to(dev).transpose(1, 2), y[6:].clamp(min=0).repeat(2, 2)[:, :5]
    assert torch.equal(ED.preference_loss(pairs, labels)[1], ED.preference_loss(pairs.contiguous(), labels)[1])


def weighted(mask, seed=3):
    """Tokens that count by a weight: 0 where the mask is 0, else 0.25 to 2, one of them negative."""
    w = mask * (0.25 + 1.75 * torch.rand(mask.shape, generator=torch.Generator().manual_seed(seed))).to(mask.device)
    w[0, 5] = -0.5
    return w


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("clip,kl", [(0.0, 0.0), (0.2, 0.1)])
@pytest.mark.parametrize("kind", ["weights", "one_row"])
def test_grpo_mask_of_weights(dev, clip, kl, kind):
    m = model(dev)
    t = rl.GRPOTrainer(m, group_size=4, beta=0.04, clip_eps=clip, kl_coef=kl)
    if kl:
        t.ref_model = model(dev, seed=7).eval()
    ids, mask, _ = batch(dev)
    mask = weighted(mask) if kind == "weights" else mask[1:2]
    rewards = torch.tensor([1.0, 0.2, -0.5, 0.7])
    got, loss = stepped_gradients(t, lambda: t.train_step(ids, mask, rewards))
    adv = t.advantages(rewards).to(dev)[:, None]

    def plain():
        lp, k = lp64(m, ids), mask[:, 1:]
        n = k.sum(-1).clamp(min=1)
        per = -torch.exp(lp - lp.detach()) * adv if clip else -adv * lp
        out = ((per * k).sum(-1) / n).mean()
        if kl:
            with torch.no_grad():
                r = lp64(t.ref_model, ids)
            out = out + kl * (((torch.exp(r - lp) - (r - lp) - 1) * k).sum(-1) / n).mean()
        return out
    want, wloss = plain_gradients(m, plain)
    same(got, want * (1 - 0.01 * 0.04), dev)
    assert loss == pytest.approx(wloss, rel=1e-4, abs=1e-4) and t.last_loss() == loss


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("given", [False, True])
def test_ppo_mask_of_weights(dev, given):
    m = model(dev)
    t = rl.PPOTrainer(m)
    ids, mask, g = batch(dev)
    mask = weighted(mask).abs()
    k = mask[:, 1:]
    old = None
    if given:
        with torch.no_grad():
            old = (lp64(m, ids) + 0.1 * torch.randn(4, 16, generator=g).to(dev)).masked_fill(k == 0, float("nan"))
    coef, rewards = t.kl_coef, [1.0, 0.0, -1.0, 0.5]
    v = t.values(ids).detach()
    got, (loss, vloss, kl) = stepped_gradients(t, lambda: t.train_step(ids, mask, torch.tensor(rewards), old))
    advs = []
    for b, r1 in enumerate(rewards):
        r = torch.zeros(16)
        r[int(k[b].nonzero().max())] = r1
        advs.append(rl.gae(r, torch.cat([v[b, :16].cpu(), torch.zeros(1)]), 0.99, 0.95)[0])
    adv = torch.stack(advs).to(dev)
    adv = (adv - (adv * k).sum() / k.sum()) / (adv[k > 0].std() + 1e-8)
    seen = {}

    def plain():
        lp = lp64(m, ids)
        o = lp.detach() if old is None else old.nan_to_num(0.0)
        r = torch.exp(lp - o)
        pol = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv)
        seen["kl"] = float((((o - lp) * k).sum() / k.sum()).detach())
        return (pol * k).sum() / k.sum() + coef * ((o - lp) * k).sum() / k.sum()
    want, wloss = plain_gradients(m, plain)
    same(got, want, dev)
    assert loss == pytest.approx(wloss, rel=1e-3, abs=1e-3) and kl == pytest.approx(seen["kl"], abs=1e-3)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["weights", "one_row"])
def test_dpo_mask_of_weights(dev, kind):
    m, ref = model(dev), model(dev, seed=3)
    t = rl.DPOTrainer(m, ref, beta=0.3)
    seen = []
    t.set_log_callback(lambda *a: seen.append(a))
    (c, cm, _), (r, rm, _) = batch(dev, S=17), batch(dev, S=12, seed=5)
    cm, rm = (weighted(cm), weighted(rm, 4)) if kind == "weights" else (cm[1:2], rm)
    got, (loss, acc) = stepped_gradients(t, lambda: t.train_step(c, r, cm, rm))
    f = lambda q, i, k: (lp64(q, i) * k[:, 1:]).sum(-1)
    with torch.no_grad():
        rc, rr = f(ref, c, cm), f(ref, r, rm)
        gap = float((f(m, c, cm) - rc).mean())
        order = float((((f(m, c, cm) - rc) - (f(m, r, rm) - rr)) > 0).float().mean())

    def plain():
        return -torch.nn.functional.logsigmoid(0.3 * ((f(m, c, cm) - rc) - (f(m, r, rm) - rr))).mean()
    want, wloss = plain_gradients(m, plain)
    same(got, want, dev)
    assert loss == pytest.approx(wloss, rel=1e-4 if dev == "cpu" else 2e-2) and (acc == order or dev == "cuda")
    assert seen[0][0] == loss and seen[0][1] == pytest.approx(gap, abs=1e-4 if dev == "cpu" else 14 * 8 * 2 ** -9)      # a product of other rows may round a logit to its neighbour, in 14 tokens at most


@pytest.mark.parametrize("dev", DEVICES)
def test_ppo_on_its_own_tokens(dev):
    """Without older log-probabilities the ratio is 1 to the last bit: no token is outside of a clip of width 0, and the KL estimate is 0, which leaves its coefficient alone when
    that is the target."""
    m = model(dev)
    t = rl.PPOTrainer(m, clip=0.0, kl_target=0.0, kl_coef=0.1)
    ids, mask, _ = batch(dev)
    v, k = t.values(ids).detach(), mask[:, 1:]
    rewards = [1.0, 0.0, -1.0, 0.5]
    got, (loss, _, kl) = stepped_gradients(t, lambda: t.train_step(ids, mask, torch.tensor(rewards)))
    assert kl == 0.0 and t.kl_coef == 0.1 and t.last_kl() == 0.0
    advs = []
    for b, r1 in enumerate(rewards):
        r = torch.zeros(16)
        r[int(k[b].nonzero().max())] = r1
        advs.append(rl.gae(r, torch.cat([v[b, :16].cpu(), torch.zeros(1)]), 0.99, 0.95)[0])
    adv = torch.stack(advs).to(dev)
    adv = (adv - (adv * k).sum() / k.sum()) / (adv[k > 0].std() + 1e-8)

    def plain():
        lp = lp64(m, ids)
        return -(torch.exp(lp - lp.detach()) * adv * k).sum() / k.sum() + 0.1 * ((lp.detach() - lp) * k).sum() / k.sum()
    want, wloss = plain_gradients(m, plain)
    same(got, want, dev)
    assert loss == pytest.approx(wloss, rel=1e-4, abs=1e-5)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n,beta", [((1, 3), 0.3), ((4, 1), 0.3), ((4, 4), 0.0), ((4, 4), -0.2)])
def test_dpo_of_one_answer_against_several(dev, n, beta):
    """One answer on a side makes a pair with each of the other side's, and a beta that is not above 0 is taken as it is."""
    m, ref = model(dev), model(dev, seed=3)
    t = rl.DPOTrainer(m, ref, beta=beta)
    (c, cm, _), (r, rm, _) = batch(dev, n=n[0], S=17), batch(dev, n=n[1], S=12, seed=5)
    got, (loss, acc) = stepped_gradients(t, lambda: t.train_step(c, r, cm, rm))
    f = lambda q, i, k: (lp64(q, i) * k[:, 1:]).sum(-1)

    def plain():
        with torch.no_grad():
            rc, rr = f(ref, c, cm), f(ref, r, rm)
        return -torch.nn.functional.logsigmoid(beta * ((f(m, c, cm) - rc) - (f(m, r, rm) - rr))).mean()
    want, wloss = plain_gradients(m, plain)
    if beta:
        same(got, want, dev)
    else:
        assert not got.any() and not want.any()
    assert loss == pytest.approx(wloss, rel=1e-4 if dev == "cpu" else 2e-2)


def test_dpo_of_answers_that_do_not_pair():
    t = rl.DPOTrainer(model("cpu"))
    (c, cm, _), (r, rm, _) = batch("cpu", n=2), batch("cpu", n=4)
    before = t.flat.params.clone()
    with pytest.raises(ValueError):
        t.train_step(c, r, cm, rm)
    assert torch.equal(t.flat.params, before) and t.steps == 0


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("variant,policy", [("EXPERT_CHOICE", "none"), ("SPARSE_TOPK", "token_drop")])
def test_dpo_of_a_mixture_whose_tokens_compete(dev, variant, policy):
    """A chosen answer's logits depend neither on the rejected answer nor on padding to its length."""
    base = TransformerConfig(vocab_size=96, hidden_size=128, num_layers=2, num_heads=2, ffn_hidden_size=192, max_seq_len=64, init_std=0.1)
    mixture = lambda seed: create_moe_variant(variant, base, MoEAllConfig(num_experts=4, top_k=2, expert_hidden=64, capacity_factor=0.75, capacity_policy=policy), device=dev,
                                              dtype=torch.float32 if dev == "cpu" else torch.bfloat16, seed=seed)
    m, ref = mixture(0), mixture(3)
    t = rl.DPOTrainer(m, ref, beta=0.3)
    (c, cm, _), (r, rm, _) = batch(dev, S=17), batch(dev, S=12, seed=5)
    with torch.no_grad():
        both = m(torch.cat([c, torch.nn.functional.pad(r, (0, 5))]))[:4]
        assert (both - m(c)).abs().max() > 0.02                       # they do compete
    got, (loss, acc) = stepped_gradients(t, lambda: t.train_step(c, r, cm, rm))

    def plain():
        f = lambda q, i, k: (lp64(q, i) * k[:, 1:]).sum(-1)
        with torch.no_grad():
            rc, rr = f(ref, c, cm), f(ref, r, rm)
        return -torch.nn.functional.logsigmoid(0.3 * ((f(m, c, cm) - rc) - (f(m, r, rm) - rr))).mean()
    want, wloss = plain_gradients(m, plain)
    same(got, want, dev)
    assert loss == pytest.approx(wloss, rel=1e-4 if dev == "cpu" else 2e-2)
