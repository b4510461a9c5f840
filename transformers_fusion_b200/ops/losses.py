"""Losses of post-training on logits, and the scoring of given tokens.

* ``logprobs_fwd`` / ``logprobs_bwd``: log-probabilities of given tokens and the gradient of the logits; ``token_logprobs`` is both as one
  autograd function.
* ``policy_loss_fwd_bwd``: clipped policy loss with a KL term.
* ``preference_loss_fwd_bwd``: loss of paired answers on their log-ratios to a reference model.
* ``distill_loss_fwd_bwd``: KL divergence from a teacher's stored top logits.
* ``linear_logprobs``: log-probabilities of given tokens from hidden states and the head's weight, for passes that want no gradient.

As in ``ops/functional.py``: CUDA tensors go to the sm_100a kernels (``csrc/kernels/token_losses.cu``, ``linear_logprobs.cu``), CPU
tensors run the plain PyTorch statement of the same mathematics.

Logits are [T, V] or [B, S, V], bfloat16 or float32, of any strides with a dense last dimension (rows may start at any element).  Targets are
int64 or int32 of the logits' leading shape; rows whose target is ``ignore_index`` are not read, their statistics and gradients are 0.  A
target outside the vocabulary makes its row's results NaN.  ``out`` takes the gradient: another tensor of the logits' shape and type, or the
logits themselves, which are then overwritten; None makes a new one.  It shares no memory with the other inputs (but for teacher's
logits that are the student's, row for row).  Per-row results and losses are float32.

Reference counterparts: log-probabilities, ratio clipping and KL terms of the RL trainers (src/trainer/trainer_rl.cpp:557-1350)."""
from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import c_i, c_ll, c_p, check

MAX_TOP = 1024          # entries of a teacher's row
PIPE_CLUSTERS = 296     # most clusters of one launch, each with three sums of 8 bytes in the workspace
SCORE_ROWS = 1 << 15    # most rows of one launch of linear_logprobs, whose workspace holds their hidden states and 8 bytes a row per 128 of the vocabulary (512 MB of these)

_KL = {"k3": 0, "k1": 1, "log_ratio": 2}
_MEAN = {"tokens": 0, "sequences": 1, "sum": 2}
_KIND = {"sigmoid": 0, "hinge": 1, "squared": 2}

# Arguments of the C entry points travel as packed structures (natural alignment, as the compiler lays them out): a call of a small loss is a few
# microseconds of GPU time, and a ctypes structure of twenty fields would cost as much again.
_ROWS = struct.Struct("@PPqqqqiiiiP0P")                      # z, dz, zb, zs, db, ds, T, S, V, f32, status
_POLICY = struct.Struct("@PiqPPPiiiifffPPPPPP0P")            # targets, idx64, ignore, adv, old, ref, adv_seq, ratio, kl, mean, lo, hi, kl_coef, n_valid, logp, out, ws, denom, counter
_PREFERENCE = struct.Struct("@PiqPiiffPPPPPPPP0P")           # targets, idx64, ignore, ref, kind, average, beta, smooth, loss, margins, logp, lp64, stats, coef, terms, counter
_DISTILL = struct.Struct("@PPiiifPPPPPP0P")                  # ids, z, idx64, top_f32, K, tau, n_valid, kl, loss, ws, denom, counter
_SCORE = struct.Struct("@PPqqPiqiiiPPPPPPqPiPqP0P")          # x, w, ldx, ldw, targets, idx64, ignore, M, V, H, logp, lse, rows, row_of, col_of, xc, ldc, part, parts, z, ldz, zy

_lib.register("tfb_token_logprobs", [c_p, c_p, c_i, c_ll, c_p, c_p, c_p])
_lib.register("tfb_token_logprobs_bwd", [c_p, c_p, c_i, c_ll, c_p, c_p, c_p])
_lib.register("tfb_policy_loss", [c_p, c_p, c_p])
_lib.register("tfb_preference_loss", [c_p, c_p, c_p])
_lib.register("tfb_distill_loss", [c_p, c_p, c_p])
_lib.register("tfb_linear_logprobs", [c_p, c_p, c_p])


# ---------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------
def _check_logits(logits):
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits: [T, V] or [B, S, V], got {tuple(logits.shape)}")
    if logits.dtype is not torch.bfloat16 and logits.dtype is not torch.float32:
        raise ValueError(f"logits: bfloat16 or float32, got {logits.dtype}")
    if logits.shape[-1] == 0:
        raise ValueError("logits: an empty vocabulary")
    if logits.stride(-1) != 1 and logits.shape[-1] != 1:
        raise ValueError("logits: the last dimension has to be dense")


def _check_index(idx, shape, name, device):
    if idx.dtype is not torch.int64 and idx.dtype is not torch.int32:
        raise ValueError(f"{name}: int64 or int32, got {idx.dtype}")
    if idx.shape != shape or idx.device != device:
        raise ValueError(f"{name}: {tuple(shape)} on {device} wanted, got {tuple(idx.shape)} on {idx.device}")
    return idx if idx.is_contiguous() else idx.contiguous()


def _check_f32(t, shape, name, device):
    """A float32 tensor of this shape, dense; None stays None."""
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape != shape or t.device != device:
        raise ValueError(f"{name}: float32 {tuple(shape)} on {device} wanted, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _check_n_valid(n_valid, device):
    if n_valid is None:
        return None
    if n_valid.numel() != 1:
        raise ValueError("n_valid: one value")
    return _check_f32(n_valid.reshape(1), torch.Size((1,)), "n_valid", device)


def _one_of(value, choices, name):
    if value not in choices:
        raise ValueError(f"{name}: one of {sorted(choices)}, got {value!r}")
    return choices[value]


def _gradient(logits, out, want_grad, *inputs):
    """Where the gradient goes: None, ``out``, or a new tensor.  ``inputs``: what else the call reads (None: not given)."""
    if not want_grad:
        if out is not None:
            raise ValueError("out: without want_grad there is no gradient")
        return None
    if out is None:
        return torch.empty_like(logits)          # rows of the same alignment as those of the logits where they are dense
    if out.device == logits.device and out.numel():
        a, b = _span(out)
        for t in inputs:
            if t is not None and t.numel():
                first, last = _span(t)
                # (a teacher's logits that are the student's, entry by entry, are read before their row is written)
                if first < b and a < last and not (first == a and t.shape == out.shape and t.stride() == out.stride()):
                    raise ValueError("out: overlaps an input that is not the logits")
    if out is logits and logits.is_contiguous():
        return out
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out: the logits' shape, type and device")
    if out.stride(-1) != 1 and out.shape[-1] != 1:
        raise ValueError("out: the last dimension has to be dense")
    reach = out.shape[-1]
    for stride, n in sorted((out.stride(i), out.shape[i]) for i in range(out.dim() - 1) if out.shape[i] > 1):
        if stride < reach:
            raise ValueError("out: its rows overlap")
        reach = stride * (n - 1) + reach
    if out.numel() and not (out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()):
        (first, last), (a, b) = _span(out), _span(logits)
        if not (last <= a or b <= first):
            raise ValueError("out: overlaps the logits without being them")
    return out


def _span(t):
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)))


_status = {}            # device index -> address of its status word


def _rows(logits, grad=None):
    st, sh, dev = logits.stride(), logits.shape, logits.device.index
    status = _status.get(dev)
    if status is None:
        status = _status[dev] = _lib.status_word(logits.device).data_ptr()
    d, dz = ((0, 0, 0), 0) if grad is None else (grad.stride(), grad.data_ptr())
    f32 = logits.dtype is torch.float32
    if len(sh) == 2:
        return _ROWS.pack(logits.data_ptr(), dz, 0, st[0], 0, d[0], sh[0], max(sh[0], 1), sh[1], f32, status)
    return _ROWS.pack(logits.data_ptr(), dz, st[0], st[1], d[0], d[1], sh[0] * sh[1], max(sh[1], 1), sh[2], f32, status)


def _call(device, what, launches, fn, *args, out=None):
    """fn(*args, stream) with the tensors' device current: streams and kernels belong to the device that is.  ``out``: a caller's tensor that is written, of which autograd
    has to know (a graph that still needs its values raises in its backward pass)."""
    if out is not None:
        increment_version(out)
    index = device.index
    if index == torch.cuda.current_device():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(index)), what, launches)
        return
    with torch.cuda.device(index):
        check(fn(*args, torch._C._cuda_getCurrentRawStream(index)), what, launches)


def _empty(device, *sizes, dtype=torch.float32):
    return torch.empty(sizes, dtype=dtype, device=device)


def _at(t):
    return 0 if t is None else t.data_ptr()


def _softmax64(z):
    """CPU statement: (z - m, m, log of the sum of exp(z - m)) in float64, m the maximum of a row: apart, since m + log S is m where m is large."""
    z = z.double()
    m = z.max(-1).values
    d = z - torch.where(m == -math.inf, torch.zeros_like(m), m)[..., None]
    return d, m, torch.exp(d).sum(-1).log()


def _taken(z, targets, ignore_index):
    """CPU statement: (kept rows, target clamped into the vocabulary, log p of the target, 0 on the other rows, what ``_softmax64`` gives)."""
    keep = targets != ignore_index
    y = targets.long()
    inside = (y >= 0) & (y < z.shape[-1])
    y = y.clamp(0, z.shape[-1] - 1)
    d, m, ls = _softmax64(z)
    lp = d.gather(-1, y[..., None])[..., 0] - ls
    lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
    return keep, y, torch.where(keep, lp, torch.zeros((), dtype=torch.float64)), (d, m, ls)


def _row_gradient(y, c, soft, keep, grad):
    """CPU statement: grad = c (onehot(y) - softmax z) on the kept rows."""
    g = -torch.exp(soft[0] - soft[2][..., None])
    g.scatter_add_(-1, y[..., None], torch.ones_like(g[..., :1]))
    grad.detach().copy_(torch.where(keep[..., None], g * c[..., None], torch.zeros((), dtype=g.dtype)).to(grad.dtype))


# ---------------------------------------------------------------------------------------------
# log-probabilities of given tokens
# ---------------------------------------------------------------------------------------------
def logprobs_fwd(logits, targets, ignore_index: int = -100):
    """(log softmax(logits)[target], stats), float32: the first of the targets' shape, ``stats`` [2, *shape] the maximum m of every row and the log of its
    sum of exp(z - m), whose sum is logsumexp(z); all 0 on ignored rows."""
    _check_logits(logits)
    targets = _check_index(targets, logits.shape[:-1], "targets", logits.device)
    if not logits.is_cuda:
        keep, _, lp, (_, m, ls) = _taken(logits.detach(), targets, ignore_index)
        return lp.float(), torch.where(keep, torch.stack([m, ls]), torch.zeros((), dtype=m.dtype)).float()
    lp, stats = _empty(logits.device, *targets.shape), _empty(logits.device, 2, *targets.shape)
    if targets.numel():
        _call(logits.device, "token_logprobs", 1, _lib.lib().tfb_token_logprobs, _rows(logits), targets.data_ptr(), targets.dtype is torch.int64, int(ignore_index),
              lp.data_ptr(), stats.data_ptr())
    return lp, stats


def logprobs_bwd(dlogp, logits, targets, stats, ignore_index: int = -100, out=None):
    """d logits = dlogp (onehot(target) - softmax(logits)); ``stats`` as ``logprobs_fwd`` gave them."""
    _check_logits(logits)
    targets = _check_index(targets, logits.shape[:-1], "targets", logits.device)
    dlogp = _check_f32(dlogp, targets.shape, "dlogp", logits.device)
    stats = _check_f32(stats, torch.Size((2, *targets.shape)), "stats", logits.device)
    grad = _gradient(logits, out, True, targets, dlogp, stats)
    if not logits.is_cuda:
        keep, y, lp, soft = _taken(logits.detach(), targets, ignore_index)
        c = torch.where(lp.isnan(), lp, dlogp.detach().double())
        _row_gradient(y, c, soft, keep, grad)
        return grad
    if targets.numel():
        _call(logits.device, "token_logprobs_bwd", 1, _lib.lib().tfb_token_logprobs_bwd, _rows(logits, grad), targets.data_ptr(), targets.dtype is torch.int64,
              int(ignore_index), stats.data_ptr(), dlogp.data_ptr(), out=out)
    return grad


def _statement(logits, targets, ignore_index):
    """What ``token_logprobs`` computes, in operations that any transformation goes through; and (kept rows, clamped targets, logits that are 0 on the other rows)."""
    keep, V = targets != ignore_index, logits.shape[-1]
    z = torch.where(keep[..., None], logits.float(), torch.zeros((), device=logits.device))
    y = targets.long()
    inside, y = (y >= 0) & (y < V), y.clamp(0, V - 1)
    lp = torch.log_softmax(z, -1).gather(-1, y[..., None])[..., 0]
    lp = torch.where(inside, lp, torch.full((), math.nan, device=logits.device))
    return torch.where(keep, lp, torch.zeros((), device=logits.device)), (keep, y, z)


def _transformed(*tensors):
    """Whether a tensor belongs to a function transformation (vmap, grad, jvp ...) or carries a tangent: a kernel sees neither."""
    return (any(torch._C._functorch.is_functorch_wrapped_tensor(t) or torch._C._functorch.is_legacy_batchedtensor(t) for t in tensors)
            or forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors if t.is_floating_point()))


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index):
        lp, stats = logprobs_fwd(logits, targets, ignore_index)
        ctx.save_for_backward(logits, targets, stats)
        ctx.ignore_index = ignore_index
        return lp

    @staticmethod
    def backward(ctx, dlogp):
        logits, targets, stats = ctx.saved_tensors
        if torch.is_grad_enabled() or _transformed(dlogp):
            # a gradient that is differentiated again (create_graph), or one of many at once
            lp, (keep, y, z) = _statement(logits, targets, ctx.ignore_index)
            c = torch.where(keep, torch.where(lp.isnan(), lp, dlogp.float()), torch.zeros((), device=logits.device))
            hot = torch.zeros_like(z).scatter_(-1, y[..., None], 1.0)
            return (c[..., None] * (hot - torch.softmax(z, -1))).to(logits.dtype), None, None
        return logprobs_bwd(dlogp.float(), logits, targets, stats, ctx.ignore_index), None, None


def token_logprobs(logits, targets, ignore_index: int = -100):
    """Log-probabilities of given tokens, float32 of the targets' shape, with the gradient of the logits.  Second derivatives, forward-mode ones and the
    transformations of ``torch.func`` go through tensor operations."""
    if _transformed(logits, targets):
        _check_logits(logits)
        if targets.shape != logits.shape[:-1]:
            raise ValueError(f"targets: {tuple(logits.shape[:-1])} wanted, got {tuple(targets.shape)}")
        return _statement(logits, targets, ignore_index)[0]
    return _TokenLogprobs.apply(logits, targets, ignore_index)


# ---------------------------------------------------------------------------------------------
# policy
# ---------------------------------------------------------------------------------------------
class PolicyLoss(NamedTuple):
    loss: torch.Tensor                     # scalar
    kl: torch.Tensor                       # scalar: mean of the KL estimate (0 without reference log-probabilities)
    clipped: torch.Tensor                  # scalar: share of the tokens whose gradient the clip took
    logp: torch.Tensor                     # log-probabilities of the tokens
    dlogits: Optional[torch.Tensor]


@torch.no_grad()
def _policy_statement(logits, targets, advantages, old, ref, lo, hi, ratio, kl_coef, kl, mean, n_valid, ignore_index, grad):
    keep, y, lp, soft = _taken(logits, targets, ignore_index)
    zero = torch.zeros((), dtype=torch.float64)
    A = (advantages[:, None] if advantages.dim() < targets.dim() else advantages).double().expand(lp.shape)
    clipped = torch.zeros_like(lp)
    if ratio:
        r = torch.exp(lp - old.double()) if old is not None else torch.exp(lp - lp)
        s = ds = r * A
        c = r.clamp(1 - lo, 1 + hi) * A
        clipped = (c < s).double()
        s, ds = torch.where(c < s, c, s), torch.where(c < s, zero, ds)
    else:
        s, ds = A * lp, A
    k, dk = torch.zeros_like(lp), torch.zeros_like(lp)
    if ref is not None:
        x = ref.double() - lp
        k, dk = {"k3": lambda: (torch.where(x == math.inf, x, torch.expm1(x) - x), -torch.expm1(x)), "k1": lambda: (x, -torch.ones_like(x)),
                 "log_ratio": lambda: (-x, torch.ones_like(x))}[kl]()
    w = keep.double()
    if mean == "tokens":
        w = w / (n_valid.double() if n_valid is not None else w.sum().clamp(min=1))
    elif mean == "sequences":
        w = w.view(-1, targets.shape[-1])
        w = (w / (max(len(w), 1) * w.sum(1, keepdim=True).clamp(min=1))).view(keep.shape)
    total = lambda v: torch.where(keep, w * v, zero).sum().float()
    loss, dloss = (kl_coef * k - s, kl_coef * dk - ds) if kl_coef != 0 else (-s, -ds)
    if grad is not None:
        _row_gradient(y, torch.where(lp.isnan(), lp, w * dloss), soft, keep, grad)
    return PolicyLoss(total(loss), total(k), total(clipped), lp.float(), grad)


def policy_loss_fwd_bwd(logits, targets, advantages, old_logprobs=None, ref_logprobs=None, *, clip=0.2, kl_coef: float = 0.0, kl: str = "k3",
                        mean: str = "tokens", n_valid=None, ignore_index: int = -100, want_grad: bool = True, out=None) -> PolicyLoss:
    """Policy loss of sampled tokens and its gradient with respect to the logits, in one pass over them.

    Per token, with lp its log-probability, A its advantage, r = exp(lp - old): -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl_coef * KL.  ``clip`` is
    one bound for both sides, (lo, hi), or None: no clip.  Without ``old_logprobs`` the tokens are the policy's own: r is 1 and its gradient that
    of lp; without a clip as well the objective is A lp itself.  KL against ``ref_logprobs``, x = ref - lp.  On tokens that the policy sampled, KL(policy || reference) is
    the mean of "k3" exp(x) - 1 - x and of "log_ratio" -x (lp - ref; often called k1 elsewhere).  On tokens that the reference sampled (an older policy, whose
    log-probabilities are passed as ``ref_logprobs``), KL(reference || policy) is the mean of "k1" x.  The two have opposite signs: "k1" on the policy's own tokens has a mean
    of -KL(policy || reference).

    ``advantages``: one per token, or [B], one per sequence.  ``mean``: over all "tokens" (``n_valid``, one float32 value above 0 on the device, replaces their
    number, for a batch in several calls), over the "sequences" of each one's mean over its tokens (a sequence without tokens counts as 0), or "sum"."""
    _check_logits(logits)
    dev = logits.device
    targets = _check_index(targets, logits.shape[:-1], "targets", dev)
    kl_kind, mean_kind = _one_of(kl, _KL, "kl"), _one_of(mean, _MEAN, "mean")
    if n_valid is not None and mean != "tokens":
        raise ValueError("n_valid: belongs to the mean over tokens")
    if kl_coef != 0.0 and ref_logprobs is None:
        raise ValueError("kl_coef: wants reference log-probabilities")
    adv_seq = logits.dim() == 3 and advantages.dim() == 1
    advantages = _check_f32(advantages, targets.shape[:1] if adv_seq else targets.shape, "advantages", dev)
    old, ref = _check_f32(old_logprobs, targets.shape, "old_logprobs", dev), _check_f32(ref_logprobs, targets.shape, "ref_logprobs", dev)
    n_valid = _check_n_valid(n_valid, dev)
    lo, hi = (math.inf, math.inf) if clip is None else (float(clip[0]), float(clip[1])) if isinstance(clip, (tuple, list)) else (float(clip), float(clip))
    if not (lo >= 0 and hi >= 0):
        raise ValueError(f"clip: bounds of 0 or more, got {clip!r}")
    ratio = old is not None or clip is not None
    grad = _gradient(logits, out, want_grad, targets, advantages, old, ref, n_valid)
    B, S = targets.shape if targets.dim() == 2 else (1, targets.shape[0])
    if not logits.is_cuda:
        return _policy_statement(logits, targets, advantages, old, ref, lo, hi, ratio, kl_coef, kl, mean, n_valid, ignore_index, grad)
    lp = _empty(dev, *targets.shape)
    if not lp.numel():
        z = torch.zeros((), device=dev)
        return PolicyLoss(z, z, z, lp, grad)
    T = lp.numel()
    n_ws = 6 * PIPE_CLUSTERS + 3 * T
    sums, work = _empty(dev, 3), _empty(dev, n_ws + B + 1)
    ws = work.data_ptr()
    arg = _POLICY.pack(targets.data_ptr(), targets.dtype is torch.int64, int(ignore_index), advantages.data_ptr(), _at(old), _at(ref), adv_seq, ratio, kl_kind, mean_kind,
                       1 - lo, 1 + hi, float(kl_coef), _at(n_valid), lp.data_ptr(), sums.data_ptr(), ws, ws + 4 * n_ws, ws + 4 * (n_ws + B))
    _call(dev, "policy_loss", 2, _lib.lib().tfb_policy_loss, _rows(logits, grad), arg, out=out)
    return PolicyLoss(*sums.unbind(), lp, grad)


# ---------------------------------------------------------------------------------------------
# preferences
# ---------------------------------------------------------------------------------------------
class PreferenceLoss(NamedTuple):
    loss: torch.Tensor                     # scalar: mean over the pairs
    margins: torch.Tensor                  # [N] beta times the difference of the log-ratios: > 0 where the chosen answer is preferred
    logp: torch.Tensor                     # [2N] log-probabilities of the answers (their means with ``average``)
    dlogits: Optional[torch.Tensor]


@torch.no_grad()
def _preference_statement(logits, targets, ref, beta, kind, label_smoothing, average, ignore_index, grad):
    N = len(targets) // 2
    keep, y, lp, soft = _taken(logits, targets, ignore_index)
    n = keep.sum(1).clamp(min=1).double() if average else torch.ones(2 * N, dtype=torch.float64)
    L = lp.sum(1) / n
    d = L - (ref.double() if ref is not None else 0)
    h = d[:N] - d[N:]
    x = beta * h
    if kind == "sigmoid":
        l = torch.log1p(torch.exp(-x.abs())) + (-x).clamp(min=0) + (label_smoothing * x if label_smoothing else 0)
        dl = beta * (label_smoothing - torch.sigmoid(-x))
    elif kind == "hinge":
        l, dl = (1 - x).clamp(min=0), torch.where(x.isnan(), x, -beta * (x < 1).double())
    else:
        l, dl = (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta)
    if grad is not None:
        c = torch.cat([dl, -dl]) / max(N, 1) / n
        _row_gradient(y, c[:, None].expand(lp.shape), soft, keep, grad)
    return PreferenceLoss((l.sum() / max(N, 1)).float(), x.float(), L.float(), grad)


def preference_loss_fwd_bwd(logits, targets, ref_logprobs=None, *, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0,
                            average: bool = False, ignore_index: int = -100, want_grad: bool = True, out=None) -> PreferenceLoss:
    """Loss of N pairs of answers and its gradient: logits [2N, S, V] and targets [2N, S] hold the N chosen answers first, then the N rejected
    ones, each padded with ``ignore_index``.

    L_i is the sum of the log-probabilities of answer i (``average``: their mean), ``ref_logprobs`` [2N] the same under the reference model (None: 0), h
    the difference (L - ref) of the chosen answer less that of the rejected one.  ``kind``: "sigmoid" -(1 - e) log sigmoid(beta h) - e log sigmoid(-beta h)
    with e = ``label_smoothing``, "hinge" max(0, 1 - beta h), "squared" (h - 1 / (2 beta))^2."""
    _check_logits(logits)
    dev = logits.device
    if logits.dim() != 3 or logits.shape[0] % 2:
        raise ValueError(f"logits: [2N, S, V], got {tuple(logits.shape)}")
    targets = _check_index(targets, logits.shape[:-1], "targets", dev)
    loss_kind = _one_of(kind, _KIND, "kind")
    if not 0 < beta < math.inf:
        raise ValueError(f"beta: more than 0, got {beta}")
    if not 0 <= label_smoothing < 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError(f"label_smoothing: in [0, 0.5), of the sigmoid loss, got {label_smoothing} ({kind})")
    N, S = logits.shape[0] // 2, logits.shape[1]
    ref = _check_f32(ref_logprobs, torch.Size((2 * N,)), "ref_logprobs", dev)
    grad = _gradient(logits, out, want_grad, targets, ref)
    if not logits.is_cuda:
        return _preference_statement(logits, targets, ref, beta, kind, label_smoothing, average, ignore_index, grad)
    margins, L = _empty(dev, N), _empty(dev, 2 * N)
    if N == 0 or S == 0:
        # no pairs, or only empty answers: nothing depends on the logits
        L.zero_()
        d = L if ref is None else -ref
        x = beta * (d[:N] - d[N:])
        l = {"sigmoid": torch.nn.functional.softplus(-x) + label_smoothing * x, "hinge": (1 - x).clamp(min=0), "squared": (x / beta - 0.5 / beta) ** 2}[kind]
        return PreferenceLoss(l.sum() / max(N, 1), x, L, grad)
    T = 2 * N * S
    loss, lp64, work = _empty(dev), _empty(dev, T, dtype=torch.float64), _empty(dev, 2 * T + 3 * N + 1)
    ws = work.data_ptr()
    arg = _PREFERENCE.pack(targets.data_ptr(), targets.dtype is torch.int64, int(ignore_index), _at(ref), loss_kind, bool(average), float(beta), float(label_smoothing),
                           loss.data_ptr(), margins.data_ptr(), L.data_ptr(), lp64.data_ptr(), ws, ws + 8 * T, ws + 8 * T + 8 * N, ws + 8 * T + 12 * N)
    _call(dev, "preference_loss", 3 if want_grad else 2, _lib.lib().tfb_preference_loss, _rows(logits, grad), arg, out=out)
    return PreferenceLoss(loss, margins, L, grad)


# ---------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------
class DistillLoss(NamedTuple):
    loss: torch.Tensor                     # scalar: temperature^2 times the mean of kl over the rows with entries
    kl: torch.Tensor                       # per row, at the temperature
    dlogits: Optional[torch.Tensor]


@torch.no_grad()
def _distill_statement(logits, top_ids, top_logits, temperature, n_valid, grad):
    V = logits.shape[-1]
    ids = top_ids.long()
    keep, have = ids[..., 0] >= 0, (ids >= 0) & (ids < V)
    bad = (ids >= V).any(-1) & keep
    zero = torch.zeros((), dtype=torch.float64)
    lq = torch.log_softmax(torch.where(have, top_logits.double() / temperature, torch.full((), -math.inf, dtype=torch.float64)), -1)
    q = torch.where(have, lq.exp(), zero)
    z, _, ls = _softmax64(logits.double() / temperature)
    lp = z.gather(-1, ids.clamp(0, V - 1)) - ls[..., None]
    kl = torch.where(have & (q != 0), q * (lq - lp), zero).sum(-1)
    kl = torch.where(keep, torch.where(bad, torch.full_like(kl, math.nan), kl), zero)
    w = 1.0 / (n_valid.double() if n_valid is not None else keep.sum().clamp(min=1).double())
    if grad is not None:
        d = torch.exp(z - ls[..., None])
        d.scatter_add_(-1, ids.clamp(0, V - 1), -q)
        d = torch.where(bad[..., None], torch.full_like(d, math.nan), d) * (temperature * w)
        grad.copy_(torch.where(keep[..., None], d, zero).to(grad.dtype))
    return DistillLoss((kl.sum() * temperature ** 2 * w).float().reshape(()), kl.float(), grad)


def distill_loss_fwd_bwd(logits, top_ids, top_logits, *, temperature: float = 1.0, n_valid=None, want_grad: bool = True, out=None) -> DistillLoss:
    """Distillation from the top logits of a teacher, and its gradient, in one pass over the student's logits.

    ``top_ids`` (int64 or int32) and ``top_logits`` (bfloat16 or float32) are the logits' leading shape + [K], K up to 1024: the teacher's best
    tokens of every row with their logits (or log-probabilities: only differences count).  Negative ids are entries that are not there; a row
    whose first id is negative has none and is not trained on.  With q the soft-max of a row's entries at the temperature and p that of the
    student's whole row, KL = sum q (log q - log p); loss = temperature^2 mean KL.  An id that comes twice counts twice.  A row with entries whose
    teacher logits are all -inf, or with an id outside the vocabulary, gives NaN.  ``n_valid`` (one float32 value above 0 on the device) replaces
    the number of rows with entries."""
    _check_logits(logits)
    dev, V = logits.device, logits.shape[-1]
    if top_ids.dim() != logits.dim() or top_ids.shape[-1] < 1 or top_ids.shape[-1] > MAX_TOP:
        raise ValueError(f"top_ids: {tuple(logits.shape[:-1])} + [K] wanted, K up to {MAX_TOP}, got {tuple(top_ids.shape)}")
    K = top_ids.shape[-1]
    top_ids = _check_index(top_ids, torch.Size((*logits.shape[:-1], K)), "top_ids", dev)
    if top_logits.shape != top_ids.shape or top_logits.device != dev or top_logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"top_logits: bfloat16 or float32 {tuple(top_ids.shape)} on {dev} wanted, got {top_logits.dtype} {tuple(top_logits.shape)} on {top_logits.device}")
    top_logits = top_logits.contiguous()
    if not 0 < temperature < math.inf:
        raise ValueError(f"temperature: more than 0, got {temperature}")
    n_valid = _check_n_valid(n_valid, dev)
    grad = _gradient(logits, out, want_grad, top_ids, top_logits, n_valid)
    rows = logits.shape[:-1]
    if not logits.is_cuda:
        return _distill_statement(logits, top_ids, top_logits, temperature, n_valid, grad)
    kl = _empty(dev, *rows)
    T = kl.numel()
    if not T:
        return DistillLoss(torch.zeros((), device=dev), kl, grad)
    n_ws = 6 * PIPE_CLUSTERS + T
    loss, work = _empty(dev), _empty(dev, n_ws + 2)
    ws = work.data_ptr()
    arg = _DISTILL.pack(top_ids.data_ptr(), top_logits.data_ptr(), top_ids.dtype is torch.int64, top_logits.dtype is torch.float32, K, float(temperature), _at(n_valid),
                        kl.data_ptr(), loss.data_ptr(), ws, ws + 4 * n_ws, ws + 4 * n_ws + 4)
    _call(dev, "distill_loss", 2, _lib.lib().tfb_distill_loss, _rows(logits, grad), arg, out=out)
    return DistillLoss(loss, kl, grad)


# ---------------------------------------------------------------------------------------------
# scoring from hidden states
# ---------------------------------------------------------------------------------------------
def _tma_ready(t):
    """Rows that start at 16-byte boundaries."""
    if t.stride(-1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def linear_logprobs(x, weight, targets, ignore_index: int = -100):
    """Log-probabilities of given tokens under a head, and the logsumexp of its logits, without the logits of many rows in memory (those of up to 64 rows, or 128 at widths of
    2048 and more, stand in a float32 workspace on the GPU): x [..., H], weight [V, H] (bfloat16, or
    float32 on the CPU), targets of x's leading shape -> (logp, lse), float32, both 0 where the target is ``ignore_index``.  For passes that want
    no gradient (reference models, older policies, evaluation); with one use ``token_logprobs`` on the logits."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        raise ValueError("linear_logprobs has no gradient: call it under torch.no_grad(), or use token_logprobs")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.numel() == 0:
        raise ValueError(f"x [..., H] and weight [V, H], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x.dtype != weight.dtype or x.device != weight.device:
        raise ValueError(f"x and weight: one type and device, got {x.dtype} on {x.device} and {weight.dtype} on {weight.device}")
    targets = _check_index(targets, x.shape[:-1], "targets", x.device)
    x2, y = x.reshape(-1, x.shape[-1]), targets.view(-1)
    if not x.is_cuda:
        if not x.is_floating_point():
            raise ValueError(f"x: a floating type, got {x.dtype}")
        keep, _, lp, (_, m, ls) = _taken(x2.float() @ weight.float().t(), y, ignore_index)
        return lp.float().view(targets.shape), torch.where(keep, m + ls, torch.zeros((), dtype=m.dtype)).float().view(targets.shape)
    if x.dtype is not torch.bfloat16 or x.shape[-1] % 8:
        raise ValueError(f"x: bfloat16 of a width that is a multiple of 8 on the GPU, got {x.dtype} {tuple(x.shape)}")
    x2, w, dev = _tma_ready(x2), _tma_ready(weight), x.device
    lp, lse = _empty(dev, *targets.shape), _empty(dev, *targets.shape)
    (V, H), M = w.shape, y.numel()
    if not M:
        return lp, lse
    n = min(M, SCORE_ROWS, max(256, (1 << 27) // (4 * -(-V // 256))))
    # workspace: parts of a row's statistics (two values per half a tile), compacted rows and their number; the logits of few rows
    ldz = -(-V // 4) * 4 if n <= 128 and n * V <= 1 << 27 else 0
    parts = 4 * -(-V // (128 if n <= 128 else 256)) * n
    xc, work = _empty(dev, n, H, dtype=torch.bfloat16), _empty(dev, parts + ldz * n + 3 * n + 1)
    ws = work.data_ptr()
    zy, rows = ws + 4 * (parts + ldz * n), ws + 4 * (parts + ldz * n + n)
    status = _lib.status_word(dev).data_ptr()
    for a in range(0, M, n):
        arg = _SCORE.pack(x2.data_ptr() + 2 * a * x2.stride(0), w.data_ptr(), x2.stride(0), w.stride(0), y.data_ptr() + y.element_size() * a, y.dtype is torch.int64,
                          int(ignore_index), min(n, M - a), V, H, lp.data_ptr() + 4 * a, lse.data_ptr() + 4 * a, rows, rows + 4, rows + 4 + 4 * n, xc.data_ptr(), H, ws, 0,
                          ws + 4 * parts if ldz else 0, ldz, zy)
        _call(dev, "linear_logprobs", 3, _lib.lib().tfb_linear_logprobs, arg, status)
    return lp, lse
