"""Distillation from a teacher's top logits (csrc/distill.hip).

``top_logits`` takes from a teacher's logits what a student's loss needs of them: the k largest of
each row, their classes, and the row's log-sum-exp. ``distill_loss`` is the loss against that, with
or without labels. GPU tensors run the native kernels; CPU tensors (and reference mode) take the
PyTorch path below, whose gradients are autograd's.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from .. import _native
from .functional import _C, _ref

MAX_CLASSES = 1 << 18
MAX_K = 1024
MIN_TEMPERATURE = 2.0 ** -64     # csrc/distill.h kDistillMinTemp; its reciprocal is the largest
REST = 2.0 ** -20        # csrc/distill.h kDistillRest
_REDUCTION = ("none", "mean", "sum")
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class TopLogits(NamedTuple):
    """A teacher's answer: ``values`` [..., k] (descending), ``indices`` [..., k] (int32; a
    negative one marks an entry that is not kept) and ``lse`` [...] (fp32), the log-sum-exp of all
    logits / temperature (None where no rest of the mass is wanted)."""
    values: torch.Tensor
    indices: torch.Tensor
    lse: torch.Tensor | None = None


def _check_logits(logits, name="logits"):
    if logits.dim() < 1:
        raise ValueError(f"{name} must have a class dimension")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"{name} must be fp32, bf16 or fp16, got {logits.dtype}")
    if not 1 <= logits.shape[-1] <= MAX_CLASSES:
        raise ValueError(f"{name} has {logits.shape[-1]} classes: 1 to {MAX_CLASSES} are supported")


def _check_temperature(t):
    t = float(t)
    if not MIN_TEMPERATURE <= t <= 1 / MIN_TEMPERATURE:
        raise ValueError(f"temperature must be positive, 2^-64 to 2^64, got {t}")
    return t


def _name_bad_class(logits, indices, target, ignore_index):
    """Debug mode: name a class outside the row on the host (the kernel NaN-poisons its row)."""
    n = logits.shape[-1]
    bad = [("index", indices, indices >= n)]
    if target is not None:
        bad.append(("target", target, (target != ignore_index) & ((target < 0) | (target >= n))))
    for name, x, b in bad:
        if bool(b.any()):
            at = b.nonzero()[0].tolist()
            raise IndexError(f"distill_loss: {name} {int(x[tuple(at)])} at {at} is outside [0, {n})")


def top_logits(logits, k, temperature=1.0):
    """The ``k`` largest logits of each row of ``logits`` [..., classes] as :class:`TopLogits`.

    Descending; among equal logits the lowest class comes first, and NaN counts as the largest.
    ``lse`` is taken at ``temperature``, that of the loss that will use it; the values are the
    logits as they are. Not differentiable, backward or forward: a teacher's answer is data to its
    student.
    """
    if not _ref(logits):
        return TopLogits(*_C().top_logits(logits, k, temperature))
    _check_logits(logits)
    t = _check_temperature(temperature)
    n = logits.shape[-1]
    k = int(k)
    if not 1 <= k <= min(n, MAX_K):
        raise ValueError(f"k must be 1 to {min(n, MAX_K)}, got {k}")
    with torch.no_grad():
        logits = forward_ad.unpack_dual(logits).primal
        z = logits.float()
        values, indices = torch.sort(z, dim=-1, descending=True, stable=True)
        lse = torch.logsumexp(z.double() / t, -1).float()
        return TopLogits(values[..., :k].to(logits.dtype), indices[..., :k].to(torch.int32), lse)


def _finite_max(x):
    m = x.detach().amax(1, keepdim=True)
    return torch.where(torch.isfinite(m), m, torch.zeros_like(m))


def _ref_distill(z, values, indices, lse, target, t, alpha, tail, ignore_index):
    """The rows' losses in 64 bits, differentiable in ``z`` [rows, classes]."""
    z = z.double()
    n, v = z.shape
    used = (indices >= 0).any(1) if alpha != 0 else torch.zeros(n, dtype=torch.bool, device=z.device)
    if target is not None and alpha != 1:
        used = used | (target != ignore_index)
    z = torch.where(used[:, None], z, torch.zeros_like(z))   # (no term: not looked at)
    logq = F.log_softmax(z / t, 1)
    idx = indices.long()
    kept = idx >= 0
    bad = (idx >= v).any(1)
    idx = idx.clamp(0, v - 1)
    tv = values.double() / t
    base = (lse.double()[:, None] if tail
            else torch.logsumexp(tv.masked_fill(~kept, -math.inf), 1, keepdim=True))
    has = kept.any(1) & (base[:, 0] != -math.inf) & (alpha != 0)
    live = kept & has[:, None]
    logp = torch.where(live, tv - base, torch.full_like(tv, -math.inf))
    p = logp.exp()
    # (a class without mass takes no part, whatever the student gives it: 0 log 0 = 0)
    use = live & (p != 0)
    lq = torch.where(use, logq.gather(1, idx), torch.zeros_like(p))
    loss = (p * (torch.where(use, logp, torch.zeros_like(p)) - lq)).sum(1)
    if tail:
        inside = torch.zeros(n, v + 1, dtype=torch.bool, device=z.device)
        inside.scatter_(1, torch.where(live, idx, torch.full_like(idx, v)), True)
        inside = inside[:, :v]
        rest = 1.0 - p.sum(1)
        rest = torch.where(has & ~inside.all(1) & ~(rest < REST), rest, torch.zeros_like(rest))
        some = rest != 0
        zt = z / t
        outer = torch.where(some[:, None], zt.masked_fill(inside, -math.inf), torch.zeros_like(zt))
        # (logarithms of sums apart from their bases: where the classes not kept stand as far from the others
        # as the type's lowest value, they are below the distance's last bit, and the shares with them)
        top_z, top_outer = _finite_max(zt), _finite_max(outer)
        lrest = ((outer - top_outer).exp().sum(1).log() - (zt - top_z).exp().sum(1).log()
                 + (top_outer - top_z)[:, 0])
        loss = loss + torch.where(some, rest * (torch.where(some, rest, torch.ones_like(rest)).log()
                                                - lrest), torch.zeros_like(rest))
    loss = torch.where(has, loss * (alpha * t * t), torch.zeros_like(loss))
    if target is not None and alpha != 1:
        hit = target != ignore_index
        bad = bad | (hit & ((target < 0) | (target >= v)))
        y = target.clamp(0, v - 1)[:, None]
        ce = -F.log_softmax(z, 1).gather(1, y)[:, 0]
        loss = loss + torch.where(hit, (1 - alpha) * ce, torch.zeros_like(ce))
    return loss * torch.where(bad, math.nan, 1.0).to(loss)


def distill_loss(logits, top, target=None, temperature=1.0, alpha=None, tail=False,
                 reduction="mean", ignore_index=-100):
    """Loss of a student's ``logits`` [..., classes] against a teacher's ``top`` logits.

    With q = softmax(logits / T) a row's loss is

        alpha T^2 KL(p || q) + (1 - alpha) cross_entropy(logits, target)

    ``tail=False``: p is the softmax of the kept teacher logits / T among themselves.
    ``tail=True``: p is the teacher's own probability of each kept class, exp(value / T - lse), and
    the mass it leaves to all other classes is one more term, against the mass q leaves to them
    (``top.lse`` must have been taken at the same T). A rest below 2^-20 counts as none.

    ``target`` [...] holds int64 classes; ``alpha`` defaults to 1 without it and must be given with
    it. Rows may keep fewer logits (negative indices); a row that keeps none has no teacher term, a
    row whose target is ``ignore_index`` no label term, and a row with neither is not looked at:
    loss and gradient 0. ``reduction``: "mean" over all rows, "sum", or "none". A class outside
    the row makes its loss and gradient NaN.

    Teacher's side is data: gradients flow to ``logits`` alone, once and in reverse mode. Forward and backward can be captured,
    together or apart. As with every autograd function, no eager graph of the same leaves may be alive
    while a backward is captured.
    """
    if alpha is None:
        if target is not None:
            raise ValueError("alpha (the weight of the teacher's term) must be given with a target")
        alpha = 1.0
    values, indices, lse = top if len(top) == 3 else (*top, None)
    if not _ref(logits):
        if _native._debug:
            _name_bad_class(logits, indices, target if alpha != 1 else None, ignore_index)
        return _C().distill_loss(logits, values, indices, lse, target, temperature, alpha, tail,
                                 reduction, ignore_index, _native._debug)
    _check_logits(logits)
    t = _check_temperature(temperature)
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction must be one of {_REDUCTION}, got {reduction!r}")
    alpha = float(alpha)
    if not 0 <= alpha <= 1:
        raise ValueError(f"alpha must be in [0, 1], got {alpha}")
    if target is None and alpha != 1:
        raise ValueError("alpha below 1 needs a target")
    lead = logits.shape[:-1]
    k = values.shape[-1] if values.dim() else 0
    if values.shape[:-1] != lead or indices.shape != values.shape or values.dim() < 1:
        raise ValueError(f"top values {tuple(values.shape)} and indices {tuple(indices.shape)} do "
                         f"not fit logits {tuple(logits.shape)}")
    if not 1 <= k <= MAX_K:
        raise ValueError(f"1 to {MAX_K} kept logits a row are supported, got {k}")
    if values.dtype not in _FLOATS or indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"top values must be fp32, bf16 or fp16 and indices int32 or int64, got "
                        f"{values.dtype}, {indices.dtype}")
    if tail:
        if lse is None:
            raise ValueError("tail=True needs the teacher's lse")
        if lse.shape != lead or lse.dtype != torch.float32:
            raise ValueError(f"lse must be fp32 of shape {tuple(lead)}")
    if target is not None and (target.shape != lead or target.dtype != torch.int64):
        raise ValueError(f"target must be int64 of shape {tuple(lead)}")
    for name, x in (("values", values), ("indices", indices), ("lse", lse), ("target", target)):
        if x is not None and x.device != logits.device:
            raise ValueError(f"{name} is on {x.device}, the logits are on {logits.device}")
        if x is not None and x.requires_grad:
            raise ValueError(f"{name} requires grad: a teacher's answer is data, detach it")

    rows = _ref_distill(logits.reshape(-1, logits.shape[-1]), values.reshape(-1, k),
                        indices.reshape(-1, k), lse.reshape(-1) if tail else None,
                        target.reshape(-1) if target is not None else None, t, alpha, tail,
                        ignore_index)
    if reduction == "none":
        return rows.float().view(lead)
    return (rows.mean() if reduction == "mean" else rows.sum()).float()
