"""top_logits / distill_loss on the CPU reference path: against the formulas written out row by row
in Python floats, gradients against differences, rows without terms, and every refusal.

Tolerances: the reference path computes in 64 bits and returns fp32 (half a step: 2^-24 relative);
a central difference of step h has an error of h^2 times the third derivative (order 1 here) and
2^-53 / h of rounding: 1e-10 + 1e-11 at h = 1e-5.
"""
import math

import pytest
import torch

from pytorch_cifar_amd.nn import functional as PF
from pytorch_cifar_amd.ops.distill import _ref_distill

HALF = 2.0 ** -24


def row_loss(z, values, idx, lse, y, t, alpha, tail, ignore=-100):
    """One row, from the definition."""
    v = len(z)

    def softmax(x):
        m = max(x)
        e = [math.exp(a - m) for a in x]
        return [a / sum(e) for a in e]

    loss = 0.0
    pairs = [(a, i) for a, i in zip(values, idx) if i >= 0]
    if pairs and alpha:
        q = softmax([a / t for a in z])
        if tail:
            p = [math.exp(a / t - lse) for a, _ in pairs]
        else:
            p = softmax([a / t for a, _ in pairs])
        kd = sum(a * math.log(a / q[i]) for a, (_, i) in zip(p, pairs) if a > 0)
        inside = {i for _, i in pairs}
        rest = 1 - sum(p)
        if tail and len(inside) < v and rest >= 2.0 ** -20:
            kd += rest * math.log(rest / sum(q[j] for j in range(v) if j not in inside))
        loss += alpha * t * t * kd
    if y is not None and y != ignore and alpha != 1:
        loss -= (1 - alpha) * math.log(softmax(z)[y])
    return loss


def case(r=7, v=13, k=5, t=2.0, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    teacher = (3 * torch.randn(r, v, generator=g)).to(dtype)
    z = (2 * torch.randn(r, v, generator=g)).to(dtype)
    y = torch.randint(0, v, (r,), generator=g)
    return z, PF.top_logits(teacher, k, t), y, teacher


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("labels", [False, True])
@pytest.mark.parametrize("k", [1, 5, 13])
def test_matches_the_definition(tail, labels, k):
    z, top, y, _ = case(k=k)
    top.indices[2, k // 2:] = -1            # fewer kept
    top.indices[3] = -1                     # none
    if k > 1:
        top.indices[4, 1] = top.indices[4, 0]   # a class twice
    y[5] = -100
    alpha = 0.6 if labels else 1.0
    got = PF.distill_loss(z, top, y if labels else None, temperature=2.0, alpha=alpha, tail=tail,
                          reduction="none")
    for i in range(z.shape[0]):
        want = row_loss(z[i].tolist(), top.values[i].tolist(), top.indices[i].tolist(),
                        top.lse[i].item(), y[i].item() if labels else None, 2.0, alpha, tail)
        # terms of order 10 in 64 bits, then one rounding
        assert abs(got[i].item() - want) <= HALF * abs(want) + 1e-13
    total = got.double().sum().item()
    for red, scale in (("sum", 1.0), ("mean", 1.0 / z.shape[0])):
        one = PF.distill_loss(z, top, y if labels else None, temperature=2.0, alpha=alpha, tail=tail,
                              reduction=red).item()
        assert abs(one - total * scale) <= 2 * HALF * got.double().abs().sum().item() * scale


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_matches_differences(tail):
    z, top, y, _ = case()
    top.indices[3] = -1
    top.indices[4, 1] = top.indices[4, 0]
    y[3] = -100
    z = z.double().requires_grad_(True)

    def f(x):
        return _ref_distill(x, top.values, top.indices, top.lse, y, 2.0, 0.6, tail, -100).sum()

    (g,) = torch.autograd.grad(f(z), z)
    h = 1e-5
    for i in range(z.shape[0]):
        for j in range(z.shape[1]):
            d = torch.zeros_like(z)
            d[i, j] = h
            fd = (f(z + d) - f(z - d)).item() / (2 * h)
            assert abs(g[i, j].item() - fd) <= 2e-9
    assert (g[3] == 0).all()


def test_top_logits_order_and_ties():
    z = torch.tensor([[1.0, 3.0, 3.0, -0.0, 0.0, 3.0], [-math.inf] * 6,
                      [0.0, math.nan, 9.0, math.inf, -1.0, 2.0]])
    top = PF.top_logits(z, 4)
    assert top.indices.tolist() == [[1, 2, 5, 0], [0, 1, 2, 3], [1, 3, 2, 5]]
    assert top.indices.dtype == torch.int32 and top.values.dtype == z.dtype
    assert top.lse[1] == -math.inf and math.isnan(top.lse[2].item())
    assert PF.top_logits(z, 6).indices[0].tolist() == [1, 2, 5, 0, 3, 4]


def test_shapes_and_empty():
    z = torch.randn(2, 3, 11)
    top = PF.top_logits(z, 4)
    assert top.values.shape == (2, 3, 4) and top.lse.shape == (2, 3)
    assert PF.distill_loss(z, top, reduction="none").shape == (2, 3)
    assert PF.distill_loss(z, top[:2]).shape == ()
    e = PF.top_logits(torch.zeros(0, 11), 4)
    assert e.values.shape == (0, 4) and e.lse.shape == (0,)
    assert PF.distill_loss(torch.zeros(0, 11), e, reduction="sum").item() == 0


def test_rows_without_terms_are_not_looked_at():
    z, top, y, _ = case()
    z[3] = math.nan
    top.indices[3] = -1
    y[3] = -100
    z.requires_grad_(True)
    loss = PF.distill_loss(z, top, y, temperature=2.0, alpha=0.5, tail=True)
    loss.backward()
    assert torch.isfinite(loss) and (z.grad[3] == 0).all() and torch.isfinite(z.grad).all()


def test_bad_classes_poison_their_row():
    z, top, y, _ = case()
    top.indices[1, 0] = z.shape[1]
    y[2] = z.shape[1]
    loss = PF.distill_loss(z, top, y, temperature=2.0, alpha=0.5, reduction="none")
    assert torch.isnan(loss).tolist() == [i in (1, 2) for i in range(z.shape[0])]


def test_same_answer_as_the_teacher_is_no_loss():
    # student = teacher: every q equals its p, up to the roundings of lse (2^-24 of |lse| < 16)
    _, top, _, teacher = case()
    z = teacher.clone().requires_grad_(True)
    loss = PF.distill_loss(z, top, temperature=2.0, tail=True)
    loss.backward()
    # KL is second order in the difference of lse; the gradient is first order
    assert abs(loss.item()) <= 1e-5 and z.grad.abs().max() <= 4 * 16 * HALF


@pytest.mark.parametrize("kw, err", [
    (dict(temperature=0.0), ValueError), (dict(temperature=math.inf), ValueError),
    (dict(alpha=1.5), ValueError), (dict(alpha=0.5), ValueError), (dict(reduction="max"), ValueError),
    (dict(target=torch.zeros(7, dtype=torch.int64)), ValueError),
    (dict(target=torch.zeros(7, dtype=torch.int32), alpha=0.5), ValueError),
    (dict(target=torch.zeros(6, dtype=torch.int64), alpha=0.5), ValueError),
])
def test_distill_refusals(kw, err):
    z, top, _, _ = case()
    with pytest.raises(err):
        PF.distill_loss(z, top, **kw)


def test_distill_refuses_what_does_not_fit():
    z, top, _, _ = case()
    T = PF.TopLogits
    with pytest.raises(ValueError):
        PF.distill_loss(z, T(top.values, top.indices, None), tail=True)
    with pytest.raises(ValueError):
        PF.distill_loss(z, T(top.values, top.indices, top.lse[:3]), tail=True)
    with pytest.raises(ValueError):
        PF.distill_loss(z, T(top.values, top.indices, top.lse.double()), tail=True)
    with pytest.raises(ValueError):
        PF.distill_loss(z[:3], top)
    with pytest.raises(ValueError):
        PF.distill_loss(z, T(top.values[:, :2], top.indices, None))
    with pytest.raises(TypeError):
        PF.distill_loss(z, T(top.values.double(), top.indices, None))
    with pytest.raises(TypeError):
        PF.distill_loss(z, T(top.values, top.indices.short(), None))
    with pytest.raises(TypeError):
        PF.distill_loss(z.double(), top)
    with pytest.raises(ValueError):
        PF.distill_loss(z, T(top.values.requires_grad_(True), top.indices, None))
    with pytest.raises(ValueError):
        PF.distill_loss(torch.zeros(7, 0), top)


@pytest.mark.parametrize("z, k, kw, err", [
    (torch.zeros(2, 5), 6, {}, ValueError), (torch.zeros(2, 5), 0, {}, ValueError),
    (torch.zeros(2, 5), 1, dict(temperature=-1.0), ValueError),
    (torch.zeros(2, 5, dtype=torch.int32), 1, {}, TypeError),
    (torch.zeros(1, 2000), 1025, {}, ValueError), (torch.zeros(()), 1, {}, ValueError),
    (torch.zeros(1, (1 << 18) + 1), 1, {}, ValueError),
])
def test_top_logits_refusals(z, k, kw, err):
    with pytest.raises(err):
        PF.top_logits(z, k, **kw)


def test_gradient_of_the_rest_under_a_mask():
    """All classes but the kept one masked by the type's lowest value: the mass that the teacher leaves to
    them is shared by them alike."""
    z = torch.full((1, 300), torch.finfo(torch.float32).min)
    z[0, 5] = 1.0
    top = PF.TopLogits(torch.zeros(1, 1), torch.full((1, 1), 5, dtype=torch.int32), torch.full((1,), 0.01))
    z.requires_grad_(True)
    PF.distill_loss(z, top, tail=True).backward()
    rest = 1 - math.exp(-top.lse.item())
    want = torch.full((300,), -rest / 299, dtype=torch.float64)
    want[5] = rest                          # (q = 1 there, and p = 1 - rest)
    assert ((z.grad[0].double() - want).abs() <= 2 * HALF * want.abs()).all()


def test_gradient_of_the_rest_below_a_huge_logit():
    """The kept class at half of the type's largest number: the others share the rest by their own softmax."""
    z = torch.randn(1, 300, generator=torch.Generator().manual_seed(1))
    z[0, 5] = torch.finfo(torch.float32).max / 2
    top = PF.TopLogits(torch.zeros(1, 1), torch.full((1, 1), 5, dtype=torch.int32), torch.full((1,), 0.01))
    z.requires_grad_(True)
    PF.distill_loss(z, top, tail=True).backward()
    rest = 1 - math.exp(-top.lse.item())
    others = z.detach().double()[0]
    others[5] = -math.inf
    want = -rest * torch.softmax(others, 0)
    want[5] = rest
    assert ((z.grad[0].double() - want).abs() <= 2 * HALF * want.abs()).all()


def test_a_teachers_answer_has_no_tangent():
    from torch.autograd import forward_ad as fa

    z, top, y, _ = case()
    with fa.dual_level():
        dual = fa.make_dual(z, torch.ones_like(z) * torch.arange(z.shape[1]))
        assert fa.unpack_dual(PF.top_logits(dual, 3).values).tangent is None
        assert fa.unpack_dual(PF.top_logits(dual, 3).lse).tangent is None
        # the loss's is that of its gradient
        out = fa.unpack_dual(PF.distill_loss(dual, top, y, temperature=2.0, alpha=0.5, tail=True))
    x = z.clone().requires_grad_(True)
    PF.distill_loss(x, top, y, temperature=2.0, alpha=0.5, tail=True).backward()
    want = (x.grad.double() * torch.arange(z.shape[1])).sum().item()
    # 91 elements rounded to fp32, times 12 at most, and the sum rounded
    assert abs(out.tangent.item() - want) <= HALF * (12 * x.grad.double().abs().sum().item() + abs(want))


@pytest.mark.parametrize("t", [2.0 ** -65, 2.0 ** 65, 1e-300, 1e300, math.nan])
def test_temperatures_out_of_range(t):
    z, top, _, teacher = case()
    with pytest.raises(ValueError, match="temperature"):
        PF.top_logits(teacher, 3, t)
    with pytest.raises(ValueError, match="temperature"):
        PF.distill_loss(z, top, temperature=t)
