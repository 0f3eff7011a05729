"""gated_linear on the CPU reference path, its module, and its refusals.

Tolerances: the path computes in fp32 here; a sum of n products is off by at most (n + 1) 2^-24 of the
sum of their magnitudes, and the activation and the product add a few roundings of the result.
"""
import pytest
import torch

from pytorch_cifar_amd import nn as pnn
from pytorch_cifar_amd.nn import functional as PF

U = 2.0 ** -24
ACTS = {"swish": lambda x: x * torch.sigmoid(x), "sigmoid": torch.sigmoid, "relu": torch.relu,
        None: lambda x: x}


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("lead", [(), (3,), (2, 5), (0,)])
def test_matches_the_formula(act, lead):
    torch.manual_seed(0)
    x, wg, wu = torch.randn(*lead, 7), torch.randn(9, 7), torch.randn(9, 7)
    h = PF.gated_linear(x, wg, wu, act)
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    want = ACTS[act](g) * u
    dg, du = ((x.double().abs() @ w.double().abs().t()) * 8 * U for w in (wg, wu))
    # |act'| <= 1.1
    tol = 1.1 * dg * u.abs() + ACTS[act](g).abs() * du + dg * du + 8 * U * want.abs()
    assert h.shape == (*lead, 9) and ((h.double() - want).abs() <= tol).all()


def test_feature_maps_are_rows_of_pixels():
    torch.manual_seed(0)
    x, wg, wu = torch.randn(2, 7, 3, 4), torch.randn(5, 7), torch.randn(5, 7)
    y = PF.gated_linear(x, wg, wu)
    assert y.shape == (2, 5, 3, 4)
    rows = PF.gated_linear(x.permute(0, 2, 3, 1).reshape(-1, 7), wg, wu)
    assert torch.allclose(y.permute(0, 2, 3, 1).reshape(-1, 5), rows, rtol=8 * U, atol=64 * U)


def test_gradients_match_differences():
    torch.manual_seed(0)
    for act in ("swish", "sigmoid", None):
        x, wg, wu = (torch.randn(*s, dtype=torch.float64) for s in ((4, 6), (5, 6), (5, 6)))
        f = lambda x, wg, wu: ACTS[act](x @ wg.t()) * (x @ wu.t())   # noqa: E731
        h = 1e-3
        leaves = [t.float().requires_grad_(True) for t in (x, wg, wu)]
        w = torch.randn(4, 5)
        grads = torch.autograd.grad((PF.gated_linear(*leaves, act) * w).sum(), leaves)
        for i, t in enumerate((x, wg, wu)):
            d = torch.randn_like(t)
            args = [[x, wg, wu], [x, wg, wu]]
            args[0][i], args[1][i] = t + h * d, t - h * d
            fd = ((f(*args[0]) - f(*args[1])) * w).sum() / (2 * h)
            got = (grads[i].double() * d).sum()
            # h^2 times a third derivative (below 1e3 here), and 40 fp32 roundings of terms below 1e2
            assert abs(got - fd) <= 1e-3 + 40 * 100 * U


def test_module():
    torch.manual_seed(0)
    m = pnn.GatedLinear(6, 11, act="sigmoid")
    assert sorted(m.state_dict()) == ["weight_gate", "weight_up"]
    assert m.weight_gate.shape == (11, 6) and m.weight_gate.abs().max() <= 6 ** -0.5
    x = torch.randn(3, 6)
    assert torch.equal(m(x), PF.gated_linear(x, m.weight_gate, m.weight_up, "sigmoid"))
    m(x).sum().backward()
    assert m.weight_gate.grad.shape == (11, 6) and m.weight_up.grad.abs().sum() > 0
    assert m(x.bfloat16()).dtype == torch.bfloat16


W = torch.zeros(9, 7)


@pytest.mark.parametrize("args, err", [
    ((torch.zeros(2, 6), W, W), ValueError), ((torch.zeros(2, 7), W, W[:8]), ValueError),
    ((torch.zeros(2, 7), W[0], W[0]), ValueError), ((torch.zeros(2, 7), W, W, "gelu"), ValueError),
    ((torch.zeros(2, 7).long(), W, W), TypeError), ((torch.zeros(2, 7), W.double(), W.double()), TypeError),
    ((torch.zeros(2, 7), W, W.bfloat16()), TypeError),
    ((torch.zeros(2, 7), W.bfloat16(), W.bfloat16()), TypeError),
    ((torch.zeros(2, 0), W[:, :0], W[:, :0]), ValueError), ((torch.zeros(()), W, W), ValueError),
    ((torch.zeros(2, 7), W[:0], W[:0]), ValueError), ((torch.zeros(2, 7, 3, 6), W[:, :6], W[:, :6]), ValueError),
])
def test_refusals(args, err):
    with pytest.raises(err):
        PF.gated_linear(*args)


def test_rows_of_four_dimensions():
    """[batch, heads, tokens, width] beside feature maps: `dim` says which, and nothing is guessed."""
    torch.manual_seed(0)
    wg, wu = torch.randn(5, 7), torch.randn(5, 7)

    def check(h, rows):
        g, u = rows.double() @ wg.double().t(), rows.double() @ wu.double().t()
        dg, du = ((rows.double().abs() @ w.double().abs().t()) * 8 * U for w in (wg, wu))
        a = ACTS["swish"](g)
        tol = 1.1 * dg * u.abs() + a.abs() * du + dg * du + 8 * U * (a * u).abs()
        assert h.shape == (*rows.shape[:-1], 5) and ((h.double() - a * u).abs() <= tol).all()

    for shape in ((2, 3, 4, 7), (2, 7, 3, 7)):
        x = torch.randn(*shape)
        check(PF.gated_linear(x, wg, wu, dim=-1), x)
        m = pnn.GatedLinear(7, 5, dim=-1)
        m.load_state_dict({"weight_gate": wg, "weight_up": wu})
        check(m(x).detach(), x)
        assert "dim=-1" in repr(m)
        with pytest.raises(ValueError, match="dim"):
            PF.gated_linear(x, wg, wu)
    for x in (torch.randn(2, 7, 3, 7), torch.randn(2, 7, 3, 4)):
        check(PF.gated_linear(x, wg, wu, dim=1).permute(0, 2, 3, 1), x.permute(0, 2, 3, 1))
    for dim, x in ((0, x), (3, x), (1, x[0]), (1, torch.randn(2, 3, 4, 7))):
        with pytest.raises(ValueError):
            PF.gated_linear(x, wg, wu, dim=dim)
