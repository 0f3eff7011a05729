"""The native gated_linear against its formula in 64 bits.

Tolerances. A projection's fp32 sum of n products is off by at most (n + 2) 2^-24 of the sum of their
magnitudes; the activation's exponential and quotient by 32 2^-24 relative. Through act and act'
(slopes at most 1.1) these give the error of h, dg and du; h is rounded to its type (half a step,
eps / 2), and so are dg and du in 16 bits, before the products that give dx and dW, whose own fp32
sums and last rounding come on top. All are carried through with the magnitudes of the operands.

Such a bound holds for every element, and is far above what roundings that are independent add up to.
So the 2-norm is held as well: the rounding of dg / du and of the result, each at most half a step of
its elements, are independent, and together at most sqrt(2) of one.
"""
import pytest
import torch

from pytorch_cifar_amd import nn as pnn
from pytorch_cifar_amd.nn import functional as PF

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# rows, width, hidden
SIZES = [(1, 8, 8), (1, 1, 1), (3, 5, 7), (2, 264, 40), (1, 1000, 333), (17, 96, 640), (130, 129, 131),
         (257, 64, 300), (64, 512, 1365), (5, 4096, 264), (300, 72, 1100)]
# ... for which a product is run in tiles of 192 rows: the forward, dx, dW; of 256: the forward, dx, dW,
# dW and dx in splits
LARGE = [(4100, 136, 2056), (4100, 4104, 40), (72, 2056, 4104),
         (577, 32, 8257), (6987, 1594, 32), (40, 1044, 4899), (2460, 136, 9555), (10190, 131, 2366)]


def act_of(g, act):
    """act(g) and its slope in 64 bits."""
    if act == "relu":
        return g.clamp_min(0), (g > 0).double()
    if act is None:
        return g, torch.ones_like(g)
    s = torch.sigmoid(g)
    return (g * s, s * (1 + g * (1 - s))) if act == "swish" else (s, s * (1 - s))


def inputs(m, c, f, dtype, seed=0, device="cuda", wdtype=None):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    return (n(m, c).to(dtype).to(device), (n(f, c) * c ** -0.5).to(wdtype or dtype).to(device),
            (n(f, c) * c ** -0.5).to(wdtype or dtype).to(device), n(m, f).to(dtype).to(device))


def check(x, wg, wu, dh, act, got):
    """got: h, dx, dwg, dwu (any None) against the formula in 64 bits on the GPU."""
    dtype = x.dtype
    half = torch.finfo(dtype).eps / 2
    xd, gd, ud, d = (t.double() for t in (x, wg.to(dtype), wu.to(dtype), dh))
    m, c = xd.shape
    f = gd.shape[0]
    g, u = xd @ gd.t(), xd @ ud.t()
    eg, eu = ((c + 2) * U * (xd.abs() @ w.abs().t()) for w in (gd, ud))
    a, s = act_of(g, act)
    ea = 1.1 * eg + 32 * U * a.abs()
    es = 1.1 * eg + 32 * U * (s.abs() + (s * g).abs())
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu + 4 * U * h.abs()
    want, tol = {"h": h}, {"h": eh + half * (h.abs() + eh) + tiny}
    if any(t is not None for t in got[1:]):
        dg, du = d * u * s, d * a
        rnd = half if dtype != torch.float32 else 0.0
        edg = d.abs() * (es * (u.abs() + eu) + s.abs() * eu) + 4 * U * dg.abs()
        edg = edg + rnd * (dg.abs() + edg) + tiny
        edu = d.abs() * ea + 4 * U * du.abs()
        edu = edu + rnd * (du.abs() + edu) + tiny
        want["dx"] = dg @ gd + du @ ud
        tol["dx"] = edg @ gd.abs() + edu @ ud.abs() + (2 * f + 2) * U * (dg.abs() @ gd.abs() + du.abs() @ ud.abs())
        want["dwg"], want["dwu"] = dg.t() @ xd, du.t() @ xd
        tol["dwg"] = edg.t() @ xd.abs() + (m + 2) * U * (dg.abs().t() @ xd.abs())
        tol["dwu"] = edu.t() @ xd.abs() + (m + 2) * U * (du.abs().t() @ xd.abs())
    norm = {"h": 1.0, "dx": 2 ** 0.5, "dwg": 2 ** 0.5, "dwu": 2 ** 0.5}
    for name, t in zip(("h", "dx", "dwg", "dwu"), got):
        if t is None:
            continue
        w, e = want[name], tol[name]
        out = torch.finfo(t.dtype).eps / 2
        if name != "h":
            e = e + out * (w.abs() + e) + tiny
        off = (t.double() - w).abs()
        assert t.shape == w.shape and torch.isfinite(t).all(), name
        assert (off <= e).all(), (name, (off / e).max().item())
        if dtype != torch.float32 and act != "relu":   # (relu's slope jumps: an element may be off whole)
            # what fp32 sums add to the norm is at most their share of the elements' bound
            extra = (e - half * w.abs()).clamp_min(0) if name == "h" else None
            bound = norm[name] * half * w.norm()
            bound = bound + (extra.norm() if extra is not None else 64 * max(m, c, f) * U * w.norm())
            assert (t.double() - w).norm() <= bound + tiny * w.numel() ** 0.5, name


def run(x, wg, wu, dh, act):
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    h = PF.gated_linear(*leaves, act)
    return (h.detach(), *torch.autograd.grad(h, leaves, dh))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, c, f", SIZES)
def test_forward_and_gradients(m, c, f, dtype):
    x, wg, wu, dh = inputs(m, c, f, dtype)
    got = run(x, wg, wu, dh, "swish")
    assert all(t.dtype == dtype for t in got)
    check(x, wg, wu, dh, "swish", got)
    with torch.no_grad():
        assert torch.equal(PF.gated_linear(x, wg, wu), got[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, c, f", LARGE)
def test_large_tiles(m, c, f, dtype):
    x, wg, wu, dh = inputs(m, c, f, dtype)
    check(x, wg, wu, dh, "sigmoid", run(x, wg, wu, dh, "sigmoid"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["sigmoid", "relu", "silu", None])
def test_activations(act, dtype):
    x, wg, wu, dh = inputs(70, 88, 104, dtype, 1)
    got = run(x, wg, wu, dh, act)
    if act == "relu":
        # next to a gate of zero the slope may be either: such units' gradients are left out
        g = x.double() @ wg.double().t()
        near = g.abs() <= 90 * U * (x.double().abs() @ wg.double().abs().t())
        dh = dh.masked_fill(near, 0)
        got = run(x, wg, wu, dh, act)
    check(x, wg, wu, dh, "swish" if act == "silu" else act, got)


def test_gradients_match_differences():
    x, wg, wu, w = inputs(6, 20, 12, torch.float32, 2)
    _, *grads = run(x, wg, wu, w, "swish")
    f = lambda a: ((act_of(a[0] @ a[1].t(), "swish")[0] * (a[0] @ a[2].t())) * w.double()).sum()   # noqa: E731
    base = [t.double() for t in (x, wg, wu)]
    h = 1e-4
    for i in range(3):
        d = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        fd = ((f(up) - f(down)) / (2 * h)).item()
        got = (grads[i].double() * d).sum().item()
        # h^2 times a third derivative (sums of 72 terms, below 1e4), 40 fp32 roundings of the terms
        terms = (grads[i].double().abs() * d.abs()).sum().item()
        assert abs(got - fd) <= 1e-4 + 64 * 40 * U * terms


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp32_masters(dtype):
    x, wg, wu, dh = inputs(50, 72, 56, dtype, 3, wdtype=torch.float32)
    got = run(x, wg, wu, dh, "swish")
    assert got[0].dtype == got[1].dtype == dtype and got[2].dtype == got[3].dtype == torch.float32
    check(x, wg, wu, dh, "swish", got)
    low = run(x, wg.to(dtype), wu.to(dtype), dh, "swish")
    assert torch.equal(low[0], got[0]) and torch.equal(low[1], got[1])
    assert torch.equal(low[2], got[2].to(dtype)) and torch.equal(low[3], got[3].to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    m, c, f = 33, 40, 48
    x, wg, wu, dh = inputs(m, c, f, dtype, 4)
    base = run(x, wg, wu, dh, "swish")
    packed = torch.cat([wg, wu])                       # both halves of one matrix
    wide = torch.zeros(m, 3 * c + 8, dtype=dtype, device="cuda")
    wide[:, 8:8 + c] = x
    odd = torch.zeros(m, c + 3, dtype=dtype, device="cuda")
    odd[:, 1:1 + c] = x
    every = torch.zeros(2 * m, c, dtype=dtype, device="cuda")
    every[::2] = x
    dwide = torch.zeros(m, f + 5, dtype=dtype, device="cuda")
    dwide[:, 5:] = dh
    for xv in (wide[:, 8:8 + c], odd[:, 1:1 + c], every[::2], x.t().contiguous().t()):
        for dv in (dh, dwide[:, 5:], dh.t().contiguous().t()):
            for a, b in zip(run(xv, *packed.chunk(2), dv, "swish"), base):
                assert torch.equal(a, b)
    wpad = torch.zeros(f, c + 16, dtype=dtype, device="cuda")
    wpad[:, :c] = wg
    for a, b in zip(run(x, wpad[:, :c], wu, dh, "swish"), base):
        assert torch.equal(a, b)
    one = x[:1].expand(m, c)
    check(one, wg, wu, dh, "swish", run(one, wg, wu, dh, "swish"))
    # a gradient that is one number spread out
    leaf = x.detach().requires_grad_(True)
    PF.gated_linear(leaf, wg, wu).sum().backward()
    ones = torch.ones_like(dh)
    assert torch.equal(leaf.grad, run(x, wg, wu, ones, "swish")[1])


def test_shapes_feature_maps_and_no_rows():
    x, wg, wu, dh = inputs(24, 16, 40, torch.bfloat16, 5)
    h = PF.gated_linear(x, wg, wu)
    assert torch.equal(PF.gated_linear(x.view(2, 3, 4, 16).permute(0, 3, 1, 2), wg, wu),
                       h.view(2, 3, 4, 40).permute(0, 3, 1, 2))
    assert torch.equal(PF.gated_linear(x.view(2, 12, 16), wg, wu), h.view(2, 12, 40))
    assert torch.equal(PF.gated_linear(x[0], wg, wu), PF.gated_linear(x[:1], wg, wu)[0])
    leaves = [t.requires_grad_(True) for t in (x[:0].detach(), wg, wu)]
    e = PF.gated_linear(*leaves)
    assert e.shape == (0, 40)
    dx, dwg, dwu = torch.autograd.grad(e, leaves, torch.zeros_like(e))
    assert dx.shape == (0, 16) and not dwg.any() and not dwu.any()


def test_only_some_gradients():
    x, wg, wu, dh = inputs(20, 24, 32, torch.bfloat16, 6)
    base = run(x, wg, wu, dh, "swish")
    for k in range(3):
        leaves = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, wg, wu))]
        (g,) = torch.autograd.grad(PF.gated_linear(*leaves), leaves[k], dh)
        assert torch.equal(g, base[k + 1])


def test_values_stay_in_their_rows():
    """NaN and infinity in one row, or in a weight's, reach what is computed from it alone."""
    x, wg, wu, dh = inputs(200, 64, 136, torch.bfloat16, 7)
    base = run(x, wg, wu, dh, "swish")
    bad = x.clone()
    bad[131, 5] = float("nan")
    h, dx, _, _ = run(bad, wg, wu, dh, "swish")
    keep = torch.arange(200) != 131
    assert torch.equal(h[keep], base[0][keep]) and torch.equal(dx[keep], base[1][keep])
    assert h[131].isnan().all()
    w2 = wg.clone()
    w2[70] = float("inf")
    h, _, dwg, _ = run(x, w2, wu, dh, "swish")
    cols = torch.arange(136) != 70
    assert torch.equal(h[:, cols], base[0][:, cols]) and torch.equal(dwg[cols], base[2][cols])


@pytest.mark.parametrize("act", ["swish", "relu", None])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_are_those_of_the_formula(dtype, act):
    """One infinity in a row, one in a weight, a NaN in another: the same infinities and NaN as the
    formula's, and finite values where it has them. (The rows are few enough for one sum a unit.)"""
    for m in (5, 300):
        x, wg, wu, dh = inputs(m, 64, 136, dtype, 7)
        x[3, 9] = float("inf")
        wg[20, 4] = -float("inf")
        wu[30, 5] = float("nan")
        wg[:, 9] = wg[:, 9].float().abs().clamp_min(2.0 ** -6).to(dtype)   # (a product of 1 and of 8 bits each)
        h = PF.gated_linear(x, wg, wu, act)
        g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
        want = {"swish": g * torch.sigmoid(g), "relu": torch.relu(g), None: g}[act] * u
        want = torch.where(g.isnan(), g, want)
        assert torch.equal(h.isnan(), want.isnan())
        assert torch.equal(h.double()[want.isinf()], want[want.isinf()])
        assert torch.isfinite(h[torch.isfinite(want)]).all()


def test_other_stream_and_same_bits():
    x, wg, wu, dh = inputs(100, 520, 2100, torch.bfloat16, 8)
    first = run(x, wg, wu, dh, "swish")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = run(x, wg, wu, dh, "swish")
    s.synchronize()
    for a, b, c in zip(first, second, run(x, wg, wu, dh, "swish")):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("m, c, f", [(1, 512, 264), (48, 100, 300)])
def test_captured_and_replayed(m, c, f):
    """Forward and backward in two graphs, replayed in turn over new rows with eager work between;
    each replay against the eager result, bit by bit."""
    x, wg, wu, dh = inputs(m, c, f, torch.bfloat16, 9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(x, wg, wu, dh, "swish")
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(x, wg, wu, dh, "swish")
        graphs.append((g, out))
    for i in range(6):
        nx, _, _, nd = inputs(m, c, f, torch.bfloat16, 20 + i)
        x.copy_(nx)
        dh.copy_(nd)
        want = run(x, wg, wu, dh, "swish")
        g, out = graphs[i % 2]
        g.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    m, c, f = 280000, 8192, 8
    x = torch.zeros(m, c, dtype=torch.bfloat16, device="cuda")
    tail, wg, wu, dh_tail = inputs(300, c, f, torch.bfloat16, 10)
    x[-300:] = tail
    dh = torch.zeros(m, f, dtype=torch.bfloat16, device="cuda")
    dh[-300:] = dh_tail
    h, dx, dwg, dwu = run(x, wg, wu, dh, "swish")
    check(tail, wg, wu, dh_tail, "swish", (h[-300:], dx[-300:], None, None))
    assert not h[:-300].any() and not dx[:-300].any()
    # the zero rows add nothing but their places in the sums
    half = 2.0 ** -8
    want = run(tail, wg, wu, dh_tail, "swish")
    # The small call keeps dg and du in two parts, of error below 2^-16 of them, the large one rounds
    # each once: its sums are off by at most half a step of every |dg_mf| |x_mc|, that is
    # half * |dg|^T |x|, however the terms' signs fall. (1.1: fp32's share and that of the two parts.)
    xd, gd, ud, d = (t.double() for t in (tail, wg, wu, dh_tail))
    act, slope = act_of(xd @ gd.t(), "swish")
    terms = [(d * (xd @ ud.t()) * slope).abs().t() @ xd.abs(), (d * act).abs().t() @ xd.abs()]
    for a, b, e in zip((dwg, dwu), want[2:], terms):
        # ... and two roundings of those sums: a step apart
        assert ((a.double() - b.double()).abs() <= 1.1 * half * e
                + 2 * half * b.double().abs() + 1e-3 * b.double().abs().max()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m, c, f", [(1, 96, 264), (2, 8, 1000), (7, 333, 40), (22, 24, 89), (200, 520, 1365)])
def test_small_products_round_once(m, c, f, dtype):
    """In small layers dg and du are kept in two parts: what is left of their rounding is below 2^-16
    (bf16; fp16 2^-22, or 2^-25 where the second part is subnormal) of each, and the gradients are
    off by half a step of themselves and the sums' share."""
    x, wg, wu, dh = inputs(m, c, f, dtype, 12)
    half = torch.finfo(dtype).eps / 2
    _, *grads = run(x, wg, wu, dh, "swish")
    xd, gd, ud, d = (t.double() for t in (x, wg, wu, dh))
    g, u = xd @ gd.t(), xd @ ud.t()
    a, s = act_of(g, "swish")
    dg, du = d * u * s, d * a
    # relative errors of dg and du: two parts, and fp32 projections (of c terms) through slopes below 1.1
    mag = xd.abs() @ gd.abs().t(), xd.abs() @ ud.abs().t()
    e = 1.2 * (c + 40) * U
    near = d.abs() * (e * mag[1] * (s.abs() + 0.1) + e * mag[0] * (u.abs() + 1)) + 2.0 ** -25
    eg, eu = (near + (half * half + 8 * U) * t.abs() for t in (dg, du))
    want = dg @ gd + du @ ud, dg.t() @ xd, du.t() @ xd
    off = (eg @ gd.abs() + eu @ ud.abs() + (2 * f + 2) * 2 * U * (dg.abs() @ gd.abs() + du.abs() @ ud.abs()),
           eg.t() @ xd.abs() + (m + 2) * 2 * U * (dg.abs().t() @ xd.abs()),
           eu.t() @ xd.abs() + (m + 2) * 2 * U * (du.abs().t() @ xd.abs()))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for got, w, o in zip(grads, want, off):
        assert ((got.double() - w).abs() <= half * (w.abs() + o) + o + tiny).all()


def test_module_trains_in_bf16():
    torch.manual_seed(0)
    m = pnn.GatedLinear(48, 80).cuda()
    x = torch.randn(30, 48, device="cuda").bfloat16()
    dh = torch.randn(30, 80, device="cuda").bfloat16()
    h = m(x)
    h.backward(dh)
    assert m.weight_gate.grad.dtype == torch.float32
    check(x, m.weight_gate.detach(), m.weight_up.detach(), dh, "swish",
          (h.detach(), None, m.weight_gate.grad, m.weight_up.grad))


def test_changed_weights_are_noticed():
    x, wg, wu, dh = inputs(8, 16, 16, torch.bfloat16, 11)
    wg.requires_grad_(True)
    h = PF.gated_linear(x, wg, wu)
    with torch.no_grad():
        wg.mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        h.backward(dh)


def test_second_derivatives_are_refused():
    x, wg, wu, dh = inputs(8, 16, 24, torch.bfloat16, 12)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(PF.gated_linear(x, wg, wu), x, dh, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.float().sum().backward()


def test_refusals_on_the_gpu():
    x, wg, wu, dh = inputs(8, 16, 24, torch.bfloat16, 12)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")   # noqa: E731
    for err, args in [
            (ValueError, (x, wg.cpu(), wu)), (TypeError, (x, wg.half(), wu.half())),
            (TypeError, (x, wg.float(), wu)), (ValueError, (x[:, :8], wg, wu)),
            (ValueError, (x, wg, wu[:16])), (ValueError, (x, wg[0], wu[0])),
            (ValueError, (x, wg, wu, "gelu")), (TypeError, (x.long(), wg, wu)),
            (TypeError, (x.double(), wg.double(), wu.double())), (ValueError, (x, wg[:0], wu[:0])),
            (ValueError, (z(2, 0), z(4, 0), z(4, 0))), (ValueError, (z(1, 16)[0, 0], wg, wu)),
            (ValueError, (z(1, 1).expand((1 << 30) + 1, 1), z(4, 1), z(4, 1))),
            (ValueError, (z(1, (1 << 19) + 8), z(1, (1 << 19) + 8), z(1, (1 << 19) + 8)))]:
        with pytest.raises(err):
            PF.gated_linear(*args)


@pytest.mark.parametrize("m, c, f, dtype, wdtype", [
    (4096, 2048, 5504, torch.bfloat16, None), (1021, 512, 1365, torch.float32, None),
    (300, 1028, 2056, torch.float16, None), (37, 1000, 2003, torch.bfloat16, torch.float32)])
def test_same_bits_whatever_the_memory_held(m, c, f, dtype, wdtype):
    """Every output, workspace and padded copy is written before it is read: the same bits after memory
    full of NaN, of ones and of zeros."""
    x, wg, wu, dh = inputs(m, c, f, dtype, 13, wdtype=wdtype)
    first = None
    for value in (float("nan"), 1.0, 0.0):
        torch.cuda.empty_cache()
        held = [torch.full((n,), value, device="cuda") for n in (1 << 28, 1 << 26, 1 << 24, 1 << 18)]
        del held                      # (kept by the allocator: what follows is cut out of it)
        got = run(x, wg, wu, dh, "swish")
        first = got if first is None else first
        for a, b in zip(got, first):
            assert torch.equal(a, b)
    check(x, wg, wu, dh, "swish", first)


@pytest.mark.parametrize("act", ["swish", "sigmoid", "relu", None])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_of_the_gradients_are_those_of_the_formula(dtype, act):
    """One infinity in a row, a weight or an incoming gradient: the gradients' infinities and NaN are
    the formula's, and finite values stay finite."""
    for where in ("x", "wg", "wu", "dh", "wg of a zero"):
        for m in (5, 300):
            x, wg, wu, dh = inputs(m, 64, 136, dtype, 7)
            # away from zero, so that no rounding makes one (0 times an infinity is NaN)
            x, wg, wu, dh = (t.sign() * (t.abs() + 2.0 ** -3) for t in (x, wg, wu, dh))
            {"x": x, "wg": wg, "wu": wu, "dh": dh, "wg of a zero": wg}[where][3, 9] = float("inf")
            if where == "wg of a zero":
                x[1, 9] = 0.0
                if act == "relu":
                    continue          # (a gate of NaN has no side)
            got = run(x, wg, wu, dh, act)
            xd, gd, ud, d = (t.double().cpu() for t in (x, wg, wu, dh))
            g, u = xd @ gd.t(), xd @ ud.t()
            a, s = act_of(g, act)
            dg, du = d * u * s, d * a
            want = (a * u, dg @ gd + du @ ud, dg.t() @ xd, du.t() @ xd)
            for name, t, w in zip(("h", "dx", "dwg", "dwu"), got, want):
                t = t.double().cpu()
                assert torch.equal(t.isnan(), w.isnan()), (where, m, name)
                assert torch.equal(t[w.isinf()], w[w.isinf()]), (where, m, name)
                assert torch.isfinite(t[torch.isfinite(w)]).all(), (where, m, name)


@pytest.mark.parametrize("c", [1, 2, 3])
@pytest.mark.parametrize("bits", [0x3f80ffff, 0x3f80feff, 0x3fff7f7f, 0x3f808080, 0x3f817fff, 0x3fffffff])
def test_fp32_products_of_three_parts(bits, c):
    """fp32 products are six of their operands' three bf16 parts. A projection of c equal terms: what is
    left out is 2^-24 of each, the fp32 sum of the largest parts' products rounds c times by a step at
    most, and the smaller parts' (2^-7 of them) sums by 2^-6 together; h is their product, rounded once."""
    v = torch.tensor(bits, dtype=torch.int32).view(torch.float32).item()
    for s in (1.0, -1.0):
        x = torch.full((70, c), v, device="cuda")
        wg, wu = torch.full((40, c), v, device="cuda"), torch.full((40, c), s * v, device="cuda")
        h = PF.gated_linear(x, wg, wu, None)
        want = s * (c * v * v) ** 2
        step = 2 * (1 + 2 * c + 2.0 ** -4) + 1
        assert ((h.double() - want).abs() <= step * U * abs(want)).all(), ((h.double() / want - 1).abs().max() / U)


def test_fp32_operands_that_bf16_does_not_hold():
    """Finite numbers that round to infinity in bf16."""
    big = torch.finfo(torch.float32).max
    x, wg, wu, dh = inputs(80, 24, 40, torch.float32, 14)
    x[3, 5], x[4] = big, 0.0
    wg[:, 5] = wg[:, 5].sign() * 2.0 ** -120
    wu[:, 5] = 0.0
    x[4, 2], wg[7, 2], wg[8] = -big, 1.0, 0.0
    wu[:, 2] = 2.0 ** -100
    wg[8, 2] = 2.0 ** -100
    h = PF.gated_linear(x, wg, wu, None)
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    want = g * u
    mag = (x.double().abs() @ wg.double().abs().t()) * u.abs() + g.abs() * (x.double().abs() @ wu.double().abs().t())
    fine = want.abs() < 2.0 ** 127
    assert ((h.double() - want).abs() <= 64 * U * mag)[fine].all()
    assert h.isnan().sum() == 0


def test_rows_of_four_dimensions():
    x, wg, wu, dh = inputs(24, 16, 40, torch.bfloat16, 15)
    base = run(x, wg, wu, dh, "swish")
    for shape in ((2, 3, 4), (1, 16, 1), (2, 12, 1)):
        n = shape[0] * shape[1] * shape[2]
        leaves = [t.detach().requires_grad_(True) for t in (x[:n].view(*shape, 16), wg, wu)]
        h = PF.gated_linear(*leaves, dim=-1)
        (dx,) = torch.autograd.grad(h, leaves[:1], dh[:n].view(*shape, 40))
        assert torch.equal(h.view(n, 40), base[0][:n]) and torch.equal(dx.view(n, 16), base[1][:n])
        with pytest.raises(ValueError, match="dim"):
            PF.gated_linear(*leaves)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad as fa

    args = inputs(8, 16, 24, torch.bfloat16, 16)[:3]
    with fa.dual_level():
        for i in range(3):
            for leaf in (args[i], args[i].clone().requires_grad_(True)):
                mixed = list(args)
                mixed[i] = fa.make_dual(leaf, torch.ones_like(leaf))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    PF.gated_linear(*mixed)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: PF.gated_linear(x, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
