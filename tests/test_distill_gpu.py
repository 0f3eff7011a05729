"""The native top_logits / distill_loss kernels against the 64-bit reference path on the CPU.

Tolerances. e_j = exp((z_j - max)/T) has a relative error of at most (3 x + 4) 2^-24, x = |z_j -
max| / T: one rounding each of the difference, of log2(e)/T and of the product, each worth x 2^-24
in the exponent, and 2 steps of the exponential instruction. A sum adds one rounding a term that a
thread holds (at most 256). With x at most X, the row's spread, a sum or a share of it is off by
at most C = (3 X + 260) 2^-24 relative, the logarithm of a sum by C absolute. The loss holds two
such logarithms times alpha T^2 and one times 1 - alpha; a gradient element holds shares of them
times alpha T and 1 - alpha, and is then rounded to its type: half a step, eps / 2 (in fp16 at least
half of its smallest number, 2^-25).
"""
import math

import pytest
import torch

from pytorch_cifar_amd.nn import functional as PF
from pytorch_cifar_amd.ops.distill import _ref_distill

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = [(3, 1, 1), (1024, 10, 5), (5, 64, 64), (4, 65, 3), (7, 513, 100), (9, 2047, 512),
         (5, 4097, 17), (3, 8200, 1024), (4, 33001, 256), (2, 50257, 64), (3, 65540, 5),
         (2, 131072, 64), (2, 262144, 1000)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(r, v, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(r, v, generator=g)).to(dtype)


def spread(z, t):
    z = z.double()
    f = torch.where(torch.isfinite(z), z, torch.zeros_like(z))
    return ((f.amax() - f.amin()) / min(t, 1.0)).item()


def check_top(z, k, t=1.0, gpu=None):
    want = PF.top_logits(z, k, t)
    got = PF.top_logits(z.cuda() if gpu is None else gpu, k, t)
    assert got.indices.dtype == torch.int32 and got.values.dtype == z.dtype
    assert torch.equal(got.indices.cpu(), want.indices)
    a, b = got.values.cpu(), want.values
    assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) and torch.equal(a.isnan(), b.isnan())
    c = (3 * spread(z, t) + 260) * U
    lse, ref = got.lse.cpu().double(), torch.logsumexp(z.double() / t, -1)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.nan_to_num(lse[~fine]), torch.nan_to_num(ref[~fine]))
    assert ((lse - ref)[fine].abs() <= c + U * ref[fine].abs()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r, v, k", SIZES)
def test_top_logits(r, v, k, dtype):
    check_top(make(r, v, dtype), k, 2.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [6, 300, 5000, 40000, 200000])
def test_top_logits_hard_rows(v, dtype):
    k = min(v, 200)
    z = make(15, v, dtype, 1)
    z[12, :2 * v // 3] = -math.inf
    z[13, :v // 3] = torch.finfo(dtype).min
    z[14] = -torch.arange(v).to(dtype)
    z[0] = -math.inf
    z[1] = 1.0                                    # all equal
    z[2] = torch.randint(0, 3, (v,)).to(dtype)    # few values
    z[3, v // 2:] = -math.inf
    z[4, v // 3] = math.nan
    z[5, 1] = math.inf
    z[6] = torch.finfo(dtype).min
    z[7, 3:] = torch.finfo(dtype).min
    z[8] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0).to(dtype)
    z[9] = torch.arange(v).to(dtype)
    z[10] = math.nan
    z[11] = -math.inf
    z[11, v - 1] = 2.0
    top = PF.top_logits(z.cuda(), k)
    want = PF.top_logits(z, k)
    assert torch.equal(top.indices.cpu(), want.indices)
    check_top(z[[0, 1, 2, 3, 5, 8, 11, 12]], k)
    lse = top.lse.cpu()
    assert lse[0] == -math.inf and lse[5] == math.inf
    assert lse[4].isnan() and lse[10].isnan()
    assert abs(lse[11].item() - 2.0) <= 300 * U


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [130, 500, 2048, 2500, 4000, 8100, 9000, 33000])
@pytest.mark.parametrize("k", [1, 24, 33, 65, 100, 129, 160, 257, 500, 800, 1024])
def test_top_logits_on_both_sides_of_each_rule(v, k, dtype):
    """Bounds by threads' maxima, by chunks', by counting; few threads and many; places counted and
    searched; rows in random order, ascending, descending, masked at one end, of few values."""
    z = make(7, v, dtype, 6)
    z[1] = z[1].sort()[0]
    z[2] = z[2].sort(descending=True)[0]
    z[3, v // 3:] = -math.inf
    z[4, :v // 2] = torch.finfo(dtype).min
    z[5] = z[5].round()
    z[6, v // 2] = math.nan
    check_top(z, min(k, v))


def test_top_logits_strided_rows():
    buf = make(9, 1003, torch.bfloat16).cuda()
    for view in (buf[:, 1:778], buf[::2, 3:500], buf[:, :1], buf[2:3].expand(4, 1003), buf.t()):
        check_top(view.cpu(), min(view.shape[1], 9), gpu=view)


def distill_inputs(r, v, k, dtype, t, seed=3, labels=True):
    teacher = make(r, v, dtype, seed)
    z = (0.6 * teacher.float() + make(r, v, torch.float32, seed + 1, 1.5)).to(dtype)
    top = PF.top_logits(teacher, k, t)
    y = torch.randint(0, v, (r,), generator=torch.Generator().manual_seed(seed))
    return z, top, (y if labels else None)


def oracle(z, top, y, t, alpha, tail, seeds=None):
    """Rows' losses and the gradient of (seeds . losses) in 64 bits."""
    x = z.detach().cpu().double().requires_grad_(True)
    c = [a.cpu() if a is not None else None for a in (top.values, top.indices, top.lse, y)]
    loss = _ref_distill(x, *c, t, alpha, tail, -100)
    w = torch.ones_like(loss) if seeds is None else seeds.double().cpu()
    (g,) = torch.autograd.grad((loss * w).sum(), x)
    return loss.detach(), g


def tolerances(z, t, alpha, grad, seeds=1.0):
    z = z.detach().cpu().double()
    c = (3 * spread(z, t) + 260) * U
    loss = 2 * c * (alpha * t * t + 1 - alpha)
    q = alpha * t * torch.softmax(z / t, 1) + (1 - alpha) * torch.softmax(z, 1)
    return loss, lambda dtype: (2 * c * (q.nan_to_num() + grad.abs()) * seeds
                                + torch.finfo(dtype).eps / 2 * grad.abs()
                                + (2.0 ** -25 if dtype == torch.float16 else 1e-37))


def gpu_top(top):
    return PF.TopLogits(*(a.cuda() if a is not None else None for a in top))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r, v, k", SIZES)
@pytest.mark.parametrize("tail, labels, t", [(False, True, 4.0), (True, True, 1.0), (True, False, 2.0)])
def test_distill(r, v, k, dtype, tail, labels, t):
    alpha = 0.7 if labels else 1.0
    z, top, y = distill_inputs(r, v, k, dtype, t, labels=labels)
    if r > 2:
        top.indices[0, k // 2:] = -1
        top.indices[2] = -1
        if labels:
            y[1] = -100
            y[2] = -100
    if k > 2:
        top.indices[1, 2] = top.indices[1, 0]      # a class twice
    want, grad = oracle(z, top, y, t, alpha, tail)
    tl, tg = tolerances(z, t, alpha, grad)
    x = z.cuda().requires_grad_(True)
    kw = dict(temperature=t, alpha=alpha, tail=tail)
    args = (gpu_top(top), y.cuda() if labels else None)
    rows = PF.distill_loss(x.detach(), *args, reduction="none", **kw)
    assert ((rows.cpu().double() - want).abs() <= tl + 2 * U * want.abs()).all()
    loss = PF.distill_loss(x, *args, reduction="sum", **kw)
    loss.backward(PF.unit_grad(loss))
    # (the pass with a gradient may sum a row in another order than the one without: each row of it is
    # held to the oracle's by the same bound, and their sum by the bounds' sum and its own rounding)
    assert abs(loss.item() - want.sum().item()) <= r * tl + 3 * U * want.abs().sum().item()
    assert x.grad.dtype == dtype
    assert ((x.grad.cpu().double() - grad).abs() <= tg(dtype)).all()
    if r > 2 and labels:
        assert (x.grad[2] == 0).all() and rows[2] == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_reductions_and_seeds(dtype):
    r, v, k, t = 6, 777, 9, 2.0
    z, top, y = distill_inputs(r, v, k, dtype, t)
    seeds = torch.tensor([1.0, 0.0, -2.5, 0.125, 1.0, 3.0])
    kw = dict(temperature=t, alpha=0.5, tail=True)
    args = (gpu_top(top), y.cuda())
    x = z.cuda().requires_grad_(True)
    _, grad = oracle(z, top, y, t, 0.5, True, seeds)
    _, tg = tolerances(z, t, 0.5, grad, 1 + seeds.abs()[:, None].double())
    loss = PF.distill_loss(x, *args, reduction="none", **kw)
    (g,) = torch.autograd.grad(loss, x, seeds.cuda())
    # (the factor is applied to a gradient that was rounded before: a second half step)
    half = torch.finfo(dtype).eps / 2
    extra = half * grad.abs() + (2.0 ** -23 if dtype == torch.float16 else 0)
    assert ((g.cpu().double() - grad).abs() <= tg(dtype) + extra).all()
    # the mean, by another seed, twice over a retained graph
    _, one = oracle(z, top, y, t, 0.5, True, torch.full((r,), 3.0 / r))
    _, tg = tolerances(z, t, 0.5, one)
    loss = PF.distill_loss(x, *args, **kw)
    seed = torch.tensor(3.0, device="cuda")
    a = torch.autograd.grad(loss, x, seed, retain_graph=True)[0]
    a0 = a.clone()
    a.add_(1.0)                       # what a caller does to its gradient is its own affair
    b = torch.autograd.grad(loss, x, seed)[0]
    assert torch.equal(a0, b)
    extra = half * one.abs() + (2.0 ** -23 if dtype == torch.float16 else 0)
    assert ((b.cpu().double() - one).abs() <= tg(dtype) + extra).all()


def test_gradient_matches_differences():
    z, top, y = distill_inputs(3, 40, 7, torch.float32, 2.0)
    kw = dict(temperature=2.0, alpha=0.6, tail=True, reduction="sum")
    x = z.cuda().requires_grad_(True)
    PF.distill_loss(x, gpu_top(top), y.cuda(), **kw).backward()
    ref = lambda d: _ref_distill(d, *top, y, 2.0, 0.6, True, -100).sum().item()   # noqa: E731
    h = 1e-4
    c = (3 * spread(z, 2.0) + 260) * U
    for i in range(3):
        for j in range(0, 40, 3):
            d = torch.zeros(3, 40, dtype=torch.float64)
            d[i, j] = h
            fd = (ref(z.double() + d) - ref(z.double() - d)) / (2 * h)
            # h^2 / 6 times a third derivative below 1, and the kernel's own C
            assert abs(x.grad[i, j].item() - fd) <= h * h + 8 * c


def test_strides_types_and_shapes():
    z, top, y = distill_inputs(12, 515, 20, torch.float32, 1.0)
    big = torch.full((12, 1031), math.nan)
    big[:, 3:518] = z
    big = big.cuda()
    kw = dict(alpha=0.5, tail=True, reduction="none")
    base = PF.distill_loss(z.cuda(), gpu_top(top), y.cuda(), **kw)
    assert torch.equal(PF.distill_loss(big[:, 3:518], gpu_top(top), y.cuda(), **kw), base)
    assert torch.equal(PF.distill_loss(z.cuda().t().contiguous().t(), gpu_top(top), y.cuda(), **kw), base)
    T = PF.TopLogits
    g = gpu_top(top)
    assert torch.equal(PF.distill_loss(z.cuda(), T(g.values, g.indices.long(), g.lse), y.cuda(), **kw), base)
    wide = torch.cat([g.values, g.values], 1)[:, :20]
    assert torch.equal(PF.distill_loss(z.cuda(), T(wide, g.indices, g.lse), y.cuda(), **kw), base)
    half = T(g.values.bfloat16(), g.indices, g.lse)
    same = T(half.values.float(), g.indices, g.lse)
    assert torch.equal(PF.distill_loss(z.cuda(), half, y.cuda(), **kw),
                       PF.distill_loss(z.cuda(), same, y.cuda(), **kw))
    nd = PF.distill_loss(z.cuda().view(3, 4, 515), T(g.values.view(3, 4, 20), g.indices.view(3, 4, 20),
                                                     g.lse.view(3, 4)), y.cuda().view(3, 4), **kw)
    assert torch.equal(nd, base.view(3, 4))
    x = big.clone().requires_grad_(True)
    PF.distill_loss(x[:, 3:518], g, y.cuda(), alpha=0.5, tail=True).backward()
    assert (x.grad[:, :3] == 0).all() and (x.grad[:, 518:] == 0).all()
    assert torch.isfinite(x.grad).all() and (x.grad[:, 3:518] != 0).any()


def test_masked_classes_and_empty_rows():
    """Classes masked by -inf or the type's lowest value; rows without terms may hold anything."""
    for dtype in DTYPES:
        z, top, y = distill_inputs(8, 300, 6, dtype, 1.0)
        teacher = make(8, 300, dtype, 3)
        teacher[:, 200:] = -math.inf
        top = PF.top_logits(teacher, 6)
        y = top.indices[:, 1].long()
        low = torch.finfo(dtype).min
        z[0, 200:] = -math.inf
        z[1, 200:] = low
        z[2] = math.nan
        top.indices[2], y[2] = -1, -100
        z[3] = -math.inf
        top.indices[3], y[3] = -1, -100
        z[4] = low                                    # uniform
        top.values[5] = -math.inf                     # a teacher's row of no mass
        top.lse[5] = -math.inf
        y[5] = -100
        z[6, 7] = math.nan
        rows = {}
        for tail in (False, True):
            x = z.cuda().requires_grad_(True)
            loss = PF.distill_loss(x, gpu_top(top), y.cuda(), alpha=0.5, tail=tail, reduction="none")
            loss.backward(torch.ones_like(loss))
            want, grad = oracle(z, top, y, 1.0, 0.5, tail)
            keep = [0, 1, 4, 7]
            tl, tg = tolerances(z[[0, 7]], 1.0, 0.5, grad[[0, 7]])
            assert ((loss.cpu().double() - want).abs()[keep] <= tl + 2 * U * want.abs()[keep]).all()
            assert ((x.grad.cpu().double() - grad).abs()[[0, 7]] <= tg(dtype)).all()
            # a row of one value has q = 1/300 everywhere: shares without rounding of a spread
            assert ((x.grad.cpu().double() - grad).abs()[4] <= torch.finfo(dtype).eps
                    * (grad[4].abs() + 1 / 300) + 2.0 ** -25).all()
            assert (x.grad[1, 200:] == 0).all()
            for i in (2, 3, 5):
                assert loss[i] == 0 and (x.grad[i] == 0).all()
            assert loss[6].isnan()
            rows[tail] = loss.detach()
        assert torch.isfinite(rows[False][keep]).all()


def test_bad_classes_poison_their_row():
    z, top, y = distill_inputs(4, 50, 3, torch.float32, 1.0)
    top.indices[1, 0], y[2], y[3] = 50, 50, -7
    x = z.cuda().requires_grad_(True)
    loss = PF.distill_loss(x, gpu_top(top), y.cuda(), alpha=0.5, reduction="none")
    loss.backward(torch.ones_like(loss))
    assert loss.isnan().tolist() == [False, True, True, True]
    assert x.grad.isnan().all(1).tolist() == [False, True, True, True]


def test_debug_mode_names_a_bad_class():
    import pytorch_cifar_amd as pca

    z, top, y = distill_inputs(4, 50, 3, torch.float32, 1.0)
    top.indices[1, 2] = 50
    pca.set_debug_sync(True)
    try:
        with pytest.raises(IndexError, match="50"):
            PF.distill_loss(z.cuda(), gpu_top(top))
    finally:
        pca.set_debug_sync(False)


def test_no_rows():
    top = PF.top_logits(torch.zeros(0, 33, device="cuda"), 4)
    assert top.values.shape == (0, 4)
    x = torch.zeros(0, 33, device="cuda", requires_grad=True)
    loss = PF.distill_loss(x, top, reduction="sum")
    loss.backward()
    assert loss.item() == 0 and x.grad.shape == (0, 33)
    assert PF.distill_loss(x, top).isnan()


def test_other_stream_and_same_bits():
    z, top, y = distill_inputs(64, 5003, 50, torch.bfloat16, 2.0)
    x, g, yc = z.cuda().requires_grad_(True), gpu_top(top), y.cuda()
    torch.cuda.synchronize()

    def both():
        loss = PF.distill_loss(x, g, yc, temperature=2.0, alpha=0.5, tail=True)
        return (loss.detach(), *torch.autograd.grad(loss, x), *PF.top_logits(x, 50, 2.0))

    first = both()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = both()
    s.synchronize()
    third = both()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_and_replayed():
    """The teacher's selection, the loss and its gradient in one graph, replayed over new logits with
    eager work between; each replay against the eager result, bit by bit."""
    dev = "cuda"
    t = torch.empty(32, 1000, device=dev)
    z = torch.empty(32, 1000, device=dev)
    y = torch.empty(32, dtype=torch.int64, device=dev)

    def fill(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        t.copy_(3 * torch.randn(32, 1000, generator=g, device=dev))
        z.copy_(2 * torch.randn(32, 1000, generator=g, device=dev))
        y.copy_(torch.randint(0, 1000, (32,), generator=g, device=dev))

    def step():
        x = z.detach().requires_grad_(True)
        loss = PF.distill_loss(x, PF.top_logits(t, 20, 2.0), y, temperature=2.0, alpha=0.5, tail=True)
        (d,) = torch.autograd.grad(loss, x, PF.unit_grad(loss))
        return loss.detach(), d

    fill(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for i in range(6):
        fill(10 + i)
        want = step()
        gr, out = graphs[i % 2]
        gr.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    r, v, k = 17000, 131072, 3
    z = torch.zeros(r, v, dtype=torch.bfloat16, device="cuda")
    z[-1] = make(1, v, torch.bfloat16).cuda()[0]
    top = PF.top_logits(z, k)
    want = PF.top_logits(z[-1:].cpu(), k)
    assert torch.equal(top.indices[-1:].cpu(), want.indices)
    assert top.indices[:-1].cpu().tolist() == [[0, 1, 2]] * (r - 1)
    x = z.requires_grad_(True)
    loss = PF.distill_loss(x, top, reduction="sum")
    (d,) = torch.autograd.grad(loss, x)
    last = x.detach()[-1:].cpu()
    _, grad = oracle(last, want, None, 1.0, 1.0, False)
    _, tg = tolerances(last, 1.0, 1.0, grad)
    assert ((d[-1:].cpu().double() - grad).abs() <= tg(torch.bfloat16)).all()
    assert torch.equal(d[0], d[-2])


@pytest.mark.parametrize("r, v", [((1 << 26) + 5, 2), ((1 << 21) + 3, 70)])
def test_more_rows_than_a_launch_holds(r, v):
    """A launch has less than 2^32 threads: rows on both sides of its parts, against small calls."""
    g = torch.Generator(device="cuda").manual_seed(5)
    z = torch.randn(r, v, generator=g, device="cuda", dtype=torch.bfloat16)
    y = torch.randint(0, v, (r,), generator=g, device="cuda")
    top = PF.top_logits(z, 1, 2.0)

    def run(z, top, y):
        x = z.detach().requires_grad_(True)
        loss = PF.distill_loss(x, top, y, temperature=2.0, alpha=0.5, tail=True, reduction="none")
        (d,) = torch.autograd.grad(loss, x, torch.full_like(loss, 3.0))
        return loss.detach(), d

    loss, d = run(z, top, y)
    for at in (0, (1 << 21) - 4, r - 8):
        rows = slice(at, at + 8)
        t = PF.top_logits(z[rows], 1, 2.0)
        assert all(torch.equal(a[rows], b) for a, b in zip(top, t))
        want = run(z[rows], t, y[rows])
        assert torch.equal(loss[rows], want[0]) and torch.equal(d[rows], want[1])


def test_backward_in_a_graph_of_its_own():
    """Forward and backward captured apart: replays of the backward alone, each with its own seed."""
    z, top, y = distill_inputs(32, 1000, 20, torch.float32, 2.0)
    z, top, y = z.cuda(), gpu_top(top), y.cuda()
    seed = torch.ones(32, device="cuda")
    args = dict(temperature=2.0, alpha=0.5, reduction="none")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = z.detach().requires_grad_(True)
        torch.autograd.grad(PF.distill_loss(x, top, y, **args), x, seed)
        del x
    torch.cuda.current_stream().wait_stream(s)
    x = z.detach().requires_grad_(True)
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=s):
        loss = PF.distill_loss(x, top, y, **args)
    with torch.cuda.graph(backward, pool=forward.pool(), stream=s):
        (d,) = torch.autograd.grad(loss, x, seed)
    for i in range(3):
        forward.replay()
        for scale in (1.0, 3.0, 0.5):
            seed.fill_(scale)
            backward.replay()
            w = z.detach().requires_grad_(True)
            (want,) = torch.autograd.grad(PF.distill_loss(w, top, y, **args), w, seed)
            assert torch.equal(d, want)
        z.add_(0.25 * i)


def test_refusals_on_the_gpu():
    z, top, y = distill_inputs(4, 50, 3, torch.float32, 1.0)
    g = gpu_top(top)
    with pytest.raises(ValueError):
        PF.distill_loss(z.cuda(), top)                       # the teacher's side on the host
    with pytest.raises(ValueError):
        PF.distill_loss(z.cuda(), g, y, alpha=0.5)
    with pytest.raises(ValueError):
        PF.top_logits(z.cuda(), 51)
    from pytorch_cifar_amd import _native

    with pytest.raises(ValueError):
        _native.lib().top_logits(z, 1, 1.0)


def test_second_derivatives_are_refused():
    z, top, y = distill_inputs(4, 50, 3, torch.float32, 1.0)
    x = z.cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(PF.distill_loss(x, gpu_top(top)), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


def test_changed_logits_are_noticed():
    z, top, y = distill_inputs(4, 50, 3, torch.float32, 1.0)
    x = z.cuda().requires_grad_(True)
    w = x * 1.0
    loss = PF.distill_loss(w, gpu_top(top))
    w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


@pytest.mark.parametrize("kw, err", [
    (dict(temperature=0.0), ValueError), (dict(temperature=math.inf), ValueError),
    (dict(alpha=1.5), ValueError), (dict(alpha=0.5), ValueError), (dict(reduction="max"), ValueError),
    (dict(target=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(target=torch.zeros(4, dtype=torch.int32), alpha=0.5), ValueError),
    (dict(target=torch.zeros(3, dtype=torch.int64), alpha=0.5), ValueError),
])
def test_argument_refusals(kw, err):
    z, top, _ = distill_inputs(4, 50, 3, torch.float32, 1.0)
    kw = {k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()}
    with pytest.raises(err):
        PF.distill_loss(z.cuda(), gpu_top(top), **kw)


def test_refuses_what_does_not_fit():
    z, top, _ = distill_inputs(7, 50, 5, torch.float32, 1.0)
    z, top, T = z.cuda(), gpu_top(top), PF.TopLogits
    for err, args, kw in [
            (ValueError, (z, T(top.values, top.indices, None)), dict(tail=True)),
            (ValueError, (z, T(top.values, top.indices, top.lse[:3])), dict(tail=True)),
            (ValueError, (z, T(top.values, top.indices, top.lse.double())), dict(tail=True)),
            (ValueError, (z[:3], top), {}),
            (ValueError, (z, T(top.values[:, :2], top.indices, None)), {}),
            (TypeError, (z, T(top.values.double(), top.indices, None)), {}),
            (TypeError, (z, T(top.values, top.indices.short(), None)), {}),
            (TypeError, (z.double(), top), {}),
            (ValueError, (z, T(top.values.clone().requires_grad_(True), top.indices, None)), {}),
            (ValueError, (torch.zeros(7, 0, device="cuda"), top), {})]:
        with pytest.raises(err):
            PF.distill_loss(*args, **kw)
    for err, args, kw in [
            (ValueError, (z, 51), {}), (ValueError, (z, 0), {}), (ValueError, (z, 1), dict(temperature=-1.0)),
            (TypeError, (z.int(), 1), {}), (ValueError, (torch.zeros(1, 2000, device="cuda"), 1025), {}),
            (ValueError, (torch.zeros((), device="cuda"), 1), {}),
            (ValueError, (torch.zeros(1, (1 << 18) + 1, device="cuda"), 1), {})]:
        with pytest.raises(err):
            PF.top_logits(*args, **kw)


def oracle_on_gpu(z, top, y, t, alpha, tail, seeds):
    """oracle() on the GPU, for rows too many for the CPU."""
    x = z.detach().double().requires_grad_(True)
    loss = _ref_distill(x, *top, y, t, alpha, tail, -100)
    (g,) = torch.autograd.grad((loss * seeds.double()).sum(), x)
    return loss.detach(), g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r, v, tail", [(2048, 4099, False), (1500, 9001, True)])
def test_seeds_reach_the_gradient_before_its_rounding(r, v, tail, dtype):
    """A loss scale of 2^16 over the mean, and a seed a row: one rounding, of what the seed has
    multiplied. (The shares of thousands of classes, divided by the rows, are below fp16's numbers.)"""
    t, k, alpha = 2.0, 16, 0.5
    z, top, y = distill_inputs(r, v, k, dtype, t)
    z, top, y = z.cuda(), gpu_top(top), y.cuda()
    g = torch.Generator(device="cuda").manual_seed(9)
    x = z.detach().requires_grad_(True)
    kw = dict(temperature=t, alpha=alpha, tail=tail)
    each = torch.exp2(torch.randint(-8, 17, (r,), generator=g, device="cuda").float()) / r
    each[::5] = 1.0
    for reduction, seed, rows in (("mean", torch.tensor(65536.0, device="cuda"), torch.full((r,), 65536.0 / r)),
                                  ("none", each, each)):
        loss = PF.distill_loss(x, top, y, reduction=reduction, **kw)
        (got,) = torch.autograd.grad(loss, x, seed)
        rows = rows.cuda()
        _, want = oracle_on_gpu(z, top, y, t, alpha, tail, rows)
        c = (3 * spread(z, t) + 260) * U
        q = alpha * t * torch.softmax(z.double() / t, 1) + (1 - alpha) * torch.softmax(z.double(), 1)
        tol = (2 * c * (q * rows.double()[:, None] + want.abs()) + torch.finfo(dtype).eps / 2 * want.abs()
               + (2.0 ** -25 if dtype == torch.float16 else 1e-37))
        assert ((got.double() - want).abs() <= tol).all()
        if dtype == torch.float16 and reduction == "mean":
            # what half of the smallest number is reached by is not zero
            assert (got[want.abs() > 2.0 ** -24] != 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_seed_of_one_is_the_unit_seed(dtype):
    z, top, y = distill_inputs(70, 1003, 9, dtype, 2.0)
    top, y = gpu_top(top), y.cuda()
    kw = dict(temperature=2.0, alpha=0.5, tail=True)
    x = z.cuda().requires_grad_(True)
    grads = []
    for seed in ("unit", None, 1.0, "again"):
        loss = PF.distill_loss(x, top, y, **kw)
        s = PF.unit_grad(loss) if seed in ("unit", "again") else None if seed is None else torch.tensor(1.0, device="cuda")
        if seed == "again":
            torch.autograd.grad(loss, x, s, retain_graph=True)
        grads.append(torch.autograd.grad(loss, x, s)[0])
    assert all(torch.equal(g, grads[0]) for g in grads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [70, 1000, 9000, 70000])
@pytest.mark.parametrize("t, labels, k", [(1.0, False, 1), (2.0, True, 3), (0.7, True, 1), (0.1, False, 3)])
def test_rest_far_below_the_kept(v, dtype, t, labels, k):
    """A student whose kept classes stand far above all others (gaps in z / T): the rest's mass has a
    logarithm and shares where it is too small a part of the row for 32 bits."""
    gaps = [30.0, 50.0, 54.0, 57.0, 62.0, 80.0, 86.0, 90.0, 100.0, 200.0, 700.0, 100.0]
    r, alpha = len(gaps), 0.6 if labels else 1.0
    z = make(r, v, torch.float32, 21, 1.0)
    idx = torch.stack([torch.randperm(v, generator=torch.Generator().manual_seed(i))[:k] for i in range(r)])
    z.scatter_(1, idx, (torch.tensor(gaps)[:, None] + torch.arange(k)) * t)
    z[11] = -math.inf                       # nothing but the kept and one more
    z[11, idx[11]] = 3.0
    z[11, (idx[11, 0] + 1) % v if k == 1 else next(j for j in range(v) if j not in idx[11].tolist())] = 3.0 - 150 * t
    z = z.to(dtype)
    values = t * torch.arange(k).float().expand(r, k).contiguous()
    # the kept classes hold 0.99 of the teacher's mass
    lse = torch.logsumexp(values.double() / t, 1).sub(math.log(0.99)).float()
    top = PF.TopLogits(values, idx.int(), lse)
    y = None
    if labels:
        y = idx[:, 0].clone()
        y[1::2] = (y[1::2] + 1) % v         # (some are kept classes, most of these are not)
        y[11] = idx[11, 0]
    want, grad = oracle(z, top, y, t, alpha, True)
    x = z.cuda().requires_grad_(True)
    kw = dict(temperature=t, alpha=alpha, tail=True, reduction="none")
    loss = PF.distill_loss(x, gpu_top(top), y.cuda() if labels else None, **kw)
    loss.backward(torch.ones_like(loss))
    alone = PF.distill_loss(x.detach(), gpu_top(top), y.cuda() if labels else None, **kw)
    for i in range(r):
        tl, tg = tolerances(z[i:i + 1], t, alpha, grad[i:i + 1])
        for got in (loss, alone):
            assert abs(got[i].item() - want[i].item()) <= tl + 2 * U * want[i].abs(), (i, got[i], want[i])
        off = (x.grad[i].cpu().double() - grad[i]).abs()
        # Exponentials below 2^-126 of their base are zero in 32 bits. The rest's mass is 2^-60 of its base
        # at least (it takes another below), so what is zero has a share of the rest below 2^-66, and
        # alpha T rest times it of the gradient; the teacher's rest is 0.01.
        lost = alpha * t * 0.01 * 2.0 ** -66
        assert (off <= tg(dtype)[0] + lost).all(), (i, off.max())


def test_rest_without_classes():
    """All other classes masked by -inf: the teacher gives them mass, the student none."""
    z = torch.full((2, 300), -math.inf)
    z[:, 5] = 1.0
    z[1, 6:] = torch.finfo(torch.float32).min
    top = PF.TopLogits(torch.zeros(2, 1), torch.full((2, 1), 5, dtype=torch.int32), torch.full((2,), 0.01))
    want, _ = oracle(z, top, None, 1.0, 1.0, True)
    x = z.cuda().requires_grad_(True)
    loss = PF.distill_loss(x, gpu_top(top), tail=True, reduction="none")
    loss.backward(torch.ones_like(loss))
    assert loss[0] == math.inf
    # (the rest's logarithm is the mask's value over T: all but the rest's share of it is rounding)
    assert abs(loss[1].item() / want[1].item() - 1) <= 8 * U
    # the student's mass is all at class 5 (q = 1, p = 1 - rest), that of the others is shared by the 294
    # that are not at -inf alike: gradients rest and -rest / 294
    rest = 1 - math.exp(-top.lse[1].item())
    by_hand = torch.zeros(300, dtype=torch.float64)
    by_hand[5], by_hand[6:] = rest, -rest / 294
    assert ((x.grad[1].cpu().double() - by_hand).abs() <= 600 * U * by_hand.abs()).all()


@pytest.mark.parametrize("v", [300, 1000, 2000, 8192, 40000, 150000])
@pytest.mark.parametrize("low", [-86.0, -88.0, -89.0, -90.0, -95.0, -100.0])
def test_first_chunks_far_below_the_rest(v, low):
    """The classes that threads meet first stand some 90 below the largest, what follows them near it: a
    thread's sum is far above its base, and its base as far below the row's."""
    for first in (64 * 4, 256 * 4, 1024 * 4):
        z = make(6, v, torch.float32, 31, 0.5) - 10.0
        z[:, :first] = low
        z[2:4] = torch.where(torch.arange(v) < first, low, -14.0)
        z[:, 5] = 0.0
        z[1, 5], z[1, v - 1] = low, 0.0
        check_top(z, min(v, 7))
        top = PF.TopLogits(torch.zeros(6, 1), torch.full((6, 1), v // 2, dtype=torch.int32), torch.full((6,), 0.5))
        y = torch.full((6,), v - 1)
        for t, tail in ((1.0, True), (2.0, False), (0.9, True)):
            want, grad = oracle(z, top, y, t, 0.5, tail)
            tl, tg = tolerances(z, t, 0.5, grad)
            x = z.cuda().requires_grad_(True)
            loss = PF.distill_loss(x, gpu_top(top), y.cuda(), temperature=t, alpha=0.5, tail=tail, reduction="none")
            loss.backward(torch.ones_like(loss))
            assert ((loss.cpu().double() - want).abs() <= tl + 2 * U * want.abs()).all()
            assert ((x.grad.cpu().double() - grad).abs() <= tg(torch.float32)).all()


@pytest.mark.parametrize("v", [300, 2000, 9000, 40000])
@pytest.mark.parametrize("t", [1.0, 2.0, 0.5])
def test_classes_masked_by_some_millions(v, t):
    """Masks near -2^22 / log2(e) T, below which a thread takes no base from its first classes: what it
    has summed by then counts as little as before."""
    z = make(12, v, torch.float32, 41, 1.0)
    for i, steps in enumerate((-200.0, -100.0, -20.0, -4.0, -1.0, -0.5, 0.0, 0.5, 1.0, 20.0, 200.0, -126.0)):
        z[i, :v - 40] = (steps - 4194304.0) / 1.4426950408889634 * t
    real = z[:, v - 40:]
    lse = PF.top_logits(z.cuda(), 7, t).lse.cpu().double()
    ref = torch.logsumexp(z.double() / t, 1)
    # (the row's own classes spread over some 10: what is masked has a share of 0, with any error)
    assert ((lse - ref).abs() <= (3 * spread(real, t) + 260) * U + U * ref.abs()).all()
    top = PF.TopLogits(torch.zeros(12, 1), torch.full((12, 1), v - 3, dtype=torch.int32), torch.full((12,), 0.5))
    y = torch.full((12,), v - 1)
    for tail in (False, True):
        want, grad = oracle(z, top, y, t, 0.5, tail)
        tl, tg = tolerances(real, t, 0.5, grad[:, v - 40:])
        x = z.cuda().requires_grad_(True)
        loss = PF.distill_loss(x, gpu_top(top), y.cuda(), temperature=t, alpha=0.5, tail=tail, reduction="none")
        loss.backward(torch.ones_like(loss))
        assert ((loss.cpu().double() - want).abs() <= tl + 2 * U * want.abs()).all()
        assert ((x.grad.cpu().double() - grad).abs()[:, v - 40:] <= tg(torch.float32)).all()
        assert not x.grad[:, :v - 40].any()


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad as fa

    z, top, y = distill_inputs(4, 50, 3, torch.float32, 1.0)
    z, top = z.cuda(), gpu_top(top)
    with fa.dual_level():
        for leaf in (z, z.clone().requires_grad_(True)):
            dual = fa.make_dual(leaf, torch.ones_like(leaf))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                PF.distill_loss(dual, top)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                PF.distill_loss(dual[:2, 1:40], PF.TopLogits(*(a[:2] for a in top)))
        values = fa.make_dual(top.values, torch.ones_like(top.values))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            PF.distill_loss(z, PF.TopLogits(values, top.indices, top.lse))
        # data, as in reverse mode
        assert fa.unpack_dual(PF.top_logits(fa.make_dual(z, torch.ones_like(z)), 3).values).tangent is None
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: PF.distill_loss(x, top), (z,), (torch.ones_like(z),))


def check_streamed(z, t, terms, x_loss, want, x_grad, grad, alpha, seeds):
    """Losses and gradients on the GPU, where a thread sums `terms` terms of a row."""
    c = (3 * spread(z, t) + terms + 4) * U
    assert ((x_loss.double() - want).abs() <= 2 * c * (alpha * t * t + 1 - alpha) + 2 * U * want.abs()).all()
    if x_grad is None:
        return
    q = alpha * t * torch.softmax(z.double() / t, 1) + (1 - alpha) * torch.softmax(z.double(), 1)
    tol = 2 * c * (q * seeds.double()[:, None] + grad.abs()) + torch.finfo(z.dtype).eps / 2 * grad.abs()
    tol += 2.0 ** -25 if z.dtype == torch.float16 else 1e-37
    assert ((x_grad.double() - grad).abs() <= tol).all()


# rows and chunks of 16 bytes: streamed by 256, 512 or 1024 threads with a gradient and without (a row of
# up to 8192 chunks takes fewer threads than a longer one, and few rows take more)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r, chunks", [(530, 1030), (530, 8190), (530, 8300), (1030, 1251), (1030, 8190), (1030, 8193),
                                       (1100, 2500), (300, 1500)])
def test_distill_streamed_by_few_threads(r, chunks, dtype):
    if dtype == torch.float32:
        v = chunks * 4 - 3
    else:
        v = chunks * 8 - 5
    t, alpha, k = 2.0, 0.7, 33
    g = torch.Generator(device="cuda").manual_seed(r + chunks)
    teacher = (3 * torch.randn(r, v, generator=g, device="cuda")).to(dtype)
    z = (0.6 * teacher.float() + 1.5 * torch.randn(r, v, generator=g, device="cuda")).to(dtype)
    top = PF.top_logits(teacher, k, t)
    del teacher
    y = torch.randint(0, v, (r,), generator=g, device="cuda")
    top.indices[3, 7:] = -1
    top.indices[5] = -1
    top.indices[6, 3] = top.indices[6, 1]
    y[7::50] = -100
    seeds = torch.rand(r, generator=g, device="cuda") + 0.5
    terms = (chunks + 255) // 256 * (4 if dtype == torch.float32 else 8)      # (256 threads: the most)
    for tail in (True, False):
        kw = dict(temperature=t, alpha=alpha, tail=tail, reduction="none")
        x = z.detach().requires_grad_(True)
        loss = PF.distill_loss(x, top, y, **kw)
        (got,) = torch.autograd.grad(loss, x, seeds)
        alone = PF.distill_loss(z, top, y, **kw)
        for at in range(0, r, 265):               # (64 bits of some rows at a time)
            s = slice(at, min(at + 265, r))
            part = PF.TopLogits(*(a[s] for a in top))
            want, grad = oracle_on_gpu(z[s], part, y[s], t, alpha, tail, seeds[s])
            check_streamed(z[s], t, terms, loss.detach()[s], want, got[s], grad, alpha, seeds[s])
            check_streamed(z[s], t, terms, alone[s], want, None, None, alpha, seeds[s])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r, chunks, k", [(520, 1030, 5), (520, 1251, 120), (520, 8192, 256), (520, 8193, 256), (300, 2000, 100),
                                          (520, 16384, 384), (520, 16385, 300), (300, 6000, 640), (300, 4000, 700),
                                          (300, 1100, 1024), (200, 3000, 200)])
def test_top_logits_streamed_by_few_threads(r, chunks, k, dtype):
    v = chunks * 4 - 3 if dtype == torch.float32 else chunks * 8 - 5
    g = torch.Generator(device="cuda").manual_seed(r + chunks)
    z = (3 * torch.randn(r, v, generator=g, device="cuda")).to(dtype)
    z[1] = z[1].sort()[0]
    z[2] = z[2].sort(descending=True)[0]
    z[3, v // 3:] = -math.inf
    z[4, :v // 2] = torch.finfo(dtype).min
    z[5] = z[5].float().round().to(dtype)
    z[6, v // 2] = math.nan
    z[7] = 1.0
    top = PF.top_logits(z, k, 2.0)
    some = list(range(9)) + [r // 2, r - 2, r - 1]
    want = PF.top_logits(z[some].cpu(), k, 2.0)
    assert torch.equal(top.indices[some].cpu(), want.indices)
    # all rows: descending, each value where it says, no class twice, nothing left out above the last
    for at in range(0, r, 130):
        s = slice(at, min(at + 130, r))
        f = torch.nan_to_num(z[s].float(), nan=math.inf)
        vals = f.gather(1, top.indices[s].long())
        assert torch.equal(vals, torch.nan_to_num(top.values[s].float(), nan=math.inf))
        assert (vals[:, :-1] >= vals[:, 1:]).all()
        order = top.indices[s].sort(1)[0]
        assert (order[:, 1:] > order[:, :-1]).all()
        assert ((f > vals[:, -1:]).sum(1) < k).all()
        keep = torch.tensor([i for i in range(at, s.stop) if i != 6], device="cuda") - at
        # C of a thread's most terms (256 threads)
        terms = (chunks + 255) // 256 * (4 if dtype == torch.float32 else 8)
        rows = z[s][keep]
        c = (3 * spread(rows.masked_fill(rows <= torch.finfo(dtype).min, 0), 2.0) + terms + 4) * U
        ref = torch.logsumexp(rows.double() / 2.0, 1)
        assert ((top.lse[s][keep].double() - ref).abs() <= c + U * ref.abs()).all()
    assert top.lse[6].isnan()


def test_temperatures_at_the_ends_of_their_range():
    for t in (2.0 ** -64, 2.0 ** 64):
        z, top, y = distill_inputs(4, 50, 3, torch.float32, 1.0)
        z.mul_(t)
        teacher = make(4, 50, torch.float32, 3) * t
        top = PF.top_logits(teacher, 3, t)
        got = PF.top_logits(teacher.cuda(), 3, t)
        assert torch.equal(got.indices.cpu(), top.indices)
        assert ((got.lse.cpu() - top.lse).abs() <= 300 * U * top.lse.abs()).all()
    for t in (2.0 ** -65, 2.0 ** 65, 1e-40, 1e-300, 1e300):
        with pytest.raises(ValueError):
            PF.top_logits(z.cuda(), 3, t)
        with pytest.raises(ValueError):
            PF.distill_loss(z.cuda(), gpu_top(top), temperature=t)
