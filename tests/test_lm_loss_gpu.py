"""Vocabulary cross entropy and its gradients (ops/csrc/loss_kernels.hip via
models/train_ops.py lm_loss) against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def _ref(h, table, labels, reduction, ignore, g):
    """loss, dh, dtable in 64 bits, by the formulas."""
    H = h.shape[-1]
    x, e, y = h.reshape(-1, H).double(), table.double(), labels.reshape(-1).long()
    keep = y != ignore
    yk = torch.where(keep, y, 0)
    z = x @ e.t()
    lse = torch.logsumexp(z, 1)
    each = torch.where(keep, lse - z.gather(1, yk[:, None])[:, 0], 0.0)
    n = keep.sum()
    w = {"mean": g / n if n else g, "sum": g, "none": g.reshape(-1)}[reduction].double() * keep
    d = torch.exp(z - lse[:, None])
    d[torch.arange(len(y), device=d.device), yk] -= 1.0
    d = d * w[:, None]
    loss = {"mean": each.sum() / n, "sum": each.sum(), "none": each.reshape(labels.shape)}[reduction]
    return loss, (d @ e).reshape(h.shape), d.t() @ x


def _run(h, table, labels, reduction, ignore, g):
    from smsgate_amd.models import train_ops

    h, table = h.detach().requires_grad_(), table.detach().requires_grad_()
    loss = train_ops.lm_loss(h, table, labels, reduction=reduction, ignore_index=ignore)
    return (loss.detach(), *torch.autograd.grad(loss, (h, table), g))


def _check(h, table, labels, reduction="mean", ignore=-100, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed + 99)
    g = torch.rand(labels.shape if reduction == "none" else (), generator=gen, device=dev) + 0.1
    got, want = _run(h, table, labels, reduction, ignore, g), _ref(h, table, labels, reduction, ignore, g)
    u, t = U[h.dtype], h.dtype
    assert got[0].dtype == torch.float32 and got[0].shape == want[0].shape
    # a logit: H products, exact in fp32, summed in fp32: off by at most H 2^-24 sum |h e|;
    # L by as much and the rounding of a few operations on values of its size
    zmax = float((h.reshape(-1, h.shape[-1]).double().abs() @ table.double().abs().t()).max())
    tol = (2 * h.shape[-1] + 16) * 2.0 ** -24 * max(zmax, 1.0)
    n = max(1, int((labels != ignore).sum()))
    if reduction == "sum":
        tol = tol * n + 2.0 ** -24 * (n / 1024 + 32) * abs(float(want[0]))
    elif reduction == "mean":
        tol += 2.0 ** -24 * (n / 1024 + 32) * abs(float(want[0]))
    assert float((got[0].double() - want[0]).abs().max()) <= tol
    # gradients, relative 2-norms: d rounded to the type (u) and the result rounded (u), with
    # fp32 sums far below; p in d is off by up to `tol` relative, against |d| = 1 at most
    for name, x, y in zip(("dh", "dtable"), got[1:], want[1:]):
        assert x.dtype == t and x.shape == y.shape, name
        grain = 2.0 ** -25 * math.sqrt(y.numel()) if t == torch.float16 else 0.0  # fp16's subnormal step
        other = float((table if name == "dh" else h).double().norm())
        gsum = float((g.double().expand(labels.shape) if reduction == "none" else g.double()).norm())
        err = float((x.double() - y).norm())
        assert err <= 2 * u * float(y.norm()) + grain + tol * gsum * other, (name, err, float(y.norm()))
    flat = (labels == ignore).reshape(-1)
    assert not got[1].reshape(-1, h.shape[-1])[flat].any()
    return got


def _inputs(N, V, H, dtype, kept=1.0, seed=0, lean=4.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    table = torch.randn(V, H, generator=g, device=dev) * 0.1
    labels = torch.randint(0, V, (N,), generator=g, device=dev)
    h = torch.randn(N, H, generator=g, device=dev) * 0.3
    h = h + lean * torch.rand(N, 1, generator=g, device=dev) * table[labels]
    labels[torch.rand(N, generator=g, device=dev) >= kept] = -100
    return h.to(dtype), table.to(dtype), labels


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N,V,H,kept", [(1, 1, 8, 1.0), (1, 2, 64, 1.0), (61, 8192, 256, 0.5), (65, 100, 72, 0.9),
                                        (255, 1000, 128, 1.0), (257, 257, 200, 0.7), (4099, 4161, 192, 0.8),
                                        (600, 33001, 136, 0.3)])
def test_loss_matches_definition(dtype, reduction, N, V, H, kept):
    """Small and big tiles, sizes on both sides of every tile, hidden sizes that are not a
    multiple of 64, more than one piece of the vocabulary."""
    h, table, labels = _inputs(N, V, H, dtype, kept, seed=N)
    if (labels == -100).all():
        labels[0] = 0
    _check(h, table, labels, reduction, seed=N)


def test_loss_pieces():
    """Rows enough for the vocabulary to be taken in several pieces."""
    h, table, labels = _inputs(40000, 9000, 64, torch.bfloat16, 0.2, seed=3)
    _check(h, table, labels)


def test_loss_shapes_and_label_types():
    h, table, labels = _inputs(6 * 35, 777, 64, torch.bfloat16, 0.6, seed=5)
    _check(h.view(6, 35, 64), table, labels.view(6, 35), "none")
    _check(h.view(6, 35, 64), table, labels.view(6, 35).int())
    # views: rows of a wider matrix, off a 16-byte border, labels with a stride
    wide = torch.zeros(210, 70, dtype=torch.bfloat16, device=dev)
    wide[:, 3:67] = h
    flat = torch.zeros(777 * 64 + 1, dtype=torch.bfloat16, device=dev)
    flat[1:] = table.reshape(-1)
    two = torch.stack([labels, labels], 1)
    a = _check(h, table, labels)
    b = _check(wide[:, 3:67], flat[1:].view(777, 64), two[:, 0])
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    # another ignore_index, one that is an id
    _check(h, table, torch.where(labels < 0, 5, labels), ignore=5)


def test_loss_large_logits():
    """Logits of some hundreds: one id takes all, losses of 0 and of hundreds."""
    h, table, labels = _inputs(300, 513, 128, torch.bfloat16, 1.0, seed=7)
    _check(h * 100, table * 2, labels, "none")


def test_loss_nothing_labelled():
    from smsgate_amd.models import train_ops

    h, table, labels = _inputs(70, 200, 64, torch.bfloat16)
    labels.fill_(-100)
    for reduction in ("mean", "sum", "none"):
        g = torch.ones(labels.shape if reduction == "none" else (), device=dev)
        loss, dh, dt = _run(h, table, labels, reduction, -100, g)
        assert loss.isnan().all() if reduction == "mean" else not loss.any()
        assert not dh.any() and not dt.any()
    assert train_ops.lm_loss(h, table, labels, reduction="sum") == 0


def test_loss_label_of_no_row_is_loud():
    h, table, labels = _inputs(70, 200, 64, torch.bfloat16)
    for bad in (200, -1, 2 ** 31 - 1, -2 ** 40):
        y = labels.clone()
        y[3] = bad
        loss, dh, dt = _run(h, table, y, "none", -100, torch.ones(70, device=dev))
        assert loss[3].isnan() and not loss[:3].isnan().any() and not loss[4:].isnan().any()
        assert dh[3].isnan().all() and not dh[:3].isnan().any() and dt.isnan().all()


def test_loss_gradient_against_differences():
    """The directional derivative of the mean in h and table against central differences of
    the 64-bit definition."""
    h, table, labels = _inputs(90, 333, 64, torch.bfloat16, 0.7, seed=11)
    _, dh, dt = _run(h, table, labels, "mean", -100, torch.ones((), device=dev))
    keep = labels >= 0

    def f(a, b):
        z = a[keep] @ b.t()
        return (torch.logsumexp(z, 1) - z.gather(1, labels[keep][:, None])[:, 0]).mean()

    gen = torch.Generator(device=dev).manual_seed(13)
    for d, which in ((dh, 0), (dt, 1)):
        x = [h.double(), table.double()]
        e = torch.randn(x[which].shape, generator=gen, device=dev, dtype=torch.float64)
        hi, lo = list(x), list(x)
        hi[which], lo[which] = x[which] + 1e-4 * e, x[which] - 1e-4 * e
        want, got = float(f(*hi) - f(*lo)) / 2e-4, float((d.double() * e).sum())
        # the gradient is off by at most 2 u of its norm, in a direction that e meets at random (4 sigma)
        assert abs(got - want) <= 4 * 2 * 2.0 ** -8 * float(d.double().norm()) + 1e-7, (which, got, want)


def test_loss_repeats_partial_gradients_and_no_grad():
    from smsgate_amd.models import train_ops

    h, table, labels = _inputs(500, 4000, 192, torch.bfloat16, 0.5, seed=17)
    one = torch.ones((), device=dev)
    first = _run(h, table, labels, "mean", -100, one)
    for _ in range(3):
        for x, y in zip(_run(h, table, labels, "mean", -100, one), first):
            assert torch.equal(x, y)
    with torch.no_grad():
        assert torch.equal(train_ops.lm_loss(h, table, labels), first[0])
    a = h.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(train_ops.lm_loss(a, table, labels), a)[0], first[1])
    b = table.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(train_ops.lm_loss(h, b, labels), b)[0], first[2])


def test_loss_graph():
    """Captured, and replayed on other states and labels (another number of labelled rows)
    between eager calls."""
    from smsgate_amd.models import train_ops

    for N, V, H, reduction in ((61, 500, 64, "mean"), (2100, 9000, 128, "none")):
        h, table, labels = _inputs(N, V, H, torch.bfloat16, 0.5)
        h.requires_grad_(), table.requires_grad_()
        g = torch.ones(N if reduction == "none" else (), device=dev)

        def step(a, b):
            loss = train_ops.lm_loss(a, b, labels, reduction=reduction)
            return (loss.detach(), *torch.autograd.grad(loss, (a, b), g))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(h, table)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(h, table)
        for i in range(4):
            h2, t2, y2 = _inputs(N, V, H, torch.bfloat16, 0.2 * (i + 1), seed=i)
            with torch.no_grad():
                h.copy_(h2), table.copy_(t2), labels.copy_(y2)
            want = step(h2.requires_grad_(), t2.requires_grad_())
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(res, want):
                assert torch.equal(x, y), (N, i)
