"""How near lm_loss's gradients (ops/csrc/loss_kernels.hip) come to what their types allow, in
units of the exact result's own rounding to the type.

A gradient has that rounding (1 by definition) and the roundings of d, the product's operand,
about as much again; fp32 sums and exponentials are far below.  They are independent, so they
add in quadrature: about sqrt(2), which 1.6 bounds.  An emulation of the roundings on the CPU
holds the same bound, and breaks it with a mistake of 1 % in d or in its labels' terms."""
import pytest
import torch

SHAPES = [(61, 8192, 256, 0.5, 1.0), (65, 100, 72, 0.9, 1.0), (255, 1000, 128, 1.0, 1.0), (257, 257, 200, 0.7, 1.0),
          (600, 3301, 136, 0.3, 1.0), (300, 513, 128, 1.0, 40.0)]
LARGE = [(4099, 4161, 192, 0.8, 1.0), (600, 33001, 136, 0.3, 1.0), (9000, 17000, 64, 0.2, 1.0), (14464, 8192, 256, 0.33, 1.0),
         (9001, 8191, 128, 0.9, 1.0)]


def _inputs(N, V, H, kept, grow, dtype):
    """h, table, labels (-100: left out) and a weight a row, on the CPU."""
    g = torch.Generator().manual_seed(N + V)
    table = torch.randn(V, H, generator=g) * 0.1
    labels = torch.randint(0, V, (N,), generator=g)
    h = torch.randn(N, H, generator=g) * 0.3 + 4.0 * torch.rand(N, 1, generator=g) * table[labels]
    labels[torch.rand(N, generator=g) >= kept] = -100
    return (h * grow).to(dtype), table.to(dtype), labels, torch.rand(N, generator=g) + 0.25


def _exact(h, table, labels, w, dtype=None, mistake=lambda d: d):
    """dh and dtable of sum(w loss) over the labelled rows, in 64 bits by the formulas (dtype:
    with d rounded to it, as the kernel does)."""
    on = labels >= 0
    x, e, y = h[on].double(), table.double(), labels[on]
    d = torch.softmax(x @ e.t(), 1)
    d[torch.arange(len(y), device=d.device), y] -= 1.0
    if dtype is not None:
        f = 1024.0 if dtype == torch.float16 else 1.0
        d = (mistake(d) * f).to(dtype).double() / f
    d = d * w[on].double()[:, None]
    dh = torch.zeros(h.shape, dtype=torch.float64, device=h.device)
    dh[on] = d @ e
    return dh, d.t().contiguous() @ x


def _far(got, want, dtype):
    """The farther gradient's distance, the exact one's own rounding being 1."""
    return max(float((x.to(dtype).double() - y).norm() / (y.to(dtype).double() - y).norm()) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_the_bound_passes_the_roundings_and_no_mistake(shape, dtype):
    args = _inputs(*shape, dtype)
    want = _exact(*args)
    assert _far(_exact(*args, dtype), want, dtype) <= 1.6
    assert _far(_exact(*args, dtype, lambda d: 1.01 * d), want, dtype) > 1.6
    assert _far(_exact(*args, dtype, lambda d: torch.where(d < 0, 1.01 * d, d)), want, dtype) > 1.6
    assert _far([torch.zeros_like(t) for t in want], want, dtype) > 100


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES + LARGE)
def test_gradients_are_as_near_as_their_roundings(shape, dtype, reduction):
    from smsgate_amd.models import train_ops

    h, table, labels, w = (t.to("cuda") for t in _inputs(*shape, dtype))
    h.requires_grad_(), table.requires_grad_()
    n = int((labels >= 0).sum())
    # an incoming gradient that keeps fp16's results in its normal range
    by = w if reduction == "none" else torch.tensor(float(n) if reduction == "mean" else 1.0, device="cuda")
    loss = train_ops.lm_loss(h, table, labels, reduction=reduction)
    got = torch.autograd.grad(loss, (h, table), by)
    want = _exact(h.detach(), table.detach(), labels, w if reduction == "none" else torch.ones_like(w))
    far = _far(got, want, dtype)
    assert far <= 1.6, far
