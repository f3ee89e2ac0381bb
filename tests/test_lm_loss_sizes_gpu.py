"""lm_loss (ops/csrc/loss_kernels.hip) on both sides of its rules on sizes: rows numbered by
every block or by one, tiles small or large, the hidden gradient in one share or many."""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N,V,H,kept", [
    (1023, 300, 72, 0.5), (1024, 300, 72, 1.0), (1025, 300, 72, 0.5), (1024, 300, 72, 0.0), (1025, 300, 72, 0.0),
    (1024, 33000, 64, 0.02), (1600, 33000, 200, 0.9), (5000, 17000, 64, 0.1), (17000, 9000, 64, 0.01),
])
def test_rules_on_sizes(N, V, H, kept, reduction):
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(N + V)
    h = torch.randn(N, H, generator=g, device=dev).bfloat16().requires_grad_()
    table = (torch.randn(V, H, generator=g, device=dev) * 0.3).bfloat16().requires_grad_()
    labels = torch.randint(0, V, (N,), generator=g, device=dev)
    labels[torch.rand(N, generator=g, device=dev) >= kept] = -100
    on = labels >= 0
    n = int(on.sum())
    by = torch.randn(N, generator=g, device=dev) if reduction == "none" else torch.ones((), device=dev)
    loss = train_ops.lm_loss(h, table, labels, reduction=reduction)
    dh, dt = torch.autograd.grad(loss, (h, table), by)
    x, e, y = h.detach()[on].double(), table.detach().double(), labels[on]
    z = x @ e.t()
    lse = torch.logsumexp(z, 1)
    each = lse - z.gather(1, y[:, None])[:, 0]
    w = by[on].double() if reduction == "none" else torch.full((n,), 1.0 / n if reduction == "mean" and n else 1.0,
                                                               device=dev, dtype=torch.float64)
    d = torch.exp(z - lse[:, None])
    d[torch.arange(n, device=dev), y] -= 1.0
    d *= w[:, None]
    want = torch.zeros(N, H, dtype=torch.float64, device=dev)
    want[on] = d @ e
    # z: H products summed in fp32, so off by at most H 2^-24 sum |x e| (4 standard
    # deviations of it and more); the loss adds roundings of values of z's size
    tol = (H + 16) * 2.0 ** -24 * float((x.abs() @ e.abs().t()).max()) if n else 0.0
    if reduction == "none":
        assert not loss[~on].any() and (n == 0 or float((loss.double()[on] - each).abs().max()) <= tol)
    elif n == 0:
        assert torch.isnan(loss) if reduction == "mean" else float(loss) == 0.0
    else:
        ref = float(each.sum() if reduction == "sum" else each.mean())
        assert abs(float(loss) - ref) <= tol * (n if reduction == "sum" else 1) + 2.0 ** -20 * abs(ref)
    # d rounded to bf16 as an operand and the result rounded: 2^-8 each, relative norms
    assert not dh[~on].any()
    assert float((dh.double() - want).norm()) <= 2 * 2.0 ** -8 * float(want.norm())
    wt = d.t().contiguous() @ x
    assert float((dt.double() - wt).norm()) <= 2 * 2.0 ** -8 * float(wt.norm())
