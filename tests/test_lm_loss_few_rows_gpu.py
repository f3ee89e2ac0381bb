"""lm_loss's gradients over few rows (ops/csrc/loss_kernels.hip), where one row's rounding of d
would show as it is: they are the exact result's own rounding to the type and nothing more (1 in
its units; 1.1 leaves room for fp32's)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N,V,H,kept", [(1, 100, 128, 1.0), (1, 70001, 64, 1.0), (2, 500, 576, 1.0), (3, 8192, 256, 1.0),
                                        (5, 33, 72, 0.7), (17, 1000, 960, 1.0), (61, 8192, 256, 0.5), (64, 577, 64, 1.0),
                                        (100, 70001, 200, 0.9), (128, 2000, 128, 1.0)])
def test_few_rows(N, V, H, kept, reduction, dtype):
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(N + V + H)
    table = (torch.randn(V, H, generator=g, device=dev) * 0.05).to(dtype)
    labels = torch.randint(0, V, (N,), generator=g, device=dev)
    lean = 12.0 * torch.rand(N, 1, generator=g, device=dev)
    h = torch.randn(N, H, generator=g, device=dev) + lean * table[labels].float() / (0.05 * H ** 0.5)
    h = (h * torch.rsqrt(h.square().mean(-1, keepdim=True))).to(dtype)
    labels[torch.rand(N, generator=g, device=dev) >= kept] = -100
    labels[0] = V - 1
    on = labels >= 0
    n = int(on.sum())
    w = torch.rand(N, generator=g, device=dev) + 0.25
    h.requires_grad_(), table.requires_grad_()
    # an incoming gradient that keeps fp16's results in its normal range
    by = w * 16 if reduction == "none" else torch.tensor(16.0 * n if reduction == "mean" else 16.0, device=dev)
    loss = train_ops.lm_loss(h, table, labels, reduction=reduction)
    dh, dt = torch.autograd.grad(loss, (h, table), by)
    x, e, y = h.detach()[on].double(), table.detach().double(), labels[on]
    d = torch.softmax(x @ e.t(), 1)
    d[torch.arange(n, device=dev), y] -= 1.0
    d = d * 16 * (w[on].double()[:, None] if reduction == "none" else 1.0)
    for got, want in ((dh[on], d @ e), (dt, d.t().contiguous() @ x)):
        own = float((want.to(dtype).double() - want).norm())
        assert float((got.double() - want).norm()) <= 1.1 * own + 1e-6 * float(want.norm())
    assert not dh[~on].any()


@pytest.mark.parametrize("N,V", [(61, 8192), (100, 70001)])
def test_few_rows_each_gradient_alone_and_again(N, V):
    """Only one input asks for a gradient, the backward runs twice: the same bits."""
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(N)
    h = torch.randn(N, 256, generator=g, device=dev).bfloat16()
    table = (torch.randn(V, 256, generator=g, device=dev) * 0.1).bfloat16()
    labels = torch.randint(-1, V, (N,), generator=g, device=dev)
    a, b = h.clone().requires_grad_(), table.clone().requires_grad_()
    loss = train_ops.lm_loss(a, b, labels, ignore_index=-1)
    want = torch.autograd.grad(loss, (a, b), retain_graph=True)
    for x, y in zip(torch.autograd.grad(loss, (a, b)), want):
        assert torch.equal(x, y)
    a, b = h.clone().requires_grad_(), table.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(train_ops.lm_loss(a, table, labels, ignore_index=-1), a)[0], want[0])
    assert torch.equal(torch.autograd.grad(train_ops.lm_loss(h, b, labels, ignore_index=-1), b)[0], want[1])
