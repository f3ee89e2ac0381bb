"""lm_loss (ops/csrc/loss_kernels.hip) on rows that are nearly sure of their label, at logits of
hundreds: the label's term 1 - p is far below the rounding of the logits' logarithm of a sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def _rows(N, V, top, gap, dtype, seed):
    """Hidden states and a table whose logits are exact in fp32 in whatever order they are
    summed (multiples of 1/8 below 2^10): a shift of about ``top`` that every id shares, and
    60 columns of signs of which the label has all, the others about half."""
    g = torch.Generator(device=dev).manual_seed(seed)
    signs = torch.randint(0, 2, (V, 60), generator=g, device=dev) * 2.0 - 1.0
    labels = torch.randint(0, V, (N,), generator=g, device=dev)
    table = torch.zeros(V, 64, device=dev)
    h = torch.zeros(N, 64, device=dev)
    table[:, 0], h[:, 0] = 8.0, top / 8
    table[:, 4:] = signs
    h[:, 4:] = gap * signs[labels]
    return h.to(dtype), table.to(dtype), labels


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top", [0, 128, 320, 896])
@pytest.mark.parametrize("N,V,gap", [(40, 500, 0.25), (40, 500, 0.375), (1100, 3000, 0.375), (3000, 30000, 0.375)])
def test_nearly_sure_rows(dtype, top, N, V, gap):
    """1 - p of 1e-3 to 1e-6.  Small tiles and large, one and many labels a tile."""
    from smsgate_amd.models import train_ops

    h, table, labels = _rows(N, V, top, gap, dtype, seed=N + V + top)
    h.requires_grad_(), table.requires_grad_()
    each = train_ops.lm_loss(h, table, labels, reduction="none")
    # (a gradient of 2^10: fp16 holds what comes of it)
    dh, dt = torch.autograd.grad(each, (h, table), torch.full((N,), 1024.0, device=dev))
    x, e = h.detach().double(), table.detach().double()
    z = x @ e.t()
    at = torch.arange(N, device=dev)
    zy = z[at, labels]
    others = torch.exp(z - zy[:, None])
    others[at, labels] = 0.0
    s = others.sum(1)  # of the other ids over the label
    want = torch.log1p(s)
    d = others / (1 + s)[:, None]
    d[at, labels] = -s / (1 + s)
    assert float(s.max()) < 0.1 and float(s.min()) > 1e-8
    # e^x is off by the rounding of its argument (|x| up to 50, its product with log2 e and the
    # difference with the sum's logarithm) and an ulp or two: 160 2^-24; sums of positive terms
    # add a rounding each of 64 at most that lie one above the other (a lane's, its wave's, the
    # tiles')
    fp32 = (160 + 64) * 2.0 ** -24
    assert float(((each.detach().double() - want).abs() / want).max()) <= 2 * fp32
    # d rounded to the type as an operand (fp16: of 1024 d, at least 2^-25 off), the gradient
    # rounded; products summed in fp32, 2 roundings of each 32-wide step and of the shares
    u = U[dtype]
    tiny = 2.0 ** -35 if dtype == torch.float16 else 0.0
    grain = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for got, ref, size, many in ((dh, d @ e, d.abs() @ e.abs(), V), (dt, d.t() @ x, d.abs().t() @ x.abs(), N)):
        other = float(max(e.abs().max() if got is dh else x.abs().max(), 0.0))
        tol = 1024 * (size * (u + 2 * fp32 + many / 8 * 2.0 ** -24) + ref.abs() * u + many * tiny * other) + grain
        err = (got.double() - 1024 * ref).abs()
        assert (err <= tol).all(), (float((err / tol).nan_to_num().max()), "dh" if got is dh else "dtable")


def test_one_id():
    """Nothing but the label: p = 1, the loss and both gradients exactly 0."""
    from smsgate_amd.models import train_ops

    h = (torch.randn(70, 64, device=dev) * 30).bfloat16().requires_grad_()
    table = torch.randn(1, 64, device=dev).bfloat16().requires_grad_()
    each = train_ops.lm_loss(h, table, torch.zeros(70, dtype=torch.long, device=dev), reduction="none")
    dh, dt = torch.autograd.grad(each.sum(), (h, table))
    assert not each.any() and not dh.any() and not dt.any()


def test_lost_rows():
    """The label far below the others: p = 0, its term -1, the loss the difference."""
    from smsgate_amd.models import train_ops

    h, table, labels = _rows(50, 300, 128, 0.5, torch.bfloat16, 3)
    away = (labels + 1) % 300
    h.requires_grad_(), table.requires_grad_()
    each = train_ops.lm_loss(h, table, away, reduction="none")
    (dh,) = torch.autograd.grad(each.sum(), h)
    z = h.detach().double() @ table.detach().double().t()
    lse = torch.logsumexp(z, 1)
    at = torch.arange(50, device=dev)
    want = lse - z[at, away]
    assert float((each.detach().double() - want).abs().max()) <= 4 * 2.0 ** -24 * float(want.max())
    d = torch.exp(z - lse[:, None])
    d[at, away] -= 1.0
    assert float((dh.double() - d @ table.detach().double()).norm()) <= 2 * 2.0 ** -8 * float(dh.double().norm())
    assert math.isfinite(float(each.detach().sum()))
