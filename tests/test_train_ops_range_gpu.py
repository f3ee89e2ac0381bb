"""The training operators (models/train_ops.py) with values at the ends of their types' ranges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


def _gen(seed):
    return torch.Generator(device=dev).manual_seed(seed)


def test_attention_of_one_position_off_16_bytes():
    from smsgate_amd.models import train_ops

    base = torch.randn(3, 65, generator=_gen(1), device=dev).bfloat16()
    off = [base[i].view(1, 1, 1, 65)[..., 1:].detach().requires_grad_() for i in range(3)]
    on = [t.detach().clone().requires_grad_() for t in off]
    a, b = train_ops.tiled_attention(*off), train_ops.tiled_attention(*on)
    assert torch.equal(a, b) and torch.equal(a.view(-1), off[2].view(-1))
    g = torch.ones_like(a)
    for x, y in zip(torch.autograd.grad(a, off, g), torch.autograd.grad(b, on, g)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("D", [64, 128])
def test_fp16_scaling_ignores_rows_behind_the_sequence(D):
    """The factor on fp16's dS comes from the rows inside the sequences alone."""
    from smsgate_amd.models import train_ops

    g = _gen(2)
    B, T, nh, nkv = 3, 90, 6, 2
    q, k, v = (torch.randn(B, h, T, D, generator=g, device=dev).half() for h in (nh, nkv, nkv))
    dout = (torch.randn(B, T, nh * D, generator=g, device=dev) * 1e-4).half()
    lens = [90, 37, 0]
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    res = []
    for fill in (0.0, 6e4, math.inf, math.nan):
        x = [t.clone() for t in (q, k, v, dout)]
        for b, n in enumerate(lens):
            x[3][b, n:] = fill
            for t in x[:3]:
                t[b, :, n:] = fill
        leaves = [t.requires_grad_() for t in x[:3]]
        out = train_ops.tiled_attention(*leaves, lengths=lengths)
        res.append((out.detach(), *torch.autograd.grad(out, leaves, x[3])))
    for other in res[1:]:
        for a, b in zip(res[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [2, 50, 200])
def test_fp16_gradients_of_large_values(T):
    """v of 1000 along do: dP of 64000, dS beyond fp16, dq and dk within it."""
    from smsgate_amd.models import train_ops

    g = _gen(3)
    q, k = (0.02 * torch.randn(1, 2, T, 64, generator=g, device=dev) for _ in range(2))
    sign = torch.where(torch.rand(1, 2, T, 1, generator=g, device=dev) < 0.5, -1.0, 1.0)
    sign[:, :, 0], sign[:, :, 1] = -1.0, 1.0
    v = (1000 * sign).expand(1, 2, T, 64).contiguous()
    q, k, v = (t.half().requires_grad_() for t in (q, k, v))
    dout = torch.ones(1, T, 128, device=dev).half()
    out = train_ops.tiled_attention(q, k, v, causal=False)
    got = torch.autograd.grad(out, (q, k, v), dout)
    Q, K, V = (t.detach().double() for t in (q, k, v))
    p = torch.softmax(Q @ K.transpose(-1, -2).contiguous() / 8, -1)
    do = dout.double().view(1, T, 2, 64).transpose(1, 2)
    dp = do @ V.transpose(-1, -2).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / 8
    want = (ds @ K, ds.transpose(-1, -2).contiguous() @ Q, p.transpose(-1, -2).contiguous() @ do)
    # roundings to fp16 of at most u each: dS and the result, and D from the rounded out with
    # what that rounding took (u^2); doubled for the norm of sums of signs
    for x, y in zip(got, want):
        assert torch.isfinite(x).all()
        assert float((x.double() - y).norm()) <= 4 * 2.0 ** -11 * float(y.norm())


@pytest.mark.parametrize("T", [130, 300])
@pytest.mark.parametrize("step", [1, 2])
def test_first_keys_without_weight(T, step):
    """Products of -infinity for a row's first 64 keys: the row is the mean of the others."""
    from smsgate_amd.models import train_ops

    g = _gen(4)
    q, k = (torch.zeros(1, 2, T, 64, device=dev) for _ in range(2))
    q[:, :, ::step, 0] = 3e38
    k[:, :, :64, 0] = -3e38
    v = torch.randn(1, 2, T, 64, generator=g, device=dev).bfloat16()
    out = train_ops.tiled_attention(q.bfloat16(), k.bfloat16(), v, causal=False).view(T, 2, 64).double()
    V = v[0].double()
    some, every = V[:, 64:].mean(1), V.mean(1)
    # P is 1 exactly or 0: out's rounding, and fp32 sums
    for rows, want in ((out[::step], some), (out[1::2][:0 if step == 1 else T], every)):
        if not len(rows):
            continue
        assert float((rows - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())


def test_an_infinite_incoming_gradient_stays_in_its_row():
    from smsgate_amd.models import train_ops

    g = _gen(5)
    h = torch.randn(200, 64, generator=g, device=dev).bfloat16().requires_grad_()
    table = torch.randn(300, 64, generator=g, device=dev).bfloat16()
    labels = torch.randint(0, 300, (200,), generator=g, device=dev)
    labels[7] = -100
    w = torch.rand(200, generator=g, device=dev) + 0.5
    res = []
    for bad in (0.25, math.inf, -math.inf, math.nan):
        w[3], w[7] = bad, bad  # row 7 is ignored: no effect
        each = train_ops.lm_loss(h, table, labels, reduction="none")
        (dh,) = torch.autograd.grad(each, h, w)
        res.append(dh)
    keep = torch.arange(200, device=dev) != 3
    for dh in res[1:]:
        assert torch.equal(dh[keep], res[0][keep]) and not torch.isfinite(dh[3]).all()


def test_logits_at_the_ends_of_fp32():
    """Differences of logits beyond what e^x's argument may be multiplied to."""
    from smsgate_amd.models import train_ops

    h = torch.zeros(3, 8, device=dev)
    h[:, 0] = 1e19
    table = torch.zeros(70, 8, device=dev)
    table[0, 0], table[69, 0] = 3e19, -3e19
    h, table = h.bfloat16().requires_grad_(), table.bfloat16().requires_grad_()
    labels = torch.tensor([0, 5, 69], device=dev)
    each = train_ops.lm_loss(h, table, labels, reduction="none")
    top = float(h[0, 0].double() * table[0, 0].double())
    assert float(each[0]) == 0.0 and abs(float(each[1]) / top - 1) < 1e-6 and float(each[2]) == math.inf
    dh, dt = torch.autograd.grad(each[:2].sum(), (h, table))
    assert not dh[0].any() and float(dh[1, 0]) == float(table[0, 0]) and not dh[2].any()
    assert float(dt[0, 0]) == float(h[0, 0]) and float(dt[5, 0]) == -float(h[0, 0])
