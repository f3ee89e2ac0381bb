"""fp16 gradients of tiled_attention (ops/csrc/attn_grad_kernels.hip): the factor that keeps dS
within the type is a sequence's own."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


def _inputs(B, T, nh, nkv, D, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    q, k, v = (torch.randn(B, h, T, D, generator=g, device=dev).half() for h in (nh, nkv, nkv))
    # an incoming gradient near fp16's smallest: dS is lost if it is not scaled
    return q, k, v, (torch.randn(B, T, nh * D, generator=g, device=dev) * 2.0 ** -12).half()


def _run(q, k, v, dout, causal, lengths=None):
    from smsgate_amd.models import train_ops

    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = train_ops.tiled_attention(*leaves, causal=causal, lengths=lengths)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [20, 61, 200])
@pytest.mark.parametrize("fill", [math.inf, -math.inf, math.nan, 60000.0])
@pytest.mark.parametrize("where", ["dout", "v"])
def test_one_sequence_does_not_move_the_others(D, T, fill, where):
    """An infinity, NaN or an outlier in one sequence: the others' bits stay."""
    B, nh, nkv, bad = 5, 4, 2, 2
    clean = _inputs(B, T, nh, nkv, D, seed=T + D)
    dirty = [t.clone() for t in clean]
    if where == "dout":
        dirty[3][bad, T // 2, 3] = fill
    else:
        dirty[2][bad, 1, T // 2, 5] = fill
    keep = [b for b in range(B) if b != bad]
    for x, y in zip(_run(*clean, True), _run(*dirty, True)):
        assert torch.equal(x[keep], y[keep])


@pytest.mark.parametrize("B", [1, 3, 130, 257])
@pytest.mark.parametrize("causal", [True, False])
def test_a_sequence_is_the_same_alone(B, causal):
    """Batches of every number of blocks a sequence, gradients of very different sizes."""
    T, nh, nkv, D = 70, 2, 1, 64
    q, k, v, dout = _inputs(B, T, nh, nkv, D, seed=B)
    dout = (dout.float() * 2.0 ** (torch.arange(B, device=dev) % 20 - 2)[:, None, None]).half()
    lens = torch.tensor([(T, 33, 1, 0, 65)[b % 5] for b in range(B)], dtype=torch.int32, device=dev)
    many = _run(q, k, v, dout, causal, lens)
    for b in sorted({0, 1, B // 2, B - 1} & set(range(B))):
        one = _run(*(t[b:b + 1] for t in (q, k, v, dout)), causal, lens[b:b + 1])
        for x, y in zip(many, one):
            assert torch.equal(x[b:b + 1], y)


@pytest.mark.parametrize("T", [61, 200])
def test_an_infinite_row_leaves_the_other_rows_of_dq(T):
    """An infinity in one row of the incoming gradient: dq of the other rows is what it was
    (to the roundings of another factor, 2^-11 each of dS and dq, doubled)."""
    q, k, v, dout = _inputs(1, T, 4, 2, 64, seed=9)
    a = _run(q, k, v, dout, True)
    dout[0, 7, :] = math.inf
    b = _run(q, k, v, dout, True)
    rows = [i for i in range(T) if i != 7]
    x, y = a[1][:, :, rows].double(), b[1][:, :, rows].double()
    assert float((x - y).norm()) <= 4 * 2.0 ** -11 * float(x.norm()) + 2.0 ** -25 * math.sqrt(x.numel())
    assert not torch.isfinite(b[1][:, :, 7]).all()
