"""How near tiled_attention (ops/csrc/attn_grad_kernels.hip) comes to what its types allow, in
units of the exact result's own rounding to the type.

Besides the result's rounding (1 by definition) an error may have the roundings of what is
summed: a product's operands, each about 1 where its terms are rounded to the type, 0 where the
kernel keeps what the rounding took (P up to 32 rows, dS up to 64) or where D is taken from the
unrounded output.  They are independent, so they add in quadrature: 1, or about sqrt(2), and
1.1 and 1.6 bound them.  The same bounds are held against an emulation of the roundings on the
CPU, which passes them and fails one when a kept part is left out."""
import math

import pytest
import torch

CASES = [(T, causal, dtype) for T in (20, 32, 50, 64, 200) for causal in (True, False)
         for dtype in (torch.bfloat16, torch.float16)]
HEADS, GROUPS, D = 6, 3, 64


def _inputs(T, dtype, shift, seed):
    """q, k, v and dout, on the CPU in 64 bits, of values that the type holds; ``shift``: a
    common part of v, which P dP - P D takes out again and the roundings of P and o do not."""
    g = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    q, k, v, dout = normal(HEADS, T, D), normal(GROUPS, T, D), normal(GROUPS, T, D) + shift, normal(HEADS, T, D)
    return [t.to(dtype).double() for t in (q, k, v, dout)]


def _exact(q, k, v, dout, causal, dtype=None, drop=()):
    """out, dq, dk, dv by the formulas.  ``dtype``: with the kernel's roundings to it, and those
    that ``drop`` names too."""
    T, scale = q.shape[1], D ** -0.5

    def kept(t, factor=1.0):
        return t if dtype is None else (t * factor).to(dtype).double() / factor

    def fine(t, name, most, factor):
        return t if dtype is None or (T <= most and name not in drop) else kept(t, factor)

    f = (256.0, 64.0) if dtype == torch.float16 else (1.0, 1.0)  # (powers of two that fp16 is given)
    rep = HEADS // GROUPS
    K, V = (t.repeat_interleave(rep, 0) for t in (k, v))
    s = (q @ K.transpose(1, 2)) * scale
    if causal:
        s = s.masked_fill(torch.ones(T, T).triu(1).bool(), -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    total = e.sum(-1, keepdim=True)
    o = fine(e, "P", 32, f[0]) @ V / total
    out = kept(o)
    p = e / total
    ds = p * (dout @ V.transpose(1, 2) - (dout * (out if "o" in drop else o)).sum(-1, keepdim=True))
    ds = fine(ds, "dS", 64, f[1])
    dk, dv = ds.transpose(1, 2) @ q * scale, fine(p, "P", 32, f[0]).transpose(1, 2) @ dout
    return out, kept(ds @ K * scale), *(kept(t.view(GROUPS, rep, T, D).sum(1)) for t in (dk, dv))


def _errors(got, want, dtype):
    """Each result's distance from the exact one, the exact one's own rounding being 1."""
    return [float((x - y).norm() / (y.to(dtype).double() - y).norm()) for x, y in zip(got, want)]


def _bounds(T, shift):
    """out, dq, dk, dv"""
    p, ds = 1.1 if T <= 32 else 1.6, 1.1 if T <= 32 else 1.2 if T <= 64 else 1.6
    if shift and T > 32:  # with P rounded, the common part's share of o's error reaches dP - D
        ds = 5.0          # (2 to 3.1; 8.8 and more from the rounded o)
    return p, ds, ds, p


def _dist(T, causal, dtype, shift, drop=()):
    x = _inputs(T, dtype, shift, seed=T)
    return _errors(_exact(*x, causal, dtype, drop), _exact(*x, causal), dtype)


@pytest.mark.parametrize("T,causal,dtype", CASES)
def test_the_bounds_pass_the_roundings_as_they_are(T, causal, dtype):
    for shift in (0.0, 8.0):
        assert all(e <= b for e, b in zip(_dist(T, causal, dtype, shift), _bounds(T, shift)))


@pytest.mark.parametrize("T,causal,dtype", CASES)
def test_the_bounds_miss_no_part_left_out(T, causal, dtype):
    def fails(shift, *drop):
        return any(e > b for e, b in zip(_dist(T, causal, dtype, shift, drop), _bounds(T, shift)))

    assert fails(8.0, "o")
    assert T > 64 or fails(0.0, "dS")
    assert T > 32 or fails(0.0, "P")


@pytest.mark.gpu
@pytest.mark.parametrize("T,causal,dtype", CASES)
@pytest.mark.parametrize("shift", [0.0, 8.0])
def test_attention_is_as_near_as_its_roundings(T, causal, dtype, shift):
    from smsgate_amd.models import train_ops

    x = _inputs(T, dtype, shift, seed=T)
    q, k, v = (t[None].to("cuda", dtype).requires_grad_() for t in x[:3])
    dout = x[3].transpose(0, 1).reshape(1, T, HEADS * D).to("cuda", dtype)
    out = train_ops.tiled_attention(q, k, v, causal=causal)
    got = [t.detach()[0].double().cpu() for t in (out, *torch.autograd.grad(out, (q, k, v), dout))]
    got[0] = got[0].view(T, HEADS, D).transpose(0, 1)
    err = _errors(got, _exact(*x, causal), dtype)
    assert all(e <= b for e, b in zip(err, _bounds(T, shift))), err
