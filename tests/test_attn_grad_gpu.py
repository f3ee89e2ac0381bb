"""Attention of whole sequences and its gradients (ops/csrc/attn_grad_kernels.hip via
models/train_ops.py tiled_attention) against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def _ref(q, k, v, dout, scale, causal, lens):
    """out, dq, dk, dv in 64 bits, by the formulas, one sequence at a time."""
    B, nh, T, D = q.shape
    nkv = k.shape[1]
    rep = nh // nkv
    out = torch.zeros(B, T, nh, D, dtype=torch.float64, device=q.device)
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v))
    for b in range(B):
        n = lens[b]
        if n == 0:
            continue
        for h in range(nh):
            Q, K, V = q[b, h, :n].double(), k[b, h // rep, :n].double(), v[b, h // rep, :n].double()
            s = (Q @ K.t()) * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
            p = torch.softmax(s, -1)
            o = p @ V
            do = dout[b, :n].reshape(n, nh, D)[:, h].double()
            ds = p * (do @ V.t() - (do * o).sum(-1, keepdim=True)) * scale
            out[b, :n, h] = o
            dq[b, h, :n] = ds @ K
            dk[b, h // rep, :n] += ds.t() @ Q
            dv[b, h // rep, :n] += p.t() @ do
    return out.reshape(B, T, nh * D), dq, dk, dv


def _run(q, k, v, dout, scale, causal, lengths):
    from smsgate_amd.models import train_ops

    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = train_ops.tiled_attention(q, k, v, scale, causal=causal, lengths=lengths)
    return (out, *torch.autograd.grad(out, (q, k, v), dout))


def _check(q, k, v, dout, causal, lens, scale=None):
    B, nh, T, D = q.shape
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    got = _run(q, k, v, dout, scale, causal, lengths)
    lens = [T] * B if lens is None else [min(max(n, 0), T) for n in lens]
    want = _ref(q, k, v, dout, D ** -0.5 if scale is None else scale, causal, lens)
    u = U[q.dtype]
    # Relative 2-norms.  A value rounded to the type is off by at most u.  out: P rounded
    # (u), out rounded (u).  dv: P and dv (2 u).  dq, dk: D from the rounded out (its error
    # of up to 2 u |do||o| is at most 2 u of the dP it is taken from in norm), dS rounded
    # (u), result rounded (u): 4 u.  Twice that for the norm of a difference that cancels
    # (dP - D): 8 u.  fp32 sums and exp2 are far below u.
    for name, x, y, tol in zip(("out", "dq", "dk", "dv"), got, want, (2, 8, 8, 2)):
        assert x.shape == y.shape and x.dtype == q.dtype, name
        err, norm = float((x.double() - y).norm()), float(y.norm())
        # one key: P = 1, dP = D up to rounding, dS is rounding alone against |dP| (dq, dk = 0)
        floor = 0.0 if name in ("out", "dv") else float(dout.double().norm() * v.double().norm()) * 4 * u * \
            max(float(q.double().norm()), float(k.double().norm())) / math.sqrt(v.numel()) / math.sqrt(q.numel()) \
            if max(lens) <= 1 else 0.0
        assert err <= tol * u * norm + floor, (name, err / max(norm, 1e-30), tol * u)
    for b, n in enumerate(lens):  # behind the sequence: zeros
        assert not got[0][b, n:].any() and not any(g[b, :, n:].any() for g in got[1:])
    return got


def _inputs(B, T, nh, nkv, D, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g, device=dev).to(dtype)

    return normal(B, nh, T, D), normal(B, nkv, T, D), normal(B, nkv, T, D), normal(B, T, nh * D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,T,nh,nkv", [(1, 1, 4, 2), (2, 2, 3, 1), (3, 31, 2, 2), (2, 33, 9, 3), (2, 64, 4, 1), (1, 65, 6, 3),
                                        (2, 129, 3, 3), (1, 200, 6, 2), (1, 517, 4, 2)])
def test_attention_matches_definition(dtype, D, causal, B, T, nh, nkv):
    """Lengths on both sides of every tile (32 rows a wave, 64 keys a tile, 1 / 2 / 4 waves),
    heads shared or not, joined per query head or not."""
    _check(*_inputs(B, T, nh, nkv, D, dtype, seed=T), causal, None)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,lens", [(61, [61, 1, 0, 40, 32, 33]), (150, [0, 150, 64, 65, 149]), (300, [300, 128, 7]),
                                    (40, [-3, 1000])])
def test_attention_padded_batch(causal, T, lens):
    """Padding holds infinities and NaN; an empty sequence; lengths out of range are clamped."""
    q, k, v, dout = _inputs(len(lens), T, 6, 3, 64, torch.bfloat16, seed=7)
    clean = _check(q, k, v, dout, causal, lens)
    dirty = [t.clone() for t in (q, k, v, dout)]
    for b, n in enumerate(lens):
        n = min(max(n, 0), T)
        for i, x in enumerate((math.nan, math.inf, -math.inf, math.nan)):
            (dirty[i][b, :, n:] if i < 3 else dirty[i][b, n:]).fill_(x)
    got = _run(*dirty, None, causal, torch.tensor(lens, dtype=torch.int32, device=dev))
    for x, y in zip(got, clean):
        assert torch.equal(x, y)


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_attention_peaked_and_flat(scale):
    """Scores of some hundreds (the running maximum rises late, one key takes all) and
    nearly equal ones."""
    q, k, v, dout = _inputs(1, 300, 4, 2, 64, torch.bfloat16, seed=11)
    k = k * torch.linspace(0.1, 4.0, 300, device=dev)[:, None].to(k.dtype)
    _check(q, k, v, dout, True, None, scale)
    _check(q, k, v, dout, False, [257], scale)


def test_attention_small_fp16_gradients():
    """An incoming gradient near fp16's smallest: dS would vanish if it were not scaled.
    The results are 2^-24 grained (subnormal), so they are compared after a rounding of 2^-25."""
    q, k, v, dout = _inputs(1, 260, 4, 2, 64, torch.float16, seed=13)
    dout = (dout.float() * 2.0 ** -12).half()
    got = _run(q, k, v, dout, None, True, None)
    want = _ref(q, k, v, dout, 0.125, True, [260])
    for x, y, tol in zip(got[1:], want[1:], (8, 8, 2)):
        assert float((x.double() - y).norm()) <= tol * 2.0 ** -11 * float(y.norm()) + 2.0 ** -25 * math.sqrt(y.numel())


def test_attention_gradient_against_differences():
    """The directional derivative of sum(out * dout) in q, k and v against central
    differences of the 64-bit definition."""
    q, k, v, dout = _inputs(1, 70, 4, 2, 64, torch.bfloat16, seed=17)
    _, dq, dk, dv = _run(q, k, v, dout, None, True, None)

    def f(a, b, c):
        p = torch.softmax((a @ b.repeat_interleave(2, 1).transpose(-1, -2) * 0.125).masked_fill(
            torch.ones(70, 70, dtype=torch.bool, device=dev).triu(1), -math.inf), -1)
        return ((p @ c.repeat_interleave(2, 1)).transpose(1, 2).reshape(1, 70, 256) * dout.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i, d in enumerate((dq, dk, dv)):
        e = torch.randn(x[i].shape, generator=torch.Generator(device=dev).manual_seed(i), device=dev, dtype=torch.float64)
        hi, lo = [t.clone() for t in x], [t.clone() for t in x]
        hi[i] += 1e-4 * e
        lo[i] -= 1e-4 * e
        want, got = float(f(*hi) - f(*lo)) / 2e-4, float((d.double() * e).sum())
        # each of the N summands is off by at most 8 u of the gradient's norm, in a random direction
        assert abs(got - want) <= 8 * 2.0 ** -8 * float(d.double().norm()) * 4, (i, got, want)


def test_attention_views_and_repeats():
    """Rows of a fused [B, T, heads, D] projection, an odd view that has to be copied, an
    expanded gradient; the same bits on every run."""
    B, T, nh, nkv, D = 2, 150, 6, 2, 64
    g = torch.Generator(device=dev).manual_seed(19)
    qkv = torch.randn(B, T, nh + 2 * nkv, D, generator=g, device=dev).bfloat16()
    q, k, v = (t.transpose(1, 2) for t in qkv.split([nh, nkv, nkv], 2))
    dout = torch.randn(B, T, nh * D, generator=g, device=dev).bfloat16()
    first = _check(q, k, v, dout, True, [150, 77])
    for _ in range(3):
        for x, y in zip(_run(q, k, v, dout, None, True, torch.tensor([150, 77], dtype=torch.int32, device=dev)), first):
            assert torch.equal(x, y)
    odd = torch.randn(B, nh, T, D + 3, generator=g, device=dev).bfloat16()[..., 3:]
    _check(odd, k, v, dout, False, None)
    _check(q, k, v, dout[:1, :1].expand(B, T, nh * D), True, None)
    _check(q, k[:, :1].expand(B, 2, T, D), v[:, :1].expand(B, 2, T, D), dout, True, None)


def test_attention_graph_and_stream():
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(23)
    for dtype, T in ((torch.bfloat16, 61), (torch.float16, 300)):
        q, k, v, dout = (t.requires_grad_(i < 3) for i, t in enumerate(_inputs(2, T, 6, 2, 64, dtype)))
        lengths = torch.tensor([T, T // 2], dtype=torch.int32, device=dev)

        def step(a, b, c):
            o = train_ops.tiled_attention(a, b, c, lengths=lengths)
            return (o, *torch.autograd.grad(o, (a, b, c), dout))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(q, k, v)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(q, k, v)
        for i in range(4):
            with torch.no_grad():
                for t in (q, k, v, dout):
                    t.copy_(torch.randn(t.shape, generator=g, device=dev))
                lengths.copy_(torch.tensor([T - i, 5 * i], dtype=torch.int32))
            want = step(*(t.detach().clone().requires_grad_() for t in (q, k, v)))
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(res, want):
                assert torch.equal(x, y), i


def test_attention_no_grad_and_partial_grad():
    from smsgate_amd.models import train_ops

    q, k, v, dout = _inputs(1, 100, 4, 2, 64, torch.bfloat16)
    with torch.no_grad():
        a = train_ops.tiled_attention(q, k, v)
    b = train_ops.tiled_attention(q.requires_grad_(), k, v)
    assert torch.equal(a, b) and not a.requires_grad
    (dq,) = torch.autograd.grad(b, q, dout)
    assert torch.equal(dq, _run(q, k, v, dout, None, True, None)[1])
